"""Calls under a torch dispatch mode (make_fx's trace, a FakeTensorMode) go through their custom ops, so a trace holds the
call and not one call's result. Without a GPU the trace runs on fake tensors."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from nablaengine_b200 import synthetic, torch_ffi


def _targets(graph):
    return [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]


def test_layer_norm_is_an_operation_of_the_trace():
    x, w, b = torch.randn(4, 6), torch.ones(6), torch.zeros(6)
    fx = make_fx(lambda *a: torch_ffi.layer_norm(*a), tracing_mode="fake")(x, w, b)
    assert any("nabla_b200.layer_norm" in t for t in _targets(fx))
    stat = torch.ones(4)
    fx = make_fx(lambda *a: torch_ffi.layer_norm_backward(*a), tracing_mode="fake")(x, x, stat, stat, w, b)
    assert any("nabla_b200.layer_norm_backward" in t for t in _targets(fx))


def test_its_gradient_is_too():
    def grad(x, w, b):
        x = x.detach().requires_grad_()
        return torch.autograd.grad(torch_ffi.layer_norm(x, w, b).square().sum(), x)[0]

    fx = make_fx(grad, tracing_mode="fake")(torch.randn(4, 6), torch.ones(6), torch.zeros(6))
    targets = _targets(fx)
    assert any("nabla_b200.layer_norm." in t for t in targets)
    assert any("nabla_b200.layer_norm_backward" in t for t in targets)


def test_the_step_is_too():
    s = {k: torch.from_numpy(v) for k, v in synthetic.states(2, 0).items()}
    state = [s[k] for k in ("qpos", "qvel", "warm", "ctrl", "friction", "com")]
    for call in (torch_ffi.step, torch_ffi.forward):
        fx = make_fx(lambda *a: call(*a), tracing_mode="fake")(*state)
        assert any("nabla_b200.forward" in t for t in _targets(fx))


def test_the_gradient_calls_say_that_they_cannot_be_traced():
    """They write in place and have no operation that a trace could hold."""
    for call in (lambda g: torch_ffi.grad_norm([g])[0], lambda g: torch_ffi.clip_grad_norm([g], 1.0)[0]):
        for mode in ("real", "fake"):
            with pytest.raises(NotImplementedError, match="traced"):
                make_fx(call, tracing_mode=mode)(torch.randn(5))
