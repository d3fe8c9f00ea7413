"""Forward-mode derivatives (torch.autograd.forward_ad, torch.func.jvp) are refused, not dropped: a tensor that carries a
tangent would come back without one, a derivative of zero."""
import pytest
import torch
from torch.autograd import forward_ad

from nablaengine_b200 import synthetic, torch_ffi


def _state():
    s = {k: torch.from_numpy(v) for k, v in synthetic.states(2, 0).items()}
    return [s[k] for k in ("qpos", "qvel", "warm", "ctrl", "friction", "com")]


def _calls(dual):
    """Every differentiable call, and the training operators', with `dual` made of the tensor that is looked at first."""
    x, stat = torch.randn(4, 6), torch.ones(4)
    yield lambda: torch_ffi.layer_norm(dual(x))
    yield lambda: torch_ffi.layer_norm_forward(dual(x))
    yield lambda: torch_ffi.layer_norm_backward(x, dual(x), stat, stat)
    yield lambda: torch_ffi.grad_norm([dual(x), x])
    yield lambda: torch_ffi.clip_grad_norm([dual(x)], 1.0)
    for k in (0, 1, 3):
        state = _state()
        state[k] = dual(state[k])
        yield lambda state=state: torch_ffi.step(*state)
    state = _state()
    yield lambda: torch_ffi.kinematics(dual(state[0]), state[1], state[5])


@pytest.mark.parametrize("requires_grad", [False, True])
def test_a_tangent_is_refused(requires_grad):
    with forward_ad.dual_level():
        for call in _calls(lambda t: forward_ad.make_dual(t.clone().requires_grad_(requires_grad), torch.ones_like(t))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_without_a_tangent_nothing_is_refused_for_it():
    """CPU tensors are, as ever (TypeError), inside a dual level too."""
    with forward_ad.dual_level():
        for call in _calls(lambda t: t):
            with pytest.raises(TypeError):
                call()


def test_jvp_is_refused():
    q, v, w, u, f, c = _state()
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda u: torch_ffi.step(q, v, w, u, f, c)[1], (u,), (torch.ones_like(u),))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda q: torch_ffi.kinematics(q, v, c)[1], (q,), (torch.ones_like(q),))
