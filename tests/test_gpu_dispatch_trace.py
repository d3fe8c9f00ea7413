"""A trace of the calls on real tensors (make_fx), run on other inputs, gives those inputs' results; and a dispatch mode
that only looks on changes nothing."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def test_layer_norm_and_its_gradient():
    torch = _torch()
    from torch.fx.experimental.proxy_tensor import make_fx
    from nablaengine_b200 import torch_ffi

    def run(x, w, b):
        y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
        xs = x.detach().requires_grad_()
        z = torch_ffi.layer_norm(xs, w, b)
        return (y, mean, rstd, z.detach(), torch.autograd.grad(z.square().sum(), xs)[0],
                *torch_ffi.layer_norm_backward(y, x, mean, rstd, w, b))

    inputs = [(torch.randn(30, 36, device="cuda"), torch.rand(36, device="cuda"), torch.rand(36, device="cuda"))
              for _ in range(2)]
    fx = make_fx(run)(*inputs[0])
    for args in inputs:
        for a, c in zip(fx(*args), run(*args)):
            assert torch.equal(a, c)


def test_the_step():
    torch = _torch()
    from torch.fx.experimental.proxy_tensor import make_fx
    from nablaengine_b200 import synthetic, torch_ffi
    states = []
    for seed in (0, 1):
        s = {k: torch.from_numpy(v).cuda() for k, v in synthetic.states(8, seed).items()}
        states.append([s[k] for k in ("qpos", "qvel", "warm", "ctrl", "friction", "com")])
    fx = make_fx(lambda *a: torch_ffi.step(*a))(*states[0])
    for state in states:
        for a, c in zip(fx(*state), torch_ffi.step(*state)):
            assert torch.equal(a, c)


def test_a_mode_that_looks_on():
    torch = _torch()
    from torch.utils._python_dispatch import TorchDispatchMode
    from nablaengine_b200 import torch_ffi

    class Seen(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    x, w = torch.randn(30, 36, device="cuda"), torch.rand(36, device="cuda")
    want = torch_ffi.layer_norm_forward(x, w)
    g = [torch.randn(100, device="cuda")]
    clipped = [g[0].clone()]
    norm = torch_ffi.clip_grad_norm(clipped, 1.0)
    with Seen():
        got = torch_ffi.layer_norm_forward(x, w)
        norm2 = torch_ffi.clip_grad_norm(g, 1.0)
    assert any("nabla_b200.layer_norm" in n for n in Seen.names)
    assert all(torch.equal(a, c) for a, c in zip((*got, *norm2, *g), (*want, *norm, *clipped)))


def test_clipping_inside_a_compiled_function():
    """torch.compile leaves its graph for the call: other inputs of the compiled function get their own results."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    torch_ffi.init()

    def run(g):
        g = g * 2.0
        norm, bad = torch_ffi.clip_grad_norm([g], 1.0)
        return g + 1.0, norm, bad

    compiled = torch.compile(run)
    for _ in range(3):
        g = torch.randn(1000, device="cuda")
        for a, c in zip(compiled(g), run(g)):
            assert torch.allclose(a, c, rtol=1e-6, atol=1e-6)
