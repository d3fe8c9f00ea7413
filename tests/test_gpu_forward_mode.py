"""Forward-mode derivatives of the training operators on the GPU are refused, in every form in which they are asked for."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.mark.parametrize("requires_grad", [False, True])
def test_tangents_are_refused(requires_grad):
    torch = _torch()
    from torch.autograd import forward_ad
    from nablaengine_b200 import torch_ffi
    x, w = torch.randn(8, 36, device="cuda"), torch.ones(36, device="cuda")
    y, mean, rstd = torch_ffi.layer_norm_forward(x, w)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.clone().requires_grad_(requires_grad), torch.ones_like(t))

        for call in (lambda: torch_ffi.layer_norm(dual(x), w), lambda: torch_ffi.layer_norm(x, dual(w)),
                     lambda: torch_ffi.layer_norm(x, w, dual(w)), lambda: torch_ffi.layer_norm_forward(dual(x)),
                     lambda: torch_ffi.layer_norm_backward(dual(y), x, mean, rstd, w),
                     lambda: torch_ffi.layer_norm_backward(y, x, mean, dual(rstd), w),
                     lambda: torch_ffi.grad_norm([x, dual(w)]), lambda: torch_ffi.clip_grad_norm([dual(x)], 1.0),
                     lambda: torch_ffi.clip_grad_norm([x], 1.0, out=[dual(x)])):
            with pytest.raises(NotImplementedError):
                call()
        # tensors without a tangent are taken, here too
        assert torch.equal(torch_ffi.layer_norm(x, w), y)


def test_functional_transforms_are_refused():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    x, w = torch.randn(8, 36, device="cuda"), torch.ones(36, device="cuda")
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: torch_ffi.layer_norm(t, w), (x,), (torch.ones_like(x),))
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: torch_ffi.grad_norm([t])[0], (x,), (torch.ones_like(x),))
