"""What the training operators say about arguments they cannot take: the reason given is the reason there is. Every call
here is refused on the host."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def test_shared_memory_is_named_as_that():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    flat = torch.randn(100, device="cuda")
    for grads, out in (([flat, flat], None), ([flat[:60], flat[40:]], None), ([flat[:50]], [flat[10:60]]),
                       ([flat[:50], flat[50:]], [flat[50:], flat[:50]]), ([flat[:50], flat[50:51]], [None, flat[3:4]])):
        out = out and [torch.zeros(50, device="cuda") if o is None else o for o in out]
        with pytest.raises(ValueError, match="share memory"):
            torch_ffi.clip_grad_norm(grads, 1.0, out=out)


def test_another_error_of_the_library_is_not_called_shared_memory():
    """cudaErrorInvalidValue for another reason (here: sums at an address that the entry refuses) is a RuntimeError."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    g = torch.randn(8, device="cuda")
    stats = torch.zeros(3, dtype=torch.float64, device="cuda")[1:]  # (8 bytes off the 16 that two doubles want)
    with pytest.raises(RuntimeError, match="nb_g1_grad_scale"):
        torch_ffi._native().grad_clip([g], [g], 1.0, 1e-6, False, stats)
