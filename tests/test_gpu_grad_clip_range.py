"""Clipping where the coefficient is below float32's normal range: gradients close to float32's end, or a small bound. The
tolerances are those of test_gpu_grad_clip.py."""
import pytest

from test_gpu_grad_clip import SHAPES, U, _check_outs, _grads, _reference

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _check(grads, max_norm, zero=False, out=None):
    """The clipped values; the norm is told in float32, infinite where it rounds to that."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    norm, bad, ref = _reference(grads, max_norm, 1e-6, zero)
    n, b = torch_ffi.clip_grad_norm(grads, max_norm, nonfinite="zero" if zero else "keep", out=out)
    told = float(torch.tensor(norm, dtype=torch.float64).float())
    assert float(n) == told or abs(float(n) - norm) <= 5 * U * norm
    assert int(b) == bad
    _check_outs(grads if out is None else out, ref)


@pytest.mark.parametrize("dtypes", [["f32"], ["bf16"], ["f32", "bf16"]])
@pytest.mark.parametrize("shapes", ["one value", "odd", "policy", "long", "three tables"])
@pytest.mark.parametrize("max_norm", [1e-1, 1e-3, 1e-5])
def test_subnormal_coefficients(shapes, dtypes, max_norm):
    """Coefficients of 3e-38 to 1e-44 (three tables: many parts of the list), in place and into float32 tensors."""
    torch = _torch()
    grads = _grads(SHAPES[shapes], dtypes, scale=1e36)
    _check(grads, max_norm, out=[torch.empty(g.shape, device="cuda") for g in grads])
    _check(grads, max_norm)


def test_a_norm_beyond_float32():
    """The squares' root is beyond the largest float32: the norm that is told is infinite, the values are still clipped."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    g = torch.full((10_000,), 3e38, device="cuda")
    norm, bad = torch_ffi.clip_grad_norm([g], 1.0)
    assert float(norm) == float("inf") and int(bad) == 0
    assert ((g.double() - 0.01).abs() <= 0.01 * 8 * U).all()


def test_non_finite_values_zeroed_under_a_subnormal_coefficient():
    torch = _torch()
    grads = _grads(SHAPES["odd"], ["f32"], scale=1e36)
    grads[2][1, 1] = float("nan")
    grads[4][-1] = float("-inf")
    _check(grads, 1e-3, zero=True)
    assert all(torch.isfinite(g).all() for g in grads)


def test_an_infinite_bound():
    """norm + eps <= infinity holds for an infinite norm too: nothing is scaled; a NaN norm scales by NaN."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    inf, nan = float("inf"), float("nan")
    for scale in (1.0, 1e38):
        g = [torch.tensor([1.0 * scale, -inf], device="cuda"), torch.tensor([3.0], device="cuda")]
        norm, bad = torch_ffi.clip_grad_norm(g, inf)
        assert float(norm) == inf and int(bad) == 1
        assert torch.equal(g[0], torch.tensor([1.0 * scale, -inf], device="cuda")) and g[1].tolist() == [3.0]
    g = [torch.tensor([1.0, nan, inf], device="cuda")]
    norm, bad = torch_ffi.clip_grad_norm(g, inf)
    assert torch.isnan(norm) and int(bad) == 2 and torch.isnan(g[0]).all()
    g = [torch.tensor([1.0, nan, inf], device="cuda")]
    torch_ffi.clip_grad_norm(g, inf, nonfinite="zero")
    assert g[0].tolist() == [1.0, 0.0, 0.0]
