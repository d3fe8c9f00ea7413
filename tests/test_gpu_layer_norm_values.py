"""Every value of layer norm's results (torch_ffi.layer_norm_forward and _backward) against the definition in 64 bits,
by checks that a NaN fails: every kernel's widths, the parameters' forms, and rows between poisoned neighbours."""
import pytest

import layer_norm_checks as checks

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _check(x, w, b, gy, eps=1e-5):
    _torch()
    from nablaengine_b200 import torch_ffi
    y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b, eps)
    checks.check_forward(x, w, b, eps, y, mean, rstd)
    checks.check_backward(gy, x, mean, rstd, w, b, *torch_ffi.layer_norm_backward(gy, x, mean, rstd, w, b))


# widths of every spread of a row over lanes, odd ones among them: inside a warp, over several, split over a cluster,
# and beyond what is held in registers; row counts that fill no block and that fill many
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [
    (1, 1), (1, 2), (5, 7), (9, 32), (17, 35), (64, 64), (257, 71), (4096, 100), (31, 128), (130, 255), (61, 256),
    (300, 512), (45, 513), (50, 1001), (20, 1024), (301, 2048), (19, 2047), (151, 4100), (6, 4096), (3, 8191),
    (160, 8192), (331, 8208), (97, 9001), (70, 12000), (33, 16384), (40, 20001), (35, 32768), (5, 32769), (3, 65537),
    (100003, 5), (70001, 1), (40000, 9)])
def test_sizes_and_types(rows, cols, dtype):
    x, w, b, gy = checks.inputs(rows, cols, dtype, seed=rows + cols)
    _check(x, w, b, gy)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("affine", ["", "same", "weight", "bias"])
@pytest.mark.parametrize("rows,cols", [(70, 100), (33, 101), (9, 4096), (5, 9000)])
def test_parameter_forms(rows, cols, affine, dtype):
    x, w, b, gy = checks.inputs(rows, cols, dtype, affine and "same")
    _check(x, None if affine == "bias" else w, None if affine == "weight" else b, gy)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("pad,shift", [(1, 0), (0, 1), (8, 8), (13, 3), (29, 2)])
@pytest.mark.parametrize("cols", [1, 35, 64, 100, 520, 1001, 2048, 6000, 9000, 17000, 33000])
def test_rows_between_poisoned_neighbours(cols, pad, shift, dtype):
    """x and g_y column slices of wider buffers of NaN, and a dense x inside one: what lies beside a row stays out."""
    torch = _torch()
    rows = 67
    x, w, b, gy = checks.inputs(rows, cols, dtype, seed=cols + pad)
    wide = torch.full((rows, shift + cols + pad), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, shift:shift + cols] = x
    gwide = torch.full((rows, cols + shift + 2 * pad), float("nan"), dtype=x.dtype, device="cuda")
    gwide[:, pad:pad + cols] = gy
    _check(wide[:, shift:shift + cols], w, b, gwide[:, pad:pad + cols])
    flat = torch.full((rows * cols + 3 + 61,), float("nan"), dtype=x.dtype, device="cuda")
    flat[3:3 + rows * cols] = x.reshape(-1)
    params = torch.full((2, cols + 4), float("nan"), device="cuda")
    params[0, 1:1 + cols], params[1, 3:3 + cols] = w, b
    _check(flat[3:3 + rows * cols].view(rows, cols), params[0, 1:1 + cols], params[1, 3:3 + cols], gy)


@pytest.mark.parametrize("eps", [0.0, 1e-12, 1e-3, 1.0])
def test_eps(eps):
    x, w, b, gy = checks.inputs(40, 129, "f32")
    _check(x, w, b, gy, eps)


def test_offsets_scales_and_rows_of_one_value():
    x, w, b, gy = checks.inputs(64, 100, "f32")
    x[3], x[7] = 0.0, -17.25
    for other in (x, x + 1.0e4, x * 1.0e-18, x * 1.0e15):
        _check(other, w, b, gy)


def _check_sums(rows, cols, dtype):
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    gy, x, mean, rstd = checks.exact_sums_inputs(rows, cols, dtype, seed=rows + cols)
    one = torch.ones(cols, device="cuda")
    _, gw, gb = torch_ffi.layer_norm_backward(gy, x, mean, rstd, one, one)
    checks.check_exact_sums(gy, x, mean, rstd, gw, gb)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [
    (1, 100), (2, 33), (100003, 5), (300_000, 2), (70001, 1), (40_000, 9), (262_143, 64), (131_073, 100), (20011, 3),
    (5000, 1001), (4099, 512), (1023, 4100), (301, 8192), (333, 8208), (777, 12000), (333, 16384), (350, 32768),
    (70, 32769), (129, 40001)])
def test_column_sums_take_every_row_once(rows, cols, dtype):
    _check_sums(rows, cols, dtype)


@pytest.mark.parametrize("cols", [512, 1001])
def test_column_sums_take_every_row_beyond_32_bits(cols):
    """More than 2^31 values, and rows on either side of that offset."""
    _check_sums(2 ** 31 // cols + 1000, cols, "bf16")


@pytest.mark.parametrize("cols", [100, 5000, 20001, 40000])
def test_beyond_float32s_squares(cols):
    """The stated limit of the float32 sums: where the squared deviations' sum is infinite, rstd is 0 and y the bias."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    x, w, b, _ = checks.inputs(4, cols, "f32")
    x[1] *= 1e25
    y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
    assert float(rstd[1]) == 0.0 and torch.equal(y[1], b) and torch.isfinite(mean).all()
    rest = [0, 2, 3]
    checks.check_forward(x[rest], w, b, 1e-5, y[rest], mean[rest], rstd[rest])
