"""The checks of layer_norm_checks.py see what they are for: correctly rounded results pass, and results with a planted
mistake do not."""
import pytest
import torch

import layer_norm_checks as checks


def _results(dtype, rows=9, cols=33):
    """Inputs and the results that the definition gives, rounded to the results' types."""
    x, w, b, gy = checks.inputs(rows, cols, dtype, device="cpu")
    y, mean, rstd = checks.forward64(x, w, b, 1e-5)
    forward = [y.to(x.dtype), mean.float(), rstd.float()]
    gx, gw, gb = checks.backward64(gy, x, forward[1], forward[2], w)
    return x, w, b, gy, forward, [gx.to(x.dtype), gw.float(), gb.float()]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_rounded_results_pass(dtype):
    x, w, b, gy, forward, backward = _results(dtype)
    checks.check_forward(x, w, b, 1e-5, *forward)
    checks.check_backward(gy, x, forward[1], forward[2], w, b, *backward)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 7.0])
@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("which", range(3))
def test_a_wrong_value_fails(which, whole, value):
    """One value, or all of them, of any of the results: NaN, an infinity or another number."""
    x, w, b, gy, forward, backward = _results("f32")
    at = slice(None) if whole else 5
    for good, check in ((forward, lambda r: checks.check_forward(x, w, b, 1e-5, *r)),
                        (backward, lambda r: checks.check_backward(gy, x, forward[1], forward[2], w, b, *r))):
        wrong = [t.clone() for t in good]
        wrong[which].view(-1)[at] = value
        with pytest.raises(AssertionError):
            check(wrong)


@pytest.mark.parametrize("rows,cols", [(1000, 7), (100003, 5)])
def test_column_sums_that_miss_one_row_fail(rows, cols):
    """The sums of all rows pass; those without one row, with one row twice, or with a NaN do not."""
    gy, x, mean, rstd = checks.exact_sums_inputs(rows, cols, "f32", device="cpu")
    terms = gy * (x - mean[:, None]) * rstd[:, None]
    gw, gb = terms.sum(0, dtype=torch.float64).float(), gy.sum(0, dtype=torch.float64).float()
    checks.check_exact_sums(gy, x, mean, rstd, gw, gb)
    for row in (0, rows // 2, rows - 1):
        for sign in (-1, 1):
            with pytest.raises(AssertionError):
                checks.check_exact_sums(gy, x, mean, rstd, gw, gb + sign * gy[row])
            with pytest.raises(AssertionError):
                checks.check_exact_sums(gy, x, mean, rstd, gw + sign * (terms[row] + terms[row - 1]) + gy[row], gb)
    with pytest.raises(AssertionError):
        checks.check_exact_sums(gy, x, mean, rstd, gw * float("nan"), gb)
