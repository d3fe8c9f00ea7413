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
