"""Checks of layer norm results against the definition in 64 bits, for tests on the CPU and on the GPU.

The bounds are worked out from the formulas, value by value, with u = 2^-24: a float32 sum of n terms t_i in which no
value passes through more than k additions is off by at most k u sum |t_i|; k = n / 8 + 16 covers any split of a row over
8 or more lanes. A result in bfloat16 or float16 adds half a unit in its last place. Every comparison is written so that
a NaN fails it.
"""
import torch

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_ulp(v, dtype):
    """Half a unit in the last place of v in dtype (with float16's smallest step below its normal range)."""
    rel, low = {torch.float32: (U, 0.0), torch.bfloat16: (2.0 ** -8, 0.0),
                torch.float16: (2.0 ** -11, 2.0 ** -25)}[dtype]
    return v.abs() * rel + low


def within(name, got, want, tol):
    """Every value of `got` within `tol` of `want` (a NaN on either side is not)."""
    ok = (got.double() - want).abs() <= tol
    assert ok.all(), f"{name}: {int((~ok).sum())} of {ok.numel()} values beyond their bound"


def inputs(rows, cols, dtype, affine="f32", seed=0, device="cuda"):
    """x, weight, bias (None where `affine` is empty, of x's type where it is "same") and the cotangent."""
    g = torch.Generator(device=device).manual_seed(seed)

    def rnd(*s):
        return torch.randn(s, device=device, generator=g)

    dtype = DTYPES[dtype]
    x = (rnd(rows, cols) * torch.exp(0.5 * rnd(cols)) + 0.5 * rnd(cols)).to(dtype)
    kind = dtype if affine == "same" else torch.float32
    w, b = (1 + 0.2 * rnd(cols)).to(kind), (0.1 * rnd(cols)).to(kind)
    return x, (w if affine else None), (b if affine else None), rnd(rows, cols).to(dtype)


def forward64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1)
    d = x - mean[..., None]
    rstd = ((d * d).mean(-1) + eps).rsqrt()
    y = d * rstd[..., None]
    y = y if w is None else y * w.double()
    return (y if b is None else y + b.double()), mean, rstd


def backward64(gy, x, mean, rstd, w):
    """(g_x, g_weight, g_bias) from the given statistics."""
    rows, n = x.reshape(-1, x.shape[-1]).shape
    x, g = x.reshape(rows, n).double(), gy.reshape(rows, n).double()
    r = rstd.reshape(rows, 1).double()
    xh = (x - mean.reshape(rows, 1).double()) * r
    h = g if w is None else g * w.double()
    gx = r * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
    return gx, (g * xh).sum(0), g.sum(0)


def check_forward(x, w, b, eps, y, mean, rstd):
    k = x.shape[-1] / 8 + 16
    ry, rm, rr = forward64(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    assert mean.dtype == rstd.dtype == torch.float32 and mean.shape == rstd.shape == x.shape[:-1]
    xd = x.double()
    em = k * U * xd.abs().mean(-1) + U * rm.abs()  # the mean's error
    within("mean", mean, rm, em + 1e-40)
    er = rr * (k * U + 4 * U + 0.5 * (em * rr) ** 2)  # rstd's: half the variance's relative error, the root's
    within("rstd", rstd, rr, er)
    xh = (xd - rm[..., None]) * rr[..., None]
    wv = torch.ones_like(xh) if w is None else w.double().expand_as(xh)
    tol = wv.abs() * (rr[..., None] * (em[..., None] + U * xd.abs()) + xh.abs() * (er / rr)[..., None])
    tol = tol + 4 * U * ((wv * xh).abs() + (0 if b is None else b.double().abs())) + half_ulp(ry, x.dtype)
    within("y", y, ry, tol)


def check_backward(gy, x, mean, rstd, w, b, gx, gw, gb):
    rows, n = x.reshape(-1, x.shape[-1]).shape
    k, kr = n / 8 + 16, rows / 16 + 320  # (columns: no value passes through more additions than this)
    x2, g2 = x.reshape(rows, n).double(), gy.reshape(rows, n).double()
    m, r = mean.reshape(rows, 1).double(), rstd.reshape(rows, 1).double()
    xh = (x2 - m) * r
    exh = r * U * (x2.abs() + m.abs()) + 3 * U * xh.abs()  # the normalised value's error
    h = g2 if w is None else g2 * w.double()
    c1, c2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    rx, rw, rb = backward64(gy, x, mean, rstd, w)
    e1 = k * U * h.abs().mean(1, keepdim=True)
    e2 = k * U * (h * xh).abs().mean(1, keepdim=True) + (h.abs() * exh).mean(1, keepdim=True)
    tol = r * (e1 + xh.abs() * e2 + exh * c2.abs() + 6 * U * (h.abs() + c1.abs() + (xh * c2).abs()))
    assert gx.dtype == x.dtype and gx.shape == x.shape and gx.is_contiguous()
    within("g_x", gx.reshape(rows, n), rx, tol + half_ulp(rx, x.dtype))
    assert (gw is None) == (w is None) and (gb is None) == (b is None)
    if w is not None:
        assert gw.dtype == w.dtype and gw.shape == (n,)
        within("g_weight", gw, rw,
               kr * U * (g2 * xh).abs().sum(0) + (g2.abs() * exh).sum(0) + half_ulp(rw, w.dtype))
    if b is not None:
        assert gb.dtype == b.dtype and gb.shape == (n,)
        within("g_bias", gb, rb, kr * U * g2.abs().sum(0) + half_ulp(rb, b.dtype))


def exact_sums_inputs(rows, cols, dtype, seed=0, device="cuda"):
    """(g_y, x, mean, rstd) whose column sums float32 holds exactly in any order: g_y is 1 or -1 everywhere, so that every
    row counts in every column, and (x - mean) rstd is a whole number of at most 3 (3 rows < 2^24)."""
    assert 3 * rows < 2 ** 24
    g = torch.Generator(device=device).manual_seed(seed)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi + 1, shape, dtype=torch.int8, device=device, generator=g)

    gy = whole(0, 1, rows, cols).mul_(2).sub_(1).to(DTYPES[dtype])
    x = whole(-2, 2, rows, cols).to(DTYPES[dtype])
    return gy, x, whole(0, 1, rows).float(), torch.ones(rows, device=device)


def check_exact_sums(gy, x, mean, rstd, gw, gb):
    """g_weight and g_bias of exact_sums_inputs, to the last bit: a row left out, taken twice or read from another place
    shows."""
    rows = x.shape[0]
    want = torch.zeros((2, x.shape[1]), dtype=torch.int64, device=x.device)
    step = max(1, (1 << 25) // x.shape[1])
    for r in range(0, rows, step):
        s = slice(r, min(r + step, rows))
        g = gy[s].to(torch.int8)
        xh = ((x[s].float() - mean[s, None]) * rstd[s, None]).to(torch.int8)
        want[0] += (g * xh).sum(0, dtype=torch.int64)
        want[1] += g.sum(0, dtype=torch.int64)
    for name, got, sums in (("g_weight", gw, want[0]), ("g_bias", gb, want[1])):
        assert got.dtype == torch.float32 and got.shape == sums.shape
        wrong = got.double() != sums.double()
        assert not wrong.any(), f"{name}: {int(wrong.sum())} of {wrong.numel()} columns"
