"""Layer norm (torch_ffi.layer_norm, its forward and backward) against its definition in 64 bits.

The tolerances are bounds worked out from the formulas, value by value, with u = 2^-24: a float32 sum of n terms t_i in
which no value passes through more than k additions is off by at most k u sum |t_i|; k = n / 8 + 16 covers any split of
a row over 8 or more lanes. A result in bfloat16 or float16 adds half a unit in its last place.
"""
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _dtype(name):
    torch = _torch()
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def _half_ulp(v, dtype):
    """Half a unit in the last place of v in dtype (with float16's smallest step below its normal range)."""
    torch = _torch()
    rel, low = {torch.float32: (U, 0.0), torch.bfloat16: (2.0 ** -8, 0.0),
                torch.float16: (2.0 ** -11, 2.0 ** -25)}[dtype]
    return v.abs() * rel + low


def _inputs(rows, cols, dtype, affine, seed=0, offset=0.5):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    x = (rnd(rows, cols) * torch.exp(0.5 * rnd(cols)) + offset * rnd(cols)).to(dtype)
    pt = dtype if affine == "same" else torch.float32
    w, b = (1 + 0.2 * rnd(cols)).to(pt), (0.1 * rnd(cols)).to(pt)
    gy = rnd(rows, cols).to(dtype)
    return x, (w if affine else None), (b if affine else None), gy


def _forward64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1)
    d = x - mean[..., None]
    rstd = ((d * d).mean(-1) + eps).rsqrt()
    y = d * rstd[..., None]
    y = y if w is None else y * w.double()
    return (y if b is None else y + b.double()), mean, rstd


def _check_forward(x, w, b, eps, y, mean, rstd):
    torch = _torch()
    n = x.shape[-1]
    k = n / 8 + 16
    ry, rm, rr = _forward64(x, w, b, eps)
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    assert mean.dtype == rstd.dtype == torch.float32 and mean.shape == rstd.shape == x.shape[:-1]
    xd = x.double()
    em = k * U * xd.abs().mean(-1) + U * rm.abs()  # the mean's error
    assert ((mean.double() - rm).abs() <= em + 1e-40).all()
    er = rr * (k * U + 4 * U + 0.5 * (em * rr) ** 2)  # rstd's: half the variance's relative error, the root's
    assert ((rstd.double() - rr).abs() <= er).all()
    xh = (xd - rm[..., None]) * rr[..., None]
    wv = torch.ones_like(xh) if w is None else w.double().expand_as(xh)
    tol = wv.abs() * (rr[..., None] * (em[..., None] + U * xd.abs()) + xh.abs() * (er / rr)[..., None])
    tol = tol + 4 * U * ((wv * xh).abs() + (0 if b is None else b.double().abs())) + _half_ulp(ry, x.dtype)
    bad = (y.double() - ry).abs() > tol
    worst = float(((y.double() - ry).abs() / tol).max())
    assert not bad.any(), f"{int(bad.sum())} values beyond the bound, by up to {worst:.3g}"


def _check_backward(gy, x, mean, rstd, w, b, gx, gw, gb):
    torch = _torch()
    rows, n = x.reshape(-1, x.shape[-1]).shape
    k, kr = n / 8 + 16, rows / 16 + 320  # (columns: no value passes through more additions than this)
    x2, g2 = x.reshape(rows, n).double(), gy.reshape(rows, n).double()
    m, r = mean.reshape(rows, 1).double(), rstd.reshape(rows, 1).double()
    xh = (x2 - m) * r
    exh = r * U * (x2.abs() + m.abs()) + 3 * U * xh.abs()  # the normalised value's error
    h = g2 if w is None else g2 * w.double()
    c1, c2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    ref = r * (h - c1 - xh * c2)
    e1 = k * U * h.abs().mean(1, keepdim=True)
    e2 = k * U * (h * xh).abs().mean(1, keepdim=True) + (h.abs() * exh).mean(1, keepdim=True)
    tol = r * (e1 + xh.abs() * e2 + exh * c2.abs() + 6 * U * (h.abs() + c1.abs() + (xh * c2).abs()))
    if gx is not None:
        assert gx.dtype == x.dtype and gx.shape == x.shape and gx.is_contiguous()
        bad = (gx.reshape(rows, n).double() - ref).abs() > tol + _half_ulp(ref, x.dtype)
        assert not bad.any(), int(bad.sum())
    if w is None:
        assert gw is None
    else:
        rw = (g2 * xh).sum(0)
        assert gw.dtype == w.dtype and gw.shape == (n,)
        tw = kr * U * (g2 * xh).abs().sum(0) + (g2.abs() * exh).sum(0) + _half_ulp(rw, w.dtype)
        assert ((gw.double() - rw).abs() <= tw).all()
    if b is None:
        assert gb is None
    else:
        rb = g2.sum(0)
        assert gb.dtype == b.dtype and gb.shape == (n,)
        assert ((gb.double() - rb).abs() <= kr * U * g2.abs().sum(0) + _half_ulp(rb, b.dtype)).all()


def _both(x, w, b, gy, eps=1e-5):
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b, eps)
    _check_forward(x, w, b, eps, y, mean, rstd)
    gx, gw, gb = torch_ffi.layer_norm_backward(gy, x, mean, rstd, w, b)
    _check_backward(gy, x, mean, rstd, w, b, gx, gw, gb)
    torch.cuda.synchronize()


# one row and one column, widths around the vector and warp lengths, the policy's widths, wide rows (beyond a block's
# registers and beyond its shared memory), row counts that fill no block and that fill many waves
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", [
    (1, 1), (3, 1), (1, 2), (5, 7), (2, 8), (1, 31), (9, 32), (4, 33), (17, 35), (33, 36), (64, 64), (257, 71),
    (100, 99), (4096, 100), (129, 127), (31, 128), (7, 129), (130, 255), (61, 256), (40, 257), (300, 512), (45, 513),
    (77, 1000), (50, 1001), (20, 1024), (19, 2047), (301, 2048), (6, 4096), (151, 4100), (3, 8191), (160, 8192),
    (2, 16384),
    (2, 16385), (1, 40000), (3, 65537), (1, 300001), (100003, 5), (500, 8192), (331, 8208), (97, 9001), (700, 12000),
    (333, 16384), (40, 20001), (350, 32768), (5, 32769), (3001, 64), (77, 63), (20011, 3),
    (70001, 1), (300_000, 2), (40_000, 9)])
def test_sizes_and_types(rows, cols, dtype):
    x, w, b, gy = _inputs(rows, cols, _dtype(dtype), "f32", seed=rows + cols)
    _both(x, w, b, gy)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("affine", ["", "same", "weight", "bias"])
@pytest.mark.parametrize("rows,cols", [(70, 100), (33, 101), (9, 4096), (600, 512)])
def test_parameter_forms(rows, cols, affine, dtype):
    x, w, b, gy = _inputs(rows, cols, _dtype(dtype), affine and "same")
    _both(x, None if affine == "bias" else w, None if affine == "weight" else b, gy)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad,shift", [(1, 0), (0, 1), (8, 0), (8, 8), (13, 3), (4, 4), (29, 2)])
@pytest.mark.parametrize("cols", [35, 64, 100, 520, 2048, 6000, 9000, 17000])
def test_strided_rows_and_shifted_starts(cols, pad, shift, dtype):
    """x a column slice of a wider buffer, g_y a slice of another: rows that start at any address."""
    torch = _torch()
    rows = 67
    x, w, b, gy = _inputs(rows, cols, _dtype(dtype), "f32", seed=cols + pad)
    wide = torch.full((rows, shift + cols + pad), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, shift:shift + cols] = x
    gwide = torch.full((rows, cols + shift + 2 * pad), float("nan"), dtype=x.dtype, device="cuda")
    gwide[:, pad:pad + cols] = gy
    _both(wide[:, shift:shift + cols], w, b, gwide[:, pad:pad + cols])
    # the parameters at odd addresses, and a dense x that starts at one
    flat = torch.empty(rows * cols + 3, dtype=x.dtype, device="cuda")
    flat[3:] = x.reshape(-1)
    w2, b2 = torch.empty(cols + 1, device="cuda"), torch.empty(cols + 3, device="cuda")
    w2[1:], b2[3:] = w, b
    _both(flat[3:].view(rows, cols), w2[1:], b2[3:], gy)


def test_leading_dimensions_and_shared_rows():
    torch = _torch()
    x, w, b, gy = _inputs(6 * 5 * 4, 36, torch.float32, "f32")
    _both(x.view(6, 5, 4, 36), w, b, gy.view(6, 5, 4, 36))
    _both(x.view(6, 5, 4, 36)[:, :, 1:2], w, b, gy.view(6, 5, 4, 36)[:, :, 2:3])  # rows 4 * 36 apart
    _both(x[0], w, b, gy[0])  # one dimension: 0-d statistics
    _both(x[:1].expand(50, 36), w, b, gy[:50])  # one row in every place (stride 0)


def test_rows_of_one_value_offsets_and_scales():
    """Rows whose variance is 0, a mean far above the spread, and values near the ends of float32's range."""
    torch = _torch()
    x, w, b, gy = _inputs(64, 100, torch.float32, "f32")
    x[3], x[7] = 0.0, -17.25
    _both(x, w, b, gy)
    _both(x + 1.0e4, w, b, gy)
    _both(x * 1.0e-18, w, b, gy)
    _both(x * 1.0e15, w, b, gy)


@pytest.mark.parametrize("eps", [0.0, 1e-12, 1e-3, 1.0])
def test_eps(eps):
    torch = _torch()
    x, w, b, gy = _inputs(40, 129, torch.float32, "f32")
    _both(x, w, b, gy, eps)


def test_nan_and_inf_stay_in_their_rows():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    for cols in (35, 100, 512, 5000):
        x, w, b, gy = _inputs(96, cols, torch.float32, "f32")
        clean = torch_ffi.layer_norm_forward(x, w, b)
        cg = torch_ffi.layer_norm_backward(gy, x, clean[1], clean[2], w, b)[0]
        x[5, 3], x[40, cols - 1], x[77, 0] = float("nan"), float("inf"), float("-inf")
        y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
        gx, gw, gb = torch_ffi.layer_norm_backward(gy, x, mean, rstd, w, b)
        hit = torch.zeros(96, dtype=torch.bool, device="cuda")
        hit[[5, 40, 77]] = True
        assert torch.equal(y[~hit], clean[0][~hit]) and torch.equal(gx[~hit], cg[~hit])
        assert not torch.isfinite(y[hit]).any() and torch.isnan(gx[hit]).all()
        assert torch.isnan(gw).all() and torch.isfinite(gb).all()


@pytest.mark.parametrize("cols", [6001, 8192, 12000, 20001, 40000])
def test_nan_stays_in_its_row_where_a_row_takes_many_warps(cols):
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    x, w, b, gy = _inputs(9, cols, torch.bfloat16, "f32")
    clean = torch_ffi.layer_norm_forward(x, w, b)
    cg = torch_ffi.layer_norm_backward(gy, x, clean[1], clean[2], w, b)[0]
    x[4, cols // 2] = float("nan")
    y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
    gx = torch_ffi.layer_norm_backward(gy, x, mean, rstd, w, b)[0]
    rest = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(gx[rest], cg[rest])
    assert torch.isnan(y[4]).all() and torch.isnan(gx[4]).all()


@pytest.mark.parametrize("cols", [512, 1001])
def test_offsets_beyond_32_bits(cols):
    """More than 2^31 values: the last rows equal those rows alone, bit for bit (a row does not depend on the others),
    and the column sums the sums of the halves', both within this file's bound for column sums."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    rows = 2 ** 31 // cols + 1000
    seed = torch.Generator(device="cuda").manual_seed(cols)
    part = (torch.randn(1 << 16, cols, device="cuda", generator=seed) * 2 + 1).to(torch.bfloat16)
    x = part.repeat(rows // (1 << 16) + 1, 1)[:rows]
    g = x.flip(1) if cols % 2 else x
    w, b = torch.rand(cols, device="cuda"), torch.rand(cols, device="cuda")
    y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
    gx, gw, gb = torch_ffi.layer_norm_backward(g, x, mean, rstd, w, b)
    tail = slice(rows - 777, rows)
    ty, tm, tr = torch_ffi.layer_norm_forward(x[tail].clone(), w, b)
    tgx = torch_ffi.layer_norm_backward(g[tail].clone(), x[tail].clone(), tm, tr, w, b)[0]
    assert torch.equal(y[tail], ty) and torch.equal(mean[tail], tm) and torch.equal(rstd[tail], tr)
    assert torch.equal(gx[tail], tgx)
    half = rows // 2
    parts = [torch_ffi.layer_norm_backward(g[s].clone(), x[s].clone(), mean[s].clone(), rstd[s].clone(), w, b)
             for s in (slice(0, half), slice(half, rows))]
    n = 1 << 16  # (the values repeat after n rows)
    xh = (x[:n].float() - mean[:n, None]) * rstd[:n, None]
    sizes = ((g[:n].float() * xh).abs().sum(0), g[:n].float().abs().sum(0))
    for whole, a, c, size in zip((gw, gb), parts[0][1:], parts[1][1:], sizes):
        bound = 2 * (rows / 16 + 320) * U * size * (rows / n + 1)  # (the whole's and the halves' together)
        assert ((whole - (a + c)).abs() <= bound).all()


def test_no_rows():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    w, b = torch.ones(36, device="cuda"), torch.zeros(36, device="cuda")
    for shape in ((0, 36), (4, 0, 36)):
        x = torch.zeros(shape, device="cuda")
        y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
        assert y.shape == shape and mean.shape == shape[:-1]
        gx, gw, gb = torch_ffi.layer_norm_backward(x, x, mean, rstd, w, b)
        assert gx.shape == shape and not gw.any() and not gb.any()


@pytest.mark.parametrize("rows,cols,dtype", [(37, 36, "f32"), (513, 100, "f32"), (64, 512, "bf16"), (3, 6000, "f32")])
def test_autograd_equals_the_explicit_calls(rows, cols, dtype):
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    x, w, b, gy = _inputs(rows, cols, _dtype(dtype), "f32")
    _, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
    ref = torch_ffi.layer_norm_backward(gy, x, mean, rstd, w, b)
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    y = torch_ffi.layer_norm(xs, ws, bs)
    assert torch.equal(y, torch_ffi.layer_norm(x, w, b))
    y.backward(gy)
    for a, c in zip((xs.grad, ws.grad, bs.grad), ref):
        assert torch.equal(a, c)
    # parts of the inputs alone
    w2 = w.clone().requires_grad_()
    torch_ffi.layer_norm(x, w2, b).backward(gy)
    assert torch.equal(w2.grad, ref[1])
    x2 = x.clone().requires_grad_()
    torch_ffi.layer_norm(x2, w, b).backward(gy)
    assert torch.equal(x2.grad, ref[0])
    # a broadcast cotangent (sum's)
    x3 = x.clone().requires_grad_()
    torch_ffi.layer_norm(x3, w, b).sum().backward()
    one = torch.ones_like(x)
    assert torch.equal(x3.grad, torch_ffi.layer_norm_backward(one, x, mean, rstd, w, b)[0])


@pytest.mark.parametrize("rows,cols", [(16, 5), (64, 100), (8, 1001)])
def test_gradient_against_differences(rows, cols):
    """Along random directions, the kernel's gradients against central differences of the 64-bit definition: step h
    leaves a truncation error of h^2 / 6 of the third derivative (h = 1e-4: below 1e-6 of the value for directions of
    the inputs' own size) and the gradients' float32 error; 1e-4 of the sum of the terms' sizes covers both."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    x, w, b, gy = _inputs(rows, cols, torch.float32, "f32", seed=3)
    _, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
    grads = torch_ffi.layer_norm_backward(gy, x, mean, rstd, w, b)
    g = torch.Generator(device="cuda").manual_seed(9)
    for which in range(3):
        p = [x.double(), w.double(), b.double()]
        d = torch.randn(p[which].shape, device="cuda", generator=g, dtype=torch.float64)
        loss = []
        for s in (1e-4, -1e-4):
            q = [t + s * d if i == which else t for i, t in enumerate(p)]
            loss.append((_forward64(q[0], q[1], q[2], 1e-5)[0] * gy.double()).sum())
        diff = float(loss[0] - loss[1]) / 2e-4
        terms = grads[which].double() * d
        assert abs(float(terms.sum()) - diff) <= 1e-4 * float(terms.abs().sum())


def test_repeats_bit_for_bit_and_on_another_stream():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    x, w, b, gy = _inputs(5000, 512, torch.float32, "f32")
    ref = torch_ffi.layer_norm_forward(x, w, b)
    gref = torch_ffi.layer_norm_backward(gy, x, ref[1], ref[2], w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            out = torch_ffi.layer_norm_forward(x, w, b)
            gout = torch_ffi.layer_norm_backward(gy, x, out[1], out[2], w, b)
    torch.cuda.current_stream().wait_stream(side)
    for a, c in zip(ref + gref, out + gout):
        assert torch.equal(a, c)


def test_captured_and_compiled():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    x, w, b, gy = _inputs(300, 100, torch.float32, "f32")
    torch_ffi.init()

    def run():
        y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
        return (y,) + torch_ffi.layer_norm_backward(gy, x, mean, rstd, w, b)

    ref = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for t in out:
        t.zero_()
    graph.replay()
    for a, c in zip(ref, out):
        assert torch.equal(a, c)

    def loss(x, w, b):
        return torch_ffi.layer_norm(x, w, b)

    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    y = torch.compile(loss, fullgraph=True)(xs, ws, bs)
    y.backward(gy)
    for a, c in zip((y, xs.grad, ws.grad, bs.grad), ref):
        assert torch.equal(a, c)


def test_refusals():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    x, w, b, gy = _inputs(8, 36, torch.float32, "f32")
    y, mean, rstd = torch_ffi.layer_norm_forward(x, w, b)
    for bad in (x.cpu(), x.double(), x.t(), x[:, ::2], torch.zeros((), device="cuda"), torch.zeros(4, 0, device="cuda"),
                x.view(2, 4, 36)[:, ::3].transpose(0, 1), None, torch._neg_view(x)):
        with pytest.raises(TypeError):
            torch_ffi.layer_norm(bad)
    for bad in (w[:35], w.cpu(), w.double(), w.half(), torch.ones(72, device="cuda")[::2], w.view(1, 36)):
        with pytest.raises(TypeError):
            torch_ffi.layer_norm(x, bad)
        with pytest.raises(TypeError):
            torch_ffi.layer_norm(x, None, bad)
    with pytest.raises(TypeError):
        torch_ffi.layer_norm(x.half(), w, b.half())  # two types of parameters
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            torch_ffi.layer_norm(x, w, b, eps)
    for args in ((gy[:7], x, mean, rstd), (gy.half(), x, mean, rstd), (gy, x, mean[:7], rstd),
                 (gy, x, mean, rstd.double()), (gy, x, mean, rstd[:1].expand(8)), (gy.t(), x, mean, rstd)):
        with pytest.raises(TypeError):
            torch_ffi.layer_norm_backward(*args, w, b)
    xs = x.clone().requires_grad_()
    gx, = torch.autograd.grad(torch_ffi.layer_norm(xs, w, b).square().sum(), xs, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        gx.sum().backward()
