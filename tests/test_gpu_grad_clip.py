"""The global gradient norm and clipping (torch_ffi.grad_norm, clip_grad_norm) against their definition in 64 bits.

Tolerances, with u = 2^-24: the sum of squares is held in 64 bits, over groups of at most 8 squares summed in float32
(off by at most 8 u), so the norm is off by at most 4 u and its own rounding; the coefficient likewise, and a clipped
value by one product more: 8 u of its size, and half a unit in the last place of a 16-bit output.
"""
import math

import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _torch():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _grads(shapes, dtypes, seed=0, scale=1.0):
    torch = _torch()
    g = torch.Generator(device="cuda").manual_seed(seed)
    types = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
    return [(torch.randn(s, device="cuda", generator=g) * scale * (1 + k % 3)).to(types[dtypes[k % len(dtypes)]])
            for k, s in enumerate(shapes)]


def _reference(grads, max_norm, eps, zero):
    """(norm, bad, clipped tensors) in 64 bits."""
    torch = _torch()
    vals = [g.double() for g in grads]
    bad = sum(int((~torch.isfinite(v)).sum()) for v in vals)
    if zero:
        vals = [torch.where(torch.isfinite(v), v, 0.0) for v in vals]
    norm = math.sqrt(math.fsum(float((v * v).sum()) for v in vals))
    c = 1.0 if norm + eps <= max_norm else max_norm / (norm + eps)
    return norm, bad, [v * c for v in vals]


def _check_outs(outs, ref):
    torch = _torch()
    for o, r in zip(outs, ref):
        rel, low = {torch.float32: (0.0, 2.0 ** -150), torch.bfloat16: (2.0 ** -8, 2.0 ** -134),
                    torch.float16: (2.0 ** -11, 2.0 ** -25)}[o.dtype]
        assert ((o.double() - r).abs() <= r.abs() * (8 * U + rel) + low).all()


def _check(grads, max_norm, eps=1e-6, zero=False, out=None):
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    mode = "zero" if zero else "keep"
    norm, bad, ref = _reference(grads, max_norm, eps, zero)
    n1, b1 = torch_ffi.grad_norm(grads, nonfinite=mode)
    kept = [g.clone() for g in grads]
    outs = grads if out is None else out
    n2, b2 = torch_ffi.clip_grad_norm(grads, max_norm, eps=eps, nonfinite=mode, out=out)
    for n, b in ((n1, b1), (n2, b2)):
        assert n.dtype == torch.float32 and b.dtype == torch.int64 and n.dim() == b.dim() == 0
        assert abs(float(n) - norm) <= 5 * U * norm + 2.0 ** -150 and int(b) == bad  # (2^-150: half the last subnormal)
    _check_outs(outs, ref)
    if out is not None:
        assert all(torch.equal(g.nan_to_num(7.0), k.nan_to_num(7.0)) for g, k in zip(grads, kept))
    return norm


SHAPES = {
    "one value": [(1,)], "one": [(1000,)], "odd": [(1,), (7,), (33, 5), (8191,), (8192,), (8193,), (3, 3, 3)],
    "policy": [(100,), (100,), (128, 100), (128,), (128,), (29, 128), (29,)], "empty ones": [(0,), (5,), (0, 4), (6,)],
    "many": [(k % 37 + 1,) for k in range(500)], "long": [(3_000_001,), (17,), (1_000_000,)],
    "ctrl": [(8, 4096, 29)], "last of one launch": [(524_287,), (1,)], "first of two": [(524_288,), (1,)],
    "one table": [(k % 50 + 1,) for k in range(96)], "a tensor more": [(k % 50 + 1,) for k in range(97)],
    "three tables": [(k % 9 * 100 + 1,) for k in range(2000)],
}


@pytest.mark.parametrize("dtypes", [["f32"], ["bf16"], ["f16"], ["f32", "bf16", "f16"]])
@pytest.mark.parametrize("shapes", SHAPES)
def test_shapes_and_types(shapes, dtypes):
    for max_norm in (0.5, 1e9, 0.0):
        _check(_grads(SHAPES[shapes], dtypes), max_norm)


@pytest.mark.parametrize("dtypes", [["f32"], ["bf16"], ["f16", "bf16", "f32"]])
@pytest.mark.parametrize("wide", [False, True])
def test_into_other_tensors(dtypes, wide):
    torch = _torch()
    for shapes in ("odd", "many", "long"):
        grads = _grads(SHAPES[shapes], dtypes)
        for max_norm in (2.0, 1e9):
            out = [torch.full(g.shape, float("nan"), dtype=torch.float32 if wide else g.dtype, device="cuda")
                   for g in grads]
            _check(grads, max_norm, out=out)


def test_no_gradients():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    for grads in ([], [torch.zeros(0, device="cuda")], [torch.zeros(5, device="cuda")]):
        for norm, bad in (torch_ffi.grad_norm(grads), torch_ffi.clip_grad_norm(grads, 1.0),
                          torch_ffi.clip_grad_norm(grads, 0.0, eps=0.0)):
            assert float(norm) == 0.0 and int(bad) == 0
        assert all(not g.any() for g in grads)


@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e-42])
def test_squares_beyond_float32(scale):
    """Gradients whose squares overflow or underflow float32: the sum of squares is held in 64 bits."""
    torch = _torch()
    grads = _grads(SHAPES["odd"], ["f32"], scale=scale)
    assert _check(grads, 0.1 * scale, eps=0.0) > 0
    mixed = _grads([(100,)], ["f32"], scale=1e-30) + _grads([(50_000,)], ["bf16"], scale=1e25)
    _check(mixed, 1e9)
    sparse = [torch.zeros(10_000, device="cuda")]
    sparse[0][7777] = 1e-25  # alone among zeros
    _check(sparse, 1.0)


@pytest.mark.parametrize("shapes", ["odd", "policy", "long", "many"])
@pytest.mark.parametrize("dtypes", [["f32"], ["f16", "bf16"]])
def test_nonfinite_zeroed(shapes, dtypes):
    torch = _torch()
    grads = _grads(SHAPES[shapes], dtypes)
    for k, v in enumerate((float("nan"), float("inf"), float("-inf"))):
        g = grads[k % len(grads)]
        g.view(-1)[(k * 31) % g.numel()] = v
        g.view(-1)[-1] = v
    grads[-1].view(-1)[0] = float("nan")
    _check(grads, 0.25, zero=True)
    assert all(torch.isfinite(g).all() for g in grads)
    all_bad = [torch.full((777,), float("nan"), device="cuda")]
    assert _check(all_bad, 1.0, zero=True) == 0.0 and not all_bad[0].any()


def test_nonfinite_kept():
    """As the arithmetic has it: an infinite norm scales by 0, a NaN norm by NaN; a bound of infinity scales nothing."""
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    inf, nan = float("inf"), float("nan")
    g = [torch.tensor([1.0, inf, -2.0], device="cuda"), torch.tensor([3.0], device="cuda")]
    norm, bad = torch_ffi.clip_grad_norm(g, 1.0)
    assert float(norm) == inf and int(bad) == 1
    assert g[0].tolist()[0] == 0.0 and math.isnan(g[0].tolist()[1]) and g[1].tolist() == [0.0]
    g = [torch.tensor([1.0, nan], device="cuda"), torch.tensor([3.0], device="cuda")]
    norm, bad = torch_ffi.clip_grad_norm(g, 1.0)
    assert math.isnan(float(norm)) and int(bad) == 1 and all(torch.isnan(t).all() for t in g)
    g = _grads(SHAPES["odd"], ["f32"])
    kept = [t.clone() for t in g]
    torch_ffi.clip_grad_norm(g, inf)
    assert all(torch.equal(a, c) for a, c in zip(g, kept))


def test_layouts_and_addresses():
    """Transposed gradients, slices of one buffer that start at odd addresses, and the values between them kept."""
    torch = _torch()
    base = torch.randn(6, 40, 50, device="cuda")
    g = [base.permute(2, 0, 1), torch.randn(300, 7, device="cuda").t()]
    _check(g, 1.0)
    for dtype in (torch.float32, torch.bfloat16):
        buf = torch.randn(100_000, device="cuda").to(dtype)
        cuts = [1, 4, 12, 13, 1000, 9999, 50_001, 99_990]
        parts = [buf[a + 1:b] for a, b in zip(cuts, cuts[1:])]
        keep = buf[cuts].clone()
        _check(parts, 0.5)
        assert torch.equal(buf[cuts], keep)
        out = torch.full((100_003,), 5.0, device="cuda")
        _check(parts, 0.1, out=[out[a + 3:b + 2] for a, b in zip(cuts, cuts[1:])])
        assert (out[[c + 2 for c in cuts]] == 5.0).all() and (out[:4] == 5.0).all()


def test_repeats_bit_for_bit_streams_and_capture():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    torch_ffi.init()
    grads = _grads(SHAPES["long"], ["f32", "bf16"])
    outs = [torch.empty_like(g) for g in grads]
    ref = torch_ffi.clip_grad_norm(grads, 1.0, out=outs)
    ref_outs = [o.clone() for o in outs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            again = torch_ffi.clip_grad_norm(grads, 1.0, out=outs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ref[0], again[0]) and all(torch.equal(a, c) for a, c in zip(outs, ref_outs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = torch_ffi.clip_grad_norm(grads, 1.0, out=outs)
    for g in grads:
        g.mul_(2.0)
    graph.replay()
    assert float(cap[0]) == pytest.approx(2 * float(ref[0]), rel=1e-6)
    _check_outs(outs, _reference(grads, 1.0, 1e-6, False)[2])


def test_offsets_beyond_32_bits():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    g = torch.zeros(2 ** 31 + 4099, dtype=torch.bfloat16, device="cuda")
    at = [0, 7, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 4098]
    g[at] = torch.tensor([3.0, -4.0, 12.0, 84.0, 3612.0], dtype=torch.bfloat16, device="cuda")
    exact = math.sqrt(sum(float(v) ** 2 for v in g[at]))
    before = g[at].double()
    norm, bad = torch_ffi.clip_grad_norm([g], 1.0)
    assert abs(float(norm) - exact) <= 5 * U * exact and int(bad) == 0
    _check_outs([g[at]], [before / (exact + 1e-6)])
    assert int((g != 0).sum()) == len(at)


def test_in_place_is_seen_by_autograd():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    g = torch.randn(8, device="cuda")
    before = g._version
    torch_ffi.clip_grad_norm([g], 1.0)
    assert g._version > before


def test_agrees_with_the_rollouts_reduction():
    torch = _torch()
    from nablaengine_b200 import rollout, torch_ffi
    g = torch.randn(4, 256, 29, device="cuda")
    g[1, 7, 3] = float("nan")
    vec = rollout.reduce_stats(torch.zeros((), device="cuda"), g)
    norm, bad = torch_ffi.grad_norm([g], nonfinite="zero")
    assert float(norm) == pytest.approx(float(vec[1]) ** 0.5, rel=6 * U) and int(bad) == 1


def test_refusals():
    torch = _torch()
    from nablaengine_b200 import torch_ffi
    g = torch.randn(64, 8, device="cuda")
    for bad in (g, [g.cpu()], [g.double()], [g[:, ::2]], [g.expand(3, 64, 8)], [None], [g, g.int()], [g[::2]],
                [torch._neg_view(g)]):
        with pytest.raises(TypeError):
            torch_ffi.grad_norm(bad)
        with pytest.raises(TypeError):
            torch_ffi.clip_grad_norm(bad, 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            torch_ffi.clip_grad_norm([g], bad)
        with pytest.raises(ValueError):
            torch_ffi.clip_grad_norm([g], 1.0, eps=bad)
    with pytest.raises(ValueError):
        torch_ffi.grad_norm([g], nonfinite="drop")
    h = g.half()
    for out in ([], [g, g], [g[:63]], [g.t().contiguous().t()], [h], [g.double()]):
        with pytest.raises(TypeError):
            torch_ffi.clip_grad_norm([g], 1.0, out=out)
    with pytest.raises(TypeError):
        torch_ffi.clip_grad_norm([h], 1.0, out=[g.bfloat16()])
    flat = torch.randn(100, device="cuda")
    keep = flat.clone()
    for grads, out in (([flat, flat], None), ([flat[:60], flat[40:]], None), ([flat[:50]], [flat[10:60]]),
                       ([flat[:50], flat[50:]], [flat[50:], flat[:50]])):
        with pytest.raises(ValueError):
            torch_ffi.clip_grad_norm(grads, 1.0, out=out)
    assert torch.equal(flat, keep)
    torch_ffi.grad_norm([flat, flat])  # (nothing is written: the same tensor may be given twice)
