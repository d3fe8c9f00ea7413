"""The gradient norm and clipping in two calls (the sums of a part, then the clip by the parts' common sums), which a
process group's ranks make, against the definition over all parts in 64 bits. The tolerances are those of
test_gpu_grad_clip.py."""
import pytest

from test_gpu_grad_clip import SHAPES, U, _check_outs, _grads, _reference

pytestmark = pytest.mark.gpu


def _native():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nablaengine_b200 import torch_ffi
    return torch, torch_ffi._native()


def _clip_parts(parts, max_norm, zero, outs_of):
    """Both calls for every part of the list, the sums added up between them as an all-reduce does. outs_of: the outputs
    of a part. Compares all of it with the whole list's reference."""
    torch, native = _native()
    whole = [g for p in parts for g in p]
    norm, bad, ref = _reference(whole, max_norm, 1e-6, zero)
    sums = [native.grad_sumsq(p, zero)[0] for p in parts]
    for s, p in zip(sums, parts):
        own = _reference(p, max_norm, 1e-6, zero)
        assert s.dtype == torch.float64 and int(s[1]) == own[1]
        assert abs(float(s[0]) - own[0] ** 2) <= 9 * U * own[0] ** 2
    total = torch.stack(sums).sum(0)
    at = 0
    for p in parts:
        outs = outs_of(p)
        for n, b in (native.grad_clip(p, None, 0.0, 0.0, zero, total),
                     native.grad_clip(p, outs, max_norm, 1e-6, zero, total)):
            assert abs(float(n) - norm) <= 5 * U * norm + 2.0 ** -150 and int(b) == bad
        _check_outs(outs, ref[at:at + len(p)])
        at += len(p)


@pytest.mark.parametrize("dtypes", [["f32"], ["bf16"], ["f16", "bf16", "f32"]])
@pytest.mark.parametrize("shapes", ["one value", "odd", "empty ones", "one table", "long", "three tables"])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_parts_of_a_list(shapes, dtypes, max_norm):
    """The first part, the second, and an empty one; in place and into float32 tensors."""
    torch, _ = _native()
    grads = _grads(SHAPES[shapes], dtypes)
    half = len(grads) // 2
    split = [grads[:half], grads[half:], []]
    _clip_parts(split, max_norm, False, lambda p: [torch.full(g.shape, float("nan"), device="cuda") for g in p])
    _clip_parts(split, max_norm, False, lambda p: p)


@pytest.mark.parametrize("shapes", ["odd", "long", "three tables"])
def test_non_finite_values_of_one_part_count_in_all(shapes):
    torch, _ = _native()
    for first in (True, False):
        grads = _grads(SHAPES[shapes], ["f32", "bf16"])
        half = len(grads) // 2
        hit = (grads[:half] if first else grads[half:])[0].view(-1)
        hit[0], hit[-1] = float("inf"), float("nan")
        _clip_parts([grads[:half], grads[half:]], 0.25, True, lambda p: p)
        assert all(torch.isfinite(g).all() for g in grads)


def test_non_finite_values_kept():
    """One part's NaN makes the common norm NaN, and with it every part's values."""
    torch, native = _native()
    a, b = [torch.tensor([1.0, float("nan")], device="cuda")], [torch.tensor([3.0], device="cuda")]
    total = native.grad_sumsq(a, False)[0] + native.grad_sumsq(b, False)[0]
    for part in (a, b):
        norm, bad = native.grad_clip(part, part, 1.0, 1e-6, False, total)
        assert torch.isnan(norm) and int(bad) == 1 and torch.isnan(part[0]).all()


def test_a_process_group_of_one_rank():
    torch, _ = _native()
    import torch.distributed as dist
    from nablaengine_b200 import torch_ffi
    dist.init_process_group("nccl", store=dist.HashStore(), rank=0, world_size=1)
    try:
        for zero in (False, True):
            grads = _grads(SHAPES["odd"], ["f32", "bf16"])
            if zero:
                grads[0][0] = float("nan")
            norm, bad, ref = _reference(grads, 0.5, 1e-6, zero)
            mode = "zero" if zero else "keep"
            for n, b in (torch_ffi.grad_norm(grads, nonfinite=mode, group=dist.group.WORLD),
                         torch_ffi.clip_grad_norm(grads, 0.5, nonfinite=mode, group=dist.group.WORLD)):
                assert abs(float(n) - norm) <= 5 * U * norm and int(b) == bad
            _check_outs(grads, ref)
    finally:
        dist.destroy_process_group()
