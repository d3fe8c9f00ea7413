"""The training operators' host side without a GPU: what the C entries refuse before any launch, the torch API's
refusal of CPU tensors, and the norm over the ranks of a process group (gloo, the device calls stood in for)."""
import ctypes
import os
import socket

import pytest
import torch

from nablaengine_b200 import capi, torch_ffi

INVALID = 1  # cudaErrorInvalidValue
NUL = ctypes.c_void_p(0)
AT = ctypes.c_void_p(1 << 20)  # an address that nothing reads: every call here is refused first


def test_layer_norm_entries_refuse_bad_arguments():
    lib = capi.load()

    def forward(rows=4, cols=36, stride=36, dtype=0, x=AT, wtype=0, w=NUL, b=NUL, eps=1e-5, y=AT, mean=AT, rstd=AT):
        return lib.nb_g1_layer_norm_forward(NUL, rows, cols, stride, dtype, x, wtype, w, b, eps, y, mean, rstd)

    def backward(rows=4, cols=36, gs=36, s=36, dtype=0, g=AT, x=AT, mean=AT, rstd=AT, wtype=0, w=AT, gx=AT, gw=AT,
                 gb=AT, work=AT):
        return lib.nb_g1_layer_norm_backward(NUL, rows, cols, gs, s, dtype, g, x, mean, rstd, wtype, w, gx, gw, gb,
                                             work)

    assert forward(rows=0, x=NUL, y=NUL, mean=NUL, rstd=NUL) == 0  # no rows: a no-op
    odd = ctypes.c_void_p((1 << 20) + 1)
    for kw in (dict(rows=-1), dict(cols=0), dict(cols=-3), dict(cols=1 << 40), dict(stride=-1), dict(dtype=3),
               dict(dtype=-1), dict(dtype=0, wtype=1), dict(dtype=1, wtype=2), dict(x=NUL), dict(y=NUL),
               dict(mean=NUL), dict(rstd=NUL), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
               dict(x=odd), dict(y=odd), dict(w=odd), dict(b=odd), dict(mean=odd), dict(rstd=odd)):
        assert forward(**kw) == INVALID, kw
    for kw in (dict(rows=-1), dict(cols=0), dict(gs=-1), dict(s=-1), dict(dtype=7), dict(dtype=2, wtype=1),
               dict(g=NUL), dict(x=NUL), dict(mean=NUL), dict(rstd=NUL), dict(work=NUL), dict(gx=odd), dict(g=odd),
               dict(gw=odd), dict(mean=odd), dict(rstd=odd), dict(work=ctypes.c_void_p((1 << 20) + 8))):
        assert backward(**kw) == INVALID, kw
    assert lib.nb_g1_layer_norm_work_bytes(4096, 100) > 0
    assert lib.nb_g1_layer_norm_work_bytes(-1, 100) < 0 and lib.nb_g1_layer_norm_work_bytes(1, 0) < 0


def _arrays(*tensors):
    """(count, addresses, sizes, types) of (address, size, type) triples."""
    n = len(tensors)
    return (n, (ctypes.c_void_p * n)(*[t[0] for t in tensors]), (ctypes.c_longlong * n)(*[t[1] for t in tensors]),
            (ctypes.c_int * n)(*[t[2] for t in tensors]))


def _clip(grads, outs, max_norm=1.0, eps=1e-6, work=AT):
    n, g, sizes, types = _arrays(*grads)
    _, o, _, out_types = _arrays(*outs)
    return capi.load().nb_g1_grad_clip(NUL, n, g, o, sizes, types, out_types, 0, max_norm, eps, work, AT, AT)


def test_grad_entries_refuse_bad_arguments():
    lib = capi.load()
    base = 1 << 20
    one = [(base, 10, 0)]
    for kw in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(eps=-1.0), dict(eps=float("nan"))):
        assert _clip(one, one, **kw) == INVALID, kw
    for many in ([(base, 1 << 20, 0)], [(base + 4096 * k, 10, 0) for k in range(97)]):  # (a short list needs no work)
        for work in (NUL, ctypes.c_void_p((1 << 20) + 8)):
            assert _clip(many, many, work=work) == INVALID
    for bad in ([(None, 10, 0)], [(base, -1, 0)], [(base, 10, 3)], [(base + 2, 10, 0)], [(base + 1, 10, 1)]):
        assert _clip(bad, bad) == INVALID, bad
        n, g, sizes, types = _arrays(*bad)
        assert lib.nb_g1_grad_sumsq(NUL, n, g, sizes, types, 0, AT, AT) == INVALID
        assert lib.nb_g1_grad_scale(NUL, n, g, g, sizes, types, types, 0, 1.0, 0.0, AT, NUL, NUL) == INVALID
    assert lib.nb_g1_grad_sumsq(NUL, -1, NUL, NUL, NUL, 0, AT, AT) == INVALID
    assert lib.nb_g1_grad_work_bytes(-1) < 0 and lib.nb_g1_grad_work_bytes(0) > 0
    assert lib.nb_g1_grad_work_bytes(1000) >= lib.nb_g1_grad_work_bytes(10)


def test_grad_results_refuse_odd_addresses_and_impossible_sizes():
    lib = capi.load()
    base = 1 << 20
    n, g, sizes, types = _arrays((base, 10, 0))
    for norm, bad in ((base + 2, base), (base, base + 4)):
        at = ctypes.c_void_p(norm), ctypes.c_void_p(bad)
        assert lib.nb_g1_grad_clip(NUL, n, g, g, sizes, types, types, 0, 1.0, 0.0, AT, *at) == INVALID
        assert lib.nb_g1_grad_scale(NUL, n, g, g, sizes, types, types, 0, 1.0, 0.0, AT, *at) == INVALID
    for size in ((1 << 40) + 1, (1 << 63) - 1):
        assert _clip([(base, size, 0)], [(base, size, 0)]) == INVALID


def test_grad_entries_refuse_shared_memory():
    """Any two of the spans that a clip touches, one of them written, unless it is a tensor scaled in place."""
    a = 1 << 20
    grads = [(a, 100, 0), (a + 4096, 100, 1)]
    for outs in ([(a, 100, 0), (a + 396, 100, 1)],           # an output over another output's end
                 [(a + 8192, 100, 0), (a + 8192, 100, 1)],   # two outputs at one place
                 [(a + 4, 100, 0), (a + 8192, 100, 1)],      # an output shifted against its gradient
                 [(a + 8192, 100, 0), (a + 4096, 100, 0)],   # in place, but in another type
                 [(a + 4100, 100, 0), (a + 16384, 100, 1)],  # an output in another gradient
                 [(a + 4096 - 396, 100, 0), (a + 16384, 100, 1)]):
        assert _clip(grads, outs) == INVALID, outs
    assert _clip([(a, 100, 0), (a, 100, 0)], [(a, 100, 0), (a, 100, 0)]) == INVALID    # one tensor given twice
    assert _clip([(a, 100, 0), (a + 200, 100, 0)], [(a, 100, 0), (a + 200, 100, 0)]) == INVALID


def test_torch_api_refuses_cpu_tensors():
    x = torch.zeros(4, 36)
    for call in (lambda: torch_ffi.layer_norm(x), lambda: torch_ffi.layer_norm_forward(x),
                 lambda: torch_ffi.layer_norm_backward(x, x, x[:, 0], x[:, 0]),
                 lambda: torch_ffi.grad_norm([x]), lambda: torch_ffi.clip_grad_norm([x], 1.0)):
        with pytest.raises(TypeError):
            call()


class _StandIn:
    """The compiled host module's two calls on CPU tensors."""

    @staticmethod
    def grad_sumsq(grads, zero):
        s = sum(float((g.double() ** 2).sum()) for g in grads)
        return torch.tensor([s, 0.0], dtype=torch.float64),

    @staticmethod
    def grad_clip(grads, outs, max_norm, eps, zero, stats):
        norm = float(stats[0]) ** 0.5
        for o, g in zip(outs or (), grads):
            o.copy_(g * min(1.0, max_norm / (norm + eps)))
        return torch.tensor(norm), stats[1].long()


def _rank_main(rank, world, port, out):
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    torch_ffi._NATIVE[:] = [_StandIn]
    g = torch.Generator().manual_seed(5)
    full = torch.randn(2, 1000, generator=g)
    mine = [full[rank].clone()]
    n1, _ = torch_ffi.grad_norm(mine, group=dist.group.WORLD)
    n2, _ = torch_ffi.clip_grad_norm(mine, 2.0, group=dist.group.WORLD)
    torch.save((n1, n2, mine[0]), f"{out}.{rank}")
    dist.destroy_process_group()


def test_two_ranks_clip_by_their_common_norm(tmp_path):
    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = str(tmp_path / "r")
    mp.start_processes(_rank_main, args=(2, port, out), nprocs=2, join=True, start_method="spawn")
    full = torch.randn(2, 1000, generator=torch.Generator().manual_seed(5))
    norm = full.double().norm()
    for rank in range(2):
        n1, n2, mine = torch.load(f"{out}.{rank}")
        assert float(n1) == float(n2) == pytest.approx(float(norm), rel=1e-6)
        assert torch.allclose(mine, full[rank] * float(2.0 / (norm + 1e-6)), rtol=1e-6, atol=0)
