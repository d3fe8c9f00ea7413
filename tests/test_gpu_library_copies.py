"""Two copies of libnabla_g1.so in one process: what one prepares (a kernel's shared memory, its clusters) is not taken for
the other's, and both give the same bits."""
import ctypes
import shutil

import pytest

pytestmark = pytest.mark.gpu


def test_a_second_copy_prepares_its_own_kernels(tmp_path):
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nablaengine_b200 import build, capi, torch_ffi
    product = capi.load()
    path = tmp_path / "libnabla_g1_copy.so"
    shutil.copy(build.LIB, path)
    copy = ctypes.CDLL(str(path))
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for name in ("nb_g1_layer_norm_forward", "nb_g1_layer_norm_backward", "nb_g1_grad_clip"):
        f = getattr(copy, name)
        f.argtypes, f.restype = getattr(product, name).argtypes, ctypes.c_int

    def p(t):
        return ctypes.c_void_p(t.data_ptr())

    # rows of one block and rows of a cluster, each with more shared memory than a kernel has unasked
    for rows, cols in ((300, 4096), (40, 20001)):
        x, g = (torch.randn(rows, cols, device="cuda") for _ in range(2))
        w, b = torch.rand(cols, device="cuda"), torch.rand(cols, device="cuda")
        want = torch_ffi.layer_norm_forward(x, w, b)
        got = [torch.full_like(t, float("nan")) for t in want]
        assert copy.nb_g1_layer_norm_forward(stream, rows, cols, cols, 0, p(x), 0, p(w), p(b), 1e-5, *map(p, got)) == 0
        assert all(torch.equal(a, c) for a, c in zip(got, want))
        want = torch_ffi.layer_norm_backward(g, x, got[1], got[2], w, b)
        grads = [torch.full_like(t, float("nan")) for t in want]
        work = torch.empty(product.nb_g1_layer_norm_work_bytes(rows, cols), dtype=torch.uint8, device="cuda")
        assert copy.nb_g1_layer_norm_backward(stream, rows, cols, cols, cols, 0, p(g), p(x), p(got[1]), p(got[2]), 0,
                                              p(w), *map(p, grads), p(work)) == 0
        assert all(torch.equal(a, c) for a, c in zip(grads, want))
    # a short list: one cluster of 16 blocks, which a kernel does not have unasked either
    g = torch.randn(5000, device="cuda")
    out, other = torch.empty_like(g), torch.empty_like(g)
    norm, bad = torch_ffi.clip_grad_norm([g], 1.0, out=[out])
    n, k = torch.zeros((), device="cuda"), torch.zeros((), dtype=torch.int64, device="cuda")
    one = (ctypes.c_void_p * 1)
    assert copy.nb_g1_grad_clip(stream, 1, one(g.data_ptr()), one(other.data_ptr()), (ctypes.c_longlong * 1)(5000),
                                (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(0), 0, 1.0, 1e-6, ctypes.c_void_p(0), p(n),
                                p(k)) == 0
    assert torch.equal(out, other) and torch.equal(n, norm) and int(k) == int(bad) == 0
