"""How the blocks' column sums of layer norm's backward meet: in trees, in which a large term does not swallow the others
one by one."""
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cols", [64, 100, 128])
@pytest.mark.parametrize("rows_of_one", ["one block's", "one of each block's"])
def test_a_large_term_leaves_the_others(rows_of_one, cols, dtype):
    """A column with 2^24 in row 0 and 1 in 31 other rows, either those of the first block's other groups or one in each
    of 31 further blocks. Over 4096 rows of these widths a group takes at most 2 rows, a warp of the second kernel at
    most 5 blocks' sums, and 32 groups and 32 warps meet in trees: 2 + 5 + 5 + 5 = 17 additions at most, so each column
    is within 17 u of the sum of its terms' sizes (one after the other, all 31 ones would be lost)."""
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nablaengine_b200 import torch_ffi
    g = torch.zeros(4096, cols, device="cuda", dtype=getattr(torch, dtype))
    g[0] = 2.0 ** 24
    g[range(1, 32) if rows_of_one == "one block's" else range(32, 1024, 32)] = 1.0
    x = torch.ones_like(g)
    mean, rstd, one = torch.zeros(4096, device="cuda"), torch.ones(4096, device="cuda"), torch.ones(cols, device="cuda")
    _, gw, gb = torch_ffi.layer_norm_backward(g, x, mean, rstd, one, one)
    want = 2.0 ** 24 + 31
    for sums in (gw, gb):
        assert ((sums.double() - want).abs() <= 17 * U * want).all(), (sums.double() - want).abs().max()
