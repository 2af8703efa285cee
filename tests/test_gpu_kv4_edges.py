"""The low-precision attention layer's kernels where they can go wrong unnoticed: work items of one key tile, values that are not finite
in calls whose keys are split, loose bounds, offsets that fall, operands off their alignment, and every key counted once."""
import pytest

from test_gpu_kv4 import Questions

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def G(dcd):
    import torch
    assert torch.cuda.is_available()
    import gpu_util
    return gpu_util


# ---------------------------------------------------------------------------------------------
# items of one key tile
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("causal", [False, True])
def test_items_of_one_key_tile_behind_each_other(G, hd, causal):
    """Twenty items a CTA, nearly all of a single key tile, whose sums differ by up to a hundred times: each row is divided by its own
    sum, whichever group of warps has the tile and however far the other one is behind."""
    import torch
    lens = [(1 + (37 * i) % 120, 130 + i)[i % 29 == 28] for i in range(200)]
    c = Questions(lens, 0, 16, 16, hd, causal, False)
    c.launch(G)
    c.check(rows=range(0, 200, 3))
    first = c.out.clone()
    for _ in range(3):
        c.out.fill_(-7.0)
        c.launch(G)
        torch.cuda.synchronize()
        assert torch.equal(first, c.out)
