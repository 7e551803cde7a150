"""Eviction whose rows a second launch moves: in place the CTAs split a row's
columns, into other blocks the rows.  That form is taken where a (sequence, K/V
head) keeps more than 128 KB, or where the new lengths are written over the old
ones.  Bit for bit against the reference."""
import pytest

from test_gpu_bounded import evict_case

pytestmark = pytest.mark.gpu


def above_one_launch(D):
    """A budget that keeps more than 128 KB of K and V rows."""
    return (128 << 10) // (4 * D) + 37


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("D,dt", [(8, "fp16"), (16, "bf16"), (40, "bf16"), (72, "fp16"), (80, "fp16"), (96, "bf16"),
                                  (144, "fp16"), (200, "bf16"), (256, "fp16")])
def test_head_dims(cuda, in_place, D, dt):
    n = above_one_launch(D)
    evict_case(110, [2 * n + 5, n + 1, n - 3], 16, 2, D, dt, n, 3, n // 3, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bs,layout", [(1, "slot"), (5, "slot"), (5, "head"), (16, "head"), (24, "slot"), (128, "head")])
@pytest.mark.parametrize("D", [40, 128])
def test_block_sizes_and_layouts(cuda, in_place, bs, layout, D):
    n = above_one_launch(D)
    evict_case(111, [n + 300, 3 * n, 0, n], bs, 3, D, "fp16", n, 5, 60, layout=layout, in_place=in_place)


@pytest.mark.parametrize("D", [8, 40, 64, 80, 96, 128, 144, 256])
@pytest.mark.parametrize("layout", ["slot", "head"])
def test_few_rows_with_lengths_written_over(cuda, D, layout):
    evict_case(112, [500, 20, 64, 65], 16, 3, D, "bf16", 64, 3, 5, layout=layout, in_place=True, alias=True)
    evict_case(113, [500, 20, 64, 65], 16, 3, D, "bf16", 64, 3, 5, layout=layout, alias=True)
