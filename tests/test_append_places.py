"""An append into a cache whose blocks, positions or heads lie in one place is
refused: which of the rows would stay is nobody's to say."""
import pytest

from test_kv4 import append, cache16


@pytest.mark.parametrize("which", ["stride_block", "stride_slot", "stride_head"])
def test_rows_that_would_be_written_to_one_place(which):
    assert append(cache16(**{which: 0})) == -1


@pytest.mark.gpu
def test_dimensions_of_one_need_no_stride(cuda):
    import torch

    import b2engine as b2
    x = torch.randn(1, 9, 1, 64, device="cuda").half()
    k, v = (torch.zeros(16, 64, dtype=torch.float16, device="cuda") for _ in "kv")
    one = lambda t: t.as_strided((1, 16, 1, 64), (0, 64, 0, 1))  # noqa: E731
    kv = b2.PagedKV(one(k), one(v), torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                    torch.tensor([9], dtype=torch.int32, device="cuda"))
    kv.c.stride_block = kv.c.stride_head = 0
    b2.paged_kv_append(kv, x, x)
    assert torch.equal(k[:9], x[0, :, 0]) and torch.equal(v[:9], x[0, :, 0]) and not k[9:].any()
