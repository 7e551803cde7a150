"""A list of no blocks is refused, whatever the cache: a tensor without elements has
no address, which the library takes for no list at all."""
import pytest
import torch

import b2engine as b2
from test_gpu_kv4 import make, make16, ws_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 16])
def test_a_list_of_no_blocks_is_refused(cuda, bits):
    q, kv, _, _ = (make if bits == 4 else make16)(1, [40, 3], 8, 2, 64, 16, "fp16")
    out = torch.full_like(q, 7.0)
    for shape in ((2, 2, 0), (0,)):
        with pytest.raises(ValueError, match="blocks"):
            b2.paged_decode_gqa(q, kv, out, blocks=torch.zeros(shape, dtype=torch.int32, device="cuda"), ws=ws_for(kv, 8))
    torch.cuda.synchronize()
    assert (out == 7).all()
