"""The bounded-cache example takes rows that lie anywhere, and a call that is refused
leaves the layer as it was."""
import os
import sys

import pytest
import torch

EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "serving-engine_b200", "examples")
sys.path.insert(0, EXAMPLES)

pytestmark = pytest.mark.gpu


def layer():
    from bounded_cache import BoundedLayer
    torch.manual_seed(3)
    return BoundedLayer(2, 4, 2, 64, capacity=64, budget=32, sinks=2, recent=8)


def new(n, h):
    return torch.randn(2, n, h, 64, device="cuda").bfloat16()


def moved(x, by):
    """The same numbers `by` elements into a buffer."""
    return torch.zeros(x.numel() + by, dtype=x.dtype, device="cuda")[by:].view(x.shape).copy_(x)


def spread(x, axis):
    """The same numbers with the elements of a row far apart."""
    return x.transpose(-1, axis).contiguous().transpose(-1, axis)


def test_rows_that_lie_anywhere(cuda):
    a, b = layer(), layer()
    q, k, v = new(40, 4), new(40, 2), new(40, 2)
    a.prefill(q, k, v)
    b.prefill(q, moved(k, 1), moved(v, 4))
    tokens = [(new(1, 4)[:, 0], new(1, 2)[:, 0], new(1, 2)[:, 0]) for _ in range(30)]
    for i, (q1, k1, v1) in enumerate(tokens):
        a.decode(q1, k1, v1)
        b.decode(q1, *((moved(k1, 3), moved(v1, 2)) if i % 2 else (spread(k1, 1), spread(v1, 0))))
    assert a.rows == b.rows == a.seq_lens.tolist() == b.seq_lens.tolist()
    assert torch.equal(a.kv.k, b.kv.k) and torch.equal(a.kv.v, b.kv.v) and torch.equal(a.scores, b.scores)


def test_refused_rows_change_nothing(cuda):
    a = layer()
    with pytest.raises(ValueError):
        a.prefill(new(20, 4), new(20, 1), new(20, 1))
    assert a.rows == [0, 0] == a.seq_lens.tolist()
    a.prefill(new(20, 4), new(20, 2), new(20, 2))
    for k in (new(1, 1)[:, 0], new(1, 2)[:, 0].float(), new(1, 2)[:1, 0]):
        with pytest.raises(ValueError):
            a.decode(new(1, 4)[:, 0], k, k)
        assert a.rows == [20, 20] == a.seq_lens.tolist()
    a.decode(new(1, 4)[:, 0], new(1, 2)[:, 0], new(1, 2)[:, 0])
    assert a.rows == [21, 21] == a.seq_lens.tolist()
