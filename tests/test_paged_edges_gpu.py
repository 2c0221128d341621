"""The paged attention and its writer at the edges of what their documentation allows. Definition, tolerances and the
makers of inputs: tests/test_paged_gpu.py."""

import pytest
import torch
from test_paged_gpu import check, make, reference

from byteprof_b200 import _lib

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("nh,nkv,hd", [(8, 8, 128), (16, 8, 64)])
@pytest.mark.parametrize("order", ["EERE", "EEEEEEEERR", "REEEEEEEEEEEER", "ERERERERERER"])
def test_many_rows_of_empty_sequences_beside_long_ones(order, nh, nkv, hd):
    """E: 300 rows that see nothing (a slot of a captured graph without a cache), R: 300 rows over 2300 positions. Each E is
    two items for each of 8 kv heads, so that CTAs take several of them in a row and a long one behind them. No other
    sequence's values may change: the long ones equal the definition, the empty ones are zero, run after run."""
    n = 300
    cache, q, table, starts, kv = make([n] * len(order), [2000 * (c == "R") for c in order], nh, nkv, hd, 64, seed=len(order))
    empty = torch.tensor([c == "E" for c in order], device="cuda")
    lens = torch.where(empty, 0, kv).int()
    y = cache.attend(q, table, starts, lens)
    for i, c in enumerate(order):
        part = slice(i * n, (i + 1) * n)
        if c == "E":
            assert (y[part] == 0).all()
        else:
            one = torch.tensor([0, n], dtype=torch.int32, device="cuda")
            check(y[part], *reference(cache, q[part], table[i:i + 1], one, kv[i:i + 1]))
    for _ in range(20):
        assert torch.equal(cache.attend(q, table, starts, lens), y)
    assert _lib.device_errors() == 0
