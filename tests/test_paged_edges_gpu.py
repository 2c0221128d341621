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


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("news,befores,nh,nkv,hd,page", [
    ([200], [100], 4, 2, 128, 16), ([333, 1, 150], [0, 700, 77], 8, 2, 64, 32), ([700], [1300], 3, 1, 128, 16),
    ([5], [300], 8, 2, 128, 16), ([9, 1, 3], [0, 64, 500], 4, 4, 64, 8), ([17], [40], 1, 1, 128, 64), ([3], [0], 40, 5, 64, 16)])
def test_a_value_that_is_not_finite_stays_with_the_rows_that_see_it(news, befores, nh, nkv, hd, page, value):
    """One value of one kv head at one new position after the other: the rows before it, and the other kv heads, are as
    without it; the rows that see it are not finite where it weighs in."""
    cache, q, table, starts, kv = make(news, befores, nh, nkv, hd, page, seed=31)
    want, mag = reference(cache, q, table, starts, kv)
    g = nh // nkv
    for s, (n, before) in enumerate(zip(news, befores)):
        a = starts[s].item()
        for i in sorted({0, 1, n // 3, n // 2, n - 2, n - 1} & set(range(n))):
            p, head, dim = before + i, i % nkv, (13 * i) % hd
            at = (table[s, p // page].item(), p % page, head, dim)
            kept = cache.v_pages[at].clone()
            cache.v_pages[at] = value
            y = cache.attend(q, table, starts, kv)
            cache.v_pages[at] = kept
            heads = slice(head * g, (head + 1) * g)
            assert not torch.isfinite(y[a + i:a + n, heads, dim].float()).any()
            y[a + i:a + n, heads] = want[a + i:a + n, heads].to(BF16)
            check(y, want, mag)
