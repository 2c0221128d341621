"""The paged attention and its writer at the edges of what their documentation allows. Definition, tolerances and the
makers of inputs: tests/test_paged_gpu.py."""

import pytest
import torch
from test_paged_gpu import append_reference, check, make, reference

from byteprof_b200 import _lib
from byteprof_b200.optim.decode_ops import rope_tables
from byteprof_b200.optim.paged import PagedCache

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("nh,nkv,hd", [(8, 8, 128), (16, 8, 64)])
@pytest.mark.parametrize("order", ["EERE", "EEEEEEEERR", "REEEEEEEEEEEER", "ERERERERERER", "E" * 20 + "RR" + "E" * 18 + "R"])
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


@pytest.mark.parametrize("news,befores,nh,nkv,hd,page", [
    # one token per tile of 128 rows (65 to 128 heads per kv head), and the first group of two
    ([130], [40], 71, 1, 128, 16), ([5, 90], [300, 0], 142, 2, 64, 32), ([77, 1, 40], [0, 513, 128], 128, 1, 128, 64),
    ([60], [100], 65, 1, 64, 8), ([50, 33], [7, 200], 64, 1, 128, 16), ([9], [1500], 130, 2, 64, 64),
    # more heads than a tile has rows: the 16-row kernel, tiles within a token and across two
    ([1], [700], 256, 1, 128, 16), ([40, 3], [0, 250], 256, 1, 64, 32), ([20], [90], 400, 2, 128, 64), ([1, 7], [33, 0], 129, 1, 64, 8),
    ([2], [65], 1024, 1, 128, 16), ([3, 1], [1000, 5], 1024, 4, 64, 16)])
def test_large_head_groups(news, befores, nh, nkv, hd, page):
    cache, q, table, starts, kv = make(news, befores, nh, nkv, hd, page, seed=nh)
    y = cache.attend(q, table, starts, kv)
    check(y, *reference(cache, q, table, starts, kv))
    assert torch.equal(y, cache.attend(q, table, starts, kv))


def test_append_with_the_most_heads():
    """1024 query heads: what a thread keeps in registers is a fraction of the row. A sum of squares has 512 terms in each of a
    thread's two accumulators: 2^-15 of it at most, half of that after the root, beside the usual tolerance."""
    nh, nkv, hd, n = 1024, 4, 128, 5
    cache, _, table, starts, kv = make([n], [30], nh, nkv, hd, 16, seed=41)
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g, device="cuda").to(BF16)
    qn = (1 + 0.1 * torch.randn(nh * hd, generator=g, device="cuda")).to(BF16)
    kn = (1 + 0.1 * torch.randn(nkv * hd, generator=g, device="cuda")).to(BF16)
    cos, sin = rope_tables(64, hd, 10000.0, torch.device("cuda"))
    q = cache.append(qkv, nh, table, starts, kv, qn, kn, cos, sin)
    pos = torch.arange(30, 30 + n, device="cuda")
    (wq, sq), (wk, sk) = append_reference(qkv, nh, nkv, hd, pos, qn, kn, cos, sin, 1e-6)
    at = table.long()[0, pos // 16], pos % 16
    for y, w, s in ((q, wq, sq), (cache.k_pages[at], wk, sk)):
        assert ((y.double() - w).abs() <= (2.0**-8 + 2.0**-16) * w.abs() + 2.0**-20 * s).all()
    assert torch.equal(cache.v_pages[at], qkv[:, (nh + nkv) * hd:].view(n, nkv, hd))


@pytest.mark.parametrize("n", [1, 40])
def test_lengths_up_to_the_end_of_32_bits(n):
    """A table of 2^23 entries that all name one page of 256. Up to position 2^31 - 257 a row sees the same keys again and
    again, so its result is that of the page alone (here all its values are 1: any weights give 1, up to the sums' drift); the
    largest lengths are past the table."""
    page = 256
    cache = PagedCache(*(torch.ones(1, page, 1, 64, dtype=BF16, device="cuda") for _ in range(2)))
    table = torch.zeros(1, 2**31 // page, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    q = torch.randn(n, 1, 64, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(BF16)
    last = 2**31 - 256
    for kv, live in ((last, n), (last + 3, max(n - 3, 0)), (2**31 - 1, 0)):
        y = cache.attend(q, table, starts, torch.tensor([kv], dtype=torch.int32, device="cuda"))
        assert ((y[:live].float() - 1).abs() < 2.0**-5).all() and torch.isnan(y[live:]).all()
        kv = torch.tensor([kv], dtype=torch.int32, device="cuda")
        own = PagedCache.zeros(1, page, 1, 64, torch.device("cuda"))
        x = own.append(torch.ones(n, 3 * 64, dtype=BF16, device="cuda"), 1, table, starts, kv)
        assert (x[:live] == 1).all() and torch.isnan(x[live:]).all()
    assert _lib.device_errors() == 0


def test_ever_new_sizes_do_not_pile_up():
    cache, q, table, starts, kv = make([1500], [3], 2, 2, 64, 16, seed=51)
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for rows in range(1, 1500):
        cache.attend(q[:rows], table, one, kv)
    assert len(cache._ws_bytes) <= 1024
    check(cache.attend(q, table, starts, kv), *reference(cache, q, table, starts, kv))
