"""The paged cache's writer and the attention over it (csrc/paged_append.cu, paged_attn.cu, paged_attn_tc.cu) against
their definitions in float64.

Tolerances. append: one rounding to bf16 of an fp32 value whose chain (norm, weight, rotation) has about six roundings
of 2^-24: half a bf16 step, 2^-8 |y|, plus 2^-20 of the rotated pair's size (the two products may cancel).
attend: the result's rounding gives 2^-8 |y|; the weights' rounding gives at most 2^-8 sum_j p_j |v_j| (each
weight is off by half a step), and the same again covers exp2's and the sums' fp32 errors (under 2^-12): in
all 2^-8 |y| + 1.25 * 2^-8 sum_j p_j |v_j|, element by element."""

import numpy as np
import pytest
import torch

from byteprof_b200 import _lib
from byteprof_b200.optim.decode_ops import rope_tables
from byteprof_b200.optim.paged import PagedCache

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def make(news, befores, nh, nkv, hd, page, seed=0, spare=2, extra_cols=1):
    """A pool with shuffled pages; what no sequence holds (tails, spare pages) is NaN. Lengths as given."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = [a + b for a, b in zip(news, befores)]
    need = [max(0, -(-x // page)) for x in kv]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(news), max([1] + need) + extra_cols), -7, dtype=torch.int32)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = order[at:at + c].int()
        at += c
    kp = torch.full((pool, page, nkv, hd), float("nan"), dtype=BF16, device="cuda")
    vp = torch.full_like(kp, float("nan"))
    for i, n in enumerate(kv):
        for p in range(-(-n // page)):
            m = min(page, n - p * page)
            for t in (kp, vp):
                t[table[i, p], :m] = torch.randn(m, nkv, hd, generator=g, device="cuda").to(BF16)
    q = (2 * torch.randn(sum(news), nh, hd, generator=g, device="cuda")).to(BF16)
    starts = torch.tensor(np.cumsum([0] + list(news)), dtype=torch.int32, device="cuda")
    return (PagedCache(kp, vp), q, table.cuda(), starts, torch.tensor(kv, dtype=torch.int32, device="cuda"))


def reference(cache, q, table, starts, kv_len, scale=None):
    """(out, sum_j p_j |v_j|) in float64, rows of no sequence NaN."""
    nh, hd, g = q.shape[1], q.shape[2], q.shape[1] // cache.nkv
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    st, kv, tab = starts.tolist(), kv_len.tolist(), table.long()
    for s in range(len(kv)):
        a, b = st[s], min(st[s + 1], q.shape[0])
        at = torch.arange(kv[s], device="cuda")
        page, off = tab[s, at // cache.page_size], at % cache.page_size
        k, v = (t[page, off].double().repeat_interleave(g, 1) for t in (cache.k_pages, cache.v_pages))
        x = torch.einsum("thd,jhd->htj", q[a:b].double(), k) * (hd ** -0.5 if scale is None else scale)
        pos = torch.arange(kv[s] - (st[s + 1] - a), kv[s], device="cuda")[: b - a]
        x = x.masked_fill(at[None] > pos[:, None], float("-inf"))
        p = torch.softmax(x, -1).nan_to_num(0.0) if kv[s] else x
        out[a:b] = torch.einsum("htj,jhd->thd", p, v)
        mag[a:b] = torch.einsum("htj,jhd->thd", p, v.abs())
    return out, mag


def check(y, want, mag):
    err = (y.double() - want).abs()
    tol = 2.0**-8 * want.abs() + 1.25 * 2.0**-8 * mag + 1e-30
    worst = (err / tol).nan_to_num(float("inf")).max().item() if err.numel() else 0.0
    assert worst <= 1.0, worst


FEW = [
    ([1], [0], 1, 1, 128, 16), ([1], [63], 16, 16, 128, 16), ([1], [64], 16, 16, 128, 8), ([1], [1022], 16, 16, 64, 256),
    ([1, 1, 1], [0, 700, 33], 32, 8, 128, 64), ([5], [3001], 16, 16, 128, 32), ([3, 1, 2], [9, 0, 128], 8, 1, 64, 16),
    ([1] * 67, list(range(0, 670, 10)), 6, 2, 64, 8), ([2], [0], 40, 5, 128, 16), ([1], [20000], 8, 1, 128, 64),
    ([1, 4, 1], [5000, 17, 1], 7, 1, 128, 128), ([17], [200], 3, 3, 64, 16),
]
MANY = [
    ([130], [0], 4, 2, 128, 16), ([128], [0], 1, 1, 128, 128), ([257], [511], 4, 4, 128, 64), ([300, 1, 77], [0, 900, 5], 8, 2, 64, 32),
    ([1000], [0], 6, 2, 64, 8), ([129, 127, 1], [1, 0, 128], 16, 16, 128, 256), ([700], [1300], 3, 1, 128, 16),
    ([64, 511, 33, 200], [100, 3, 0, 1024], 14, 2, 64, 64), ([333], [77], 5, 5, 128, 8),
    ([128], [30000], 1, 1, 128, 16), ([130], [20000], 2, 1, 64, 256), ([700], [0], 8, 1, 64, 16), ([2000], [37], 12, 1, 128, 32),
    ([33] * 600, [i % 50 for i in range(600)], 1, 1, 64, 16), ([0, 500, 0, 1, 0], [0, 3, 9, 2, 0], 4, 4, 128, 16),
]


FEW.append(([1] * 1100, [(7 * i) % 90 for i in range(1100)], 2, 1, 64, 32))


@pytest.mark.parametrize("news,befores,nh,nkv,hd,page", FEW + MANY)
def test_attend_against_the_definition(news, befores, nh, nkv, hd, page):
    cache, q, table, starts, kv = make(news, befores, nh, nkv, hd, page, seed=len(news) + nh)
    y = cache.attend(q, table, starts, kv)
    check(y, *reference(cache, q, table, starts, kv))
    assert torch.equal(y, cache.attend(q, table, starts, kv))  # the same bits again


@pytest.mark.parametrize("news,befores", [([1, 1], [5, 900]), ([200, 40], [0, 300])])
def test_attend_strided_rows_scale_and_out(news, befores):
    cache, q, table, starts, kv = make(news, befores, 4, 2, 128, 16, seed=3)
    wide = torch.zeros(q.shape[0], 6 * 128 + 8, dtype=BF16, device="cuda")
    qs = wide[:, 8:8 + 4 * 128].view(-1, 4, 128)
    qs.copy_(q)
    ow = torch.full((q.shape[0] + 2, 5 * 128), 7.0, dtype=BF16, device="cuda")
    out = ow[1:-1, :4 * 128].view(-1, 4, 128)
    y = cache.attend(qs, table, starts, kv, scale=0.25, out=out)
    assert y.data_ptr() == out.data_ptr()
    check(y, *reference(cache, q, table, starts, kv, 0.25))
    assert (ow[0] == 7).all() and (ow[-1] == 7).all() and (ow[1:-1, 4 * 128:] == 7).all()


@pytest.mark.parametrize("news,befores", [([1, 1, 1], [30, 0, 7]), ([150, 160, 140], [30, 0, 7])])
def test_rows_that_see_nothing_are_zero_and_rows_behind_the_last_sequence_are_left(news, befores):
    cache, q, table, starts, kv = make(news, befores, 4, 2, 64, 16, seed=5)
    kv2 = kv.clone()
    kv2[1] = 0                      # an empty sequence with rows
    if news[2] > 1:
        kv2[2] = news[2] - 3        # its first three rows lie before position 0
    want, mag = reference(cache, q, table, starts, kv)
    pad = torch.cat([q, q[:3]])
    out = torch.full_like(pad, 9.0)
    y = cache.attend(pad, table, starts, kv2, out=out)
    a, b = starts[1].item(), starts[2].item()
    check(y[:a], want[:a], mag[:a])
    assert (y[a:b] == 0).all()
    assert (y[q.shape[0]:] == 9).all()
    if news[2] > 1:
        assert (y[b:b + 3] == 0).all()
        w2, m2 = reference(cache, q[b + 3:], table[2:], torch.tensor([0, news[2] - 3], dtype=torch.int32), kv2[2:])
        check(y[b + 3:q.shape[0]], w2, m2)


@pytest.mark.parametrize("n", [1, 200])
def test_empty_sequences_between_others(n):
    cache, q, table, starts, kv = make([n, n], [100, 40], 4, 4, 128, 16, seed=6)
    tab = torch.cat([table[:1], table[:1], table[1:], table[1:]])
    st = torch.tensor([0, n, n, 2 * n, 2 * n], dtype=torch.int32, device="cuda")
    kv4 = torch.stack([kv[0], kv[0], kv[1], kv[1]])
    assert torch.equal(cache.attend(q, tab, st, kv4), cache.attend(q, table, starts, kv))
    check(cache.attend(q, tab, st, kv4), *reference(cache, q, table, starts, kv))


@pytest.mark.parametrize("news", [[1, 1], [140, 150]])
def test_a_page_outside_the_pool_gives_nan_rows_from_its_first_position(news):
    cache, q, table, starts, kv = make(news, [100, 100], 2, 1, 64, 16, seed=7)
    want, mag = reference(cache, q, table, starts, kv)
    for bad in (-1, cache.num_pages, 2**31 - 1):
        t = table.clone()
        t[1, 6] = bad  # positions 96..111 of sequence 1: every one of its rows sees them
        y = cache.attend(q, t, starts, kv)
        check(y[:news[0]], want[:news[0]], mag[:news[0]])
        assert torch.isnan(y[news[0]:]).all()
    if news[1] > 1:
        t = table.clone()
        t[1, 9] = -1  # positions 144..: rows before them are untouched
        y = cache.attend(q, t, starts, kv)
        check(y[:news[0] + 44], want[:news[0] + 44], mag[:news[0] + 44])
        assert torch.isnan(y[news[0] + 44:]).all()


@pytest.mark.parametrize("news", [[1], [130]])
def test_a_length_past_the_table_gives_nan_where_it_is_seen(news):
    cache, q, table, starts, kv = make(news, [100], 2, 2, 64, 16, seed=8, extra_cols=0)
    y = cache.attend(q, table, starts, kv + 1000)
    assert torch.isnan(y).all()
    short = table[:, :-1].contiguous()
    cap = short.shape[1] * 16
    want, mag = reference(cache, q, table, starts, kv)
    y = cache.attend(q, short, starts, kv)
    seen = max(0, cap - 100)  # rows at positions below the table's end
    check(y[:seen], want[:seen], mag[:seen])
    assert torch.isnan(y[seen:]).all()


@pytest.mark.parametrize("news", [[1, 1, 1, 1], [100, 200, 1, 60]])
def test_one_graph_serves_every_length_on_another_stream(news):
    cache, q, table, starts, kv = make(news, [500, 20, 1000, 3], 8, 2, 128, 16, seed=9)
    cache.attend(q, table, starts, kv)
    torch.cuda.synchronize()
    out = torch.empty_like(q)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    lens = kv.clone()
    with torch.cuda.graph(graph, stream=side):
        cache.attend(q, table, starts, lens, out=out)
    full, mag = reference(cache, q, table, starts, kv)
    for cut in (0, 1, 3):
        lens.copy_(kv - cut)
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want, m2 = reference(cache, q, table, starts, lens)
        check(out, want, m2)


def test_two_streams_at_once_do_not_share_scratch():
    sets = [make([1], [6000 + 100 * i], 8, 8, 128, 64, seed=20 + i) for i in range(2)]
    want = [c.attend(q, t, s, k) for c, q, t, s, k in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (c, q, t, s, k) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                got[i].append(c.attend(q, t, s, k))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


@pytest.mark.parametrize("dominant", [0, 99, 150])
def test_one_dominant_key_far_above_the_rest(dominant):
    """The running maximum has to move: one key scores hundreds above all others, early, late and on the diagonal."""
    for news in ([1], [151]):
        cache, q, table, starts, kv = make(news, [151 - news[0]], 2, 2, 128, 16, seed=11)
        q.fill_(4.0)
        cache.k_pages[table[0, dominant // 16].item(), dominant % 16] = 4.0
        check(cache.attend(q, table, starts, kv), *reference(cache, q, table, starts, kv))


# ---- the writer ----------------------------------------------------------------------------------------
def append_reference(qkv, nh, nkv, hd, pos, qn, kn, cos, sin, eps):
    x = qkv.double()
    res = []
    for part, w in ((x[:, :nh * hd], qn), (x[:, nh * hd:(nh + nkv) * hd], kn)):
        y = part
        if w is not None:
            y = y / torch.sqrt(y.pow(2).mean(1, keepdim=True) + eps) * w.double()
        y = y.view(len(pos), -1, hd)
        size = y.abs()
        if cos is not None:
            c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
            a, b = y[..., :hd // 2], y[..., hd // 2:]
            size = (a.abs() + b.abs()).repeat(1, 1, 2)
            y = torch.cat([a * c - b * s, b * c + a * s], -1)
        res.append((y, size))
    return res


@pytest.mark.parametrize("news,befores,nh,nkv,hd,page,norm,rope", [
    ([1], [0], 16, 16, 128, 16, True, True), ([5, 1, 300], [0, 77, 12], 32, 8, 128, 64, True, True),
    ([40], [3], 6, 2, 64, 8, True, False), ([33, 2], [64, 0], 4, 4, 64, 256, False, True), ([9], [1], 1, 1, 128, 16, False, False)])
def test_append_against_the_definition(news, befores, nh, nkv, hd, page, norm, rope):
    cache, _, table, starts, kv = make(news, befores, nh, nkv, hd, page, seed=13)
    g = torch.Generator(device="cuda").manual_seed(1)
    T, width = sum(news), (nh + 2 * nkv) * hd
    buf = torch.randn(T, width + 8, generator=g, device="cuda").to(BF16)
    qkv = buf[:, :width]
    qn = (1 + 0.1 * torch.randn(nh * hd, generator=g, device="cuda")).to(BF16) if norm else None
    kn = (1 + 0.1 * torch.randn(nkv * hd, generator=g, device="cuda")).to(BF16) if norm else None
    cos, sin = rope_tables(max(kv.tolist()), hd, 500000.0, torch.device("cuda")) if rope else (None, None)
    k0, v0 = cache.k_pages.clone(), cache.v_pages.clone()
    q = cache.append(qkv, nh, table, starts, kv, qn, kn, cos, sin, eps=1e-6)
    pos = torch.cat([torch.arange(b, a + b) for a, b in zip(news, befores)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news)).cuda()
    (wq, sq), (wk, sk) = append_reference(qkv, nh, nkv, hd, pos, qn, kn, cos, sin, 1e-6)
    page_of, off = table.long()[seq, pos // page], pos % page
    for y, w, s in ((q, wq, sq), (cache.k_pages[page_of, off], wk, sk)):
        assert ((y.double() - w).abs() <= 2.0**-8 * w.abs() + 2.0**-20 * s).all()
    assert torch.equal(cache.v_pages[page_of, off], qkv[:, (nh + nkv) * hd:].view(T, nkv, hd))
    k0[page_of, off] = cache.k_pages[page_of, off]
    v0[page_of, off] = cache.v_pages[page_of, off]
    assert torch.equal(k0.view(torch.int16), cache.k_pages.view(torch.int16))  # nothing else was written
    assert torch.equal(v0.view(torch.int16), cache.v_pages.view(torch.int16))


def test_append_outside_the_cache_or_tables_writes_nan_and_no_cache_row():
    cache, _, table, starts, kv = make([4, 3], [20, 0], 2, 1, 64, 8, seed=14)
    cos, sin = rope_tables(22, 64, 10000.0, torch.device("cuda"))  # positions 22, 23 of sequence 0 are outside
    qkv = torch.randn(9, 4 * 64, device="cuda").to(BF16)
    kv2 = kv.clone()
    kv2[1] = 2                                                    # its first row lies before position 0
    table[1, 0] = cache.num_pages                                 # and the others in no page
    k0 = cache.k_pages.clone()
    out = torch.full((9, 2, 64), 5.0, dtype=BF16, device="cuda")
    q = cache.append(qkv, 2, table, starts, kv2, None, None, cos, sin, out=out)
    assert not torch.isnan(q[:2]).any() and torch.isnan(q[2:7]).all() and (q[7:] == 5).all()
    changed = (k0.view(torch.int16) != cache.k_pages.view(torch.int16)).flatten(1).any(1)
    assert changed.sum() == 1 and changed[table[0, 2].long()]


def test_chunks_of_a_prompt_equal_the_whole_and_single_tokens():
    """A prompt appended and attended at once, in ragged chunks and token by token: the caches are the same bits, the
    outputs agree within both results' tolerances."""
    nh, nkv, hd, page, n = 8, 2, 128, 16, 333
    g = torch.Generator(device="cuda").manual_seed(15)
    qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g, device="cuda").to(BF16)
    cos, sin = rope_tables(n, hd, 10000.0, torch.device("cuda"))
    w = torch.ones(nh * hd, dtype=BF16, device="cuda"), torch.ones(nkv * hd, dtype=BF16, device="cuda")
    table = torch.randperm(-(-n // page), device="cuda").int()[None]
    results = []
    for chunks in ([n], [100, 1, 130, 2, 100], [1] * n):
        cache = PagedCache.zeros(table.shape[1], page, nkv, hd, torch.device("cuda"))
        ys, at = [], 0
        for c in chunks:
            starts = torch.tensor([0, c], dtype=torch.int32, device="cuda")
            kv = torch.tensor([at + c], dtype=torch.int32, device="cuda")
            q = cache.append(qkv[at:at + c], nh, table, starts, kv, *w, cos, sin)
            ys.append(cache.attend(q, table, starts, kv))
            at += c
        results.append((cache, torch.cat(ys), q))
    full = results[0]
    starts, kv = torch.tensor([0, n], dtype=torch.int32, device="cuda"), torch.tensor([n], dtype=torch.int32, device="cuda")
    want, mag = reference(full[0], full[2], table, starts, kv)
    for cache, y, _ in results:
        assert torch.equal(cache.k_pages, full[0].k_pages) and torch.equal(cache.v_pages, full[0].v_pages)
        check(y, want, mag)
    assert _lib.device_errors() == 0


def test_no_rows_and_no_sequences():
    cache, q, table, starts, kv = make([1], [5], 2, 2, 64, 8)
    assert cache.attend(q[:0], table, starts * 0, kv).shape == (0, 2, 64)
    out = torch.full_like(q, 3.0)
    cache.attend(q, table[:0], starts[:1], kv[:0], out=out)
    assert (out == 3).all()


@pytest.mark.parametrize("news", [[1, 2], [70, 90]])
def test_a_table_of_no_pages_has_no_positions(news):
    cache, q, table, starts, kv = make(news, [5, 0], 4, 2, 64, 8)
    assert torch.isnan(cache.attend(q, table[:, :0], starts, kv)).all()
    assert (cache.attend(q, table[:, :0], starts, kv * 0) == 0).all()
    before = cache.k_pages.clone()
    assert torch.isnan(cache.append(torch.ones(sum(news), 8 * 64, dtype=BF16, device="cuda"), 4, table[:, :0], starts, kv)).all()
    assert torch.equal(cache.k_pages.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("n", [1, 100])
def test_sequences_may_share_pages(n):
    """Three sequences continue one prefix of 64 positions (two pages), each with pages of its own behind it."""
    cache, q, table, starts, kv = make([n] * 3, [64, 64, 64], 4, 2, 128, 32)
    table[1:, :2] = table[0, :2]
    check(cache.attend(q, table, starts, kv), *reference(cache, q, table, starts, kv))


@pytest.mark.parametrize("news,befores", [([1, 2], [300, 77]), ([130, 200], [300, 77])])
def test_a_pool_of_more_than_32_bits(news, befores):
    """Pages whose first value is more than 2^32 elements, and 2^33 bytes, behind the pool's."""
    small, q, table, starts, kv = make(news, befores, 8, 4, 128, 64)
    pool = 2**32 // (64 * 4 * 128) + 64
    big = PagedCache(*(torch.empty(pool, 64, 4, 128, dtype=BF16, device="cuda") for _ in range(2)))
    far = torch.where(table >= 0, table + (pool - small.num_pages), table)
    for a, b in ((big.k_pages, small.k_pages), (big.v_pages, small.v_pages)):
        a[-small.num_pages:] = b
    y = big.attend(q, far, starts, kv)
    check(y, *reference(small, q, table, starts, kv))
    qkv = torch.randn(sum(news), 16 * 128, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(BF16)
    assert torch.equal(big.append(qkv, 8, far, starts, kv), small.append(qkv, 8, table, starts, kv))
    for a, b in ((big.k_pages, small.k_pages), (big.v_pages, small.v_pages)):
        assert torch.equal(a[-small.num_pages:].view(torch.int16), b.view(torch.int16))
