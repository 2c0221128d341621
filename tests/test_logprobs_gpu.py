"""token_logprobs (csrc/logprobs.cu) against float64.

Tolerance: sums of up to 131072 positive fp32 terms, each thread's share of at most some hundred added in a chain and
the shares merged in a tree, so a relative error below 300 * 2^-24 of the sums; exp2 adds 2^-22, the difference m - x
2^-24 |m - x|. log turns the sum's relative error into an absolute one: 2^-15 covers logprob's and the entropy's
absolute errors (entropy: T / (1 + R), at most log V = 12 times the sums' relative errors), plus 2^-22 relative."""

import numpy as np
import pytest
import torch

from byteprof_b200.optim.decode_ops import decode_finish, token_logprobs

pytestmark = pytest.mark.gpu


def want(x, ids, top):
    z = torch.log_softmax(x.double(), 1)
    p = z.exp()
    ent = -(torch.where(p > 0, p * z, torch.zeros_like(z))).sum(1)
    v, i = torch.sort(x.float(), dim=1, descending=True, stable=True)
    return z.gather(1, ids[:, None])[:, 0], ent, z.gather(1, i[:, :top]), i[:, :top]


def close(a, b):
    assert ((a.double() - b).abs() <= 2.0**-15 + 2.0**-22 * b.abs()).all(), (a.double() - b).abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 0), (5, 7, 3), (9, 31, 31), (3, 512, 20), (64, 513, 32),
                                            (2, 2048, 1), (2, 2049, 5), (1, 100352, 20), (7, 100352, 32), (33, 8191, 5),
                                            (200, 5000, 0), (1, 131072, 32), (170, 4097, 4)])
def test_against_float64(dtype, rows, vocab, top):
    g = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (3 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype)
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    lp, ent, tl, ti = token_logprobs(x, ids, top)
    wl, we, wt, wi = want(x, ids, top)
    close(lp, wl)
    close(ent, we)
    if top:
        assert torch.equal(ti, wi)
        close(tl, wt)
    else:
        assert tl is None and ti is None
    again = token_logprobs(x, ids, top)
    assert torch.equal(lp, again[0]) and torch.equal(ent, again[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(600, 1025, 3), (601, 8192, 32), (600, 8193, 32), (593, 20001, 6), (600, 33000, 5),
                                            (3, 1024, 9), (3, 1025, 9), (2, 1500, 0)])
def test_many_rows_and_the_lengths_where_the_split_changes(dtype, rows, vocab, top):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (2 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype)
    x[0] = 1.5  # ties alone
    x[1, : vocab - 2] = float("-inf")
    ids = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    ids[1] = vocab - 1
    lp, ent, tl, ti = token_logprobs(x, ids, top)
    wl, we, wt, wi = want(x, ids, top)
    close(lp, wl)
    close(ent, we)
    if top:
        assert torch.equal(ti, wi)
        seen = wt > float("-inf")  # row 1 has two values
        close(tl[seen], wt[seen])
        assert torch.equal(tl > float("-inf"), seen)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [300, 6001, 40000])
def test_unaligned_strided_rows_and_ties(dtype, vocab):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    buf = torch.randint(-3, 4, (5, vocab + 13), generator=g, device="cuda").to(dtype)  # seven values: ties everywhere
    for off in (0, 1, 3, 5):
        x = buf[:, off:off + vocab]
        ids = torch.randint(0, vocab, (5,), generator=g, device="cuda")
        lp, ent, tl, ti = token_logprobs(x, ids, 32)
        wl, we, wt, wi = want(x, ids, 32)
        close(lp, wl), close(ent, we), close(tl, wt)
        assert torch.equal(ti, wi)


@pytest.mark.parametrize("order", ["up", "down", "flat"])
@pytest.mark.parametrize("vocab", [1000, 50001])
def test_sorted_and_flat_rows(order, vocab):
    x = torch.arange(vocab, device="cuda", dtype=torch.float32)[None] / vocab
    x = {"up": x, "down": -x, "flat": x * 0 + 5}[order].contiguous()
    ids = torch.tensor([vocab // 2], device="cuda")
    lp, ent, tl, ti = token_logprobs(x, ids, 20)
    wl, we, wt, wi = want(x, ids, 20)
    close(lp, wl), close(ent, we), close(tl, wt)
    assert torch.equal(ti, wi)


@pytest.mark.parametrize("vocab", [512, 100352])
@pytest.mark.parametrize("mask", [float("-inf"), torch.finfo(torch.float32).min])
def test_masked_vocabularies(vocab, mask):
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.full((4, vocab), mask, device="cuda")
    keep = torch.tensor([3, 17, vocab - 1], device="cuda")
    x[0, keep] = torch.tensor([1.0, 2.0, 0.5], device="cuda")
    x[1, 100] = -7.0
    x[2] = torch.randn(vocab, generator=g, device="cuda")
    x[2, ::2] = mask
    ids = torch.tensor([17, 100, 1, 0], device="cuda")
    lp, ent, tl, ti = token_logprobs(x, ids, 5)
    wl, we, wt, wi = want(x, ids, 5)
    close(lp[:3], wl[:3]), close(ent[:3], we[:3])
    assert torch.equal(ti, wi)
    assert torch.equal(tl[0, 3:], wt[0, 3:].float())  # -inf stays -inf, the lowest value its distance
    if mask == float("-inf"):
        assert torch.isnan(lp[3]) and torch.isnan(ent[3])  # nothing has a probability
    else:
        close(lp[3:], wl[3:]), close(ent[3:], we[3:])


@pytest.mark.parametrize("vocab", [512, 100352])
def test_certain_tokens_keep_the_small_rest(vocab):
    """p = 1 - 1e-11: log p and the entropy are tiny and keep their relative precision (2^-15 of it, not of 1)."""
    x = torch.full((1, vocab), -20.0, device="cuda")
    x[0, 7] = 20.0
    lp, ent, _, _ = token_logprobs(x, torch.tensor([7], device="cuda"), 0)
    rest = (vocab - 1) * np.exp(-40.0)
    assert abs(lp.item() + np.log1p(rest)) <= 2.0**-15 * rest
    assert abs(ent.item() - (np.log1p(rest) + 40 * rest / (1 + rest))) <= 2.0**-15 * 41 * rest


@pytest.mark.parametrize("vocab", [512, 20000])
def test_non_finite_rows_and_ids_outside(vocab):
    x = torch.randn(5, vocab, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x[0, 5] = float("nan")
    x[1, 9] = float("inf")
    x[4, vocab - 1] = float("nan")
    x[4, 11] = float("inf")
    ids = torch.tensor([0, 9, -1, vocab, 0], device="cuda")
    lp, ent, tl, ti = token_logprobs(x, ids, 3)
    assert torch.isnan(lp).all() and torch.isnan(ent[[0, 1, 4]]).all() and not torch.isnan(ent[2:4]).any()
    assert ti[0, 0] == 5 and ti[1, 0] == 9 and ti[4, :2].tolist() == [vocab - 1, 11]
    assert torch.isnan(tl[[0, 1, 4]]).all() and not torch.isnan(tl[2:4]).any()
    out = torch.zeros(2, dtype=torch.long, device="cuda")
    for r in range(5):  # the first alternative is the decode step's argmax
        assert decode_finish(x[r].contiguous(), None, out)[0] == ti[r, 0]


def test_no_ids_no_rows():
    x = torch.randn(3, 50, device="cuda")
    lp, ent, tl, ti = token_logprobs(x, None, 2)
    assert lp is None and ent.shape == (3,) and torch.equal(ti[:, 0], x.argmax(1))
    lp, ent, tl, ti = token_logprobs(x[:0], torch.zeros(0, dtype=torch.long, device="cuda"), 2)
    assert lp.shape == (0,) and ti.shape == (0, 2)


def test_captured_and_replayed():
    x = torch.randn(6, 9000, device="cuda")
    ids = torch.arange(6, device="cuda")
    token_logprobs(x, ids, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = token_logprobs(x, ids, 4)
    x.copy_(torch.randn(6, 9000, device="cuda"))
    ids.add_(100)
    graph.replay()
    for a, b in zip(got, token_logprobs(x, ids, 4)):
        assert torch.equal(a, b)


def test_rows_more_than_32_bits_apart():
    x = torch.empty(3, 2**31 + 64, dtype=torch.bfloat16, device="cuda")[:, :3000]
    x.copy_(torch.randn(3, 3000, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda"))
    ids = torch.tensor([0, 2999, 17], device="cuda")
    for a, b in zip(token_logprobs(x, ids, 4), token_logprobs(x.contiguous(), ids, 4)):
        assert torch.equal(a, b)
