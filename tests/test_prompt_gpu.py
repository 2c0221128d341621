"""A prompt in one pass through the framework's own paths: BolmoDecoder.prefill and score (local scans, GlobalBlock.chunk
over the decoder's caches, int8 products, token_logprobs), and Int8Linear with 8-bit activations.

The prompt pass and the byte loop round to bf16 at the same places but sum in other orders (and the loop rounds k once
more), so neither is the other's reference: both are compared with the fp32 decoder of the same weights, and the
prompt pass may be at most twice as far from it as the loop."""

import numpy as np
import pytest
import torch
import torch.nn as nn

from byteprof_b200 import _lib
from byteprof_b200.optim.bolmo_e2e import BolmoDecoder, GlobalBlock
from byteprof_b200.optim.decode_ops import rope_tables, token_logprobs
from byteprof_b200.optim.paged import PagedCache
from byteprof_b200.quant.int8 import int8_linear, quantize_rowwise_int8
from byteprof_b200.quant.integrate import Int8Linear, apply_quantization

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
SMALL = dict(d=512, local_heads=4, local_dh=128, local_ffn=704, global_layers=3, global_heads=4, global_ffn=1024,
             max_patches=128, fused_glob=False, fused_local=False)


def text(n, seed=0):
    return np.random.RandomState(seed).randint(0, 256, n).tolist()


def fed(dec, ids, opened):
    rows = []
    for b, o in zip(ids, opened):
        dec.feed(b, o)
        rows.append(dec.logits[0].double().clone())
    return torch.stack(rows)


@pytest.mark.parametrize("n", [1, 2, 40, 150])
def test_prefill_is_as_near_to_fp32_as_the_byte_loop(n):
    ids = text(n + 6)
    chunk, loop, exact = (BolmoDecoder(precision=p, **SMALL) for p in ("bf16", "bf16", "fp32"))
    logits, flags, opened = chunk.prefill(ids[:n])
    assert logits.shape == (n, 512) and opened[0] and opened[1:] == flags[:-1] and chunk.patches == sum(opened)
    want, step = fed(exact, ids[:n], opened), fed(loop, ids[:n], opened)
    e_chunk, e_loop = (logits.double() - want).norm().item(), (step - want).norm().item()
    assert e_chunk <= 2 * e_loop, (e_chunk, e_loop)
    # the loop goes on behind the prompt
    more = [flags[-1], True, False, True, True, False]
    want, step, cont = (fed(d, ids[n:], more) for d in (exact, loop, chunk))
    assert (cont - want).norm() <= 2 * (step - want).norm()
    assert chunk.patches == loop.patches and int(chunk.pos) == int(loop.pos)


def test_two_prefills_continue_each_other_and_reset():
    ids = text(90, 3)
    a, b = BolmoDecoder(**SMALL), BolmoDecoder(**SMALL)
    whole, flags, opened = a.prefill(ids)
    first, f1, o1 = b.prefill(ids[:33])
    second, f2, o2 = b.prefill(ids[33:], first_patch=f1[-1])
    got = torch.cat([first, second])
    # the same model in two cuts: other row counts, the same roundings; a flag near its threshold may differ
    if o1 + o2 == opened:
        exact = BolmoDecoder(precision="fp32", **SMALL)
        want = fed(exact, ids, opened)
        assert (got.double() - want).norm() <= 2 * (whole.double() - want).norm()
    b.reset()
    again, _, _ = b.prefill(ids)
    assert torch.equal(again, whole)


def test_score_is_the_log_softmax_of_the_prefill():
    ids = text(80, 5)
    dec = BolmoDecoder(**SMALL)
    lp, ent, tl, ti = dec.score(ids, top=5)
    dec.reset()
    logits, _, _ = dec.prefill(ids)
    z = torch.log_softmax(logits[:-1].double(), 1)
    nxt = torch.tensor(ids[1:], device="cuda")
    # (tolerance: tests/test_logprobs_gpu.py)
    assert ((lp.double() - z.gather(1, nxt[:, None])[:, 0]).abs() <= 2.0**-15 + 2.0**-22 * z.abs().max()).all()
    assert ((ent.double() + (z.exp() * z).sum(1)).abs() <= 2.0**-15 + 2.0**-22 * 7).all()
    assert torch.equal(ti, torch.sort(logits[:-1], dim=1, descending=True, stable=True)[1][:, :5])


def test_prefill_in_8_bits_stays_near():
    """Rounding x and w to 8 bits (step amax / 127, amax at most 4.5 standard deviations of a row) adds at most 1.5 % to
    each of the 4 products of 3 blocks, which add up like independent errors: 1.5 % * sqrt(2 * 12) = 7 % at the patch
    values; the logits see them beside the exact local path."""
    ids = text(120, 7)
    a, b = BolmoDecoder(**SMALL), BolmoDecoder(**SMALL)
    b.quantize_prompt()
    x, _, _ = a.prefill(ids)
    y, _, _ = b.prefill(ids)
    assert not torch.equal(x, y)
    assert (x - y).norm() <= 0.07 * x.norm()


def test_a_prompt_that_does_not_fit_changes_nothing():
    ids = text(60, 9)
    a = BolmoDecoder(**{**SMALL, "max_patches": 16})
    b = BolmoDecoder(**{**SMALL, "max_patches": 16})
    with pytest.raises(RuntimeError, match="patches"):
        a.prefill(ids)
    assert a.patches == 0 and a.parity == 0
    assert torch.equal(fed(a, ids[:4], [True, False, True, False]), fed(b, ids[:4], [True, False, True, False]))
    with pytest.raises(ValueError, match="first byte"):
        BolmoDecoder(**SMALL).prefill(ids, first_patch=False)
    with pytest.raises(ValueError, match="byte ids"):
        b.prefill([600])
    with pytest.raises(ValueError, match="bf16"):
        BolmoDecoder(precision="fp32", **SMALL).prefill(ids)
    with pytest.raises(ValueError, match="two bytes"):
        b.score([1])


def test_a_cache_of_no_whole_pages_is_refused_and_nothing_changes():
    ids = text(5, 11)
    a = BolmoDecoder(**{**SMALL, "max_patches": 20})
    b = BolmoDecoder(**{**SMALL, "max_patches": 20})
    with pytest.raises(ValueError, match="multiple of 8"):
        a.prefill(ids)
    opened = [True, False, True, True, False]
    assert torch.equal(fed(a, ids, opened), fed(b, ids, opened))


def test_a_block_takes_packed_sequences_and_single_tokens():
    """Three prompts packed into one chunk equal the three by themselves, within the rounding of the block's bf16 output,
    and a further token each (the few-row kernels) equals the longer prompts' last rows within what 8-bit activations
    make of it: an attention output that another order of sums moves by d (a bf16 rounding of it, in the mean half of its
    largest: 2^-9 * 0.8 sigma) moves its 8-bit code by a whole step s = amax / 127 (0.035 sigma at amax = 4.5) with probability d / s, so
    the product's inputs differ by sqrt(d s) = 0.0075 sigma in the root mean square; the block's three products in a row
    make sqrt(3) of that, 0.013 sigma: 0.8 * 0.013 / 0.8 = 0.013 of the mean, under 2^-6."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(1)
    blk = GlobalBlock(512, 4, 1024, 64, gen, dev)
    blk.quantize_prompt()
    cos, sin = rope_tables(256, 128, 500000.0, dev)
    lens = [70, 1, 133]
    xs = [torch.randn(n + 1, 512, generator=gen, device=dev).to(BF16) for n in lens]
    pages = torch.arange(24, dtype=torch.int32, device=dev).view(3, 8)[:, torch.randperm(8, device=dev)]

    def run(cache, which, rows, kv):
        start = torch.tensor([0] + np.cumsum([r.shape[0] for r in rows]).tolist(), dtype=torch.int32, device=dev)
        return blk.chunk(torch.cat(rows), cache, pages[which].contiguous(), start, torch.tensor(kv, dtype=torch.int32, device=dev), cos, sin)

    caches = [PagedCache.zeros(24, 32, 4, 128, dev) for _ in range(2)]
    packed = run(caches[0], [0, 1, 2], [x[:-1] for x in xs], lens)
    alone = torch.cat([run(caches[1], [i], [x[:-1]], [n]) for i, (x, n) in enumerate(zip(xs, lens))])
    assert torch.equal(caches[0].k_pages, caches[1].k_pages) and torch.equal(caches[0].v_pages, caches[1].v_pages)
    scale = alone.double().abs().mean()
    assert (packed.double() - alone.double()).abs().mean() <= 2.0**-7 * scale
    step = run(caches[0], [0, 1, 2], [x[-1:] for x in xs], [n + 1 for n in lens])
    full = PagedCache.zeros(24, 32, 4, 128, dev)
    want = [run(full, [i], [x], [n + 1])[-1:] for i, (x, n) in enumerate(zip(xs, lens))]
    assert (step.double() - torch.cat(want).double()).abs().mean() <= 2.0**-6 * scale
    assert torch.equal(caches[0].k_pages, full.k_pages)


def test_prompt_operators_run_on_a_side_stream_and_in_a_graph():
    """append, attend, int8_linear and token_logprobs as one captured pass, replayed with new inputs."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(2)
    nh, nkv, hd, t, vocab = 8, 2, 64, 50, 700
    cache = PagedCache.zeros(16, 16, nkv, hd, dev)
    pages = torch.randperm(16, device=dev).int()[None]
    start, kv = torch.tensor([0, t], dtype=torch.int32, device=dev), torch.tensor([t], dtype=torch.int32, device=dev)
    cos, sin = rope_tables(256, hd, 10000.0, dev)
    w, ws = quantize_rowwise_int8((torch.randn(vocab, nh * hd, generator=gen, device=dev) * 0.05).to(BF16))
    qkv = torch.randn(t, (nh + 2 * nkv) * hd, generator=gen, device=dev).to(BF16)
    ids = torch.randint(0, vocab, (t,), generator=gen, device=dev)

    def run():
        q = cache.append(qkv, nh, pages, start, kv, None, None, cos, sin)
        y = int8_linear(cache.attend(q, pages, start, kv).view(t, nh * hd), w, ws)
        return token_logprobs(y, ids, 4)

    run()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        got = run()
    for i in range(3):
        qkv.copy_(torch.randn(t, (nh + 2 * nkv) * hd, generator=gen, device=dev))
        kv.fill_(t + 20 * i)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = run()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    assert _lib.device_errors() == 0


@pytest.mark.parametrize("bias", [None, BF16, torch.float32])
def test_int8_linear_module(bias):
    lin = nn.Linear(256, 300, bias=bias is not None, dtype=BF16, device="cuda")
    if bias is not None:
        lin.bias = nn.Parameter(lin.bias.detach().to(bias))
    m = Int8Linear(lin, act="int8")
    for shape in ((1, 256), (2, 5, 256), (130, 256), (0, 256)):
        x = torch.randn(*shape, device="cuda").to(BF16)
        y = m(x)
        assert y.shape == (*shape[:-1], 300)
        if x.numel():
            want = int8_linear(x.view(-1, 256), m.q, m.scale, lin.bias.detach() if bias == BF16 else None).view(y.shape)
            assert torch.equal(y, want + lin.bias if bias == torch.float32 else want)
    assert "int8 x int8" in repr(m)
    assert m(torch.randn(3, 256, device="cuda")).dtype == torch.float32 if bias != BF16 else True  # fp32: the dequantized product
    with pytest.raises(ValueError, match="act"):
        Int8Linear(lin, act="fp8")


def test_apply_quantization_with_8_bit_activations():
    """The scheme swaps the selected linears; the products are `int8_linear`'s."""
    model = nn.Module()
    model.model = nn.Module()
    model.model.layers = nn.ModuleList([nn.ModuleDict({"self_attn": nn.ModuleDict({"q_proj": nn.Linear(128, 96, bias=False)}),
                                                       "mlp": nn.ModuleDict({"down_proj": nn.Linear(256, 128, bias=False)})})])
    model.lm_head = nn.Linear(128, 64, bias=False)
    model.to("cuda", BF16)
    w = model.model.layers[0]["self_attn"]["q_proj"].weight.detach().clone()
    stats = apply_quantization(model, "blocks", "int8_w8a8")
    q_proj = model.model.layers[0]["self_attn"]["q_proj"]
    assert stats["n_linears"] == 2 and isinstance(model.lm_head, nn.Linear)
    assert isinstance(q_proj, Int8Linear) and q_proj.act == "int8"
    for rows in (1, 40, 300):
        x = torch.randn(rows, 128, device="cuda").to(BF16)
        assert torch.equal(q_proj(x), int8_linear(x, *quantize_rowwise_int8(w)))
