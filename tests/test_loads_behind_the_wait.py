"""A kernel that starts under the one before it (programmatic dependent launch) may read what that one writes only behind
its wait. `ldg16` and `ldg_stream16` are plain functions of an address to the compiler, which may move them above the
wait, so they are for constants; `ld16` stays where it is written. The sources are read for the first half; on the GPU,
each operand of the kind goes through a chain of early-started kernels over reused buffers."""

import re
from pathlib import Path

import pytest
import torch

CSRC = Path(__file__).resolve().parent.parent / "byteprof_b200" / "csrc"
BF16 = torch.bfloat16


def test_only_weights_are_loaded_by_movable_loads():
    weights = {"w", "wl"}
    seen = 0
    for f in sorted(CSRC.glob("*.cu")):
        text = f.read_text()
        if "pdl_wait_prior_grids();" not in text:
            continue
        for arg in re.findall(r"\bldg(?:_stream)?16\(\s*([A-Za-z_][\w.]*)", text):
            seen += 1
            assert arg in weights or arg.startswith("wr"), f"{f.name}: {arg} is loaded by a load that may move above the wait"
    assert seen > 0


def test_the_load_of_activations_cannot_move():
    text = (CSRC / "bp_common.cuh").read_text()
    body = text[text.index("uint4 ld16("):]
    body = body[:body.index("return r;")]
    assert "asm volatile(" in body and '"memory"' in body and ".nc" not in body


def pages_of(n, page, dev):
    return torch.arange(-(-n // page), dtype=torch.int32, device=dev)[None]


def consumers(dev):
    """name -> (width of the buffer that the kernel before writes, the consumer of [rows, width])."""
    from byteprof_b200.optim.bolmo_local import rmsnorm
    from byteprof_b200.optim.decode_ops import swiglu, token_logprobs
    from byteprof_b200.optim.paged import PagedCache
    from byteprof_b200.optim.skinny import skinny_mm
    from byteprof_b200.quant.int8 import int8_linear, quantize_rowwise_int8, quantize_tokens_int8

    g = torch.Generator(device=dev).manual_seed(1)
    nh, nkv, hd, page = 8, 2, 128, 16
    cache = PagedCache.zeros(8, page, nkv, hd, dev)
    cache.k_pages.normal_(generator=g)
    cache.v_pages.normal_(generator=g)
    table = pages_of(128, page, dev)
    w = (torch.randn(512, 1024, generator=g, device=dev) * 0.05).to(BF16)
    w8 = quantize_rowwise_int8(w)
    norm = torch.ones(1024, dtype=BF16, device=dev)

    def tables(t):
        return table, torch.tensor([0, t], dtype=torch.int32, device=dev), torch.tensor([100], dtype=torch.int32, device=dev)

    at = {t: tables(t) for t in (1, 4, 16)}

    def attend(x):
        return cache.attend(x.view(-1, nh, hd), *at[x.shape[0]])

    def append(x):
        own = PagedCache(cache.k_pages.clone(), cache.v_pages.clone())
        return own.append(x, nh, *at[x.shape[0]])

    return {
        "append": (nh * hd + 2 * nkv * hd, append), "attend": (nh * hd, attend),
        "int8_linear": (1024, lambda x: int8_linear(x, *w8)), "quantize": (1024, lambda x: quantize_tokens_int8(x)[0]),
        "norm": (1024, lambda x: rmsnorm(x, norm, 1e-6)), "swiglu": (1024, lambda x: swiglu(x)),
        "skinny": (1024, lambda x: skinny_mm(x, w)), "logprobs": (1024, lambda x: token_logprobs(x, None, 4)[2]),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 16])
@pytest.mark.parametrize("name", ["append", "attend", "int8_linear", "quantize", "norm", "swiglu", "skinny", "logprobs"])
def test_a_chain_over_one_buffer_equals_the_calls_apart(name, rows):
    from byteprof_b200.optim.skinny import skinny_mm

    dev = torch.device("cuda")
    width, consume = consumers(dev)[name]
    g = torch.Generator(device=dev).manual_seed(2)
    w = (torch.randn(width, 2048, generator=g, device=dev) * 0.05).to(BF16)
    xs = [torch.randn(rows, 2048, generator=g, device=dev).to(BF16) for _ in range(24)]
    buf = torch.empty(rows, width, dtype=BF16, device=dev)
    apart = []
    for x in xs:
        skinny_mm(x, w, out=buf)
        torch.cuda.synchronize()
        apart.append(consume(buf).clone())
        torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):  # back to back, each started under the one before
        chained = [consume(skinny_mm(x, w, out=buf)) for x in xs]
    for _ in range(3):
        buf.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(chained, apart))
