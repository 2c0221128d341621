"""Refusals of the prompt operators before any device work: the C ABI's status codes and the Python checks."""

import ctypes

import pytest
import torch

from byteprof_b200 import _lib
from byteprof_b200.optim.decode_ops import token_logprobs
from byteprof_b200.optim.paged import PagedCache
from byteprof_b200.quant.int8 import int8_linear, int8_mm, quantize_tokens_int8

P = ctypes.c_void_p(256)
BF16 = torch.bfloat16


def attention(**kw):
    a = dict(q=P, ldq=256, k=P, v=P, num_pages=4, page_size=16, pages=P, ld_pages=4, max_pages=4, q_start=P, kv_len=P,
             seqs=1, rows=1, nh=2, nkv=2, hd=128, scale=0.1, out=P, ldo=256, ws=P, ws_bytes=0, stream=None)
    a.update(kw)
    return _lib.lib().bp_paged_attention(*a.values()), _lib.lib().bp_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(rows=-1), 1, b"negative"), (dict(nh=3), 1, b"multiple"), (dict(nkv=0), 1, b"multiple"), (dict(nh=2048, nkv=1), 1, b"1024"),
    (dict(hd=96), 2, b"head_dim"), (dict(page_size=24), 2, b"page_size"), (dict(page_size=4), 2, b"page_size"),
    (dict(page_size=512), 2, b"page_size"), (dict(rows=1 << 21), 2, b"2^20"), (dict(num_pages=0), 1, b"no pages"),
    (dict(num_pages=1 << 27), 2, b"2^31"), (dict(q=None), 1, b"NULL"), (dict(pages=None), 1, b"NULL"),
    (dict(ldq=255), 1, b"strides"), (dict(ld_pages=3), 1, b"strides"), (dict(scale=0.0), 1, b"scale"),
    (dict(scale=float("nan")), 1, b"scale"), (dict(q=ctypes.c_void_p(264)), 3, b"aligned"), (dict(ldo=260), 3, b"aligned"),
    (dict(rows=0, q=None), 0, b""), (dict(seqs=0, pages=None), 0, b"")])
def test_attention_statuses(kw, status, msg):
    st, err = attention(**kw)
    assert st == status and msg in err


def append(**kw):
    a = dict(qkv=P, ldqkv=768, qn=P, kn=P, cos=P, sin=P, max_pos=64, pages=P, ld_pages=4, max_pages=4, q_start=P, kv_len=P,
             seqs=1, rows=1, k=P, v=P, num_pages=4, page_size=16, nh=2, nkv=2, hd=128, eps=1e-6, q=P, ldq=256, stream=None)
    a.update(kw)
    return _lib.lib().bp_paged_append(*a.values()), _lib.lib().bp_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(seqs=-1), 1, b"negative"), (dict(hd=80), 2, b"head_dim"), (dict(page_size=12), 2, b"page_size"), (dict(qn=None), 1, b"both"),
    (dict(sin=None), 1, b"both"), (dict(ldqkv=767), 1, b"strides"), (dict(ldqkv=772), 3, b"aligned"),
    (dict(k=ctypes.c_void_p(8)), 3, b"aligned"), (dict(rows=0, qkv=None), 0, b"")])
def test_append_statuses(kw, status, msg):
    st, err = append(**kw)
    assert st == status and msg in err


def mm(**kw):
    a = dict(x=P, ldx=64, xs=P, w=P, ldw=64, ws=P, wsd=0, bias=None, y=P, ldy=8, yd=0, M=2, N=8, K=64, stream=None)
    a.update(kw)
    return _lib.lib().bp_int8_mm(*a.values()), _lib.lib().bp_last_error()


@pytest.mark.parametrize("kw,status,msg", [
    (dict(M=-1), 1, b"negative"), (dict(yd=2), 1, b"output dtype"), (dict(wsd=3), 1, b"scale dtype"), (dict(y=None), 1, b"NULL"),
    (dict(ldx=63), 1, b"strides"), (dict(ldy=7), 1, b"strides"), (dict(K=131072, ldx=131072, ldw=131072), 2, b"131071"),
    (dict(xs=ctypes.c_void_p(258)), 3, b"alignment"), (dict(M=0, y=None), 0, b""), (dict(N=0, y=None), 0, b"")])
def test_int8_statuses(kw, status, msg):
    st, err = mm(**kw)
    assert st == status and msg in err


def test_quantizer_and_logprobs_statuses():
    L = _lib.lib()
    need = L.bp_int8_linear_workspace_bytes(3, 50)
    assert need == 256 + 3 * 64 and L.bp_int8_linear_workspace_bytes(0, 50) == 0
    lin = (P, 50, P, 50, P, 0, None, P, 8, 0, 3, 8, 50)
    assert L.bp_int8_linear(*lin, P, need - 1, None) == 1 and b"workspace" in L.bp_last_error()
    assert L.bp_int8_linear(*lin, ctypes.c_void_p(264), need, None) == 3
    assert L.bp_int8_linear(*lin[:10], 0, 8, 50, None, 0, None) == 0
    assert L.bp_quantize_rows_int8(P, 63, P, 64, P, 2, 64, None) == 1
    assert L.bp_quantize_rows_int8(None, 64, P, 64, P, 2, 64, None) == 1
    assert L.bp_quantize_rows_int8(None, 0, None, 0, None, 0, 64, None) == 0
    args = dict(x=P, ld=100, dt=1, ids=P, lp=P, ent=P, tl=P, ti=P, rows=2, vocab=100, top=5, stream=None)

    def lp(**kw):
        return L.bp_token_logprobs(*{**args, **kw}.values())
    assert lp(dt=2) == 1 and lp(top=33) == 1 and lp(top=5, vocab=4) == 1 and lp(ld=99) == 1 and lp(ids=None) == 1
    assert lp(ent=None) == 1 and lp(tl=None) == 1 and lp(vocab=0, top=0) == 1 and lp(rows=0) == 0
    assert lp(x=ctypes.c_void_p(258)) == 3 and lp(ti=ctypes.c_void_p(260)) == 3


def test_python_refusals():
    z = torch.zeros(2, 16, 2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="contiguous bf16"):
        PagedCache(z.float(), z.float())
    with pytest.raises(ValueError, match="contiguous bf16"):
        PagedCache(z.transpose(1, 2), z.transpose(1, 2))
    with pytest.raises(ValueError, match="same shape"):
        PagedCache(z, z[:1])
    with pytest.raises(ValueError, match="page_size"):
        PagedCache(z[:, :12].contiguous(), z[:, :12].contiguous())
    with pytest.raises(ValueError, match="head_dim"):
        PagedCache(*(torch.zeros(2, 16, 2, 96, dtype=BF16),) * 2)
    with pytest.raises(ValueError, match="multiple"):
        PagedCache.over(torch.zeros(100, 2, 64, dtype=BF16), torch.zeros(100, 2, 64, dtype=BF16))
    c = PagedCache.over(torch.zeros(128, 2, 64, dtype=BF16), torch.zeros(128, 2, 64, dtype=BF16))
    assert (c.num_pages, c.page_size, c.nkv, c.hd) == (2, 64, 2, 64)
    i32 = dict(dtype=torch.int32)
    q, pages, st, kv = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(1, 2, **i32), torch.tensor([0, 3], **i32), torch.tensor([3], **i32)
    with pytest.raises(ValueError, match="CUDA"):
        c.attend(q, pages, st, kv)
    with pytest.raises(ValueError, match="int32"):
        c.attend(q, pages.long(), st, kv)
    with pytest.raises(ValueError, match="agree"):
        c.attend(q, pages, st[:1], kv)
    with pytest.raises(ValueError, match="multiple"):
        c.attend(q[:, :3], pages, st, kv)
    with pytest.raises(ValueError, match="bf16"):
        c.attend(q.float(), pages, st, kv)
    with pytest.raises(ValueError, match="contiguous"):
        c.attend(q.transpose(1, 2).contiguous().transpose(1, 2), pages, st, kv)
    qkv = torch.zeros(3, 8 * 64, dtype=BF16)
    with pytest.raises(ValueError, match="qkv"):
        c.append(qkv[:, :-1], 4, pages, st, kv)
    with pytest.raises(ValueError, match="together"):
        c.append(qkv, 4, pages, st, kv, q_norm=torch.zeros(256, dtype=BF16))
    with pytest.raises(ValueError, match="norm weights"):
        c.append(qkv, 4, pages, st, kv, torch.zeros(255, dtype=BF16), torch.zeros(128, dtype=BF16))
    with pytest.raises(ValueError, match="cos and sin"):
        c.append(qkv, 4, pages, st, kv, cos=torch.zeros(8, 32), sin=torch.zeros(8, 31))
    i8 = torch.zeros(3, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="agree on K"):
        int8_mm(i8, torch.ones(3), i8[:, :32], torch.ones(3))
    with pytest.raises(ValueError, match="scale must"):
        int8_mm(i8, torch.ones(3, dtype=torch.float64), i8, torch.ones(3))
    with pytest.raises(ValueError, match="w_scale"):
        int8_mm(i8, torch.ones(3), i8, torch.ones(2))
    with pytest.raises(ValueError, match="bias"):
        int8_mm(i8, torch.ones(3), i8, torch.ones(3), torch.ones(3))
    with pytest.raises(ValueError, match="out must be"):
        int8_mm(i8, torch.ones(3), i8, torch.ones(3), out=torch.zeros(3, 4))
    with pytest.raises(ValueError, match="overlap"):
        int8_mm(i8[:1].expand(3, 64), torch.ones(3), i8, torch.ones(3))
    with pytest.raises(ValueError, match="CUDA"):
        int8_mm(i8, torch.ones(3), i8, torch.ones(3))
    with pytest.raises(ValueError, match="bf16"):
        quantize_tokens_int8(torch.zeros(3, 8))
    x16, one = torch.zeros(3, 64, dtype=BF16), torch.ones(3)
    for call in (lambda: quantize_tokens_int8(x16[0]), lambda: int8_linear(x16[0], i8, one)):
        with pytest.raises(ValueError, match="2-D"):
            call()
    with pytest.raises(ValueError, match="unit column"):
        int8_linear(x16.t().contiguous().t(), i8, one)
    with pytest.raises(ValueError, match="bf16 or fp32"):
        int8_linear(x16, i8, one, out=torch.zeros(3, 3, dtype=torch.int8))
    with pytest.raises(ValueError, match="CUDA"):
        int8_linear(x16, i8, one)
    x = torch.zeros(2, 9)
    with pytest.raises(ValueError, match="top"):
        token_logprobs(x, None, 10)
    with pytest.raises(ValueError, match="ids"):
        token_logprobs(x, torch.zeros(2), 1)
    with pytest.raises(ValueError, match="bf16 or fp32"):
        token_logprobs(x.half(), None)
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(x, torch.zeros(2, dtype=torch.long))
