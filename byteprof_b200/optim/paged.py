"""Paged KV cache of an attention layer: its writer and the attention of new tokens over it (csrc/paged_append.cu,
paged_attn.cu, paged_attn_tc.cu).

`decode_ops.DecodeAttention` attends one position of one sequence over a static cache. `PagedCache` takes any
number of new positions of any number of sequences in one call: a prompt's chunk, drafted tokens, or a token each of
a batch of streams. Sequences are packed one behind the other in the rows of q; `q_start` int32 [S + 1] holds
their bounds, `kv_len` int32 [S] the cached length of each including its new rows, `pages` int32 [S, max_pages] the
page of every `page_size` positions. All three live on the device and are read there: nothing is planned on the host,
and a captured graph serves every length. bf16 only; CUDA tensors only; a missing library raises.
"""

from __future__ import annotations

import torch

from .. import _lib


_BF16, _I32, _F32 = torch.bfloat16, torch.int32, torch.float32


class PagedCache:
    """k_pages and v_pages [num_pages, page_size, n_kv_heads, head_dim], bf16 and contiguous (`PagedCache.zeros` makes
    them; `PagedCache.over` lays pages over a static [max_pos, n_kv_heads, head_dim] cache). page_size is a power of
    two from 8 to 256, head_dim 64 or 128."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor):
        for t in (k_pages, v_pages):
            if t.dtype != torch.bfloat16 or t.dim() != 4 or not t.is_contiguous():
                raise ValueError("pages must be contiguous bf16 [num_pages, page_size, n_kv_heads, head_dim]")
        if k_pages.shape != v_pages.shape or k_pages.device != v_pages.device:
            raise ValueError("k_pages and v_pages must have the same shape and device")
        self.num_pages, self.page_size, self.nkv, self.hd = k_pages.shape
        if self.page_size not in (8, 16, 32, 64, 128, 256):
            raise ValueError(f"page_size must be a power of two from 8 to 256, got {self.page_size}")
        if self.hd not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {self.hd}")
        self.k_pages, self.v_pages = k_pages, v_pages
        self._ws_bytes: dict[tuple[int, int, int, int], int] = {}

    @classmethod
    def zeros(cls, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device: torch.device) -> "PagedCache":
        return cls(*(torch.zeros(num_pages, page_size, n_kv_heads, head_dim, dtype=torch.bfloat16, device=device)
                     for _ in range(2)))

    @classmethod
    def over(cls, k_cache: torch.Tensor, v_cache: torch.Tensor, page_size: int = 64) -> "PagedCache":
        """The same memory as a static cache [max_pos, n_kv_heads, head_dim]: page i holds the positions i * page_size
        and up (max_pos a multiple of page_size; the page table of its one sequence is 0, 1, 2, ...)."""
        if k_cache.dim() != 3 or k_cache.shape[0] % page_size:
            raise ValueError(f"a [max_pos, n_kv_heads, head_dim] cache with max_pos a multiple of {page_size} expected")
        return cls(*(t.view(-1, page_size, *t.shape[1:]) for t in (k_cache, v_cache)))

    def _where(self, pages: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor) -> tuple[int, int, int]:
        """(S, max_pages, row stride of pages) of a call's tables."""
        if pages.dtype is not _I32 or pages.dim() != 2 or q_start.dtype is not _I32 or q_start.dim() != 1 or \
                kv_len.dtype is not _I32 or kv_len.dim() != 1:
            raise ValueError("pages [S, max_pages], q_start [S + 1] and kv_len [S] must be int32")
        seqs, width = pages.shape
        ld, one = pages.stride()
        if (one != 1 and width > 1) or q_start.stride(0) != 1 or (kv_len.stride(0) != 1 and seqs > 1):
            raise ValueError("pages, q_start and kv_len need unit stride along their last dimension")
        if q_start.shape[0] != seqs + 1 or kv_len.shape[0] != seqs:
            raise ValueError("pages [S, max_pages], q_start [S + 1] and kv_len [S] must agree on S")
        return seqs, width, ld if seqs > 1 else width

    def append(self, qkv: torch.Tensor, nh: int, pages: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, cos: torch.Tensor | None = None,
               sin: torch.Tensor | None = None, eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
        """qkv [T, (nh + 2 n_kv_heads) * head_dim] bf16 (rows may be strided), q | k | v of each new row: writes k
        and v to the pages of their positions and returns q [T, nh, head_dim]. q and k are RMS-normalised over their
        widths (q_norm [nh * head_dim], k_norm, bf16; None: not) and rotated (cos / sin fp32 [max_pos, head_dim / 2] as
        `decode_ops.rope_tables` makes them; None: not). A row whose position is outside the tables or the cache gives
        a NaN q and writes nothing; rows behind q_start[S] are left alone."""
        hd, nkv = self.hd, self.nkv
        if qkv.dtype is not _BF16 or qkv.dim() != 2 or qkv.shape[1] != (nh + 2 * nkv) * hd:
            raise ValueError(f"qkv must be bf16 [T, {(nh + 2 * nkv) * hd}]")
        rows, width = qkv.shape
        ldx, one = qkv.stride()
        if one != 1:
            raise ValueError("qkv must have unit column stride")
        seqs, max_pages, ldp = self._where(pages, q_start, kv_len)
        if (q_norm is None) != (k_norm is None) or (cos is None) != (sin is None):
            raise ValueError("q_norm and k_norm, and cos and sin, come together")
        qn = kn = cp = sp = None
        if q_norm is not None:
            if q_norm.dtype is not _BF16 or q_norm.numel() != nh * hd or not q_norm.is_contiguous() or \
                    k_norm.dtype is not _BF16 or k_norm.numel() != nkv * hd or not k_norm.is_contiguous():
                raise ValueError(f"norm weights must be contiguous bf16 of {nh * hd} and {nkv * hd} values")
            qn, kn = q_norm.data_ptr(), k_norm.data_ptr()
        max_pos = 0
        if cos is not None:
            max_pos = cos.shape[0]
            if cos.dtype is not _F32 or sin.dtype is not _F32 or cos.shape != (max_pos, hd // 2) or sin.shape != cos.shape or \
                    not cos.is_contiguous() or not sin.is_contiguous():
                raise ValueError("cos and sin must be contiguous fp32 [max_pos, head_dim / 2]")
            cp, sp = cos.data_ptr(), sin.data_ptr()
        dev = _lib.device_of(qkv, self.k_pages, pages, q_start, kv_len, q_norm, k_norm, cos, sin, out)
        if out is None:
            q, ldq = qkv.new_empty((rows, nh, hd)), nh * hd
        else:
            q, ldq = out, _head_rows("out", out, rows, nh, hd)
        _lib.launch(dev, "bp_paged_append", qkv.data_ptr(), ldx if rows > 1 else width, qn, kn, cp, sp, max_pos,
                    pages.data_ptr(), ldp, max_pages, q_start.data_ptr(), kv_len.data_ptr(), seqs, rows,
                    self.k_pages.data_ptr(), self.v_pages.data_ptr(), self.num_pages, self.page_size, nh, nkv, hd, eps,
                    q.data_ptr(), ldq)
        return q

    def attend(self, q: torch.Tensor, pages: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor,
               scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """q [T, nh, head_dim] bf16 -> [T, nh, head_dim]: causal attention of every row over its sequence's cached
        positions up to its own (softmax scale head_dim ** -0.5 unless given). A row that sees nothing gives zeros; a
        row that should see a page outside the cache gives NaN; rows behind q_start[S] are left alone."""
        if q.dim() != 3 or q.shape[2] != self.hd:
            raise ValueError(f"q must be [T, nh, {self.hd}]")
        rows, nh, hd = q.shape
        if nh % self.nkv or nh == 0:
            raise ValueError(f"nh = {nh} must be a multiple of n_kv_heads = {self.nkv}")
        seqs, max_pages, ldp = self._where(pages, q_start, kv_len)
        ldq = _head_rows("q", q, rows, nh, hd)
        dev = _lib.device_of(q, self.k_pages, pages, q_start, kv_len, out)
        if out is None:
            y, ldo = q.new_empty((rows, nh, hd)), nh * hd
        else:
            y, ldo = out, _head_rows("out", out, rows, nh, hd)
        need = self._ws_bytes.get((rows, seqs, nh, dev))
        if need is None:
            with torch.cuda.device(dev):
                need = int(_lib.lib().bp_paged_attention_workspace_bytes(rows, seqs, nh, self.nkv, hd))
            if len(self._ws_bytes) >= 1024:  # a server's batches have ever new sizes
                self._ws_bytes.clear()
            self._ws_bytes[(rows, seqs, nh, dev)] = need
        # scratch of this call alone, from torch's allocator: calls on several streams and captured graphs share none
        ws = q.new_empty(need // 2)
        _lib.launch(dev, "bp_paged_attention", q.data_ptr(), ldq, self.k_pages.data_ptr(), self.v_pages.data_ptr(),
                    self.num_pages, self.page_size, pages.data_ptr(), ldp, max_pages, q_start.data_ptr(), kv_len.data_ptr(),
                    seqs, rows, nh, self.nkv, hd, hd ** -0.5 if scale is None else scale, y.data_ptr(), ldo, ws.data_ptr(),
                    need)
        return y


def _head_rows(name: str, t: torch.Tensor, rows: int, nh: int, hd: int) -> int:
    """The row stride of a bf16 [rows, nh, hd] tensor whose rows are contiguous."""
    if t.dtype is not _BF16 or t.shape != (rows, nh, hd):
        raise ValueError(f"{name} must be bf16 [{rows}, {nh}, {hd}]")
    ld, lh, one = t.stride()
    if one != 1 or (nh > 1 and lh != hd):
        raise ValueError(f"{name} must have contiguous (heads, head_dim) rows")
    return ld if rows > 1 else nh * hd
