"""int8 weight-only GEMV (one activation row), the per-row int8 quantizer, and the int8 x int8 product.

Same API as byteprof/quant/triton_int8.py:33-55: `gemv_int8(x, w, scale, cfg=None, out=None)`
and `quantize_rowwise_int8(w)`. The GEMV runs the skinny kernel family with M = 1
(bp_gemv_int8); `cfg` is accepted and ignored.

Beyond byteprof: the product in 8-bit integers for any number of rows (csrc/int8_mm.cu, int8_mm_tc.cu), the
activations quantized too, one scale per token: `quantize_tokens_int8(x)`, `int8_mm(q, scale, w, w_scale)`, and both in
one call, `int8_linear(x, w, w_scale)`.
"""

from __future__ import annotations

import torch

from .. import _lib

DEFAULT_CFG = (2, 1024, 2)  # the reference's Triton (BN, BK, warps); no meaning for the B200 kernel


def default_cfg(n_out: int) -> tuple[int, int, int]:
    return (2, 512, 2) if n_out <= 1024 else DEFAULT_CFG


def gemv_int8(x: torch.Tensor, w: torch.Tensor, scale: torch.Tensor, cfg: tuple[int, int, int] | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """x: [1, K] bf16, w: [N, K] int8, scale: [N] bf16 -> [1, N] (dtype of `out`, default x.dtype)."""
    n, k = w.shape
    if x.numel() != k:
        raise ValueError(f"x must hold one row of K = {k} values, got shape {tuple(x.shape)}")
    if w.dtype != torch.int8 or scale.numel() != n:
        raise ValueError("w must be int8 [N, K] and scale [N]")
    if x.dtype != torch.bfloat16:
        raise ValueError(f"x must be bf16, got {x.dtype}")
    y = out if out is not None else torch.empty(1, n, dtype=x.dtype, device=x.device)
    if y.numel() != n or not y.is_contiguous():
        raise ValueError("out must be a contiguous [1, N] tensor")
    if n == 0:
        return y
    _lib.require_cuda(x, w, scale, y)
    x = x.contiguous()
    if scale.dtype != torch.bfloat16:
        scale = scale.to(torch.bfloat16)
    with _lib.on_device(x):
        ws, ws_bytes = _lib.skinny_workspace(x.device, 1, n, k, _lib.BP_DTYPE_INT8)
        _lib.call("bp_gemv_int8", x.data_ptr(), w.contiguous().data_ptr(), scale.contiguous().data_ptr(), y.data_ptr(),
                  _lib.dtype_code(y.dtype), n, k, ws, ws_bytes, _lib.stream_of(x))
    return y


def quantize_rowwise_int8(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Symmetric per-output-row int8: w ~ q * scale[:, None]; scale in the weight's dtype.

    The scale max|row| / 127 (clamped below at 1e-12) is rounded to the weight dtype before q is
    computed, so q is quantized against the scale that is stored (byteprof/quant/triton_int8.py:50-55).
    Offline weight preparation: runs wherever w lives."""
    wf = w.float()
    scale = (wf.abs().amax(dim=1) / 127.0).clamp_min(1e-12).to(w.dtype)
    q = torch.round(wf / scale.float()[:, None]).clamp_(-127, 127).to(torch.int8)
    return q.contiguous(), scale


def _rows_of(name: str, t: torch.Tensor) -> int:
    """The row stride of a 2-D tensor with unit column stride."""
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D")
    rows, cols = t.shape
    ld, one = t.stride()
    if one != 1 and cols > 1:
        raise ValueError(f"{name} must have unit column stride")
    if rows <= 1:
        return (cols + 15) // 16 * 16  # one row: its stride means nothing
    if ld < cols:
        raise ValueError(f"{name}'s rows overlap")
    return ld


def quantize_tokens_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x bf16 [M, K] (rows may be strided) -> (q int8 [M, K], scale fp32 [M]): scale = max(max|row| / 127, 1e-12) and
    q = rint(row / scale). A row holding Inf or NaN gets a NaN scale. q's rows start at multiples of 16 bytes."""
    if x.dtype != torch.bfloat16:
        raise ValueError("x must be bf16 [M, K]")
    ldx = _rows_of("x", x)
    m, k = x.shape
    q = torch.empty(m, -(-k // 16) * 16, dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    _lib.launch(_lib.device_of(x), "bp_quantize_rows_int8", x.data_ptr(), ldx, q.data_ptr(), q.shape[1], scale.data_ptr(), m, k)
    return q[:, :k], scale


def _operands(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias, out, m: int, k: int):
    """Checks the weights' side of a product with x; returns (device, ldw, w_scale's code, y, ldy, y's code)."""
    if w.dtype is not torch.int8:
        raise ValueError("w must be int8 [N, K]")
    ldw = _rows_of("w", w)
    n, kw = w.shape
    if kw != k:
        raise ValueError(f"the operands must agree on K, got {k} and {kw}")
    wsd = _SCALE_CODE.get(w_scale.dtype)
    if wsd is None or w_scale.shape != (n,) or not w_scale.is_contiguous():
        raise ValueError("w_scale must be a contiguous bf16 or fp32 [N]")
    if bias is not None and (bias.dtype is not torch.bfloat16 or bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous bf16 [N]")
    if out is not None and (out.dtype not in _SCALE_CODE or out.shape != (m, n)):
        raise ValueError(f"out must be bf16 or fp32 [{m}, {n}]")
    dev = _lib.device_of(x, w, w_scale, bias, out)
    if out is None:
        return dev, ldw, wsd, x.new_empty((m, n), dtype=torch.bfloat16), n, _lib.BP_DTYPE_BF16
    return dev, ldw, wsd, out, _rows_of("out", out), _SCALE_CODE[out.dtype]


_SCALE_CODE = {torch.bfloat16: _lib.BP_DTYPE_BF16, torch.float32: _lib.BP_DTYPE_F32}


def int8_mm(q: torch.Tensor, scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """q int8 [M, K] with fp32 scale [M], w int8 [N, K] with bf16 or fp32 w_scale [N], bias bf16 [N] or None ->
    scale[m] * w_scale[n] * sum_k q w + bias [M, N] (bf16, or the type of `out`: bf16 or fp32). The integer sum is
    exact; one rounding at the end."""
    if q.dtype != torch.int8:
        raise ValueError("q must be int8 [M, K]")
    ldq = _rows_of("q", q)
    m, k = q.shape
    if scale.dtype != torch.float32 or scale.shape != (m,) or not scale.is_contiguous() or scale.device != q.device:
        raise ValueError("scale must be a contiguous fp32 [M] on q's device")
    dev, ldw, wsd, y, ldy, yd = _operands(q, w, w_scale, bias, out, m, k)
    _lib.launch(dev, "bp_int8_mm", q.data_ptr(), ldq, scale.data_ptr(), w.data_ptr(), ldw, w_scale.data_ptr(), wsd,
                _lib.ptr(bias), y.data_ptr(), ldy, yd, m, w.shape[0], k)
    return y


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """x bf16 [M, K] times int8 weights [N, K] with both operands in 8 bits: `quantize_tokens_int8`, then `int8_mm`, in
    one call of the library (the same bits)."""
    if x.dtype != torch.bfloat16:
        raise ValueError("x must be bf16 [M, K]")
    ldx = _rows_of("x", x)
    m, k = x.shape
    dev, ldw, wsd, y, ldy, yd = _operands(x, w, w_scale, bias, out, m, k)
    need = (4 * m + 255) // 256 * 256 + m * ((k + 15) // 16 * 16)  # bp_int8_linear_workspace_bytes
    ws = x.new_empty((need + 1) // 2)
    _lib.launch(dev, "bp_int8_linear", x.data_ptr(), ldx, w.data_ptr(), ldw, w_scale.data_ptr(), wsd, _lib.ptr(bias),
                y.data_ptr(), ldy, yd, m, w.shape[0], k, ws.data_ptr(), need)
    return y
