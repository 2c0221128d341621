"""The 8-bit product at the edges of what its documentation allows. Definition and tolerances: tests/test_int8_mm_gpu.py."""

import pytest
import torch
import torch.nn as nn
from test_int8_mm_gpu import check, ints, scales

from byteprof_b200 import _lib
from byteprof_b200.optim.decode_ops import token_logprobs
from byteprof_b200.quant.int8 import int8_linear, int8_mm, quantize_tokens_int8
from byteprof_b200.quant.integrate import Int8Linear

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_pairs_of_ctas_one_behind_the_other_and_beside_other_kernels():
    """Products on pairs of CTAs (more than 128 rows, enough tiles), each followed on the same SMs by kernels that lay their
    own barriers where the pair's were, from two streams: nothing of a pair may arrive after its end."""
    sets = []
    for i, (m, n, k) in enumerate([(700, 5000, 256), (300, 9000, 128), (1025, 4608, 144)]):
        q, s, w, ws = ints(m, k, 10 + i), scales(m, 20 + i), ints(n, k, 30 + i), scales(n, 40 + i, BF16)
        y = int8_mm(q, s, w, ws)
        check(y, q, s, w, ws)
        sets.append(((q, s, w, ws), y))
    logits = torch.randn(300, 30000, device="cuda").to(BF16)
    want = token_logprobs(logits, None, 3)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for r in range(60):
        with torch.cuda.stream(streams[r % 2]):
            args, y = sets[r % 3]
            got.append((int8_mm(*args), y, token_logprobs(logits, None, 3)))
    torch.cuda.synchronize()
    for y, ref, lp in got:
        assert torch.equal(y, ref)
        assert all(torch.equal(a, b) for a, b in zip(lp[1:], want[1:]))
    assert _lib.device_errors() == 0


@pytest.mark.parametrize("rows", [1, 2, 40, 300])
def test_the_module_takes_any_strides(rows):
    lin = nn.Linear(256, 96, bias=True, dtype=BF16, device="cuda")
    m = Int8Linear(lin, act="int8")
    x = torch.randn(256, rows, device="cuda").to(BF16)
    assert torch.equal(m(x.t()), m(x.t().contiguous()))                        # transposed
    wide = torch.randn(rows, 2, 512, device="cuda").to(BF16)
    for view in (wide[..., ::2], wide[..., :256], wide[:1].expand(rows, 2, 512)[..., 3:259], wide[0, 0, :256].expand(rows, 256)):
        y = m(view)
        assert y.shape == (*view.shape[:-1], 96) and torch.equal(y, m(view.contiguous()))


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("m", [1, 20, 100, 260, 1025])
def test_exactly_the_block_is_written(m, dtype):
    """Every width behind a multiple of 8, in rows that are 16-byte aligned: what lies behind the block stays."""
    k = 64
    for n in [*range(145, 161), 2039, 2042, 2044]:
        q, s, w, ws = ints(m, k, n), scales(m, 1), ints(n, k, 2), scales(n, 3, BF16)
        for ld in (-(-n // 8) * 8, -(-n // 8) * 8 + 8):
            buf = torch.full((m + 1, ld), 7.0, dtype=dtype, device="cuda")
            y = int8_mm(q, s, w, ws, out=buf[:m, :n])
            assert (buf[:m, n:] == 7).all() and (buf[m] == 7).all(), (n, ld)
            check(y, q, s, w, ws)


@pytest.mark.parametrize("m", [1, 20, 100, 300])
def test_what_lies_between_the_rows_does_not_count(m):
    """Every K behind a multiple of 16 in rows of 16-byte steps (the tensor cores' form), with values between the rows of both
    operands; and the bf16 rows of a fused call."""
    for k in [*range(1, 18), 100, 113, 127, 129, 2047]:
        ld = -(-k // 16) * 16
        q, w = ints(m, k, k, ld=ld + 16, lo=-128), ints(150, k, 7, ld=ld, lo=-128)
        s, ws = scales(m, 1), scales(150, 3, BF16)
        check(int8_mm(q, s, w, ws), q, s, w, ws)
        x = torch.randn(m, ld + 8, device="cuda").to(BF16)[:, :k]
        q2, s2 = quantize_tokens_int8(x)
        assert torch.equal(int8_linear(x, w, ws), int8_mm(q2, s2, w, ws))
        check(int8_mm(q2, s2, w, ws), q2, s2, w, ws)
