"""The product in 8-bit integers (csrc/int8_mm.cu, int8_mm_tc.cu) against integer arithmetic on the host.

Tolerance of y: the integer sum is exact; as fp32 it has one rounding (2^-24), the two scales and the bias one
each: 4 * 2^-24 of |value| (and of |bias| for the addition) before y's own rounding: 2^-24 more for fp32, 2^-8 for bf16."""

import numpy as np
import pytest
import torch
import torch.nn as nn

from byteprof_b200.quant.int8 import gemv_int8, int8_linear, int8_mm, quantize_rowwise_int8, quantize_tokens_int8
from byteprof_b200.quant.integrate import Int8Linear

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def ints(rows, k, seed, ld=None, lo=-127):
    g = torch.Generator(device="cuda").manual_seed(seed)
    full = torch.randint(lo, 128, (rows, ld or k), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    return full[:, :k]


def scales(n, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(n, generator=g, device="cuda") * 0.02 + 1e-3).to(dtype)


def check(y, q, s, w, ws, bias=None):
    acc = q.cpu().double() @ w.cpu().double().t()  # exact: below 2^53
    val = acc * s.cpu().double()[:, None] * ws.cpu().double()
    want, size = val, val.abs()
    if bias is not None:
        want, size = val + bias.cpu().double(), size + bias.cpu().double().abs()
    tol = 4 * 2.0**-24 * size + (2.0**-24 if y.dtype == torch.float32 else 2.0**-8) * (want.abs() + 4 * 2.0**-24 * size)
    err = (y.cpu().double() - want).abs()
    assert (err <= tol).all(), (err - tol).max().item()


SHAPES = [(1, 1, 1), (1, 8192, 2048), (3, 37, 100), (16, 2048, 2048), (17, 129, 64), (33, 1000, 272), (64, 64, 8192),
          (100, 300, 17), (127, 256, 48), (128, 128, 128), (129, 257, 144), (250, 2048, 512), (509, 2048, 1040),
          (1, 100352, 256), (2, 5, 131056), (700, 513, 2048), (1025, 640, 96), (2500, 4001, 272),
          (385, 13000, 1040), (4097, 4608, 16)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_product_against_integer_arithmetic(m, n, k, dtype):
    q, w = ints(m, k, 1, ld=-(-k // 16) * 16), ints(n, k, 2)
    s, ws = scales(m, 3), scales(n, 4, BF16)
    y = int8_mm(q, s, w, ws, out=torch.empty(m, n, dtype=dtype, device="cuda"))
    check(y, q, s, w, ws)


@pytest.mark.parametrize("m,n,k", [(5, 130, 256), (200, 300, 512), (40, 77, 50)])
def test_bias_fp32_scales_strides_and_surroundings(m, n, k):
    q, w = ints(m, k, 5, ld=k + 48 if k % 16 == 0 else k + 3, lo=-128), ints(n, k, 6, ld=k + 32, lo=-128)
    s, ws = scales(m, 7), scales(n, 8)
    bias = torch.randn(n, device="cuda").to(BF16)
    for dtype in (BF16, torch.float32):
        buf = torch.full((m + 2, n + 5), 7.0, dtype=dtype, device="cuda")
        y = int8_mm(q, s, w, ws, bias, out=buf[1:-1, 2:2 + n])
        check(y, q, s, w, ws, bias)
        assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[:, :2] == 7).all() and (buf[:, 2 + n:] == 7).all()


@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (40, 256, 1024), (300, 300, 256)])
def test_aligned_and_unaligned_operands_give_the_same_bits(m, n, k):
    q, w, s, ws = ints(m, k, 9), ints(n, k, 10), scales(m, 11), scales(n, 12, BF16)
    y = int8_mm(q, s, w, ws)
    big = torch.zeros(n, k + 1, dtype=torch.int8, device="cuda")
    big[:, 1:] = w
    assert torch.equal(y, int8_mm(q, s, big[:, 1:], ws))  # odd row stride and base: the CUDA cores


def test_extreme_sums_do_not_wrap():
    k = 131071  # 131071 * 128 * 128 < 2^31
    q = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((130, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
    w[1::2] = 127
    one = torch.ones(130, device="cuda")
    for m in (1, 2):
        y = int8_mm(q[:m], one[:m], w, one, out=torch.empty(m, 130, device="cuda"))
        assert (y[:, 0::2] == float(k * 16384)).all() and (y[:, 1::2] == float(-k * 128 * 127)).all()


def test_a_row_does_not_depend_on_the_others():
    w, ws = ints(700, 512, 13), scales(700, 14, BF16)
    q, s = ints(300, 512, 15), scales(300, 16)
    y = int8_mm(q, s, w, ws)
    for m in (1, 7, 33, 150):
        assert torch.equal(int8_mm(q[:m], s[:m], w, ws), y[:m])


# ---- the rows' quantizer --------------------------------------------------------------------------------
@pytest.mark.parametrize("m,k", [(1, 2048), (3, 64), (5, 1), (7, 50), (2, 20000), (300, 8192)])
def test_quantizer_equals_correctly_rounded_division(m, k):
    g = torch.Generator(device="cuda").manual_seed(m + k)
    x = (torch.randn(m, k + 8, generator=g, device="cuda") * 3).to(BF16)[:, :k]
    q, s = quantize_tokens_int8(x)
    xn = x.float().cpu().numpy()
    amax = np.abs(xn).max(1).astype(np.float32)
    sn = np.maximum(amax / np.float32(127), np.float32(1e-12))
    assert np.array_equal(s.cpu().numpy(), sn)
    assert np.array_equal(q.cpu().numpy(), np.rint(xn / sn[:, None]).astype(np.int8))


def test_quantizer_on_zeros_ties_tiny_and_non_finite_rows():
    x = torch.zeros(6, 64, device="cuda")
    x[1, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])       # scale 1: ties go to even
    x[2, 3] = float("inf")
    x[3, 5] = float("nan")
    x[4, 0] = 1e-30                                          # below the smallest scale
    x[5, :2] = torch.tensor([float.fromhex("0x1.fep127"), -1e30])
    q, s = quantize_tokens_int8(x.to(BF16))
    assert s[0].item() == np.float32(1e-12) and (q[0] == 0).all()
    assert q[1, :4].tolist() == [127, 0, 2, -2] and s[1].item() == 1.0
    assert torch.isnan(s[2:4]).all() and (q[2:4] == 0).all()
    assert (q[4] == 0).all() and s[4].item() == np.float32(1e-12)
    assert q[5, 0].item() == 127
    w, ws = ints(40, 64, 1), scales(40, 2)
    y = int8_mm(q, s, w, ws)
    assert torch.isnan(y[2:4]).all() and not torch.isnan(y[[0, 1, 4]]).any()


@pytest.mark.parametrize("m,n,k", [(1, 8192, 2048), (1, 40000, 512), (16, 700, 512), (5, 33, 8), (7, 130, 200), (2, 20000, 4096), (1, 300, 8192), (2, 513, 264),
                                   (8, 260, 1000)])
def test_few_rows_quantized_inside_equal_the_two_calls(m, n, k):
    """One or two rows quantize in the product's own launch: the same bits, NaN rows and zero rows among them."""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn(m, k + 8, generator=g, device="cuda").to(BF16)[:, :k]
    if m > 4:
        x[1] = 0
        x[2, k - 1] = float("nan")
        x[3, 0] = float("-inf")
    if m == 2:
        x[1, k - 1] = float("nan")
    w, ws = ints(n, k, 21, ld=-(-k // 16) * 16), scales(n, 22, BF16)
    bias = torch.randn(n, generator=g, device="cuda").to(BF16)
    for dtype in (BF16, torch.float32):
        a, b = (torch.empty(m, n, dtype=dtype, device="cuda") for _ in range(2))
        int8_linear(x, w, ws, bias, out=a)
        int8_mm(*quantize_tokens_int8(x), w, ws, bias, out=b)
        assert torch.equal(a.view(torch.int16 if dtype == BF16 else torch.int32), b.view(torch.int16 if dtype == BF16 else torch.int32))
        assert torch.isnan(a).any(1).tolist() == [(m > 4 and i in (2, 3)) or (m == 2 and i == 1) for i in range(m)]


@pytest.mark.parametrize("m", [1, 30, 200])
def test_linear_is_the_two_calls_and_near_the_bf16_product(m):
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, 1024, generator=g, device="cuda").to(BF16)
    w = (torch.randn(700, 1024, generator=g, device="cuda") * 0.02).to(BF16)
    wq, ws = quantize_rowwise_int8(w)
    y = int8_linear(x, wq, ws)
    assert torch.equal(y, int8_mm(*quantize_tokens_int8(x), wq, ws))
    # against the weight-only product: each activation is off by at most half a scale step
    ref = x.double() @ (wq.double() * ws.double()[:, None]).t()
    step = x.double().abs().amax(1, keepdim=True) / 254
    bound = step * (wq.double() * ws.double()[:, None]).abs().sum(1) + 2.0**-8 * ref.abs() + 1e-3
    assert ((y.double() - ref).abs() <= bound).all()
    if m == 1:
        assert ((gemv_int8(x, wq, ws).double() - y.double()).abs() <= 2 * bound).all()


def test_empty_products():
    q, s, w, ws = ints(4, 32, 1), scales(4, 2), ints(6, 32, 3), scales(6, 4)
    assert int8_mm(q[:0], s[:0], w, ws).shape == (0, 6)
    assert int8_mm(q, s, w[:0], ws[:0]).shape == (4, 0)
    assert (int8_mm(q[:, :0], s, w[:, :0], ws) == 0).all()
    b = torch.arange(6, device="cuda").to(BF16)
    assert torch.equal(int8_mm(q[:, :0], s, w[:, :0], ws, b), b.expand(4, 6))


def test_captured_and_replayed_with_new_inputs():
    g = torch.Generator(device="cuda").manual_seed(5)
    wq, ws = ints(384, 512, 6), scales(384, 7, BF16)
    x = torch.randn(100, 512, generator=g, device="cuda").to(BF16)
    int8_linear(x, wq, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int8_linear(x, wq, ws)
    for _ in range(3):
        x.copy_(torch.randn(100, 512, generator=g, device="cuda"))
        graph.replay()
        assert torch.equal(y, int8_linear(x, wq, ws))


@pytest.mark.parametrize("m,n,k", [(129, 2000, 64), (300, 4097, 48), (1000, 5003, 32), (70, 3001, 256), (128, 4000, 128), (700, 1281, 4096)])
@pytest.mark.parametrize("off", [0, 1, 2, 4])
def test_rows_of_the_result_that_start_anywhere(m, n, k, off):
    """Results in a buffer whose rows start at odd, 4-byte and 8-byte places, both types: the values, and nothing beside them."""
    q, w, s, ws = ints(m, k, 30), ints(n, k, 31), scales(m, 32), scales(n, 33)
    want = int8_mm(q, s, w, ws, out=torch.empty(m, (n + 7) // 8 * 8, device="cuda")[:, :n])
    for dtype in (BF16, torch.float32):
        buf = torch.full((m + 1, n + 2 * off + 3), 5.0, dtype=dtype, device="cuda")
        int8_mm(q, s, w, ws, out=buf[:m, off:off + n])
        assert torch.equal(buf[:m, off:off + n], want.to(dtype))
        assert (buf[:m, :off] == 5).all() and (buf[:m, off + n:] == 5).all() and (buf[m] == 5).all()


def test_a_result_of_more_than_32_bits():
    m, n, k = 40003, 65600, 32
    x, s, w, ws = ints(m, k, 8), scales(m, 9), ints(n, k, 10), scales(n, 11)
    y = int8_mm(x, s, w, ws)
    rows = torch.tensor([0, 1, 32767, 32768, m - 129, m - 1], device="cuda")
    assert torch.equal(y[rows], int8_mm(x[rows].contiguous(), s[rows].contiguous(), w, ws))
