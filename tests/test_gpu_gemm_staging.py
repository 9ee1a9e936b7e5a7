"""GPU: the FP8 and bf16 products on CTA pairs at sizes that end inside a tile.

The epilogue stages its output in two pieces taken in turn, and a piece behind the last row or column is not stored.  Every kind
of the kernel runs with several tiles a pair, with rows that end in the lower and in the upper half of a tile's 256 and columns
that end after each number of pieces.  The operands are small integers (and powers of two as scales), so every sum is exact in
FP32 and the outputs are compared to the bit; bf16 outputs are those sums rounded once.
"""
import pytest
import torch

from tests.util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
DTYPES = [torch.float32, torch.bfloat16]
ROWS = [2048, 2064, 2128, 2160, 2272]
COLS = [2048 + r for r in (0, 32, 64, 96, 128, 160, 192, 224)]


def ints(seed, rows, cols, dtype):
    return torch.randint(-3, 4, (rows, cols), generator=gen(seed)).float().to(dtype).to(DEV)


def planes(seed, blocks, rows):
    return torch.randint(-2, 3, (blocks, rows), generator=gen(seed), dtype=torch.int8).to(DEV)


def values(codes, exps, bs):
    return codes.double() * torch.exp2(exps.t().double()).repeat_interleave(bs, dim=1)


def same(out, want, times):
    for _ in range(times):
        assert torch.equal(out(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n", COLS)
def test_per_tensor(m, n, dtype):
    from tcfp_b200.kernels import fused_dual_gemm_backward_dx, fused_dual_gemm_forward

    k = 384
    one, half = torch.ones(1, device=DEV), torch.full((1,), 0.5, device=DEV)
    a, hi, lo = ints(1, m, k, E4), ints(2, n, k, E4), ints(3, n, k, E4)
    first, second = a.double() @ hi.double().t(), a.double() @ lo.double().t()
    same(lambda: fused_dual_gemm_forward(a, hi, lo, one, one, half, out_dtype=dtype), (first + 0.5 * second).to(dtype), 3)
    same(lambda: fused_dual_gemm_forward(a, hi, None, one, one, None, out_dtype=dtype), first.to(dtype), 3)
    g, hi_t, lo_t = ints(4, m, k, E5), ints(5, k, n, E4), ints(6, k, n, E4)
    first, second = g.double() @ hi_t.double(), g.double() @ lo_t.double()
    same(lambda: fused_dual_gemm_backward_dx(g, hi_t, lo_t, one, one, half, out_dtype=dtype), (first + 0.5 * second).to(dtype), 3)
    same(lambda: fused_dual_gemm_backward_dx(g, hi_t, None, one, one, None, out_dtype=dtype), first.to(dtype), 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n", COLS)
def test_block_scaled(m, n, dtype):
    from tcfp_b200.kernels import fused_block_scaled_backward_dx, fused_block_scaled_dual_gemm_forward

    k, bs = 384, 32
    a, hi, lo = ints(11, m, k, E4), ints(12, n, k, E4), ints(13, n, k, E4)
    ea, eh, el = planes(14, k // bs, m), planes(15, k // bs, n), planes(16, k // bs, n)
    x = values(a, ea, bs)
    first, second = x @ values(hi, eh, bs).t(), x @ values(lo, el, bs).t()
    same(lambda: fused_block_scaled_dual_gemm_forward(a, hi, lo, ea, eh, el, bs, out_dtype=dtype), (first + second).to(dtype), 3)
    same(lambda: fused_block_scaled_dual_gemm_forward(a, hi, None, ea, eh, None, bs, out_dtype=dtype), first.to(dtype), 3)
    # dX: exponents of 0, so that the weight re-targeted for the other contraction keeps its integers
    g, eg = ints(17, m, k, E5), planes(18, k // bs, m)
    hi_t, lo_t = ints(19, k, n, E4), ints(20, k, n, E4)
    zero = torch.zeros(n // bs, k, dtype=torch.int8, device=DEV)
    want = (values(g, eg, bs) @ (hi_t.double() + lo_t.double())).to(dtype)
    for exact in (False, True):
        same(lambda: fused_block_scaled_backward_dx(g, hi_t, lo_t, eg, zero, zero, bs, out_dtype=dtype, exact_bf16=exact), want, 3)


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n", COLS)
def test_weight_gradients(m, n):
    from tcfp_b200.kernels import bf16_weight_grad, fp8_weight_grad

    tokens = 320
    one = torch.ones(1, device=DEV)
    g, x = ints(21, tokens, m, E5), ints(22, tokens, n, E4)
    want = g.double().t() @ x.double()
    for dtype in DTYPES:
        same(lambda: fp8_weight_grad(g, x, one, one, out_dtype=dtype), want.to(dtype), 3)
    x16 = x.to(torch.bfloat16)
    same(lambda: bf16_weight_grad(g.to(torch.bfloat16), x16), want.float(), 3)
    # 257 needs nine bits: a head of 256 and a tail
    same(lambda: bf16_weight_grad(257.0 * g.float(), x16), (257.0 * want).float(), 3)
