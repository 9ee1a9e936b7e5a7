"""GPU: the operators that end in 8 bits in front of a linear layer (norm with
the residual's addition, gated activation, row quantizer), their backward
passes and the int8 product, against their definitions in 64 bits.

Tolerances.  u = 2^-24 is half a step of FP32 relative to the value, bf16 and
E4M3 round by at most 2^-8 and 2^-4 of the value (E4M3 below 2^-6: by 2^-10).

* norm: a thread adds at most 32 squares, at most 10 tree steps follow, and
  the division, the addition of eps and rsqrtf (2 ulp = 4u) join: rstd is off by
  at most (32 + 10 + 2 + 4) u / 2 + 4u < 32 u, y by two more roundings: Y = 40 u.
* gate: the product -g log2 e is off by 2 u of itself, 2 |g| u of the power of
  two; that instruction adds 2^-22, the addition u, the reciprocal 2 u, two
  products 2 u; with |g| <= 40 y = g * sigma * u is off by at most 89 u of itself:
  G = 128 u.  Where 1 + e^-g passes 2^126 the reciprocal is 0, for a value below
  |u| * 88 * 2^-126.
* a code of step s is off by s / 2 and by what y is off.
"""
import pytest
import torch

from tests.util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24
Y = 40 * U
G = 128 * U
EPS = 1e-5
DTYPES = [torch.bfloat16, torch.float32]


def stream(seed, rows, width, dtype):
    g = gen(seed)
    x = torch.randn(rows, width, generator=g) * (0.5 + torch.rand(width, generator=g))
    x[:, ::97] *= 20.0
    x[rows // 2] = 0.0                       # a padded token
    return x.to(dtype).to(DEV)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check_row_codes(q, y, rel):
    """int8 codes with a scale for each row against y in 64 bits, y known to ``rel`` of itself."""
    s = q.scales.double()
    want = y.abs().amax(1).clamp(min=1e-12) / 127
    assert ((s - want).abs() <= (rel + 2 * U) * want).all()
    code = q.codes.double()
    assert code.abs().max() <= 127
    off = (code * s[:, None] - y).abs()
    # half a step, the roundings of the reciprocal and of the product, and y's own error
    assert (off <= s[:, None] * (0.5 + 127 * 2.001 * U) + rel * y.abs()).all()
    if q.bf16 is not None:
        v = code * s[:, None]
        assert ((q.bf16.double() - v).abs() <= (2.0**-8 + 2 * U) * v.abs()).all()


def check_block_codes(q, y, rel):
    rows, width = y.shape
    bs = q.block_size
    blocks = y.reshape(rows, -1, bs)
    am = blocks.abs().amax(2).clamp(min=1e-12)
    e = q.scales.t().double()
    # the exponent is that of an amax within its error; 2 u more for the quotient by 448
    lo, hi = (torch.ceil(torch.log2(am * f / 448)).clamp(min=-126) for f in (1 - rel - 4 * U, 1 + rel + 4 * U))
    assert ((e >= lo) & (e <= hi)).all()
    v = q.codes.float().double().reshape(blocks.shape) * torch.exp2(e)[:, :, None]
    assert ((v - blocks).abs() <= (2.0**-4 + rel) * blocks.abs() + torch.exp2(e)[:, :, None] * 2.0**-10).all()
    if q.bf16 is not None:
        assert torch.equal(q.bf16.double(), v.reshape(y.shape))        # four significant bits: exact in bf16
    # the packed scale factors are those of the exponent planes, filled up with 2^0 along K
    sf = q.scales._tcfp_sf[0].cpu()
    kb = width // bs
    kg = (kb + 3) // 4
    want = torch.full((rows, kg * 4), 127, dtype=torch.int64)
    want[:, :kb] = (q.scales.t().cpu().long() + 127).clamp(min=0)
    r, k = torch.meshgrid(torch.arange(rows), torch.arange(kg * 4), indexing="ij")
    at = ((r // 128) * kg + k // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + k % 4
    assert torch.equal(sf[at].long(), want)


def check_codes(q, y, rel):
    (check_row_codes if q.block_size is None else check_block_codes)(q, y, rel)


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------

ROW_SHAPES = [(1, 4096), (3, 1), (5, 7), (2, 333), (33, 1000), (17, 2731), (130, 64), (9, 5120), (3, 11008), (2, 32768), (1, 32761)]
# many rows, not a multiple of what a block takes: 2 and 4 chunks a thread, one warp a row and more
ROW_SHAPES += [(2371, 264), (2371, 512), (2371, 520), (2370, 1024), (2371, 1032), (2371, 2048), (2371, 4096), (2371, 8192), (1201, 8200), (1203, 12296)]
BLOCK_SHAPES = [(1, 128), (33, 384), (130, 4096), (257, 640), (3, 11008), (2, 32768), (1201, 8320), (907, 32768)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("add", [True, False])
@pytest.mark.parametrize("shape,bs", [(s, None) for s in ROW_SHAPES] + [(s, b) for s in BLOCK_SHAPES for b in (32, 64, 128)])
def test_norm_forward(shape, bs, add, dtype):
    from tcfp_b200.kernels import add_rms_norm_quantize

    rows, width = shape
    x = stream(1, rows, width, dtype)
    r = stream(2, rows, width, dtype) if add else None
    w = (1 + 0.1 * torch.randn(width, generator=gen(3))).to(DEV)
    q, h, rstd = add_rms_norm_quantize(x, w, r, EPS, block_size=bs, want_bf16=True)
    want_h = x if r is None else x + r
    assert torch.equal(h, want_h) and h.dtype == dtype
    hd = want_h.double()
    want_r = (hd.square().mean(1) + EPS).rsqrt()
    assert ((rstd.double() - want_r).abs() <= 32 * U * want_r).all()
    check_codes(q, hd * want_r[:, None] * w.double(), Y)
    assert torch.equal(q.dequantize(), q.bf16) and q.shape == x.shape and q.dtype == dtype


def norm_loss(x, r, w, gy, gh):
    h = x if r is None else x + r
    y = h * (h.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
    return (y * gy).sum() + ((h * gh).sum() if gh is not None else 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (2, 7), (33, 1000), (700, 96), (1300, 512), (9, 9000), (3, 17001), (4, 20480), (2, 32768)])
@pytest.mark.parametrize("with_h", [True, False])
def test_norm_backward(shape, with_h, dtype):
    from tcfp_b200.kernels import add_rms_norm_backward

    rows, width = shape
    h = stream(4, rows, width, dtype)
    w = (1 + 0.1 * torch.randn(width, generator=gen(5))).to(DEV)
    gy = torch.randn(rows, width, generator=gen(6)).to(dtype).to(DEV)
    gh = torch.randn(rows, width, generator=gen(7)).to(dtype).to(DEV) if with_h else None
    hd, wd, gyd = h.double(), w.double(), gy.double()
    ghd = None if gh is None else gh.double()
    rstd = (hd.square().mean(1) + EPS).rsqrt()
    dx, dw = add_rms_norm_backward(gy, h, rstd.float(), w, gh)
    hat = hd * rstd[:, None]
    g = gyd * wd
    want = rstd[:, None] * (g - hat * (g * hat).mean(1, keepdim=True)) + (0 if ghd is None else ghd)
    # terms of the sum, each off by a few u; the mean by (32 + 10 + 4) u of the sum of magnitudes, rstd in by u
    size = rstd[:, None] * (g.abs() + hat.abs() * (g * hat).abs().mean(1, keepdim=True)) + (0 if ghd is None else ghd.abs())
    assert dx.dtype == dtype and dw.dtype == torch.float32
    assert ((dx.double() - want).abs() <= 64 * U * size + half_step(dtype) * want.abs()).all()
    # a block adds the rows it owns in order, then at most 148 * 4 partial sums are joined: fewer additions than rows + 16
    assert ((dw.double() - (gyd * hat).sum(0)).abs() <= (min(rows, 1000) + 16) * U * (gyd * hat).abs().sum(0)).all()
    again = add_rms_norm_backward(gy, h, rstd.float(), w, gh)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    # differences of the definition in 64 bits, along one direction in x and one in w; the step's own error is of its square
    gen_d = gen(8)
    dirx = torch.randn(rows, width, generator=gen_d).double().to(DEV)
    dirw = torch.randn(width, generator=gen_d).double().to(DEV)
    step = 1e-6
    for dirv, args in ((dirx, lambda t: (hd + t * dirx, None, wd, gyd, ghd)), (dirw, lambda t: (hd, None, wd + t * dirw, gyd, ghd))):
        slope = (norm_loss(*args(step)) - norm_loss(*args(-step))) / (2 * step)
        got = (dx.double() * dirv).sum() if dirv is dirx else (dw.double() * dirv).sum()
        room = ((64 * U * size + half_step(dtype) * want.abs()) * dirx.abs()).sum() if dirv is dirx else \
            ((min(rows, 1000) + 16) * U * (gyd * hat).abs().sum(0) * dirw.abs()).sum()
        # the step: 64-bit cancellation 2^-52 |loss| / step, and the third derivative (of the order of rstd^3) times step^2
        scale = (gyd * hat * wd).abs().sum() + (0 if ghd is None else (ghd * hd).abs().sum())
        third = step**2 * (size * dirv.abs()).sum() * (rstd.max() * dirv.abs().max() * 8) ** 2
        assert (slope - got).abs() <= room + 1e-9 * scale + third


# ---------------------------------------------------------------------------
# gated activation
# ---------------------------------------------------------------------------

def gate_up(seed, rows, width, dtype):
    x = 2 * torch.randn(rows, 2 * width, generator=gen(seed))
    x[rows // 2] = 0.0
    if width > 8:
        x[0, :8] = torch.tensor([40.0, -40.0, 0.0, -0.0, 1e-30, 30.0, -30.0, 12.0])
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("shape,bs", [(s, None) for s in ROW_SHAPES + [(2, 40000), (1, 50001)]]
                         + [(s, b) for s in BLOCK_SHAPES for b in (32, 64, 128)])
def test_gate_forward(shape, bs, packed, dtype):
    from tcfp_b200.kernels import silu_mul_quantize

    rows, width = shape
    x = gate_up(9, rows, width, dtype)
    if packed:
        q = silu_mul_quantize(x, block_size=bs, want_bf16=True)
    else:
        q = silu_mul_quantize(x[:, :width], x[:, width:], block_size=bs, want_bf16=True)
    g, u = x[:, :width].double(), x[:, width:].double()
    assert q.shape == (rows, width)
    check_codes(q, g * torch.sigmoid(g) * u, G)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (2, 7), (33, 1000), (17, 2731), (3, 11008), (2, 40000)])
def test_gate_backward(shape, packed, dtype):
    from tcfp_b200.kernels import silu_mul_backward

    rows, width = shape
    x = gate_up(10, rows, width, dtype)
    dy = torch.randn(rows, width, generator=gen(11)).to(dtype).to(DEV)
    g, u, d = x[:, :width].double(), x[:, width:].double(), dy.double()
    if packed:
        both = silu_mul_backward(dy, x)
        assert both.shape == x.shape
        dg, du = both[:, :width], both[:, width:]
    else:
        dg, du = silu_mul_backward(dy, x[:, :width], x[:, width:])
    assert dg.dtype == dtype and du.dtype == dtype
    sig = torch.sigmoid(g)
    want_u = d * g * sig
    want_g = d * u * sig * (1 + g * (1 - sig))
    assert ((du.double() - want_u).abs() <= G * want_u.abs() + half_step(dtype) * want_u.abs()).all()
    # 1 - sigma cancels for large g: off by u of 1, times g; d(1 - sigma) is bounded by G sigma
    size = (d * u).abs() * sig * (1 + g.abs() * (1 - sig) + g.abs() * sig)
    assert ((dg.double() - want_g).abs() <= 2 * G * size + half_step(dtype) * want_g.abs()).all()
    if dtype == torch.float32:
        step = 1e-6
        f = lambda gg, uu: gg * torch.sigmoid(gg) * uu * d  # noqa: E731
        num_g = (f(g + step, u) - f(g - step, u)) / (2 * step)
        # 64-bit cancellation over the step, and the third derivative of silu (at most 1) times the square of the step
        room = 2 * G * size + half_step(dtype) * want_g.abs() + 1e-9 * (f(g, u).abs() + (d * u).abs())
        assert ((dg.double() - num_g).abs() <= room).all()


def test_gate_limits():
    """Far from zero silu is 0 or g; a NaN or an infinity stays in its row (int8) or its place (E4M3)."""
    from tcfp_b200.kernels import silu_mul_quantize

    g = torch.tensor([[-200.0, 200.0, -89.0, 88.0, 0.0, 0.0, 0.0, 1.0]], device=DEV).repeat(1, 4)
    q = silu_mul_quantize(g, torch.ones_like(g), block_size=32, want_bf16=True)
    gd = g.double()
    check_block_codes(q, torch.where(gd < -87, 0.0, gd * torch.sigmoid(gd)), G)
    x = torch.ones(4, 64, device=DEV)
    x[1, 5] = float("nan")
    x[2, 6] = float("inf")
    x[3, 7] = float("-inf")
    q = silu_mul_quantize(x, torch.ones_like(x))
    assert q.scales.isfinite().tolist() == [True, False, False, False]
    q = silu_mul_quantize(x, torch.ones_like(x), block_size=32, want_bf16=True)
    assert q.bf16.isnan().nonzero().tolist() == [[1, 5], [3, 7]]          # -inf * sigma(-inf) is not a number
    assert torch.equal(q.bf16[0], q.bf16[1, 32:].repeat(2))


def test_norm_limits():
    """Zero rows give zero codes; a row that holds a NaN or an infinity is not finite, its neighbours are untouched."""
    from tcfp_b200.kernels import add_rms_norm_quantize

    w = torch.ones(64, device=DEV)
    x = torch.ones(4, 64, device=DEV)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 6] = float("inf")
    q, _, rstd = add_rms_norm_quantize(x, w)
    assert torch.equal(q.codes[0], torch.zeros(64, dtype=torch.int8, device=DEV)) and q.scales[0] == torch.tensor(1e-12) / 127
    assert q.scales.isfinite().tolist() == [True, False, False, True] and (q.codes[3] == 127).all()
    q, _, _ = add_rms_norm_quantize(x, w, block_size=32, want_bf16=True)
    assert (q.bf16[0] == 0).all() and q.bf16[1].isnan().all() and q.bf16[2, 6].isnan() and q.bf16[3].isfinite().all()


# ---------------------------------------------------------------------------
# row quantizer and int8 product
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROW_SHAPES + [(2, 40000), (1, 50001), (5000, 128)])
def test_int8_quantize_rows(shape, dtype):
    """The codes are defined to the bit: the product with the reciprocal in FP32, rounded half to even."""
    from tcfp_b200.kernels import int8_quantize_rows

    x = stream(12, *shape, dtype)
    x[0, 0] = 127.0
    if shape[1] > 8:                            # exact ties, either side of them
        x[0] = x[0].clamp(-100, 100)
        x[0, :8] = torch.tensor([127.0, 0.5, 1.5, -0.5, 2.5, 63.5, -64.5, 126.5]).to(dtype)
    q = int8_quantize_rows(x, want_bf16=True)
    # a quotient of FP32 numbers formed in 64 bits and rounded is the FP32 quotient (53 >= 2 * 24 + 2); torch divides by a
    # number by multiplying with its reciprocal, which is not
    f = x.double()
    s = (f.abs().amax(1).float().clamp(min=1e-12).double() / 127).float()
    assert torch.equal(q.scales, s)
    # the product of two FP32 numbers is exact in 64 bits
    assert torch.equal(q.codes.float(), torch.round((f * (1 / s.double()).float().double()[:, None]).float()))
    check_row_codes(q, x.double(), 0.0)
    assert q.codes.stride(0) % 16 == 0


def codes(seed, rows, k, lo=-127):
    return torch.randint(lo, 128, (rows, k), generator=gen(seed), dtype=torch.int8).to(DEV)


def check_product(a, b, sa, sb, bias, dtype):
    from tcfp_b200.kernels import int8_matmul

    out = int8_matmul(a, b, sa, sb, bias=bias, out_dtype=dtype)
    prod = (a.double() @ b.double().t()) * (sa.double()[:, None] * sb.double())     # below 2^53: exact
    want = prod if bias is None else prod + bias.double()
    # conversion of the sum, two factors, the addition: four roundings; then the output's
    room = 4 * U * (prod.abs() + want.abs()) + (half_step(dtype) * want.abs() if dtype == torch.bfloat16 else 0)
    assert out.shape == want.shape and out.dtype == dtype
    assert ((out.double() - want).abs() <= room).all()
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 128, 16), (1, 4096, 4096), (2, 100, 15), (3, 1001, 2031), (7, 22016, 512), (16, 256, 129), (17, 640, 384),
    (31, 130, 11008), (32, 4096, 1024), (33, 129, 127), (64, 1024, 4096), (65, 300, 640), (100, 7, 333), (128, 2048, 256),
    (129, 1000, 1000), (200, 4096, 640), (256, 256, 256), (257, 513, 1030), (300, 11008, 128), (512, 1536, 2048),
    (777, 333, 4097), (1024, 4096, 512), (2049, 1025, 96), (4096, 384, 4096), (3000, 8192, 160)])
def test_int8_product(m, n, k, dtype):
    g = gen(m + n + k)
    sa, sb = (torch.rand(m, generator=g) + 0.01).to(DEV), (torch.rand(n, generator=g) * 1e-3 + 1e-5).to(DEV)
    a, b = codes(1 + m, m, k), codes(2 + n, n, k)
    check_product(a, b, sa, sb, None, dtype)
    check_product(a, b, sa, sb, torch.randn(n, generator=g).to(DEV), dtype)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_int8_product_extreme_sums(m):
    """The largest sum there is, 131071 products of -128 * -128, is below 2^31 and comes out exact."""
    k = 131071
    a = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    b = torch.full((130, k), -128, dtype=torch.int8, device=DEV)
    b[1] = 127
    one = torch.ones(m, device=DEV)
    out = check_product(a, b, one, torch.ones(130, device=DEV), None, torch.float32)
    assert (out[:, 0].double() == float(torch.tensor(16384.0 * k, dtype=torch.float32))).all()


@pytest.mark.parametrize("m", [1, 50, 700])
def test_int8_product_views(m):
    """Operands that start anywhere and have any row pitch; scales of zero and infinity."""
    big_a, big_b = codes(20, m + 1, 1111), codes(21, 301, 999)
    sa, sb = torch.rand(m, generator=gen(22)).to(DEV), torch.rand(300, generator=gen(23)).to(DEV)
    check_product(big_a[1:, 3:900], big_b[1:, 5:902], sa, sb, None, torch.float32)
    check_product(big_a[1:, :897], codes(24, 897, 300).t(), sa, sb, None, torch.bfloat16)
    from tcfp_b200.kernels import int8_matmul

    sa[0], sb[1] = 0.0, float("inf")
    a, b = big_a[1:, :500], big_b[1:, :500]
    out = int8_matmul(a, b, sa, sb)
    assert (out[0, 2:] == 0).all() and not out[:, 1].isfinite().any() and out[:, 2:].isfinite().all()


def test_strides_and_leading_dimensions():
    """Views with a row pitch, an odd start or more dimensions give what their dense copies give: the same bytes, except
    where a norm's row starts off a 16-byte boundary.  Its narrow loads give the threads other columns, so the sum of
    squares has another order: both are within Y of the definition."""
    from tcfp_b200.kernels import add_rms_norm_backward, add_rms_norm_quantize, int8_quantize_rows, silu_mul_quantize

    big, wide = stream(13, 40, 1100, torch.bfloat16), stream(17, 40, 1104, torch.bfloat16)
    w = torch.ones(512, device=DEV)
    for view in (big[:, :512], big[:, 3:515], big[::3, 8:520], big.t()[:512, :].t(), big[:, :512].reshape(2, 20, 512),
                 big[:1, :512].expand(6, 512), big[:, :512][:0], wide[:, 512:1024], wide[1::2, 8:520]):
        dense = view.contiguous().clone()
        for bs in (None, 64):
            a, b = add_rms_norm_quantize(view, w, view, block_size=bs), add_rms_norm_quantize(dense, w, dense, block_size=bs)
            assert torch.equal(a[1], b[1]) and a[1].shape == view.shape
            if bs is not None or (view.data_ptr() % 16 == 0 and view.stride(-2) % 8 == 0):
                assert torch.equal(a[0].codes.view(torch.uint8), b[0].codes.view(torch.uint8))
                assert torch.equal(a[0].scales, b[0].scales) and torch.equal(a[2], b[2])
            else:
                assert ((a[0].scales - b[0].scales).abs() <= 2 * Y * b[0].scales).all()
                assert ((a[0].codes.int() - b[0].codes.int()).abs() <= 1).all()
            ga, gb = silu_mul_quantize(view, view, block_size=bs), silu_mul_quantize(dense, dense, block_size=bs)
            assert torch.equal(ga.codes.view(torch.uint8), gb.codes.view(torch.uint8)) and ga.shape == view.shape
        assert torch.equal(int8_quantize_rows(view).codes, int8_quantize_rows(dense).codes)
        if view.numel():
            rstd = a[2]
            ra = add_rms_norm_backward(view, view, rstd, w, view)
            rb = add_rms_norm_backward(dense, dense, rstd, w, dense)
            # an unaligned view goes through the narrow loads, whose threads own other columns: another order of the same sums
            assert (ra[0].float() - rb[0].float()).abs().max() <= 2.0**-7 * rb[0].float().abs().max() and ra[0].shape == view.shape
            assert (ra[1] - rb[1]).abs().max() <= 1e-5 * rb[1].abs().max()


def test_codes_padding_is_left_alone():
    """What lies behind a row's codes up to its pitch is not written."""
    import ctypes

    from tcfp_b200 import _C

    x = stream(14, 5, 37, torch.float32)
    held = torch.full((5, 48), 77, dtype=torch.int8, device=DEV)
    s = torch.empty(5, device=DEV)
    _C.check(_C.load().tcfp_int8_quantize_rows(x.data_ptr(), 37, _C.F32, held.data_ptr(), 48, s.data_ptr(), None, 5, 37,
                                               ctypes.c_void_p(_C.stream())))
    assert (held[:, 37:] == 77).all()


def test_empty_inputs():
    from tcfp_b200 import kernels as K

    x = torch.empty(0, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    for bs in (None, 32):
        q, h, rstd = K.add_rms_norm_quantize(x, w, x, block_size=bs, want_bf16=True)
        assert q.codes.shape == (0, 64) and h.shape == (0, 64) and rstd.shape == (0,) and q.dequantize().shape == (0, 64)
        assert K.silu_mul_quantize(x, block_size=bs).shape == (0, 32)
    dx, dw = K.add_rms_norm_backward(x, x, torch.empty(0, device=DEV), w)
    assert dx.shape == (0, 64) and (dw == 0).all()
    assert K.silu_mul_backward(torch.empty(0, 32, device=DEV), x).shape == (0, 64)
    q = K.int8_quantize_rows(x)
    assert K.int8_matmul(q.codes, codes(1, 8, 64), q.scales, torch.ones(8, device=DEV)).shape == (0, 8)


def test_another_stream_and_a_captured_graph():
    """The whole chain on a side stream, and captured and replayed with new inputs, gives the eager bytes."""
    from tcfp_b200 import kernels as K

    w = torch.ones(256, device=DEV)
    w1, w2 = K.int8_quantize_rows(stream(15, 1024, 256, torch.float32)), K.int8_quantize_rows(stream(16, 256, 512, torch.float32))

    def chain(x, r):
        q, h, rstd = K.add_rms_norm_quantize(x, w, r)
        gu = K.int8_matmul(q.codes, w1.codes, q.scales, w1.scales, out_dtype=torch.bfloat16)
        q2 = K.silu_mul_quantize(gu)
        y = K.int8_matmul(q2.codes, w2.codes, q2.scales, w2.scales, out_dtype=torch.bfloat16)
        dx, dw = K.add_rms_norm_backward(y, h, rstd, w, h)
        return y, h, dx, dw, K.silu_mul_backward(q2.dequantize(), gu)

    for rows in (3, 400):
        ins = [(stream(30 + i, rows, 256, torch.bfloat16), stream(40 + i, rows, 256, torch.bfloat16)) for i in range(3)]
        eager = [chain(*i) for i in ins]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = chain(*ins[0])
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(other, eager[0]))
        x, r = (t.clone() for t in ins[0])
        graphs = []
        for _ in range(2):                                     # two graphs captured one after the other share nothing
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = chain(x, r)
            graphs.append((g, out))
        for i, want in zip(ins, eager):
            x.copy_(i[0])
            r.copy_(i[1])
            for g, _ in graphs:
                g.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    """Calls that overlap on two streams share nothing."""
    from tcfp_b200 import kernels as K

    w = torch.ones(2048, device=DEV)
    xs = [stream(50 + i, 1500, 2048, torch.bfloat16) for i in range(2)]
    b = K.int8_quantize_rows(stream(52, 640, 2048, torch.float32))

    def work(x):
        q, h, rstd = K.add_rms_norm_quantize(x, w, x)
        y = K.int8_matmul(q.codes, b.codes, q.scales, b.scales)
        few = K.int8_matmul(q.codes[:9], b.codes, q.scales[:9], b.scales)
        return (y, few, *K.add_rms_norm_backward(x, h, rstd, w))

    want = [work(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(work(x))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


def test_offsets_past_32_bits():
    """The last rows of tensors of more than 2^31 elements are those of the same rows alone."""
    from tcfp_b200 import kernels as K

    rows, width = 140_000, 16_384
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=DEV)
    tail = stream(60, 9, width, torch.bfloat16)
    x[-9:] = tail
    w = torch.ones(width, device=DEV)
    for bs in (None, 64):
        q, _, rstd = K.add_rms_norm_quantize(x, w, block_size=bs)
        q9, _, rstd9 = K.add_rms_norm_quantize(tail, w, block_size=bs)
        assert torch.equal(q.codes[-9:].view(torch.uint8), q9.codes.view(torch.uint8)) and torch.equal(rstd[-9:], rstd9)
        assert torch.equal(q.scales[-9:] if bs is None else q.scales[:, -9:], q9.scales)
        assert (q.codes[0].view(torch.uint8) == 0).all()
        del q
        g, g9 = K.silu_mul_quantize(x, block_size=bs), K.silu_mul_quantize(tail, block_size=bs)
        assert torch.equal(g.codes[-9:].view(torch.uint8), g9.codes.view(torch.uint8))
        del g
    dx, dw = K.add_rms_norm_backward(x, x, rstd, w)
    dx9, dw9 = K.add_rms_norm_backward(tail, tail, rstd9, w)
    assert torch.equal(dx[-9:], dx9) and (dw - dw9).abs().max() <= 1e-5 * dw9.abs().max()      # other rows add zeros in another order
    del dx
    d = K.silu_mul_backward(x[:, :width // 2], x)
    assert torch.equal(d[-9:], K.silu_mul_backward(tail[:, :width // 2], tail))
    del d, x
    m, n = 70_000, 32_768
    a, b = codes(61, m, 64), codes(62, n, 64)
    sa, sb = torch.rand(m, generator=gen(63)).to(DEV), torch.rand(n, generator=gen(64)).to(DEV)
    out = K.int8_matmul(a, b, sa, sb, out_dtype=torch.bfloat16)
    assert torch.equal(out[-300:], K.int8_matmul(a[-300:], b, sa[-300:], sb, out_dtype=torch.bfloat16))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [40, 264, 1000, 1001, 2048, 4096, 8192, 9000])
def test_norm_backward_keeps_inside_its_workspace(width, dtype):
    """Not a byte behind tcfp_rms_norm_backward_workspace_bytes() is written, whichever shape the call takes."""
    from tcfp_b200 import _C

    lib = _C.load()
    for rows in (1, 300, 5000):
        x = stream(70, rows, width, dtype)
        w, rstd = torch.ones(width, device=DEV), torch.ones(rows, device=DEV)
        n = lib.tcfp_rms_norm_backward_workspace_bytes(rows, width)
        guard = 4 * width * 600                       # a margin larger than any other shape's workspace
        ws = torch.full((n + guard,), 113, dtype=torch.uint8, device=DEV)
        dx, dw = torch.empty_like(x), torch.empty(width, device=DEV)
        _C.check(lib.tcfp_rms_norm_backward(x.data_ptr(), width, x.data_ptr(), width, rstd.data_ptr(), _C.dtype_code(x),
                                            w.data_ptr(), _C.F32, None, 0, dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), rows,
                                            width, _C.stream()))
        assert (ws[n:] == 113).all()


def test_capture_after_copies_memsets_and_joins():
    """The operators start early only behind another kernel: captured behind a copy, a memset, another library kernel and the
    join of two streams they replay the eager bytes."""
    from tcfp_b200 import kernels as K

    rows, d = 200, 512
    w = torch.ones(d, device=DEV)
    wq = K.int8_quantize_rows(stream(80, 384, d, torch.float32))
    src = [stream(81 + i, rows, d, torch.bfloat16) for i in range(3)]
    x, r = torch.empty_like(src[0]), torch.empty_like(src[0])
    side = torch.cuda.Stream()

    def step(first, second):
        x.copy_(first)                                        # copy -> row kernel
        q0 = K.int8_quantize_rows(x)
        r.zero_()                                             # memset -> row kernel
        q1, h, rstd = K.add_rms_norm_quantize(x, w, r)
        x.add_(second)                                        # library kernel -> product, whose other input came from a row kernel
        y = K.int8_matmul(q1.codes, wq.codes, q1.scales, wq.scales)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            z = K.int8_matmul(q0.codes, wq.codes, q0.scales, wq.scales)
        few = K.int8_matmul(q1.codes[:3], wq.codes, q1.scales[:3], wq.scales)
        torch.cuda.current_stream().wait_stream(side)         # join -> row kernel
        return y, z, few, *K.add_rms_norm_backward(x, h, rstd, w, x), K.silu_mul_quantize(x).codes

    eager = [[t.clone() for t in step(src[i], src[i + 1])] for i in range(2)]
    first, second = src[0].clone(), src[1].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(first, second)
    for i in (0, 1, 0):
        first.copy_(src[i])
        second.copy_(src[i + 1])
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, eager[i]):
            assert torch.equal(a, b)
