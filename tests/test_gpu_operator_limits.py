"""GPU: the operators at the ends of their documented ranges."""
import pytest
import torch

from tests.util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("block", [32, 128])
@pytest.mark.parametrize("width", [1 << 26, 65535 * 1024, 65535 * 1024 + 128])
def test_widest_gated_rows(width, block):
    """A block of columns knows nothing of its row: the codes and exponents of one row of up to 2^26 columns are those of the
    same values as many rows."""
    from tcfp_b200.kernels import silu_mul_quantize

    piece = torch.randn(2, 1 << 20, generator=gen(1)).to(torch.bfloat16).to(DEV)
    gate = (piece[0] * torch.exp2(torch.arange(64, device=DEV).remainder(5).float())[:, None].to(torch.bfloat16)).reshape(-1)[:width]
    up = piece[1].repeat(64)[:width]
    gate, up = gate[None], up[None]
    q = silu_mul_quantize(gate, up, block_size=block, want_bf16=True)
    cut = width // 128
    rows = silu_mul_quantize(gate.view(cut, 128), up.view(cut, 128), block_size=block, want_bf16=True)
    assert q.codes.shape == (1, width) and torch.equal(q.codes.view(torch.uint8).view(cut, 128), rows.codes.view(torch.uint8))
    assert torch.equal(q.scales.view(cut, 128 // block), rows.scales.t())
    assert torch.equal(q.bf16.view(cut, 128), rows.bf16)


def test_gate_backward_in_32_bits():
    """FP32 gradients stay in 32 bits, so sigma is formed with the exponential of the library: 2 ulp = 4 u of itself (u = 2^-24),
    the addition and the reciprocal a u each, S = 6 u in all, also far from zero.  du = d g sigma: two products more.  dg = d sigma
    u f with f = 1 + g (1 - sigma): 1 - sigma is off by S sigma + u (1 - sigma), f by |g| times that and u, three products more."""
    from tcfp_b200.kernels import silu_mul_backward

    U = 2.0**-24
    S = 6 * U
    n = 1 << 20
    gate = (torch.rand(64, n // 64, generator=gen(2)) * 120 - 80).to(DEV)
    gate[0, :8] = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 40.0, -80.0, 87.0, -87.0])
    up, d = torch.randn(64, n // 64, generator=gen(3)).to(DEV), torch.randn(64, n // 64, generator=gen(4)).to(DEV)
    dg, du = silu_mul_backward(d, gate, up)
    g, u, dd = gate.double(), up.double(), d.double()
    sig = 1 / (1 + torch.exp(-g))
    rest = 1 / (1 + torch.exp(g))
    f = 1 + g * rest
    tiny = 2.0**-120             # products that leave the normal numbers
    assert ((du.double() - dd * g * sig).abs() <= (S + 2 * U) * 1.0001 * (dd * g * sig).abs() + tiny).all()
    room = (dd * u).abs() * sig * ((S + 4 * U) * f.abs() + g.abs() * (S * sig + U * rest)) * 1.0001
    assert ((dg.double() - dd * u * sig * f).abs() <= room + tiny).all()
    # far out sigma is 0 or 1, and a NaN stays one
    far = torch.tensor([[-1000.0, 1000.0, float("nan"), 2.0]], device=DEV)
    dg, du = silu_mul_backward(torch.ones_like(far), far, torch.ones_like(far))
    assert dg[0, :2].tolist() == [0.0, 1.0] and du[0, :2].tolist() == [0.0, 1000.0]
    assert dg[0].isnan().tolist() == du[0].isnan().tolist() == [False, False, True, False]
