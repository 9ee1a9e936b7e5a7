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
