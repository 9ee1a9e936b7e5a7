"""GPU: the block-scaled layers and the operators in front of them under torch.inference_mode give the bytes they give under
torch.no_grad, and train afterwards."""
import pytest
import torch

from tests.test_gpu_operator_layers import layer, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("error_feedback", [True, False])
def test_operators_and_layers(error_feedback):
    from tcfp_b200.nn import QuantizedRMSNorm, silu_mul

    norm = QuantizedRMSNorm(128, scale_block_size=64).to(DEV)
    up, down = layer(128, 512, error_feedback=error_feedback), layer(256, 128, error_feedback=error_feedback)
    x = rand(51, 33, 128, dtype=torch.bfloat16)

    def block(t):
        q, h = norm(t, t)
        return h + down(silu_mul(up(q), block_size=64)), up(t)

    with torch.inference_mode():
        first, second = block(x), block(x.clone())
    with torch.no_grad():
        want = block(x)
    for got in (first, second):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    xg = x.clone().requires_grad_()
    out, _ = block(xg)
    out.float().sum().backward()
    assert torch.equal(out, want[0]) and xg.grad.isfinite().all() and up.weight.grad.isfinite().all()
    with torch.no_grad():                       # a new weight is quantized anew
        up.weight.mul_(2.0)
        down.weight.mul_(0.5)
        third = block(x)
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(block(x), third))


def test_an_edited_plane_is_packed_again():
    from tcfp_b200 import kernels as K

    x, w = rand(52, 40, 128), rand(53, 64, 128)
    with torch.inference_mode():
        a, ea = K.block_quantize_fp8(x, 64)
        b, eb = K.block_quantize_fp8(w, 64)
        one = K.block_scaled_gemm(a, b, ea, eb, 64)
        ea += 1
        assert torch.equal(K.block_scaled_gemm(a, b, ea, eb, 64), 2 * one)
