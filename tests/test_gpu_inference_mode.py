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


@pytest.mark.parametrize("residual", [True, False])
def test_input_gradient_product(residual):
    """The weight re-targeted for the input gradient is formed again where its operands have no version counter."""
    from tcfp_b200 import kernels as K

    w, g = rand(54, 192, 128), rand(55, 70, 192, dtype=torch.bfloat16)

    def product(edit):
        hi, lo, eh, el = K.fused_dual_quantize_fp8(w, 64, torch.zeros_like(w))
        if not residual:
            lo = el = None
        gq, eg = K.block_quantize_fp8(g, 64, torch.float8_e5m2)
        one = K.fused_block_scaled_backward_dx(gq, hi, lo, eg, eh, el, 64)
        if edit:
            eh += 1
            if residual:
                el += 1
        return one, K.fused_block_scaled_backward_dx(gq, hi, lo, eg, eh, el, 64)

    want, _ = product(False)
    with torch.inference_mode():
        one, two = product(True)
    assert torch.equal(one, want) and torch.equal(two, 2 * want)
