"""GPU: an operator whose output feeds two layers gets the sum of their gradients, bit for bit."""
import pytest
import torch

from tests.test_gpu_operator_layers import layer, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_one_norm_two_layers(rows):
    """Each layer's gradient of the shared codes, taken by itself; their sum in bf16, the type of the stream, through the norm's
    backward pass with the stream's own gradient; then the sum over the rows of a broadcast input."""
    from tcfp_b200 import kernels as K
    from tcfp_b200.nn import add_rms_norm

    d = 256
    # without error feedback, so that a second forward pass quantizes the same weight
    a, b = layer(d, 128, error_feedback=False), layer(d, 192, error_feedback=False)
    w = (1 + 0.1 * rand(31, d)).requires_grad_()
    x, r = rand(32, rows, d, dtype=torch.bfloat16).requires_grad_(), rand(33, rows, d, dtype=torch.bfloat16)
    ga, gb = rand(34, rows, 128, dtype=torch.bfloat16), rand(35, rows, 192, dtype=torch.bfloat16)
    gh = rand(36, rows, d, dtype=torch.bfloat16)

    q, h = add_rms_norm(x, w, r, block_size=64)
    (da,) = torch.autograd.grad(a(q), q._handle, ga, retain_graph=True)
    (db,) = torch.autograd.grad(b(q), q._handle, gb, retain_graph=True)
    assert da.dtype == db.dtype == torch.bfloat16 and da.abs().max() > 0 and db.abs().max() > 0
    rstd = K.add_rms_norm_quantize(x, w, r, 1e-5, block_size=64)[2]
    dx, dw = K.add_rms_norm_backward(da + db, h.detach(), rstd, w, gh)
    torch.autograd.backward([a(q), b(q), h], [ga, gb, gh])
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)

    row = rand(37, 1, d, dtype=torch.bfloat16).requires_grad_()
    q, h = add_rms_norm(row.expand(rows, d), w, r, block_size=64)
    (da,) = torch.autograd.grad(a(q), q._handle, ga, retain_graph=True)
    (db,) = torch.autograd.grad(b(q), q._handle, gb, retain_graph=True)
    rstd = K.add_rms_norm_quantize(row.expand(rows, d), w, r, 1e-5, block_size=64)[2]
    dx, _ = K.add_rms_norm_backward(da + db, h.detach(), rstd, w)
    torch.autograd.backward([a(q), b(q)], [ga, gb])
    assert torch.equal(row.grad, dx.sum(0, keepdim=True))


def test_one_gate_two_layers():
    from tcfp_b200 import kernels as K
    from tcfp_b200.nn import silu_mul

    a, b = layer(128, 64, error_feedback=False), layer(128, 192, error_feedback=False)
    x = rand(38, 70, 256, dtype=torch.bfloat16).requires_grad_()
    ga, gb = rand(39, 70, 64, dtype=torch.bfloat16), rand(40, 70, 192, dtype=torch.bfloat16)
    q = silu_mul(x, block_size=64)
    (da,) = torch.autograd.grad(a(q), q._handle, ga, retain_graph=True)
    (db,) = torch.autograd.grad(b(q), q._handle, gb, retain_graph=True)
    torch.autograd.backward([a(q), b(q)], [ga, gb])
    assert torch.equal(x.grad, K.silu_mul_backward(da + db, x))
