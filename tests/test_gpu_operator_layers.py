"""GPU: the operators that hand a layer its 8-bit input, as a user has them:
``nn.add_rms_norm`` / ``silu_mul`` in front of ``TCFPLinear`` and ``Int8Linear``,
the decoder block built of them, int8 conversion."""
import copy

import pytest
import torch
import torch.nn.functional as F

from tests.util import gen, rel_fro

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen(seed)).to(dtype).to(DEV)


def layer(k, n, bs=64, **kw):
    from tcfp_b200.nn import TCFPLinear

    m = TCFPLinear(k, n, bias=True, use_tensor_cores=True, scale_block_size=bs, out_dtype=torch.bfloat16, **kw).to(DEV)
    with torch.no_grad():
        m.weight.copy_(rand(1, n, k) * 0.05)
        m.bias.copy_(rand(2, n) * 0.1)
    return m


@pytest.mark.parametrize("bs", [32, 64, 128])
@pytest.mark.parametrize("shape", [(1, 1), (3, 37), (2, 200)])
def test_norm_in_front_of_a_layer(bs, shape):
    """The layer multiplies the norm's codes as they are, and the gradients are those of the parts, bit for bit: the
    layer's own dX for those codes through the norm's backward pass, joined by the stream's gradient."""
    from tcfp_b200 import kernels as K
    from tcfp_b200.nn import QuantizedRMSNorm

    d, n = 384, 256
    lin = layer(d, n, bs)
    norm = QuantizedRMSNorm(d, scale_block_size=bs).to(DEV)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * rand(3, d))
    x = rand(4, *shape, d, dtype=torch.bfloat16).requires_grad_()
    r = rand(5, *shape, d, dtype=torch.bfloat16).requires_grad_()
    q, h = norm(x, r)
    y = lin(q)
    assert y.shape == (*shape, n) and h.shape == x.shape and q.shape == x.shape
    gy, gh = rand(6, *shape, n, dtype=torch.bfloat16), rand(7, *shape, d, dtype=torch.bfloat16)
    torch.autograd.backward([y, h], [gy, gh])

    q2, h2, rstd = K.add_rms_norm_quantize(x, norm.weight, r, 1e-5, block_size=bs)
    assert torch.equal(h2, h) and torch.equal(q2.codes.view(torch.uint8), q.codes.view(torch.uint8))
    err = lin._error_state._buffers[""]
    w_hi, w_lo, s_hi, s_lo = K.fused_dual_quantize_fp8(lin.weight.detach(), bs, torch.zeros_like(err), update_error=False)
    want = K.fused_block_scaled_dual_gemm_forward(q2.codes, w_hi, w_lo, q2.scales, s_hi, s_lo, bs, bias=lin.bias.detach(),
                                                  out_dtype=torch.bfloat16)
    assert torch.equal(y.reshape(-1, n), want)
    g2 = gy.reshape(-1, n)
    g8, gs, gb = K.block_quantize_fp8(g2, bs, torch.float8_e5m2, want_colsum=True)
    dq = K.fused_block_scaled_backward_dx(g8, w_hi, w_lo, gs, s_hi, s_lo, bs, out_dtype=torch.bfloat16)
    dx, dw = K.add_rms_norm_backward(dq.reshape(x.shape), h2, rstd, norm.weight, gh)
    assert torch.equal(x.grad, dx) and torch.equal(r.grad, dx) and torch.equal(norm.weight.grad, dw)
    assert torch.equal(lin.bias.grad, gb)
    assert torch.equal(lin.weight.grad, K.bf16_weight_grad(g2, K.block_dequantize_bf16(q2.codes, q2.scales, bs)))


def test_norm_gradient_paths():
    """One norm feeding two layers, a stream that nobody uses, an output that nobody uses, inputs without gradient, a bf16
    weight, an input that was broadcast."""
    from tcfp_b200.nn import add_rms_norm, dequantized

    d = 256
    a, b = layer(d, 128), layer(d, 192)
    w = torch.ones(d, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    row = rand(8, 1, d, dtype=torch.bfloat16).requires_grad_()
    x = row.expand(40, d)
    r = rand(9, 40, d, dtype=torch.bfloat16)
    q, h = add_rms_norm(x, w, r, block_size=64)
    (a(q).float().sum() + b(q).float().sum()).backward()
    assert row.grad.shape == (1, d) and w.grad.dtype == torch.bfloat16 and r.grad is None and row.grad.isfinite().all()
    ga, gw = row.grad.clone(), w.grad.clone()
    # the same two losses one after the other: bf16 gradients of the codes, summed by autograd in one case and not in the
    # other, so equal within their roundings: three of half a step each, against the largest term of every sum
    row.grad = w.grad = None
    for m in (a, b):
        q, _ = add_rms_norm(x, w, r, block_size=64)
        m(q).float().sum().backward()
    assert (row.grad.float() - ga.float()).abs().max() <= 3 * 2.0**-8 * 40 * ga.float().abs().max()
    assert (w.grad.float() - gw.float()).abs().max() <= 3 * 2.0**-8 * 2 * gw.float().abs().max()
    # only the stream
    row.grad = w.grad = None
    q, h = add_rms_norm(x, w, r, block_size=64)
    h.float().sum().backward()
    assert torch.equal(row.grad.float(), torch.full((1, d), 40.0, device=DEV)) and w.grad is None
    # only the codes, without a residual
    leaf = rand(10, 40, d).requires_grad_()
    q, same = add_rms_norm(leaf, w.detach(), block_size=64)
    assert same is leaf
    dequantized(q).float().square().sum().backward()
    assert leaf.grad.isfinite().all() and leaf.grad.abs().max() > 0
    with torch.no_grad():
        q, _ = add_rms_norm(leaf, w, block_size=64)
        assert not a(q).requires_grad


def test_gradients_match_the_formula_through_the_chain():
    """norm -> values -> gate -> values with FP32 inputs and int8 codes: the gradients are those of the operators in 64 bits
    at the points the codes stand for (the rounding passes them through)."""
    from tcfp_b200.nn import add_rms_norm, dequantized, silu_mul

    d = 96
    x, r = rand(11, 31, d).requires_grad_(), rand(12, 31, d).requires_grad_()
    w = (1 + 0.1 * rand(13, d)).requires_grad_()
    q, h = add_rms_norm(x, w, r)
    s = silu_mul(h[:, :48] * 1.0, h[:, 48:] * 1.0)
    gq, gs = rand(14, 31, d), rand(15, 31, 48)
    loss = (dequantized(q).float() * gq).sum() + (dequantized(s).float() * gs).sum() + h.sum()
    loss.backward()
    xd, rd, wd = (t.detach().double().requires_grad_() for t in (x, r, w))
    hd = xd + rd
    y = hd * (hd.square().mean(1, keepdim=True) + 1e-5).rsqrt() * wd
    # dequantized() is a bf16 tensor: the gradients that reach it are rounded to bf16
    round16 = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    ((y * round16(gq)).sum() + (F.silu(hd[:, :48]) * hd[:, 48:] * round16(gs)).sum() + hd.sum()).backward()
    size = xd.grad.abs() + 1 + gq.double().abs().amax() * 4
    assert ((x.grad - xd.grad).abs() <= 200 * U * size).all() and torch.equal(x.grad, r.grad)
    assert ((w.grad - wd.grad).abs() <= 64 * U * (gq.double().abs() * y.detach().abs()).sum(0) + 64 * U).all()


def test_layer_refusals_on_the_gpu():
    from tcfp_b200.nn import Int8Linear, TCFPLinear, add_rms_norm, silu_mul

    x = rand(16, 4, 128, dtype=torch.bfloat16).requires_grad_()
    w = torch.ones(128, device=DEV)
    q64, _ = add_rms_norm(x, w, block_size=64)
    q8, _ = add_rms_norm(x, w)
    with pytest.raises(ValueError, match="block_size"):
        layer(128, 128, 32)(q64)
    with pytest.raises(ValueError, match="block_size"):
        layer(128, 128, 64)(q8)
    with pytest.raises(ValueError, match="scale_block_size=None"):
        TCFPLinear(128, 128, use_tensor_cores=True).to(DEV)(q8)
    with pytest.raises(ValueError, match="input features"):
        layer(256, 128, 64)(q64)
    with pytest.raises(ValueError, match="hp_grad_weight"):
        layer(128, 128, 64, hp_grad_weight=True)(q64)
    i8 = Int8Linear(128, 64, device=DEV)
    with pytest.raises(RuntimeError, match="no backward"):
        i8(q8)
    with pytest.raises(RuntimeError, match="no backward"):
        i8(x)
    with torch.no_grad():
        with pytest.raises(ValueError, match="E4M3"):
            i8(q64)
        with pytest.raises(ValueError, match="input features"):
            i8(x[:, :64])
    for bad in (dict(residual=x[:2]), dict(residual=x.float()), dict(eps=-1.0), dict(eps=float("nan")), dict(block_size=48),
                dict(block_size=True)):
        with pytest.raises(ValueError):
            add_rms_norm(x, w, **bad)
    with pytest.raises(ValueError, match="weight"):
        add_rms_norm(x, w[:64])
    with pytest.raises(TypeError):
        add_rms_norm(x.half(), w)
    with pytest.raises(ValueError, match="32768"):
        add_rms_norm(torch.zeros(1, 32769, device=DEV), torch.ones(32769, device=DEV))
    with pytest.raises(ValueError, match="divisible"):
        silu_mul(torch.zeros(2, 96, device=DEV), block_size=32)


def test_warmup_and_fallback_take_the_values():
    """A layer in warm-up or switched to plain F.linear multiplies the values the codes stand for."""
    from tcfp_b200.nn import add_rms_norm

    lin = layer(128, 64, 64, warmup_steps=1)
    x = rand(17, 5, 128).requires_grad_()
    q, _ = add_rms_norm(x, torch.ones(128, device=DEV), block_size=64)
    y = lin(q)
    assert torch.equal(y, F.linear(q.dequantize().float(), lin.weight, lin.bias))
    y.sum().backward()
    assert x.grad.isfinite().all()
    lin.fallback_to_bf16()
    assert torch.equal(lin(q), y)
    lin.restore_tcfp()
    assert lin(q).dtype == torch.bfloat16


@pytest.mark.parametrize("rows", [1, 64, 300])
def test_training_step_of_a_block_replays_from_a_graph(rows):
    """norm -> layer -> gate -> layer, forward and backward captured and replayed with new inputs: the eager bytes."""
    from tcfp_b200.nn import QuantizedRMSNorm, silu_mul

    norm, up, down = QuantizedRMSNorm(128, scale_block_size=64).to(DEV), layer(128, 512), layer(256, 128)
    params = [norm.weight, *up.parameters(), *down.parameters()]

    def step(x, r):
        q, h = norm(x, r)
        out = h + down(silu_mul(up(q), block_size=64))
        return (out, *torch.autograd.grad(out.float().square().mean(), [x, r, *params]))

    x, r = (rand(s, rows, 128, dtype=torch.bfloat16).requires_grad_() for s in (18, 19))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x, r)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(x, r)
    for seed in (20, 21):
        with torch.no_grad():
            x.copy_(rand(seed, rows, 128, dtype=torch.bfloat16))
            r.copy_(rand(seed + 5, rows, 128, dtype=torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(x, r)):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# decoder
# ---------------------------------------------------------------------------

def decoder(**kw):
    from tcfp_b200.workloads import build_decoder

    torch.manual_seed(0)
    return build_decoder(2, 256, 4, 512, 64, **kw).to(DEV)


def exact_decoder(m, x):
    """The decoder's mathematics in FP32 with its FP32 weights, nothing quantized."""
    h = x
    for blk in m.layers:
        B, T, d = h.shape
        n = F.rms_norm(h, (d,), blk.norm1.weight, blk.norm1.eps)
        q, k, v = (t.reshape(B, T, blk.heads_local, blk.head_dim).transpose(1, 2)
                   for t in F.linear(n, blk.qkv.inner.weight).split(blk.qkv.local_sizes, -1))
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True).transpose(1, 2).reshape(B, T, d)
        h = h + F.linear(a, blk.o.inner.weight)
        n = F.rms_norm(h, (d,), blk.norm2.weight, blk.norm2.eps)
        g, u = F.linear(n, blk.gate_up.inner.weight).chunk(2, -1)
        h = h + F.linear(F.silu(g) * u, blk.down.inner.weight)
    return h


def test_decoder_with_fused_operators():
    """The block with the operators is as near to the unquantized mathematics as the block of plain passes: both make the
    same E4M3 and bf16 roundings except that the operators leave out one to bf16.  The errors are sums over 10^5 values, so
    they agree to a few per cent; 10 % are allowed."""
    plain, fused = decoder(), decoder(fused_ops=True)
    fused.load_state_dict(plain.state_dict())
    x = rand(22, 2, 96, 256, dtype=torch.bfloat16)
    gy = rand(23, 2, 96, 256, dtype=torch.bfloat16)
    xe = x.float().requires_grad_()
    ye = exact_decoder(plain, xe)
    ge = torch.autograd.grad(ye, [xe, *plain.parameters()], gy.float())
    got = []
    for m in (plain, fused):
        xm = x.clone().requires_grad_()
        y = m(xm)
        got.append((y, *torch.autograd.grad(y, [xm, *m.parameters()], gy)))
    names = ["out", "x", *dict(plain.named_parameters())]
    for name, e, a, b in zip(names, (ye, *ge), *got):
        assert a.shape == b.shape and a.dtype == b.dtype
        assert rel_fro(b, e) <= 1.1 * rel_fro(a, e) + 1e-3, (name, rel_fro(a, e), rel_fro(b, e))
    # one block called by itself
    one = plain.layers[0](x)
    assert rel_fro(fused.layers[0](x), one) <= 0.02 and fused.layers[0](x).dtype == one.dtype


def test_int8_linear():
    """Within what rounding the operands to int8 can do: x and w are off by half a step s_x, s_w each."""
    from tcfp_b200.nn import Int8Linear

    for k, n, shape, dtype in ((256, 192, (1,), torch.bfloat16), (333, 100, (3, 50), torch.float32), (4096, 512, (300,), torch.bfloat16)):
        lin = torch.nn.Linear(k, n).to(DEV)
        m = Int8Linear.from_linear(lin)
        assert m.out_dtype == torch.float32 and m.weight_codes.shape == (n, (k + 15) // 16 * 16)
        x = rand(24, *shape, k, dtype=dtype)
        y = m(x)
        assert y.shape == (*shape, n) and y.dtype == torch.float32
        xd, wd = x.double().reshape(-1, k), lin.weight.detach().double()
        sx, sw = xd.abs().amax(1, keepdim=True) / 127, wd.abs().amax(1) / 127
        want = xd @ wd.t() + lin.bias.detach().double()
        # half a step, a little more where the FP32 quotient rounds a tie the other way
        room = 0.5001 * (xd.abs().sum(1, keepdim=True) * sw + wd.abs().sum(1) * sx) + 0.26 * k * sx * sw + 1e-5
        assert ((y.double().reshape(-1, n) - want).abs() <= room).all()
        # what was saved is what runs
        other = Int8Linear(k, n, device=DEV)
        other.load_state_dict(copy.deepcopy(m.state_dict()))
        assert torch.equal(other(x), y)
        assert m(x[:0]).shape == (*((0,) + shape[1:]), n)


def test_convert_to_int8():
    """A trained decoder answers in int8: the stream's update is within what the roundings do.  A row of n values rounded to
    int8 is off by max/127/sqrt(12), 0.9 % of its deviation for the 4 deviations a Gaussian row reaches and 2.5 % for the
    heavier gated product; a product of two roundings joins to 1.3 %, the chain of a block (q/k/v, o; gate and up, down) to
    below 5 %, two blocks to 7 %: 10 % are allowed."""
    from tcfp_b200.nn import Int8Linear, convert_to_int8

    m = decoder(fused_ops=True)
    exact = copy.deepcopy(m)
    convert_to_int8(m)
    assert sum(isinstance(s, Int8Linear) for s in m.modules()) == 8
    for T in (1, 7, 200):
        x = rand(25, 1, T, 256, dtype=torch.bfloat16)
        with torch.no_grad():
            y, e = m(x), exact_decoder(exact, x.float())
        assert y.shape == x.shape and y.dtype == torch.bfloat16
        assert float((y.double() - e.double()).norm() / (e.double() - x.double()).norm()) <= 0.1
    seq = torch.nn.Sequential(torch.nn.Linear(64, 64), torch.nn.Sequential(torch.nn.Linear(64, 32))).to(DEV)
    seq.add_module("head", torch.nn.Linear(32, 8).to(DEV))
    convert_to_int8(seq)
    assert isinstance(seq[0], Int8Linear) and isinstance(seq[1][0], Int8Linear) and isinstance(seq.head, torch.nn.Linear)


def test_int8_models_survive_casts_and_attention_modules():
    from tcfp_b200.nn import Int8Linear, convert_to_int8

    class Net(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.attn = torch.nn.MultiheadAttention(64, 2, batch_first=True)
            self.fc = torch.nn.Linear(64, 48)

        def forward(self, x):
            return self.fc(self.attn(x, x, x)[0])

    net = convert_to_int8(Net().to(DEV))
    assert isinstance(net.fc, Int8Linear) and not isinstance(net.attn.out_proj, Int8Linear)
    x = rand(26, 2, 5, 64)
    with torch.no_grad():
        y = net(x)
        scale = net.fc.weight_scale.clone()
        net.to(torch.bfloat16)
        assert net.fc.weight_scale.dtype == net.fc.bias.dtype == torch.float32 and torch.equal(net.fc.weight_scale, scale)
        # attention in bf16: 8 bits in and out, a softmax of 5 terms
        assert rel_fro(net(x.to(torch.bfloat16)), y) <= 0.05


def test_sequence_parallel_io_passes_quantized_codes():
    """With the collectives of one rank the layer's gathers see the codes and planes of the operator."""
    from tcfp_b200.nn import LayerHooks, add_rms_norm
    from tcfp_b200.tp import SequenceParallelIO

    class Doubling(SequenceParallelIO):      # two ranks that hold the same tokens
        def gather_rows(self, t):
            return torch.cat([t.view(torch.uint8), t.view(torch.uint8)]).view(t.dtype)

        def gather_planes(self, planes):
            return torch.cat([planes, planes], dim=1)

        def scatter_rows_async(self, full):
            n = full.shape[0] // 2
            return None, full[:n] + full[n:]

    lin = layer(128, 64, error_feedback=False)      # with it the second forward quantizes the weight plus the first one's error
    x = rand(27, 160, 128, dtype=torch.bfloat16).requires_grad_()
    w = torch.ones(128, device=DEV)
    y = lin(add_rms_norm(torch.cat([x, x]), w, block_size=64)[0])       # the same number of rows: the same tiles and sums
    gy = rand(28, 160, 64, dtype=torch.bfloat16)
    (gx,) = torch.autograd.grad(lin(add_rms_norm(x, w, block_size=64)[0]), x, gy)
    lin._hooks = LayerHooks(sp=Doubling())
    z = lin(add_rms_norm(x, w, block_size=64)[0])
    assert torch.equal(z, y)
    (gz,) = torch.autograd.grad(z, x, torch.cat([gy, gy]))
    # twice every gradient, formed by an addition of two equal bf16 numbers: exact until the norm's own rounding
    assert (gz.float() - 2 * gx.float()).abs().max() <= 2 * 2.0**-8 * gx.float().abs().max()


def test_convert_to_int8_refuses_communicating_layers():
    from tcfp_b200.nn import LayerHooks, TCFPLinear, convert_to_int8

    lin = TCFPLinear(64, 64, use_tensor_cores=True).to(DEV)
    lin._hooks = LayerHooks(out_hook=lambda y: None)
    with pytest.raises(ValueError, match="ranks"):
        convert_to_int8(torch.nn.Sequential(lin))
