"""Cases of the operators around an 8-bit linear layer: the RMS norm with the residual's addition and an 8-bit
output, the gated activation with an 8-bit output, both directions of each, and the matrix product of 8-bit
integers with a scale for each token and each channel.

``run`` computes a case in its plain form, elementary torch operations in 32 bits, or, where ``own`` is true, with
the calls of ``tcfp_b200.kernels``.  Quantized outputs come back as the values they stand for.
"""
import math

import torch

own = False

EPS = 1e-5


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
# op "norm" / "gate": rows x width, dtype, block (scale block of the E4M3 codes; 0: int8 with a scale for each row),
# backward; "norm" also add (with a residual).  op "linear": rows x k activations times an n x k weight; codes: the
# activations are codes already.  op "mlp": norm, gate/up product, gated activation, down product.

def listed():
    return [
        # one token of a decoder with d = 4096 being generated: latency
        dict(name="norm_int8_one_token", op="norm", rows=1, width=4096, dtype="bf16", block=0, add=True, backward=False),
        # the training step of the decoder workload: 8 x 4096 tokens, block-64 codes for the product behind the norm
        dict(name="norm_block64_train", op="norm", rows=32768, width=4096, dtype="bf16", block=64, add=True, backward=False),
        # ... and its backward pass, the residual stream's gradient joining
        dict(name="norm_backward_train", op="norm", rows=32768, width=4096, dtype="bf16", block=64, add=True, backward=True),
        # a ragged batch in 32 bits, a width no vector divides, nothing to add
        dict(name="norm_int8_f32_odd", op="norm", rows=1003, width=2731, dtype="f32", block=0, add=False, backward=False),
        # the feed-forward activation of the same decoder over half a step's tokens
        dict(name="gate_block64_train", op="gate", rows=16384, width=11008, dtype="bf16", block=64, backward=False),
        dict(name="gate_backward_train", op="gate", rows=16384, width=11008, dtype="bf16", block=64, backward=True),
        # a few sequences at once, an odd width
        dict(name="gate_int8_ragged", op="gate", rows=37, width=1365, dtype="bf16", block=0, backward=False),
        # prompts through the fused q/k/v projection
        dict(name="linear_prompts", op="linear", rows=8192, n=12288, k=4096, dtype="bf16", bias=False, codes=False),
        # one token through the fused gate/up projection: the weight's bytes are the time
        dict(name="linear_one_token", op="linear", rows=1, n=22016, k=4096, dtype="bf16", bias=False, codes=False),
        # 32 sequences generating together, the down projection
        dict(name="linear_32_tokens", op="linear", rows=32, n=4096, k=11008, dtype="bf16", bias=False, codes=False),
        # sizes that no tile divides, with a bias and a 32-bit output
        dict(name="linear_odd", op="linear", rows=333, n=1001, k=2031, dtype="f32", bias=True, codes=True),
        # the operators together: the feed-forward half of a block for 16 sequences
        dict(name="mlp_16_tokens", op="mlp", rows=16, width=4096, hidden=11008, dtype="bf16"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "gate", "gate", "linear", "linear", "linear", "mlp"])
    if op == "linear":
        codes = rng.random() < 0.3
        return dict(op=op, rows=_log_uniform(rng, 1, 8192), n=_log_uniform(rng, 64, 12288), k=_log_uniform(rng, 64, 4096),
                    dtype=rng.choice(["bf16", "f32"]) if codes else "bf16", bias=rng.random() < 0.5, codes=codes)
    if op == "mlp":
        return dict(op=op, rows=_log_uniform(rng, 1, 1024), width=_log_uniform(rng, 256, 4096),
                    hidden=_log_uniform(rng, 512, 11008), dtype="bf16")
    block = rng.choice([0, 0, 32, 64, 128])
    width = _log_uniform(rng, 64, 4096 if op == "norm" else 11008)
    width = max(width // block, 1) * block if block else width
    case = dict(op=op, rows=_log_uniform(rng, 1, 16384), width=width, dtype=rng.choice(["bf16", "bf16", "f32"]), block=block,
                backward=rng.random() < 0.4)
    if op == "norm":
        case["add"] = rng.random() < 0.7
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _stream(g, rows, width, dtype):
    """A residual stream: channels of different sizes, a few large ones, the last rows of a padded batch zero."""
    x = torch.randn(rows, width, generator=g, device="cuda") * (0.5 + torch.rand(width, generator=g, device="cuda"))
    x[:, ::509] *= 20.0
    if rows > 8:
        x[rows - rows // 16 - 1:] = 0.0
    return x.to(dtype)


def _codes(g, rows, k):
    """A matrix held as int8 codes with a scale for each row; rows start on 16-byte boundaries."""
    w = torch.randn(rows, k, generator=g, device="cuda") * 0.02
    scale = w.abs().amax(dim=1) / 127.0
    held = torch.zeros(rows, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    held[:, :k] = torch.round(w / scale[:, None]).clamp(-127, 127).to(torch.int8)
    return held[:, :k], scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case=case)
    op, rows = case["op"], case["rows"]
    if op == "norm":
        width, dt = case["width"], _dtype(case)
        s["weight"] = 1.0 + 0.1 * torch.randn(width, generator=g, device="cuda")
        if not case["backward"]:
            s["x"] = _stream(g, rows, width, dt)
            s["residual"] = _stream(g, rows, width, dt) if case["add"] else None
        else:
            # what the forward pass kept, and the gradients that arrive
            s["h"] = _stream(g, rows, width, dt)
            s["rstd"] = torch.rsqrt(s["h"].double().square().mean(dim=1) + EPS).float()
            s["grad"] = (torch.randn(rows, width, generator=g, device="cuda") * 0.01).to(dt)
            s["grad_h"] = (torch.randn(rows, width, generator=g, device="cuda") * 0.01).to(dt) if case["add"] else None
    elif op == "gate":
        width, dt = case["width"], _dtype(case)
        s["gate_up"] = torch.randn(rows, 2 * width, generator=g, device="cuda", dtype=dt) * 1.5
        if case["backward"]:
            s["grad"] = (torch.randn(rows, width, generator=g, device="cuda") * 0.01).to(dt)
    elif op == "linear":
        s["w"], s["w_scale"] = _codes(g, case["n"], case["k"])
        s["bias"] = torch.randn(case["n"], generator=g, device="cuda") if case["bias"] else None
        if case["codes"]:
            s["a"], s["a_scale"] = _codes(g, rows, case["k"])
        else:
            s["x"] = torch.randn(rows, case["k"], generator=g, device="cuda").to(torch.bfloat16)
    else:
        width, hidden = case["width"], case["hidden"]
        s["weight"] = 1.0 + 0.1 * torch.randn(width, generator=g, device="cuda")
        s["x"] = _stream(g, rows, width, torch.bfloat16)
        s["residual"] = _stream(g, rows, width, torch.bfloat16)
        s["w"], s["w_scale"] = _codes(g, 2 * hidden, width)
        s["w2"], s["w2_scale"] = _codes(g, width, hidden)
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------

def _block_values(y, block):
    """Values of E4M3 codes with a power of two for each block."""
    v = y.reshape(y.shape[0], -1, block)
    e = torch.ceil(torch.log2(v.abs().amax(dim=2, keepdim=True).clamp(min=1e-12).double() / 448.0)).clamp(min=-126.0).float()
    code = (v * torch.exp2(-e)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return (code.float() * torch.exp2(e)).reshape(y.shape)


def _row_codes(y):
    """int8 codes (as 32-bit numbers) with a scale for each row."""
    scale = y.abs().amax(dim=1).clamp(min=1e-12) / 127.0
    return torch.round(y / scale[:, None]).clamp(-127.0, 127.0), scale


def _quantized(y, block):
    if block:
        return {"values": _block_values(y, block).to(torch.bfloat16)}
    code, scale = _row_codes(y)
    return {"values": (code * scale[:, None]).to(torch.bfloat16), "scales": scale}


def _norm(x, residual, weight):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).mean(dim=1) + EPS)
    return h, rstd, hf * rstd[:, None] * weight.float()


def _gated(gate_up):
    gate, up = gate_up.float().chunk(2, dim=1)
    return gate / (1.0 + torch.exp(-gate)) * up


def _product(code, scale, w, w_scale, bias, dtype):
    out = (code.float() @ w.float().t()) * scale[:, None] * w_scale
    return (out if bias is None else out + bias).to(dtype)


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "norm" and not case["backward"]:
        h, rstd, y = _norm(s["x"], s["residual"], s["weight"])
        out = dict(_quantized(y, case["block"]), rstd=rstd)
        if case["add"]:
            out["h"] = h
        return out
    if op == "norm":
        hat = s["h"].float() * s["rstd"][:, None]
        dy = s["grad"].float()
        g = dy * s["weight"]
        dx = s["rstd"][:, None] * (g - hat * (g * hat).mean(dim=1, keepdim=True))
        if case["add"]:
            dx = dx + s["grad_h"].float()
        return {"dx": dx.to(s["h"].dtype), "dw": (dy * hat).sum(dim=0)}
    if op == "gate" and not case["backward"]:
        return _quantized(_gated(s["gate_up"]), case["block"])
    if op == "gate":
        gate, up = s["gate_up"].float().chunk(2, dim=1)
        dy = s["grad"].float()
        sig = 1.0 / (1.0 + torch.exp(-gate))
        d = torch.cat([dy * up * sig * (1.0 + gate * (1.0 - sig)), dy * gate * sig], dim=1)
        return {"d_gate_up": d.to(s["gate_up"].dtype)}
    if op == "linear":
        code, scale = (s["a"], s["a_scale"]) if case["codes"] else _row_codes(s["x"].float())
        return {"out": _product(code, scale, s["w"], s["w_scale"], s["bias"], _dtype(case))}
    h, _, y = _norm(s["x"], s["residual"], s["weight"])
    gate_up = _product(*_row_codes(y), s["w"], s["w_scale"], None, torch.bfloat16)
    return {"h": h, "out": _product(*_row_codes(_gated(gate_up)), s["w2"], s["w2_scale"], None, torch.bfloat16)}


def _own(s):
    from tcfp_b200 import kernels as K

    case = s["case"]
    op = case["op"]
    if op == "norm" and not case["backward"]:
        q, h, rstd = K.add_rms_norm_quantize(s["x"], s["weight"], s["residual"], EPS, block_size=case["block"] or None,
                                             want_bf16=True)
        out = {"values": q.bf16, "rstd": rstd}
        if not case["block"]:
            out["scales"] = q.scales
        if case["add"]:
            out["h"] = h
        return out
    if op == "norm":
        dx, dw = K.add_rms_norm_backward(s["grad"], s["h"], s["rstd"], s["weight"], s["grad_h"])
        return {"dx": dx, "dw": dw}
    if op == "gate" and not case["backward"]:
        q = K.silu_mul_quantize(s["gate_up"], block_size=case["block"] or None, want_bf16=True)
        return {"values": q.bf16} if case["block"] else {"values": q.bf16, "scales": q.scales}
    if op == "gate":
        return {"d_gate_up": K.silu_mul_backward(s["grad"], s["gate_up"])}
    if op == "linear":
        if case["codes"]:
            a, a_scale = s["a"], s["a_scale"]
        else:
            q = K.int8_quantize_rows(s["x"])
            a, a_scale = q.codes, q.scales
        return {"out": K.int8_matmul(a, s["w"], a_scale, s["w_scale"], bias=s["bias"], out_dtype=_dtype(case))}
    q, h, _ = K.add_rms_norm_quantize(s["x"], s["weight"], s["residual"], EPS)
    gate_up = K.int8_matmul(q.codes, s["w"], q.scales, s["w_scale"], out_dtype=torch.bfloat16)
    q = K.silu_mul_quantize(gate_up)
    return {"h": h, "out": K.int8_matmul(q.codes, s["w2"], q.scales, s["w2_scale"], out_dtype=torch.bfloat16)}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the least a pass has to move and compute
# ---------------------------------------------------------------------------

def work(case):
    op, rows = case["op"], case["rows"]
    if op == "linear":
        n, k = case["n"], case["k"]
        out = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": rows * k * (1 if case["codes"] else 2) + n * k + rows * n * out + 4 * n, "flops": 2.0 * rows * n * k}
    if op == "mlp":
        d, f = case["width"], case["hidden"]
        return {"bytes": 3 * d * f + rows * d * 2 * 4 + 4 * (2 * d + 2 * f), "flops": 6.0 * rows * d * f}
    n = rows * case["width"]
    e = 2 if case["dtype"] == "bf16" else 4
    scales = n / case["block"] if case["block"] else 4 * rows
    if op == "norm":
        tail = 4 * case["width"] + 4 * rows
        if case["backward"]:
            return {"bytes": n * e * (4 if case["add"] else 3) + 2 * tail, "flops": 14.0 * n}
        return {"bytes": n * (e * (3 if case["add"] else 1) + 1 + 2) + scales + tail, "flops": 10.0 * n}
    if case["backward"]:
        return {"bytes": 5 * e * n, "flops": 14.0 * n}
    return {"bytes": n * (2 * e + 1 + 2) + scales, "flops": 10.0 * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _e4m3_exact(v):
    """Nearest E4M3 number, ties to even: a step is 2^(exponent - 3), from 2^-9 up."""
    a = v.abs().clamp(max=448.0)
    _, e = torch.frexp(a)
    step = torch.pow(2.0, (e.double() - 4.0).clamp(min=-9.0))
    return torch.sign(v) * (torch.round(a / step) * step).clamp(max=448.0)


def _exact_quantized(y, block):
    rows, width = y.shape
    if block:
        blocks = y.view(rows, width // block, block)
        top = blocks.abs().max(dim=-1).values.clamp_min(1e-12)
        unit = torch.pow(2.0, torch.ceil(torch.log2(top / 448.0)).clamp_min(-126.0)).unsqueeze(-1)
        return {"values": (_e4m3_exact(blocks / unit) * unit).view(rows, width)}
    s = y.abs().max(dim=1, keepdim=True).values.clamp_min(1e-12) / 127.0
    return {"values": torch.round(y / s) * s, "scales": s.squeeze(1)}


def _exact_norm(x, residual, weight):
    # the stream is kept in the inputs' type: its rounding belongs to the definition
    h = x.double() if residual is None else (x.double() + residual.double()).to(x.dtype).double()
    power = torch.einsum("ij,ij->i", h, h) / h.shape[1]
    return h, (power + EPS) ** -0.5, h * ((power + EPS) ** -0.5)[:, None] * weight.double()


def _exact_codes(y):
    s = (y.abs().max(dim=1, keepdim=True).values.clamp_min(1e-12) / 127.0).float().double()
    return torch.round(y / s), s


def _exact_linear(code, s, w, w_scale):
    return torch.mm(code.double(), w.double().t()) * (s.double().reshape(-1, 1) * w_scale.double().reshape(1, -1))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm" and not case["backward"]:
        h, rstd, y = _exact_norm(s["x"], s["residual"], s["weight"])
        out = dict(_exact_quantized(y, case["block"]), rstd=rstd)
        if case["add"]:
            out["h"] = h
        return out
    if op == "norm":
        h, r, dy = s["h"].double(), s["rstd"].double().unsqueeze(1), s["grad"].double()
        g = dy * s["weight"].double()
        along = torch.einsum("ij,ij->i", g, h).unsqueeze(1) / h.shape[1]
        dx = r * g - r ** 3 * along * h
        if case["add"]:
            dx += s["grad_h"].double()
        return {"dx": dx, "dw": torch.einsum("ij,ij,i->j", dy, h, r.squeeze(1))}
    if op == "gate":
        f = case["width"]
        gate, up = s["gate_up"][:, :f].double(), s["gate_up"][:, f:].double()
        sig = torch.sigmoid(gate)
        if not case["backward"]:
            return _exact_quantized(gate * sig * up, case["block"])
        dy = s["grad"].double()
        return {"d_gate_up": torch.cat([dy * up * (sig + gate * sig * (1 - sig)), dy * gate * sig], dim=1)}
    if op == "linear":
        code, scale = (s["a"], s["a_scale"]) if case["codes"] else _exact_codes(s["x"].double())
        out = _exact_linear(code, scale, s["w"], s["w_scale"])
        return {"out": out if s["bias"] is None else out + s["bias"].double()}
    h, _, y = _exact_norm(s["x"], s["residual"], s["weight"])
    f = case["hidden"]
    gu = _exact_linear(*_exact_codes(y), s["w"], s["w_scale"]).to(torch.bfloat16).double()  # kept in 16 bits between the two
    return {"h": h, "out": _exact_linear(*_exact_codes(gu[:, :f] * torch.sigmoid(gu[:, :f]) * gu[:, f:]), s["w2"], s["w2_scale"])}
