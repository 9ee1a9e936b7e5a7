"""Launch wrappers with the names and return conventions of the reference's
``tcfp/kernels.py`` (:1537-2469), backed by ``libtcfp_b200.so``.

Every wrapper allocates its outputs with torch (as the reference's do,
tcfp/kernels.py:1572, 1699-1700, 1806-1813), hands raw pointers and the current
stream to the C ABI, and raises on failure -- there is no Triton and no CPU
path behind these names.

Additions the reference does not have, all keyword-only and optional:
``seed`` / ``offset`` for the stochastic residual (the reference draws a fresh
seed per launch, tcfp/kernels.py:1828-1831), ``update_error`` (read the error
buffer without writing it, replacing the clone at tcfp/nn/__init__.py:607-608)
and ``out_dtype``.
"""
from __future__ import annotations

import math

import torch

from . import _C

_FP8_E4M3_MAX = 448.0
_FP8_E5M2_MAX = 57344.0
_FP8_DTYPES = (torch.float8_e4m3fn, torch.float8_e5m2)


def is_triton_available() -> bool:
    """Capability probe kept under its reference name (tcfp/kernels.py:1537):
    True when the fused kernels can run, i.e. the library loads on sm_100."""
    return _C.is_available()


def _fmt(t: torch.Tensor) -> int:
    if t.dtype == torch.float8_e4m3fn:
        return _C.E4M3
    if t.dtype == torch.float8_e5m2:
        return _C.E5M2
    raise TypeError(f"expected an FP8 tensor, got {t.dtype}")


def _out_code(dtype: torch.dtype) -> int:
    if dtype == torch.float32:
        return _C.F32
    if dtype == torch.bfloat16:
        return _C.BF16
    raise TypeError(f"out_dtype must be float32 or bfloat16, got {dtype}")


def _scalar(t: torch.Tensor) -> torch.Tensor:
    assert t.numel() == 1 and t.dtype == torch.float32, "scales must be 1-element float32 tensors"
    return t


# ---------------------------------------------------------------------------
# packed scale factors ride along with the reference-layout exponent planes
# ---------------------------------------------------------------------------

def _alloc_sf(rows: int, K: int, bs: int, device) -> torch.Tensor:
    n = _C.load().tcfp_sf_packed_bytes(rows, K, bs)
    return torch.empty(n, dtype=torch.uint8, device=device)


def packed_scale_rows(sf: torch.Tensor, r0: int, r1: int, K: int, block_size: int) -> torch.Tensor:
    """The part of a packed scale-factor array that covers rows ``[r0, r1)``
    of its operand (``r0`` a multiple of 128: chunks hold 128 rows each)."""
    assert r0 % 128 == 0, "row slices of packed scale factors start on multiples of 128"
    per_row_block = ((K // block_size + 3) // 4) * 512
    return sf[(r0 // 128) * per_row_block:((r1 + 127) // 128) * per_row_block]


def _attach_sf(exps: torch.Tensor, sf: torch.Tensor, block_size: int) -> None:
    # the packed copy is only valid for the bytes it was packed from: remember the plane's
    # version counter and address so that an in-place edit or a re-bound storage repacks.  An inference tensor has no
    # counter: its plane is packed again where it is used
    if exps.is_inference():
        return
    exps._tcfp_sf = (sf, exps._version, exps.data_ptr(), block_size)


def pack_block_scales(exps: torch.Tensor, block_size: int) -> torch.Tensor:
    """int8 exponent plane ``(K // bs, rows)`` -> packed E8M0 chunk array.
    A quantizer of this module attaches the packed copy it wrote in the same
    pass; it is reused only while the plane is unmodified."""
    cached = getattr(exps, "_tcfp_sf", None)
    if cached is not None:
        sf, version, addr, bs = cached
        if version == exps._version and addr == exps.data_ptr() and bs == block_size:
            return sf
    assert exps.dtype == torch.int8 and exps.ndim == 2 and exps.is_contiguous()
    num_kb, rows = exps.shape
    K = num_kb * block_size
    sf = _alloc_sf(rows, K, block_size, exps.device)
    _C.check(_C.load().tcfp_pack_scales(_C.ptr(exps), _C.ptr(sf), rows, K, block_size, _C.stream()))
    return sf


# ---------------------------------------------------------------------------
# per-tensor dual GEMM (tcfp/kernels.py:1545-1666)
# ---------------------------------------------------------------------------

def fused_dual_gemm_forward(act_fp8, w_hi_fp8, w_lo_fp8, act_inv, w_hi_inv, w_lo_inv, *,
                            bias=None, out_dtype=torch.float32, out=None):
    """``(act @ W_hi.T) * s + (act @ W_lo.T) * s`` -> ``(M, N)``
    (tcfp/kernels.py:1545-1601).  ``w_lo_fp8`` / ``w_lo_inv`` may be ``None``."""
    M, K = act_fp8.shape
    N, K2 = w_hi_fp8.shape
    assert K == K2 and (w_lo_fp8 is None or w_lo_fp8.shape == (N, K)), (
        f"Shape mismatch: act({M},{K}), w_hi({N},{K2}), w_lo{None if w_lo_fp8 is None else tuple(w_lo_fp8.shape)}"
    )
    assert act_fp8.is_contiguous() and w_hi_fp8.is_contiguous(), "operands must be contiguous"
    if out is None:
        out = torch.empty((M, N), device=act_fp8.device, dtype=out_dtype)
    else:
        assert out.shape == (M, N) and out.dtype == out_dtype and out.is_contiguous(), "bad out buffer"
    _C.check(_C.load().tcfp_dual_gemm(
        _C.ptr(act_fp8), _fmt(act_fp8), _C.ptr(w_hi_fp8), _C.ptr(w_lo_fp8),
        _C.ptr(_scalar(act_inv)), _C.ptr(_scalar(w_hi_inv)), _C.ptr(None if w_lo_inv is None else _scalar(w_lo_inv)),
        _C.ptr(bias), _C.ptr(out), _out_code(out_dtype), M, N, K, 0, _C.stream()))
    return out


def fused_dual_gemm_backward_dx(grad_fp8, w_hi_fp8, w_lo_fp8, grad_inv, w_hi_inv, w_lo_inv, *,
                                out_dtype=torch.float32):
    """``(grad @ W_hi) * s + (grad @ W_lo) * s`` -> ``(M, D_in)``
    (tcfp/kernels.py:1604-1666); the weights stay in their ``(D_out, D_in)``
    layout."""
    M, D_out = grad_fp8.shape
    D_out2, D_in = w_hi_fp8.shape
    assert D_out == D_out2 and (w_lo_fp8 is None or w_lo_fp8.shape == (D_out, D_in)), (
        f"Shape mismatch: grad({M},{D_out}), w_hi({D_out2},{D_in})"
    )
    assert grad_fp8.is_contiguous() and w_hi_fp8.is_contiguous(), "operands must be contiguous"
    out = torch.empty((M, D_in), device=grad_fp8.device, dtype=out_dtype)
    _C.check(_C.load().tcfp_dual_gemm(
        _C.ptr(grad_fp8), _fmt(grad_fp8), _C.ptr(w_hi_fp8), _C.ptr(w_lo_fp8),
        _C.ptr(_scalar(grad_inv)), _C.ptr(_scalar(w_hi_inv)), _C.ptr(None if w_lo_inv is None else _scalar(w_lo_inv)),
        None, _C.ptr(out), _out_code(out_dtype), M, D_in, D_out, 1, _C.stream()))
    return out


def fp8_weight_grad(grad_fp8, act_fp8, grad_inv, act_inv, *, out_dtype=torch.float32):
    """``dW = (grad^T @ act) * (s_g * s_a)`` -> ``(D_out, D_in)`` from the
    gradient ``(M, D_out)`` and the saved activation codes ``(M, D_in)`` as
    they are (tcfp/nn/__init__.py:546-555 without the transposed copies)."""
    M, D_out = grad_fp8.shape
    M2, D_in = act_fp8.shape
    assert M == M2, f"Shape mismatch: grad({M},{D_out}), act({M2},{D_in})"
    assert grad_fp8.is_contiguous() and act_fp8.is_contiguous(), "operands must be contiguous"
    out = torch.empty((D_out, D_in), device=grad_fp8.device, dtype=out_dtype)
    _C.check(_C.load().tcfp_dw_gemm(
        _C.ptr(grad_fp8), _fmt(grad_fp8), _C.ptr(act_fp8), _C.ptr(_scalar(grad_inv)), _C.ptr(_scalar(act_inv)),
        _C.ptr(out), _out_code(out_dtype), M, D_out, D_in, _C.stream()))
    return out


def split_bf16(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """FP32 tensor -> ``(head, tail)`` bf16 with ``head = bf16(x)`` and
    ``tail = bf16(x - head)``: ``head + tail`` carries 16 significant bits of
    ``x``.  One pass (the three torch operations it replaces move 22 B/elem)."""
    assert x.dtype == torch.float32 and x.is_cuda
    x = x.contiguous()
    if x.numel() % 4 != 0:
        head = x.to(torch.bfloat16)
        return head, (x - head.float()).to(torch.bfloat16)
    head = torch.empty_like(x, dtype=torch.bfloat16)
    tail = torch.empty_like(head)
    _C.check(_C.load().tcfp_split_bf16(_C.ptr(x), _C.ptr(head), _C.ptr(tail), x.numel(), _C.stream()))
    return head, tail


def bf16_weight_grad(grad: torch.Tensor, act_bf16: torch.Tensor) -> torch.Tensor:
    """``dW = grad^T @ act`` -> ``(D_out, D_in)`` FP32 for an FP32 (or bf16)
    gradient ``(M, D_out)`` and a bf16 activation ``(M, D_in)``: the gradient
    is split into a bf16 head and tail (16 significant bits) and both ride one
    bf16 tensor-core GEMM -- the FP32 matmul of tcfp/nn/__init__.py:744-750 at
    about a tenth of its time.  Returns a transposed view (the kernel produces
    dW^T)."""
    M, D_out = grad.shape
    M2, D_in = act_bf16.shape
    assert M == M2 and act_bf16.dtype == torch.bfloat16
    if grad.dtype == torch.bfloat16:
        # nothing to split: compute dW = grad^T @ act directly (grad is the transposed operand)
        out = torch.empty((D_out, D_in), device=grad.device, dtype=torch.float32)
        _C.check(_C.load().tcfp_bf16_dw_gemm(_C.ptr(grad.contiguous()), _C.ptr(act_bf16.contiguous()), None, _C.ptr(out),
                                             _C.F32, M, D_out, D_in, _C.stream()))
        return out
    g_lo = None
    if grad.dtype == torch.float32:
        g_hi, g_lo = split_bf16(grad)
    else:
        g_hi = grad.to(torch.bfloat16)
    out = torch.empty((D_in, D_out), device=grad.device, dtype=torch.float32)
    _C.check(_C.load().tcfp_bf16_dw_gemm(_C.ptr(act_bf16.contiguous()), _C.ptr(g_hi), _C.ptr(g_lo), _C.ptr(out),
                                         _C.F32, M, D_in, D_out, _C.stream()))
    return out.t()


# ---------------------------------------------------------------------------
# block quantizers (tcfp/kernels.py:1675-1875)
# ---------------------------------------------------------------------------

def _colsum_workspace(R: int, C: int, device) -> torch.Tensor:
    return torch.empty(_C.load().tcfp_colsum_workspace_bytes(R, C), dtype=torch.uint8, device=device)


def block_quantize_fp8(tensor, block_size=128, fp8_dtype=torch.float8_e4m3fn, *, want_bf16=False, want_colsum=False):
    """Per-block FP8 quantization (tcfp/kernels.py:1675-1722).  Returns
    ``(fp8 (M,K), int8 exponents (K // bs, M))``; with ``want_bf16`` a third
    tensor holds the dequantized values as bf16; with ``want_colsum`` a third
    tensor holds the FP32 column sums of the input (the bias gradient when the
    input is an output gradient), accumulated in the same pass."""
    M, K = tensor.shape
    assert K % block_size == 0, f"K ({K}) must be divisible by block_size ({block_size})"
    assert tensor.is_contiguous(), "input must be contiguous"
    num_kb = K // block_size
    out = torch.empty((M, K), device=tensor.device, dtype=fp8_dtype)
    scales = torch.empty((num_kb, M), device=tensor.device, dtype=torch.int8)
    sf = _alloc_sf(M, K, block_size, tensor.device)
    if want_colsum:
        assert not want_bf16, "want_colsum and want_bf16 are separate variants"
        colsum = torch.empty(K, device=tensor.device, dtype=torch.float32)
        _C.check(_C.load().tcfp_quantize_colsum(
            _C.ptr(tensor), _C.dtype_code(tensor), _C.ptr(out), _C.ptr(scales), _C.ptr(sf), M, K, block_size, _fmt(out),
            _C.ptr(colsum), _C.ptr(_colsum_workspace(M, K, tensor.device)), _C.stream()))
        _attach_sf(scales, sf, block_size)
        return out, scales, colsum
    deq = torch.empty((M, K), device=tensor.device, dtype=torch.bfloat16) if want_bf16 else None
    _C.check(_C.load().tcfp_quantize(
        _C.ptr(tensor), _C.dtype_code(tensor), _C.ptr(out), _C.ptr(scales), _C.ptr(sf), _C.ptr(deq),
        M, K, block_size, _fmt(out), None, None, 0, 0, 0, None, _C.stream()))
    _attach_sf(scales, sf, block_size)
    if want_bf16:
        return out, scales, deq
    return out, scales


def block_dequantize_fp8(fp8_tensor, block_scales, block_size):
    """``(M, K)`` FP32 from codes and int8 exponents (tcfp/kernels.py:1725-1746);
    torch ops, exactly as in the reference."""
    M, K = fp8_tensor.shape
    blocked = fp8_tensor.float().reshape(M, K // block_size, block_size)
    float_scales = torch.exp2(block_scales.float())
    return (blocked * float_scales.t().unsqueeze(-1)).reshape(M, K)


def block_dequantize_bf16(fp8_tensor, block_scales, block_size, *, sentinel_zero=False):
    """Codes + exponents -> bf16 values (exact: at most 4 significant bits)."""
    M, K = fp8_tensor.shape
    out = torch.empty((M, K), device=fp8_tensor.device, dtype=torch.bfloat16)
    _C.check(_C.load().tcfp_block_dequantize_bf16(
        _C.ptr(fp8_tensor), _C.ptr(block_scales), _C.ptr(out), M, K, block_size, _fmt(fp8_tensor),
        1 if sentinel_zero else 0, _C.stream()))
    return out


_srr_seed_gen: torch.Generator | None = None


def _fresh_seed() -> int:
    # one 31-bit seed per launch, drawn on the host (the reference draws it on
    # the device and synchronises to fetch it, tcfp/kernels.py:1828-1831)
    global _srr_seed_gen
    if _srr_seed_gen is None:
        _srr_seed_gen = torch.Generator(device="cpu")
        _srr_seed_gen.manual_seed(torch.initial_seed() & 0x7FFFFFFF)
    return int(torch.randint(0, 2**31, (1,), generator=_srr_seed_gen).item())


def fused_dual_quantize_fp8(weight, block_size=128, error_buf=None, stochastic_lo=False, *,
                            seed=None, offset=0, update_error=True):
    """W -> ``(w_hi, w_lo, scales_hi, scales_lo)`` in one kernel
    (tcfp/kernels.py:1749-1875).  ``error_buf`` is read and, unless
    ``update_error=False``, overwritten in place with
    ``W - deq(W_hi) - deq(W_lo)``."""
    assert weight.is_contiguous(), "Weight must be contiguous (N, K) row-major"
    N, K = weight.shape
    assert K % block_size == 0, f"K ({K}) must be divisible by block_size ({block_size})"
    if stochastic_lo and error_buf is not None:
        raise ValueError(
            "stochastic_lo and error_buf are mutually exclusive: "
            "SRR eliminates the need for error feedback buffers."
        )
    if error_buf is not None:
        assert error_buf.dtype == torch.float32, "error_buf must be float32"
        assert error_buf.shape == (N, K), f"error_buf shape {tuple(error_buf.shape)} != weight shape {(N, K)}"
        assert error_buf.is_contiguous(), "error_buf must be contiguous"
    num_kb = K // block_size
    dev = weight.device
    w_hi = torch.empty((N, K), device=dev, dtype=torch.float8_e4m3fn)
    w_lo = torch.empty((N, K), device=dev, dtype=torch.float8_e4m3fn)
    scales_hi = torch.empty((num_kb, N), device=dev, dtype=torch.int8)
    scales_lo = torch.empty((num_kb, N), device=dev, dtype=torch.int8)
    sf_hi = _alloc_sf(N, K, block_size, dev)
    sf_lo = _alloc_sf(N, K, block_size, dev)
    if stochastic_lo:
        mode = _C.Q_SRR
        if seed is None:
            seed = _fresh_seed()
    elif error_buf is not None:
        mode = _C.Q_EF if update_error else _C.Q_EF_READONLY
    else:
        mode = _C.Q_NONE
    _C.check(_C.load().tcfp_dual_quantize(
        _C.ptr(weight), _C.dtype_code(weight), _C.ptr(error_buf), _C.ptr(w_hi), _C.ptr(w_lo),
        _C.ptr(scales_hi), _C.ptr(scales_lo), _C.ptr(sf_hi), _C.ptr(sf_lo), N, K, block_size, mode,
        int(seed or 0), int(offset), None, None, None, None, _C.stream()))
    _attach_sf(scales_hi, sf_hi, block_size)
    _attach_sf(scales_lo, sf_lo, block_size)
    return w_hi, w_lo, scales_hi, scales_lo


# ---------------------------------------------------------------------------
# block-scaled GEMMs (tcfp/kernels.py:1878-2149, 2326-2469)
# ---------------------------------------------------------------------------

def fused_block_scaled_dual_gemm_forward(act_fp8, w_hi_fp8, w_lo_fp8, act_scales, w_hi_scales, w_lo_scales,
                                         block_size, sparse_threshold=0.0, persistent=True, launch_mult=1, *,
                                         bias=None, out_dtype=torch.float32, out=None, act_sf=None):
    """Block-scaled 2-GEMM forward (tcfp/kernels.py:1939-2028).  The tuning
    arguments of the reference are accepted and ignored: the kernel is always
    persistent with one CTA per SM.  ``act_sf`` passes the packed activation
    scale factors explicitly (a row slice of a larger operand's array);
    ``act_scales`` is then not consulted."""
    M, K = act_fp8.shape
    N, K2 = w_hi_fp8.shape
    assert K == K2 and (w_lo_fp8 is None or w_lo_fp8.shape == (N, K)), (
        f"Shape mismatch: act({M},{K}), w_hi({N},{K2})"
    )
    assert K % block_size == 0, f"K ({K}) must be divisible by block_size ({block_size})"
    sf_a = act_sf if act_sf is not None else pack_block_scales(act_scales, block_size)
    sf_hi = pack_block_scales(w_hi_scales, block_size)
    sf_lo = pack_block_scales(w_lo_scales, block_size) if w_lo_fp8 is not None else None
    if out is None:
        out = torch.empty((M, N), device=act_fp8.device, dtype=out_dtype)
    else:
        assert out.shape == (M, N) and out.dtype == out_dtype and out.is_contiguous(), "bad out buffer"
    _C.check(_C.load().tcfp_block_dual_gemm(
        _C.ptr(act_fp8), _C.ptr(sf_a), _C.ptr(w_hi_fp8), _C.ptr(sf_hi), _C.ptr(w_lo_fp8), _C.ptr(sf_lo),
        _C.ptr(bias), _C.ptr(out), _out_code(out_dtype), M, N, K, block_size, _C.stream()))
    return out


def block_scaled_gemm(a_fp8, b_fp8, scales_a, scales_b, block_size=128):
    """Single block-scaled GEMM (tcfp/kernels.py:1878-1936): the dual kernel
    with the residual operand left out."""
    M, K = a_fp8.shape
    N, K2 = b_fp8.shape
    assert K == K2, f"K mismatch: A ({K}) vs B ({K2})"
    assert K % block_size == 0, f"K ({K}) not divisible by block_size ({block_size})"
    return fused_block_scaled_dual_gemm_forward(a_fp8, b_fp8, None, scales_a, scales_b, None, block_size)


# Widest layer (output features) for which the prologue-fused kernel is dispatched by default.  Measured on a
# B200 at M = 32768, K = 4096, block 64: fused 166 / 270 / 392 / 402 us against 105 / 124 / 146 / 164 us for the
# block quantizer followed by the GEMM at N = 128 / 256 / 384 / 512 -- the converters re-quantize the activation
# tile for every 128-column tile and set the pace of the K loop -- so the separate route wins at every width and
# the default never fuses; ``fuse=True`` selects the fused kernel explicitly.
FUSED_ACT_MAX_N = 0


def fused_act_quant_dual_gemm_forward(act, w_hi_fp8, w_lo_fp8, w_hi_scales, w_lo_scales, block_size,
                                      sparse_threshold=0.0, persistent=True, launch_mult=1,
                                      save_side_outputs=True, *, bias=None, out_dtype=torch.float32, fuse=None):
    """Activation quantize + block-scaled 2-GEMM (tcfp/kernels.py:2031-2149).
    Returns ``(output, act_fp8, act_scales)``; the side outputs are ``None``
    when ``save_side_outputs`` is False.

    ``fuse=True`` runs ONE kernel that quantizes the bf16 activation tiles in
    the GEMM prologue (``tcfp_block_dual_gemm_fused_act``); ``fuse=False``
    runs the block quantizer and then the GEMM.  The default picks the fused
    kernel for bf16 activations and ``N <= FUSED_ACT_MAX_N`` (0: the two-kernel
    route measured faster at every width).  Both produce the same side-output
    bytes."""
    M, K = act.shape
    N, K2 = w_hi_fp8.shape
    assert K == K2 and w_lo_fp8.shape == (N, K), f"Shape mismatch: act({M},{K}), w_hi({N},{K2})"
    assert K % block_size == 0, f"K ({K}) must be divisible by block_size ({block_size})"
    fusable = act.dtype == torch.bfloat16 and act.is_contiguous()
    if fuse is None:
        fuse = fusable and N <= FUSED_ACT_MAX_N
    if fuse:
        assert fusable, "the fused kernel takes a contiguous bfloat16 activation"
        out = torch.empty((M, N), device=act.device, dtype=out_dtype)
        act_fp8 = act_scales = None
        if save_side_outputs:
            act_fp8 = torch.empty((M, K), device=act.device, dtype=torch.float8_e4m3fn)
            act_scales = torch.empty((K // block_size, M), device=act.device, dtype=torch.int8)
        # keep the packed scale arrays alive in locals until the launch is queued: a temporary freed between the
        # two pack launches would hand its block to the second one
        sf_hi = pack_block_scales(w_hi_scales, block_size)
        sf_lo = pack_block_scales(w_lo_scales, block_size)
        _C.check(_C.load().tcfp_block_dual_gemm_fused_act(
            _C.ptr(act), _C.ptr(w_hi_fp8), _C.ptr(sf_hi), _C.ptr(w_lo_fp8), _C.ptr(sf_lo), _C.ptr(bias), _C.ptr(out),
            _out_code(out_dtype), _C.ptr(act_fp8), _C.ptr(act_scales), M, N, K, block_size, _C.stream()))
        return out, act_fp8, act_scales
    act_fp8, act_scales = block_quantize_fp8(act, block_size, torch.float8_e4m3fn)
    out = fused_block_scaled_dual_gemm_forward(act_fp8, w_hi_fp8, w_lo_fp8, act_scales, w_hi_scales, w_lo_scales,
                                               block_size, bias=bias, out_dtype=out_dtype)
    if save_side_outputs:
        return out, act_fp8, act_scales
    return out, None, None


def block_retarget(w_hi_fp8, w_lo_fp8, w_hi_scales, w_lo_scales, block_size):
    """One launch of ``tcfp_block_retarget``: ``(hi_t, lo_t, t_hi, t_lo)`` with
    the codes transposed to ``(D_in, D_out)`` and int8 exponent planes
    ``(D_out // bs, D_in)``; ``lo`` entries ``None`` without ``w_lo_fp8``."""
    D_out, D_in = w_hi_fp8.shape
    assert w_hi_fp8.is_contiguous() and w_hi_scales.is_contiguous(), "operands must be contiguous"
    assert w_hi_scales.shape == (D_in // block_size, D_out), "scales must be (D_in // block_size, D_out)"
    dev = w_hi_fp8.device
    hi_t = torch.empty((D_in, D_out), device=dev, dtype=torch.float8_e4m3fn)
    t_hi = torch.empty((D_out // block_size, D_in), device=dev, dtype=torch.int8)
    lo_t = t_lo = None
    if w_lo_fp8 is not None:
        assert w_lo_fp8.is_contiguous() and w_lo_scales.is_contiguous(), "operands must be contiguous"
        lo_t = torch.empty((D_in, D_out), device=dev, dtype=torch.float8_e4m3fn)
        t_lo = torch.empty((D_out // block_size, D_in), device=dev, dtype=torch.int8)
    _C.check(_C.load().tcfp_block_retarget(
        _C.ptr(w_hi_fp8), _C.ptr(w_lo_fp8), _C.ptr(w_hi_scales), _C.ptr(w_lo_scales), _C.ptr(hi_t), _C.ptr(lo_t),
        _C.ptr(t_hi), _C.ptr(t_lo), D_out, D_in, block_size, _C.stream()))
    return hi_t, lo_t, t_hi, t_lo


def retarget_block_weights(w_hi_fp8, w_lo_fp8, w_hi_scales, w_lo_scales, block_size):
    """Quantized weight ``(D_out, D_in)`` with scales along ``D_in`` -> the
    operands of the input-gradient GEMM: codes transposed to ``(D_in, D_out)``
    and scale factors along ``D_out`` (``tcfp_block_retarget``).  Returns
    ``(hi_t, lo_t, sf_hi_t, sf_lo_t)`` (``lo`` entries ``None`` without
    ``w_lo_fp8``).  The result depends only on the quantized weight; it is
    kept on ``w_hi_fp8`` and reused while none of the four inputs changes, so
    gradient-accumulation micro-batches pay for it once."""
    D_out, D_in = w_hi_fp8.shape
    if any(t is not None and t.is_inference() for t in (w_hi_fp8, w_hi_scales, w_lo_fp8, w_lo_scales)):
        # no version counter tells of a change: nothing is kept
        hi_t, lo_t, t_hi, t_lo = block_retarget(w_hi_fp8, w_lo_fp8, w_hi_scales, w_lo_scales, block_size)
        return hi_t, lo_t, pack_block_scales(t_hi, block_size), None if t_lo is None else pack_block_scales(t_lo, block_size)
    key = (w_hi_fp8._version, w_hi_scales._version, w_hi_scales.data_ptr(), block_size,
           None if w_lo_fp8 is None else (w_lo_fp8.data_ptr(), w_lo_fp8._version, w_lo_scales._version))
    cached = getattr(w_hi_fp8, "_tcfp_dx", None)
    if cached is not None and cached[0] == key:
        return cached[1]
    hi_t, lo_t, t_hi, t_lo = block_retarget(w_hi_fp8, w_lo_fp8, w_hi_scales, w_lo_scales, block_size)
    out = (hi_t, lo_t, pack_block_scales(t_hi, block_size), None if t_lo is None else pack_block_scales(t_lo, block_size))
    w_hi_fp8._tcfp_dx = (key, out)
    return out


def fused_block_scaled_backward_dx(grad_fp8, w_hi_fp8, w_lo_fp8, grad_scales, w_hi_scales, w_lo_scales, block_size,
                                   persistent=True, launch_mult=1, *, out_dtype=torch.float32, exact_bf16=False,
                                   grad_bf16=None):
    """Block-scaled dX ``(M, D_in)`` (tcfp/kernels.py:2326-2425).  The weight
    scales run along ``D_in`` but dX contracts over ``D_out``: the quantized
    weight is re-targeted once per weight version (:func:`retarget_block_weights`)
    and the product runs on the FP8 block-scaled tensor-core path, like the
    forward.  ``exact_bf16=True`` takes the other route: every operand is
    dequantized to bf16 (exact) and multiplied on the bf16 tensor-core path at
    half the rate."""
    M, D_out = grad_fp8.shape
    D_out2, D_in = w_hi_fp8.shape
    assert D_out == D_out2 and (w_lo_fp8 is None or w_lo_fp8.shape == (D_out, D_in)), (
        f"Shape mismatch: grad({M},{D_out}), w_hi({D_out2},{D_in})"
    )
    assert D_out % block_size == 0, f"D_out={D_out} must be divisible by block_size={block_size}"
    assert D_in % block_size == 0, f"D_in={D_in} must be divisible by block_size={block_size}"
    out = torch.empty((M, D_in), device=grad_fp8.device, dtype=out_dtype)
    if exact_bf16:
        if grad_bf16 is None:
            grad_bf16 = block_dequantize_bf16(grad_fp8, grad_scales, block_size)
        hi = block_dequantize_bf16(w_hi_fp8, w_hi_scales, block_size)
        lo = None
        if w_lo_fp8 is not None:
            lo = block_dequantize_bf16(w_lo_fp8, w_lo_scales, block_size, sentinel_zero=True)
        _C.check(_C.load().tcfp_bf16_dual_gemm(
            _C.ptr(grad_bf16), _C.ptr(hi), _C.ptr(lo), None, _C.ptr(out), _out_code(out_dtype),
            M, D_in, D_out, 1, _C.stream()))
        return out
    assert grad_fp8.dtype == torch.float8_e5m2 and grad_fp8.is_contiguous(), "gradient codes must be contiguous E5M2"
    hi_t, lo_t, sf_hi_t, sf_lo_t = retarget_block_weights(w_hi_fp8, w_lo_fp8, w_hi_scales, w_lo_scales, block_size)
    sf_g = pack_block_scales(grad_scales, block_size)
    _C.check(_C.load().tcfp_block_dx_gemm(
        _C.ptr(grad_fp8), _C.ptr(sf_g), _C.ptr(hi_t), _C.ptr(sf_hi_t), _C.ptr(lo_t), _C.ptr(sf_lo_t), _C.ptr(out),
        _out_code(out_dtype), M, D_in, D_out, block_size, _C.stream()))
    return out


def fused_block_scaled_dual_gemm_backward_dx(grad_fp8, w_hi_fp8, w_lo_fp8, grad_scales, w_hi_scales, w_lo_scales,
                                             block_size):
    """Reference name of the dX dispatch (tcfp/kernels.py:2428-2469)."""
    return fused_block_scaled_backward_dx(grad_fp8, w_hi_fp8, w_lo_fp8, grad_scales, w_hi_scales, w_lo_scales,
                                          block_size=block_size)


# ---------------------------------------------------------------------------
# operators that end in 8 bits in front of a linear layer, and the int8 product
# (no counterpart in the reference, whose layer quantizes a stored 16-bit activation)
# ---------------------------------------------------------------------------

class QuantizedActivation:
    """An activation that exists in 8 bits only.

    ``codes`` is ``(rows, width)`` for an activation of ``shape``
    ``(..., width)``.  ``block_size`` 32/64/128: E4M3 codes and int8 exponent
    planes ``(width // block_size, rows)`` in ``scales``, what
    :func:`block_quantize_fp8` returns.  ``block_size`` ``None``: int8 codes
    and one float scale for each row; the rows start on 16-byte boundaries.
    ``bf16`` holds the values the codes stand for if they were asked for.
    ``dtype`` is the type of the tensor the activation was computed from.

    It is neither a tensor nor a pytree node: a full backward hook on a module
    that takes one is given ``None`` for it, and a wrapper that looks for tensors
    in a module's inputs or outputs does not see the path of its gradient."""

    def __init__(self, codes, scales, block_size, shape, dtype, bf16=None):
        self.codes, self.scales, self.block_size = codes, scales, block_size
        self.shape, self.dtype, self.bf16 = shape, dtype, bf16
        # stands for the activation in the autograd graph (see nn.add_rms_norm); its values are never read
        self._handle = None

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self) -> torch.Tensor:
        """The values the codes stand for, bf16, in ``shape``."""
        if self.bf16 is not None:
            return self.bf16.reshape(self.shape)
        if self.codes.numel() == 0:
            return torch.empty(self.shape, dtype=torch.bfloat16, device=self.device)
        if self.block_size is not None:
            with torch.cuda.device(self.device):
                return block_dequantize_bf16(self.codes, self.scales, self.block_size).reshape(self.shape)
        return (self.codes.float() * self.scales[:, None]).to(torch.bfloat16).reshape(self.shape)


def _rows_of(t: torch.Tensor, who: str, name: str) -> tuple[torch.Tensor, int]:
    """``(..., width)`` f32 or bf16 -> ``(rows, width)`` with unit column
    stride, and the row pitch in elements; a view where the strides allow."""
    if not t.is_cuda:
        raise RuntimeError(f"{who}: tcfp_b200 runs on CUDA (sm_100) tensors only, got a {t.device} {name}")
    _C.dtype_code(t)
    shape = t.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{who}: {name} needs a last dimension of at least 1, got shape {tuple(shape)}")
    if t.requires_grad:
        t = t.detach()
    if len(shape) != 2:
        t = t.reshape(math.prod(shape[:-1]), shape[-1])
    rows, width = t.shape
    ld, unit = t.stride()
    if unit != 1 and width > 1:
        t = t.contiguous()
        ld = width
    # the pitch of a single row is never used: give it one that does not stand in the way of wide accesses
    return t, ld if rows > 1 else -(-width // 16) * 16


def _same(t: torch.Tensor | None, like: torch.Tensor, who: str, name: str, like_name: str) -> None:
    if t is not None and (t.shape != like.shape or t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{who}: {name} ({tuple(t.shape)}, {t.dtype}, {t.device}) must match {like_name} "
                         f"({tuple(like.shape)}, {like.dtype}, {like.device})")


def _vector(t: torch.Tensor, n: int, device, who: str, name: str, dtypes=(torch.float32,)) -> torch.Tensor:
    if t.shape != (n,) or t.dtype not in dtypes or t.device != device:
        raise ValueError(f"{who}: {name} must be a ({n},) tensor of {' or '.join(str(d) for d in dtypes)} on {device}, got "
                         f"{tuple(t.shape)} {t.dtype} on {t.device}")
    if t.requires_grad:
        t = t.detach()
    return t.contiguous()


def _launch(device: torch.device, fn, *args) -> None:
    """Calls a C entry point on ``device``'s current stream."""
    if device.index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _C.stream())
    if rc != 0:
        _C.check(rc)


def _pitch16(t: torch.Tensor, ld: int) -> bool:
    return t.data_ptr() % 16 == 0 and (ld * t.element_size()) % 16 == 0


def _dense_like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, requires_grad=False) if t.is_contiguous() else t.new_empty(t.shape)


def _check_block(block_size, width: int, who: str) -> None:
    if block_size is None:
        return
    if block_size not in (32, 64, 128):
        raise ValueError(f"{who}: block_size must be 32, 64, 128 or None (int8, one scale for each row), got {block_size}")
    if width % block_size != 0:
        raise ValueError(f"{who}: width ({width}) must be divisible by block_size ({block_size})")


def _alloc_quantized(x: torch.Tensor, rows: int, width: int, block_size, want_bf16: bool, shape) -> tuple:
    """The outputs of a row quantizer: ``(QuantizedActivation, sf or None,
    row pitch of the codes)``."""
    dev = x.device
    # empty_strided is the cheapest allocation there is (1.5 us of host time; empty 2.4, a slice of a padded one 1.7 more)
    new = torch.empty_strided
    deq = new((rows, width), (width, 1), dtype=torch.bfloat16, device=dev) if want_bf16 else None
    if block_size is not None:
        codes = new((rows, width), (width, 1), dtype=torch.float8_e4m3fn, device=dev)
        scales = new((width // block_size, rows), (rows, 1), dtype=torch.int8, device=dev)
        sf = _alloc_sf(rows, width, block_size, dev)
        _attach_sf(scales, sf, block_size)
        pitch = width
    else:
        # the int8 product reads rows that start on 16-byte boundaries
        pitch = -(-width // 16) * 16
        codes = new((rows, width), (pitch, 1), dtype=torch.int8, device=dev)
        scales = new((rows,), (1,), dtype=torch.float32, device=dev)
        sf = None
    return QuantizedActivation(codes, scales, block_size, shape, x.dtype, deq), sf, pitch


def add_rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-5, *,
                          block_size: int | None = None, want_bf16: bool = False):
    """RMS norm with the residual's addition and an output in 8 bits, one
    pass: ``h = x + residual`` (rounded to ``x.dtype``), ``y = h *
    rsqrt(mean(h^2) + eps) * weight`` in FP32, quantized.  Returns
    ``(QuantizedActivation of y, h, rstd)`` with ``rstd`` ``(rows,)`` FP32;
    without a residual ``h`` is ``x``.  ``x`` is ``(..., width)`` FP32 or bf16
    with ``width <= 32768``, ``weight`` ``(width,)`` FP32 or bf16."""
    who = "add_rms_norm_quantize"
    x2d, ld_x = _rows_of(x, who, "x")
    _same(residual, x, who, "residual", "x")
    rows, width = x2d.shape
    _check_block(block_size, width, who)
    if width > 32768:
        raise ValueError(f"{who}: width ({width}) must be at most 32768")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"{who}: eps must be finite and not negative, got {eps}")
    w = _vector(weight, width, x.device, who, "weight", (torch.float32, torch.bfloat16))
    r2d, ld_r = (None, 0) if residual is None else _rows_of(residual, who, "residual")
    if block_size is not None:
        if not _pitch16(x2d, ld_x):
            x2d, ld_x = x2d.clone(memory_format=torch.contiguous_format), width
        if r2d is not None and not _pitch16(r2d, ld_r):
            r2d, ld_r = r2d.clone(memory_format=torch.contiguous_format), width
        if w.data_ptr() % 16:
            w = w.clone()
    q, sf, pitch = _alloc_quantized(x, rows, width, block_size, want_bf16, x.shape)
    h = None if residual is None else _dense_like(x)
    rstd = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=x.device)
    if rows > 0:
        _launch(x.device, _C.load().tcfp_add_rms_norm_quantize, x2d.data_ptr(), ld_x, _C.ptr(r2d), ld_r, _C.dtype_code(x2d),
                w.data_ptr(), _C.dtype_code(w), eps, _C.ptr(h), rstd.data_ptr(), q.codes.data_ptr(), pitch,
                q.scales.data_ptr(), _C.ptr(sf), _C.ptr(q.bf16), rows, width, block_size or 0)
    return q, x if h is None else h, rstd


def add_rms_norm_backward(grad: torch.Tensor, h: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor,
                          grad_h: torch.Tensor | None = None):
    """Gradients of :func:`add_rms_norm_quantize`, the rounding to 8 bits
    taken as the identity: ``grad`` is that of the normalised output,
    ``grad_h`` that of the stream ``h`` (``None``: zero).  Returns ``(dx,
    dw)``: ``dx`` (``h.dtype``, for ``x`` and the residual alike) and ``dw``
    ``(width,)`` FP32.  Repeated calls return identical bits."""
    who = "add_rms_norm_backward"
    h2d, ld_h = _rows_of(h, who, "h")
    _same(grad, h, who, "grad", "h")
    _same(grad_h, h, who, "grad_h", "h")
    rows, width = h2d.shape
    if width > 32768:
        raise ValueError(f"{who}: width ({width}) must be at most 32768")
    w = _vector(weight, width, h.device, who, "weight", (torch.float32, torch.bfloat16))
    rstd = _vector(rstd, rows, h.device, who, "rstd")
    if rows == 0:
        return torch.empty_like(h), torch.zeros(width, dtype=torch.float32, device=h.device)
    g2d, ld_g = _rows_of(grad, who, "grad")
    d2d, ld_d = (None, 0) if grad_h is None else _rows_of(grad_h, who, "grad_h")
    dx = _dense_like(h)
    dw = torch.empty_strided((width,), (1,), dtype=torch.float32, device=h.device)
    lib = _C.load()
    if h.device.index == torch._C._cuda_getDevice():      # the workspace goes by the device's number of SMs
        nbytes = lib.tcfp_rms_norm_backward_workspace_bytes(rows, width)
    else:
        with torch.cuda.device(h.device):
            nbytes = lib.tcfp_rms_norm_backward_workspace_bytes(rows, width)
    ws = h.new_empty(nbytes, dtype=torch.uint8)
    _launch(h.device, lib.tcfp_rms_norm_backward, g2d.data_ptr(), ld_g, h2d.data_ptr(), ld_h, rstd.data_ptr(), _C.dtype_code(h2d),
            w.data_ptr(), _C.dtype_code(w), _C.ptr(d2d), ld_d, dx.data_ptr(), dw.data_ptr(), ws.data_ptr(), rows, width)
    return dx, dw


def _gate_up(gate: torch.Tensor, up: torch.Tensor | None, who: str):
    """Gate and up as ``(rows, width, shape, gate address, pitch, up address,
    pitch, tensors that hold them)``: two tensors, or the halves of one packed
    ``(..., 2 * width)`` tensor."""
    if up is None:
        shape = gate.shape
        if not shape or shape[-1] % 2 != 0:
            raise ValueError(f"{who}: a packed gate_up needs an even last dimension, got shape {tuple(shape)}")
        both, ld = _rows_of(gate, who, "gate_up")
        rows, width = both.shape[0], shape[-1] // 2
        at = both.data_ptr()
        shape = shape[:-1] + (width,)
        out = rows, width, shape, at, ld, at + width * both.element_size(), ld, both
    else:
        _same(up, gate, who, "up", "gate")
        g2d, ld_g = _rows_of(gate, who, "gate")
        u2d, ld_u = _rows_of(up, who, "up")
        out = *g2d.shape, gate.shape, g2d.data_ptr(), ld_g, u2d.data_ptr(), ld_u, (g2d, u2d)
    if out[1] > _MAX_ROW:
        raise ValueError(f"{who}: width ({out[1]}) must be at most {_MAX_ROW}")
    return out


_MAX_ROW = 1 << 26


def silu_mul_quantize(gate: torch.Tensor, up: torch.Tensor | None = None, *, block_size: int | None = None,
                      want_bf16: bool = False) -> QuantizedActivation:
    """``silu(gate) * up`` in FP32, quantized, one pass.  ``up=None``: ``gate``
    is the packed ``(..., 2 * width)`` output of a fused gate/up projection."""
    who = "silu_mul_quantize"
    rows, width, shape, at_g, ld_g, at_u, ld_u, held = _gate_up(gate, up, who)
    _check_block(block_size, width, who)
    if block_size is not None:
        e = gate.element_size()
        if at_g % 16 or at_u % 16 or ld_g * e % 16 or ld_u * e % 16:
            g2d, u2d = held if up is not None else (held[:, :width], held[:, width:])
            held = g2d.clone(memory_format=torch.contiguous_format), u2d.clone(memory_format=torch.contiguous_format)
            at_g, at_u, ld_g, ld_u = held[0].data_ptr(), held[1].data_ptr(), width, width
    q, sf, pitch = _alloc_quantized(gate, rows, width, block_size, want_bf16, shape)
    if rows > 0:
        _launch(gate.device, _C.load().tcfp_silu_mul_quantize, at_g, ld_g, at_u, ld_u, _C.dtype_code(gate), q.codes.data_ptr(),
                pitch, q.scales.data_ptr(), _C.ptr(sf), _C.ptr(q.bf16), rows, width, block_size or 0)
    return q


def silu_mul_backward(grad: torch.Tensor, gate: torch.Tensor, up: torch.Tensor | None = None):
    """Gradients of :func:`silu_mul_quantize`, the rounding to 8 bits taken as
    the identity: ``(dgate, dup)``, or one packed tensor where ``gate`` is
    packed."""
    who = "silu_mul_backward"
    rows, width, shape, at_g, ld_g, at_u, ld_u, held = _gate_up(gate, up, who)
    if grad.shape != shape or grad.dtype != gate.dtype or grad.device != gate.device:
        raise ValueError(f"{who}: grad must be {tuple(shape)} {gate.dtype} on {gate.device}, got {tuple(grad.shape)} "
                         f"{grad.dtype} on {grad.device}")
    d2d, ld_d = _rows_of(grad, who, "grad")
    dg = _dense_like(gate)
    du = None if up is None else _dense_like(gate)
    if rows > 0:
        at = dg.data_ptr()
        ld = 2 * width if up is None else width
        _launch(gate.device, _C.load().tcfp_silu_mul_backward, d2d.data_ptr(), ld_d, at_g, ld_g, at_u, ld_u, _C.dtype_code(gate),
                at, ld, at + width * gate.element_size() if up is None else du.data_ptr(), ld, rows, width)
    return dg if up is None else (dg, du)


def int8_quantize_rows(x: torch.Tensor, *, want_bf16: bool = False) -> QuantizedActivation:
    """``(..., width)`` FP32 or bf16 -> int8 codes with one FP32 scale for each
    row, ``s = max(amax, 1e-12) / 127``, ``code = round(x * (1 / s))`` (FP32,
    ties to even): a token's scale for an activation, an output channel's for a weight
    ``(N, K)``."""
    who = "int8_quantize_rows"
    x2d, ld = _rows_of(x, who, "x")
    rows, width = x2d.shape
    if width > _MAX_ROW:
        raise ValueError(f"{who}: width ({width}) must be at most {_MAX_ROW}")
    q, _, pitch = _alloc_quantized(x, rows, width, None, want_bf16, x.shape)
    if rows > 0:
        _launch(x.device, _C.load().tcfp_int8_quantize_rows, x2d.data_ptr(), ld, _C.dtype_code(x2d), q.codes.data_ptr(), pitch,
                q.scales.data_ptr(), _C.ptr(q.bf16), rows, width)
    return q


def _int8_operand(t: torch.Tensor, who: str, name: str) -> tuple[torch.Tensor, int]:
    if not t.is_cuda:
        raise RuntimeError(f"{who}: tcfp_b200 runs on CUDA (sm_100) tensors only, got a {t.device} {name}")
    if t.dtype != torch.int8 or t.ndim != 2:
        raise TypeError(f"{who}: {name} must be a 2-D int8 tensor, got {t.ndim}-D {t.dtype}")
    rows, width = t.shape
    ld, unit = t.stride()
    pitch = -(-width // 16) * 16
    if t.data_ptr() % 16 or (unit != 1 and width > 1) or (rows > 1 and (ld % 16 or ld < width)):
        held = t.new_empty((rows, pitch))[:, :width]
        held.copy_(t)
        return held, pitch
    return t, ld if rows > 1 else pitch


def int8_matmul(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``(a @ b.T) * a_scale[:, None] * b_scale + bias`` -> ``(M, N)`` for int8
    ``a (M, K)`` and ``b (N, K)`` with one FP32 scale for each row of either.
    The integer sum is exact (``K <= 131071``); the scales and the bias are
    applied in FP32 and the result is rounded once.  Operands whose rows do
    not start on 16-byte boundaries are copied to such rows first
    (:func:`int8_quantize_rows` lays its codes out that way)."""
    who = "int8_matmul"
    code = _out_code(out_dtype)
    a, ld_a = _int8_operand(a, who, "a")
    b, ld_b = _int8_operand(b, who, "b")
    (M, K), (N, K2) = a.shape, b.shape
    if K != K2 or a.device != b.device:
        raise ValueError(f"{who}: a ({M}, {K}) on {a.device} and b ({N}, {K2}) on {b.device} do not fit")
    if not 1 <= K <= 131071 or N < 1:
        raise ValueError(f"{who}: K ({K}) must be in [1, 131071] and N ({N}) at least 1")
    a_scale = _vector(a_scale, M, a.device, who, "a_scale")
    b_scale = _vector(b_scale, N, a.device, who, "b_scale")
    if bias is not None:
        bias = _vector(bias, N, a.device, who, "bias", (torch.float32, torch.bfloat16)).float()
    out = torch.empty_strided((M, N), (N, 1), dtype=out_dtype, device=a.device)
    if M > 0:
        _launch(a.device, _C.load().tcfp_int8_gemm, a.data_ptr(), ld_a, a_scale.data_ptr(), b.data_ptr(), ld_b,
                b_scale.data_ptr(), _C.ptr(bias), out.data_ptr(), code, M, N, K)
    return out
