"""CPU: what the operators in front of a linear layer and the int8 product
refuse, in Python and at the C entry points (no launch is reached)."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from tcfp_b200 import _C, build

    build.build()
    return _C.load()


def refused(lib, rc, code, text):
    from tcfp_b200 import _C

    assert rc == code and text in _C.last_error(), (rc, _C.last_error())


def test_norm_entry_point_refusals(lib):
    f = lib.tcfp_add_rms_norm_quantize
    ok = dict(x=4096, ld=64, r=None, ld_r=0, dt=0, w=4096, wdt=0, eps=1e-5, h=None, rstd=None, codes=4096, ldc=64, scale=4096,
              sf=None, deq=None, rows=4, width=64, bs=0)

    def call(**kw):
        a = dict(ok, **kw)
        return f(a["x"], a["ld"], a["r"], a["ld_r"], a["dt"], a["w"], a["wdt"], a["eps"], a["h"], a["rstd"], a["codes"], a["ldc"],
                 a["scale"], a["sf"], a["deq"], a["rows"], a["width"], a["bs"], None)

    for kw in (dict(x=None), dict(w=None), dict(codes=None), dict(scale=None)):
        refused(lib, call(**kw), -1, "NULL")
    refused(lib, call(dt=2), -1, "dtype")
    refused(lib, call(wdt=7), -1, "dtype")
    refused(lib, call(rows=0), -1, "rows")
    refused(lib, call(rows=1 << 31), -1, "rows")
    refused(lib, call(width=0), -1, "width")
    refused(lib, call(width=32769, ld=32769, ldc=32769), -2, "width")
    refused(lib, call(r=4096, ld_r=64), -1, "h_out")
    refused(lib, call(ldc=63), -1, "ld_codes")
    refused(lib, call(bs=16), -1, "block_size")
    refused(lib, call(bs=128), -1, "multiple")
    refused(lib, call(bs=32, ldc=80), -1, "dense")
    refused(lib, call(bs=32, x=4100), -1, "aligned")
    refused(lib, call(bs=32, ld=65), -1, "aligned")
    refused(lib, call(sf=4096), -1, "sf_out")


def test_gate_and_row_entry_point_refusals(lib):
    gate = lib.tcfp_silu_mul_quantize
    refused(lib, gate(4096, 64, None, 64, 0, 4096, 64, 4096, None, None, 4, 64, 0, None), -1, "NULL")
    refused(lib, gate(4096, 64, 4096, 64, 0, 4096, 64, 4096, None, None, 4, 1 << 27, 0, None), -2, "width")
    refused(lib, gate(4096, 64, 4100, 64, 0, 4096, 64, 4096, None, None, 4, 64, 32, None), -1, "aligned")
    rows = lib.tcfp_int8_quantize_rows
    refused(lib, rows(4096, 64, 3, 4096, 64, 4096, None, 4, 64, None), -1, "dtype")
    refused(lib, rows(4096, 64, 0, 4096, 32, 4096, None, 4, 64, None), -1, "ld_codes")
    back = lib.tcfp_silu_mul_backward
    refused(lib, back(4096, 64, 4096, 64, None, 64, 0, 4096, 64, 4096, 64, 4, 64, None), -1, "NULL")
    refused(lib, back(4096, 64, 4096, 64, 4096, 64, 0, 4096, 64, 4096, 64, 0, 64, None), -1, "rows")
    norm = lib.tcfp_rms_norm_backward
    refused(lib, norm(4096, 64, 4096, 64, 4096, 0, 4096, 0, None, 0, 4096, 4096, None, 4, 64, None), -1, "NULL")
    refused(lib, norm(4096, 64, 4096, 64, 4096, 0, 4096, 0, None, 0, 4096, 4096, 4096, 4, 40000, None), -2, "width")
    assert lib.tcfp_rms_norm_backward_workspace_bytes(0, 64) == 0
    assert lib.tcfp_rms_norm_backward_workspace_bytes(3, 64) >= 64 * 4          # at least one row of partial sums


def test_product_entry_point_refusals(lib):
    f = lib.tcfp_int8_gemm
    ok = dict(a=4096, lda=64, sa=4096, b=4096, ldb=64, sb=4096, bias=None, out=4096, dt=0, M=4, N=4, K=64)

    def call(**kw):
        a = dict(ok, **kw)
        return f(a["a"], a["lda"], a["sa"], a["b"], a["ldb"], a["sb"], a["bias"], a["out"], a["dt"], a["M"], a["N"], a["K"], None)

    for name in ("a", "sa", "b", "sb", "out"):
        refused(lib, call(**{name: None}), -1, "NULL")
    refused(lib, call(dt=5), -1, "dtype")
    for name in ("M", "N", "K"):
        refused(lib, call(**{name: 0}), -1, "M ")
    refused(lib, call(K=131072, lda=131072, ldb=131072), -2, "overflow")
    for kw in (dict(lda=72), dict(ldb=48), dict(a=4104), dict(b=4097)):
        refused(lib, call(**kw), -1, "16-byte")


def test_python_refusals():
    from tcfp_b200 import kernels as K

    x = torch.zeros(2, 64)
    for f in (lambda: K.add_rms_norm_quantize(x, torch.ones(64)), lambda: K.silu_mul_quantize(x), lambda: K.int8_quantize_rows(x),
              lambda: K.int8_matmul(x.to(torch.int8), x.to(torch.int8), torch.ones(2), torch.ones(2)),
              lambda: K.add_rms_norm_backward(x, x, torch.ones(2), torch.ones(64)), lambda: K.silu_mul_backward(x[:, :32], x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    with pytest.raises(ValueError, match="even"):
        K.silu_mul_quantize(torch.zeros(2, 7))
    with pytest.raises(ValueError, match="must match"):
        K.silu_mul_quantize(x, torch.zeros(2, 32))
    with pytest.raises(TypeError, match="out_dtype"):
        K.int8_matmul(x.to(torch.int8), x.to(torch.int8), torch.ones(2), torch.ones(2), out_dtype=torch.float16)


def test_module_refusals():
    from tcfp_b200.nn import Int8Linear, QuantizedRMSNorm, convert_to_int8

    for kw in (dict(d=96, scale_block_size=64), dict(d=128, scale_block_size=48)):
        with pytest.raises(ValueError, match="scale_block_size"):
            QuantizedRMSNorm(**kw)
    with pytest.raises(ValueError, match="out_dtype"):
        Int8Linear(16, 16, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="131071"):
        Int8Linear(131072, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        convert_to_int8(torch.nn.Sequential(torch.nn.Linear(16, 16)))
    layer = Int8Linear(30, 5)
    assert layer.weight_codes.shape == (5, 32) and set(layer.state_dict()) == {"weight_codes", "weight_scale", "bias"}
    assert layer.to(torch.bfloat16).weight_scale.dtype == torch.float32 and layer.bias.dtype == torch.float32
    assert Int8Linear(16, 16, bias=False).to(torch.float64).weight_scale.dtype == torch.float32


def test_column_parallel_parts_and_packed_output():
    from tcfp_b200.tp import ColumnParallelLinear

    layer = ColumnParallelLinear(8, (32, 16), layer_factory=lambda i, o, b, **kw: torch.nn.Linear(i, o, b))
    x = torch.randn(3, 8)
    parts, packed = layer(x), layer(x, packed=True)
    assert [p.shape[-1] for p in parts] == [32, 16] and torch.equal(torch.cat(parts, dim=-1), packed)
