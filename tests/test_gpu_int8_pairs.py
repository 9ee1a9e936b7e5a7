"""GPU: the int8 product on CTA pairs with one group of epilogue warps (K from 2048 on), against its definition in 64 bits.

The epilogue stages its output in two pieces taken in turn; a piece that lies outside the output is not stored, and the next
rewrite of the buffers has to wait for the right store all the same.  So the sizes end a tile after every number of pieces
(64 columns of bf16, 32 of FP32), in the lower half of a tile's 256 rows and in the upper one, with several tiles a pair.
"""
import pytest
import torch

from tests.test_gpu_operators import DTYPES, check_product, codes
from tests.util import gen

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:DEBUG")]
DEV = "cuda"


def kernels_of(call, tmp_path):
    """The text of a graph of what `call` launches: the kernels' names are in it."""
    g = torch.cuda.CUDAGraph(keep_graph=True)
    g.enable_debug_mode()
    with torch.cuda.graph(g):
        call()
    path = tmp_path / "graph.dot"
    g.debug_dump(str(path))
    return path.read_text()


def check(m, n, k, dtype, tmp_path, groups=1):
    from tcfp_b200.kernels import int8_matmul

    g = gen(m + n + k)
    sa, sb = (torch.rand(m, generator=g) + 0.01).to(DEV), (torch.rand(n, generator=g) * 1e-3 + 1e-5).to(DEV)
    bias = torch.randn(n, generator=g).to(DEV)
    a, b = codes(1 + m, m, k), codes(2 + n, n, k)
    # a changed choice between the kernels must not take these sizes away from the one they test
    text = kernels_of(lambda: int8_matmul(a, b, sa, sb, out_dtype=dtype), tmp_path)
    assert f"int8_pair_kernelILb{int(dtype == torch.bfloat16)}ELi{groups}E" in text, text
    out = check_product(a, b, sa, sb, None, dtype)
    for _ in range(3):
        assert torch.equal(check_product(a, b, sa, sb, None, dtype), out)
    check_product(a, b, sa, sb, bias, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [2560 + r for r in (0, 8, 32, 64, 72, 96, 128, 136, 160, 192, 200, 224)])
@pytest.mark.parametrize("m", [2048, 2049, 2148, 2176, 2248])
def test_every_end_of_a_tile(m, n, dtype, tmp_path):
    check(m, n, 2048, dtype, tmp_path)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(2100, 2561, 2048), (2305, 2729, 2500), (2048, 2564, 2049)])
def test_rows_off_16_byte_boundaries(m, n, k, dtype, tmp_path):
    check(m, n, k, dtype, tmp_path)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(256, 9600, 2048), (200, 9640, 4096), (4196, 4168, 4097), (8192, 1032, 2304), (1030, 8288, 11008)])
def test_one_and_many_tiles_a_pair(m, n, k, dtype, tmp_path):
    check(m, n, k, dtype, tmp_path)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shorter_rows_have_two_groups(dtype, tmp_path):
    for m, n, k in ((2148, 2632, 2047), (2176, 2560, 100), (2049, 2573, 640)):
        check(m, n, k, dtype, tmp_path, groups=2)


def test_extreme_sums():
    """The largest sum there is, 131071 products of -128 * -128, is below 2^31 and comes out exact."""
    k = 131071
    a = torch.full((2200, k), -128, dtype=torch.int8, device=DEV)
    b = torch.full((2312, k), -128, dtype=torch.int8, device=DEV)
    b[1] = 127
    out = check_product(a, b, torch.ones(2200, device=DEV), torch.ones(2312, device=DEV), None, torch.float32)
    assert (out[:, 0].double() == float(torch.tensor(16384.0 * k, dtype=torch.float32))).all()
