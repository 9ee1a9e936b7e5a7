"""CPU: a column-parallel layer around an inner layer that is no TCFPLinear hands a QuantizedActivation on: one rank, and two
over gloo.  The inner layer is a stand-in that multiplies the tensor behind the activation's gradient."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from tests.test_tp_gloo import _free_port


class TakesCodes(torch.nn.Module):
    def __init__(self, i, o):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.randn(o, i))

    def forward(self, q):
        from tcfp_b200.kernels import QuantizedActivation

        assert isinstance(q, QuantizedActivation)
        return (q.codes.float() if q._handle is None else q._handle) @ self.weight.t()


def activation(x):
    from tcfp_b200.kernels import QuantizedActivation

    q = QuantizedActivation(torch.zeros(x.shape, dtype=torch.int8), torch.ones(x.shape[0]), None, x.shape, x.dtype)
    q._handle = x
    return q


def build(**kw):
    from tcfp_b200.tp import ColumnParallelLinear

    torch.manual_seed(0)
    return ColumnParallelLinear(8, (32, 16), granule=16, layer_factory=lambda i, o, b, **k: TakesCodes(i, o), **kw)


@pytest.mark.parametrize("sequence_parallel", [False, True])
def test_one_rank(sequence_parallel):
    layer = build(sequence_parallel=sequence_parallel)
    x = torch.randn(3, 8, requires_grad=True)
    q = activation(x)
    parts = layer(q)
    assert [p.shape for p in parts] == [(3, 32), (3, 16)] and torch.equal(torch.cat(parts, 1), x @ layer.inner.weight.t())
    layer(q, packed=True).sum().backward()
    # sums of 48 FP32 numbers in two orders: 47 roundings of 2^-24 of the magnitudes in either
    w = layer.inner.weight.detach().double()
    assert ((x.grad.double() - w.sum(0)).abs() <= 48 * 2.0**-24 * w.abs().sum(0)).all() and q._handle is x
    q._handle = None
    assert layer(q, packed=True).shape == (3, 48)


def _worker(rank, world, port, ret):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from tcfp_b200.tp import ColumnParallelLinear

        torch.manual_seed(0)
        layer = ColumnParallelLinear(8, 32, granule=16, layer_factory=lambda i, o, b, **k: TakesCodes(i, o))
        with torch.no_grad():
            layer.inner.weight.copy_(torch.arange(16 * 8).reshape(16, 8) * (rank + 1))
        x = torch.ones(3, 8, requires_grad=True)
        q = activation(x)
        layer(q).sum().backward()
        # integers: the sum over the ranks is exact
        ok = torch.equal(x.grad, 3 * torch.arange(16 * 8).reshape(16, 8).sum(0).float().expand(3, 8))
        try:
            ColumnParallelLinear(8, 32, granule=16, sequence_parallel=True, layer_factory=lambda i, o, b, **k: TakesCodes(i, o))(q)
            ok = False
        except TypeError as e:
            ok &= "TCFPLinear" in str(e)
        ret[rank] = ok
    finally:
        dist.destroy_process_group()


def test_two_ranks():
    with mp.Manager() as manager:
        ret = manager.dict()
        mp.spawn(_worker, args=(2, _free_port(), ret), nprocs=2, join=True)
        assert dict(ret) == {0: True, 1: True}
