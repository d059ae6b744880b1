"""Which path the tensor-parallel layers take for batches with and without adapters;
no GPU: the projection, the exchange and the communicator are stand-ins."""

import pytest
import torch

from sglite_b200.tp import ColumnParallelAWQLinear, RowParallelAWQLinear


class _Method:
    def __init__(self):
        self.calls = []

    def create_weights(self, k, n):
        return {"qweight": torch.zeros(1), "_act_dtype": torch.bfloat16, "_group_size": 128}

    def apply_weights(self, weights, x, bias=None, out=None, adapters=None, batch=None):
        self.calls.append((adapters, batch))
        return torch.full((x.shape[0], 8), 1.0 if adapters is None else 2.0)


class _Exchange:
    max_rows, max_n = 64, 1024

    def gemm_allreduce(self, x, blob, k, n, G):
        return torch.full((x.shape[0], n), 10.0)


class _Comm:
    def all_reduce(self, y):
        return y * 100


X = torch.zeros((3, 16), dtype=torch.bfloat16)


def test_a_layer_without_adapters_takes_the_steps_batch():
    """One batch serves every projection of a step; where a projection has no adapters
    no row uses one, and the output is the projection's own."""
    batch = object()
    col = ColumnParallelAWQLinear(_Method(), 16, 8)
    assert torch.equal(col.forward(X, batch), col.forward(X)) and col.method.calls == [(None, None)] * 2
    row = RowParallelAWQLinear(_Method(), 32, 8, 2, _Comm(), exchange=_Exchange())
    assert torch.equal(row.forward(X, batch), torch.full((3, 8), 10.0)) and not row.method.calls  # still fused
    row = RowParallelAWQLinear(_Method(), 32, 8, 2, _Comm())
    assert torch.equal(row.forward(X, batch), torch.full((3, 8), 100.0))


def test_a_layer_with_adapters_uses_them_before_the_all_reduce():
    batch, adapters = object(), object()
    for layer, want in ((ColumnParallelAWQLinear(_Method(), 16, 8), 2.0),
                        (RowParallelAWQLinear(_Method(), 16, 8, 1), 2.0),
                        (RowParallelAWQLinear(_Method(), 32, 8, 2, _Comm(), exchange=_Exchange()), 200.0)):
        layer.adapters = adapters
        assert torch.equal(layer.forward(X, batch), torch.full((3, 8), want))
        assert layer.method.calls == [(adapters, batch)]
    assert torch.equal(layer.forward(X), torch.full((3, 8), 10.0))  # a batch without adapters


def test_rows_that_need_the_communicator_say_so_before_any_work():
    """An exchange alone serves batches without adapters and bias up to its size."""
    row = RowParallelAWQLinear(_Method(), 32, 8, 2, exchange=_Exchange())
    assert torch.equal(row.forward(X), torch.full((3, 8), 10.0))
    row.adapters = object()
    for x, lora in ((X, object()), (torch.zeros((65, 16), dtype=torch.bfloat16), None)):
        with pytest.raises(ValueError, match="comm"):
            row.forward(x, lora)
    assert not row.method.calls
