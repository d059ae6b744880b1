"""Host logic of the operators around the projections at the edges of what their
documentation allows; no GPU."""

import pytest
import torch

from sglite_b200 import ops


def _gate_as_kernel_reads(gate, x, n):
    """[rows, n] of what the kernel reads at gate[m * row + c * col], or None where an
    element would lie outside the gate's own memory."""
    row, col = ops._gate_strides(gate, x, n)
    at = torch.arange(x.numel() // n)[:, None] * row + torch.arange(n) * col
    held = gate.storage_offset() + at
    if int(held.max()) >= gate.untyped_storage().nbytes() // gate.element_size():
        return None
    return torch.as_strided(gate, (gate.untyped_storage().nbytes() // gate.element_size(),), (1,), 0)[held]


@pytest.mark.parametrize("make", [
    lambda: torch.randn(1, 4, 64).transpose(0, 1),             # [4, 1, 64]: the middle stride is arbitrary
    lambda: torch.randn(1, 4, 1).transpose(0, 1),              # [4, 1, 1]
    lambda: torch.randn(4, 64).as_strided((4, 1, 64), (64, 7, 1)),
    lambda: torch.randn(4, 1).as_strided((4, 1, 1), (1, 5, 9)),
    lambda: torch.randn(4, 1, 64), lambda: torch.randn(4, 1, 1), lambda: torch.randn(64),
    lambda: torch.randn(1, 1, 64), lambda: torch.randn(1, 64), lambda: torch.randn(1), lambda: torch.tensor(0.5)])
def test_gate_of_three_dimensions_is_read_where_it_stands(make):
    gate, x = make(), torch.zeros(4, 1, 64)
    got = _gate_as_kernel_reads(gate, x, 64)
    assert got is not None
    assert torch.equal(got, gate.expand(x.shape).reshape(4, 64))


@pytest.mark.parametrize("make", [
    lambda: torch.randn(2, 3, 64), lambda: torch.randn(2, 3, 1), lambda: torch.randn(6, 128)[:, 64:].unflatten(0, (2, 3)).contiguous()])
def test_gate_rows_over_two_batch_dimensions(make):
    gate, x = make(), torch.zeros(2, 3, 64)
    assert torch.equal(_gate_as_kernel_reads(gate, x, 64), gate.expand(x.shape).reshape(6, 64))


@pytest.mark.parametrize("make", [
    lambda: torch.randn(6, 128)[:, 64:], lambda: torch.randn(6, 5)[:, 2:3], lambda: torch.randn(64).expand(6, 64),
    lambda: torch.randn(1, 1).expand(6, 1)])
def test_gate_of_two_dimensions_keeps_its_row_stride(make):
    gate, x = make(), torch.zeros(6, 64)
    assert torch.equal(_gate_as_kernel_reads(gate, x, 64), gate.expand(x.shape))


def test_gates_that_do_not_broadcast_are_refused():
    x = torch.zeros(4, 1, 64)
    for gate in (torch.zeros(4, 64), torch.zeros(4), torch.zeros(3, 1, 64), torch.zeros(4, 2, 64), torch.zeros(4, 1, 2),
                 torch.zeros(64, 4, 1).permute(1, 2, 0), torch.zeros(2, 64).expand(4, 2, 64)):
        with pytest.raises(ValueError):
            ops._gate_strides(gate, x, 64)
