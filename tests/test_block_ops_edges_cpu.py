"""Host logic of the operators around the projections at the edges of what their
documentation allows; no GPU."""

import contextlib
import ctypes

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


@pytest.mark.parametrize("ids", [
    torch.zeros((3, 8), dtype=torch.int32)[:, :2], torch.zeros((1, 2), dtype=torch.int32).expand(3, 2),
    torch.zeros((3, 1), dtype=torch.int32).expand(3, 2), torch.zeros((2, 3), dtype=torch.int32).T])
def test_topk_sum_reads_ids_by_their_rows(monkeypatch, ids):
    """The kernel reads M * topk ids one after the other: what it gets has to hold them."""
    seen = {}

    def record(name, *args):
        ptr, n = args[4].value, ids.numel()
        seen["ids"] = torch.frombuffer((ctypes.c_int32 * n).from_address(ptr), dtype=torch.int32).clone().view(ids.shape)

    ids = ids.clone() if ids.is_contiguous() else ids
    if ids.untyped_storage().nbytes() >= 4 * ids.numel():
        ids.copy_(torch.arange(ids.numel()).view(ids.shape))
    monkeypatch.setattr(ops, "call", record)
    monkeypatch.setattr(ops, "_check_cuda", lambda *ts: ts[0].device)
    monkeypatch.setattr(ops, "_DeviceGuard", contextlib.nullcontext)
    monkeypatch.setattr(ops, "_stream", lambda dev: None)
    y3, out = torch.zeros((6, 8), dtype=torch.bfloat16), torch.zeros((3, 8), dtype=torch.bfloat16)
    try:
        ops.moe_topk_sum(y3, 3, 2, ids, 0, 4, out)
    except ValueError:
        return  # refusing the layout is right as well
    assert torch.equal(seen["ids"], ids)


@pytest.mark.parametrize("ids", [torch.zeros((3, 2), dtype=torch.int64), torch.zeros((3, 1), dtype=torch.int32),
                                 torch.zeros((2, 2), dtype=torch.int32)])
def test_topk_sum_refuses_other_ids(monkeypatch, ids):
    monkeypatch.setattr(ops, "call", lambda *a: pytest.fail("reached the kernel"))
    monkeypatch.setattr(ops, "_check_cuda", lambda *ts: ts[0].device)
    y3, out = torch.zeros((6, 8), dtype=torch.bfloat16), torch.zeros((3, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.moe_topk_sum(y3, 3, 2, ids, 0, 4, out)
