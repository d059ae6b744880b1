"""Host logic of the operators around the projections at the edges of what their
documentation allows; no GPU."""

import contextlib
import ctypes
import math
import os
import struct
import subprocess

import pytest
import torch

from sglite_b200 import _lib, ops
from sglite_b200.moe import AWQB200MoeBackend, AWQExpertWeights, DenseExpertWeights
from sglite_b200.rotary import RotaryEmbedding, rotary_frequencies


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


LONG = {"rope_type": "longrope", "short_factor": [1.0, 1.5, 2.0, 2.5], "long_factor": [4.0, 8.0, 16.0, 32.0], "factor": 32.0,
        "original_max_position_embeddings": 4096}


def test_longrope_with_two_lists_needs_the_length_it_is_for():
    """A checkpoint's entry with both lists: the short one up to the original length,
    the long one beyond, and no guess."""
    plain = rotary_frequencies(8, 1e4)[0]
    with pytest.raises(ValueError, match="max_length"):
        rotary_frequencies(8, 1e4, LONG)
    with pytest.raises(ValueError, match="max_length"):
        RotaryEmbedding(2, 1, 8, scaling=LONG)
    for length, key in ((1, "short_factor"), (4096, "short_factor"), (4097, "long_factor"), (131072, "long_factor")):
        inv, f = rotary_frequencies(8, 1e4, LONG, max_length=length)
        assert torch.allclose(inv, plain / torch.tensor(LONG[key], dtype=torch.float64), rtol=1e-15)
        assert math.isclose(f, math.sqrt(1 + math.log(32) / math.log(4096)))  # of the model, not of the length
        layer = RotaryEmbedding(2, 1, 8, scaling=LONG, max_length=length)
        assert torch.equal(layer.inv_freq(torch.device("cpu")), inv) and layer.scale == f
    with pytest.raises(ValueError):
        rotary_frequencies(8, 1e4, {**LONG, "original_max_position_embeddings": None, "attention_factor": 1.0},
                           max_length=100)
    with pytest.raises(ValueError):  # the list that applies has another length
        rotary_frequencies(8, 1e4, {**LONG, "short_factor": [1.0]}, max_length=100)


def test_longrope_without_a_choice_to_make():
    plain = rotary_frequencies(8, 1e4)[0]
    long = plain / torch.tensor(LONG["long_factor"], dtype=torch.float64)
    one = {k: v for k, v in LONG.items() if k != "short_factor"}
    for entry, length in ((one, None), (one, 100), ({**LONG, "short_factor": LONG["long_factor"]}, None)):
        assert torch.allclose(rotary_frequencies(8, 1e4, entry, max_length=length)[0], long, rtol=1e-15)
    named = {**LONG, "factors": LONG["short_factor"]}  # said outright
    assert torch.allclose(rotary_frequencies(8, 1e4, named)[0], plain / torch.tensor(LONG["short_factor"], dtype=torch.float64))
    short = {k: v for k, v in LONG.items() if k != "long_factor"}
    with pytest.raises(ValueError):  # nothing for lengths beyond the original one
        rotary_frequencies(8, 1e4, short)
    with pytest.raises(ValueError):
        rotary_frequencies(8, 1e4, short, max_length=5000)
    assert torch.allclose(rotary_frequencies(8, 1e4, short, max_length=4096)[0],
                          plain / torch.tensor(LONG["short_factor"], dtype=torch.float64))


def test_what_lora_keeps_between_calls_is_bounded(monkeypatch):
    """Prompts come with any number of rows: nothing may be kept for each of them."""
    monkeypatch.setattr(ops, "_device_of", lambda t: -1)  # the other tensors' device here
    monkeypatch.setattr(ops, "_run", lambda *a: None)
    monkeypatch.setattr(ops, "_LORA_BYTES", {}, raising=False)
    a, b = torch.zeros((2, 8, 16), dtype=torch.bfloat16), torch.zeros((2, 8, 8), dtype=torch.bfloat16)
    offsets = torch.zeros(3, dtype=torch.int32)
    for M in range(1, 3001):
        x, base = torch.empty((M, 16), dtype=torch.bfloat16), torch.empty((M, 8), dtype=torch.bfloat16)
        ops.lora(x, a, b, torch.empty(M, dtype=torch.int32), offsets, base)
    kept = sum(len(v) for v in vars(ops).values() if isinstance(v, dict) and v is not vars(ops).get("__builtins__"))
    kept += sum(v.cache_info().currsize for v in vars(ops).values() if hasattr(v, "cache_info"))
    assert kept < 1500


def test_packed_structures_have_the_size_that_c_reads(tmp_path):
    """Field offsets and sizes as a C compiler lays the structures out."""
    names = {"awqb_gated_add_rmsnorm": ("awqb_gated_norm_args", "dtype"), "awqb_rotary": ("awqb_rotary_args", "dtype"),
             "awqb_grouped_gemm": ("awqb_grouped_gemm_args", "ldo"), "awqb_lora": ("awqb_lora_args", "workspace_bytes")}
    assert set(names) == set(_lib.ARGS)
    lines = [f'printf("{k} %zu %zu\\n", sizeof({t}), offsetof({t}, {last}));' for k, (t, last) in names.items()]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "awqb200.h"\nint main(void) {\n' + "\n".join(lines)
                   + "\nreturn 0;\n}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "sizes")], check=True)
    for line in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size, last = line.split()
        form = _lib.ARGS[name].format
        fields = form.removesuffix("0q")
        assert _lib.ARGS[name].size == int(size), name
        assert struct.calcsize(fields) - struct.calcsize("@" + fields[-1]) == int(last), name


def test_empty_features_are_refused_as_such(monkeypatch):
    """No features: a ValueError that says so, whatever the gate."""
    monkeypatch.setattr(ops, "_device_of", lambda t: -1)
    monkeypatch.setattr(ops, "_raw_stream", lambda i: 0)
    monkeypatch.setattr(ops, "_cur_device", lambda: -1)
    x, w = torch.zeros((3, 0), dtype=torch.bfloat16), torch.zeros(0, dtype=torch.bfloat16)
    for gate in (None, torch.zeros((3, 0), dtype=torch.bfloat16), w, torch.zeros((3, 1), dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="N=0"):
            ops.gated_add_rmsnorm(x, x, w, 1e-6, gate=gate)


def test_experts_take_plain_tensors_one_by_one(monkeypatch):
    """Plain [E, N, K] tensors stand for 16-bit experts in both calls, beside
    DenseExpertWeights too; a plain tensor beside AWQ experts is refused."""
    seen = []
    backend = AWQB200MoeBackend()
    monkeypatch.setattr(backend, "_dense_experts", lambda x, w1, w2, tw, ids: seen.append((w1, w2)) or x)
    monkeypatch.setattr(ops, "moe_topk_softmax", lambda g, k, r: (torch.zeros(3, k), torch.zeros((3, k), dtype=torch.int32)))
    x, w1, w2 = (torch.zeros(s, dtype=torch.float16) for s in ((3, 64), (4, 32, 64), (4, 64, 16)))
    ids = torch.zeros((3, 2), dtype=torch.int32)
    for a, b in ((w1, w2), (DenseExpertWeights(w1), w2), (w1, DenseExpertWeights(w2))):
        backend.forward(x, a, b, torch.zeros(3, 4), 2, True)
        backend.experts(x, a, b, torch.zeros(3, 2), ids)
    assert len(seen) == 6
    assert all(isinstance(w, DenseExpertWeights) and w.num_experts == 4 for pair in seen for w in pair)
    with pytest.raises(ValueError, match="different experts"):  # the plain ones are experts 0 .. 3
        backend.forward(x, DenseExpertWeights(w1, 4, 8), w2, torch.zeros(3, 8), 2, True)
    awq = AWQExpertWeights(torch.zeros((1, 16), dtype=torch.uint8), 16, 64, 16, torch.float16)
    with pytest.raises(ValueError, match="both"):
        backend.experts(x, w1[:1], awq, torch.zeros(3, 2), ids)
