"""Refusals and host logic of the operators around the projections; no GPU. Every
C-ABI refusal comes before any GPU work, so made-up addresses are never read."""

import math

import pytest
import torch

from sglite_b200 import _lib, ops
from sglite_b200.lora import LoraAdapters
from sglite_b200.moe import AWQB200MoeBackend, DenseExpertWeights
from sglite_b200.rotary import RotaryEmbedding, rotary_frequencies

P = 256  # an aligned address that nothing reads


def _call(name, args):
    """args as in include/awqb200.h, packed where the entry point takes a structure."""
    fn = getattr(_lib.lib(), name)
    if name not in _lib.ARGS:
        return fn(*args)
    return fn(_lib.ARGS[name].pack(*(0 if v is None else v for v in args[:-1])), args[-1])


def _refused(name, args, status, text):
    assert _call(name, args) == status
    assert text in _lib.lib().awqb_last_error()


def _replace(args, **at):
    out = list(args)
    for k, v in at.items():
        out[int(k[1:])] = v
    return out


NORM = [P, 4096, P, 4096, 0, P, P, 4096, 1, 0, 1.0, P, 0.0, P, 4096, P, 4096, 4, 4096, 1e-6, 1, None]


@pytest.mark.parametrize("change,text", [
    ({"_18": 4100}, b"multiple of 8"), ({"_18": 16392, "_1": 16392}, b"at most"), ({"_1": 4088}, b"row strides"),
    ({"_3": 4100}, b"row strides"), ({"_9": 4}, b"activation"), ({"_19": -1.0}, b"eps"), ({"_8": 2}, b"gate_col"),
    ({"_7": 4090}, b"row stride"), ({"_5": None, "_11": None}, b"weights must be given"), ({"_0": None}, b"null"),
    ({"_15": None}, b"null"), ({"_13": None}, b"null"), ({"_0": 8}, b"16-byte"), ({"_6": 8}, b"16-byte"),
    ({"_20": 5}, b"dtype"), ({"_17": -1}, b"")])
def test_gated_norm_refusals(change, text):
    _refused("awqb_gated_add_rmsnorm", _replace(NORM, **change), 1, text)


ROT = [P, 4096, 128, 32, P, 1024, 128, 8, P, 1, P, 128, 128, 4, 0, 1.0, P, P, 1e-6, P, 4096, 128, P, 1024, 128, 1, None]


@pytest.mark.parametrize("change,text", [
    ({"_12": 100}, b"head_dim"), ({"_12": 264}, b"head_dim"), ({"_11": 130}, b"rot_dim"), ({"_11": 3}, b"rot_dim"),
    ({"_11": 0}, b"rot_dim"), ({"_3": 0}, b"sizes"), ({"_7": -1}, b"sizes"), ({"_1": 4100}, b"strides"),
    ({"_24": 4}, b"strides"), ({"_8": None}, b"null"), ({"_4": None}, b"null"), ({"_19": 8}, b"16-byte"),
    ({"_25": 9}, b"dtype"), ({"_18": -1.0}, b"eps"), ({"_21": 0}, b"overlap"), ({"_20": 0}, b"overlap"),
    ({"_20": 4088}, b"overlap"), ({"_23": 1016}, b"overlap"), ({"_24": 120}, b"overlap")])
def test_rotary_refusals(change, text):
    _refused("awqb_rotary", _replace(ROT, **change), 1, text)


GROUP = [P, 100, 0, 8, P, P, None, 0, None]


@pytest.mark.parametrize("change,text", [
    ({"_3": 0}, b"groups"), ({"_3": 1025}, b"groups"), ({"_1": -1}, b"number of ids"), ({"_0": None}, b"null"),
    ({"_5": None}, b"null"), ({"_1": 20000}, b"workspace"), ({"_2": 1 << 40}, b"first id")])
def test_group_rows_refusals(change, text):
    _refused("awqb_group_rows", _replace(GROUP, **change), 1, text)


GG = [P, 64, 256, P, 8, 256, 512, P, 1, 0, None, None, P, 64, 512, None]


@pytest.mark.parametrize("change,text", [
    ({"_5": 260}, b"K="), ({"_5": 0}, b"K="), ({"_6": 516}, b"N="), ({"_6": 520, "_9": 1}, b"multiple of 16"),
    ({"_4": 0}, b"experts"), ({"_4": 1025}, b"experts"), ({"_2": 248}, b"row strides"), ({"_14": 504}, b"row strides"),
    ({"_2": 260}, b"row strides"), ({"_13": 63}, b"out has"), ({"_1": -1}, b"rows"), ({"_0": None}, b"null"),
    ({"_7": None}, b"null"), ({"_12": 8}, b"16-byte"), ({"_8": 2}, b"dtype"), ({"_6": 1 << 21}, b"N=")])
def test_grouped_gemm_refusals(change, text):
    _refused("awqb_grouped_gemm", _replace(GG, **change), 1, text)


LORA = [P, 16, 256, 256, P, P, 4, 16, 512, 1, 512, 0, 0, 0, P, P, None, P, 512, P, 512, 1, P, 1 << 30, None]


@pytest.mark.parametrize("change,text", [
    ({"_3": 100}, b"K="), ({"_7": 12}, b"rank"), ({"_7": 136}, b"rank"), ({"_7": 0}, b"rank"), ({"_6": 0}, b"adapters"),
    ({"_6": 2000}, b"adapters"), ({"_9": 5}, b"slices"), ({"_9": 0}, b"slices"), ({"_8": 500}, b"N="),
    ({"_9": 2, "_10": 256, "_11": 128}, b"add up"), ({"_9": 2, "_10": 508, "_11": 4}, b"slice width"),
    ({"_10": 0}, b"slice width"), ({"_2": 248}, b"row strides"), ({"_18": 500}, b"row strides"),
    ({"_20": 508}, b"row strides"), ({"_23": 16}, b"workspace"), ({"_22": None}, b"workspace"), ({"_0": None}, b"null"),
    ({"_14": None}, b"null"), ({"_19": 8}, b"16-byte"), ({"_21": 3}, b"dtype"), ({"_20": 520}, b"in place")])
def test_lora_refusals(change, text):
    _refused("awqb_lora", _replace(LORA, **change), 1, text)


def test_a_missing_structure_is_refused():
    for name in _lib.ARGS:
        assert getattr(_lib.lib(), name)(None, None) == 1
        assert b"args" in _lib.lib().awqb_last_error()


def test_nothing_to_do_is_ok():
    assert _call("awqb_gated_add_rmsnorm", _replace(NORM, _0=None, _17=0)) == 0
    assert _call("awqb_rotary", _replace(ROT, _0=None, _13=0)) == 0
    assert _call("awqb_grouped_gemm", _replace(GG, _0=None, _1=0)) == 0
    assert _call("awqb_lora", _replace(LORA, _0=None, _1=0)) == 0


def test_wrappers_refuse_cpu_tensors_and_bad_shapes():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.gated_add_rmsnorm(x, x, w, 1e-6)
    with pytest.raises(ValueError):
        ops.gated_add_rmsnorm(x.float(), x, w, 1e-6)
    with pytest.raises(ValueError):
        ops.rotary(x.view(4, 1, 64), None, torch.arange(4), torch.ones(32, dtype=torch.float64))
    with pytest.raises(ValueError):
        ops.grouped_gemm(x, torch.zeros(2, 8, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.grouped_gemm(x, torch.zeros(2, 8, 56, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.lora(x, torch.zeros(1, 8, 64, dtype=torch.bfloat16), torch.zeros(1, 8, 8, dtype=torch.bfloat16),
                 torch.zeros(4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), x[:, :8])
    with pytest.raises(ValueError):
        ops.group_rows(torch.zeros(4, dtype=torch.int32), 2)


def test_dense_expert_weights_and_mixed_experts():
    with pytest.raises(ValueError):
        DenseExpertWeights(torch.zeros(2, 8, 8))  # float32
    w1, w2 = (DenseExpertWeights(torch.zeros(s, dtype=torch.float16), 2, 8) for s in ((4, 32, 64), (4, 64, 16)))
    assert (w1.num_experts, w1.N, w1.K, w1.e_end) == (4, 32, 64, 6)
    ids = torch.zeros((3, 2), dtype=torch.int32)
    with pytest.raises(ValueError):  # w2 of other experts
        AWQB200MoeBackend().experts(torch.zeros(3, 64, dtype=torch.float16), w1, DenseExpertWeights(w2.w, 0, 8),
                                    torch.zeros(3, 2), ids)
    with pytest.raises(ValueError):  # shapes
        AWQB200MoeBackend().experts(torch.zeros(3, 32, dtype=torch.float16), w1, w2, torch.zeros(3, 2), ids)


def test_frequencies_follow_their_formulas():
    inv, f = rotary_frequencies(128, 10000.0)
    assert f == 1.0 and inv.dtype == torch.float64
    assert torch.allclose(inv, torch.tensor([10000.0 ** (-2 * j / 128) for j in range(64)], dtype=torch.float64), rtol=1e-14)
    assert torch.allclose(rotary_frequencies(128, 10000.0, {"type": "linear", "factor": 8})[0], inv / 8, rtol=1e-14)
    sc = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    l3 = rotary_frequencies(128, 500000.0, sc)[0]
    base = rotary_frequencies(128, 500000.0)[0]
    wave = 2 * math.pi / base
    assert torch.equal(l3[wave < 8192 / 4.0], base[wave < 8192 / 4.0])
    assert torch.allclose(l3[wave > 8192], base[wave > 8192] / 8, rtol=1e-14)
    mid = (wave >= 8192 / 4.0) & (wave <= 8192)
    assert bool(((l3[mid] <= base[mid]) & (l3[mid] >= base[mid] / 8)).all()) and bool(mid.any())
    y, f = rotary_frequencies(128, 1e6, {"type": "yarn", "factor": 4, "original_max_position_embeddings": 32768})
    full = rotary_frequencies(128, 1e6)[0]
    assert math.isclose(f, 0.1 * math.log(4) + 1)
    turns = 32768 * full / (2 * math.pi)
    assert torch.equal(y[turns > 33], full[turns > 33])  # fast pairs stay
    assert torch.allclose(y[turns < 0.7], full[turns < 0.7] / 4, rtol=1e-14)
    assert torch.allclose(rotary_frequencies(8, 1e4, {"type": "longrope", "factors": [1, 2, 3, 4]})[0],
                          rotary_frequencies(8, 1e4)[0] / torch.tensor([1.0, 2, 3, 4], dtype=torch.float64))


@pytest.mark.parametrize("rot,scaling", [(7, None), (0, None), (8, {"type": "linear"}), (8, {"type": "linear", "factor": 0.5}),
                                         (8, {"type": "spiral", "factor": 2}), (8, {"type": "longrope", "factors": [1]}),
                                         (8, {"type": "yarn", "factor": 2}), (8, {"type": "dynamic", "factor": 2}),
                                         (8, {"type": "longrope", "long_factor": [1, 2, 3, 4]}),
                                         (8, {"type": "llama3", "factor": 2, "original_max_position_embeddings": 10,
                                              "low_freq_factor": 4, "high_freq_factor": 4})])
def test_frequency_refusals(rot, scaling):
    with pytest.raises(ValueError):
        rotary_frequencies(rot, 10000.0, scaling)


def test_factors_on_the_turned_elements():
    yarn = {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096}
    m = 0.1 * math.log(40)
    assert math.isclose(rotary_frequencies(64, 1e4, yarn)[1], m + 1)
    assert math.isclose(rotary_frequencies(64, 1e4, {**yarn, "mscale": 0.707, "mscale_all_dim": 0.707})[1], 1.0)
    assert math.isclose(rotary_frequencies(64, 1e4, {**yarn, "mscale": 0.5, "mscale_all_dim": 0.25})[1],
                        (0.5 * m + 1) / (0.25 * m + 1))
    long = {"type": "longrope", "long_factor": [1, 2, 3, 4], "factor": 32, "original_max_position_embeddings": 4096}
    assert math.isclose(rotary_frequencies(8, 1e4, long)[1], math.sqrt(1 + math.log(32) / math.log(4096)))
    # without rounding the ramp's ends to whole pairs, it runs from one exact pair to the other
    exact = rotary_frequencies(64, 1e4, {**yarn, "truncate": False})[0] / rotary_frequencies(64, 1e4)[0]
    lo, hi = (64 * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(1e4)) for t in (32, 1))
    for j in range(32):
        r = min(max((j - lo) / (hi - lo), 0), 1)
        assert math.isclose(float(exact[j]), 1 - r + r / 40, rel_tol=1e-12)


def test_rotary_layer_refuses_other_widths():
    with pytest.raises(ValueError):
        RotaryEmbedding(8, 2, 64).forward(torch.zeros(3, 64), torch.arange(3))


def test_stacked_adapters_equal_the_sum_of_their_parts():
    """Zero-padded ranks and absent slices change no sum; shards add up / concatenate."""
    g = torch.Generator().manual_seed(0)
    K, widths = 32, (16, 8)

    def pair(r, n):
        return torch.randn((r, K), generator=g), torch.randn((n, r), generator=g)

    ads = [[pair(4, 16), pair(10, 8)], [None, pair(3, 8)]]
    s = LoraAdapters.stack(ads, widths, scales=[1.0, 2.0])
    assert s.a.shape == (2, 32, K) and s.b.shape == (2, 24, 16) and s.slices == widths
    x = torch.randn((5, K), generator=g)

    def product(ad, l, x):
        h = x @ ad.a[l].T
        at, out, r = 0, [], ad.b.shape[2]
        for i, w in enumerate(ad.slices):
            out.append(h[:, i * r:(i + 1) * r] @ ad.b[l, at:at + w].T)
            at += w
        return torch.cat(out, dim=1)

    for l, ad in enumerate(ads):
        want = torch.cat([torch.zeros(5, w) if p is None else x @ p[0].T @ p[1].T for p, w in zip(ad, widths)], dim=1)
        assert torch.allclose(product(s, l, x), want, atol=1e-4)
        row = [s.shard("row", r, 2) for r in range(2)]
        assert torch.allclose(sum(product(p, l, xs) for p, xs in zip(row, x.chunk(2, dim=1))), want, atol=1e-4)
        col = [product(s.shard("column", r, 2), l, x).split([8, 4], dim=1) for r in range(2)]
        assert torch.allclose(torch.cat([torch.cat([c[i] for c in col], dim=1) for i in range(2)], dim=1), want, atol=1e-4)
    with pytest.raises(ValueError):
        LoraAdapters.stack([[None]], (8,))
    with pytest.raises(ValueError):
        LoraAdapters.stack([[pair(4, 16)]], (8,))
    with pytest.raises(ValueError):
        s.shard("column", 0, 3)
