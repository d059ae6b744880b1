"""Microscaled 4-bit floating point without a GPU: the oracle's own formats, the layout
of weight scales, argument structures and refusals. Every refusal of the C entry points
comes before any GPU work, so made-up addresses are never read."""

import os
import struct
import subprocess

import pytest
import torch

from oracle.fp4_ref import BLOCK, E4M3, GRID, nearest, pack, quantize_ref, values_ref
from sglite_b200 import _lib, ops

P = 256  # an aligned address that nothing reads


def _refused(name, args, change, text):
    args = list(args)
    for k, v in change.items():
        args[int(k[1:])] = v
    fn = getattr(_lib.lib(), name)
    assert fn(_lib.FP4_ARGS[name].pack(*(0 if v is None else v for v in args)), None) == 1
    assert text in _lib.lib().awqb_last_error()


Q = [P, 8, 256, 256, 0, 1, P, None, 1, None, 8, P, P]


@pytest.mark.parametrize("change,text", [
    ({"_3": 240}, b"K="), ({"_3": 0}, b"K="), ({"_3": -32}, b"K="), ({"_4": 2}, b"format"), ({"_4": -1}, b"format"),
    ({"_5": 2}, b"dtype"), ({"_2": 248}, b"row stride"), ({"_2": 260}, b"row stride"), ({"_10": 9}, b"index"),
    ({"_1": -1, "_10": -1}, b"rows"), ({"_8": 0, "_7": P}, b"per_row"), ({"_0": None}, b"null"), ({"_11": None}, b"null"),
    ({"_12": None}, b"null"), ({"_0": 8}, b"16-byte"), ({"_11": 8}, b"16-byte"), ({"_12": 8}, b"16-byte"),
    ({"_4": 1}, b"scale")])
def test_quantize_refusals(change, text):
    _refused("awqb_fp4_quantize", Q, change, text)


def test_quantize_takes_an_empty_index():
    """A list of no rows has no address; nothing is launched for it."""
    args = list(Q)
    args[10], args[11], args[12] = 0, None, None
    assert _lib.lib().awqb_fp4_quantize(_lib.FP4_ARGS["awqb_fp4_quantize"].pack(*(0 if v is None else v for v in args)), None) == 0


D = [P, P, 8, 256, 0, 1, P, P, 256]


@pytest.mark.parametrize("change,text", [
    ({"_3": 48}, b"K="), ({"_4": 7}, b"format"), ({"_5": -1}, b"dtype"), ({"_8": 252}, b"row stride"), ({"_8": 8}, b"row stride"),
    ({"_2": -1}, b"rows"), ({"_0": None}, b"null"), ({"_1": None}, b"null"), ({"_7": None}, b"null"), ({"_7": 24}, b"16-byte"),
    ({"_4": 1}, b"scale")])
def test_dequantize_refusals(change, text):
    _refused("awqb_fp4_dequantize", D, change, text)


NORM = [P, 256, P, 256, P, P, 256, 8, 256, 1e-6, 0, 1, P, P, P]


@pytest.mark.parametrize("change,text", [
    ({"_8": 250}, b"K="), ({"_8": 16416, "_1": 16416, "_3": 16416, "_6": 16416}, b"at most"), ({"_1": 8}, b"row strides"),
    ({"_3": 255}, b"row strides"), ({"_6": 0}, b"row strides"), ({"_9": -1.0}, b"eps"), ({"_9": float("nan")}, b"eps"),
    ({"_10": 3}, b"format"), ({"_11": 3}, b"dtype"), ({"_0": None}, b"null"), ({"_4": None}, b"null"),
    ({"_5": None}, b"null"), ({"_13": None}, b"null"), ({"_14": None}, b"null"), ({"_4": 8}, b"16-byte"), ({"_7": -1}, b"rows"),
    ({"_10": 1}, b"scale")])
def test_add_rmsnorm_refusals(change, text):
    _refused("awqb_fp4_add_rmsnorm", NORM, change, text)


G = [P, P, 64, 256, P, P, 8, 512, P, 0, 1, P, P, None, 0, None, None, P, 64, 512]


@pytest.mark.parametrize("change,text", [
    ({"_3": 264}, b"K="), ({"_3": 0}, b"K="), ({"_7": 516}, b"N="), ({"_7": 0}, b"N="), ({"_7": 520, "_14": 1}, b"multiple of 16"),
    ({"_6": 0}, b"experts"), ({"_6": 1025}, b"experts"), ({"_8": None}, b"offsets"), ({"_13": P}, b"bias"),
    ({"_19": 504}, b"row stride"), ({"_19": 516}, b"row stride"), ({"_18": 63}, b"out has"), ({"_2": -1}, b"row count"),
    ({"_9": 2}, b"format"), ({"_10": 2}, b"dtype"), ({"_0": None}, b"null"), ({"_1": None}, b"null"), ({"_4": None}, b"null"),
    ({"_5": None}, b"null"), ({"_17": None}, b"null"), ({"_0": 8}, b"16-byte"), ({"_1": 8}, b"16-byte"), ({"_4": 8}, b"16-byte"),
    ({"_5": 8}, b"16-byte"), ({"_17": 8}, b"16-byte"), ({"_7": 1 << 29}, b"N="), ({"_9": 1}, b"scale")])
def test_gemm_refusals(change, text):
    _refused("awqb_fp4_gemm", G, change, text)


@pytest.mark.parametrize("E,N", [(1, 0x7ffffff8), (1, 0x7fffff08), (8, 1 << 28), (1024, 1 << 60)])
def test_weights_of_more_rows_than_coordinates_are_refused(E, N):
    """Up to where the last tile's rows still count in 32 bits; E * N itself may pass 64."""
    _refused("awqb_fp4_gemm", G, {"_6": E, "_7": N, "_19": N}, b"N=")


def test_null_arguments_are_refused():
    for name in _lib.FP4_ARGS:
        assert getattr(_lib.lib(), name)(None, None) == 1


def test_packed_structures_have_the_size_that_c_reads(tmp_path):
    names = {n: (f"{n}_args", last) for n, last in
             (("awqb_fp4_quantize", "scales"), ("awqb_fp4_dequantize", "ldo"), ("awqb_fp4_add_rmsnorm", "scales"),
              ("awqb_fp4_gemm", "ldo"))}
    assert set(names) == set(_lib.FP4_ARGS)
    lines = [f'printf("{k} %zu %zu\\n", sizeof({t}), offsetof({t}, {last}));' for k, (t, last) in names.items()]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "awqb200.h"\nint main(void) {\n' + "\n".join(lines)
                   + "\nreturn 0;\n}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "sizes")], check=True)
    for line in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size, last = line.split()
        fields = _lib.FP4_ARGS[name].format.removesuffix("0q")
        assert _lib.FP4_ARGS[name].size == int(size), name
        assert struct.calcsize(fields) - struct.calcsize("@" + fields[-1]) == int(last), name


# ---------------------------------------------------------------- the oracle and the layouts
def test_oracle_formats():
    assert torch.equal(E4M3.float(), torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float())
    v = torch.tensor([0.25, 0.2500001, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.0000001, 100.0], dtype=torch.float64)
    assert GRID[nearest(v, GRID)].tolist() == [0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6]
    s = torch.rand(5000, dtype=torch.float64) * 448
    assert torch.equal(E4M3[nearest(s.float().double(), E4M3)].float(), s.float().to(torch.float8_e4m3fn).float())
    for fmt in BLOCK:
        x = torch.randn(7, 96) * 3
        values, byte = quantize_ref(x, fmt)
        assert torch.equal(values_ref(pack(values, byte, fmt), byte, fmt), values)
        assert float((values - x).norm() / x.norm()) < 0.2


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("shape", [(8, 32), (128, 256), (200, 800), (3, 136, 96)])
def test_laid_out_scales(fmt, shape):
    N, K = shape[-2:]
    b = BLOCK[fmt]
    s = torch.randint(1, 256, (*shape[:-1], K // b), dtype=torch.uint8)
    t = ops.fp4_lay_out_scales(s, fmt)
    assert t.shape == (*shape[:-2], -(-N // 128), -(-K // 256), 64 // b, 32, 4, 4) and t.is_contiguous()
    flat, want = t.reshape(-1, *t.shape[len(shape) - 2:]), s.reshape(-1, N, K // b)
    n, k = torch.meshgrid(torch.arange(N), torch.arange(K // b), indexing="ij")
    k0 = k * b
    got = flat[:, n // 128, k0 // 256, k0 % 256 // (4 * b), n % 32, n % 128 // 32, k % 4]
    assert torch.equal(got, want)
    assert int(t.count_nonzero()) == s.numel()  # zero everywhere else
    assert torch.equal(ops.fp4_lay_out_scales(s.view(torch.int8), fmt), t)


@pytest.mark.parametrize("bad", [torch.zeros(4, dtype=torch.uint8), torch.zeros((4, 4))])
def test_scales_to_lay_out_are_bytes(bad):
    with pytest.raises(ValueError):
        ops.fp4_lay_out_scales(bad, "nvfp4")


# ---------------------------------------------------------------- refusals of the wrappers
@pytest.fixture
def here(monkeypatch):
    """Lets CPU tensors pass for CUDA ones up to the call itself, which must not be reached."""
    def reached(*a):
        raise AssertionError("the call was made")
    monkeypatch.setattr(ops, "_device_of", lambda t: -1)
    monkeypatch.setattr(ops, "_run", reached)


def _rows(M, K, fmt):
    c, s = ops.fp4_rows_empty(M, K, fmt, "cpu")
    return c.zero_(), s.zero_()


def test_wrappers_refuse(here):
    T = torch.bfloat16
    x = torch.zeros((4, 64), dtype=T)
    one = torch.ones(1)
    i32 = torch.zeros(4, dtype=torch.int32)
    for kw in ({"fmt": "fp4"}, {"fmt": "mxfp4", "scale": one}, {"scale": one.double()}, {"scale": torch.ones(2)},
               {"index": i32.long()}, {"index": i32[::2]}, {"per_row": 2}, {"count": i32}, {"count": torch.zeros(1)},
               {"out": _rows(3, 64, "nvfp4")}, {"out": _rows(4, 96, "nvfp4")}, {"out": _rows(4, 64, "nvfp4")[::-1]}):
        with pytest.raises(ValueError):
            ops.fp4_quantize(x, kw.pop("fmt", "nvfp4"), **kw)
    with pytest.raises(ValueError):
        ops.fp4_quantize(x.float(), "nvfp4")
    with pytest.raises(ValueError):
        ops.fp4_quantize(x.T, "nvfp4")
    c, s = _rows(4, 64, "nvfp4")
    for args in ((c.int(), s), (c, s[:, :3]), (c, s.int()), (c[:, ::2], s)):
        with pytest.raises(ValueError):
            ops.fp4_dequantize(*args, "nvfp4", T)
    with pytest.raises(ValueError):
        ops.fp4_dequantize(c, s, "nvfp4", torch.float32)
    with pytest.raises(ValueError):
        ops.fp4_dequantize(c, s, "nvfp4", T, out=torch.zeros((4, 60), dtype=T))
    w = torch.zeros(64, dtype=T)
    for args, kw in (((x, x.half(), w), {}), ((x, x[:2], w), {}), ((x, x, w[:32]), {}), ((x, x, w.half()), {}),
                     ((x, None, w), {"residual_out": x}), ((x, x, w), {"residual_out": x.half()}), ((x, x, w), {"scale": w})):
        with pytest.raises(ValueError):
            ops.fp4_add_rmsnorm(*args, 1e-6, "nvfp4", **kw)


def test_products_refuse(here):
    T = torch.bfloat16
    c, s = _rows(4, 64, "nvfp4")
    w = torch.zeros((32, 32), dtype=torch.uint8)
    ws = ops.fp4_lay_out_scales(torch.zeros((32, 4), dtype=torch.uint8), "nvfp4")
    for args, kw in (((c, s, w[:, :16], ws), {}), ((c, s, w.int(), ws), {}), ((c, s, w, ws[..., :2]), {}),
                     ((c, s, w[None], ws[None]), {}), ((c, s, w, ws), {"bias": torch.zeros(32)}),
                     ((c, s, w, ws), {"bias": torch.zeros(16, dtype=T)}), ((c, s, w, ws), {"x_scale": torch.ones(2)}),
                     ((c, s, w, ws), {"w_scale": torch.ones(1, dtype=T)}), ((c, s, w, ws), {"out": torch.zeros((4, 16), dtype=T)}),
                     ((c, s, w, ws), {"out": torch.zeros((4, 32), dtype=T), "silu_mul": True}), ((c, s[:, :2], w, ws), {})):
        with pytest.raises(ValueError):
            ops.fp4_gemm(*args, "nvfp4", T, **kw)
    with pytest.raises(ValueError):  # laid out for the other format
        ops.fp4_gemm(c, s, w, ws, "mxfp4", T)
    w3, ws3 = w.expand(2, 32, 32).contiguous(), ws.expand(2, *ws.shape).contiguous()
    off = torch.zeros(3, dtype=torch.int32)
    for args, kw in (((c, s, w, ws, off), {}), ((c, s, w3, ws3, off[:2]), {}), ((c, s, w3, ws3, off.long()), {}),
                     ((c, s, w3, ws, off), {}), ((c, s, w3, ws3, off), {"w_scale": torch.ones(1)}),
                     ((c, s, w3, ws3, off), {"row_map": off}), ((c, s, w3, ws3, off), {"row_scale": torch.ones(3)}),
                     ((c, s, w3, ws3, off), {"out": torch.zeros((4, 16), dtype=T)})):
        with pytest.raises(ValueError):
            ops.fp4_grouped_gemm(*args, "nvfp4", T, **kw)


def test_cpu_tensors_are_refused():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.fp4_quantize(x, "nvfp4")
    with pytest.raises(ValueError, match="CUDA"):
        ops.fp4_add_rmsnorm(x, None, x[0], 1e-6, "mxfp4")
    c, s = _rows(2, 64, "nvfp4")
    with pytest.raises(ValueError, match="CUDA"):
        ops.fp4_dequantize(c, s, "nvfp4", torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.fp4_gemm(c, s, c, s, "nvfp4", torch.float16)


# ---------------------------------------------------------------- config and linear method
def test_config():
    from sglite_b200.quantization import get_quantization_config
    from sglite_b200.quantization.fp4_b200 import FP4B200Config

    assert get_quantization_config("FP4_B200") is FP4B200Config
    for config, fmt in (({"quant_algo": "NVFP4", "group_size": 16}, "nvfp4"), ({"quant_method": "mxfp4"}, "mxfp4")):
        c = FP4B200Config.from_config(config)
        assert c.fmt == fmt and c.group_size == BLOCK[fmt] and c.get_name() == "fp4_b200"
        assert torch.bfloat16 in c.get_supported_act_dtypes() and c.get_min_capability() == 100
    for bad in ({"quant_algo": "FP8"}, {"quant_algo": "NVFP4", "group_size": 32}, {"group_size": 16}):
        with pytest.raises(ValueError):
            FP4B200Config.from_config(bad)
    with pytest.raises(ValueError):
        FP4B200Config("int4")


def test_config_of_a_checkpoint_file():
    """hf_quant_config.json keeps its entries under "quantization"."""
    from sglite_b200.quantization.fp4_b200 import FP4B200Config

    assert FP4B200Config.get_config_filenames()[0] == "hf_quant_config.json"
    inner = {"quant_algo": "NVFP4", "kv_cache_quant_algo": None, "group_size": 16, "exclude_modules": ["lm_head"]}
    assert FP4B200Config.from_config({"producer": {"name": "x", "version": "1"}, "quantization": inner}).fmt == "nvfp4"
    assert FP4B200Config.from_config({"quant_method": "modelopt_fp4"}).fmt == "nvfp4"
    for bad in ({**inner, "group_size": 32}, {**inner, "quant_algo": "FP8"}, {"group_size": 16}):
        with pytest.raises(ValueError):
            FP4B200Config.from_config({"quantization": bad})
    with pytest.raises(ValueError):  # its tensors have other names, and its global scale is the reciprocal
        FP4B200Config.from_config({"quant_method": "compressed-tensors", "format": "nvfp4-pack-quantized"})


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_created_weights(fmt):
    from sglite_b200.quantization.fp4_b200 import FP4B200Config

    method = FP4B200Config(fmt).get_linear_method()
    w = method.create_weights(96, 24)
    assert w["weight"].shape == (24, 48) and w["weight_scale"].shape == (24, 96 // BLOCK[fmt])
    assert w["weight"].packed_dim == 1 and w["weight"].pack_factor == 2 and w["weight_scale"].output_dim == 0
    assert ("input_scale" in w) == (fmt == "nvfp4") == ("weight_scale_2" in w)
    for sizes in ((80, 24), (96, 20)):
        with pytest.raises(ValueError):
            method.create_weights(*sizes)
    with pytest.raises(RuntimeError, match="CUDA"):
        method.process_weights_after_loading(w)
    with pytest.raises(RuntimeError, match="process_weights_after_loading"):
        method.apply_weights(w, torch.zeros((1, 96), dtype=torch.bfloat16))


@pytest.mark.parametrize("fmt,kind", [("nvfp4", torch.float8_e4m3fn), ("mxfp4", torch.float8_e8m0fnu)])
def test_typed_scales_of_a_checkpoint_keep_their_bits(fmt, kind):
    """Block scales typed as 8-bit floats, copied in place as loaders do, whole and by shards."""
    from sglite_b200.quantization.fp4_b200 import FP4B200Config

    method = FP4B200Config(fmt).get_linear_method()
    want = torch.randint(0, 255, (24, 96 // BLOCK[fmt]), dtype=torch.uint8)
    typed = want.view(kind)
    fills = [lambda p: p.data.copy_(typed), lambda p: p.copy_(typed), lambda p: p.copy_(other=typed),
             lambda p: p.data[:8].copy_(typed[:8]) is p.data.narrow(0, 8, 16).copy_(typed.narrow(0, 8, 16)),
             lambda p: p.data.__setitem__(slice(None), typed), lambda p: p.data.copy_(want), lambda p: p.data.copy_(want.int()),
             lambda p: [p.data[:, k:k + 1].copy_(typed[:, k:k + 1]) for k in range(typed.shape[1])]]
    for fill in fills:
        w = method.create_weights(96, 24)
        w["weight_scale"].data.zero_()
        fill(w["weight_scale"])
        assert isinstance(w["weight_scale"], torch.nn.Parameter) and w["weight_scale"].dtype == torch.uint8
        assert torch.equal(w["weight_scale"].data, want)
        assert torch.equal(ops.fp4_lay_out_scales(w["weight_scale"].data, fmt), ops.fp4_lay_out_scales(want, fmt))
    with pytest.raises(ValueError, match="bytes"):
        w["weight_scale"].data.copy_(want.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scale_of_a_tensor_is_that_of_its_finite_values(dtype):
    from sglite_b200.quantization.fp4_b200 import tensor_scale

    w = (torch.randn((8, 64), generator=torch.Generator().manual_seed(1)) * 0.02).to(dtype)
    want = w.abs().amax().float().reshape(1) / 2688
    assert torch.equal(tensor_scale(w), want)
    for bad in (float("inf"), -float("inf"), float("nan")):
        one = w.clone()
        at = int(w.abs().flatten().argmin())
        one.view(-1)[at] = bad
        assert torch.equal(tensor_scale(one), want)
    assert torch.equal(tensor_scale(torch.zeros_like(w)), torch.ones(1))
    if dtype is torch.bfloat16:
        tiny = tensor_scale((w.double() * 2.0 ** -125).to(dtype))
        assert 0 < float(1 / tiny) < float("inf")


def test_interleaved_gate_up():
    t = torch.arange(12).view(6, 2)
    assert ops.fp4_interleave_gate_up(t)[:, 0].tolist() == [0, 6, 2, 8, 4, 10]
    assert ops.fp4_interleave_gate_up(torch.arange(4), dim=-1).tolist() == [0, 2, 1, 3]
    with pytest.raises(ValueError):
        ops.fp4_interleave_gate_up(torch.zeros(3, 2))


def test_experts_from_a_checkpoint_are_checked():
    from sglite_b200.moe import FP4ExpertWeights

    w, s = torch.zeros((2, 16, 32), dtype=torch.uint8), torch.zeros((2, 16, 4), dtype=torch.uint8)
    e = FP4ExpertWeights.from_checkpoint(w, s, "nvfp4", torch.bfloat16, e_begin=2, num_global_experts=8, gate_up=True)
    assert (e.num_experts, e.N, e.K, e.e_end) == (2, 16, 64, 4)
    for bad in ((w, s[:, :, :2]), (w[0], s[0]), (w.int(), s), (w, s.float())):
        with pytest.raises(ValueError):
            FP4ExpertWeights.from_checkpoint(*bad, "nvfp4", torch.bfloat16)


def test_experts_record_the_order_of_their_rows():
    """Gate and up rows in the wrong order are refused, not multiplied to something else."""
    from sglite_b200.moe import AWQB200MoeBackend, FP4ExpertWeights

    E, H, I = 2, 64, 32
    T = torch.bfloat16

    def experts(N, K, **kw):
        w, s = torch.zeros((E, N, K // 2), dtype=torch.uint8), torch.zeros((E, N, K // 16), dtype=torch.uint8)
        return FP4ExpertWeights.from_checkpoint(w, s, "nvfp4", T, **kw)

    by_turns, plain = experts(2 * I, H, gate_up=True), experts(2 * I, H)
    assert by_turns.gate_up_interleaved and plain.gate_up_interleaved is False
    already, down = experts(2 * I, H, gate_up_interleaved=True), experts(H, I)
    assert already.gate_up_interleaved and torch.equal(already.w, plain.w)
    with pytest.raises(ValueError):
        experts(2 * I, H, gate_up=True, gate_up_interleaved=True)
    backend, x = AWQB200MoeBackend(), torch.zeros((0, H), dtype=T)  # (no rows: no kernel runs)
    none = torch.zeros((0, 2)), torch.zeros((0, 2), dtype=torch.int32)
    made = FP4ExpertWeights(by_turns.w, by_turns.w_scales, "nvfp4", T)
    for w1 in (by_turns, already, made):
        assert backend.experts(x, w1, down, *none) is x
    for w1, w2 in ((plain, down), (by_turns, experts(H, I, gate_up=True))):
        with pytest.raises(ValueError, match="by turns"):
            backend.experts(x, w1, w2, *none)
