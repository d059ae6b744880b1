"""Microscaled 4-bit floating point behind the same linear-method interface.

Weights and activations of a projection are both held in four bits (``ops.fp4_gemm``):
``nvfp4``, blocks of 16 with an e4m3 scale and one fp32 scale for the tensor, or
``mxfp4``, blocks of 32 with a power of two. The reference has no such method; the
interface is its ``LinearMethodBase`` (``layers/quantization/base_config.py:9-42``):
``create_weights`` allocates the checkpoint's tensors,
``process_weights_after_loading`` lays the block scales out once,
``apply_weights`` quantises the activations' rows and multiplies.
"""

from __future__ import annotations

from typing import Any, Dict, List, Optional, Tuple, Union

import torch
from torch.nn.parameter import Parameter

from .. import ops
from ..lora import LoraAdapters, LoraBatch
from .base_config import LinearMethodBase, QuantizationConfig, set_weight_attrs

# a tensor's rows already in four bits: (codes, scales) of ops.fp4_quantize or ops.fp4_add_rmsnorm
FP4Rows = Tuple[torch.Tensor, torch.Tensor]


class CheckpointBytes(torch.Tensor):
    """Bytes that a loader fills from a checkpoint. uint8, but a checkpoint may type them
    (scales as float8_e4m3fn or float8_e8m0fnu): copied into these, or into a slice of these,
    they keep their bits, where a plain uint8 tensor would take their values (0.5 as 0)."""

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        kwargs = kwargs or {}
        if func in (torch.Tensor.copy_, torch.Tensor.__setitem__):
            args = (args[0], *map(_as_bytes, args[1:]))
            kwargs = {k: _as_bytes(v) for k, v in kwargs.items()}
        return super().__torch_function__(func, types, args, kwargs)


def _as_bytes(value):
    if not isinstance(value, torch.Tensor) or not value.is_floating_point():
        return value
    if value.element_size() != 1:
        raise ValueError(f"bytes of a checkpoint cannot be taken from {value.dtype} values")
    return value.view(torch.uint8)


def _checkpoint_bytes(rows: int, columns: int) -> Parameter:
    return Parameter(torch.empty(rows, columns, dtype=torch.uint8).as_subclass(CheckpointBytes), requires_grad=False)


def tensor_scale(w: torch.Tensor) -> torch.Tensor:
    """The fp32 [1] scale under which the largest block scale of w's finite values is e4m3's
    largest value. (An infinity would make it infinite and all other values 0, a NaN leave it
    at 1, where small weights lose most of their bits.) At least 2^-126, so that 1 / scale is finite."""
    most = torch.nan_to_num(w, nan=0.0, posinf=0.0, neginf=0.0).abs().amax().float().reshape(1)
    return torch.where(most > 0, (most / (6.0 * 448.0)).clamp(min=2.0 ** -126), 1.0)


def quantize_weight(w: torch.Tensor, fmt: str) -> Dict[str, torch.Tensor]:
    """A 16-bit weight [N, K] as a checkpoint holds it in four bits: ``weight`` uint8
    [N, K / 2], ``weight_scale`` uint8 [N, K / 16 or K / 32] and, for nvfp4,
    ``weight_scale_2`` fp32 [1]."""
    scale = tensor_scale(w) if fmt == "nvfp4" else None
    codes, scales = ops.fp4_quantize(w, fmt, scale=scale)
    block = w.shape[1] // ops.FP4_BLOCK[fmt]
    out = {"weight": codes, "weight_scale": scales.transpose(0, 1).flatten(1)[:, :block].contiguous()}
    if scale is not None:
        out["weight_scale_2"] = scale
    return out


class FP4B200Config(QuantizationConfig):
    """Config for microscaled 4-bit weights and activations on B200."""

    def __init__(self, fmt: str) -> None:
        if fmt not in ops.FP4_FORMATS:
            raise ValueError(f"4-bit format {fmt!r}: one of {tuple(ops.FP4_FORMATS)}")
        self.fmt = fmt
        self.group_size = ops.FP4_BLOCK[fmt]
        self.weight_bits = 4
        self.pack_factor = 2  # values of a byte

    def __repr__(self) -> str:
        return f"FP4B200Config(fmt={self.fmt!r})"

    def get_name(self) -> str:
        return "fp4_b200"

    def get_supported_act_dtypes(self) -> List[torch.dtype]:
        return [torch.half, torch.bfloat16]

    def get_min_capability(self) -> int:
        return 100

    @staticmethod
    def get_config_filenames() -> List[str]:
        return ["hf_quant_config.json", "quant_config.json"]

    @classmethod
    def from_config(cls, config: Dict[str, Any]) -> "FP4B200Config":
        """``quant_algo``, ``format`` or ``quant_method`` names the format (NVFP4 / MXFP4, any
        case; modelopt_fp4 is NVFP4), at the top or, as hf_quant_config.json has it, under
        ``quantization``."""
        inner = config.get("quantization")
        config = inner if isinstance(inner, dict) else config
        fmt = str(cls.get_from_keys(config, ["quant_algo", "format", "quant_method"])).lower()
        fmt = "nvfp4" if fmt == "modelopt_fp4" else fmt
        group = config.get("group_size")
        if group is not None and fmt in ops.FP4_BLOCK and group != ops.FP4_BLOCK[fmt]:
            raise ValueError(f"{fmt} has blocks of {ops.FP4_BLOCK[fmt]}, got group_size={group}")
        return cls(fmt)

    def get_linear_method(self) -> "FP4B200LinearMethod":
        return FP4B200LinearMethod(self)

    def get_scaled_act_names(self) -> List[str]:
        return []


class FP4B200LinearMethod(LinearMethodBase):
    """Linear method over ``ops.fp4_quantize`` and ``ops.fp4_gemm``."""

    def __init__(self, quant_config: FP4B200Config):
        self.quant_config = quant_config

    def create_weights(self, input_size: int, output_size: int) -> Dict[str, Any]:
        """weight [N, K / 2] (uint8, the value with the even k in the low bits),
        weight_scale [N, K / block] (bytes, also where the checkpoint types them as 8-bit
        floats: CheckpointBytes), and for nvfp4 weight_scale_2 and input_scale (fp32 [1];
        input_scale is the scale of the activations and starts at one)."""
        block = self.quant_config.group_size
        if input_size % 32:
            raise ValueError(f"input_size={input_size} must be a multiple of 32. "
                             "This can be caused by too large tensor parallel size.")
        if output_size % 8:
            raise ValueError(f"output_size={output_size} must be a multiple of 8. "
                             "This can be caused by too large tensor parallel size.")
        weight = _checkpoint_bytes(output_size, input_size // 2)
        set_weight_attrs(weight, {"input_dim": 1, "output_dim": 0, "packed_dim": 1, "pack_factor": 2})
        scale = _checkpoint_bytes(output_size, input_size // block)
        set_weight_attrs(scale, {"input_dim": 1, "output_dim": 0})
        weights = {"weight": weight, "weight_scale": scale, "_input_size": input_size, "_output_size": output_size,
                   "_weights_processed": False}
        if self.quant_config.fmt == "nvfp4":
            for name in ("weight_scale_2", "input_scale"):
                weights[name] = Parameter(torch.ones(1, dtype=torch.float32), requires_grad=False)
        return weights

    def process_weights_after_loading(self, weights: Dict[str, Any]) -> Dict[str, Any]:
        if weights.get("_weights_processed", False):
            return weights
        weight, scale = (weights[name].data.as_subclass(torch.Tensor) for name in ("weight", "weight_scale"))
        if weight.device.type != "cuda":
            raise RuntimeError("FP4 B200 weights must be loaded on a CUDA device before their scales are laid out")
        N, K = weights["_output_size"], weights["_input_size"]
        fmt = self.quant_config.fmt
        if weight.shape != (N, K // 2) or weight.element_size() != 1 \
                or scale.shape != (N, K // ops.FP4_BLOCK[fmt]) or scale.element_size() != 1:
            raise ValueError(f"weight {tuple(weight.shape)} and weight_scale {tuple(scale.shape)} are not those of a "
                             f"{fmt} projection {K} -> {N}")
        out = dict(weights)
        out["weight"] = Parameter(weight.view(torch.uint8).contiguous(), requires_grad=False)
        out["weight_scale"] = Parameter(ops.fp4_lay_out_scales(scale, fmt), requires_grad=False)
        for name in ("weight_scale_2", "input_scale"):
            if name in weights:
                value = weights[name].data.to(weight.device, torch.float32).reshape(-1)
                if value.numel() != 1 or not bool(value > 0):  # (load time: a wait for the device is fine)
                    raise ValueError(f"{name} must be one positive number")
                out[name] = Parameter(value, requires_grad=False)
        out["_weights_processed"] = True
        return out

    def apply_weights(self, weights: Dict[str, Any], x: Union[torch.Tensor, FP4Rows],
                      bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                      adapters: Optional[LoraAdapters] = None, batch: Optional[LoraBatch] = None, *,
                      dtype: Optional[torch.dtype] = None, silu_mul: bool = False) -> torch.Tensor:
        """x W^T (+ bias). x is 16-bit [.., K], quantised here over input_scale, or rows that a
        norm (``norm.RMSNormFP4`` with this projection's input_scale) has quantised, with the
        result's ``dtype``. silu_mul: the weight's rows are gate and up by turns
        (``ops.fp4_interleave_gate_up``). adapters as in ``AWQB200LinearMethod``."""
        if not weights.get("_weights_processed", False):
            raise RuntimeError("process_weights_after_loading must run before apply_weights")
        if adapters is not None and batch is None:
            raise ValueError("adapters need the batch that says which row uses which adapter")
        fmt, K, N = self.quant_config.fmt, weights["_input_size"], weights["_output_size"]
        x_scale = weights.get("input_scale")
        n_out = N // 2 if silu_mul else N
        if isinstance(x, torch.Tensor):
            if x.shape[-1] != K:
                raise ValueError(f"x has {x.shape[-1]} features, expected K={K}")
            if dtype is not None and dtype != x.dtype:
                raise ValueError(f"dtype {dtype} is for quantised rows; x is {x.dtype}")
            dtype, shape = x.dtype, (*x.shape[:-1], n_out)
            rows = ops.fp4_quantize(x, fmt, scale=x_scale)
        else:
            if dtype is None:
                raise ValueError("quantised rows need the result's dtype")
            if adapters is not None:
                raise ValueError("adapters need the 16-bit activations")
            rows, shape = x, None
        if adapters is not None and silu_mul:
            raise ValueError("adapters add to the projection's output, which silu_mul does not leave")
        if out is not None and out.dim() != 2:
            out = out.view(-1, n_out)
        y = ops.fp4_gemm(rows[0], rows[1], weights["weight"], weights["weight_scale"], fmt, dtype, x_scale=x_scale,
                         w_scale=weights.get("weight_scale_2"), bias=bias, silu_mul=silu_mul, out=out)
        if shape is not None and len(shape) != 2:
            y = y.view(shape)
        return y if adapters is None else adapters.add_to(y, x, batch)
