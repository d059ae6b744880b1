"""Rotary position layer over ``ops.rotary``: the step between the QKV projection
and attention (``models/blocks.py:134-139``, ``layers/rotary.py``).

A long-context scaling changes the angular speeds of the pairs and, for YaRN, a
factor on the turned elements; both are worked out here once, in fp64, on the
CPU. Nothing is tabulated by position, so there is no longest position."""

from __future__ import annotations

import math
from typing import Any, Dict, Optional, Sequence, Tuple

import torch

from . import ops


def _longrope_factors(scaling: Dict[str, Any], max_length: Optional[int]) -> Sequence[float]:
    """The list of an entry that applies to sequences of up to ``max_length`` tokens."""
    if scaling.get("factors"):
        return scaling["factors"]
    short, long = list(scaling.get("short_factor") or ()), list(scaling.get("long_factor") or ())
    if not short or short == long:
        return long
    if max_length is None:
        raise ValueError("longrope with a short_factor changes with the sequences' length: say the longest one as "
                         "max_length (or name the list as 'factors')")
    original = scaling.get("original_max_position_embeddings")
    if original is None:
        raise ValueError("longrope with a short_factor needs 'original_max_position_embeddings'")
    return short if max_length <= int(original) else long


def rotary_frequencies(rot_dim: int, base: float = 10000.0, scaling: Optional[Dict[str, Any]] = None,
                       max_length: Optional[int] = None) -> Tuple[torch.Tensor, float]:
    """(inv_freq float64 [rot_dim / 2], factor on the turned elements) for a
    checkpoint's ``rope_scaling`` entry: None or "default", "linear", "llama3", "yarn",
    "longrope" (one factor per pair: ``long_factor``, with what its factor on the
    elements follows from, or ``factors`` with an ``attention_factor``, else 1).
    Where a longrope entry has a ``short_factor`` as well, ``max_length`` says how long
    sequences get: up to ``original_max_position_embeddings`` tokens take the short
    list, longer ones the long one; without it the entry is refused.
    "dynamic" is refused: its speeds change with the length that a sequence has."""
    if rot_dim < 2 or rot_dim % 2:
        raise ValueError(f"rot_dim {rot_dim} must be even and positive")
    half = rot_dim // 2
    pair = torch.arange(half, dtype=torch.float64)
    inv = torch.as_tensor(float(base), dtype=torch.float64) ** (-2.0 * pair / rot_dim)
    kind = "default" if scaling is None else str(scaling.get("rope_type", scaling.get("type", "default"))).lower()
    if kind == "default":
        return inv, 1.0

    def need(key: str) -> float:
        if scaling.get(key) is None:
            raise ValueError(f"rope_scaling of type {kind!r} needs {key!r}")
        return float(scaling[key])

    if kind == "longrope":
        factors = _longrope_factors(scaling, max_length)
        if len(factors) != half:
            raise ValueError(f"longrope needs {half} factors, got {len(factors)}")
        inv = inv / torch.tensor([float(f) for f in factors], dtype=torch.float64)
        attention = scaling.get("attention_factor")
        if attention is None and scaling.get("factors") and scaling.get("factor") is None:
            attention = 1.0
        elif attention is None:
            factor, original = need("factor"), need("original_max_position_embeddings")
            attention = math.sqrt(1.0 + math.log(factor) / math.log(original)) if factor > 1.0 else 1.0
        return inv, float(attention)
    factor = need("factor")
    if factor < 1.0:
        raise ValueError(f"rope_scaling factor {factor} must be at least 1")
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "dynamic":
        raise ValueError("rope_scaling of type 'dynamic' changes with the sequence's length: not supported")
    original = need("original_max_position_embeddings")
    if kind == "llama3":
        low, high = need("low_freq_factor"), need("high_freq_factor")
        if high <= low:
            raise ValueError("high_freq_factor must exceed low_freq_factor")
        turns = original * inv / (2.0 * math.pi)  # turns of each pair over the original context
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        return inv * keep + inv / factor * (1.0 - keep), 1.0
    if kind == "yarn":
        fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)

        def pair_of(turns: float) -> float:  # the pair that makes so many turns over the original context
            return rot_dim * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(float(base)))

        lo, hi = pair_of(fast), pair_of(slow)
        if scaling.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rot_dim - 1)
        ramp = ((pair - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        mscale = scaling.get("attention_factor")
        if mscale is None:  # with "mscale" and "mscale_all_dim", the ratio of both
            up, down = float(scaling.get("mscale") or 1.0), float(scaling.get("mscale_all_dim") or 0.0)
            mscale = (0.1 * up * math.log(factor) + 1.0) / (0.1 * down * math.log(factor) + 1.0)
        return inv * (1.0 - ramp) + inv / factor * ramp, float(mscale)
    raise ValueError(f"unknown rope_scaling type {kind!r}")


class RotaryEmbedding:
    """Rotary positions of a merged QKV projection's q and k, in place.

    With ``qk_norm`` the per-head RMSNorm of Qwen3's q and k runs in the same
    kernel; its weights are ``q_weight`` and ``k_weight`` [head_dim]. ``max_length``:
    the longest sequence, for scalings that depend on it (``rotary_frequencies``)."""

    def __init__(self, num_q_heads: int, num_kv_heads: int, head_dim: int, rot_dim: Optional[int] = None,
                 base: float = 10000.0, scaling: Optional[Dict[str, Any]] = None, interleaved: bool = False,
                 qk_norm: bool = False, eps: float = 1e-6, max_length: Optional[int] = None) -> None:
        self.num_q_heads, self.num_kv_heads, self.head_dim = num_q_heads, num_kv_heads, head_dim
        self.interleaved, self.eps = interleaved, eps
        self._inv_freq, self.scale = rotary_frequencies(rot_dim or head_dim, base, scaling, max_length)
        self._on_device: Dict[torch.device, torch.Tensor] = {}
        self.q_weight = torch.empty(head_dim) if qk_norm else None
        self.k_weight = torch.empty(head_dim) if qk_norm else None

    def inv_freq(self, device: torch.device) -> torch.Tensor:
        t = self._on_device.get(device)
        if t is None:
            t = self._on_device[device] = self._inv_freq.to(device)
        return t

    def forward(self, qkv: torch.Tensor, positions: torch.Tensor
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """qkv [M, (Hq + 2 Hk) D] -> q [M, Hq, D], k and v [M, Hk, D]: views of qkv,
        q and k turned in place. The first call on a device copies the
        frequencies there, so make it before a graph capture."""
        Hq, Hk, D = self.num_q_heads, self.num_kv_heads, self.head_dim
        if qkv.dim() != 2 or qkv.shape[1] != (Hq + 2 * Hk) * D:
            raise ValueError(f"qkv must be [tokens, {(Hq + 2 * Hk) * D}], got {tuple(qkv.shape)}")
        q = qkv[:, : Hq * D].unflatten(1, (Hq, D))
        k = qkv[:, Hq * D : (Hq + Hk) * D].unflatten(1, (Hk, D))
        v = qkv[:, (Hq + Hk) * D :].unflatten(1, (Hk, D))
        ops.rotary(q, k, positions, self.inv_freq(qkv.device), interleaved=self.interleaved, scale=self.scale,
                   q_weight=self.q_weight, k_weight=self.k_weight, eps=self.eps, q_out=q, k_out=k)
        return q, k, v
