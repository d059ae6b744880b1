"""RMSNorm layers over the library's kernels, with the interface of the
reference's ``srt/model_executor/layers/norm.py:10-47`` (``RMSNorm``,
``RMSNormFused``), and ``RMSNormGated`` for blocks with norms on both sides, a
gate or a residual scale. After a row-parallel projection whose all-reduce is fused
into the GEMM (``distributed.PeerExchange.gemm_allreduce``), the residual add
and the norm run as one more kernel, launched so that it overlaps the GEMM's
tail (programmatic dependent launch)."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ops


class RMSNorm:
    """RMSNorm over the last dimension (``norm.py:10-25``)."""

    def __init__(self, size: int, eps: float) -> None:
        self.eps = eps
        self.weight = torch.empty(size)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return ops.rmsnorm(x, self.weight, self.eps)

    def forward_inplace(self, x: torch.Tensor) -> None:
        ops.rmsnorm(x, self.weight, self.eps, out=x)


class RMSNormFused:
    """RMSNorm with the residual add fused in (``norm.py:28-47``)."""

    def __init__(self, size: int, eps: float) -> None:
        self.eps = eps
        self.weight = torch.empty(size)

    def forward(self, x: torch.Tensor,
                residual: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Without a residual: (rmsnorm(x), x). With one: residual += x and
        x = rmsnorm(residual), both in place; returns (x, residual)."""
        if residual is None:
            return ops.rmsnorm(x, self.weight, self.eps), x
        ops.fused_add_rmsnorm(x, residual, self.weight, self.eps)
        return x, residual


class RMSNormGated:
    """The norms around a block with its gate and residual scale, between one
    block's output projection and the next block's input: the optional norm
    after the block (``post_weight``), the gate, the scaled residual add and the
    norm before the next block (``weight``), in one kernel. Extends
    ``RMSNormFused`` (``norm.py:28-47``) to blocks that are normed on both sides,
    gated, or scaled; ``weight_offset`` is 1 for checkpoints that store their
    norm weights minus one."""

    def __init__(self, size: int, eps: float, post_norm: bool = True, gate_act: str = "none", scale: float = 1.0,
                 weight_offset: float = 0.0) -> None:
        self.eps = eps
        self.gate_act, self.scale, self.weight_offset = gate_act, scale, weight_offset
        self.weight = torch.empty(size)
        self.post_weight = torch.empty(size) if post_norm else None

    def forward(self, x: torch.Tensor, residual: torch.Tensor,
                gate: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(x, residual) updated in place: residual += scale * gate_act(gate) *
        rmsnorm(x), x = rmsnorm(residual). residual may be float32."""
        return ops.gated_add_rmsnorm(x, residual, self.weight, self.eps, post_weight=self.post_weight, gate=gate,
                                     gate_act=self.gate_act, scale=self.scale, weight_offset=self.weight_offset,
                                     out=x, residual_out=residual)
