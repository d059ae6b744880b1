"""Low-rank adapters of many requests beside a shared AWQ projection.

``LoraAdapters`` holds the adapters of one projection as the kernel reads them;
``LoraBatch`` says which rows of a step's batch use which adapter and serves every
projection of the step. ``AWQB200LinearMethod.apply_weights`` and the
tensor-parallel layers take both and add the adapters' products to the
projection's output in place."""

from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple

import torch

from . import ops


@dataclass
class LoraBatch:
    """The rows of a batch grouped by adapter (``ops.group_rows``)."""

    order: torch.Tensor    # int32 [M]: rows of adapter 0, of adapter 1, ..., then rows without one
    offsets: torch.Tensor  # int32 [adapters + 1]

    @classmethod
    def from_ids(cls, adapter_ids: torch.Tensor, num_adapters: int) -> "LoraBatch":
        """adapter_ids int32 [M]: each row's adapter, or a negative number for none."""
        return cls(*ops.group_rows(adapter_ids, num_adapters))


@dataclass
class LoraAdapters:
    """The adapters of one projection: a [L, slices * rank, K], b [L, N, rank], scales [L]."""

    a: torch.Tensor
    b: torch.Tensor
    scales: Optional[torch.Tensor] = None
    slices: Optional[Tuple[int, ...]] = None

    @classmethod
    def stack(cls, adapters: Sequence[Sequence[Optional[Tuple[torch.Tensor, torch.Tensor]]]],
              slices: Sequence[int], scales: Optional[Sequence[float]] = None) -> "LoraAdapters":
        """adapters[l][s] = (A [r, K], B [slices[s], r]) of adapter l on slice s, or
        None where it leaves the slice alone; ranks may differ and are padded
        with zeros to the largest one (a multiple of 8), which changes no sum."""
        pairs = [p for ad in adapters for p in ad if p is not None]
        if not pairs:
            raise ValueError("no adapter has a factor")
        if any(len(ad) != len(slices) for ad in adapters):
            raise ValueError(f"every adapter needs {len(slices)} slices")
        K, like = pairs[0][0].shape[1], pairs[0][0]
        rank = (max(A.shape[0] for A, _ in pairs) + 7) // 8 * 8
        a = torch.zeros((len(adapters), len(slices), rank, K), dtype=like.dtype, device=like.device)
        b = torch.zeros((len(adapters), sum(slices), rank), dtype=like.dtype, device=like.device)
        for l, ad in enumerate(adapters):
            at = 0
            for s, (pair, width) in enumerate(zip(ad, slices)):
                if pair is not None:
                    A, B = pair
                    if A.shape[1] != K or tuple(B.shape) != (width, A.shape[0]):
                        raise ValueError(f"adapter {l}, slice {s}: A {tuple(A.shape)} and B {tuple(B.shape)} do not "
                                         f"match K={K} and width {width}")
                    a[l, s, : A.shape[0]] = A
                    b[l, at : at + width, : A.shape[0]] = B
                at += width
        sc = None if scales is None else torch.tensor([float(v) for v in scales], dtype=torch.float32,
                                                      device=like.device)
        return cls(a.flatten(1, 2), b, sc, tuple(int(w) for w in slices))

    def shard(self, parallel: str, rank: int, world: int) -> "LoraAdapters":
        """This rank's part beside a tensor-parallel projection: "column" keeps the
        first factor and cuts every slice's outputs, "row" cuts the first
        factor's inputs (the ranks' products add up in the all-reduce)."""
        if parallel == "row":
            if self.a.shape[2] % world:
                raise ValueError(f"{self.a.shape[2]} inputs do not split over {world} ranks")
            return LoraAdapters(self.a.chunk(world, dim=2)[rank].contiguous(), self.b, self.scales, self.slices)
        if parallel != "column":
            raise ValueError(parallel)
        widths = self.slices or (self.b.shape[1],)
        if any(w % world for w in widths):
            raise ValueError(f"slices {widths} do not split over {world} ranks")
        parts: List[torch.Tensor] = [p.chunk(world, dim=1)[rank] for p in self.b.split(list(widths), dim=1)]
        return LoraAdapters(self.a, torch.cat(parts, dim=1).contiguous(), self.scales, tuple(w // world for w in widths))

    def add_to(self, y: torch.Tensor, x: torch.Tensor, batch: LoraBatch) -> torch.Tensor:
        """y += the adapters' products of x, in place; y [.., N] contiguous, x [.., K]."""
        y2 = y.view(-1, y.shape[-1])
        ops.lora(x.reshape(-1, x.shape[-1]), self.a, self.b, batch.order, batch.offsets, y2, slices=self.slices,
                 scales=self.scales, out=y2)
        return y
