"""PyTorch-facing wrappers of the C-ABI entry points.

Tensors stay owned by PyTorch; the library only receives raw pointers and the
current CUDA stream (the reference launches on the engine stream,
``model_executor/engine.py:50-51``). Nothing here falls back to PyTorch math.
"""

from __future__ import annotations

import ctypes
import functools
import math
import threading
from typing import Dict, Optional, Tuple

import torch

from ._lib import ARGS, FP4_ARGS, c_i64, call, check, lib

DTYPE_CODE = {torch.float16: 0, torch.bfloat16: 1}


def _p(t: Optional[torch.Tensor]):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


try:  # the raw handle without building a Stream object (~0.2 us instead of ~2 us)
    _raw_stream = torch._C._cuda_getCurrentRawStream
    _cur_device = torch._C._cuda_getDevice
except AttributeError:  # pragma: no cover - older torch
    def _raw_stream(idx: int) -> int:
        return torch.cuda.current_stream(idx).cuda_stream

    _cur_device = torch.cuda.current_device


def _dtype_code(dtype: torch.dtype) -> int:
    if dtype not in DTYPE_CODE:
        raise ValueError(f"activation dtype {dtype} not supported (float16 or bfloat16)")
    return DTYPE_CODE[dtype]


class _DeviceGuard:
    """Makes ``device`` current for the library's CUDA runtime calls."""

    def __init__(self, device: torch.device):
        self.idx = device.index if device.index is not None else torch.cuda.current_device()
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.idx:
            self.prev = cur
            torch.cuda.set_device(self.idx)

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)


def _check_cuda(*ts: torch.Tensor) -> torch.device:
    dev = ts[0].device
    for t in ts:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise ValueError("tensors must live on a CUDA device (there is no CPU path)")
        if t.device != dev:
            raise ValueError("tensors must live on the same device")
        if not t.is_contiguous():
            raise ValueError("tensors must be contiguous")
    return dev


# ---------------------------------------------------------------- repack
def blob_bytes(K: int, N: int, G: int) -> int:
    out = c_i64(0)
    call("awqb_blob_bytes", K, N, G, ctypes.byref(out))
    return out.value


def repack(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor, group_size: int) -> torch.Tensor:
    """AWQ (qweight [.., K, N/8], qzeros, scales) -> blob (uint8 [.., bytes])."""
    batched = qweight.dim() == 3
    qw = qweight if batched else qweight.unsqueeze(0)
    qz = qzeros if batched else qzeros.unsqueeze(0)
    sc = scales if batched else scales.unsqueeze(0)
    E, K, N8 = qw.shape
    N = N8 * 8
    G = K if group_size == -1 else group_size
    if qw.dtype != torch.int32 or qz.dtype != torch.int32:
        raise ValueError("qweight and qzeros must be int32")
    if sc.dtype not in DTYPE_CODE:
        raise ValueError("scales must be float16 or bfloat16")
    if qz.shape != (E, K // G, N8) or sc.shape != (E, K // G, N):
        raise ValueError(f"inconsistent AWQ shapes {tuple(qw.shape)} {tuple(qz.shape)} {tuple(sc.shape)}")
    dev = _check_cuda(qw, qz, sc)
    nb = blob_bytes(K, N, G)
    blob = torch.empty((E, nb), dtype=torch.uint8, device=dev)
    with _DeviceGuard(dev):
        call("awqb_repack", _p(qw), _p(qz), _p(sc), E, K, N, G, _p(blob), _stream(dev))
    return blob if batched else blob[0]


def unrepack(blob: torch.Tensor, K: int, N: int, G: int, scale_dtype: torch.dtype
             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    batched = blob.dim() == 2
    b = blob if batched else blob.unsqueeze(0)
    E = b.shape[0]
    dev = _check_cuda(b)
    qw = torch.empty((E, K, N // 8), dtype=torch.int32, device=dev)
    qz = torch.empty((E, K // G, N // 8), dtype=torch.int32, device=dev)
    sc = torch.empty((E, K // G, N), dtype=scale_dtype, device=dev)
    with _DeviceGuard(dev):
        call("awqb_unrepack", _p(b), E, K, N, G, _p(qw), _p(qz), _p(sc), _stream(dev))
    if not batched:
        return qw[0], qz[0], sc[0]
    return qw, qz, sc


def dequant(blob: torch.Tensor, K: int, N: int, G: int, dtype: torch.dtype) -> torch.Tensor:
    """W = (q - z) * s in ``dtype``: [.., K, N]."""
    batched = blob.dim() == 2
    b = blob if batched else blob.unsqueeze(0)
    E = b.shape[0]
    dev = _check_cuda(b)
    w = torch.empty((E, K, N), dtype=dtype, device=dev)
    with _DeviceGuard(dev):
        call("awqb_dequant", _p(b), E, K, N, G, _dtype_code(dtype), _p(w), _stream(dev))
    return w if batched else w[0]


# ---------------------------------------------------------------- workspace
class _WorkspacePool:
    """One zero-filled scratch buffer per device, grown on demand.

    The GEMM keeps its split-tile counters in the first 8 KiB of any workspace
    and leaves them at zero after every call that completes, so the buffer is
    zeroed only when it is (re)allocated; the rest is scratch shared by calls of
    every shape. A call whose bounded device wait gave up (``device_error``
    non-zero) can leave counters set: ``clear_device_error`` zeroes the counter
    region of every pool buffer together with the error word.

    One buffer serves every stream of a device, so pool-backed calls must not
    run concurrently on different streams (they would share counters and
    partial tiles); pass ``workspace=`` to give concurrent streams their own.
    Growing is refused while a CUDA graph is being captured: size it first
    (``reserve``) with the largest call.
    """

    def __init__(self):
        self._bufs: Dict[int, torch.Tensor] = {}
        self._lock = threading.Lock()

    def get(self, device: torch.device, nbytes: int) -> torch.Tensor:
        idx = device.index if device.index is not None else torch.cuda.current_device()
        buf = self._bufs.get(idx)
        if buf is not None and buf.numel() >= nbytes:
            return buf
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AWQ GEMM workspace must be reserved before CUDA graph capture")
        with self._lock:
            buf = self._bufs.get(idx)
            if buf is None or buf.numel() < nbytes:
                size = max(nbytes, 1 << 20)
                if buf is not None:
                    size = max(size, 2 * buf.numel())
                buf = torch.zeros(size, dtype=torch.uint8, device=torch.device("cuda", idx))
                self._bufs[idx] = buf
        return buf

    def reserve(self, device: torch.device, nbytes: int) -> None:
        self.get(device, nbytes)

    def reset_counters(self) -> None:
        """Zero the split-tile counter region of every buffer (on each
        device's current stream)."""
        with self._lock:
            for idx, buf in self._bufs.items():
                with torch.cuda.device(idx):
                    buf[:COUNTER_BYTES].zero_()


# Split-tile counters at the start of every GEMM workspace (two int32 per CTA,
# at most 1024 CTAs): kCounterBytes in awqb_gemm.cu.
COUNTER_BYTES = 8192

workspace_pool = _WorkspacePool()


_WS_BYTES: Dict[Tuple[int, int, int, int, int, int], int] = {}


def gemm_workspace_bytes(M: int, K: int, N: int, G: int, ntok: int = 0, ctas: int = 0) -> int:
    key = (M, K, N, G, ntok, ctas)
    v = _WS_BYTES.get(key)
    if v is None:
        out = c_i64(0)
        call("awqb_gemm_workspace_bytes_ex", M, K, N, G, ntok, ctas, ctypes.byref(out))
        v = _WS_BYTES[key] = out.value
    return v


def gemm_plan(M: int, K: int, N: int, G: int, ntok: int = 0, ctas: int = 0) -> Dict[str, int]:
    """The launch the GEMM makes for these sizes: token tile, CTAs, cluster size."""
    t, c, s = ctypes.c_int(0), c_i64(0), ctypes.c_int(0)
    call("awqb_gemm_plan", M, K, N, G, ntok, ctas, ctypes.byref(t), ctypes.byref(c), ctypes.byref(s))
    return {"ntok": t.value, "ctas": c.value, "cluster": s.value}


# ---------------------------------------------------------------- GEMM
def gemm(x: torch.Tensor, blob: torch.Tensor, K: int, N: int, G: int,
         bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
         ntok: int = 0, ctas: int = 0, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[..., N] = x[..., K] @ dequant(blob) (+ bias), fp32 accumulation."""
    if x.shape[-1] != K:
        raise ValueError(f"x has {x.shape[-1]} features, expected K={K}")
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    M = x2.shape[0]
    code = DTYPE_CODE.get(x.dtype)
    if code is None:
        raise ValueError(f"activation dtype {x.dtype} not supported (float16 or bfloat16)")
    if not (x2.is_cuda and blob.is_cuda):
        raise ValueError("tensors must live on a CUDA device (there is no CPU path)")
    di = x2.get_device()
    if blob.get_device() != di or not blob.is_contiguous():
        raise ValueError("blob must be a contiguous tensor on the activations' device")
    if bias is not None:
        if not bias.is_cuda or bias.get_device() != di or bias.dtype != x.dtype or bias.numel() != N \
                or not bias.is_contiguous():
            raise ValueError("bias must be a contiguous [N] tensor in the activation dtype on the same device")
    if out is None:
        out = torch.empty((M, N), dtype=x.dtype, device=x2.device)
    elif (out.shape[-1] != N or out.numel() != M * N or out.dtype != x.dtype or not out.is_contiguous()
          or not out.is_cuda or out.get_device() != di):
        raise ValueError("out must be a contiguous [M, N] tensor of the activation dtype on the same device")
    if M == 0:
        return out.reshape(*x.shape[:-1], N)
    if workspace is None:
        workspace = workspace_pool.get(x2.device, gemm_workspace_bytes(M, K, N, G, ntok, ctas))
    prev = _cur_device()
    if prev != di:
        torch.cuda.set_device(di)
    try:
        check(_gemm_ex()(x2.data_ptr(), M, K, N, G, code, blob.data_ptr(),
                         bias.data_ptr() if bias is not None else None, out.data_ptr(),
                         workspace.data_ptr(), workspace.numel(), ntok, ctas, _raw_stream(di)))
    finally:
        if prev != di:
            torch.cuda.set_device(prev)
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], N)


def gemv(x: torch.Tensor, blob: torch.Tensor, K: int, N: int, G: int, bias: Optional[torch.Tensor] = None,
         out: Optional[torch.Tensor] = None, features_per_cta: int = 0, warps: int = 0, ring: int = 0,
         silu_mul: bool = False) -> torch.Tensor:
    """The small-batch kernel (1 <= M <= 32) with an explicit feature slice per
    CTA and compute-warp count ((16, 16), (32, 16), (32, 8) or (64, 8); 0 =
    default) and ring depth (1..16; 0 = default). ``gemm`` takes it by itself
    for small M; this entry point exists for tuning and tests. silu_mul:
    interleaved gate/up blob, output [M, N/2]."""
    x2 = x.reshape(-1, K).contiguous()
    M = x2.shape[0]
    dev = _check_cuda(x2, blob)
    n_out = N // 2 if silu_mul else N
    if out is None:
        out = torch.empty((M, n_out), dtype=x.dtype, device=dev)
    with _DeviceGuard(dev):
        call("awqb_gemv_ex", _p(x2), M, K, N, G, _dtype_code(x.dtype), _p(blob), _p(bias), _p(out),
             int(features_per_cta), int(warps), int(ring), int(bool(silu_mul)), _stream(dev))
    return out.reshape(*x.shape[:-1], n_out)


GEMV_MAX_M = 16  # awqb_gemm takes the small-batch kernel up to this many rows


_GEMM_EX = None


def _gemm_ex():
    global _GEMM_EX
    if _GEMM_EX is None:
        _GEMM_EX = lib().awqb_gemm_ex
    return _GEMM_EX


def device_error(clear: bool = True) -> int:
    """Bits set by kernels whose bounded waits gave up (synchronises). With
    clear, a non-zero word is reset by ``clear_device_error``."""
    v = ctypes.c_uint32(0)
    call("awqb_device_error", ctypes.byref(v))
    if clear and v.value:
        clear_device_error()
    return v.value


def clear_device_error() -> None:
    """Reset the device error word and the split-tile counters of every pooled
    workspace: a GEMM that gave up waiting may have left its tile's arrival
    counters non-zero, which later calls sharing the workspace would take for
    other contributors' partials. Synchronises the device."""
    call("awqb_clear_device_error")
    workspace_pool.reset_counters()
    torch.cuda.synchronize()


def abi_version() -> int:
    return lib().awqb_abi_version()


# ---------------------------------------------------------------- MoE
def moe_topk_softmax(logits: torch.Tensor, topk: int, renormalize: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 softmax over router logits [M, E], top-k weights [M, k] and ids [M, k]."""
    lg = logits.float().contiguous()
    dev = _check_cuda(lg)
    M, E = lg.shape
    w = torch.empty((M, topk), dtype=torch.float32, device=dev)
    ids = torch.empty((M, topk), dtype=torch.int32, device=dev)
    with _DeviceGuard(dev):
        call("awqb_moe_topk_softmax", _p(lg), M, E, topk, int(bool(renormalize)), _p(w), _p(ids), _stream(dev))
    return w, ids


def moe_max_padded(numel: int, num_experts: int, block_m: int) -> int:
    return int(lib().awqb_moe_max_padded(numel, num_experts, block_m))


ALIGN_MULTI_CTA_MIN = 8192  # pairs from which the multi-CTA sort is faster (measured on B200)


def moe_align(topk_ids: torch.Tensor, e_begin: int, e_end: int, block_m: int,
              multi_cta: Optional[bool] = None):
    """Expert-sorted (token, k) ids padded per expert to block_m; returns
    (sorted_ids [max_padded], block_expert [max_padded / block_m], num_post_pad [1]).
    multi_cta: None picks by size; True / False force one of the two (identical) sorts."""
    ids = topk_ids.contiguous()
    dev = _check_cuda(ids)
    numel = ids.numel()
    maxp = moe_max_padded(numel, e_end - e_begin, block_m)
    sorted_ids = torch.empty(maxp, dtype=torch.int32, device=dev)
    block_expert = torch.empty((maxp + block_m - 1) // block_m, dtype=torch.int32, device=dev)
    npp = torch.empty(1, dtype=torch.int32, device=dev)
    if multi_cta is None:
        multi_cta = numel >= ALIGN_MULTI_CTA_MIN
    with _DeviceGuard(dev):
        if multi_cta:
            wsb = int(lib().awqb_moe_align_workspace_bytes(numel, e_end - e_begin))
            ws = torch.empty(max(wsb, 16), dtype=torch.uint8, device=dev)
            call("awqb_moe_align_ex", _p(ids), numel, e_begin, e_end, block_m, _p(sorted_ids), maxp,
                 _p(block_expert), _p(npp), _p(ws), ws.numel(), _stream(dev))
        else:
            call("awqb_moe_align", _p(ids), numel, e_begin, e_end, block_m, _p(sorted_ids), maxp,
                 _p(block_expert), _p(npp), _stream(dev))
    return sorted_ids, block_expert, npp


def moe_gather_rows(x: torch.Tensor, sorted_ids: torch.Tensor, num_post_pad: torch.Tensor, topk: int,
                    numel: int) -> torch.Tensor:
    dev = _check_cuda(x, sorted_ids, num_post_pad)
    rows = sorted_ids.numel()
    K = x.shape[-1]
    out = torch.empty((rows, K), dtype=x.dtype, device=dev)
    with _DeviceGuard(dev):
        call("awqb_moe_gather_rows", _p(x), K, _p(sorted_ids), _p(num_post_pad), numel, topk, rows, _p(out),
             _stream(dev))
    return out


def moe_grouped_gemm(x_sorted: torch.Tensor, blobs: torch.Tensor, K: int, N: int, G: int,
                     block_expert: torch.Tensor, num_post_pad: torch.Tensor, block_m: int,
                     out: torch.Tensor, row_map: Optional[torch.Tensor] = None,
                     row_scale: Optional[torch.Tensor] = None, num_valid: int = 0) -> torch.Tensor:
    """Grouped W4A16 GEMM over expert-sorted rows (blobs: [E, blob_bytes])."""
    dev = _check_cuda(x_sorted, blobs, block_expert, num_post_pad, out)
    rows = x_sorted.shape[0]
    nb = c_i64(0)
    call("awqb_moe_grouped_workspace_bytes", rows, K, N, G, block_m, ctypes.byref(nb))
    ws = workspace_pool.get(dev, nb.value)
    with _DeviceGuard(dev):
        call("awqb_moe_grouped_gemm", _p(x_sorted), rows, K, N, G, _dtype_code(x_sorted.dtype), _p(blobs),
             blobs.stride(0), _p(block_expert), _p(num_post_pad), block_m, _p(row_map), _p(row_scale),
             num_valid, _p(out), out.shape[-1], _p(ws), ws.numel(), _stream(dev))
    return out


_AWQ_SHIFT = (0, 16, 4, 20, 8, 24, 12, 28)  # bit offset of logical column i of a packed word


def _awq_unpack_cols(w: torch.Tensor) -> torch.Tensor:
    """[..., C/8] int32 in AWQ order -> [..., C] uint8 nibbles."""
    sh = torch.tensor(_AWQ_SHIFT, dtype=torch.int32, device=w.device)
    return ((w.unsqueeze(-1) >> sh) & 0xF).to(torch.uint8).reshape(*w.shape[:-1], w.shape[-1] * 8)


def _awq_pack_cols(q: torch.Tensor) -> torch.Tensor:
    """[..., C] nibbles -> [..., C/8] int32 in AWQ order."""
    sh = torch.tensor(_AWQ_SHIFT, dtype=torch.int64, device=q.device)
    w = (q.reshape(*q.shape[:-1], q.shape[-1] // 8, 8).to(torch.int64) << sh).sum(-1)
    return torch.where(w >= 2**31, w - 2**32, w).to(torch.int32)


def interleave_gate_up(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor,
                       bias: Optional[torch.Tensor] = None):
    """Reorder merged gate_up AWQ tensors ([..., K, 2I/8] packed, [..., K/G, 2I]
    scales) so that column 2j is gate column j and column 2j + 1 is up column j
    (the layout of gemm_silu_mul). Nibbles are moved, never changed: the
    dequantised weights are a column permutation of the originals."""
    two_i = scales.shape[-1]
    if two_i % 16 != 0:
        raise ValueError("fused SiLU-and-mul needs the intermediate size to be a multiple of 8")
    I = two_i // 2
    j = torch.arange(I, device=scales.device)
    cols = torch.stack([j, I + j], dim=1).reshape(-1)
    qw = _awq_pack_cols(_awq_unpack_cols(qweight).index_select(-1, cols.to(qweight.device)))
    qz = _awq_pack_cols(_awq_unpack_cols(qzeros).index_select(-1, cols.to(qzeros.device)))
    out = (qw.contiguous(), qz.contiguous(), scales.index_select(-1, cols).contiguous())
    if bias is not None:
        return out + (bias.index_select(-1, cols.to(bias.device)).contiguous(),)
    return out


def gemm_silu_mul(x: torch.Tensor, blob: torch.Tensor, K: int, N: int, G: int,
                  bias: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """silu(x @ W_gate) * (x @ W_up) -> [..., N/2] from an interleaved gate_up blob."""
    if x.shape[-1] != K:
        raise ValueError(f"x has {x.shape[-1]} features, expected K={K}")
    x2 = x.reshape(-1, K).contiguous()
    M = x2.shape[0]
    code = _dtype_code(x.dtype)
    dev = _check_cuda(x2, blob)
    if out is None:
        out = torch.empty((M, N // 2), dtype=x.dtype, device=dev)
    elif out.numel() != M * (N // 2) or out.dtype != x.dtype or not out.is_contiguous():
        raise ValueError("out must be a contiguous [M, N/2] tensor of the activation dtype")
    if M == 0:
        return out.reshape(*x.shape[:-1], N // 2)
    if M > SILU_FUSE_MAX_M:
        # Larger token tiles: the epilogue's SiLU work competes with the
        # dequantisers for issue slots (measured slower); run the GEMM and the
        # interleaved SiLU-and-mul kernel instead.
        h = gemm(x2, blob, K, N, G, bias=bias)
        return silu_and_mul(h, out=out.reshape(M, N // 2), interleaved=True).reshape(*x.shape[:-1], N // 2)
    ws = workspace_pool.get(dev, gemm_workspace_bytes(M, K, N, G))
    with _DeviceGuard(dev):
        call("awqb_gemm_silu_mul", _p(x2), M, K, N, G, code, _p(blob), _p(bias), _p(out), _p(ws), ws.numel(),
             _stream(dev))
    return out.reshape(*x.shape[:-1], N // 2)


# Largest batch (rows) for which the gate_up GEMM applies SiLU-and-mul in its
# epilogue (measured on B200: 1.04-1.36x faster up to 32 rows, slower from 64).
SILU_FUSE_MAX_M = 32


def moe_grouped_gemm_silu_mul(x_sorted: torch.Tensor, blobs: torch.Tensor, K: int, N: int, G: int,
                              block_expert: torch.Tensor, num_post_pad: torch.Tensor, block_m: int,
                              out: torch.Tensor) -> torch.Tensor:
    """Expert gate_up GEMM fused with SiLU-and-mul (interleaved w1): out [rows, N/2]."""
    dev = _check_cuda(x_sorted, blobs, block_expert, num_post_pad, out)
    rows = x_sorted.shape[0]
    nb = c_i64(0)
    call("awqb_moe_grouped_workspace_bytes", rows, K, N, G, block_m, ctypes.byref(nb))
    ws = workspace_pool.get(dev, nb.value)
    with _DeviceGuard(dev):
        call("awqb_moe_grouped_gemm_silu_mul", _p(x_sorted), rows, K, N, G, _dtype_code(x_sorted.dtype),
             _p(blobs), blobs.stride(0), _p(block_expert), _p(num_post_pad), block_m, _p(out), out.shape[-1],
             _p(ws), ws.numel(), _stream(dev))
    return out


def silu_and_mul(h: torch.Tensor, rows_dev: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, interleaved: bool = False) -> torch.Tensor:
    """silu(h[:, :I]) * h[:, I:] in fp32, rounded to h's dtype (interleaved:
    silu(h[:, 0::2]) * h[:, 1::2], the layout of an interleaved gate_up)."""
    dev = _check_cuda(h)
    rows, two_i = h.shape
    I = two_i // 2
    if out is None:
        out = torch.empty((rows, I), dtype=h.dtype, device=dev)
    with _DeviceGuard(dev):
        call("awqb_silu_and_mul_interleaved" if interleaved else "awqb_silu_and_mul", _p(h), rows, _p(rows_dev), I,
             _dtype_code(h.dtype), _p(out), _stream(dev))
    return out


def _check_device(*ts: torch.Tensor) -> torch.device:
    """Same CUDA device for all (layout is checked by the caller)."""
    dev = ts[0].device
    for t in ts:
        if t.device.type != "cuda":
            raise ValueError("tensors must live on a CUDA device (there is no CPU path)")
        if t.device != dev:
            raise ValueError("tensors must live on the same device")
    return dev


def _rows_2d(t: torch.Tensor, N: int) -> Tuple[torch.Tensor, int]:
    """[..., N] -> ([M, N] view of the same memory, row stride in elements)."""
    if t.shape[-1] != N or t.stride(-1) != 1:
        raise ValueError("the last dimension must be the contiguous feature dimension")
    if t.dim() == 2:
        t2 = t
    elif t.is_contiguous():
        t2 = t.view(-1, N)
    else:
        raise ValueError("tensors with more than 2 dimensions must be contiguous")
    return t2, (t2.stride(0) if t2.shape[0] > 1 else N)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x * rsqrt(mean(x^2) + eps) * weight over the last dimension, fp32 inside
    (flashinfer.rmsnorm semantics)."""
    N = x.shape[-1]
    if weight.numel() != N or weight.dtype != x.dtype or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [N] tensor in the activation dtype")
    dev = _check_device(x, weight)
    x2, ldx = _rows_2d(x, N)
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    o2, ldo = _rows_2d(out, N)
    with _DeviceGuard(dev):
        call("awqb_rmsnorm", _p(x2), _p(weight), _p(o2), x2.shape[0], N, ldx, ldo, float(eps),
             _dtype_code(x.dtype), _stream(dev))
    return out


def fused_add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float) -> None:
    """In place: residual += x; x = rmsnorm(residual) * weight, the norm taken
    over the fp32 sum (flashinfer.fused_add_rmsnorm semantics)."""
    N = x.shape[-1]
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise ValueError("residual must have the shape and dtype of x")
    if weight.numel() != N or weight.dtype != x.dtype or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous [N] tensor in the activation dtype")
    dev = _check_device(x, residual, weight)
    x2, ldx = _rows_2d(x, N)
    r2, ldr = _rows_2d(residual, N)
    with _DeviceGuard(dev):
        call("awqb_fused_add_rmsnorm", _p(x2), _p(r2), _p(weight), x2.shape[0], N, ldx, ldr, float(eps),
             _dtype_code(x.dtype), _stream(dev))


def moe_topk_sum(y3: torch.Tensor, M: int, topk: int, topk_ids: Optional[torch.Tensor], e_begin: int,
                 e_end: int, out: torch.Tensor) -> torch.Tensor:
    """out[m] = the sum of y3's rows m * topk .. m * topk + topk - 1; with topk_ids (int32
    [M, topk]) only of those whose expert is in [e_begin, e_end)."""
    ids = None if topk_ids is None else topk_ids.contiguous()
    if ids is not None and (ids.dtype != torch.int32 or ids.numel() != M * topk):
        raise ValueError(f"topk_ids must be an int32 [{M}, {topk}] tensor")
    dev = _check_cuda(y3, out, ids)
    H = y3.shape[-1]
    with _DeviceGuard(dev):
        call("awqb_moe_topk_sum", _p(y3), M, topk, H, _p(ids), e_begin, e_end, _dtype_code(y3.dtype),
             _p(out), _stream(dev))
    return out


# ---------------------------------------------------------------- around the projections
# These run once per block and token, for single tokens too, so their host side is
# kept short: one look at each tensor, one packed structure, one call.
_FN: Dict[str, object] = {}


def _entry(name: str):
    """(C function, packer of its argument structure)."""
    fn = _FN.get(name)
    if fn is None:
        layout = ARGS.get(name) or FP4_ARGS.get(name)
        fn = _FN[name] = (getattr(lib(), name), layout.pack if layout else None)
    return fn


def _run(fn, device_index: int, *args) -> None:
    """Call ``fn`` with ``device_index`` current and that device's stream last."""
    prev = _cur_device()
    if prev == device_index:
        status = fn(*args, _raw_stream(device_index))
    else:
        torch.cuda.set_device(device_index)
        try:
            status = fn(*args, _raw_stream(device_index))
        finally:
            torch.cuda.set_device(prev)
    if status:
        check(status)


def _device_of(t: torch.Tensor) -> int:
    di = t.get_device()
    if di < 0:
        raise ValueError("tensors must live on a CUDA device (there is no CPU path)")
    return di


def _wrong_device(name: str):
    return ValueError(f"{name} must live on the same CUDA device as the other tensors")


def _row_stride(t: torch.Tensor, n: int, name: str) -> int:
    """Stride between the rows of t [.., n] seen as [rows, n] (elements)."""
    if t.is_contiguous():
        return n
    s = t.stride()
    if s[-1] != 1 or t.dim() != 2:
        raise ValueError(f"{name} must have contiguous rows, and be contiguous with more than 2 dimensions")
    return s[0] if t.shape[0] > 1 else n


GATE_ACTIVATIONS = {"none": 0, "sigmoid": 1, "tanh": 2, "silu": 3}


def _gate_strides(gate: torch.Tensor, x: torch.Tensor, n: int) -> Tuple[int, int]:
    """(row, feature) strides of a gate that broadcasts over x [.., n]."""
    shape = gate.shape
    wide = len(shape) > 0 and shape[-1] == n
    if not wide and len(shape) > 0 and shape[-1] != 1:
        raise ValueError(f"gate {tuple(shape)} does not broadcast over x {tuple(x.shape)}")
    rows = math.prod(shape[:-1])
    if rows != 1 and shape[:-1] != x.shape[:-1]:
        raise ValueError(f"gate {tuple(shape)} does not broadcast over x {tuple(x.shape)}")
    if wide and gate.stride(-1) != 1:
        raise ValueError("the gate's last dimension must be the contiguous feature dimension")
    if rows <= 1:
        return 0, int(wide)
    if len(shape) == 2:
        return gate.stride(0), int(wide)
    if not gate.is_contiguous():
        raise ValueError("a gate with more than 2 dimensions must be contiguous")
    # from the shape: a contiguous tensor's dimensions of one may have any stride
    return shape[-1], int(wide)


def gated_add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor], eps: float, *,
                      post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                      gate_act: str = "none", scale: float = 1.0, weight_offset: float = 0.0,
                      out: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None
                      ) -> Tuple[Optional[torch.Tensor], torch.Tensor]:
    """The norms around a block with its gate and residual scale:
    ``b = rmsnorm(x) * (weight_offset + post_weight)`` (or x without post_weight),
    ``h = residual + scale * gate_act(gate) * b`` and
    ``y = rmsnorm(h) * (weight_offset + weight)``, fp32 inside, the second norm over
    the unrounded h. Returns (y, h); y is None without ``weight``.

    gate broadcasts over x: the shape of x, [N] or [1, N] (per channel), [.., 1]
    (per row) or one value. residual is of x's dtype or float32. ``out`` may be x
    and ``residual_out`` may be residual (in place)."""
    dtype, shape = x.dtype, x.shape
    code = _dtype_code(dtype)
    di = _device_of(x)
    N = shape[-1]
    wide = residual.dtype == torch.float32
    if residual.shape != shape or (not wide and residual.dtype != dtype):
        raise ValueError("residual must have the shape of x and its dtype or float32")
    if residual.get_device() != di:
        raise _wrong_device("residual")
    pw = pp = pg = po = ldo = gate_row = gate_col = 0
    if weight is not None:
        if weight.numel() != N or weight.dtype != dtype or not weight.is_contiguous():
            raise ValueError("weight must be a contiguous [N] tensor in the activation dtype")
        if weight.get_device() != di:
            raise _wrong_device("weight")
        pw = weight.data_ptr()
    if post_weight is not None:
        if post_weight.numel() != N or post_weight.dtype != dtype or not post_weight.is_contiguous():
            raise ValueError("post_weight must be a contiguous [N] tensor in the activation dtype")
        if post_weight.get_device() != di:
            raise _wrong_device("post_weight")
        pp = post_weight.data_ptr()
    act = GATE_ACTIVATIONS.get(gate_act)
    if act is None:
        raise ValueError(f"gate activation {gate_act!r}: one of {tuple(GATE_ACTIVATIONS)}")
    if gate is not None:
        if gate.dtype != dtype:
            raise ValueError("gate must have the activation dtype")
        if gate.get_device() != di:
            raise _wrong_device("gate")
        gate_row, gate_col = _gate_strides(gate, x, N)
        pg = gate.data_ptr()
    ldx, ldr = _row_stride(x, N, "x"), _row_stride(residual, N, "residual")
    if weight is not None:
        if out is None:
            out = torch.empty_like(x)  # (padded rows give a contiguous result)
        elif out.shape != shape or out.dtype != dtype or out.get_device() != di:
            raise ValueError("out must have the shape, dtype and device of x")
        po, ldo = out.data_ptr(), _row_stride(out, N, "out")
    elif out is not None:
        raise ValueError("out is the second norm's result: it needs weight")
    if residual_out is None:
        residual_out = torch.empty_like(residual)
    elif residual_out.shape != shape or residual_out.dtype != residual.dtype or residual_out.get_device() != di:
        raise ValueError("residual_out must have the shape, dtype and device of residual")
    fn, pack = _entry("awqb_gated_add_rmsnorm")
    _run(fn, di, pack(x.data_ptr(), ldx, residual.data_ptr(), ldr, wide, pp, pg, gate_row, gate_col, act, scale, pw,
                      weight_offset, po, ldo, residual_out.data_ptr(), _row_stride(residual_out, N, "residual_out"),
                      x.numel() // N if N else 0, N, eps, code))
    return out, residual_out


_HEADS_NOT_CONTIGUOUS = "the head dimension must be contiguous"


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, *,
           interleaved: bool = False, scale: float = 1.0, q_weight: Optional[torch.Tensor] = None,
           k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotary positions of q [M, Hq, D] and k [M, Hk, D] (slices of the merged QKV
    output will do: token and head strides are multiples of 8), after the per-head RMSNorm when
    q_weight / k_weight [D] are given. positions [M] int32 or int64; inv_freq
    float64 [rot_dim / 2] (``rotary.RotaryEmbedding`` makes it, long-context
    scalings included); the first rot_dim elements of a head turn, in pairs
    (j, j + rot_dim / 2) or, interleaved, (2j, 2j + 1). ``scale`` multiplies the
    turned elements. Tokens with a negative position are padding: their
    outputs are left as they were. ``q_out`` / ``k_out`` may be q / k (in place)."""
    dtype = q.dtype
    code = _dtype_code(dtype)
    di = _device_of(q)
    if q.dim() != 3:
        raise ValueError("q must be a [tokens, heads, head_dim] tensor")
    M, Hq, D = q.shape
    long = positions.dtype == torch.int64
    if positions.shape != (M,) or not (long or positions.dtype == torch.int32) or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32 or int64 [tokens] tensor")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 [rot_dim / 2] tensor")
    if positions.get_device() != di or inv_freq.get_device() != di:
        raise _wrong_device("positions and inv_freq")
    q0, q1, q2 = q.stride()
    if q_out is None:
        q_out = q.new_empty((M, Hq, D))
        o0, o1, o2 = Hq * D, D, 1
    elif q_out.shape != q.shape or q_out.dtype != dtype or q_out.get_device() != di:
        raise ValueError("q_out must have the shape, dtype and device of q")
    else:
        o0, o1, o2 = q_out.stride()
    if q2 != 1 or o2 != 1:
        raise ValueError(_HEADS_NOT_CONTIGUOUS)
    Hk = kp = ko = k0 = k1 = ko0 = ko1 = wq = wk = 0
    if k is not None:
        if k.dim() != 3 or k.shape[0] != M or k.shape[2] != D or k.dtype != dtype or k.get_device() != di:
            raise ValueError("k must be a [tokens, heads, head_dim] tensor with q's tokens, head_dim, dtype and device")
        Hk = k.shape[1]
        k0, k1, k2 = k.stride()
        if k_out is None:
            k_out = q.new_empty((M, Hk, D))
            ko0, ko1, ko2 = Hk * D, D, 1
        elif k_out.shape != k.shape or k_out.dtype != dtype or k_out.get_device() != di:
            raise ValueError("k_out must have the shape, dtype and device of k")
        else:
            ko0, ko1, ko2 = k_out.stride()
        if k2 != 1 or ko2 != 1:
            raise ValueError(_HEADS_NOT_CONTIGUOUS)
        kp, ko = k.data_ptr(), k_out.data_ptr()
        if Hk == 1:
            k1 = ko1 = 0
    elif k_out is not None or k_weight is not None:
        raise ValueError("k_out and k_weight need k")
    if M == 1:  # a dimension of one has no stride
        q0 = o0 = k0 = ko0 = 0
    if Hq == 1:
        q1 = o1 = 0
    if q_weight is not None:
        if q_weight.numel() != D or q_weight.dtype != dtype or not q_weight.is_contiguous() \
                or q_weight.get_device() != di:
            raise ValueError("q_weight must be a contiguous [head_dim] tensor in q's dtype on its device")
        wq = q_weight.data_ptr()
    if k_weight is not None:
        if k_weight.numel() != D or k_weight.dtype != dtype or not k_weight.is_contiguous() \
                or k_weight.get_device() != di:
            raise ValueError("k_weight must be a contiguous [head_dim] tensor in q's dtype on its device")
        wk = k_weight.data_ptr()
    fn, pack = _entry("awqb_rotary")
    _run(fn, di, pack(q.data_ptr(), q0, q1, Hq, kp, k0, k1, Hk, positions.data_ptr(), long, inv_freq.data_ptr(),
                      2 * inv_freq.numel(), D, M, interleaved, scale, wq, wk, eps, q_out.data_ptr(), o0, o1, ko, ko0,
                      ko1, code))
    return q_out, k_out


def group_rows(ids: torch.Tensor, num_groups: int, begin: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Stable grouping of rows by id: (order [n], offsets [num_groups + 1]), int32.
    ``order[offsets[g]:offsets[g + 1]]`` are the indices whose id is begin + g, in
    index order; indices whose id is in no group come last."""
    di = _device_of(ids)
    if ids.dtype != torch.int32 or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous int32 tensor")
    n = ids.numel()
    order = torch.empty(n, dtype=torch.int32, device=ids.device)
    offsets = torch.empty(max(num_groups, 0) + 1, dtype=torch.int32, device=ids.device)
    nb = int(lib().awqb_group_rows_workspace_bytes(n, num_groups))
    ws = torch.empty(nb, dtype=torch.uint8, device=ids.device) if nb > 0 else None
    _run(_entry("awqb_group_rows")[0], di, ids.data_ptr(), n, begin, num_groups, order.data_ptr(), offsets.data_ptr(),
         None if ws is None else ws.data_ptr(), nb)
    return order, offsets


def _row_map_scale(row_map: Optional[torch.Tensor], row_scale: Optional[torch.Tensor], rows: int, out_rows: int,
                   di: int) -> Tuple[int, int]:
    """Pointers of a grouped product's row_map and row_scale, checked."""
    pm = ps = 0
    if row_map is not None:
        if row_map.dtype != torch.int32 or row_map.numel() != rows or not row_map.is_contiguous() \
                or row_map.get_device() != di:
            raise ValueError("row_map must be a contiguous int32 [rows] tensor on x's device")
        pm = row_map.data_ptr()
    if row_scale is not None:
        if row_scale.dtype != torch.float32 or row_scale.numel() != out_rows or not row_scale.is_contiguous() \
                or row_scale.get_device() != di:
            raise ValueError("row_scale must be a contiguous float32 tensor on x's device, one value per row of out")
        ps = row_scale.data_ptr()
    return pm, ps


def grouped_gemm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *, out: Optional[torch.Tensor] = None,
                 silu_mul: bool = False, row_map: Optional[torch.Tensor] = None,
                 row_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Matrix products grouped by expert over 16-bit weights w [E, N, K]:
    ``y[r] = x[r] @ w[e].T`` for ``offsets[e] <= r < offsets[e + 1]``, fp32
    accumulation; with silu_mul, w holds the gate rows and then the up rows and
    ``y = silu(gate) * up`` [.., N / 2]. offsets [E + 1] int32 stays on the device
    and must not decrease.

    y[r] goes to row r of ``out``, or to row row_map[r] (int32 [rows]; no two rows to
    one; rows that map outside ``out`` are dropped), times row_scale[its row of out] (fp32) if
    given. Rows of ``out`` that nothing goes to are left as they were; without
    ``out`` a new [rows, N] tensor is returned, in which those rows are undefined."""
    dtype = x.dtype
    code = _dtype_code(dtype)
    di = _device_of(x)
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2]:
        raise ValueError(f"x {tuple(x.shape)} and w {tuple(w.shape)} must be [rows, K] and [experts, N, K]")
    if w.dtype != dtype or not w.is_contiguous() or w.get_device() != di:
        raise ValueError("w must be contiguous, of x's dtype and on its device")
    rows, K = x.shape
    E, N, _ = w.shape
    if offsets.dtype != torch.int32 or offsets.numel() != E + 1 or not offsets.is_contiguous() \
            or offsets.get_device() != di:
        raise ValueError("offsets must be a contiguous int32 [experts + 1] tensor on x's device")
    n_out = N // 2 if silu_mul else N
    if out is None:
        out = x.new_empty((rows, n_out))
    elif out.dim() != 2 or out.shape[1] != n_out or out.dtype != dtype or out.get_device() != di:
        raise ValueError(f"out must be a [rows, {n_out}] tensor of x's dtype on its device")
    out_rows = out.shape[0]
    pm, ps = _row_map_scale(row_map, row_scale, rows, out_rows, di)
    fn, pack = _entry("awqb_grouped_gemm")
    _run(fn, di, pack(x.data_ptr(), rows, _row_stride(x, K, "x"), w.data_ptr(), E, K, N, offsets.data_ptr(), code,
                      silu_mul, pm, ps, out.data_ptr(), out_rows, _row_stride(out, n_out, "out")))
    return out


@functools.lru_cache(maxsize=1024)  # a call asks for the same few sizes in every step
def _lora_workspace_bytes(M: int, K: int, N: int, L: int, rank: int, parts: int) -> int:
    v = c_i64(0)
    call("awqb_lora_workspace_bytes", M, K, N, L, rank, parts, ctypes.byref(v))
    return v.value


def lora(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, order: torch.Tensor, offsets: torch.Tensor,
         base: torch.Tensor, *, slices: Optional[Tuple[int, ...]] = None, scales: Optional[torch.Tensor] = None,
         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Low-rank adapters of many requests beside a shared projection:
    ``out[t] = base[t] + scales[l] * (x[t] @ a[l].T) @ b[l].T`` for the rows t that
    use adapter l, ``out[t] = base[t]`` for rows without one. x [M, K]; base [M, N]
    is the projection's output; ``order``, ``offsets`` are ``group_rows`` of the
    rows' adapter numbers (one call serves every projection of a step).

    slices: widths of a merged projection's parts (QKV, gate_up; at most 4), each with
    its own pair; a [L, len(slices) * rank, K] stacks their first factors, b
    [L, N, rank] the second ones. Sums are fp32. ``out`` may be base (in place); it must
    not overlap the inputs otherwise."""
    dtype = x.dtype
    code = _dtype_code(dtype)
    di = _device_of(x)
    if x.dim() != 2 or a.dim() != 3 or b.dim() != 3 or base.dim() != 2:
        raise ValueError("x [M, K], a [L, slices * rank, K], b [L, N, rank] and base [M, N] are wanted")
    M, K = x.shape
    L, N, rank = b.shape
    parts = 1 if slices is None else len(slices)
    if not 1 <= parts <= 4:
        raise ValueError(f"{parts} slices: 1..4 are supported")
    if a.shape != (L, parts * rank, K) or base.shape != (M, N):
        raise ValueError(f"inconsistent shapes: x {tuple(x.shape)}, a {tuple(a.shape)}, b {tuple(b.shape)}, "
                         f"base {tuple(base.shape)}, {parts} slices")
    if a.dtype != dtype or b.dtype != dtype or base.dtype != dtype or not a.is_contiguous() or not b.is_contiguous():
        raise ValueError("a, b and base must be of x's dtype, a and b contiguous")
    if a.get_device() != di or b.get_device() != di or base.get_device() != di or order.get_device() != di \
            or offsets.get_device() != di:
        raise _wrong_device("a, b, base, order and offsets")
    if order.dtype != torch.int32 or order.numel() != M or not order.is_contiguous():
        raise ValueError("order must be a contiguous int32 [M] tensor")
    if offsets.dtype != torch.int32 or offsets.numel() != L + 1 or not offsets.is_contiguous():
        raise ValueError("offsets must be a contiguous int32 [adapters + 1] tensor")
    ps = 0
    if scales is not None:
        if scales.dtype != torch.float32 or scales.numel() != L or not scales.is_contiguous() \
                or scales.get_device() != di:
            raise ValueError("scales must be a contiguous float32 [adapters] tensor on x's device")
        ps = scales.data_ptr()
    if out is None:
        out = x.new_empty((M, N))
    elif out.shape != (M, N) or out.dtype != dtype or out.get_device() != di:
        raise ValueError("out must have the shape, dtype and device of base")
    nb = _lora_workspace_bytes(M, K, N, L, rank, parts)
    # from the caching allocator: private to the stream, or to the graph being captured
    ws = x.new_empty((nb + 1) // 2)  # (x's values have two bytes)
    w = ((N,) if slices is None else tuple(slices)) + (0, 0, 0, 0)
    fn, pack = _entry("awqb_lora")
    _run(fn, di, pack(x.data_ptr(), M, _row_stride(x, K, "x"), K, a.data_ptr(), b.data_ptr(), L, rank, N, parts, w[0], w[1],
                      w[2], w[3], order.data_ptr(), offsets.data_ptr(), ps, base.data_ptr(),
                      _row_stride(base, N, "base"), out.data_ptr(), _row_stride(out, N, "out"), code, ws.data_ptr(), nb))
    return out


# ---------------------------------------------------------------- microscaled 4-bit floating point
# Values of a block of 4-bit numbers, codes of the formats and their blocks.
FP4_FORMATS = {"nvfp4": 0, "mxfp4": 1}
FP4_BLOCK = {"nvfp4": 16, "mxfp4": 32}


_FP4_CODE = {(fmt, dtype): (f, d) for fmt, f in FP4_FORMATS.items() for dtype, d in DTYPE_CODE.items()}


def _fp4_format(fmt: str) -> int:
    code = FP4_FORMATS.get(fmt)
    if code is None:
        raise ValueError(f"4-bit format {fmt!r}: one of {tuple(FP4_FORMATS)}")
    return code


def _fp4_code(fmt: str, dtype: torch.dtype) -> Tuple[int, int]:
    """The library's codes of a format and a 16-bit dtype."""
    both = _FP4_CODE.get((fmt, dtype))
    return both if both is not None else (_fp4_format(fmt), _dtype_code(dtype))


def _fp4_x(x: torch.Tensor) -> Tuple[int, int]:
    """(rows, K) of x [.., K]."""
    shape = x.shape
    if len(shape) == 2:
        return shape
    if not shape:
        raise ValueError("x must have rows of K values")
    return (x.numel() // shape[-1] if shape[-1] else 0), shape[-1]


def _fp4_scale(scale: torch.Tensor, n: int, fmt: str, di: int, name: str) -> int:
    """Pointer of an fp32 scale of n values."""
    if fmt != "nvfp4":
        raise ValueError(f"{name}: only nvfp4 has a scale beside its blocks' scales")
    if scale.dtype != torch.float32 or scale.numel() != n or not scale.is_contiguous() or scale.get_device() != di:
        raise ValueError(f"{name} must be a contiguous float32 [{n}] tensor on the same device")
    return scale.data_ptr()


def fp4_rows_empty(rows: int, K: int, fmt: str, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """Room for ``rows`` quantised rows of K values: codes uint8 [rows, K / 2] and scales
    uint8 [granules, rows, 16], 16 scales of a row side by side (256 k of nvfp4, 512 of mxfp4)."""
    _fp4_format(fmt)
    return _fp4_rows_new(torch.empty(0, dtype=torch.uint8, device=device), rows, K, fmt)


def _fp4_rows_new(like: torch.Tensor, rows: int, K: int, fmt: str) -> Tuple[torch.Tensor, torch.Tensor]:
    codes = like.new_empty(rows, K // 2, dtype=torch.uint8)  # (sizes one by one: half a microsecond less)
    return codes, codes.new_empty(-(-K // (16 * FP4_BLOCK[fmt])), rows, 16)


def _fp4_rows(codes: torch.Tensor, scales: torch.Tensor, fmt: str, di: int) -> Tuple[int, int]:
    """(rows, K) of quantised rows, checked."""
    shape = codes.shape
    if len(shape) != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous() or codes.get_device() != di:
        raise ValueError("codes must be a contiguous uint8 [rows, K / 2] CUDA tensor")
    rows, half = shape
    if scales.shape != (-(-half // (8 * FP4_BLOCK[fmt])), rows, 16) or scales.dtype != torch.uint8 \
            or not scales.is_contiguous() or scales.get_device() != di:
        raise ValueError(f"scales {tuple(scales.shape)} must be the contiguous uint8 [granules, rows, 16] tensor of "
                         f"{rows} {fmt} rows of K={2 * half}, on the codes' device")
    return rows, 2 * half


def fp4_quantize(x: torch.Tensor, fmt: str, *, scale: Optional[torch.Tensor] = None,
                 index: Optional[torch.Tensor] = None, per_row: int = 1, count: Optional[torch.Tensor] = None,
                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of x [.., K] (fp16 or bf16, K a multiple of 32) in 4 bits: (codes, scales), as
    ``fp4_rows_empty`` shapes them. fmt "nvfp4": blocks of 16 with an e4m3 scale each, and
    ``scale`` (fp32 [1], positive; 1 without) for all: a code stands for code * block
    scale * scale. "mxfp4": blocks of 32 with a power of two each. Roundings to nearest,
    ties to even; what is too large saturates; a block that holds an infinity or a NaN gets
    the scale NaN.

    index (int32 [rows]): row r is x's row index[r] // per_row (an expert-sorted list of
    (token, choice) pairs, with per_row choices a token); rows whose index is outside x, and
    rows from ``count`` (int32 [1], on the device) on, are left as they were."""
    fc, code = _fp4_code(fmt, x.dtype)
    di = _device_of(x)
    rows, K = _fp4_x(x)
    rows_in, pi, pc = rows, 0, 0
    if index is not None:
        if index.dtype != torch.int32 or index.dim() != 1 or not index.is_contiguous() or index.get_device() != di:
            raise ValueError("index must be a contiguous int32 [rows] tensor on x's device")
        pi, rows = index.data_ptr(), index.numel()
    elif per_row != 1:
        raise ValueError("per_row needs an index")
    if count is not None:
        if count.dtype != torch.int32 or count.numel() != 1 or count.get_device() != di:
            raise ValueError("count must be an int32 [1] tensor on x's device")
        pc = count.data_ptr()
    ps = 0 if scale is None else _fp4_scale(scale, 1, fmt, di, "scale")
    if out is None:
        out = _fp4_rows_new(x, rows, K, fmt)
    elif _fp4_rows(out[0], out[1], fmt, di) != (rows, K):
        raise ValueError(f"out must hold {rows} rows of K={K}")
    fn, pack = _entry("awqb_fp4_quantize")
    _run(fn, di, pack(x.data_ptr(), rows_in, _row_stride(x, K, "x"), K, fc, code, ps, pi, per_row, pc, rows,
                      out[0].data_ptr(), out[1].data_ptr()))
    return out


def fp4_dequantize(codes: torch.Tensor, scales: torch.Tensor, fmt: str, dtype: torch.dtype, *,
                   scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values [rows, K] that quantised rows stand for, rounded to ``dtype``."""
    fc, code = _fp4_code(fmt, dtype)
    di = _device_of(codes)
    rows, K = _fp4_rows(codes, scales, fmt, di)
    ps = 0 if scale is None else _fp4_scale(scale, 1, fmt, di, "scale")
    if out is None:
        out = codes.new_empty(rows, K, dtype=dtype)
        ldo = K
    elif out.shape != (rows, K) or out.dtype != dtype or out.get_device() != di:
        raise ValueError(f"out must be a [{rows}, {K}] tensor of {dtype} on the codes' device")
    else:
        ldo = _row_stride(out, K, "out")
    fn, pack = _entry("awqb_fp4_dequantize")
    _run(fn, di, pack(codes.data_ptr(), scales.data_ptr(), rows, K, fc, code, ps, out.data_ptr(), ldo))
    return out


def fp4_add_rmsnorm(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float, fmt: str, *,
                    scale: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None,
                    out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                    ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The residual-add RMSNorm in front of a 4-bit projection: h = x + residual,
    y = h * rsqrt(mean(h^2) + eps) * weight, quantised as ``fp4_quantize`` does, straight
    from fp32, for rows of any finite size (a row with an infinity: finite values over it are 0);
    eps is taken as fp32. Returns (codes, scales, h), h rounded to x's dtype; without a residual h is x.
    ``residual_out`` may be residual (in place) or x. K is at most 16384."""
    dtype = x.dtype
    fc, code = _fp4_code(fmt, dtype)
    di = _device_of(x)
    rows, K = _fp4_x(x)
    if weight.numel() != K or weight.dtype != dtype or not weight.is_contiguous() or weight.get_device() != di:
        raise ValueError("weight must be a contiguous [K] tensor in the activation dtype on x's device")
    pr = po = ldr = ldo = 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != dtype or residual.get_device() != di:
            raise ValueError("residual must have the shape, dtype and device of x")
        if residual_out is None:
            residual_out = torch.empty_like(residual)  # (padded rows give a contiguous result)
        elif residual_out.shape != x.shape or residual_out.dtype != dtype or residual_out.get_device() != di:
            raise ValueError("residual_out must have the shape, dtype and device of residual")
        pr, ldr = residual.data_ptr(), _row_stride(residual, K, "residual")
        po, ldo = residual_out.data_ptr(), _row_stride(residual_out, K, "residual_out")
    elif residual_out is not None:
        raise ValueError("residual_out needs residual")
    ps = 0 if scale is None else _fp4_scale(scale, 1, fmt, di, "scale")
    if out is None:
        out = _fp4_rows_new(x, rows, K, fmt)
    elif _fp4_rows(out[0], out[1], fmt, di) != (rows, K):
        raise ValueError(f"out must hold {rows} rows of K={K}")
    fn, pack = _entry("awqb_fp4_add_rmsnorm")
    _run(fn, di, pack(x.data_ptr(), _row_stride(x, K, "x"), pr, ldr, weight.data_ptr(), po, ldo, rows, K, eps, fc, code,
                      ps, out[0].data_ptr(), out[1].data_ptr()))
    return out[0], out[1], (x if residual is None else residual_out)


def fp4_lay_out_scales(scales: torch.Tensor, fmt: str) -> torch.Tensor:
    """A weight's block scales [.., N, K / 16 (nvfp4) or K / 32 (mxfp4)], as bytes in the
    order of a checkpoint, laid out for the tensor cores (once, at load): uint8
    [.., ceil(N / 128), ceil(K / 256), 4 or 2, 32, 4, 4], tiles of 128 rows by four scales,
    rows r, r + 32, r + 64 and r + 96 of a tile side by side, zero past N and K."""
    _fp4_format(fmt)
    if scales.dim() < 2 or scales.element_size() != 1:
        raise ValueError("scales must be one-byte values [.., N, K / block]")
    s = scales.view(torch.uint8)
    lead, (N, n) = s.shape[:-2], s.shape[-2:]
    per = 256 // FP4_BLOCK[fmt]  # scales of a stage of 256 k
    s = torch.nn.functional.pad(s, (0, -n % per, 0, -N % 128))
    s = s.reshape(*lead, s.shape[-2] // 128, 4, 32, s.shape[-1] // per, per // 4, 4)
    d = len(lead)
    return s.permute(*range(d), d, d + 3, d + 4, d + 2, d + 1, d + 5).contiguous()


def fp4_interleave_gate_up(t: torch.Tensor, dim: int = -2) -> torch.Tensor:
    """A merged gate_up tensor's rows (the gate's, then the up's; weight codes, block scales in
    the order of a checkpoint, or with dim=-1 a bias) by turns, as ``silu_mul`` wants them."""
    n = t.shape[dim]
    if n % 2:
        raise ValueError(f"{n} rows are not a gate's and an up's")
    turn = torch.arange(n, device=t.device).view(2, n // 2).t().reshape(-1)
    return t.index_select(dim, turn)


def _fp4_weight(w: torch.Tensor, w_scales: torch.Tensor, lead: Tuple[int, ...], N: int, K: int, fmt: str, di: int) -> None:
    """Checks quantised weights [*lead, N, K / 2] and their laid-out scales."""
    if w.dtype != torch.uint8 or not w.is_contiguous() or w.get_device() != di:
        raise ValueError("w must be a contiguous uint8 [.., N, K / 2] tensor on the rows' device")
    want = (*lead, -(-N // 128), -(-K // 256), 64 // FP4_BLOCK[fmt], 32, 4, 4)
    if w_scales.shape != want or w_scales.dtype != torch.uint8 or not w_scales.is_contiguous() \
            or w_scales.get_device() != di:
        raise ValueError(f"w_scales {tuple(w_scales.shape)} must be {want}: fp4_lay_out_scales of the weight's scales")


def fp4_gemm(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, fmt: str,
             dtype: torch.dtype, *, x_scale: Optional[torch.Tensor] = None, w_scale: Optional[torch.Tensor] = None,
             bias: Optional[torch.Tensor] = None, silu_mul: bool = False, out: Optional[torch.Tensor] = None
             ) -> torch.Tensor:
    """y = x @ w.T (+ bias) of quantised rows (codes, scales) and a quantised weight w uint8
    [N, K / 2] with ``fp4_lay_out_scales``'s w_scales, both of format fmt, fp32 sums,
    rounded to ``dtype``; x_scale, w_scale: their fp32 [1] scales (nvfp4). silu_mul: w's
    rows (and bias) are gate and up by turns, y = silu(gate) * up [rows, N / 2]."""
    fc, code = _fp4_code(fmt, dtype)
    di = _device_of(codes)
    rows, K = _fp4_rows(codes, scales, fmt, di)
    shape = w.shape
    if len(shape) != 2 or 2 * shape[1] != K:
        raise ValueError(f"w {tuple(shape)} must be a [N, K / 2] tensor, K={K}")
    N = shape[0]
    _fp4_weight(w, w_scales, (), N, K, fmt, di)
    pb = px = pw = 0
    if bias is not None:
        if bias.dtype != dtype or bias.numel() != N or not bias.is_contiguous() or bias.get_device() != di:
            raise ValueError(f"bias must be a contiguous [{N}] tensor of {dtype} on the rows' device")
        pb = bias.data_ptr()
    if x_scale is not None:
        px = _fp4_scale(x_scale, 1, fmt, di, "x_scale")
    if w_scale is not None:
        pw = _fp4_scale(w_scale, 1, fmt, di, "w_scale")
    ldo = n_out = N // 2 if silu_mul else N
    if out is None:
        out = codes.new_empty(rows, n_out, dtype=dtype)
    elif out.shape != (rows, n_out) or out.dtype != dtype or out.get_device() != di:
        raise ValueError(f"out must be a [{rows}, {n_out}] tensor of {dtype} on the rows' device")
    else:
        ldo = _row_stride(out, n_out, "out")
    fn, pack = _entry("awqb_fp4_gemm")
    _run(fn, di, pack(codes.data_ptr(), scales.data_ptr(), rows, K, w.data_ptr(), w_scales.data_ptr(), 1, N, 0, fc, code,
                      px, pw, pb, silu_mul, 0, 0, out.data_ptr(), rows, ldo))
    return out


def fp4_grouped_gemm(codes: torch.Tensor, scales: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
                     offsets: torch.Tensor, fmt: str, dtype: torch.dtype, *, x_scale: Optional[torch.Tensor] = None,
                     w_scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, silu_mul: bool = False,
                     row_map: Optional[torch.Tensor] = None, row_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``fp4_gemm`` grouped by expert: ``y[r] = x[r] @ w[e].T`` for ``offsets[e] <= r <
    offsets[e + 1]``, w uint8 [E, N, K / 2], w_scale fp32 [E] (nvfp4). offsets, out,
    row_map and row_scale as in ``grouped_gemm``; with silu_mul w's rows are gate and up
    by turns."""
    fc, code = _fp4_code(fmt, dtype)
    di = _device_of(codes)
    rows, K = _fp4_rows(codes, scales, fmt, di)
    if w.dim() != 3 or 2 * w.size(2) != K:
        raise ValueError(f"w {tuple(w.shape)} must be a [E, N, K / 2] tensor, K={K}")
    E, N, _ = w.shape
    _fp4_weight(w, w_scales, (E,), N, K, fmt, di)
    px = 0 if x_scale is None else _fp4_scale(x_scale, 1, fmt, di, "x_scale")
    pw = 0 if w_scale is None else _fp4_scale(w_scale, E, fmt, di, "w_scale")
    if offsets.dtype != torch.int32 or offsets.numel() != E + 1 or not offsets.is_contiguous() \
            or offsets.get_device() != di:
        raise ValueError("offsets must be a contiguous int32 [experts + 1] tensor on the rows' device")
    n_out = N // 2 if silu_mul else N
    if out is None:
        out = codes.new_empty(rows, n_out, dtype=dtype)
    elif out.dim() != 2 or out.shape[1] != n_out or out.dtype != dtype or out.get_device() != di:
        raise ValueError(f"out must be a [rows, {n_out}] tensor of {dtype} on the rows' device")
    out_rows = out.shape[0]
    pm, ps = _row_map_scale(row_map, row_scale, rows, out_rows, di)
    fn, pack = _entry("awqb_fp4_gemm")
    _run(fn, di, pack(codes.data_ptr(), scales.data_ptr(), rows, K, w.data_ptr(), w_scales.data_ptr(), E, N,
                      offsets.data_ptr(), fc, code, px, pw, 0, silu_mul, pm, ps, out.data_ptr(), out_rows,
                      _row_stride(out, n_out, "out")))
    return out
