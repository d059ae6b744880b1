"""64-bit restatements, from their formulas, of the operators around the
projections (test infrastructure): gated norms, rotary positions, products
grouped by expert, low-rank adapters. Each returns the exact result and, for
the products, a bound on what fp32 accumulation may be off by."""

from __future__ import annotations

import torch

U32 = 2.0 ** -23  # an fp32 addition, rounded or truncated


def half_step(dtype: torch.dtype) -> float:
    """What one rounding to ``dtype`` is off by at most, relative to the value."""
    return torch.finfo(dtype).eps / 2


def act_ref(t, name):
    return {"none": t, "sigmoid": t.sigmoid(), "tanh": t.tanh(), "silu": t * t.sigmoid()}[name]


def gated_add_rmsnorm_ref(x, residual, weight, eps, post_weight=None, gate=None, gate_act="none", scale=1.0,
                          weight_offset=0.0):
    b = x.double()
    if post_weight is not None:
        b = b / (b.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (post_weight.double() + weight_offset)
    if gate is not None:
        b = b * act_ref(gate.double(), gate_act)
    h = residual.double() + scale * b
    if weight is None:
        return None, h, b
    y = h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * (weight.double() + weight_offset)
    return y, h, b


def rotary_ref(v, positions, inv_freq, interleaved, scale, weight=None, eps=1e-6):
    """v [M, H, D]; returns the turned heads (padding tokens as if at position 0)."""
    half = inv_freq.numel()
    rot = 2 * half
    v = v.double().clone()
    if weight is not None:
        v = v / (v.pow(2).mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    angle = positions.clamp_min(0).double()[:, None] * inv_freq
    c, s = scale * angle.cos()[:, None], scale * angle.sin()[:, None]
    out = v.clone()
    i0 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i1 = i0 + 1 if interleaved else i0 + half
    out[..., i0] = v[..., i0] * c - v[..., i1] * s
    out[..., i1] = v[..., i0] * s + v[..., i1] * c
    assert rot <= v.shape[-1]
    return out


def grouped_gemm_ref(x, w, offsets, silu_mul=False):
    """(y, bound) per row of x; rows in no group are NaN. The bound is on fp32
    accumulation alone: K additions, each off by at most U32 of the sum of
    magnitudes so far."""
    E, N, K = w.shape
    n_out = N // 2 if silu_mul else N
    y = torch.full((x.shape[0], n_out), float("nan"), dtype=torch.float64, device=x.device)
    bound = torch.zeros_like(y)
    for e in range(E):
        r0, r1 = int(offsets[e]), int(offsets[e + 1])
        xe, we = x[r0:r1].double(), w[e].double()
        p, mag = xe @ we.T, (K * U32) * (xe.abs() @ we.abs().T)
        if silu_mul:
            g, u = p[:, :n_out], p[:, n_out:]
            dg, du = mag[:, :n_out], mag[:, n_out:]
            act = g * g.sigmoid()
            # |silu'| <= 1.1; the exponential, the division and two products in fp32: 8 units
            bound[r0:r1] = 1.1 * dg * (u.abs() + du) + act.abs() * du + 8 * U32 * (act * u).abs()
            p = act * u
        else:
            bound[r0:r1] = mag
        y[r0:r1] = p
    return y, bound


def lora_ref(x, a, b, ids, base, slices, scales=None, halves_eps=0.0):
    """(out, bound); ids[t] is row t's adapter (outside 0..L-1: none). halves_eps is
    what a value of the first product may be off by, relatively, when it enters
    the second one."""
    L, N, r = b.shape
    K = x.shape[1]
    out = base.double().clone()
    bound = U32 * out.abs()
    for l in range(L):
        rows = (ids == l).nonzero(as_tuple=True)[0]
        if not rows.numel():
            continue
        xe, al = x[rows].double(), a[l].double()
        h, mag = xe @ al.T, xe.abs() @ al.abs().T
        s = 1.0 if scales is None else float(scales[l])
        n0 = 0
        for i, width in enumerate(slices):
            hs, ms, bl = h[:, i * r:(i + 1) * r], mag[:, i * r:(i + 1) * r], b[l, n0:n0 + width].double()
            d = hs @ bl.T
            out[rows, n0:n0 + width] += s * d
            off = (ms * (K * U32)) @ bl.abs().T + (hs.abs() * (r * U32 + halves_eps)) @ bl.abs().T
            bound[rows, n0:n0 + width] += abs(s) * off + 4 * U32 * (abs(s) * d.abs() + out[rows, n0:n0 + width].abs())
            n0 += width
    return out, bound


def within(got, exact, bound, dtype):
    """Largest excess of |got - exact| over the bound plus one rounding to dtype
    (of a value that is itself off by the bound)."""
    tiny = float(torch.finfo(dtype).tiny) if dtype != torch.float16 else 2.0 ** -24  # steps near zero
    room = bound + half_step(dtype) * (exact.abs() + bound) + tiny
    return float(((got.double() - exact).abs() - room).max()) if got.numel() else -1.0
