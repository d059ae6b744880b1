"""The norms around a block with gate and residual scale, on the GPU against the
64-bit formula. Tolerance: one rounding of the result to its type, plus what
fp32 may lose on the way: a mean of N squares summed in a tree over at most 2^14
values (relative error below 64 * 2^-24 with every rounding counted), the
reciprocal root and a dozen products, so 2^-16 of every term that enters a sum
(twice that for values past the second norm)."""

import pytest
import torch

from oracle.block_ref import gated_add_rmsnorm_ref, half_step
from sglite_b200 import ops
from sglite_b200.norm import RMSNormGated

pytestmark = pytest.mark.gpu
FP32 = 2.0 ** -16


def _check(y, h, x, r, w, eps=1e-6, **kw):
    ey, eh, b = gated_add_rmsnorm_ref(x, r, w, eps, **kw)
    off_h = FP32 * (kw.get("scale", 1.0) * b).abs() + 2.0 ** -23 * eh.abs()
    tiny = 2.0 ** -24
    assert bool(((h.double() - eh).abs() <= off_h + half_step(h.dtype) * (eh.abs() + off_h) + tiny).all())
    if w is None:
        assert y is None
        return
    wo = (w.double() + kw.get("weight_offset", 0.0)).abs()
    rms = (eh.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    # h's own error passes the norm directly and through the root of the mean square
    off_y = wo / rms * (off_h + eh.abs() / rms * off_h.pow(2).mean(-1, keepdim=True).sqrt()) + 2 * FP32 * ey.abs()
    assert bool(((y.double() - ey).abs() <= off_y + half_step(y.dtype) * (ey.abs() + off_y) + tiny).all())


def _data(M, N, dtype, res, seed, cuda):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((M, N), generator=g) * 2).to(dtype)
    r = (torch.randn((M, N), generator=g) * 3).to(res)
    w, p = (torch.rand(N, generator=g) + 0.5).to(dtype), (torch.rand(N, generator=g) - 0.5).to(dtype)
    return x.to(cuda), r.to(cuda), w.to(cuda), p.to(cuda), g


@pytest.mark.parametrize("N", [8, 264, 1024, 2056, 4096, 5120, 8192, 8200, 16384])
@pytest.mark.parametrize("M", [1, 3, 130, 700])
@pytest.mark.parametrize("dtype,res", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                       (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
def test_post_and_pre_norm_with_gate(cuda, M, N, dtype, res):
    x, r, w, p, g = _data(M, N, dtype, res, M + N, cuda)
    gate = torch.randn((M, N), generator=g).to(dtype).to(cuda)
    x0, r0 = x.clone(), r.clone()
    y, h = ops.gated_add_rmsnorm(x, r, w, 1e-6, post_weight=p, gate=gate, gate_act="sigmoid", scale=0.3,
                                 weight_offset=1.0)
    assert h.dtype == res and y.dtype == dtype and torch.equal(x, x0) and torch.equal(r, r0)
    _check(y, h, x, r, w, post_weight=p, gate=gate, gate_act="sigmoid", scale=0.3, weight_offset=1.0)


@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh", "silu"])
@pytest.mark.parametrize("kind", ["none", "channel", "row", "one", "element"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True)])
def test_gates_and_missing_norms(cuda, act, kind, post, pre):
    M, N, dtype = 37, 1032, torch.bfloat16
    x, r, w, p, g = _data(M, N, dtype, dtype, 5, cuda)
    shape = {"none": None, "channel": (N,), "row": (M, 1), "one": (1,), "element": (M, N)}[kind]
    gate = None if shape is None else (3 * torch.randn(shape, generator=g)).to(dtype).to(cuda)
    kw = dict(post_weight=p if post else None, gate=gate, gate_act=act, scale=-1.5)
    y, h = ops.gated_add_rmsnorm(x, r, w if pre else None, 1e-5, **kw)
    _check(y, h, x, r, w if pre else None, eps=1e-5, **kw)


def test_equals_the_plain_residual_norm(cuda):
    """Without a post norm, gate or scale this is fused_add_rmsnorm: the rounded
    residual is the same to the bit."""
    x, r, w, _, _ = _data(65, 4096, torch.bfloat16, torch.bfloat16, 9, cuda)
    y, h = ops.gated_add_rmsnorm(x, r, w, 1e-6)
    x2, r2 = x.clone(), r.clone()
    ops.fused_add_rmsnorm(x2, r2, w, 1e-6)
    assert torch.equal(h, r2)
    _check(y, h, x, r, w)


def test_strides_batch_dims_in_place_and_untouched_padding(cuda):
    M, N, dtype = 12, 2048, torch.float16
    x, r, w, p, g = _data(M, N, dtype, torch.float32, 3, cuda)
    gate = torch.randn((M, 1), generator=g).to(dtype).to(cuda)
    wide = torch.full((M, N + 24), 7.0, dtype=dtype, device=cuda)
    wide[:, :N] = x
    rw = torch.full((M, N + 8), 5.0, device=cuda)
    rw[:, :N] = r
    xv, rv = wide[:, :N], rw[:, :N]
    y, h = ops.gated_add_rmsnorm(xv, rv, w, 1e-6, post_weight=p, gate=gate, out=xv, residual_out=rv)
    assert y is xv and h is rv
    _check(y, h, x, r, w, post_weight=p, gate=gate)
    assert bool((wide[:, N:] == 7).all()) and bool((rw[:, N:] == 5).all())
    x3, r3 = x.view(3, 4, N), r.view(3, 4, N)
    y3, h3 = ops.gated_add_rmsnorm(x3, r3, w, 1e-6, post_weight=p, gate=gate.view(3, 4, 1))
    assert y3.shape == (3, 4, N) and torch.equal(y3.view(M, N), xv) and torch.equal(h3.view(M, N), rv)
    gwide = torch.randn((M, 2 * N), generator=g).to(dtype).to(cuda)[:, N:]  # a gate that is half of a wider product
    y, h = ops.gated_add_rmsnorm(x, r, w, 1e-6, gate=gwide, gate_act="silu")
    _check(y, h, x, r, w, gate=gwide, gate_act="silu")


def test_extreme_rows(cuda):
    """Zero rows stay finite, an infinity or NaN stays in its row, large fp16 rows
    do not overflow the fp32 sums, no rows is a no-op."""
    N = 1024
    x = torch.zeros((4, N), dtype=torch.float16, device=cuda)
    r = torch.zeros_like(x)
    x[1] = 60000.0
    x[2, 5] = float("inf")
    x[3, 7] = float("nan")
    w = torch.ones(N, dtype=torch.float16, device=cuda)
    y, h = ops.gated_add_rmsnorm(x, r, w, 1e-6, post_weight=w)
    assert bool((y[0] == 0).all()) and bool((h[0] == 0).all())
    assert bool((h[1] == 1).all()) and bool((y[1] == 1).all())
    assert bool(torch.isnan(h[2, 5])) and bool(torch.isnan(h[3]).all())
    y, h = ops.gated_add_rmsnorm(x[:0], r[:0], w, 1e-6)
    assert y.shape == (0, N) and h.shape == (0, N)


def test_layer_in_a_graph_and_on_a_side_stream(cuda):
    M, N, dtype = 5, 2560, torch.bfloat16
    x, r, w, p, g = _data(M, N, dtype, torch.float32, 21, cuda)
    layer = RMSNormGated(N, 1e-6, gate_act="tanh", scale=0.5, weight_offset=1.0)
    layer.weight, layer.post_weight = w, p
    gate = torch.randn(N, generator=g).to(dtype).to(cuda)
    xs, rs = x.clone(), r.clone()
    layer.forward(xs, rs, gate)
    kw = dict(post_weight=p, gate=gate, gate_act="tanh", scale=0.5, weight_offset=1.0)
    _check(xs, rs, x, r, w, **kw)
    want, want_r = xs.clone(), rs.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        xs.copy_(x), rs.copy_(r)
        layer.forward(xs, rs, gate)
    side.synchronize()
    assert torch.equal(xs, want) and torch.equal(rs, want_r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(xs, rs, gate)
    for _ in range(2):
        xs.copy_(x), rs.copy_(r)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(xs, want) and torch.equal(rs, want_r)
