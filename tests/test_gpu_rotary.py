"""Rotary positions (with the per-head q/k norm) on the GPU against the 64-bit
formula. Tolerance: one rounding to the type, plus fp32: the norm's sum and root
(2^-18, at most 256 squares), the sine and cosine and three products (2^-20 of
the pair's magnitude), so 2^-17 of |a| + |b| of each pair."""

import pytest
import torch

from oracle.block_ref import half_step, rotary_ref
from sglite_b200 import ops
from sglite_b200.rotary import RotaryEmbedding, rotary_frequencies

pytestmark = pytest.mark.gpu


def _ok(got, v, pos, inv, inter, scale, w=None, eps=1e-6):
    want = rotary_ref(v, pos, inv, inter, scale, w, eps)
    # magnitude of each element's pair: turn by an angle cannot exceed |a| + |b|
    n = rotary_ref(v, torch.zeros_like(pos), inv, inter, 1.0, w, eps).abs()
    half = inv.numel()
    i0 = torch.arange(half) * 2 if inter else torch.arange(half)
    i1 = i0 + 1 if inter else i0 + half
    mag = n.clone()
    mag[..., i0] = mag[..., i1] = scale * (n[..., i0] + n[..., i1])
    off = 2.0 ** -17 * mag
    room = off + half_step(got.dtype) * (want.abs() + off) + 2.0 ** -24
    live = pos >= 0
    assert bool(((got.double() - want).abs() <= room)[live].all())


def _inv(rot, cuda):
    return rotary_frequencies(rot, 500000.0)[0].to(cuda)


@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 64), (80, 80), (80, 40), (96, 96), (192, 64), (256, 256),
                                   (128, 20), (64, 2), (8, 8), (256, 16), (40, 24)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layouts(cuda, D, rot, interleaved, norm, dtype):
    g = torch.Generator().manual_seed(D + rot)
    for M, Hq, Hk in ((1, 32, 8), (77, 5, 1), (300, 8, 2)):
        q = torch.randn((M, Hq, D), generator=g).to(dtype).to(cuda)
        k = torch.randn((M, Hk, D), generator=g).to(dtype).to(cuda)
        pos = torch.randint(0, 40000, (M,), generator=g).to(cuda)
        qw, kw = ((torch.rand(D, generator=g) + 0.5).to(dtype).to(cuda) if norm else None for _ in range(2))
        inv = _inv(rot, cuda)
        q1, k1 = ops.rotary(q, k, pos, inv, interleaved=interleaved, scale=1.25, q_weight=qw, k_weight=kw)
        _ok(q1, q, pos, inv, interleaved, 1.25, qw)
        _ok(k1, k, pos, inv, interleaved, 1.25, kw)
        if not norm:  # what is not turned passes unchanged
            assert torch.equal(q1[..., rot:], q[..., rot:]) and torch.equal(k1[..., rot:], k[..., rot:])


@pytest.mark.parametrize("M,Hq,Hk,D,rot,interleaved,norm", [
    (2600, 40, 8, 128, 128, False, True), (2401, 33, 1, 128, 64, True, True), (5000, 7, 3, 80, 80, False, False),
    (700, 64, 8, 64, 32, False, True), (2500, 1, 1, 256, 256, False, True), (2369, 128, 16, 16, 16, True, False)])
def test_many_tokens(cuda, M, Hq, Hk, D, rot, interleaved, norm):
    """Whole tokens and batches of heads per warp, heads that do not fill a batch,
    padding among them."""
    g = torch.Generator(device=cuda).manual_seed(M)
    dtype = torch.bfloat16
    q = torch.randn((M, Hq, D), generator=g, device=cuda).to(dtype)
    k = torch.randn((M, Hk, D), generator=g, device=cuda).to(dtype)
    pos = torch.randint(-200, 100000, (M,), generator=g, device=cuda)
    qw = (torch.rand(D, generator=g, device=cuda) + 0.5).to(dtype) if norm else None
    inv = _inv(rot, cuda)
    q_out, k_out = torch.full_like(q, 3.0), torch.full_like(k, 3.0)
    ops.rotary(q, k, pos, inv, interleaved=interleaved, scale=0.75, q_weight=qw, q_out=q_out, k_out=k_out)
    _ok(q_out, q, pos, inv, interleaved, 0.75, qw)
    _ok(k_out, k, pos, inv, interleaved, 0.75)  # q alone is normed
    assert bool((q_out[pos < 0] == 3).all()) and bool((k_out[pos < 0] == 3).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_merged_projection_in_place_padding_and_position_types(cuda, dtype):
    M, Hq, Hk, D = 65, 16, 2, 128
    g = torch.Generator().manual_seed(1)
    qkv0 = torch.randn((M, (Hq + 2 * Hk) * D), generator=g).to(dtype).to(cuda)
    pos = torch.randint(0, 1 << 20, (M,), generator=g).to(cuda)
    pos[::7] = -1  # padding tokens
    layer = RotaryEmbedding(Hq, Hk, D, base=1e6, qk_norm=True,
                            scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768})
    layer.q_weight = (torch.rand(D, generator=g) + 0.5).to(dtype).to(cuda)
    layer.k_weight = (torch.rand(D, generator=g) + 0.5).to(dtype).to(cuda)
    results = []
    for p in (pos, pos.to(torch.int32)):
        qkv = qkv0.clone()
        q, k, v = layer.forward(qkv, p)
        assert q.data_ptr() == qkv.data_ptr() and v.shape == (M, Hk, D)
        results.append(qkv)
    assert torch.equal(results[0], results[1])
    q0 = qkv0[:, :Hq * D].view(M, Hq, D)
    inv = layer.inv_freq(cuda)
    _ok(q, q0, pos, inv, False, layer.scale, layer.q_weight)
    _ok(k, qkv0[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D)), pos, inv, False, layer.scale, layer.k_weight)
    assert torch.equal(qkv[:, (Hq + Hk) * D:], qkv0[:, (Hq + Hk) * D:])  # v
    assert torch.equal(qkv[::7], qkv0[::7])                              # padding


@pytest.mark.parametrize("pos", [0, 1, 4097, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, 1 << 35])
def test_far_positions_keep_their_angle(cuda, pos):
    """The angle is reduced in 64 bits: its error is 2^-52 of the position's turns
    (below 2^-18 of a turn even at 2^35, but 2^-24 up to 2^29), not 2^-24 of them."""
    g = torch.Generator().manual_seed(2)
    q = torch.randn((3, 2, 128), generator=g, dtype=torch.float32).to(torch.float16).to(cuda)
    p = torch.tensor([pos, pos, 0], dtype=torch.int64, device=cuda)
    inv = _inv(128, cuda)
    q1, none = ops.rotary(q, None, p, inv)
    assert none is None
    _ok(q1, q, p, inv, False, 1.0)


def test_head_major_views_and_outputs(cuda):
    """[H, M, D] tensors and strided outputs, seen as [M, H, D]."""
    M, H, D, dtype = 33, 6, 64, torch.bfloat16
    g = torch.Generator().manual_seed(4)
    base = torch.randn((H, M, D), generator=g).to(dtype).to(cuda)
    q = base.transpose(0, 1)
    pos = torch.arange(M, device=cuda)
    inv = _inv(64, cuda)
    q_out = torch.zeros((M, H, D + 16), dtype=dtype, device=cuda)
    got, _ = ops.rotary(q, None, pos, inv, q_out=q_out[..., :D])
    _ok(got, q, pos, inv, False, 1.0)
    assert int(torch.count_nonzero(q_out[..., D:])) == 0
    want = got.clone()
    ops.rotary(q, None, pos, inv, q_out=q)
    assert torch.equal(q, want)
    e, _ = ops.rotary(q[:0], None, pos[:0], inv)
    assert e.shape == (0, H, D)


def test_graph_replay_with_new_positions(cuda):
    M, H, D, dtype = 9, 8, 128, torch.bfloat16
    g = torch.Generator().manual_seed(6)
    q = torch.randn((M, H, D), generator=g).to(dtype).to(cuda)
    pos = torch.arange(M, device=cuda)
    inv = _inv(D, cuda)
    out, _ = ops.rotary(q, None, pos, inv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary(q, None, pos, inv, q_out=out)
    for shift in (5, 1000):
        pos.add_(shift)
        graph.replay()
        torch.cuda.synchronize()
        _ok(out, q, pos, inv, False, 1.0)
