"""The operators around the projections run together, as a decoder block runs
them: norm, merged QKV projection with adapters, rotary positions, (attention
stands in as the mean of v over each key/value head's queries), output projection
with adapters, gated norms, 16-bit experts; eagerly and replayed from a graph."""

import pytest
import torch

from oracle.awq_ref import rel_err
from oracle.block_ref import gated_add_rmsnorm_ref, lora_ref, rotary_ref
from sglite_b200 import ops
from sglite_b200.lora import LoraAdapters, LoraBatch
from sglite_b200.moe import AWQB200MoeBackend
from sglite_b200.norm import RMSNormGated
from sglite_b200.quantization import AWQB200Config
from sglite_b200.rotary import RotaryEmbedding
from sglite_b200.synthetic import make_awq_weights
from sglite_b200.tp import ColumnParallelAWQLinear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 13, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_block(cuda, M, dtype):
    H, Hq, Hk, D, E, I, topk, L, r = 512, 8, 2, 64, 8, 128, 2, 4, 16
    g = torch.Generator(device=cuda).manual_seed(M)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=cuda) * std).to(dtype)

    def linear(k, n, widths, seed):
        layer = ColumnParallelAWQLinear(AWQB200Config(4, 128, True).get_linear_method(), k, n)
        w = make_awq_weights(k, n, 128, dtype, seed=seed)
        w["scales"] = w["scales"] * 0.25
        layer.load({key: w[key].to(cuda) for key in ("qweight", "qzeros", "scales")})
        layer.adapters = LoraAdapters(normal(L, len(widths) * r, k, std=k ** -0.5), normal(L, n, r, std=r ** -0.5),
                                      torch.rand(L, generator=g, device=cuda), widths)
        return layer

    widths = (Hq * D, Hk * D, Hk * D)
    qkv_proj, o_proj = linear(H, sum(widths), widths, 1), linear(Hq * D, H, (H,), 2)
    rope = RotaryEmbedding(Hq, Hk, D, base=1e6, qk_norm=True)
    rope.q_weight, rope.k_weight = 1 + normal(D, std=0.1), 1 + normal(D, std=0.1)
    norm = RMSNormGated(H, 1e-6, gate_act="sigmoid", scale=0.7, weight_offset=1.0)
    norm.weight, norm.post_weight = normal(H, std=0.1), normal(H, std=0.1)
    gate = normal(H)
    w1, w2 = normal(E, 2 * I, H, std=H ** -0.5), normal(E, H, I, std=I ** -0.5)
    router = normal(E, H, std=H ** -0.5)
    backend = AWQB200MoeBackend()
    x, residual = normal(M, H), torch.randn((M, H), generator=g, device=cuda)
    ids = torch.randint(-1, L, (M,), generator=g, device=cuda).to(torch.int32)
    pos = torch.randint(0, 100000, (M,), generator=g, device=cuda)

    def attend(v):
        return v.repeat_interleave(Hq // Hk, dim=1).reshape(M, Hq * D).contiguous()

    def block(x, residual):
        batch = LoraBatch.from_ids(ids, L)
        qkv = qkv_proj.forward(x, batch)
        q, k, v = rope.forward(qkv, pos)
        o = o_proj.forward(attend(v), batch)
        y, res = norm.forward(o, residual.clone(), gate)
        z = backend.forward(y.clone(), w1, w2, y.float() @ router.float().T, topk, True)
        return q, k, y, res, z

    got = block(x, residual)
    # each step against its formula on the step's own inputs (rel_err's bound is that of the GEMM tests)
    plain = qkv_proj.forward(x)
    qkv, _ = lora_ref(x, qkv_proj.adapters.a, qkv_proj.adapters.b, ids, plain, widths, qkv_proj.adapters.scales)
    inv = rope.inv_freq(cuda)
    q = rotary_ref(qkv[:, :Hq * D].reshape(M, Hq, D), pos, inv, False, 1.0, rope.q_weight)
    k = rotary_ref(qkv[:, Hq * D:(Hq + Hk) * D].reshape(M, Hk, D), pos, inv, False, 1.0, rope.k_weight)
    assert rel_err(got[0], q.float().cpu()) <= 1e-2 and rel_err(got[1], k.float().cpu()) <= 1e-2
    a_in = attend(qkv[:, (Hq + Hk) * D:].reshape(M, Hk, D)).to(dtype)
    o, _ = lora_ref(a_in, o_proj.adapters.a, o_proj.adapters.b, ids, o_proj.forward(a_in), (H,), o_proj.adapters.scales)
    y, res, _ = gated_add_rmsnorm_ref(o, residual, norm.weight, 1e-6, norm.post_weight, gate, "sigmoid", 0.7, 1.0)
    assert rel_err(got[2], y.float().cpu()) <= 1e-2 and rel_err(got[3], res.float().cpu()) <= 1e-2
    yk = got[2]
    tw, te = ops.moe_topk_softmax(yk.float() @ router.float().T, topk, True)
    z = torch.zeros((M, H), device=cuda)
    for j in range(topk):
        e = te[:, j].long()
        h = torch.bmm(w1[e].float(), yk.float()[..., None])[..., 0]
        h = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
        z += tw[:, j, None] * torch.bmm(w2[e].float(), h[..., None])[..., 0]
    assert rel_err(got[4], z.cpu()) <= 1e-2

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = block(x, residual)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, got))
    x.copy_(normal(M, H))  # new inputs through the same graph
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, block(x, residual)))
    assert ops.device_error() == 0


def test_offsets_past_32_bits(cuda):
    """Rows 16 MB apart, the last ones more than 2^32 elements behind the first: the
    bits are those of contiguous rows."""
    M, apart, dtype = 600, (1 << 23) + 64, torch.bfloat16
    room = torch.empty(M * apart, dtype=dtype, device=cuda).view(M, apart)
    g = torch.Generator(device=cuda).manual_seed(7)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=cuda) * std).to(dtype)

    def far(t, at):
        v = room[:, at:at + t.shape[1]]
        v.copy_(t)
        return v

    x = normal(M, 1024)
    fx = far(x, 0)
    for E, silu in ((2, False), (2, True), (32, False), (32, True)):  # many and few rows per expert
        w = normal(E, 256, 1024, std=1 / 32)
        order, offsets = ops.group_rows(torch.randint(0, E, (M,), generator=g, device=cuda).to(torch.int32), E)
        want = ops.grouped_gemm(x, w, offsets, silu_mul=silu, row_map=order)
        out = far(torch.zeros_like(want), 4096)
        ops.grouped_gemm(fx, w, offsets, silu_mul=silu, row_map=order, out=out)
        assert torch.equal(out, want)
    ids = torch.randint(-1, 3, (M,), generator=g, device=cuda).to(torch.int32)
    order, offsets = ops.group_rows(ids, 3)
    for N in (512, 16384):  # decode and prompt kernels
        a, b, base = normal(3, 64, 1024, std=1 / 32), normal(3, N, 64, std=1 / 8), normal(M, N)
        want = ops.lora(x, a, b, order, offsets, base)
        held = far(base, 4096)
        ops.lora(fx, a, b, order, offsets, held, out=held)
        assert torch.equal(held, want)
    r, gate, w = normal(M, 1024), normal(M, 1024), normal(1024)
    y, h = ops.gated_add_rmsnorm(x, r, w, 1e-6, post_weight=w, gate=gate, gate_act="silu")
    fr = far(r, 2048)
    out = ops.gated_add_rmsnorm(fx, fr, w, 1e-6, post_weight=w, gate=far(gate, 4096), gate_act="silu", out=fx,
                                residual_out=fr)
    assert torch.equal(out[0], y) and torch.equal(out[1], h)
    pos = torch.randint(0, 100000, (M,), generator=g, device=cuda)
    for rot in (128, 64, 20):  # vectors, part of the head, element by element
        inv = RotaryEmbedding(8, 2, 128, rot_dim=rot).inv_freq(cuda)
        q = normal(M, 1024)
        want, _ = ops.rotary(q.view(M, 8, 128), None, pos, inv)
        fq = far(q, 0).unflatten(1, (8, 128))
        ops.rotary(fq, None, pos, inv, q_out=fq)
        assert torch.equal(fq, want)
    assert ops.device_error() == 0
