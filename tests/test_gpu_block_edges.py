"""The operators around the projections on the GPU, at the edges of what their
documentation allows: layouts, streams, sizes and values that the operators' own
files do not reach. Bounds are those of ``oracle/block_ref.py`` unless a test derives its own."""

import pytest
import torch

from oracle.awq_ref import rel_err
from oracle.block_ref import gated_add_rmsnorm_ref, half_step, lora_ref, within
from sglite_b200 import ops
from sglite_b200.lora import LoraAdapters, LoraBatch
from sglite_b200.moe import AWQB200MoeBackend, DenseExpertWeights
from sglite_b200.quantization import AWQB200Config
from sglite_b200.synthetic import make_awq_weights
from sglite_b200.tp import RowParallelAWQLinear, shard_awq

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("B", [4, 33])
def test_gate_with_a_dimension_of_one(cuda, wide, B):
    """A decode step's [B, 1, N]: a gate made by turning [1, B, N] is contiguous, and its
    middle stride says nothing. The bits are those of the gate's own copy."""
    N, dtype = 512, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(B)
    x, r = (torch.randn((B, 1, N), generator=g, device=cuda).to(dtype) for _ in range(2))
    w = torch.rand(N, generator=g, device=cuda).to(dtype)
    gate = torch.randn((1, B, N if wide else 1), generator=g, device=cuda).to(dtype).transpose(0, 1)
    assert gate.is_contiguous() and gate.stride(1) == B * (N if wide else 1)
    y, h = ops.gated_add_rmsnorm(x, r, w, 1e-6, gate=gate, gate_act="sigmoid")
    y2, h2 = ops.gated_add_rmsnorm(x.view(B, N), r.view(B, N), w, 1e-6, gate=gate.clone().view(B, -1), gate_act="sigmoid")
    assert torch.equal(y.view(B, N), y2) and torch.equal(h.view(B, N), h2)
    ey, eh, b = gated_add_rmsnorm_ref(x, r, w, 1e-6, gate=gate, gate_act="sigmoid")
    # one rounding, and fp32's on the way (each of a few operations at most 2^-16 of a term)
    off = 2.0 ** -16 * (b.abs() + eh.abs())
    assert bool(((h.double() - eh).abs() <= off + half_step(dtype) * (eh.abs() + off)).all())


@pytest.mark.parametrize("rank", [64, 128])  # two tiles of base per group of warps, or one
@pytest.mark.parametrize("in_place", [False, True])
def test_prompt_adapters_add_to_the_base_of_this_call(cuda, rank, in_place):
    """Every element of base is its own and differs from call to call, and the adapters'
    products are known to the bit (powers of two), so a base read before it has
    arrived, from an earlier block or call, shows."""
    M, K, N, L, dtype = 1500, 64, 9000, 3, torch.bfloat16
    assert M * (N * (50 + rank) + K * rank) > 8e8  # the prompt kernels
    g = torch.Generator(device=cuda).manual_seed(rank)
    x = torch.zeros((M, K), dtype=dtype, device=cuda)
    x[:, 0] = 1
    a = torch.zeros((L, rank, K), dtype=dtype, device=cuda)
    a[:, 0, 0] = torch.tensor([1.0, 2.0, 4.0], device=cuda)
    b = torch.zeros((L, N, rank), dtype=dtype, device=cuda)
    b[:, :, 0] = 1
    ids = torch.randint(0, L, (M,), generator=g, device=cuda).to(torch.int32)
    order, offsets = ops.group_rows(ids, L)
    add = 2.0 ** ids[:, None].float()
    for _ in range(20):
        base = torch.randint(-100, 101, (M, N), generator=g, device=cuda).to(dtype)  # exact, also with 4 more
        want = (base.float() + add).to(dtype)
        got = ops.lora(x, a, b, order, offsets, base, out=base if in_place else None)
        assert torch.equal(got, want)
    assert ops.device_error() == 0


@pytest.mark.parametrize("layout", ["columns", "broadcast"])
def test_dense_experts_take_ids_and_weights_of_any_layout(cuda, layout):
    """Ids and weights that are the first columns of a wider ranking, or one row for all
    tokens: the bits are those of their contiguous copies."""
    M, E, H, I, topk, dtype = 37, 8, 128, 64, 3, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn((M, H), generator=g, device=cuda).to(dtype)
    w1 = DenseExpertWeights((torch.randn((E // 2, 2 * I, H), generator=g, device=cuda) / 11).to(dtype), 2, E)
    w2 = DenseExpertWeights((torch.randn((E // 2, H, I), generator=g, device=cuda) / 8).to(dtype), 2, E)
    tw = torch.rand((M, E), generator=g, device=cuda)
    if layout == "columns":
        tw, ids = (t[:, :topk] for t in tw.sort(dim=1, descending=True))
        ids = ids.to(torch.int32)
        ids = torch.cat([ids, torch.full_like(ids, 7)], dim=1)[:, :topk]
    else:
        ids = torch.tensor([[5, 0, 3]], dtype=torch.int32, device=cuda).expand(M, topk)
        tw = tw[:1, :topk].expand(M, topk)
    assert not ids.is_contiguous() and not tw.is_contiguous()
    backend = AWQB200MoeBackend()
    got = backend.experts(x.clone(), w1, w2, tw, ids)
    assert torch.equal(got, backend.experts(x.clone(), w1, w2, tw.contiguous(), ids.contiguous()))


# CUDA documents __expf(-g) to within 2 + floor(1.173 |g|) units (2^-23 relative) and
# __fdividef to within 2 for denominators up to 2^126, above which it gives 0. With the
# rounded sum 1 + e^-g and a last product that makes silu(g) * u and sigmoid(g) relatively
# right to (6 + 1.173 |g|) 2^-23, and 0 for g below -87.3, where they are below |g| 2^-126.
GATES = [0.0, 1e-3, 0.5, 3.0, 10.0, 19.875, 20.0, 40.0, 63.75, 79.5, 80.0, 86.0, 87.0, 87.5, 88.0, 89.0, 100.0, 120.0]


def _act_error(g):
    return (6 + 1.173 * g.abs()) * 2.0 ** -23, torch.where(g < -87.3, g.abs() + 1, 0.0) * 2.0 ** -126


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [5, 90])  # few and many rows per expert
def test_silu_mul_of_large_gates(cuda, dtype, rows):
    """One weight per feature, so that gate and up are known to the bit."""
    gates = torch.tensor([s * v for v in GATES for s in (1, -1)] * 4, device=cuda)  # 144 features
    I, K = gates.numel(), 64
    w = torch.zeros((2, 2 * I, K), dtype=dtype, device=cuda)
    w[:, :I, 0] = gates.to(dtype)
    w[:, I:, 0] = (torch.arange(I, device=cuda) % 7 - 3).to(dtype) * 4
    x = torch.zeros((rows, K), dtype=dtype, device=cuda)
    x[:, 0] = 1
    offsets = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=cuda)
    got = ops.grouped_gemm(x, w, offsets, silu_mul=True).double()
    g, u = w[0, :I, 0].double(), w[0, I:, 0].double()
    want = g / (1 + torch.exp(-g)) * u
    rel, flushed = _act_error(g)
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2  # half of the type's smallest step
    off = rel * want.abs() + flushed * u.abs()
    assert bool(((got - want).abs() <= off + half_step(dtype) * (want.abs() + off) + tiny).all())


@pytest.mark.parametrize("act", ["sigmoid", "silu", "tanh"])
def test_norm_with_large_gates(cuda, act):
    """A zero fp32 residual shows the gated branch to 24 bits."""
    N, dtype = 4096, torch.bfloat16
    vals = torch.tensor([s * v for v in GATES for s in (1, -1)])
    gate = vals.repeat(N // vals.numel() + 1)[:N].to(dtype).to(cuda)
    x = (torch.arange(3 * N, device=cuda) % 13 - 6).to(dtype).view(3, N)
    r = torch.zeros((3, N), device=cuda)
    y, h = ops.gated_add_rmsnorm(x, r, torch.ones(N, dtype=dtype, device=cuda), 1e-6, gate=gate, gate_act=act)
    g = gate.double()
    a = {"sigmoid": 1 / (1 + torch.exp(-g)), "silu": g / (1 + torch.exp(-g)), "tanh": torch.tanh(g)}[act]
    want = x.double() * a
    rel, flushed = _act_error(g)
    if act == "tanh":
        flushed = flushed * 0
    # the activation, two products and a sum with zero, each rounded once in fp32
    off = (rel + 3 * 2.0 ** -24) * want.abs() + flushed * x.double().abs() + 2.0 ** -149
    assert bool(((h.double() - want).abs() <= off).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N", [(5, 64), (1000, 16384)])  # decode and prompt kernels
def test_ranks_of_very_different_size(cuda, dtype, M, N):
    """h enters the second product as two 16-bit halves. bf16: 2^-16 of each value. fp16: a
    place's largest value (per slice) is brought to 2^14 .. 2^15, so halves are off by
    2^-22 of the value, or by half of fp16's smallest step, 2^-25, where that is more:
    2^-39 of the largest. x is one, so that h is A's column to the bit; the largest rank's
    B is 0 in half of the features, so that the small ranks stand alone there."""
    K, L = 64, 2
    assert (M * (N * 58 + K * 8) > 8e8) == (M == 1000)
    sizes = torch.tensor([60000.0, 1.3, 2.0 ** -5 * 1.7, 2.0 ** -10 * 1.1, 2.0 ** -13 * 1.9, 2.0 ** -15 * 1.37, 2.0 ** -18, 0.0])
    a = torch.zeros((L, 8, K), dtype=dtype, device=cuda)
    a[0, :, 0] = sizes.to(dtype)
    a[1, :, 0] = sizes.flip(0).to(dtype) * 0.5
    g = torch.Generator(device=cuda).manual_seed(N)
    b = (torch.rand((L, N, 8), generator=g, device=cuda) + 0.5).to(dtype)
    b[0, :, 1:] *= 256
    b[0, ::2, :3] = 0  # the large ranks leave these features alone
    b[1, ::2, 5:] = 0
    x = torch.zeros((M, K), dtype=dtype, device=cuda)
    x[:, 0] = 1
    base = torch.zeros((M, N), dtype=dtype, device=cuda)
    base[:, 1::2] = 1
    ids = (torch.arange(M, device=cuda) % 3 - 1).to(torch.int32)
    scales = torch.tensor([2.0 ** -10, 0.75 * 2.0 ** -10], device=cuda)
    got = ops.lora(x, a, b, *ops.group_rows(ids, L), base, scales=scales).double()
    for l in range(L):
        h, bl, s = a[l, :, 0].double(), b[l].double(), float(scales[l])
        off_h = half_step(dtype) ** 2 * h.abs()
        if dtype == torch.float16:
            off_h = torch.maximum(off_h, 2.0 ** -39 * h.abs().max())
        rows = (ids == l).nonzero()[:, 0]
        d = s * (bl @ h)
        want = base[rows].double() + d
        # both halves' products (16 additions), two products and the last sum, each off by 2^-23
        off = abs(s) * (bl.abs() @ (off_h + 18 * 2.0 ** -23 * h.abs())) + 2.0 ** -23 * want.abs()
        step = 2.0 ** -25 if dtype == torch.float16 else 0.0
        assert bool(((got[rows] - want).abs() <= off + half_step(dtype) * (want.abs() + off) + step).all())
    assert torch.equal(got[ids < 0], base[ids < 0].double())
    assert ops.device_error() == 0


def test_rows_that_no_expert_wrote_are_not_summed(cuda, monkeypatch):
    """Every buffer that the experts allocate starts as NaN, and the rows of choices that
    are held nowhere here are seen to be NaN still when the sum runs."""
    M, E, H, I, topk, dtype = 40, 8, 128, 64, 3, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(9)
    x = torch.randn((M, H), generator=g, device=cuda).to(dtype)
    w1 = DenseExpertWeights((torch.randn((E, 2 * I, H), generator=g, device=cuda) / 11).to(dtype))
    w2 = DenseExpertWeights((torch.randn((E, H, I), generator=g, device=cuda) / 8).to(dtype))
    ids = torch.randint(-1, 2 * E, (M, topk), generator=g, device=cuda).to(torch.int32)
    ids[3] = -1  # a token with no expert here at all
    tw = torch.rand((M, topk), generator=g, device=cuda)
    here = (ids >= 0) & (ids < E)
    backend = AWQB200MoeBackend()
    want = backend.experts(x.clone(), w1, w2, tw * here, torch.where(here, ids, 0))
    empty, topk_sum, seen = torch.empty, ops.moe_topk_sum, []

    def poisoned(*args, **kw):
        t = empty(*args, **kw)
        return t.fill_(float("nan")) if t.is_floating_point() else t

    def spy(y3, *args):
        seen.append(y3.clone())
        return topk_sum(y3, *args)

    monkeypatch.setattr(torch, "empty", poisoned)
    monkeypatch.setattr(ops, "moe_topk_sum", spy)
    got = backend.experts(x.clone(), w1, w2, tw, ids)
    monkeypatch.undo()
    bare = torch.isnan(seen[0]).all(dim=1)
    assert torch.equal(bare.view(M, topk), ~here)
    assert torch.equal(got, want) and bool((got[3] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [3, 900])  # decode and prompt kernels
def test_row_parallel_shards_with_adapters_add_up(cuda, dtype, M):
    """The two ranks of a row-parallel projection one after the other, the all-reduce a sum
    by hand: each shard is its projection's output plus its part of the adapters
    (64-bit formula), and the sum of both is the whole layer's output."""
    K, N, L, r = 512, 16384 if M == 900 else 256, 3, 32
    wq = make_awq_weights(K, N, 128, dtype, seed=5)
    method = AWQB200Config(4, 128, True).get_linear_method()
    g = torch.Generator(device=cuda).manual_seed(M)
    x = torch.randn((M, K), generator=g, device=cuda).to(dtype)
    adapters = LoraAdapters((torch.randn((L, r, K), generator=g, device=cuda) * K ** -0.5).to(dtype),
                            (torch.randn((L, N, r), generator=g, device=cuda)).to(dtype),
                            torch.rand(L, generator=g, device=cuda) + 0.5)
    ids = torch.randint(-1, L, (M,), generator=g, device=cuda).to(torch.int32)
    batch = LoraBatch.from_ids(ids, L)

    class Comm:  # takes this rank's part
        def all_reduce(self, y):
            return y

    parts = []
    for rank in range(2):
        layer = RowParallelAWQLinear(method, K, N, 2, Comm())
        layer.load({k: v.to(cuda) for k, v in shard_awq(wq, "row", rank, 2).items()})
        layer.adapters = adapters.shard("row", rank, 2)
        xs = x.chunk(2, dim=1)[rank].contiguous()
        plain, y = layer.forward(xs), layer.forward(xs, batch)
        want, bound = lora_ref(xs, layer.adapters.a, layer.adapters.b, ids, plain, (N,), adapters.scales,
                               halves_eps=half_step(dtype) ** 2)
        assert within(y, want, bound, dtype) <= 0
        assert torch.equal(y[ids < 0], plain[ids < 0])
        parts.append(y.double())
    whole = RowParallelAWQLinear(method, K, N, 1)
    whole.load({k: v.to(cuda) for k, v in wq.items() if k in ("qweight", "qzeros", "scales")})
    whole.adapters = adapters
    assert rel_err((parts[0] + parts[1]).float(), whole.forward(x, batch).float().cpu()) <= 1e-2  # that of the GEMM tests
    assert ops.device_error() == 0


@pytest.mark.parametrize("op", ["gemm 1", "gemm 64", "gemm 600", "grouped few", "grouped many", "lora decode", "lora prompt",
                                "norm", "rotary", "group_rows", "experts"])
def test_first_call_of_a_host_thread(cuda, op):
    """A thread that has made no CUDA call yet has no current context."""
    import threading

    g = torch.Generator(device=cuda).manual_seed(4)
    dtype = torch.bfloat16

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=cuda) * std).to(dtype)

    if op.startswith("gemm"):
        wq = make_awq_weights(512, 256, 128, dtype, seed=6)
        layer = RowParallelAWQLinear(AWQB200Config(4, 128, True).get_linear_method(), 512, 256, 1)
        layer.load({k: v.to(cuda) for k, v in wq.items() if k in ("qweight", "qzeros", "scales")})
        x = normal(int(op[5:]), 512)
        call = lambda: layer.forward(x)  # noqa: E731
    elif op.startswith("grouped"):
        rows = 9 if op.endswith("few") else 200
        x, w = normal(rows, 64), normal(2, 64, 64)
        offsets = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device=cuda)
        call = lambda: ops.grouped_gemm(x, w, offsets)  # noqa: E731
    elif op.startswith("lora"):
        M, N = (9, 64) if op.endswith("decode") else (1200, 16384)
        x, a, b, base = normal(M, 64), normal(2, 8, 64), normal(2, N, 8), normal(M, N)
        order, offsets = ops.group_rows(torch.arange(M, device=cuda, dtype=torch.int32) % 2, 2)
        call = lambda: ops.lora(x, a, b, order, offsets, base)  # noqa: E731
    elif op == "norm":
        x, r, w = normal(3, 64), normal(3, 64), normal(64)
        call = lambda: ops.gated_add_rmsnorm(x, r, w, 1e-6)[0]  # noqa: E731
    elif op == "rotary":
        q, pos, inv = normal(3, 2, 64), torch.arange(3, device=cuda), torch.ones(32, dtype=torch.float64, device=cuda)
        call = lambda: ops.rotary(q, None, pos, inv)[0]  # noqa: E731
    elif op == "group_rows":
        ids = torch.arange(30, device=cuda, dtype=torch.int32) % 4
        call = lambda: ops.group_rows(ids, 4)[0]  # noqa: E731
    else:
        x, w1, w2, logits = normal(5, 64), normal(4, 64, 64), normal(4, 64, 32), torch.randn((5, 4), device=cuda)
        call = lambda: AWQB200MoeBackend().forward(x.clone(), w1, w2, logits, 2, True)  # noqa: E731
    want, got = call(), []
    torch.cuda.synchronize()

    def work():
        try:
            got.append(call())
        except BaseException as e:  # compared below
            got.append(e)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert isinstance(got[0], torch.Tensor), got
    assert torch.equal(got[0], want)


def test_two_threads_on_one_stream(cuda):
    """Each call is several launches that start before the one in front has ended: launches of
    another thread's call may fall between them, and change nothing."""
    import threading

    g = torch.Generator(device=cuda).manual_seed(4)
    dtype = torch.bfloat16

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=cuda) * std).to(dtype)

    K, N = 512, 256
    wq = make_awq_weights(K, N, 128, dtype, seed=6)
    layer = RowParallelAWQLinear(AWQB200Config(4, 128, True).get_linear_method(), K, N, 1)
    layer.load({k: v.to(cuda) for k, v in wq.items() if k in ("qweight", "qzeros", "scales")})
    xs, w, offsets = normal(200, K), normal(3, 64, K, std=K ** -0.5), torch.tensor([0, 70, 90, 200], dtype=torch.int32, device=cuda)
    few, res, weight = normal(9, K), normal(200, K), normal(K)

    def others():
        return (layer.forward(xs), ops.grouped_gemm(xs, w, offsets), ops.grouped_gemm(few, w, offsets.clamp_max(9)),
                *ops.gated_add_rmsnorm(xs, res, weight, 1e-6))

    adapted = []
    for M, n in ((24, 256), (1200, 16384)):  # decode and prompt kernels
        ids = torch.randint(-1, 4, (M,), generator=g, device=cuda).to(torch.int32)
        adapted.append((normal(M, K), normal(4, 32, K, std=K ** -0.5), normal(4, n, 32), *ops.group_rows(ids, 4), normal(M, n)))

    def adapters():
        return tuple(ops.lora(x, a, b, order, off, base) for x, a, b, order, off, base in adapted)

    jobs, failures = [(others, others()), (adapters, adapters())], []
    torch.cuda.synchronize()

    def work(f, want):
        try:
            for _ in range(60):
                assert all(torch.equal(a, b) for a, b in zip(f(), want))
        except BaseException as e:  # reported by the test itself
            failures.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    assert ops.device_error() == 0
