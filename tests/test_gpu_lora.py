"""Low-rank adapters beside a projection on the GPU against the 64-bit formula,
within fp32 accumulation of both products, plus one rounding to the type. The first
product enters the second as two 16-bit halves: what the second half rounds
away is half_step^2 of the value (2^-16 for bf16, 2^-22 for fp16)."""

import pytest
import torch

from oracle.block_ref import half_step, lora_ref, within
from sglite_b200 import ops
from sglite_b200.lora import LoraAdapters, LoraBatch
from sglite_b200.quantization import AWQB200Config
from sglite_b200.synthetic import make_awq_weights

pytestmark = pytest.mark.gpu


def _case(cuda, M, K, slices, rank, L, dtype, seed=0, none=0.2, sort=False):
    g = torch.Generator(device=cuda).manual_seed(seed + M + K)
    N, S = sum(slices), len(slices)
    x = torch.randn((M, K), generator=g, device=cuda).to(dtype)
    a = (torch.randn((L, S * rank, K), generator=g, device=cuda) * K ** -0.5).to(dtype)
    b = (torch.randn((L, N, rank), generator=g, device=cuda) * rank ** -0.5).to(dtype)
    base = torch.randn((M, N), generator=g, device=cuda).to(dtype)
    ids = torch.randint(0, L, (M,), generator=g, device=cuda)
    ids[torch.rand(M, generator=g, device=cuda) < none] = -1
    if sort:
        ids = ids.sort().values
    scales = torch.rand(L, generator=g, device=cuda) + 0.5
    return x, a, b, base, ids.to(torch.int32), scales


def _check(got, x, a, b, ids, base, slices, scales):
    want, bound = lora_ref(x, a, b, ids, base, slices, scales, halves_eps=half_step(x.dtype) ** 2)
    assert within(got, want, bound, x.dtype) <= 0
    none = (ids < 0) | (ids >= b.shape[0])
    assert torch.equal(got[none], base[none])


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 64, 130, 700])
@pytest.mark.parametrize("K,slices,rank", [(4096, (512, 128, 128), 16), (64, (64,), 8), (1000, (40, 8), 24),
                                           (2560, (1032, 1032), 64), (520, (264,), 128), (8, (8,), 8),
                                           (896, (64, 32, 32, 64), 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_sizes(cuda, M, K, slices, rank, dtype):
    x, a, b, base, ids, scales = _case(cuda, M, K, slices, rank, 6, dtype)
    order, offsets = ops.group_rows(ids, 6)
    base0 = base.clone()
    got = ops.lora(x, a, b, order, offsets, base, slices=slices, scales=scales)
    assert torch.equal(base, base0)
    _check(got, x, a, b, ids, base, slices, scales)
    y = base.clone()
    assert ops.lora(x, a, b, order, offsets, y, slices=slices, scales=scales, out=y) is y  # in place
    assert torch.equal(y, got)


def _prompt(M, K, slices, rank):
    """Whether these sizes go to the prompt kernels (the rule of awqb_lora.cu): what
    follows is meant to."""
    return M * (sum(slices) * (50 + rank) + K * rank * len(slices)) > 8e8


@pytest.mark.parametrize("M,K,slices,rank", [(600, 72, (24584, 8, 1032), 8), (1300, 200, (8200, 136), 24),
                                             (300, 1000, (16008, 3000), 128), (700, 2560, (9728, 9728), 64),
                                             (2100, 1024, (4096, 1024, 1024), 32), (130, 8, (40000,), 128),
                                             (900, 14336, (4096,), 64), (1025, 4096, (1536, 512, 512, 1032), 96)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sort", [False, True])
def test_prompt_sizes(cuda, M, K, slices, rank, dtype, sort):
    """Rows in random order (copied one by one) and in order (runs), in and out of place."""
    assert _prompt(M, K, slices, rank)
    L = 6
    x, a, b, base, ids, scales = _case(cuda, M, K, slices, rank, L, dtype, sort=sort)
    order, offsets = ops.group_rows(ids, L)
    base0 = base.clone()
    got = ops.lora(x, a, b, order, offsets, base, slices=slices, scales=scales)
    assert torch.equal(base, base0)
    _check(got, x, a, b, ids, base, slices, scales)
    y = base.clone()
    ops.lora(x, a, b, order, offsets, y, slices=slices, scales=scales, out=y)
    assert torch.equal(y, got)
    assert ops.device_error() == 0


@pytest.mark.parametrize("kind", ["one", "none", "first", "last", "many", "tiles"])
def test_prompt_who_uses_which(cuda, kind):
    M, K, N, L = 1500, 256, 8192, 1024 if kind == "many" else 9
    assert _prompt(M, K, (N,), 64)
    x, a, b, base, ids, scales = _case(cuda, M, K, (N,), 64, L, torch.bfloat16)
    if kind == "tiles":  # groups of exactly one tile, one row more and one less
        ids = torch.repeat_interleave(torch.arange(9, device=cuda), torch.tensor([128, 129, 127, 0, 1, 256, 384, 0, 400], device=cuda))
        ids = torch.cat([ids, torch.full((M - ids.numel(),), -1, device=cuda)]).to(torch.int32)
    elif kind != "many":
        ids = torch.full_like(ids, {"one": 4, "none": -1, "first": 0, "last": L - 1}[kind])
    order, offsets = ops.group_rows(ids, L)
    _check(ops.lora(x, a, b, order, offsets, base, scales=scales), x, a, b, ids, base, (N,), scales)
    assert ops.device_error() == 0


def test_prompt_strides_extremes_and_graphs(cuda):
    M, K, N, r, L, dtype = 1200, 512, 8192, 64, 4, torch.float16
    assert _prompt(M, K, (N,), r)
    x, a, b, base, ids, scales = _case(cuda, M, K, (N,), r, L, dtype)
    wide_x = torch.full((M, K + 8), float("nan"), dtype=dtype, device=cuda)
    wide_x[:, :K] = x
    wide = torch.full((M, N + 16), 5.0, dtype=dtype, device=cuda)
    wide[:, :N] = base
    order, offsets = ops.group_rows(ids, L)
    y = wide[:, :N]
    ops.lora(wide_x[:, :K], a, b, order, offsets, y, scales=scales, out=y)
    _check(y, x, a, b, ids, base, (N,), scales)
    assert bool((wide[:, N:] == 5).all())
    # a first product past fp16's range
    big = ops.lora(x * 64, a * 2048, b * 2.0 ** -12, order, offsets, base)
    _check(big, x * 64, a * 2048, b * 2.0 ** -12, ids, base, (N,), None)
    # infinities and NaN stay in their rows
    x2 = x.clone()
    x2[7, 3], x2[600, 9] = float("nan"), float("inf")
    ids2 = ids.clamp_min(0)
    bad = ~torch.isfinite(ops.lora(x2, a, b, *ops.group_rows(ids2, L), base))
    assert bool(bad[7].all()) and bool(bad[600].any())
    bad[7] = bad[600] = False
    assert not bool(bad.any())
    # a graph that groups and adds, replayed with another mix of adapters
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2, f2 = ops.group_rows(ids, L)
        out = ops.lora(x, a, b, o2, f2, base, scales=scales)
    for shift in (0, 1):
        ids.add_(shift).remainder_(L + 1)
        graph.replay()
        torch.cuda.synchronize()
        _check(out, x, a, b, ids, base, (N,), scales)
    assert ops.device_error() == 0


def test_two_streams_at_once(cuda):
    """Calls that run side by side have workspaces of their own."""
    cases = [_case(cuda, M, 1024, (N,), 32, 5, torch.bfloat16, seed=i) for i, (M, N) in enumerate(((40, 512), (900, 16384)))]
    groups = [ops.group_rows(c[4], 5) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[], []]
    for _ in range(4):
        for i, (s, c, g) in enumerate(zip(streams, cases, groups)):
            with torch.cuda.stream(s):
                outs[i].append(ops.lora(c[0], c[1], c[2], g[0], g[1], c[3], scales=c[5]))
    torch.cuda.synchronize()
    for c, os in zip(cases, outs):
        for o in os:
            _check(o, c[0], c[1], c[2], c[4], c[3], (c[3].shape[1],), c[5])


@pytest.mark.parametrize("kind", ["one", "none", "first", "last", "many"])
@pytest.mark.parametrize("M", [33, 2000])
def test_who_uses_which(cuda, M, kind):
    """All rows one adapter, no row any, the ends of the range, more adapters than rows."""
    L = 300 if kind == "many" else 9
    x, a, b, base, ids, _ = _case(cuda, M, 512, (256,), 16, L, torch.bfloat16, sort=kind == "one")
    if kind != "many":
        ids = torch.full_like(ids, {"one": 4, "none": -1, "first": 0, "last": L - 1}[kind])
    order, offsets = ops.group_rows(ids, L)
    _check(ops.lora(x, a, b, order, offsets, base), x, a, b, ids, base, (256,), None)


def test_strided_rows_and_no_rows(cuda):
    M, K, N, dtype = 50, 128, 192, torch.float16
    x, a, b, base, ids, scales = _case(cuda, M, K, (N,), 16, 3, dtype)
    wide_x = torch.zeros((M, K + 8), dtype=dtype, device=cuda)
    wide_x[:, :K] = x
    wide = torch.full((M, N + 16), 5.0, dtype=dtype, device=cuda)
    wide[:, :N] = base
    order, offsets = ops.group_rows(ids, 3)
    y = wide[:, :N]
    ops.lora(wide_x[:, :K], a, b, order, offsets, y, scales=scales, out=y)
    _check(y, x, a, b, ids, base, (N,), scales)
    assert bool((wide[:, N:] == 5).all())
    assert ops.lora(x[:0], a, b, order[:0], torch.zeros_like(offsets), base[:0]).shape == (0, N)


def test_large_first_product(cuda):
    """A first product past fp16's range, brought back by a small second factor: no
    overflow on the way (each sum is within fp32)."""
    M, K, N, r, dtype = 20, 1024, 64, 16, torch.float16
    x, a, b, base, ids, _ = _case(cuda, M, K, (N,), r, 2, dtype, none=0.0)
    x, a, b = x * 64, a * 2048, b * 2.0 ** -12
    order, offsets = ops.group_rows(ids, 2)
    got = ops.lora(x, a, b, order, offsets, base)
    assert float((x[0].double() @ a[int(ids[0])].double().T).abs().max()) > 70000
    _check(got, x, a, b, ids, base, (N,), None)


def test_infinities_stay_in_their_rows(cuda):
    M, K, N, dtype = 40, 256, 128, torch.bfloat16
    x, a, b, base, ids, _ = _case(cuda, M, K, (N,), 8, 3, dtype, none=0.0)
    x[7, 3] = float("nan")
    x[20, 9] = float("inf")
    order, offsets = ops.group_rows(ids, 3)
    bad = ~torch.isfinite(ops.lora(x, a, b, order, offsets, base))
    assert bool(bad[7].all()) and bool(bad[20].any())
    bad[7] = bad[20] = False
    assert not bool(bad.any())


def test_graph_replay_with_new_groups(cuda):
    """Captured with its grouping: a replay serves another mix of adapters; two graphs
    have workspaces of their own."""
    M, K, slices, L = 24, 512, (128, 64), 5
    x, a, b, base, ids, scales = _case(cuda, M, K, slices, 16, L, torch.bfloat16)
    ops.lora(x, a, b, *ops.group_rows(ids, L), base, slices=slices, scales=scales)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            order, offsets = ops.group_rows(ids, L)
            outs.append(ops.lora(x, a, b, order, offsets, base, slices=slices, scales=scales))
        graphs.append(graph)
    for shift in (0, 1, 3):
        ids.add_(shift).remainder_(L + 1)  # id L: none
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o in outs:
            _check(o, x, a, b, ids, base, slices, scales)


def test_linear_method_and_layer_with_adapters(cuda):
    """apply_weights(adapters=): the projection's output plus each row's adapter;
    adapters of different ranks stacked from their checkpoint factors."""
    from sglite_b200.tp import ColumnParallelAWQLinear

    K, widths, dtype, M, L = 512, (256, 128), torch.bfloat16, 21, 3
    N = sum(widths)
    wq = make_awq_weights(K, N, 128, dtype, seed=1)
    method = AWQB200Config(4, 128, True).get_linear_method()
    layer = ColumnParallelAWQLinear(method, K, N)
    layer.load({k: wq[k].to(cuda) for k in ("qweight", "qzeros", "scales")})
    g = torch.Generator(device=cuda).manual_seed(2)

    def pair(r, n):
        return ((torch.randn((r, K), generator=g, device=cuda) * K ** -0.5).to(dtype),
                (torch.randn((n, r), generator=g, device=cuda)).to(dtype))

    adapters = LoraAdapters.stack([[pair(16, 256), pair(8, 128)], [None, pair(12, 128)], [pair(4, 256), None]], widths,
                                  scales=[2.0, 0.5, 1.0])
    assert adapters.a.shape == (L, 2 * 16, K) and adapters.b.shape == (L, N, 16)
    layer.adapters = adapters
    x = torch.randn((3, 7, K), generator=g, device=cuda).to(dtype)
    ids = torch.randint(-1, L, (M,), generator=g, device=cuda).to(torch.int32)
    plain = layer.forward(x)
    y = layer.forward(x, LoraBatch.from_ids(ids, L))
    assert y.shape == (3, 7, N)
    _check(y.view(M, N), x.view(M, K), adapters.a, adapters.b, ids, plain.view(M, N), widths, adapters.scales)
    with pytest.raises(ValueError):
        method.apply_weights(layer.weights, x, adapters=adapters)
