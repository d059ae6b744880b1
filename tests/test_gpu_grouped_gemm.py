"""Row grouping and the products grouped by expert on the GPU. Grouping is exact.
The products are held to the 64-bit result within the bound of fp32
accumulation (K additions) plus one rounding to the type."""

import pytest
import torch

from oracle.awq_ref import rel_err
from oracle.block_ref import grouped_gemm_ref, within
from sglite_b200 import ops
from sglite_b200.moe import AWQB200MoeBackend, DenseExpertWeights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [0, 1, 31, 1000, 8192, 10239, 10240, 40001])
@pytest.mark.parametrize("groups,begin", [(1, 0), (7, 2), (128, 0), (1024, 0), (1000, -3)])
def test_group_rows(cuda, n, groups, begin):
    g = torch.Generator().manual_seed(n + groups)
    ids = torch.randint(begin - 2, begin + groups + 2, (n,), generator=g, dtype=torch.int32)
    order, offsets = ops.group_rows(ids.to(cuda), groups, begin)
    key = torch.where((ids >= begin) & (ids < begin + groups), ids - begin, groups)
    want = torch.argsort(key, stable=True)
    count = torch.bincount(key.long(), minlength=groups + 1)[:groups]
    assert torch.equal(order.cpu().long(), want)
    assert torch.equal(offsets.cpu().long(), torch.cat([torch.zeros(1, dtype=torch.int64), count.cumsum(0)]))


def test_group_rows_ids_at_the_ends_of_their_type(cuda):
    ids = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0, -1, 3], dtype=torch.int32, device=cuda)
    order, offsets = ops.group_rows(ids, 4)
    assert order.tolist() == [2, 4, 0, 1, 3] and offsets.tolist() == [0, 1, 1, 1, 2]


def _offsets(sizes, cuda, first=0):
    return torch.tensor([first] + sizes).cumsum(0).to(cuda, torch.int32)


def _run(cuda, sizes, K, N, dtype, silu=False, pad=0, first=0, seed=0, ldx=0, ldo=0):
    g = torch.Generator(device=cuda).manual_seed(seed + K + N)
    rows = first + sum(sizes) + pad
    xw = torch.randn((rows, K + ldx), generator=g, device=cuda).to(dtype)
    x = xw[:, :K]
    w = (torch.randn((len(sizes), N, K), generator=g, device=cuda) * K ** -0.5).to(dtype)
    off = _offsets(sizes, cuda, first)
    n_out = N // 2 if silu else N
    out = torch.full((rows, n_out + ldo), 3.0, dtype=dtype, device=cuda)
    got = ops.grouped_gemm(x, w, off, out=out[:, :n_out], silu_mul=silu)
    y, bound = grouped_gemm_ref(x, w, off.cpu(), silu)
    live = slice(first, first + sum(sizes))
    assert within(got[live], y[live], bound[live], dtype) <= 0
    rest = torch.ones(rows, dtype=torch.bool)
    rest[live] = False
    assert bool((out[rest.to(cuda)] == 3).all()) and bool((out[:, n_out:] == 3).all())
    return x, w, off, got


@pytest.mark.parametrize("K,N", [(64, 64), (8, 8), (72, 264), (768, 2048), (1000, 520), (2048, 1536), (200, 16)])
@pytest.mark.parametrize("sizes", [[1], [0, 0, 5], [1, 0, 127, 128, 129], [300, 1, 0, 2, 257, 0], [16] * 9, [700]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("silu", [False, True])
def test_sizes(cuda, K, N, sizes, dtype, silu):
    if silu and N % 16:
        pytest.skip("silu_mul needs N % 16 == 0 (its refusal is tested)")
    _run(cuda, sizes, K, N, dtype, silu)


@pytest.mark.parametrize("silu", [False, True])
def test_rows_outside_the_groups_and_strides(cuda, silu):
    _run(cuda, [3, 130, 0, 60], 192, 336, torch.bfloat16, silu, pad=150, first=9, ldx=16, ldo=24)
    _run(cuda, [0, 0], 64, 64, torch.float16, silu, pad=5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_experts_and_wide_outputs(cuda, dtype):
    g = torch.Generator().manual_seed(3)
    _run(cuda, torch.randint(0, 4, (1024,), generator=g).tolist(), 64, 128, dtype)
    _run(cuda, torch.randint(0, 90, (128,), generator=g).tolist(), 2048, 1536, dtype, silu=True)
    _run(cuda, [2000, 0, 1511], 1024, 4104, dtype)
    _run(cuda, [1, 2, 3], 14336, 512, dtype)


def test_scatter_scale_and_dropped_rows(cuda):
    sizes, K, N, dtype = [40, 0, 133, 5], 256, 264, torch.bfloat16
    rows = sum(sizes)
    g = torch.Generator(device=cuda).manual_seed(8)
    x = torch.randn((rows, K), generator=g, device=cuda).to(dtype)
    w = (torch.randn((4, N, K), generator=g, device=cuda) / 16).to(dtype)
    off = _offsets(sizes, cuda)
    row_map = torch.randperm(rows, generator=g, device=cuda).to(torch.int32)
    out_rows = rows - 20  # rows that map past the end are dropped
    row_map[3] = -1
    scale = torch.rand(out_rows, generator=g, device=cuda)
    out = torch.full((out_rows, N), 9.0, dtype=dtype, device=cuda)
    ops.grouped_gemm(x, w, off, out=out, row_map=row_map, row_scale=scale)
    y, bound = grouped_gemm_ref(x, w, off.cpu())
    hit = torch.zeros(out_rows, dtype=torch.bool, device=cuda)
    ok = (row_map >= 0) & (row_map < out_rows)
    to = row_map[ok].long()
    hit[to] = True
    s = scale[to].double()[:, None]
    assert within(out[to], y[ok] * s, bound[ok] * s + 2.0 ** -23 * (y[ok] * s).abs(), dtype) <= 0
    assert bool((out[~hit] == 9).all())


def test_wrong_offsets_stay_inside_the_buffers(cuda):
    """offsets past the ends are clamped (the host cannot see them): no write
    leaves the rows, and the groups that fit are right."""
    K, N, dtype = 128, 128, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(8)
    x = torch.randn((50, K), generator=g, device=cuda).to(dtype)
    w = (torch.randn((3, N, K), generator=g, device=cuda) / 16).to(dtype)
    buf = torch.full((70, N), 9.0, dtype=dtype, device=cuda)
    out = buf[10:60]
    off = torch.tensor([-5, 20, 30, 1 << 30], dtype=torch.int32, device=cuda)
    ops.grouped_gemm(x, w, off, out=out)
    y, bound = grouped_gemm_ref(x, w, torch.tensor([0, 20, 30, 50]))
    assert within(out, y, bound, dtype) <= 0
    assert bool((buf[:10] == 9).all()) and bool((buf[60:] == 9).all())
    assert ops.device_error() == 0


def test_nan_and_infinity_stay_in_their_rows(cuda):
    K, N, dtype = 320, 256, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn((260, K), generator=g, device=cuda).to(dtype)
    x[130, 3], x[131, 3] = float("nan"), float("inf")
    w = torch.randn((2, N, K), generator=g, device=cuda).to(dtype)
    w[1, 7] = float("inf")
    off = _offsets([200, 60], cuda)
    y = ops.grouped_gemm(x, w, off)
    bad = ~torch.isfinite(y)
    assert bool(bad[130].all()) and bool(bad[131].all()) and bool(bad[200:, 7].all())
    bad[130:132] = False
    bad[200:, 7] = False
    assert not bool(bad.any())


def test_same_bits_every_time_in_a_graph_and_on_a_side_stream(cuda):
    sizes, K, N = [5, 200, 0, 77], 512, 768
    x, w, off, got = _run(cuda, sizes, K, N, torch.bfloat16)
    want = got.clone()
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.grouped_gemm(x, w, off, out=out)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.grouped_gemm(x, w, off, out=out)
    moved = _offsets([100, 100, 41, 41], cuda)
    for o in (off.clone(), moved):  # the groups may change between replays
        off.copy_(o)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        y, bound = grouped_gemm_ref(x, w, o.cpu())
        assert within(out, y, bound, torch.bfloat16) <= 0
    assert ops.device_error() == 0


@pytest.mark.parametrize("M", [1, 16, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_backend_over_dense_experts(cuda, M, dtype):
    """The MoE backend's pipeline over 16-bit experts against fp32 torch, whole and
    as two expert-parallel halves. Tolerance: that of the GEMM tests."""
    E, H, I, topk = 16, 256, 96, 4
    g = torch.Generator().manual_seed(M)
    x = torch.randn((M, H), generator=g).to(dtype).to(cuda)
    w1 = (torch.randn((E, 2 * I, H), generator=g) / 16).to(dtype).to(cuda)
    w2 = (torch.randn((E, H, I), generator=g) / 8).to(dtype).to(cuda)
    logits = torch.randn((M, E), generator=g).to(cuda)
    backend = AWQB200MoeBackend()
    y = backend.forward(x.clone(), w1, w2, logits, topk, True)
    tw, ids = ops.moe_topk_softmax(logits, topk, True)
    ref = torch.zeros((M, H), device=cuda)
    for k in range(topk):
        e = ids[:, k].long()
        h = torch.bmm(w1[e].float(), x.float()[..., None])[..., 0]
        a = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
        ref += tw[:, k, None] * torch.bmm(w2[e].float(), a[..., None])[..., 0]
    assert rel_err(y, ref.cpu()) <= 1e-2
    parts = torch.zeros((M, H), device=cuda)
    for lo in (0, E // 2):
        p1 = DenseExpertWeights(w1[lo:lo + E // 2], lo, E)
        p2 = DenseExpertWeights(w2[lo:lo + E // 2], lo, E)
        parts += backend.forward(x.clone(), p1, p2, logits, topk, True).float()
    assert rel_err(parts, ref.cpu()) <= 1e-2


def test_ids_of_no_expert_here_add_nothing(cuda):
    """The first half of the experts, with nothing said about how many there are in
    all, and padding: their choices are worth exactly those with weight zero."""
    M, E, H, I, topk, dtype = 40, 8, 128, 64, 3, torch.bfloat16
    g = torch.Generator(device=cuda).manual_seed(9)
    x = torch.randn((M, H), generator=g, device=cuda).to(dtype)
    w1 = DenseExpertWeights((torch.randn((E, 2 * I, H), generator=g, device=cuda) / 11).to(dtype))
    w2 = DenseExpertWeights((torch.randn((E, H, I), generator=g, device=cuda) / 8).to(dtype))
    ids = torch.randint(-1, 2 * E, (M, topk), generator=g, device=cuda).to(torch.int32)
    tw = torch.rand((M, topk), generator=g, device=cuda)
    here = (ids >= 0) & (ids < E)
    assert bool((~here).any()) and bool(here.any())
    backend = AWQB200MoeBackend()
    poison = torch.full((M * topk, H), float("nan"), dtype=dtype, device=cuda)
    del poison  # what the allocator hands out next is not zero
    y = backend.experts(x.clone(), w1, w2, tw, ids)
    want = backend.experts(x.clone(), w1, w2, tw * here, torch.where(here, ids, 0))
    assert torch.equal(y, want)


def test_calls_of_two_threads(cuda):
    """Both threads' launches want different amounts of shared memory of the same kernels."""
    import threading

    g = torch.Generator(device=cuda).manual_seed(3)
    jobs, failures = [], []
    for groups in (500, 1000):
        ids = torch.randint(0, groups, (4000,), generator=g, device=cuda).to(torch.int32)
        x = torch.randn((4000, 64), generator=g, device=cuda).to(torch.bfloat16)
        w = torch.randn((groups, 32, 64), generator=g, device=cuda).to(torch.bfloat16)
        order, offsets = ops.group_rows(ids, groups)
        jobs.append((ids, groups, x, w, order, offsets, ops.grouped_gemm(x, w, offsets)))
    torch.cuda.synchronize()

    def work(ids, groups, x, w, order, offsets, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(300):
                    o, f = ops.group_rows(ids, groups)
                    y = ops.grouped_gemm(x, w, f)
                    assert torch.equal(o, order) and torch.equal(f, offsets) and torch.equal(y, want)
        except BaseException as e:  # reported by the test itself
            failures.append(e)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    assert ops.device_error() == 0
