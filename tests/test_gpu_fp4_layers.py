"""Microscaled 4-bit floating point as a model uses it: the linear method, the norm in
front of it, the experts of the MoE backend, a block of them in a CUDA graph, on other
streams and at offsets past 32 bits. Each operator alone is held to its definition in
test_gpu_fp4.py; here the paths are held to the same products of the weights' values."""

import pytest
import torch

from oracle.block_ref import half_step, within
from oracle.fp4_ref import product_ref, quantize_ref, over_scale, values_ref
from sglite_b200 import ops
from sglite_b200.lora import LoraAdapters, LoraBatch
from sglite_b200.moe import AWQB200MoeBackend, DenseExpertWeights, FP4ExpertWeights
from sglite_b200.norm import RMSNormFP4
from sglite_b200.quantization import get_quantization_config
from sglite_b200.quantization.fp4_b200 import quantize_weight

pytestmark = pytest.mark.gpu

FORMATS = ["nvfp4", "mxfp4"]


def _normal(cuda, *shape, dtype=torch.bfloat16, std=1.0, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed + sum(shape))
    return (torch.randn(shape, generator=g, device=cuda) * std).to(dtype)


def _linear(cuda, fmt, K, N, dtype, seed=0, input_scale=0.01, gate_up=False):
    """(method, weights, the values that the weight is held as, its scale)."""
    method = get_quantization_config("fp4_b200")(fmt).get_linear_method()
    weights = method.create_weights(K, N)
    loaded = quantize_weight(_normal(cuda, N, K, dtype=dtype, std=K ** -0.5, seed=seed), fmt)
    values = values_ref(loaded["weight"], loaded["weight_scale"], fmt)
    for name, t in loaded.items():
        assert weights[name].shape == t.shape and weights[name].dtype == t.dtype
        weights[name] = t
    if gate_up:
        for name in ("weight", "weight_scale"):
            weights[name] = ops.fp4_interleave_gate_up(weights[name])
        values = ops.fp4_interleave_gate_up(values)
    for name in list(weights):
        if isinstance(weights[name], torch.nn.Parameter):
            weights[name] = weights[name].data.to(cuda)
    if fmt == "nvfp4":
        weights["input_scale"] = torch.full((1,), input_scale, device=cuda)
    weights = {k: torch.nn.Parameter(v, requires_grad=False) if isinstance(v, torch.Tensor) else v for k, v in weights.items()}
    return method, method.process_weights_after_loading(weights), values, loaded.get("weight_scale_2")


def _held(x, fmt, scale):
    return quantize_ref(over_scale(x.cpu(), scale), fmt)[0]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("shape", [(1,), (3,), (2, 5), (70,)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_method(cuda, fmt, shape, dtype):
    K, N = 544, 264
    method, weights, values, ws = _linear(cuda, fmt, K, N, dtype)
    x = _normal(cuda, *shape, K, dtype=dtype)
    bias = _normal(cuda, N, dtype=dtype, seed=3)
    xs = weights.get("input_scale")
    y, bound = product_ref(_held(x.reshape(-1, K), fmt, xs), values, xs, ws, bias.cpu())
    got = method.apply_weights(weights, x, bias)
    assert got.shape == (*shape, N) and got.dtype == dtype
    assert within(got.reshape(-1, N).cpu(), y, bound, dtype) <= 0
    out = torch.empty((*shape, N), dtype=dtype, device=cuda)
    assert method.apply_weights(weights, x, bias, out=out).data_ptr() == out.data_ptr() and torch.equal(out, got)
    assert method.process_weights_after_loading(weights) is weights


def test_quantised_weight_with_an_infinity_or_a_nan(cuda):
    """The block is NaN, and the others are as they are without it; so are tiny weights."""
    w = _normal(cuda, 16, 256, std=0.02)
    clean = quantize_weight(w, "nvfp4")
    for bad in (float("inf"), float("nan")):
        one = w.clone()
        one[3, 40] = bad
        got = quantize_weight(one, "nvfp4")
        values = values_ref(got["weight"], got["weight_scale"], "nvfp4") * float(got["weight_scale_2"])
        want = values_ref(clean["weight"], clean["weight_scale"], "nvfp4") * float(clean["weight_scale_2"])
        block = torch.zeros((16, 256), dtype=torch.bool)
        block[3, 32:48] = True
        assert bool(torch.isnan(values[block]).all()) and torch.equal(values[~block], want[~block])
    tiny = quantize_weight((w.double() * 2.0 ** -120).to(w.dtype), "nvfp4")
    values = values_ref(tiny["weight"], tiny["weight_scale"], "nvfp4") * float(tiny["weight_scale_2"])
    assert bool(torch.isfinite(values).all()) and bool((values != 0).any())


@pytest.mark.parametrize("fmt", FORMATS)
def test_one_row_without_a_batch_and_rows_from_the_middle(cuda, fmt):
    """x [K] as a row, and weights and x that start inside a larger tensor: the same bits."""
    K, N = 288, 136
    method, weights, _, _ = _linear(cuda, fmt, K, N, torch.bfloat16)
    x = _normal(cuda, 3, K)
    want = method.apply_weights(weights, x)
    one = method.apply_weights(weights, x[1])
    assert one.shape == (N,) and torch.equal(one, want[1])
    room = torch.zeros((7, K + 64), dtype=torch.bfloat16, device=cuda)
    room[2:5, 32:32 + K] = x
    assert torch.equal(method.apply_weights(weights, room[2:5, 32:32 + K]), want)
    more = torch.zeros((N + 3, K // 2), dtype=torch.uint8, device=cuda)
    more[3:] = weights["weight"]
    assert torch.equal(method.apply_weights(dict(weights, weight=more[3:]), x), want)
    with pytest.raises(ValueError):  # not a copy of the row for each of its uses
        ops.fp4_quantize(x[:1].expand(4, K).transpose(0, 1), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 45, 200])
def test_shards_of_a_projection(cuda, fmt, M):
    """A rank's rows (column-parallel) or k (row-parallel) of weight and weight_scale, copied into
    the tensors of create_weights: the product of just those."""
    K, N, ranks, dtype = 1152, 528, 3, torch.bfloat16
    block = ops.FP4_BLOCK[fmt]
    loaded = quantize_weight(_normal(cuda, N, K, dtype=dtype, std=K ** -0.5), fmt)
    values, ws = values_ref(loaded["weight"], loaded["weight_scale"], fmt), loaded.get("weight_scale_2")
    x = _normal(cuda, M, K, dtype=dtype)
    method = get_quantization_config("fp4_b200")(fmt).get_linear_method()

    def shard(n, k):
        w = method.create_weights(k.stop - k.start, n.stop - n.start)
        for name, per in (("weight", 2), ("weight_scale", block)):
            w[name] = torch.nn.Parameter(w[name].data.to(cuda), requires_grad=False)
            w[name].data.copy_(loaded[name][n, k.start // per:k.stop // per])
        if fmt == "nvfp4":
            w["weight_scale_2"].data, w["input_scale"].data = ws.clone(), torch.full((1,), 0.01, device=cuda)
        w = method.process_weights_after_loading(w)
        xs = w.get("input_scale")
        y, bound = product_ref(_held(x[:, k], fmt, xs), values[n, k], xs, ws)
        got = method.apply_weights(w, x[:, k])
        assert within(got.cpu(), y, bound, dtype) <= 0

    for r in range(ranks):
        shard(slice(N // ranks * r, N // ranks * (r + 1)), slice(0, K))
        shard(slice(0, N), slice(K // ranks * r, K // ranks * (r + 1)))


@pytest.mark.parametrize("fmt", FORMATS)
def test_gate_up_and_quantised_rows(cuda, fmt):
    """The norm's rows straight into gate_up with SiLU-and-mul; the gate and up halves of the
    plain projection give the same."""
    K, I, M = 512, 200, 37
    method, weights, values, ws = _linear(cuda, fmt, K, 2 * I, torch.bfloat16, gate_up=True)
    x, r = _normal(cuda, M, K), _normal(cuda, M, K, seed=9)
    norm = RMSNormFP4(K, 1e-6, fmt, weights.get("input_scale"))
    norm.weight = (torch.rand(K, device=cuda) + 0.5).to(torch.bfloat16)
    want_r = (x.float() + r.float()).to(torch.bfloat16)
    rows, r2 = norm.forward(x, r)
    assert r2.data_ptr() == r.data_ptr() and torch.equal(r, want_r)
    xv = values_ref(rows[0], rows[1].cpu().transpose(0, 1).flatten(1)[:, : K // ops.FP4_BLOCK[fmt]], fmt)
    y, bound = product_ref(xv, values, weights.get("input_scale"), ws, None, True)
    got = method.apply_weights(weights, rows, dtype=torch.bfloat16, silu_mul=True)
    assert within(got.cpu(), y, bound, torch.bfloat16) <= 0
    only, same = norm.forward(x)
    assert same is x and only[0].shape == (M, K // 2)


def test_linear_method_with_adapters(cuda):
    K, N, M, rank = 256, 128, 9, 8
    method, weights, _, _ = _linear(cuda, "nvfp4", K, N, torch.bfloat16)
    x = _normal(cuda, M, K)
    pairs = [(_normal(cuda, rank, K, std=0.05, seed=l), _normal(cuda, N, rank, std=0.05, seed=l + 7)) for l in range(2)]
    adapters = LoraAdapters(torch.stack([a for a, _ in pairs]), torch.stack([b for _, b in pairs]), None, (N,))
    ids = torch.tensor([0, 1, -1, 0, 1, 1, -1, 0, 0], dtype=torch.int32, device=cuda)
    batch = LoraBatch(*ops.group_rows(ids, 2))
    plain = method.apply_weights(weights, x)
    got = method.apply_weights(weights, x, adapters=adapters, batch=batch)
    want = ops.lora(x, adapters.a, adapters.b, batch.order, batch.offsets, plain, slices=(N,))
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        method.apply_weights(weights, x, adapters=adapters)
    with pytest.raises(ValueError):
        method.apply_weights(weights, ops.fp4_quantize(x, "nvfp4"), adapters=adapters, batch=batch, dtype=torch.bfloat16)


# ---------------------------------------------------------------- experts
def _experts(cuda, E, N, K, fmt, gate_up, lo=0, n=None, seed=0):
    n = n or E
    w, s, scale = [], [], []
    for e in range(E):
        q = quantize_weight(_normal(cuda, N, K, std=K ** -0.5, seed=seed + 31 * e), fmt)
        w.append(q["weight"]), s.append(q["weight_scale"]), scale.append(q.get("weight_scale_2"))
    part = slice(lo, lo + n)
    nv = fmt == "nvfp4"
    return FP4ExpertWeights.from_checkpoint(
        torch.stack(w)[part], torch.stack(s)[part], fmt, torch.bfloat16, torch.cat(scale)[part] if nv else None,
        torch.full((1,), 0.004, device=cuda) if nv else None, lo, E, gate_up)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 7, 130])
def test_moe_backend(cuda, fmt, M):
    """The backend is its operators one after the other; its halves over two ranks add up to
    it; and it is within the formats' own error of the experts in 16 bits."""
    E, H, I, topk = 16, 256, 96, 4
    x = _normal(cuda, M, H, seed=M)
    logits = _normal(cuda, M, E, seed=5).float()
    w1, w2 = _experts(cuda, E, 2 * I, H, fmt, True), _experts(cuda, E, H, I, fmt, False, seed=1)
    backend = AWQB200MoeBackend()
    got = backend.forward(x.clone(), w1, w2, logits, topk, True)
    tw, ids = ops.moe_topk_softmax(logits, topk, True)
    y = torch.zeros((M, topk, H), device=cuda, dtype=torch.bfloat16)
    for k in range(topk):
        for e in range(E):
            rows = (ids[:, k] == e).nonzero()[:, 0]
            if not rows.numel():
                continue
            one = lambda w: dict(x_scale=w.x_scale, w_scale=None if w.w_scale is None else w.w_scale[e:e + 1].contiguous())
            q = ops.fp4_quantize(x[rows].contiguous(), fmt, scale=w1.x_scale)
            a = ops.fp4_gemm(*q, w1.w[e], w1.w_scales[e], fmt, torch.bfloat16, silu_mul=True, **one(w1))
            q = ops.fp4_quantize(a, fmt, scale=w2.x_scale)
            off = torch.tensor([0, rows.numel()], dtype=torch.int32, device=cuda)
            kw = one(w2)
            y[rows, k] = ops.fp4_grouped_gemm(*q, w2.w[e:e + 1].contiguous(), w2.w_scales[e:e + 1].contiguous(), off, fmt,
                                              torch.bfloat16, row_scale=tw[rows, k].contiguous(), **kw)
    want = ops.moe_topk_sum(y.view(M * topk, H), M, topk, ids, 0, E, torch.empty_like(x))
    # (sums of another order of tiles: a rounding of an intermediate may fall the other way)
    scale = want.float().abs().max()
    assert float((got.float() - want.float()).abs().max() / scale) <= 0.05
    assert float((got.float() - want.float()).norm() / want.float().norm()) <= 0.01
    parts = torch.zeros((M, H), device=cuda)
    for lo in (0, E // 2):
        p1 = _experts(cuda, E, 2 * I, H, fmt, True, lo, E // 2)
        p2 = _experts(cuda, E, H, I, fmt, False, lo, E // 2, seed=1)
        parts += backend.forward(x.clone(), p1, p2, logits, topk, True).float()
    # each half is rounded to 16 bits, and so is the whole
    room = 4 * half_step(torch.bfloat16) * got.float().abs().max()
    assert float((parts - got.float()).abs().max()) <= float(room)
    d1 = torch.stack([_normal(cuda, 2 * I, H, std=H ** -0.5, seed=31 * e) for e in range(E)])
    d2 = torch.stack([_normal(cuda, H, I, std=I ** -0.5, seed=1 + 31 * e) for e in range(E)])
    dense = backend.forward(x.clone(), d1, d2, logits, topk, True).float()
    # two factors in four bits in each product: about 0.13 each (a uniform block's rounding), four in all
    assert float((got.float() - dense).norm() / dense.norm()) <= 0.5


def test_moe_backend_refuses_mixed_experts(cuda):
    w1, w2 = _experts(cuda, 4, 128, 64, "nvfp4", True), _experts(cuda, 4, 64, 64, "nvfp4", False)
    x, logits = _normal(cuda, 3, 64), torch.zeros((3, 4), device=cuda)
    backend = AWQB200MoeBackend()
    with pytest.raises(ValueError, match="both"):
        backend.forward(x, w1, DenseExpertWeights(_normal(cuda, 4, 64, 64)), logits, 2, True)
    with pytest.raises(ValueError):
        backend.forward(x.half(), w1, w2, logits, 2, True)
    empty = backend.experts(x[:0], w1, w2, torch.zeros((0, 2), device=cuda), torch.zeros((0, 2), dtype=torch.int32, device=cuda))
    assert empty.shape == (0, 64)


# ---------------------------------------------------------------- a block
class _Block:
    """norm -> projection -> norm -> gate_up -> down, and a mixture behind it."""

    def __init__(self, cuda, fmt, H=512, I=768, E=8):
        self.fmt, self.H = fmt, H
        self.o = _linear(cuda, fmt, H, H, torch.bfloat16, seed=1)
        self.gu = _linear(cuda, fmt, H, 2 * I, torch.bfloat16, seed=2, gate_up=True)
        self.down = _linear(cuda, fmt, I, H, torch.bfloat16, seed=3)
        self.norms = [RMSNormFP4(H, 1e-6, fmt, w[1].get("input_scale")) for w in (self.o, self.gu)]
        for n in self.norms:
            n.weight = torch.ones(H, dtype=torch.bfloat16, device=cuda)
        self.w1, self.w2 = _experts(cuda, E, 256, H, fmt, True), _experts(cuda, E, H, 128, fmt, False, seed=4)
        self.router = _normal(cuda, E, H, std=0.1)

    def __call__(self, x, residual):
        r = residual.clone()
        T = torch.bfloat16
        rows, r = self.norms[0].forward(x, r)
        y = self.o[0].apply_weights(self.o[1], rows, dtype=T)
        rows, r = self.norms[1].forward(y, r)
        a = self.gu[0].apply_weights(self.gu[1], rows, dtype=T, silu_mul=True)
        y = self.down[0].apply_weights(self.down[1], a)
        z = AWQB200MoeBackend().forward(y.clone(), self.w1, self.w2, (y @ self.router.T).float(), 2, True)
        return y + z, r


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 16, 77, 300])
def test_block_in_a_graph_and_on_other_streams(cuda, fmt, M):
    """Eager, captured (two graphs over the same weights, replayed by turns with new
    inputs) and on a side stream beside another call: the same bits."""
    block = _Block(cuda, fmt)
    ins = [(_normal(cuda, M, 512, seed=s), _normal(cuda, M, 512, seed=s + 50)) for s in range(4)]
    want = [block(*i) for i in ins]
    graphs = []
    for _ in range(2):
        at = [t.clone() for t in ins[0]]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            block(*at)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block(*at)
        graphs.append((g, at, out))
    for k in (1, 2, 3, 0, 2):
        for n, (g, at, out) in enumerate(graphs):
            for a, b in zip(at, ins[(k + n) % 4]):
                a.copy_(b)
            g.replay()
        torch.cuda.synchronize()
        for n, (g, at, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(k + n) % 4]))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s, i in zip(streams, ins):
        with torch.cuda.stream(s):
            got.append([block(*i) for _ in range(3)])
    torch.cuda.synchronize()
    for three, w in zip(got, want):
        for o in three:
            assert all(torch.equal(a, b) for a, b in zip(o, w))
    assert ops.device_error() == 0


def test_host_threads(cuda):
    """Calls from several host threads, their first ones among them."""
    import threading

    c = [_normal(cuda, m, 320, seed=m) for m in (1, 40, 200)]
    method, weights, _, _ = _linear(cuda, "nvfp4", 320, 1000, torch.bfloat16)
    want = [method.apply_weights(weights, x) for x in c]
    torch.cuda.synchronize()
    bad = []

    def work(n):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for k in range(30):
                y = method.apply_weights(weights, c[(n + k) % 3])
                s.synchronize()
                if not torch.equal(y, want[(n + k) % 3]):
                    bad.append((n, k))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


# ---------------------------------------------------------------- far offsets
@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_past_32_bit_offsets(cuda, fmt):
    """More than 2^31 values and more than 2^31 bytes of codes."""
    M, K = 270001, 16384
    x = torch.zeros((M, K), dtype=torch.float16, device=cuda)
    tail = _normal(cuda, 5, K, dtype=torch.float16)
    x[-5:] = tail
    codes, scales = ops.fp4_quantize(x, fmt)
    want, near = ops.fp4_quantize(tail, fmt), (codes[-5:], scales[:, -5:])
    assert torch.equal(near[0], want[0]) and torch.equal(near[1], want[1]) and not codes[:-5].any()
    del x
    back = ops.fp4_dequantize(codes, scales, fmt, torch.float16)
    assert torch.equal(back[-5:], ops.fp4_dequantize(*want, fmt, torch.float16)) and not back[-6].any()


@pytest.mark.parametrize("fmt", FORMATS)
def test_products_past_32_bit_offsets(cuda, fmt):
    """An output of more than 2^31 values, and experts of more than 2^31 bytes."""
    M, K, N = 140000, 64, 16384
    x = _normal(cuda, M, K)
    q = ops.fp4_quantize(x, fmt)
    w = quantize_weight(_normal(cuda, N, K), fmt)
    laid = ops.fp4_lay_out_scales(w["weight_scale"], fmt)
    y = ops.fp4_gemm(*q, w["weight"], laid, fmt, torch.bfloat16)
    last = ops.fp4_quantize(x[-3:].contiguous(), fmt)
    assert torch.equal(y[-3:], ops.fp4_gemm(*last, w["weight"], laid, fmt, torch.bfloat16))
    del y
    E, K, N = 70, 8192, 8192
    codes = torch.randint(0, 256, (E, N, K // 2), dtype=torch.uint8, device=cuda)
    byte = torch.full((E, N, K // ops.FP4_BLOCK[fmt]), 50 if fmt == "nvfp4" else 120, dtype=torch.uint8, device=cuda)
    laid = ops.fp4_lay_out_scales(byte, fmt)
    q = ops.fp4_quantize(_normal(cuda, E, K), fmt)
    off = torch.arange(E + 1, dtype=torch.int32, device=cuda)
    y = ops.fp4_grouped_gemm(*q, codes, laid, off, fmt, torch.bfloat16)
    one = (q[0][-1:].contiguous(), q[1][:, -1:].contiguous())
    want = ops.fp4_gemm(*one, codes[-1], laid[-1], fmt, torch.bfloat16)
    err = (y[-1:].float() - want.float()).abs().max() / want.float().abs().max()
    assert float(err) <= 2 * half_step(torch.bfloat16)  # (K is shared there: sums of another order)
