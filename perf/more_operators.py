"""What microscaled 4-bit floating point costs: quantisation, reading back, products.

Two formats of e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) that
share a scale along K: ``nvfp4``, 16 values with an e4m3 scale and one fp32 scale
for the whole tensor, and ``mxfp4``, 32 values with a power of two (e8m0).

Five operators: rows quantised and read back (``quantize``: ``fp4_quantize`` with the
rows of a mixture's experts gathered on the way, and ``fp4_dequantize``), the
residual-add RMSNorm that writes quantised rows (``norm``), the product of
quantised rows and weights (``gemm``) and the same grouped by expert (``grouped``).
``run`` computes them with elementary torch operations in 32 bits, or, with ``own``
set, through ``sglite_b200.ops``. What is held in 4 bits is returned as the
values it stands for. Sizes are those of the projections and experts that the
benchmark and the tests use (hidden sizes 2048, 4096, 8192; gate_up of 28672;
128 experts with 768 features), or generic ones.

Layouts, the same for both sides. Rows: ``codes`` uint8 [rows, K / 2], the value with
the even k in the low four bits; ``scales`` uint8 [granules, rows, 16], 16 scales
of a row side by side (256 k of nvfp4, 512 k of mxfp4), zero past K. Weights: codes
[N, K / 2]; their scales as a checkpoint has them, [N, K / 16 or K / 32], and laid out
once for the tensor cores, [N / 128, K / 256, 4 or 2, 32, 4, 4]: tiles of 128 rows
by four scales, rows r, r + 32, r + 64 and r + 96 side by side.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def listed():
    return [
        # One decoding token on its way into a projection.
        {"name": "quantise 1 token", "op": "quantize", "fmt": "nvfp4", "dtype": "bf16", "M": 1, "K": 4096, "topk": 0},
        # A decode step of 256 tokens gathered for the top 8 of its experts.
        {"name": "quantise for experts", "op": "quantize", "fmt": "nvfp4", "dtype": "bf16", "M": 256, "K": 2048, "topk": 8},
        # A prompt in front of the down projection.
        {"name": "quantise 4096 tokens", "op": "quantize", "fmt": "mxfp4", "dtype": "fp16", "M": 4096, "K": 14336, "topk": 0},
        # One token between two blocks: residual add, norm, and the next projection's input.
        {"name": "norm 1 token", "op": "norm", "fmt": "nvfp4", "dtype": "bf16", "M": 1, "K": 4096},
        # A prompt through the wide model's norms.
        {"name": "norm 4096 tokens", "op": "norm", "fmt": "mxfp4", "dtype": "bf16", "M": 4096, "K": 8192},
        # One decoding token, the merged QKV projection.
        {"name": "gemm 1 token qkv", "op": "gemm", "fmt": "nvfp4", "dtype": "bf16", "M": 1, "K": 4096, "N": 6144, "silu": False,
         "bias": False},
        # A decode batch of 32 through gate_up with SiLU-and-mul.
        {"name": "gemm 32 tokens gate_up", "op": "gemm", "fmt": "nvfp4", "dtype": "bf16", "M": 32, "K": 4096, "N": 28672,
         "silu": True, "bias": False},
        # A ragged chunk of a prompt, the down projection with a bias.
        {"name": "gemm 333 tokens down", "op": "gemm", "fmt": "mxfp4", "dtype": "fp16", "M": 333, "K": 14336, "N": 4096,
         "silu": False, "bias": True},
        # A prompt of 4096 tokens through the wide model's gate_up.
        {"name": "gemm 4096 tokens gate_up", "op": "gemm", "fmt": "nvfp4", "dtype": "bf16", "M": 4096, "K": 8192, "N": 28672,
         "silu": False, "bias": False},
        # One decode step of 16 tokens through 128 experts (top 8): most experts that are hit have one or two rows.
        {"name": "experts 16 tokens gate_up", "op": "grouped", "fmt": "nvfp4", "dtype": "bf16", "rows": 128, "K": 2048, "N": 1536,
         "E": 128, "silu": True, "pad": 0, "scatter": False},
        # A decode step of 256 tokens, the down projection with the router weights, scattered back to token order.
        {"name": "experts 256 tokens down", "op": "grouped", "fmt": "mxfp4", "dtype": "bf16", "rows": 2048, "K": 768, "N": 2048,
         "E": 128, "silu": False, "pad": 0, "scatter": True},
        # A prompt of 4096 tokens, gate_up of 128 experts, in a padded buffer: rows behind the last group stay.
        {"name": "experts 4096 tokens gate_up", "op": "grouped", "fmt": "nvfp4", "dtype": "fp16", "rows": 32768, "K": 2048,
         "N": 1536, "E": 128, "silu": True, "pad": 81, "scatter": False},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quantize", "norm", "gemm", "gemm", "grouped", "grouped"])
    head = {"op": op, "fmt": rng.choice(["nvfp4", "mxfp4"]), "dtype": rng.choice(["bf16", "fp16"])}
    if op == "quantize":
        M, K, topk = _log(rng, 1, 8192), _log(rng, 32, 16384, 32), rng.choice([0, 0, 1, 2, 8])
        while M * max(1, topk) * K > 6e7:
            M = max(1, M // 2)
        return {**head, "M": M, "K": K, "topk": topk}
    if op == "norm":
        return {**head, "M": _log(rng, 1, 4096), "K": _log(rng, 32, 16384, 32)}
    K = _log(rng, 32, 14336, 32)
    silu = rng.random() < 0.4
    if op == "gemm":
        M, N = _log(rng, 1, 8192), _log(rng, 32, 28672, 16)
        while M * K * N > 9e11:
            M //= 2
        return {**head, "M": M, "K": K, "N": N, "silu": silu, "bias": rng.random() < 0.3}
    N, E = _log(rng, 32, 14336, 16), _log(rng, 1, 160)
    while E * K * N > 4e8:
        E = max(1, E // 2)
    rows = _log(rng, 1, 32768)
    while rows * K * N > 4e11:
        rows //= 2
    return {**head, "rows": rows, "K": K, "N": N, "E": E, "silu": silu, "pad": rng.choice([0, 0, 1, 37, 200]),
            "scatter": not silu and rng.random() < 0.4}


# ---------------------------------------------------------------- the formats, in 32 bits
def _power(byte):
    """2^(byte - 127), exactly, for int32 bytes 0 .. 254."""
    return torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)


def _e2m1(v):
    """|v| to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6; ties to the even code; 6 above."""
    return torch.where(v < 2, torch.round(2 * v) / 2, torch.where(v < 4, torch.round(v), 2 * torch.round(v / 2))).clamp(max=6.0)


def _parts(u, fmt):
    """u [.., K] in 32 bits (nvfp4: already over the tensor's scale) -> (e2m1 values,
    the blocks' scales as numbers, [.., blocks, 1]), both with the block's values last."""
    b = u.unflatten(-1, (-1, BLOCK[fmt]))
    most = b.abs().amax(-1, keepdim=True)
    if fmt == "nvfp4":
        s = (most / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn).float()
    else:  # the power of two two below the largest value's own
        s = _power((torch.frexp(most)[1] + 124).clamp(min=0) * (most > 0))
    v = torch.where(s > 0, b / torch.where(s > 0, s, 1.0), 0.0)
    return torch.copysign(_e2m1(v.abs()), v), s


def _read_back(u, fmt, scale, dtype):
    v, s = _parts(u, fmt)
    w = (v * s).flatten(-2)
    return (w if scale is None else w * scale).to(dtype)


def _bytes(u, fmt):
    """u [rows, K] -> (codes [rows, K / 2], scales [rows, K / block]), uint8."""
    v, s = _parts(u, fmt)
    a = v.abs().flatten(-2)
    code = (a * 2).where(a < 2, (a + 2).where(a < 4, a / 2 + 4)).to(torch.uint8) | (torch.signbit(v.flatten(-2)).to(torch.uint8) << 3)
    pair = code.unflatten(-1, (-1, 2))
    s = s[..., 0]
    byte = s.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "nvfp4" else (torch.frexp(s)[1] + 126).to(torch.uint8)
    return pair[..., 0] | (pair[..., 1] << 4), byte


def _numbers(codes, scales, fmt):
    """The values [.., K] in 32 bits that codes [.., K / 2] and scales [.., K / block] stand for."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], dim=-1).flatten(-2)
    s = scales.view(torch.float8_e4m3fn).float() if fmt == "nvfp4" else _power(scales.int())
    return (v.unflatten(-1, (-1, BLOCK[fmt])) * s[..., None]).flatten(-2)


def _granules(scales):
    """Scales [rows, K / block] -> [granules, rows, 16], zero past K."""
    rows, n = scales.shape
    wide = torch.zeros((rows, (n + 15) // 16 * 16), dtype=torch.uint8, device=scales.device)
    wide[:, :n] = scales
    return wide.view(rows, -1, 16).transpose(0, 1).contiguous()


def _laid_out(scales, fmt):
    """Scales [E, N, K / block] -> [E, N / 128, K / 256, 4 or 2, 32, 4, 4], rounded up, zero past N and K."""
    E, N, n = scales.shape
    per = 256 // BLOCK[fmt]
    wide = torch.zeros((E, (N + 127) // 128 * 128, (n + per - 1) // per * per), dtype=torch.uint8, device=scales.device)
    wide[:, :N, :n] = scales
    t = wide.view(E, -1, 4, 32, wide.shape[2] // per, per // 4, 4)  # [E, tile, row / 32, row % 32, stage, k tile, 4]
    return t.permute(0, 1, 4, 5, 3, 2, 6).contiguous()


# ---------------------------------------------------------------- inputs
def _sizes(total, groups, salt):
    """How many of ``total`` rows each of ``groups`` gets: skewed, some none; by the case alone."""
    rng = random.Random(total * 1000003 + groups * 101 + salt)
    weight = [rng.random() ** 2 + 0.05 for _ in range(groups)]
    count = [0] * groups
    for g in rng.choices(range(groups), weight, k=total):
        count[g] += 1
    return count


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    rng = random.Random(int(seed))
    T, fmt, K, op = DTYPES[case["dtype"]], case["fmt"], case["K"], case["op"]

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, std, generator=g)

    def over_all(most):  # the scale of a tensor whose largest magnitude is about `most`
        return torch.full((1,), most / (6.0 * 448.0), device=dev) * (1 + 0.1 * torch.rand(1, generator=g, device=dev))

    channel = torch.where(torch.rand(K, generator=g, device=dev) < 0.01, 20.0, 1.0)  # a few large channels
    s = {"case": case, "scale": over_all(90.0) if fmt == "nvfp4" else None}
    if op == "quantize":
        s["x"] = (normal(case["M"], K) * channel).to(T)
        s["index"] = None
        if case["topk"]:  # the tokens in the order of the experts that they go to
            s["index"] = torch.randperm(case["M"] * case["topk"], generator=g, device=dev).to(torch.int32)
        return s
    if op == "norm":
        s["x"] = (normal(case["M"], K) * channel).to(T)
        s["residual"] = (normal(case["M"], K) * channel * 2).to(T)
        s["weight"] = (torch.rand(K, generator=g, device=dev) + 0.5).to(T)
        return s
    M, N, E = (case["M"], case["N"], 1) if op == "gemm" else (case["rows"] + case["pad"], case["N"], case["E"])
    x = normal(M, K) * channel
    s["x"], scales = _bytes(x if s["scale"] is None else x / s["scale"], fmt)
    s["xs"] = _granules(scales)
    s["w_scale"] = None
    if fmt == "nvfp4":
        s["w_scale"] = torch.cat([over_all(5.5 * K ** -0.5) for _ in range(E)])
    w, ws = [], []
    for e in range(E):
        v = normal(N, K, std=K ** -0.5)
        a, b = _bytes(v if fmt == "mxfp4" else v / s["w_scale"][e], fmt)
        w.append(a)
        ws.append(b)
    s["w"], s["ws"] = torch.stack(w), torch.stack(ws)  # with silu, gate and up rows by turns
    s["ws_laid"] = _laid_out(s["ws"], fmt)
    n_out = N // 2 if case["silu"] else N
    if op == "gemm":
        s["bias"] = normal(N, dtype=T) if case["bias"] else None
        return s
    sizes = _sizes(case["rows"], E, 1)
    rng.shuffle(sizes)
    s["offsets"] = torch.tensor([0] + sizes, dtype=torch.int64).cumsum(0).to(device=dev, dtype=torch.int32)
    s["most"], s["out"], s["row_map"], s["row_scale"] = max(sizes), normal(M, n_out, dtype=T), None, None
    if case["scatter"]:  # rows go back to their (token, choice) place with the router's weight
        s["row_map"] = torch.randperm(M, generator=g, device=dev).to(torch.int32)
        s["row_scale"] = torch.rand(M, generator=g, device=dev)
    return s


# ---------------------------------------------------------------- the operators
def run(s):
    c = s["case"]
    T, fmt = DTYPES[c["dtype"]], c["fmt"]
    if own:
        from sglite_b200 import ops

        if c["op"] == "quantize":
            codes, scales = ops.fp4_quantize(s["x"], fmt, scale=s["scale"], index=s["index"], per_row=max(1, c["topk"]))
            return ops.fp4_dequantize(codes, scales, fmt, T, scale=s["scale"])
        if c["op"] == "norm":
            codes, scales, h = ops.fp4_add_rmsnorm(s["x"], s["residual"], s["weight"], 1e-6, fmt, scale=s["scale"])
            return ops.fp4_dequantize(codes, scales, fmt, T, scale=s["scale"]), h
        if c["op"] == "gemm":
            return ops.fp4_gemm(s["x"], s["xs"], s["w"][0], s["ws_laid"][0], fmt, T, x_scale=s["scale"], w_scale=s["w_scale"],
                                bias=s["bias"], silu_mul=c["silu"])
        return ops.fp4_grouped_gemm(s["x"], s["xs"], s["w"], s["ws_laid"], s["offsets"], fmt, T, x_scale=s["scale"],
                                    w_scale=s["w_scale"], out=s["out"], silu_mul=c["silu"], row_map=s["row_map"],
                                    row_scale=s["row_scale"])
    return {"quantize": _quantize, "norm": _norm, "gemm": _gemm, "grouped": _grouped}[c["op"]](s)


def _over(u, s):
    return u if s["scale"] is None else u * (1.0 / s["scale"])


def _quantize(s):
    c = s["case"]
    x = s["x"] if s["index"] is None else s["x"][s["index"].long() // c["topk"]]
    return _read_back(_over(x.float(), s), c["fmt"], s["scale"], s["x"].dtype)


def _norm(s):
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    return _read_back(_over(y, s), s["case"]["fmt"], s["scale"], s["x"].dtype), h.to(s["x"].dtype)


def _rows(s):
    K = s["case"]["K"]
    scales = s["xs"].transpose(0, 1).flatten(1)[:, : K // BLOCK[s["case"]["fmt"]]]
    x = _numbers(s["x"], scales, s["case"]["fmt"])
    return x if s["scale"] is None else x * s["scale"]


def _weights(s, e):
    w = _numbers(s["w"][e], s["ws"][e], s["case"]["fmt"])
    return w if s["w_scale"] is None else w * s["w_scale"][e]


def _silu_mul(y):
    gate, up = y[..., 0::2], y[..., 1::2]
    return gate / (1.0 + torch.exp(-gate)) * up


def _gemm(s):
    c = s["case"]
    y = _rows(s) @ _weights(s, 0).T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["silu"]:
        y = _silu_mul(y)
    return y.to(DTYPES[c["dtype"]])


def _grouped(s):
    c = s["case"]
    at = s["offsets"][:-1, None].long() + torch.arange(s["most"], device=s["x"].device)
    real = at < s["offsets"][1:, None]
    x = _rows(s)
    w = _numbers(s["w"], s["ws"], c["fmt"])
    if s["w_scale"] is not None:
        w = w * s["w_scale"][:, None, None]
    y = torch.bmm(x[torch.where(real, at, 0)], w.transpose(1, 2))
    if c["silu"]:
        y = _silu_mul(y)
    y = y[real]  # group after group: rows offsets[0] .. offsets[E]
    if c["scatter"]:
        to = s["row_map"][: y.shape[0]].long()
        s["out"][to] = (y * s["row_scale"][to][:, None]).to(s["out"].dtype)
    else:
        s["out"][: y.shape[0]] = y.to(s["out"].dtype)
    return s["out"]


# ---------------------------------------------------------------- in 64 bits, from the definitions
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _two_to(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _below(v):
    """e with 2^e <= v < 2^(e + 1)."""
    return torch.frexp(v)[1] - 1


def _exact_blocks(u, fmt):
    """u [.., K] in 64 bits -> the values that its blocks are held as."""
    b = u.unflatten(-1, (-1, BLOCK[fmt]))
    most = b.abs().amax(-1, keepdim=True)
    if fmt == "nvfp4":  # three bits after the leading one, steps of 2^-9 below 2^-6
        q = (most / 6).clamp(max=448.0)
        step = _two_to(_below(q.clamp(min=2.0 ** -6)) - 3)
        s = torch.round(q / step) * step
    else:
        s = _two_to(_below(most.clamp(min=2.0 ** -125)) - 2)
    v = torch.where(s > 0, b.abs() / s, 0.0)
    held = torch.zeros_like(v)
    for i in range(1, 8):  # above the middle between two, or on it where the upper one's code is even
        middle = (_GRID[i - 1] + _GRID[i]) / 2
        held = torch.where((v > middle) | ((v == middle) & (i % 2 == 0)), _GRID[i], held)
    return (torch.sign(b) * held * s).flatten(-2)


def _exact_held(u, s):
    k = 1.0 if s["scale"] is None else s["scale"].double()
    return _exact_blocks(u / k, s["case"]["fmt"]) * k


def _exact_numbers(codes, scales, fmt):
    grid = torch.tensor(_GRID, dtype=torch.float64, device=codes.device)
    both = torch.stack([codes % 16, codes // 16], dim=-1).flatten(-2).long()
    v = grid[both % 8] * (1 - 2 * (both // 8))
    b = scales.double()
    if fmt == "nvfp4":
        e = torch.floor(b / 8)
        s = torch.where(e > 0, _two_to(e - 7) * (1 + (b - 8 * e) / 8), b * 2.0 ** -9)
    else:
        s = _two_to(b - 127)
    return v * s.repeat_interleave(BLOCK[fmt], dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    fmt, K = case["fmt"], case["K"]
    if case["op"] == "quantize":
        x = s["x"].double()
        if s["index"] is not None:
            x = x.repeat_interleave(case["topk"], dim=0)[s["index"].long()]
        return _exact_held(x, s)
    if case["op"] == "norm":
        h = s["x"].double() + s["residual"].double()
        return _exact_held(h / (h.pow(2).sum(1, keepdim=True) / K + 1e-6).sqrt() * s["weight"].double(), s), h
    scales = torch.cat(list(s["xs"]), dim=1)[:, : K // BLOCK[fmt]]
    x = _exact_numbers(s["x"], scales, fmt) * (1.0 if s["scale"] is None else s["scale"].double())

    def product(rows, e):
        y = rows @ _exact_numbers(s["w"][e], s["ws"][e], fmt).T * (1.0 if s["w_scale"] is None else s["w_scale"][e].double())
        if case["op"] == "gemm" and s["bias"] is not None:
            y = y + s["bias"].double()
        if case["silu"]:
            y = y.unflatten(-1, (-1, 2))
            y = y[..., 0] * torch.sigmoid(y[..., 0]) * y[..., 1]
        return y

    if case["op"] == "gemm":
        return product(x, 0)
    out, at = s["out"].double(), s["offsets"].tolist()
    for e in range(case["E"]):
        y = product(x[at[e] : at[e + 1]], e)
        if case["scatter"]:
            to = s["row_map"][at[e] : at[e + 1]].long()
            out[to] = y * s["row_scale"].double()[to, None]
        else:
            out[at[e] : at[e + 1]] = y
    return out


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once."""
    K, two = case["K"], 2  # bytes of a bf16 or fp16 value
    four = 0.5 + 1.0 / BLOCK[case["fmt"]]  # bytes of a value of four bits with its share of the scale
    if case["op"] == "quantize":
        rows = case["M"] * max(1, case["topk"])
        return {"bytes": two * case["M"] * K + rows * K * (four + two), "flops": 6.0 * rows * K}
    if case["op"] == "norm":
        return {"bytes": case["M"] * K * (4 * two + four), "flops": 12.0 * case["M"] * K}
    N = case["N"]
    n_out = N // 2 if case["silu"] else N
    if case["op"] == "gemm":
        M = case["M"]
        return {"bytes": (M + N) * K * four + two * M * n_out, "flops": 2.0 * M * N * K}
    rows = case["rows"]
    hit = sum(1 for n in _sizes(rows, case["E"], 1) if n)
    return {"bytes": (rows + hit * N) * K * four + two * rows * n_out, "flops": 2.0 * rows * N * K}
