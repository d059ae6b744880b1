"""What the decoder-block operators around the AWQ projections cost.

Four operators: matrix products grouped by expert over 16-bit weights
(``grouped``), low-rank adapters of many requests beside a shared projection
(``lora``), the norms around a block with its gate and residual scale
(``norm``) and rotary positions with the per-head q/k norm (``rotary``).
``run`` computes them with elementary torch operations in 32 bits, or, with
``own`` set, through ``sglite_b200.ops``. Sizes are those of the projections and
experts that the benchmark and the tests use (hidden sizes 2048, 2560, 4096,
8192; 128 experts with 768 features; 32 query and 8 key/value heads of 128), or
generic ones.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One decode step of 16 tokens through 128 experts (top-8): most experts that are hit have one or two rows.
        {"name": "experts 16 tokens gate_up", "op": "grouped", "dtype": "bf16", "rows": 128, "K": 2048, "N": 1536, "E": 128,
         "silu": True, "pad": 0, "scatter": False},
        # A decode step of 256 tokens, the down projection with the router weights, scattered back to token order.
        {"name": "experts 256 tokens down", "op": "grouped", "dtype": "bf16", "rows": 2048, "K": 768, "N": 2048, "E": 128,
         "silu": False, "pad": 0, "scatter": True},
        # A prompt of 4096 tokens, gate_up of 128 experts.
        {"name": "experts 4096 tokens gate_up", "op": "grouped", "dtype": "bf16", "rows": 32768, "K": 2048, "N": 1536,
         "E": 128, "silu": True, "pad": 0, "scatter": False},
        # Eight wide experts over a long prompt in a padded buffer (a captured graph's): rows behind the last group stay.
        {"name": "eight wide experts", "op": "grouped", "dtype": "fp16", "rows": 8111, "K": 4096, "N": 14336, "E": 8,
         "silu": False, "pad": 81, "scatter": False},
        # One request decoding with its adapter on the merged QKV projection.
        {"name": "adapter 1 token qkv", "op": "lora", "dtype": "bf16", "requests": 1, "tokens": 1, "K": 4096, "N0": 4096,
         "N1": 1024, "N2": 1024, "rank": 16, "adapters": 4, "plain": 0.0},
        # 64 requests decoding with 32 adapters on the down projection, some of them without one.
        {"name": "adapters 64 requests down", "op": "lora", "dtype": "bf16", "requests": 64, "tokens": 64, "K": 14336,
         "N0": 4096, "N1": 0, "N2": 0, "rank": 32, "adapters": 32, "plain": 0.15},
        # A mixed prefill of 4111 tokens of 11 requests on the merged gate_up projection.
        {"name": "adapters prefill gate_up", "op": "lora", "dtype": "fp16", "requests": 11, "tokens": 4111, "K": 4096,
         "N0": 14336, "N1": 14336, "N2": 0, "rank": 64, "adapters": 5, "plain": 0.1},
        # One token between two blocks: post-norm, gate and the next block's norm.
        {"name": "norms 1 token", "op": "norm", "dtype": "bf16", "res": "bf16", "M": 1, "N": 4096, "post": True, "pre": True,
         "gate": "channel", "act": "tanh", "scale": 1.0, "offset": 1.0},
        # A prompt through the wide model's norms, gated element by element.
        {"name": "norms 4096 tokens", "op": "norm", "dtype": "bf16", "res": "fp32", "M": 4096, "N": 8192, "post": True,
         "pre": True, "gate": "element", "act": "sigmoid", "scale": 0.22, "offset": 0.0},
        # One decoding token: q and k out of the merged projection's output, with the q/k norm.
        {"name": "rotary 1 token", "op": "rotary", "dtype": "bf16", "M": 1, "Hq": 32, "Hk": 8, "D": 128, "rot": 128,
         "interleaved": False, "qknorm": True, "far": 32768},
        # A ragged decode batch, interleaved, half of each head, far positions.
        {"name": "rotary 333 tokens part", "op": "rotary", "dtype": "fp16", "M": 333, "Hq": 64, "Hk": 8, "D": 128, "rot": 64,
         "interleaved": True, "qknorm": False, "far": 1048576},
        # A prompt's positions.
        {"name": "rotary 8192 tokens", "op": "rotary", "dtype": "bf16", "M": 8192, "Hq": 32, "Hk": 8, "D": 128, "rot": 128,
         "interleaved": False, "qknorm": True, "far": 131072},
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["grouped", "lora", "norm", "rotary"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "grouped":
        silu = rng.random() < 0.4
        K, N, E = _log(rng, 64, 8192, 8), _log(rng, 64, 14336, 16), _log(rng, 1, 160)
        while E * K * N > 5e8:
            E = max(1, E // 2)
        rows = _log(rng, 1, 32768)
        while rows * K * N > 4e11:
            rows //= 2
        return {"op": op, "dtype": dtype, "rows": rows, "K": K, "N": N, "E": E, "silu": silu,
                "pad": rng.choice([0, 0, 1, 37, 200]), "scatter": not silu and rng.random() < 0.4}
    if op == "lora":
        requests = _log(rng, 1, 128)
        tokens = max(requests, _log(rng, 1, 4096))
        parts = rng.choice([1, 1, 2, 3])
        N = [_log(rng, 64, 8192, 8) if i < parts else 0 for i in range(3)]
        return {"op": op, "dtype": dtype, "requests": requests, "tokens": tokens, "K": _log(rng, 64, 14336, 8), "N0": N[0],
                "N1": N[1], "N2": N[2], "rank": rng.choice([8, 16, 24, 32, 64, 128]), "adapters": _log(rng, 1, 64),
                "plain": rng.choice([0.0, 0.1, 0.5])}
    if op == "norm":
        pre = rng.random() < 0.85
        gate = rng.choice(["none", "channel", "row", "element"])
        return {"op": op, "dtype": dtype, "res": rng.choice([dtype, dtype, "fp32"]), "M": _log(rng, 1, 4096),
                "N": _log(rng, 64, 8192, 8), "post": rng.random() < 0.6 or not pre, "pre": pre, "gate": gate,
                "act": rng.choice(["none", "sigmoid", "tanh", "silu"]) if gate != "none" else "none",
                "scale": rng.choice([1.0, 0.22, -0.5]), "offset": rng.choice([0.0, 1.0])}
    D = rng.choice([64, 80, 96, 128, 128, 192, 256])
    M, Hq = _log(rng, 1, 8192), rng.choice([1, 7, 8, 16, 32, 40, 64])
    while M * Hq * D > 4.0e7:
        M = max(1, M // 2)
    return {"op": op, "dtype": dtype, "M": M, "Hq": Hq, "Hk": rng.choice([1, 2, 4, 8]), "D": D,
            "rot": rng.choice([D, D, D // 2, 16, 20]), "interleaved": rng.random() < 0.5, "qknorm": rng.random() < 0.5,
            "far": _log(rng, 1, 4194304)}


# ---------------------------------------------------------------- inputs
def _sizes(total, groups, salt):
    """How many of ``total`` rows each of ``groups`` gets: skewed, some none; by the case alone."""
    rng = random.Random(total * 1000003 + groups * 101 + salt)
    weight = [rng.random() ** 2 + 0.05 for _ in range(groups)]
    count = [0] * groups
    for g in rng.choices(range(groups), weight, k=total):
        count[g] += 1
    return count


def _lora_rows(case):
    """Tokens of each request and its adapter (-1: none), by the case alone."""
    R, M, L = case["requests"], case["tokens"], case["adapters"]
    rng = random.Random(M * 7919 + R * 31 + L)
    length = [1 + c for c in _sizes(M - R, R, 5)]
    adapter = [-1 if rng.random() < case["plain"] else rng.randrange(L) for _ in range(R)]
    return length, adapter


def _slices(case):
    return tuple(case[n] for n in ("N0", "N1", "N2") if case[n])


def _offsets(sizes, device):
    return torch.tensor([0] + sizes, dtype=torch.int64).cumsum(0).to(device=device, dtype=torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    rng = random.Random(int(seed))
    T = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=T):
        return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, std, generator=g)

    op = case["op"]
    if op == "grouped":
        rows, K, N, E = case["rows"], case["K"], case["N"], case["E"]
        sizes = _sizes(rows, E, 1)
        rng.shuffle(sizes)
        n_out = N // 2 if case["silu"] else N
        total = rows + case["pad"]
        s = {"case": case, "x": normal(total, K), "w": normal(E, N, K, std=K ** -0.5), "offsets": _offsets(sizes, dev),
             "most": max(sizes), "out": normal(total, n_out), "row_map": None, "row_scale": None}
        if case["scatter"]:  # rows go back to their (token, choice) place with the router's weight
            s["row_map"] = torch.randperm(total, generator=g, device=dev).to(torch.int32)
            s["row_scale"] = torch.rand(total, generator=g, device=dev)
        return s
    if op == "lora":
        M, K, r, L = case["tokens"], case["K"], case["rank"], case["adapters"]
        slices = _slices(case)
        length, adapter = _lora_rows(case)
        names = list(range(L))
        rng.shuffle(names)
        adapter = [names[a] if a >= 0 else -1 for a in adapter]
        turn = list(range(len(length)))
        rng.shuffle(turn)
        index = torch.tensor([adapter[i] for i in turn for _ in range(length[i])], dtype=torch.int64, device=dev)
        key = torch.where(index < 0, L, index)
        order = torch.argsort(key, stable=True).to(torch.int32)  # rows of adapter 0, 1, ..., then those without one
        count = torch.bincount(key, minlength=L + 1)[:L]
        offsets = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
        return {"case": case, "x": normal(M, K), "a": normal(L, len(slices) * r, K, std=K ** -0.5),
                "b": normal(L, sum(slices), r, std=0.5 * r ** -0.5), "order": order, "offsets": offsets,
                "base": normal(M, sum(slices)), "slices": slices, "most": int(count.max()),
                "scales": torch.rand(L, generator=g, device=dev) + 0.5}
    if op == "norm":
        M, N = case["M"], case["N"]
        channel = torch.where(torch.rand(N, generator=g, device=dev) < 0.01, 20.0, 1.0)  # a few large channels
        lo = -case["offset"]
        gate = {"none": None, "channel": (N,), "row": (M, 1), "element": (M, N)}[case["gate"]]
        return {"case": case, "x": (normal(M, N, dtype=torch.float32) * channel).to(T),
                "residual": (normal(M, N, dtype=torch.float32) * channel * 2).to(DTYPES[case["res"]]),
                "post": (torch.rand(N, generator=g, device=dev) + 0.5 + lo).to(T) if case["post"] else None,
                "pre": (torch.rand(N, generator=g, device=dev) + 0.5 + lo).to(T) if case["pre"] else None,
                "gate": normal(*gate) if gate else None}
    M, Hq, Hk, D = case["M"], case["Hq"], case["Hk"], case["D"]
    start = torch.randint(0, max(1, case["far"] - M), (1,), generator=g, device=dev)
    positions = (start + torch.arange(M, device=dev)).clamp_(max=case["far"])
    inv_freq = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev) / case["rot"])
    long = torch.arange(case["rot"] // 2, device=dev) >= case["rot"] // 4  # the slow half stretched for a long context
    return {"case": case, "qkv": normal(M, (Hq + 2 * Hk) * D), "positions": positions,
            "inv_freq": torch.where(long, inv_freq / 4, inv_freq), "scale": 1.0 + 0.1 * math.log(4.0),
            "qw": (torch.rand(D, generator=g, device=dev) + 0.5).to(T) if case["qknorm"] else None,
            "kw": (torch.rand(D, generator=g, device=dev) + 0.5).to(T) if case["qknorm"] else None}


# ---------------------------------------------------------------- the operators
def _qk(s):
    c = s["case"]
    M, Hq, Hk, D = c["M"], c["Hq"], c["Hk"], c["D"]
    q, k = s["qkv"][:, : Hq * D], s["qkv"][:, Hq * D : (Hq + Hk) * D]
    return q.unflatten(1, (Hq, D)), k.unflatten(1, (Hk, D))


def run(s):
    c = s["case"]
    if own:
        from sglite_b200 import ops

        if c["op"] == "grouped":
            return ops.grouped_gemm(s["x"], s["w"], s["offsets"], out=s["out"], silu_mul=c["silu"], row_map=s["row_map"],
                                    row_scale=s["row_scale"])
        if c["op"] == "lora":
            return ops.lora(s["x"], s["a"], s["b"], s["order"], s["offsets"], s["base"], slices=s["slices"],
                            scales=s["scales"])
        if c["op"] == "norm":
            return ops.gated_add_rmsnorm(s["x"], s["residual"], s["pre"], 1e-6, post_weight=s["post"], gate=s["gate"],
                                         gate_act=c["act"], scale=c["scale"], weight_offset=c["offset"])
        q, k = _qk(s)
        return ops.rotary(q, k, s["positions"], s["inv_freq"], interleaved=c["interleaved"], scale=s["scale"],
                          q_weight=s["qw"], k_weight=s["kw"], eps=1e-6)
    return {"grouped": _grouped, "lora": _lora, "norm": _norm, "rotary": _rotary}[c["op"]](s)


def _padded(offsets, most, rows):
    """Row numbers of each group, padded to the largest group's: [groups, most], and which of them are real."""
    at = offsets[:-1, None].long() + torch.arange(most, device=offsets.device)
    real = at < offsets[1:, None]
    return torch.where(real, at, rows - 1 if rows else 0), real


def _grouped(s):
    c = s["case"]
    at, real = _padded(s["offsets"], s["most"], s["x"].shape[0])
    y = torch.bmm(s["x"].float()[at], s["w"].float().transpose(1, 2))
    if c["silu"]:
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    y = y[real]  # group after group: rows offsets[0] .. offsets[E]
    if c["scatter"]:
        to = s["row_map"][: y.shape[0]].long()
        s["out"][to] = (y * s["row_scale"][to][:, None]).to(s["out"].dtype)
    else:
        s["out"][: y.shape[0]] = y.to(s["out"].dtype)
    return s["out"]


def _lora(s):
    c = s["case"]
    r, slices = c["rank"], s["slices"]
    order = s["order"].long()
    at, real = _padded(s["offsets"], s["most"], c["tokens"])
    h = torch.bmm(s["x"].float()[order[at]], s["a"].float().transpose(1, 2))
    b = s["b"].float().split(slices, dim=1)
    part = [torch.bmm(h[..., i * r : (i + 1) * r], b[i].transpose(1, 2)) for i in range(len(slices))]
    delta = torch.cat(part, dim=-1) * s["scales"][:, None, None]
    out = s["base"].float()
    out[order[at[real]]] += delta[real]
    return out.to(s["base"].dtype)


def _rms(v, weight, offset):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * (weight.to(v.dtype) + offset)


def _act(v, name):
    return {"none": lambda t: t, "sigmoid": lambda t: 1.0 / (1.0 + torch.exp(-t)), "tanh": torch.tanh,
            "silu": lambda t: t / (1.0 + torch.exp(-t))}[name](v)


def _norm(s, wide=torch.float32):
    c = s["case"]
    v = s["x"].to(wide)
    if s["post"] is not None:
        v = _rms(v, s["post"], c["offset"])
    if s["gate"] is not None:
        v = v * _act(s["gate"].to(wide), c["act"])
    h = s["residual"].to(wide) + c["scale"] * v
    y = _rms(h, s["pre"], c["offset"]) if s["pre"] is not None else None
    if wide is torch.float32:
        return (None if y is None else y.to(s["x"].dtype)), h.to(s["residual"].dtype)
    return y, h


def _rotate(v, cos, sin, rot, interleaved):
    a, b = (v[..., 0:rot:2], v[..., 1:rot:2]) if interleaved else (v[..., : rot // 2], v[..., rot // 2 : rot])
    x, y = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([x, y], dim=-1).flatten(-2) if interleaved else torch.cat([x, y], dim=-1)
    return torch.cat([turned, v[..., rot:]], dim=-1)


def _rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]  # far positions: the angle needs 64 bits
    cos, sin = ((t * s["scale"]).float()[:, None] for t in (torch.cos(angle), torch.sin(angle)))
    out = []
    for v, w in zip(_qk(s), (s["qw"], s["kw"])):
        v = v.float()
        v = v if w is None else _rms(v, w, 0.0)
        out.append(_rotate(v, cos, sin, c["rot"], c["interleaved"]).to(s["qkv"].dtype))
    return tuple(out)


# ---------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "grouped":
        out, at = s["out"].double(), s["offsets"].tolist()
        for e in range(case["E"]):
            y = s["x"][at[e] : at[e + 1]].double() @ s["w"][e].double().T
            if case["silu"]:
                I = case["N"] // 2
                y = y[:, :I] * torch.sigmoid(y[:, :I]) * y[:, I:]
            if case["scatter"]:
                to = s["row_map"][at[e] : at[e + 1]].long()
                out[to] = y * s["row_scale"].double()[to, None]
            else:
                out[at[e] : at[e + 1]] = y
        return out
    if case["op"] == "lora":
        out, at, order, r = s["base"].double(), s["offsets"].tolist(), s["order"].long(), case["rank"]
        for n in range(case["adapters"]):
            rows, n0 = order[at[n] : at[n + 1]], 0
            h = s["x"][rows].double() @ s["a"][n].double().T
            for i, width in enumerate(s["slices"]):
                out[rows, n0 : n0 + width] += s["scales"][n].double() * (
                    h[:, i * r : (i + 1) * r] @ s["b"][n, n0 : n0 + width].double().T)
                n0 += width
        return out
    if case["op"] == "norm":
        x, N = s["x"].double(), case["N"]
        if s["post"] is not None:
            x = x / (x.pow(2).sum(1, keepdim=True) / N + 1e-6).sqrt() * (s["post"].double() + case["offset"])
        if s["gate"] is not None:
            t = s["gate"].double()
            x = x * (t if case["act"] == "none" else t.sigmoid() if case["act"] == "sigmoid" else t.tanh()
                     if case["act"] == "tanh" else t * t.sigmoid())
        h = s["residual"].double() + case["scale"] * x
        if s["pre"] is None:
            return None, h
        return h / (h.pow(2).sum(1, keepdim=True) / N + 1e-6).sqrt() * (s["pre"].double() + case["offset"]), h
    M, D, rot = case["M"], case["D"], case["rot"]
    turn = torch.polar(torch.full((M, rot // 2), s["scale"], dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * s["inv_freq"])[:, None]
    both, at = [], 0
    for heads, w in ((case["Hq"], s["qw"]), (case["Hk"], s["kw"])):
        v = s["qkv"][:, at * D : (at + heads) * D].double().reshape(M, heads, D)
        at += heads
        if w is not None:
            v = v / (v.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
        first = torch.arange(0, rot, 2) if case["interleaved"] else torch.arange(rot // 2)
        second = first + (1 if case["interleaved"] else rot // 2)
        z = torch.complex(v[..., first], v[..., second]) * turn
        v[..., first], v[..., second] = z.real, z.imag
        both.append(v)
    return tuple(both)


def work(case):
    """What a pass cannot do without: inputs read once, outputs written once."""
    two = 2  # bytes of a bf16 or fp16 value
    if case["op"] == "grouped":
        rows, K, N = case["rows"], case["K"], case["N"]
        hit = sum(1 for n in _sizes(rows, case["E"], 1) if n)
        n_out = N // 2 if case["silu"] else N
        return {"bytes": two * (hit * N * K + rows * K + rows * n_out), "flops": 2.0 * rows * K * N}
    if case["op"] == "lora":
        length, adapter = _lora_rows(case)
        M, K, N, r = case["tokens"], case["K"], sum(_slices(case)), case["rank"]
        R = r * len(_slices(case))
        rows = sum(n for n, a in zip(length, adapter) if a >= 0)
        hit = len({a for a in adapter if a >= 0})
        return {"bytes": two * (rows * K + 2 * M * N + hit * (R * K + N * r)), "flops": 2.0 * rows * (R * K + N * r)}
    if case["op"] == "norm":
        M, N, res = case["M"], case["N"], 4 if case["res"] == "fp32" else 2
        gate = {"none": 0, "channel": N, "row": M, "element": M * N}[case["gate"]]
        return {"bytes": M * N * (two + 2 * res + (two if case["pre"] else 0)) + two * gate, "flops": 10.0 * M * N}
    values = case["M"] * (case["Hq"] + case["Hk"]) * case["D"]
    return {"bytes": two * 2 * values, "flops": 6.0 * values}
