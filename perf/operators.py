"""Cases and plain forms of the operators in which every token picks its own weights.

* route_experts: scores of a router, limited to the best groups, top-k, renormalised weights;
* moe_mlp: the chosen experts' SiLU-gated MLP on NVFP4 weights, from fp16 activations to the weighted sum;
* lora_add: low-rank adapters of many requests added to a shared projection's output.

``run`` computes the plain form (elementary torch operations, 32 bits, 64 for the router, whose
choice may hang on the last bit) or, with ``own`` set, calls the library's operators.
"""
import math

import numpy as np
import torch

own = False

_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # one decoded token, eight experts: the latency of a call
        dict(name="route 1x8", op="route", T=1, E=8, k=2, score="softmax", bias=False, groups=1, top_groups=1, dtype="float32"),
        # a decode batch, 256 experts in 8 groups of which 4 may be used, a bias that balances the load
        dict(name="route 64x256 grouped", op="route", T=64, E=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, dtype="float32"),
        # an odd number of tokens and of experts, half-precision logits with many ties
        dict(name="route 4097x60 bf16", op="route", T=4097, E=60, k=4, score="softmax", bias=False, groups=1, top_groups=1, dtype="bfloat16"),
        # a long prefill over many requests
        dict(name="route 32768x256 grouped", op="route", T=32768, E=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, dtype="float32"),
        # one decoded token through two of eight wide experts (the dual GEMM's widths): weights are read once
        dict(name="moe 1 of 8", op="moe", T=1, E=8, k=2, D=4096, F=14336),
        # a decode batch that touches nearly all of 64 narrow experts
        dict(name="moe 64 of 64", op="moe", T=64, E=64, k=8, D=4096, F=1536),
        # odd sizes: widths that are multiples of 64 only, ragged expert loads
        dict(name="moe 333 odd", op="moe", T=333, E=16, k=4, D=1984, F=1344),
        # a prefill: eight groups at the grouped GEMM's scale
        dict(name="moe 4096 of 8", op="moe", T=4096, E=8, k=2, D=4096, F=14336),
        # one decoded token with an adapter beside the skinny GEMM (its widths)
        dict(name="lora 1 r16", op="lora", T=1, K=4096, N=14336, r=16, n=8, run=1),
        # a decode batch of 64 requests over 32 adapters, one token each
        dict(name="lora 64 r64", op="lora", T=64, K=4096, N=14336, r=64, n=32, run=1),
        # odd sizes: mixed ranks, ragged requests, a width that is no multiple of 8
        dict(name="lora 777 odd", op="lora", T=777, K=1000, N=1003, r=48, n=9, run=37),
        # prompts of several requests beside a wide projection
        dict(name="lora 8192 r64", op="lora", T=8192, K=4096, N=14336, r=64, n=6, run=700),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["route", "moe", "lora"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _log(rng, max(2, 8 // groups), 256 // groups)
        top_groups = rng.randint(1, groups)
        k = rng.randint(1, min(8, E // groups * top_groups))
        return dict(op="route", T=_log(rng, 1, 32768), E=E, k=k, score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
                    dtype=rng.choice(["float32", "bfloat16", "float16"]))
    if op == "moe":
        E = _log(rng, 2, 64)
        D = 64 * _log(rng, 8, 64)
        F = 64 * _log(rng, 8, max(8, min(224, 8 * 4096 * 14336 // (E * D * 64))))
        k = rng.randint(1, min(8, E))
        return dict(op="moe", T=_log(rng, 1, max(1, min(4096, 8192 * 4096 * 14336 // (k * D * F)))), E=E, k=k, D=D, F=F)
    r = 16 * _log(rng, 1, 8)
    n = _log(rng, 1, min(64, 6 * 64 // r * 4))
    T = _log(rng, 1, 8192)
    K = 8 * _log(rng, 32, 512)
    N = _log(rng, 200, 14336)
    if T * r * n > 8192 * 64 * 6:   # no dearer than the largest listed case
        T = 8192 * 64 * 6 // (r * n)
    return dict(op="lora", T=T, K=K, N=N, r=r, n=n, run=_log(rng, 1, max(1, T // 2)))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _experts(g, E, rows, K):
    """Random NVFP4 weights of E experts: codes [E, rows, K/2], e4m3 scales in the 128x4 blocked layout [E, bytes]."""
    codes = torch.randint(0, 256, (E, rows, K // 2), dtype=torch.uint8, device="cuda", generator=g)
    # 2^-8 .. 2^-5.7, subnormals among them: weights of about 1/sqrt(K)
    sf = torch.randint(2, 11, (E, -(-rows // 128) * (K // 64) * 512), dtype=torch.uint8, device="cuda", generator=g)
    return codes, sf


def prepare(case, seed):
    g = _gen(seed)
    c = case
    if c["op"] == "route":
        x = (_randn(g, c["T"], c["E"]) * 1.5).to(getattr(torch, c["dtype"]))
        bias = _randn(g, c["E"]) * 0.05 if c["bias"] else None
        return dict(case=c, logits=x, bias=bias)
    if c["op"] == "moe":
        T, E, k, D, F = c["T"], c["E"], c["k"], c["D"], c["F"]
        x = _randn(g, T, D).to(torch.float16)
        score = _randn(g, T, E) + 0.5 * _randn(g, E)     # some experts are busier than others
        top, ids = score.sort(dim=1, descending=True)
        weights = torch.softmax(top[:, :k], dim=1).contiguous()
        ids = ids[:, :k].to(torch.int32).contiguous()
        st = dict(case=c, x=x, ids=ids, weights=weights, out=torch.empty_like(x))
        st["wg"], st["sg"] = _experts(g, E, F, D)
        st["wu"], st["su"] = _experts(g, E, F, D)
        st["wd"], st["sd"] = _experts(g, E, D, F)
        # the most rows that one expert gets: the plain form lays its batches out with it
        st["cap"] = int(torch.bincount(ids.flatten().long(), minlength=E).max())
        return st
    T, K, N, r, n = c["T"], c["K"], c["N"], c["r"], c["n"]
    x = _randn(g, T, K).to(torch.float16)
    a = (_randn(g, n, r, K) / math.sqrt(K)).to(torch.float16)
    b = (_randn(g, n, N, r) / math.sqrt(r)).to(torch.float16)
    base = _randn(g, T, N).to(torch.float16)
    # each request is a run of tokens with one adapter; about one in eight has none (-1)
    owner = torch.randint(0, n, (-(-T // c["run"]),), device="cuda", generator=g)
    none = torch.rand(owner.shape, device="cuda", generator=g) < 0.125
    none[0] = False
    owner = torch.where(none, torch.full_like(owner, -1), owner)
    adapters = owner.repeat_interleave(c["run"])[:T].to(torch.int32).contiguous()
    scales = torch.rand(n, device="cuda", generator=g) + 0.5
    ranks = (torch.randint(1, r // 16 + 1, (n,), device="cuda", generator=g) * 16).to(torch.int32)
    return dict(case=c, x=x, a=a, b=b, base=base, adapters=adapters, scales=scales, ranks=ranks, out=torch.empty_like(base))


# ------------------------------------------------------------------ plain forms

def _route(x, bias, k, score, groups, top_groups):
    x = x.double()
    off = torch.isnan(x) | (x == -math.inf)
    x = x.clamp(max=torch.finfo(torch.float32).max)
    low = torch.full_like(x, -math.inf)
    if score == "softmax":
        m = torch.where(off, low, x).amax(dim=1, keepdim=True)
        e = torch.where(off, torch.zeros_like(x), torch.exp(x - m))
        s = e / e.sum(dim=1, keepdim=True)
    else:
        s = torch.where(off, torch.zeros_like(x), 1 / (1 + torch.exp(-x)))
    c = s if bias is None else s + bias.double()
    key = torch.where(off, low, x if bias is None else c)
    T, E = x.shape
    if groups > 1:
        top2 = torch.where(off, low, c).view(T, groups, E // groups).sort(dim=2, descending=True).values[:, :, :2]
        gscore = torch.where(top2 > -math.inf, top2, torch.zeros_like(top2)).sum(dim=2)
        gscore = torch.where(top2[:, :, 0] > -math.inf, gscore, torch.full_like(gscore, -math.inf))
        chosen = gscore.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        allowed = torch.zeros(T, groups, dtype=torch.bool, device=x.device).scatter(1, chosen, True)
        key = torch.where(allowed.repeat_interleave(E // groups, dim=1), key, low)
    top, ids = key.sort(dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    w = torch.where(top > -math.inf, s.gather(1, ids), torch.zeros_like(top))
    total = w.sum(dim=1, keepdim=True)
    w = torch.where(total > 0, w / total, torch.zeros_like(w))
    ids = torch.where(top > -math.inf, ids, torch.full_like(ids, -1))
    return w.float(), ids.to(torch.int32)


def _decode(codes, sf, rows, K):
    """NVFP4 weights [E, rows, K/2] with blocked scales -> float32 [E, rows, K]."""
    E = codes.shape[0]
    v = torch.tensor(_E2M1, device=codes.device)
    v = torch.cat([v, -v])
    pairs = torch.stack([v.repeat(16), v.repeat_interleave(16)], dim=1)      # byte -> (low nibble, high nibble)
    w = pairs[codes.int()].view(E, rows, K // 16, 16)
    s = sf.view(torch.float8_e4m3fn).float()
    s = s.view(E, -(-rows // 128), K // 64, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(E, -1, K // 16)[:, :rows]
    return (w * s.unsqueeze(3)).view(E, rows, K)


def _quantized(x):
    """The values that NVFP4 codes and scales of x stand for: s = e4m3(amax / 6), q = e2m1(x * fl32(1 / s))."""
    b = x.view(*x.shape[:-1], -1, 16)
    s = (b.abs().amax(dim=-1, keepdim=True) / 6).clamp(max=448).to(torch.float8_e4m3fn).float()
    live = s > 0
    v = b * torch.where(live, 1 / s, torch.zeros_like(s))
    a = v.abs()
    # ties go to the even code
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
            + (a >= 3.5).int() + (a > 5).int())
    q = torch.tensor(_E2M1, device=x.device)[code] * torch.sign(v)
    return (q * s).view(x.shape)


def _moe(s):
    c = s["case"]
    T, E, k, D, F, cap = c["T"], c["E"], c["k"], c["D"], c["F"], s["cap"]
    expert = s["ids"].long().flatten()
    order = expert.sort(stable=True).indices
    first = torch.cumsum(torch.bincount(expert, minlength=E), 0) - torch.bincount(expert, minlength=E)
    place = torch.empty_like(expert)
    place[order] = torch.arange(T * k, device=expert.device) - first[expert[order]]
    slot = expert * cap + place                           # row of [E, cap] that this token's slot gets
    rows = torch.zeros(E * cap, D, device=expert.device)
    rows[slot] = _quantized(s["x"].float()).repeat_interleave(k, dim=0)
    rows = rows.view(E, cap, D)
    g = torch.bmm(rows, _decode(s["wg"], s["sg"], F, D).transpose(1, 2))
    u = torch.bmm(rows, _decode(s["wu"], s["su"], F, D).transpose(1, 2))
    h = _quantized(g / (1 + torch.exp(-g)) * u)
    y = torch.bmm(h, _decode(s["wd"], s["sd"], D, F).transpose(1, 2)).view(E * cap, D)
    return (y[slot].view(T, k, D) * s["weights"].unsqueeze(2)).sum(dim=1).to(torch.float16)


def _lora(s):
    c = s["case"]
    T, N, r, n = c["T"], c["N"], c["r"], c["n"]
    live = torch.arange(r, device="cuda") < s["ranks"].unsqueeze(1)                          # [n, r]
    a = torch.where(live.unsqueeze(2), s["a"].float(), torch.zeros((), device="cuda"))
    b = torch.where(live.unsqueeze(1), s["b"].float(), torch.zeros((), device="cuda"))
    mine = s["adapters"].unsqueeze(1) == torch.arange(n, device="cuda")                      # [T, n]
    u = (s["x"].float() @ a.view(n * r, -1).t()).view(T, n, r)
    u = torch.where(mine.unsqueeze(2), u * s["scales"].view(1, n, 1), torch.zeros((), device="cuda"))
    return (s["base"].float() + u.view(T, n * r) @ b.permute(0, 2, 1).reshape(n * r, N)).to(torch.float16)


def run(state):
    s, c = state, state["case"]
    if own:
        import __graft_entry__
        lib = __graft_entry__.load_package()
        if c["op"] == "route":
            return lib.route_experts(s["logits"], c["k"], bias=s["bias"], score=c["score"], num_groups=c["groups"],
                                     top_groups=c["top_groups"])
        if c["op"] == "moe":
            return lib.moe_mlp(s["x"], s["ids"], s["weights"], s["wg"], s["wu"], s["wd"], s["sg"], s["su"], s["sd"],
                               out=s["out"])
        return lib.lora_add(s["base"], s["x"], s["a"], s["b"], s["adapters"], scales=s["scales"], ranks=s["ranks"],
                            out=s["out"])
    if c["op"] == "route":
        return _route(s["logits"], s["bias"], c["k"], c["score"], c["groups"], c["top_groups"])
    return _moe(s) if c["op"] == "moe" else _lora(s)


def work(case):
    c = case
    if c["op"] == "route":
        size = 4 if c["dtype"] == "float32" else 2
        # a score, its sum and its comparison with the k best
        return dict(bytes=c["T"] * (c["E"] * size + c["k"] * 8) + (4 * c["E"] if c["bias"] else 0), flops=c["T"] * c["E"] * 8)
    if c["op"] == "moe":
        T, E, k, D, F = c["T"], c["E"], c["k"], c["D"], c["F"]
        active = E * (1 - (1 - k / E) ** T)               # experts that get a token
        return dict(bytes=active * 3 * D * F * 9 / 16 + T * D * 4 + T * k * 8, flops=6 * T * k * D * F)
    T, K, N, r, n = c["T"], c["K"], c["N"], c["r"], c["n"]
    requests = -(-T // c["run"])
    active = n * (1 - (1 - 1 / n) ** (requests * 7 / 8))  # adapters in use; ranks are r/2 on average
    mean = (r + 16) / 2
    return dict(bytes=T * K * 2 + T * N * 4 + active * mean * (K + N) * 2 + T * 4, flops=2 * T * 7 / 8 * mean * (K + N))


# ------------------------------------------------------------------ the definitions in 64 bits

def _route_exact(s):
    c = s["case"]
    x = s["logits"].double().cpu().numpy()
    T, E = x.shape
    k, groups = c["k"], c["groups"]
    if c["score"] == "softmax":
        p = np.exp(x - x.max(axis=1, keepdims=True))
        p /= p.sum(axis=1, keepdims=True)
    else:
        p = 1.0 / (1.0 + np.exp(-x))
    choice = p + s["bias"].double().cpu().numpy() if s["bias"] is not None else p
    rank = choice if s["bias"] is not None else x
    if groups > 1:
        per = np.sort(choice.reshape(T, groups, E // groups), axis=2)
        best = np.argsort(-per[:, :, -2:].sum(axis=2), axis=1, kind="stable")[:, :c["top_groups"]]
        keep = np.zeros((T, groups), bool)
        np.put_along_axis(keep, best, True, axis=1)
        rank = np.where(np.repeat(keep, E // groups, axis=1), rank, -np.inf)
    ids = np.argsort(-rank, axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(p, ids, axis=1)
    return torch.from_numpy(w / w.sum(axis=1, keepdims=True)), torch.from_numpy(ids.astype(np.int32))


def _grid(v, mantissa, lowest, most):
    """v >= 0 rounded to a float with so many mantissa bits, ties to even; `lowest`: the exponent of its subnormals' range."""
    e = torch.floor(torch.log2(v.clamp(min=2.0 ** (lowest - 1)))).clamp(min=lowest)
    step = torch.exp2(e - mantissa)
    return (torch.round(v / step) * step).clamp(max=most)


def _block_values(x):
    b = x.reshape(-1, 16)
    s = _grid(b.abs().amax(dim=1, keepdim=True) / 6, 3, -6, 448.0)
    inv = torch.where(s > 0, (1 / s).float().double(), torch.zeros_like(s))
    v = (b * inv).float().double()        # the definition's 32-bit reciprocal and product
    return (_grid(v.abs(), 1, 0, 6.0) * torch.sign(v) * s).reshape(x.shape)


def _weights64(codes, sf, rows, K):
    """One expert's weights, element by element from the format's definition."""
    nib = torch.stack([codes & 15, codes >> 4], dim=2).reshape(rows, K).double()
    mag, neg = nib % 8, nib >= 8
    e, m = torch.floor(mag / 2), mag % 2
    val = torch.where(e == 0, 0.5 * m, torch.exp2(e - 1) * (1 + 0.5 * m))
    row = torch.arange(rows, device=codes.device).unsqueeze(1)
    col = torch.arange(K // 16, device=codes.device).unsqueeze(0)
    at = ((row // 128) * (K // 64) + col // 4) * 512 + (row % 32) * 16 + (row % 128) // 32 * 4 + col % 4
    byte = sf[at].double()                # scales are positive: four bits of exponent, three of mantissa
    e, m = torch.floor(byte / 8), byte % 8
    scale = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e - 10))
    return torch.where(neg, -val, val) * scale.repeat_interleave(16, dim=1)


def _moe_exact(s):
    c = s["case"]
    xq = _block_values(s["x"].double())
    out = torch.zeros(c["T"], c["D"], dtype=torch.float64, device="cuda")
    for e in range(c["E"]):
        t, j = (s["ids"] == e).nonzero(as_tuple=True)
        if len(t) == 0:
            continue
        g = xq[t] @ _weights64(s["wg"][e], s["sg"][e], c["F"], c["D"]).t()
        u = xq[t] @ _weights64(s["wu"][e], s["su"][e], c["F"], c["D"]).t()
        h = _block_values(g / (1 + torch.exp(-g)) * u)
        y = h @ _weights64(s["wd"][e], s["sd"][e], c["D"], c["F"]).t()
        out.index_add_(0, t, y * s["weights"][t, j].double().unsqueeze(1))
    return out


def _lora_exact(s):
    out = s["base"].double()
    for i in range(s["case"]["n"]):
        t = (s["adapters"] == i).nonzero().flatten()
        if len(t) == 0:
            continue
        r = int(s["ranks"][i])
        u = s["x"][t].double() @ s["a"][i, :r].double().t()
        out[t] += float(s["scales"][i]) * (u @ s["b"][i, :, :r].double().t())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _route_exact(s)
    return _moe_exact(s) if case["op"] == "moe" else _lora_exact(s)
