"""Measured cases of the draft-and-evict operators: rotary positions, attention
of a tree of drafted tokens over a cache, attention weights accumulated per
cached key, and eviction from the cache by those weights.

``run`` computes a case in its plain form (elementary torch operations in 32
bits) while ``own`` is false, and calls the package's operators while it is
true.  Sizes are those of the repository's benchmark (4 KV heads, 16 query
heads, head size 256, contexts up to 128K, requests of 32K) and smaller or odd
ones of the same kind.
"""

import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}


def listed():
    return [
        # one decoded token's q and k of the benchmark layer before run() / append(): pure latency
        dict(name="rotary_token", op="rotary", B=1, N=1, Hq=16, Hkv=4, D=256, R=256, start=131072, layout="half",
             scaling="none", factor=1.0, dtype="bf16"),
        # 64 requests with a 13-token draft each, half of the head rotated, interleaved, stretched fourfold
        dict(name="rotary_drafts", op="rotary", B=64, N=13, Hq=16, Hkv=4, D=256, R=128, start=32768,
             layout="interleaved", scaling="yarn", factor=4.0, dtype="bf16"),
        # the keys and queries of a whole 64K prompt before the index build, FP32 projections
        dict(name="rotary_prompt", op="rotary", B=1, N=65536, Hq=16, Hkv=4, D=256, R=256, start=0, layout="half",
             scaling="linear", factor=2.0, dtype="fp32"),
        # five drafted tokens over short, ragged caches of three requests: latency
        dict(name="tree_short", op="tree", B=3, N=5, Hq=16, Hkv=4, D=128, T=327, ragged=True, dtype="bf16"),
        # exact decode of one token over the 128K benchmark cache: bandwidth
        dict(name="tree_token_128k", op="tree", B=1, N=1, Hq=16, Hkv=4, D=256, T=131072, ragged=False, dtype="bf16"),
        # the widest tree (64 nodes, 256 rows a KV head) over the same cache: bandwidth and tensor cores even
        dict(name="tree_64_128k", op="tree", B=1, N=64, Hq=16, Hkv=4, D=256, T=131072, ragged=False, dtype="bf16"),
        # sixteen requests up to 32K, 12 drafted tokens each, ragged lengths down to an empty cache
        dict(name="tree_requests", op="tree", B=16, N=12, Hq=16, Hkv=4, D=256, T=32768, ragged=True, dtype="bf16"),
        # eight drafted tokens over the engine's own FP8 [K | V] records of the 128K cache
        dict(name="tree_fp8_128k", op="tree", B=1, N=8, Hq=16, Hkv=4, D=256, T=131072, ragged=False, dtype="fp8"),
        # one decoded token's weights over the 128K cache
        dict(name="weights_token_128k", op="weights", B=1, N=1, Hq=16, Hkv=4, D=256, T=131072, ragged=False,
             dtype="bf16"),
        # the last 32 prompt tokens of four requests weigh their caches before the first eviction
        dict(name="weights_window", op="weights", B=4, N=32, Hq=16, Hkv=4, D=256, T=32768, ragged=True, dtype="bf16"),
        # a 128K cache halved
        dict(name="evict_128k", op="evict", B=1, Hkv=4, D=256, T=131072, keep=65536, sink=128, local=256,
             ragged=False, dtype="bf16"),
        # short ragged FP8 caches of five requests, some of them below the budget
        dict(name="evict_short", op="evict", B=5, Hkv=4, D=128, T=4103, keep=1001, sink=4, local=67, ragged=True,
             dtype="fp8"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("rotary", "tree", "tree", "weights", "evict"))
    d = rng.choice((64, 128, 256, 256))
    hkv = rng.choice((1, 2, 4, 4, 8))
    g = rng.choice((1, 2, 3, 4, 4, 8))
    if op == "rotary":
        b = _log(rng, 1, 64)
        n = _log(rng, 1, max(1, min(32768, 65536 * 4 // (b * hkv * g))))
        r = d if rng.random() < 0.5 else 2 * rng.randint(1, d // 2)
        scaling = rng.choice(("none", "linear", "ntk", "yarn"))
        return dict(op=op, B=b, N=n, Hq=hkv * g, Hkv=hkv, D=d, R=r, start=_log(rng, 1, 1 << 20) - 1,
                    layout=rng.choice(("half", "interleaved")), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 6.5)),
                    dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    b = _log(rng, 1, 32)
    t = _log(rng, 1, max(1, min(131072, 131072 * 16 // (b * hkv))))
    ragged = b > 1 and rng.random() < 0.7
    dtype = rng.choice(("bf16", "bf16", "fp8"))
    if op == "evict":
        keep = _log(rng, 1, t)
        sink = rng.randint(0, min(128, keep))
        return dict(op=op, B=b, Hkv=hkv, D=d, T=t, keep=keep, sink=sink, local=rng.randint(0, min(256, keep - sink)),
                    ragged=ragged, dtype=dtype)
    n = _log(rng, 1, max(1, min(64, 64 * 16 * 131072 * 4 // (b * hkv * g * 4 * t))))
    return dict(op=op, B=b, N=n, Hq=hkv * g, Hkv=hkv, D=d, T=t, ragged=ragged, dtype=dtype)


def _lengths(case):
    """Tokens of each cache: the full buffer, or from the full buffer evenly down to an empty cache."""
    b, t = case["B"], case["T"]
    return [t - i * t // (b - 1) if case["ragged"] and b > 1 else t for i in range(b)]


def _parents(b, n, ragged, gen):
    """Random trees of drafted tokens (-1: follows the cache); nodes past a tree's own size are unused (-2)."""
    i = torch.arange(n, device=DEV)
    back = torch.randint(0, 4, (b, n), device=DEV, generator=gen)
    p = (i - 1 - back).clamp_min(-1)
    size = n - (torch.arange(b, device=DEV) % 3 if ragged else torch.zeros(b, device=DEV, dtype=torch.int64))
    return torch.where(i[None, :] < size.clamp_min(1)[:, None], p, -2).to(torch.int32)


def _attention_inputs(case, gen):
    """Keys of a 256-component mixture per KV head, normal values, queries near
    component centres: the value distributions of the repository's benchmark."""
    b, n, hq, hkv, d, t = (case[x] for x in ("B", "N", "Hq", "Hkv", "D", "T"))
    kind = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=gen, dtype=torch.bfloat16)

    centres = normal(hkv, 256, d)
    kv = torch.empty(b, hkv, t, 2 * d, device=DEV, dtype=kind)  # [K | V] records, as the engine keeps its FP8 cache
    if case["dtype"] != "fp8":
        k, v = (torch.empty(b, hkv, t, d, device=DEV, dtype=kind) for _ in range(2))
    else:
        k, v = kv[..., :d], kv[..., d:]
    comp = torch.randint(0, 256, (b, hkv, t), device=DEV, generator=gen)
    for i in range(b):
        for h in range(hkv):
            k[i, h].copy_(centres[h][comp[i, h]] + 0.35 * normal(t, d))
            v[i, h].copy_(normal(t, d))
    pick = torch.randint(0, 256, (b, n, hq), device=DEV, generator=gen)
    head = (torch.arange(hq, device=DEV) // (hq // hkv)).expand(b, n, hq)
    q = centres[head, pick] + 0.2 * normal(b, n, hq, d)
    lengths = torch.tensor(_lengths(case), device=DEV, dtype=torch.int32)
    return q, k, v, lengths, centres, normal


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    s = dict(case=case)
    if case["op"] == "rotary":
        b, n, d, kind = case["B"], case["N"], case["D"], TYPES[case["dtype"]]
        s["q"] = torch.randn(b, n, case["Hq"], d, device=DEV, generator=gen).to(kind)
        s["k"] = torch.randn(b, case["Hkv"], n, d, device=DEV, generator=gen).to(kind)
        first = case["start"] + torch.randint(0, 64, (b, 1), device=DEV, generator=gen)
        s["positions"] = first + torch.arange(n, device=DEV)
    elif case["op"] == "evict":
        b, h, t, d = (case[x] for x in ("B", "Hkv", "T", "D"))
        kind = TYPES[case["dtype"]]
        s["k"], s["v"] = (torch.randn(b, h, t, d, device=DEV, generator=gen, dtype=torch.bfloat16).to(kind)
                          for _ in range(2))
        # heavy-tailed weights; one key in eight was never looked at
        w = torch.exp(2 * torch.randn(b, h, t, device=DEV, generator=gen))
        s["weights"] = torch.where(torch.rand(b, h, t, device=DEV, generator=gen) < 0.125, 0.0, w)
        s["lengths"] = torch.tensor(_lengths(case), device=DEV, dtype=torch.int32)
    else:
        q, k, v, lengths, centres, normal = _attention_inputs(case, gen)
        b, n, hq, hkv, d, t = (case[x] for x in ("B", "N", "Hq", "Hkv", "D", "T"))
        s.update(q=q, k_cache=k, v_cache=v, lengths=lengths)
        if case["op"] == "tree":
            s["k"] = centres[:, torch.randint(0, 256, (b, n), device=DEV, generator=gen)].transpose(0, 1).contiguous()
            s["k"] = s["k"] + 0.35 * normal(b, hkv, n, d)
            s["v"] = normal(b, hkv, n, d)
            s["parents"] = _parents(b, n, case["ragged"], gen)
        else:
            # the rows' log-sum-exp over the cache and over themselves; one row in five was not accepted
            s["lse"] = torch.empty(b, n, hq, device=DEV)
            for i in range(b):
                x = q[i].float().reshape(n, hkv, hq // hkv, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)
                z = x @ k[i].float().transpose(1, 2) * d ** -0.5
                z = z.masked_fill(torch.arange(t, device=DEV) >= lengths[i], -math.inf)
                z = torch.logaddexp(torch.logsumexp(z, 2), torch.full((), float(d) ** 0.5 * 0.5, device=DEV))
                s["lse"][i] = z.reshape(hkv, n, hq // hkv).permute(1, 0, 2).reshape(n, hq)
                del z, x
            s["rows"] = torch.rand(b, n, device=DEV, generator=gen) >= 0.2
            s["rows"][:, 0] = True
            s["weights"] = torch.rand(b, hkv, t, device=DEV, generator=gen)
    return s


# ---------------------------------------------------------------- plain forms


def _frequencies(case, kind):
    """Radians per position of each pair, and the factor on the rotated part."""
    r, factor, theta, original = case["R"], case["factor"], 10000.0, 8192.0
    i = torch.arange(0, r, 2, device=DEV, dtype=kind)
    if case["scaling"] == "ntk" and r > 2:
        theta = theta * factor ** (r / (r - 2))
    f = theta ** (-i / r)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] != "yarn":
        return f, 1.0
    # pairs that turn more than 32 times in the original context keep their
    # frequency, those that turn less than once are stretched, linear between
    low = max(math.floor(r * math.log(original / (32 * 2 * math.pi)) / (2 * math.log(theta))), 0)
    high = min(math.ceil(r * math.log(original / (2 * math.pi)) / (2 * math.log(theta))), r - 1)
    ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


def _rotate(x, cos, sin, case):
    r = case["R"]
    x = x.float()
    a, b = (x[..., :r // 2], x[..., r // 2:r]) if case["layout"] == "half" else (x[..., :r:2], x[..., 1:r:2])
    u, w = a * cos - b * sin, a * sin + b * cos
    y = torch.cat((u, w), -1) if case["layout"] == "half" else torch.stack((u, w), -1).flatten(-2)
    return torch.cat((y, x[..., r:]), -1).to(TYPES[case["dtype"]])


def _plain_rotary(s):
    f, m = _frequencies(s["case"], torch.float64)
    angle = s["positions"].double()[..., None] * f
    cos, sin = (angle.cos() * m).float(), (angle.sin() * m).float()
    return (_rotate(s["q"], cos[:, :, None], sin[:, :, None], s["case"]),
            _rotate(s["k"], cos[:, None], sin[:, None], s["case"]))


def _visible(parents):
    """[B, N, N]: node i sees node j (itself and its ancestors); no row of an unused node."""
    n = parents.shape[1]
    i = torch.arange(n, device=parents.device)
    inner = (parents >= 0) & (parents < i)
    a = torch.eye(n, device=parents.device) + (parents[..., None] == i) * inner[..., None]
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = (a @ a > 0).float()
    a = a @ a > 0
    used = inner | (parents == -1)
    return a & ~(a & ~used[:, None, :]).any(-1, keepdim=True)


def _rows(x, hkv):
    """[B, N, Hq, ...] -> [B, Hkv, N * G, ...]"""
    b, n, hq = x.shape[:3]
    x = x.reshape(b, n, hkv, hq // hkv, *x.shape[3:]).transpose(1, 2)
    return x.reshape(b, hkv, n * (hq // hkv), *x.shape[4:])


def _plain_tree(s):
    b, n, hq, hkv, d = (s["case"][x] for x in ("B", "N", "Hq", "Hkv", "D"))
    g, scale = hq // hkv, d ** -0.5
    q = _rows(s["q"].float(), hkv) * scale
    behind = torch.arange(s["case"]["T"], device=DEV) >= s["lengths"][:, None]
    v_cache = s["v_cache"].float().masked_fill(behind[:, None, :, None], 0.0)
    s1 = (q @ s["k_cache"].float().transpose(2, 3)).masked_fill_(behind[:, None, None], -math.inf)
    see = _visible(s["parents"]).repeat_interleave(g, 1)[:, None]
    s2 = (q @ s["k"].float().transpose(2, 3)).masked_fill_(~see, -math.inf)
    m = torch.maximum(s1.amax(-1), s2.amax(-1))[..., None]
    m = torch.where(m == -math.inf, 0.0, m)
    p1, p2 = torch.exp(s1.sub_(m)), torch.exp(s2 - m)
    total = p1.sum(-1, keepdim=True) + p2.sum(-1, keepdim=True)
    out = (p1 @ v_cache + p2 @ s["v"].float()) / total
    used = see.any(-1, keepdim=True)
    out = torch.where(used, out, 0.0)
    lse = torch.where(used, m + torch.log(total), -math.inf)
    out, lse = (x.reshape(b, hkv, n, g, -1).transpose(1, 2).reshape(b, n, hq, -1) for x in (out, lse))
    return out.to(torch.bfloat16), lse[..., 0]


def _plain_weights(s):
    hkv, d = s["case"]["Hkv"], s["case"]["D"]
    q = _rows(s["q"].float(), hkv) * d ** -0.5
    lse = torch.where(s["rows"][..., None], s["lse"], math.inf)
    z = (q @ s["k_cache"].float().transpose(2, 3)).sub_(_rows(lse, hkv)[..., None])
    add = torch.exp(z).sum(2)
    behind = torch.arange(s["case"]["T"], device=DEV) >= s["lengths"][:, None]
    return s["weights"] + add.masked_fill(behind[:, None], 0.0)


def _plain_evict(s):
    t, keep, sink, local = (s["case"][x] for x in ("T", "keep", "sink", "local"))
    n = s["lengths"][:, None, None]
    i = torch.arange(t, device=DEV)
    held = (i < sink) | (i >= n - local)
    rank = torch.where(held, math.inf, s["weights"])
    rank = torch.where(i >= n, -math.inf, rank)
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    j = torch.arange(keep, device=DEV)
    left = j < n
    ids = torch.sort(torch.where(left, first, t), -1).values
    at = ids.clamp_max(t - 1)
    row = at[..., None].expand(*at.shape, s["case"]["D"])
    k, v = (torch.where(left[..., None], torch.gather(x.float(), 2, row), 0.0).to(x.dtype) for x in (s["k"], s["v"]))
    w = torch.where(left, torch.gather(s["weights"], 2, at), 0.0)
    return k, v, w, torch.where(left, ids, -1).to(torch.int32), s["lengths"].clamp_max(keep)


def run(state):
    case = state["case"]
    if own:
        import seoulkv_b200 as skv

        if case["op"] == "rotary":
            return skv.rotary(state["q"], state["k"], state["positions"], rotary_dim=case["R"], layout=case["layout"],
                              scaling=case["scaling"], factor=case["factor"], original_context=8192)
        if case["op"] == "tree":
            return skv.tree_attention(state["q"], state["k_cache"], state["v_cache"], state["lengths"], state["k"],
                                      state["v"], state["parents"])
        if case["op"] == "weights":
            return skv.accumulate_weights(state["q"], state["k_cache"], state["lengths"], state["lse"],
                                          state["weights"], rows=state["rows"])
        return skv.evict(state["k"], state["v"], state["weights"], state["lengths"], keep=case["keep"],
                         sink=case["sink"], local=case["local"])
    return {"rotary": _plain_rotary, "tree": _plain_tree, "weights": _plain_weights,
            "evict": _plain_evict}[case["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "rotary":
        tokens = case["B"] * case["N"]
        values = tokens * (case["Hq"] + case["Hkv"])
        return {"bytes": 2 * values * case["D"] * e + 8 * tokens, "flops": 3 * values * case["R"]}
    lengths, h, d, t, b = _lengths(case), case["Hkv"], case["D"], case["T"], case["B"]
    held = sum(lengths)
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths)
        rows = b * case["keep"]
        return {"bytes": h * (4 * held + kept * (2 * d * e + 4) + rows * (2 * d * e + 8)) + 8 * b, "flops": h * held}
    n, hq = case["N"], case["Hq"]
    if case["op"] == "tree":
        return {"bytes": 2 * h * d * e * held + b * n * (4 * hq * d + 4 * h * d + 4 * hq + 4) + 4 * b,
                "flops": 4 * n * hq * d * (held + b * n)}
    return {"bytes": h * d * e * held + 8 * b * h * t + b * n * (2 * hq * d + 4 * hq + 1) + 4 * b,
            "flops": 2 * n * hq * d * held}


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "tree": _exact_tree, "weights": _exact_weights, "evict": _exact_evict}[case["op"]](s)


def _exact_rotary(s):
    """Each pair as a complex number, turned by exp(i * position * frequency)."""
    c = s["case"]
    r, d = c["R"], c["D"]
    base = 10000.0
    turns = []
    m = 1.0
    for i in range(r // 2):
        f = base ** (-2.0 * i / r)
        if c["scaling"] == "linear":
            f = f / c["factor"]
        elif c["scaling"] == "ntk" and r > 2:
            f = (base * c["factor"] ** (r / (r - 2))) ** (-2.0 * i / r)
        elif c["scaling"] == "yarn":
            m = 0.1 * math.log(c["factor"]) + 1.0
            lo, hi = (r * math.log(8192.0 / (x * 2.0 * math.pi)) / (2.0 * math.log(base)) for x in (32.0, 1.0))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            f = f * (1.0 - part) + (f / c["factor"]) * part
        turns.append(f)
    angle = s["positions"].double()[..., None] * torch.tensor(turns, device=DEV, dtype=torch.float64)
    turn = torch.polar(torch.full_like(angle, m), angle)

    def rotated(x, z):
        y = x.double()
        pairs = y[..., :r]
        if c["layout"] == "half":
            pairs = pairs.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        else:
            pairs = pairs.unflatten(-1, (r // 2, 2))
        w = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
        if c["layout"] == "half":
            w = w.transpose(-1, -2)
        y[..., :r] = w.reshape(*y.shape[:-1], r)
        return y

    return rotated(s["q"], turn[:, :, None, :]), rotated(s["k"], turn[:, None, :, :])


def _exact_tree(s):
    """Request by request and head by head: ancestors by walking up, softmax over the keys that a row sees."""
    c = s["case"]
    b, n, hq, hkv, d = (c[x] for x in ("B", "N", "Hq", "Hkv", "D"))
    g = hq // hkv
    out = torch.zeros(b, n, hq, d, device=DEV, dtype=torch.float64)
    lse = torch.full((b, n, hq), -math.inf, device=DEV, dtype=torch.float64)
    parents, lengths = s["parents"].tolist(), s["lengths"].tolist()
    for i in range(b):
        see = torch.zeros(n, n, dtype=torch.bool)
        for j in range(n):
            path, at = [], j
            while 0 <= at < n:
                path.append(at)
                up = parents[i][at]
                at = up if up < at else -2
            if at == -1:
                see[j, path] = True
        used = see.any(1).to(DEV)
        see = see.to(DEV)
        t = lengths[i]
        for h in range(hkv):
            x = s["q"][i, :, h * g:(h + 1) * g].double().reshape(n * g, d)
            keys = torch.cat((s["k_cache"][i, h, :t].double(), s["k"][i, h].double()))
            values = torch.cat((s["v_cache"][i, h, :t].double(), s["v"][i, h].double()))
            z = x @ keys.T / math.sqrt(d)
            z[:, t:][~see.repeat_interleave(g, 0)] = -math.inf
            z = z.reshape(n, g, t + n)[used].reshape(-1, t + n)
            if z.numel():
                out[i, used, h * g:(h + 1) * g] = (torch.softmax(z, 1) @ values).reshape(-1, g, d)
                lse[i, used, h * g:(h + 1) * g] = torch.logsumexp(z, 1).reshape(-1, g)
    return out, lse


def _exact_weights(s):
    c = s["case"]
    b, n, hq, hkv, d = (c[x] for x in ("B", "N", "Hq", "Hkv", "D"))
    g = hq // hkv
    w = s["weights"].double()
    for i, t in enumerate(s["lengths"].tolist()):
        for h in range(hkv):
            x = s["q"][i, s["rows"][i], h * g:(h + 1) * g].double().reshape(-1, d)
            less = s["lse"][i, s["rows"][i], h * g:(h + 1) * g].double().reshape(-1, 1)
            w[i, h, :t] += torch.exp(x @ s["k_cache"][i, h, :t].double().T / math.sqrt(d) - less).sum(0)
    return w


def _exact_evict(s):
    c = s["case"]
    b, hkv, d, keep = (c[x] for x in ("B", "Hkv", "D", "keep"))
    k, v = (torch.zeros(b, hkv, keep, d, device=DEV, dtype=torch.float64) for _ in range(2))
    w = torch.zeros(b, hkv, keep, device=DEV, dtype=torch.float64)
    for i, t in enumerate(s["lengths"].tolist()):
        for h in range(hkv):
            chosen = torch.arange(t, device=DEV)
            if t > keep:
                middle = s["weights"][i, h, c["sink"]:t - c["local"]]
                best = torch.sort(-middle, stable=True).indices[:keep - c["sink"] - c["local"]] + c["sink"]
                chosen = torch.cat((chosen[:c["sink"]], best.sort().values, chosen[t - c["local"]:]))
            m = chosen.numel()
            k[i, h, :m] = s["k"][i, h].double()[chosen]
            v[i, h, :m] = s["v"][i, h].double()[chosen]
            w[i, h, :m] = s["weights"][i, h, chosen].double()
    return k, v, w, None, None
