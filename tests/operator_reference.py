"""The operators' definitions in 64 bits, one sequence and head at a time, and
bounds of what their arithmetic may be off by (test infrastructure).

Half a step of rounding is finfo.eps / 2 of the value: 2^-8 in BF16, 2^-11 in
FP16, 2^-24 in FP32.
"""

import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def frequencies(r, theta=10000.0, scaling="none", factor=1.0, original=None, fast=32.0, slow=1.0, multiplier=None):
    base = theta * factor ** (r / (r - 2)) if scaling == "ntk" and r > 2 else theta
    f = [base ** (-2.0 * i / r) for i in range(r // 2)]
    m = 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":
        lo, hi = (r * math.log(original / (t * 2 * math.pi)) / (2 * math.log(theta)) for t in (fast, slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        for i in range(r // 2):
            part = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            f[i] = f[i] * (1 - part) + f[i] / factor * part
        m = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    return f, m if multiplier is None else multiplier


def rotated(x, positions, r, layout, freq, m, head_dim):
    """x [B, ., ., D] with tokens along ``head_dim``'s other axis; returns (values, bound) in 64 bits.

    Bound: cos and sin are off by the FP32 rounding of the angle (pi 2^-25),
    of the function (at most 2 units, 2^-22) and of the factor; two products
    and a sum add three roundings: below 2^-20 of |a| + |b| together; then one
    rounding to the type.
    """
    b = x.shape[0]
    pos = positions.double().expand(b, -1) if positions.ndim == 1 else positions.double()
    ang = pos[..., None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    ang = ang.unsqueeze(head_dim)
    y = x.double().clone()
    ia = torch.arange(r // 2, device=x.device) * (1 if layout == "half" else 2)
    ib = ia + (r // 2 if layout == "half" else 1)
    u, w = y[..., ia], y[..., ib]
    slack = torch.zeros_like(y)
    slack[..., ia] = slack[..., ib] = (u.abs() + w.abs()) * abs(m) * 2.0 ** -20
    y[..., ia] = m * (u * ang.cos() - w * ang.sin())
    y[..., ib] = m * (u * ang.sin() + w * ang.cos())
    turned = slack > 0
    return y, slack + torch.where(turned, y.abs() * HALF[x.dtype], 0.0) * (1 + 2.0 ** -10) + torch.where(
        turned, torch.finfo(x.dtype).smallest_normal, 0.0)


def visible(parents):
    """Per sequence: bool [N, N] of a list of parents, by walking up from each node."""
    n = len(parents)
    see = torch.zeros(n, n, dtype=torch.bool)
    for i in range(n):
        line, at = [], i
        while 0 <= at:
            line.append(at)
            up = parents[at]
            at = up if up < at and up >= -1 else -2
        if at == -1:
            see[i, line] = True
    return see


def _score_slack(q, k, scale, fp8=False):
    """FP32 accumulation of D exact products in steps of 16: each step rounds
    (or cuts) by at most 2^-23 of a partial sum, the products inside a step as
    often again; the bound is (D / 16 + 16) 2^-23 of sum |q k|.

    Over FP8 keys a query row is the sum of two e4m3 rows, hi + lo, after a
    power of two that puts its largest element x into [128, 256).  hi rounds to
    4 significant bits; what is left is a multiple of 2^-7 of hi's power of two
    and at most 2^-4 of it, so it fits lo's 4 bits unless it is below e4m3's
    last place of 2^-9.  There lo is off by at most half of that, 2^-10, which
    is 2^-10 / 128 = 2^-17 of x at most.  The score is then off by at most
    2^-17 max|q| sum |k|; and it is accumulated in twice as many steps."""
    d = q.shape[-1]
    slack = scale * (q.abs() @ k.abs().T) * (d / 16 + 16) * 2.0 ** -23
    if fp8:
        slack = 2 * slack + scale * 2.0 ** -17 * q.abs().amax(1, keepdim=True) * k.abs().sum(1)
    return slack


def tree(q, kc, vc, lengths, k, v, parents, scale=None):
    """(out, lse, out bound, lse bound).  Weights are rounded to BF16 (half a
    step of each), the result once more; scores as _score_slack says, and the
    exponential and the sums within 2^-18."""
    b, n, hq, d = q.shape
    hkv, t = kc.shape[1], kc.shape[2]
    g = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(b, n, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((b, n, hq), -math.inf, dtype=torch.float64, device=q.device)
    eo, el = torch.zeros_like(out), torch.zeros_like(lse)
    for i in range(b):
        see = visible(parents[i].tolist()).to(q.device)
        m = max(0, min(int(lengths[i]), t))
        for h in range(hkv):
            for j in range(n):
                own = see[j]
                if not own.any():
                    continue
                keys = torch.cat((kc[i, h, :m].double(), k[i, h, own].double()))
                vals = torch.cat((vc[i, h, :m].double(), v[i, h, own].double()))
                x = q[i, j, h * g:(h + 1) * g].double()
                z = x @ keys.T * scale
                p = torch.softmax(z, 1)
                out[i, j, h * g:(h + 1) * g] = p @ vals
                lse[i, j, h * g:(h + 1) * g] = torch.logsumexp(z, 1)
                dz = _score_slack(x, keys, scale, kc.dtype == torch.float8_e4m3fn).amax(1, keepdim=True) + z.abs().amax(1, keepdim=True) * 2.0 ** -22
                rel = torch.expm1(2 * dz) + 2.0 ** -18
                mass = p @ vals.abs()
                eo[i, j, h * g:(h + 1) * g] = (rel + 2.0 ** -8) * mass + out[i, j, h * g:(h + 1) * g].abs() * 2.0 ** -8 \
                    + 2.0 ** -100
                el[i, j, h * g:(h + 1) * g] = (dz + 2.0 ** -18 + lse[i, j, h * g:(h + 1) * g, None].abs() * 2.0 ** -22)[:, 0]
    return out, lse, eo, el


def weights(q, kc, lengths, lse, w, rows=None, scale=None):
    """(weights, bound): scores as above, lse * log2(e) and the subtraction
    rounded in FP32, FP32 sums."""
    b, n, hq, d = q.shape
    hkv, t = kc.shape[1], kc.shape[2]
    g = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    y = w.double().clone()
    e = y.abs() * 2.0 ** -23
    for i in range(b):
        m = max(0, min(int(lengths[i]), t))
        for h in range(hkv):
            x = q[i, :, h * g:(h + 1) * g].double().reshape(n * g, d)
            less = lse[i, :, h * g:(h + 1) * g].double().reshape(n * g, 1)
            take = less[:, 0] != -math.inf
            if rows is not None:
                take &= rows[i].repeat_interleave(g)
            x, less = x[take], less[take]
            if not m or not x.shape[0]:
                continue
            keys = kc[i, h, :m].double()
            z = x @ keys.T * scale
            p = torch.exp(z - less)
            dz = _score_slack(x, keys, scale, kc.dtype == torch.float8_e4m3fn) + (z.abs() + less.abs() + 1) * 2.0 ** -21
            y[i, h, :m] += p.sum(0)
            # (a score of -inf is exact, whatever its bound: its weight is 0)
            e[i, h, :m] += torch.where(p == 0, 0.0, p * torch.expm1(dz)).sum(0) + p.sum(0) * (x.shape[0] + 4) * 2.0 ** -24
    return y, e + y.abs() * 2.0 ** -23


def kept(w, n, keep, sink, local):
    """Kept indices of one head (ascending), by the definition: a list of Python floats."""
    n = max(0, min(n, len(w)))
    if n <= keep:
        return list(range(n))
    middle = range(sink, n - local)
    # NaN below every number; equal weights (0 and -0 alike): the lowest index first
    best = sorted(middle, key=lambda i: (w[i] != w[i], -w[i] if w[i] == w[i] else 0.0, i))[:keep - sink - local]
    return list(range(sink)) + sorted(best) + list(range(n - local, n))


def exact_turns(r, positions, theta=10000.0, factor=1.0, scaling="none"):
    """The fraction of a turn in [0, 1) of every (position, pair), as Decimal from
    60 digits (scaling: "none", "linear" or "ntk"): position * theta^(-2i/r) / (2 pi) modulo 1."""
    from decimal import Decimal, localcontext

    with localcontext() as c:
        c.prec = 60
        # pi = 48 atan(1/18) + 32 atan(1/57) - 20 atan(1/239)  (Gauss)
        def atan(x):
            total, power, i = Decimal(0), Decimal(1) / x, 0
            while abs(power) > Decimal(10) ** -62:
                total += power / (2 * i + 1) * (-1) ** i
                power, i = power / (x * x), i + 1
            return total

        turn = 2 * (48 * atan(18) + 32 * atan(57) - 20 * atan(239))
        base = Decimal(theta)
        if scaling == "ntk":
            base *= (Decimal(factor).ln() * r / (r - 2)).exp()
        f = [(base.ln() * (-2 * i) / r).exp() / (Decimal(factor) if scaling == "linear" else 1) for i in range(r // 2)]
        return [[(p * x / turn) % 1 for x in f] for p in positions]
