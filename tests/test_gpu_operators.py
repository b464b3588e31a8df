"""Operators around a decode step on the B200, against their definitions in 64
bits with the bounds that tests/operator_reference.py derives."""

import math
import pathlib
import random
import subprocess
import sys

import pytest
import torch

import seoulkv_b200 as skv
from tests import operator_reference as R

pytestmark = pytest.mark.gpu
BF, F8 = torch.bfloat16, torch.float8_e4m3fn
NAN, INF = float("nan"), float("inf")


@pytest.fixture(autouse=True)
def _no_wait_gave_up(cuda):
    yield
    skv.check_operators(cuda)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=BF):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def close(got, want, bound):
    got = got.double()
    same = torch.isfinite(got) == torch.isfinite(want)
    assert same.all(), f"{int((~same).sum())} values finite on one side alone"
    f = torch.isfinite(want)
    assert torch.equal(got[~f].nan_to_num(nan=7.0), want[~f].nan_to_num(nan=7.0))
    over = (got - want).abs()[f] - bound[f]
    assert not over.numel() or float(over.max()) <= 0, (float(over.max()), float((got - want).abs()[f].max()))


# ---------------------------------------------------------------- rotary


ROTARY = [
    dict(b=1, n=1, hq=16, hkv=4, d=256, r=256),
    dict(b=3, n=7, hq=6, hkv=2, d=128, r=64),
    dict(b=2, n=33, hq=3, hkv=3, d=80, r=36),
    dict(b=1, n=5, hq=1, hkv=1, d=66, r=2),
    dict(b=2, n=300, hq=5, hkv=1, d=64, r=62),
    dict(b=1, n=4096, hq=4, hkv=1, d=64, r=64),
]


@pytest.mark.parametrize("c", ROTARY)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
def test_rotary(c, layout, dtype):
    g = gen(1)
    q = normal(g, c["b"], c["n"], c["hq"], c["d"], dtype=dtype)
    k = normal(g, c["b"], c["hkv"], c["n"], c["d"], dtype=dtype)
    pos = torch.randint(-5000, 1 << 21, (c["b"], c["n"]), device="cuda", generator=g)
    yq, yk = skv.rotary(q, k, pos, rotary_dim=c["r"], layout=layout)
    f, m = R.frequencies(c["r"])
    close(yq, *R.rotated(q, pos, c["r"], layout, f, m, 2))
    close(yk, *R.rotated(k, pos, c["r"], layout, f, m, 1))
    # 32-bit positions, one row for all sequences
    yq, yk = skv.rotary(q, k, pos[0].int(), rotary_dim=c["r"], layout=layout)
    close(yq, *R.rotated(q, pos[0], c["r"], layout, f, m, 2))
    close(yk, *R.rotated(k, pos[0], c["r"], layout, f, m, 1))


@pytest.mark.parametrize("scaling,kw", [("linear", {}), ("ntk", {}), ("yarn", {}), ("yarn", dict(fast=16.0, slow=2.0)),
                                        ("yarn", dict(multiplier=1.5)), ("none", dict(theta=5e5))])
def test_rotary_scaling(scaling, kw):
    g = gen(2)
    q, k = normal(g, 2, 50, 4, 128, dtype=torch.float32), normal(g, 2, 1, 50, 128, dtype=torch.float32)
    pos = torch.arange(50, device="cuda") + 100000
    f, m = R.frequencies(96, scaling=scaling, factor=6.5, original=4096, **kw)
    yq, yk = skv.rotary(q, k, pos, rotary_dim=96, scaling=scaling, factor=6.5, original_context=4096,
                        theta=kw.get("theta", 1e4), beta_fast=kw.get("fast", 32.0), beta_slow=kw.get("slow", 1.0),
                        attention_factor=kw.get("multiplier"))
    close(yq, *R.rotated(q, pos, 96, "half", f, m, 2))
    close(yk, *R.rotated(k, pos, 96, "half", f, m, 1))


def test_rotary_far_positions_and_inverse():
    """Positions beyond 2^32 keep their angles; -p turns back (two roundings of angles and values)."""
    g = gen(3)
    q = normal(g, 1, 6, 2, 64, dtype=torch.float32)
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 + 5, 2 ** 33 + 7, -(2 ** 32) - 3], device="cuda")
    y, none = skv.rotary(q, None, pos)
    assert none is None
    z, _ = skv.rotary(y, None, -pos)
    assert float((z - q).abs().max()) < 8 * 2.0 ** -20 * float(q.abs().max())
    assert torch.equal(y[:, 0], q[:, 0])


def test_rotary_strides_and_in_place():
    g = gen(4)
    b, n, hq, hkv, d = 2, 9, 4, 2, 64
    pos = torch.arange(n, device="cuda") * 1000
    f, m = R.frequencies(d)
    qkv = normal(g, b, n, hq + 2 * hkv, d)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hkv].transpose(1, 2)
    before = qkv.clone()
    wq, wk = R.rotated(q, pos, d, "half", f, m, 2), R.rotated(k, pos, d, "half", f, m, 1)
    yq, yk = skv.rotary(q, k, pos)
    close(yq, *wq)
    close(yk, *wk)
    assert torch.equal(qkv, before)
    # in place, q and k parts of one projection; the V part stays
    oq, ok = skv.rotary(q, k, pos, out=(q, k))
    assert oq is q and ok is k
    assert torch.equal(q, yq) and torch.equal(k, yk)
    assert torch.equal(qkv[:, :, hq + hkv:], before[:, :, hq + hkv:])
    # into slots of larger buffers, rows on odd places
    big = torch.full((b, n + 3, hq, d + 1), 7.0, device="cuda", dtype=BF)
    kb = torch.full((b, hkv, 2 * n, d), 7.0, device="cuda", dtype=BF)
    q0, k0 = before[:, :, :hq], before[:, :, hq:hq + hkv].transpose(1, 2)
    skv.rotary(q0, k0, pos, out=(big[:, 2:2 + n, :, 1:], kb[:, :, ::2]))
    assert torch.equal(big[:, 2:2 + n, :, 1:], yq) and torch.equal(kb[:, :, ::2], yk)
    assert (big[:, :2] == 7).all() and (big[..., 0] == 7).all() and (kb[:, :, 1::2] == 7).all()
    # broadcast inputs
    one = q0[:1].expand(b, -1, -1, -1)
    close(skv.rotary(one, None, pos)[0], *R.rotated(one, pos, d, "half", f, m, 2))


def test_rotary_refuses():
    q, k, pos = torch.zeros(2, 3, 4, 64, device="cuda", dtype=BF), torch.zeros(2, 2, 3, 64, device="cuda", dtype=BF), \
        torch.arange(3, device="cuda")
    for kw in (dict(rotary_dim=65), dict(rotary_dim=66), dict(rotary_dim=0), dict(layout="other"), dict(scaling="other")):
        with pytest.raises(ValueError):
            skv.rotary(q, k, pos, **kw)
    with pytest.raises(ValueError, match="k: expected"):
        skv.rotary(q, k.float(), pos)
    with pytest.raises(ValueError, match="positions"):
        skv.rotary(q, k, pos.float())
    with pytest.raises(ValueError, match="overlaps"):
        skv.rotary(q, k, pos, out=(q[:, :, :, :], q.view(-1)[:k.numel()].view(k.shape)))
    buf = torch.zeros(q.numel() + 64, device="cuda", dtype=BF)
    with pytest.raises(ValueError, match="overlaps"):
        skv.rotary(buf[:q.numel()].view(q.shape), None, pos, out=(buf[64:].view(q.shape), None))
    with pytest.raises(ValueError, match="share"):
        skv.rotary(q, None, pos, out=(q[:1].clone().expand(2, -1, -1, -1), None))
    with pytest.raises(ValueError, match="innermost"):
        skv.rotary(q.transpose(2, 3).contiguous().transpose(2, 3), k, pos)
    with pytest.raises(ValueError, match="gradient"):
        skv.rotary(q.float().requires_grad_(), k.float(), pos)
    with pytest.raises(ValueError, match="aligned"):
        skv.rotary(buf[1:1 + q.numel()].view(q.shape), None, pos, layout="interleaved")
    # the empty call returns empty tensors
    assert skv.rotary(q[:0], k[:0], pos)[0].shape == (0, 3, 4, 64)
    assert skv.rotary(q[:, :0], k[:, :, :0], pos[:0])[1].shape == (2, 2, 0, 64)


# ---------------------------------------------------------------- tree attention


def make_parents(rng, n, kind):
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "roots":
        return [-1] * n
    if kind == "padded":  # some nodes unused, some below unused ones, some values out of range
        return [rng.choice([-1, i - 1, -2, i, n + 5, rng.randint(-1, max(-1, i - 1))]) for i in range(n)]
    return [rng.randint(-1, i - 1) for i in range(n)]


def tree_case(seed, lengths, n, hq, hkv, d, t, dtype=BF, kind="tree", sharp=1.0):
    g, rng = gen(seed), random.Random(seed)
    b = len(lengths)
    rec = normal(g, b, hkv, t, 2 * d).to(dtype)
    kc, vc = rec[..., :d], rec[..., d:]
    q = normal(g, b, n, hq, d) * sharp
    k, v = normal(g, b, hkv, n, d), normal(g, b, hkv, n, d)
    parents = torch.tensor([make_parents(rng, n, kind) for _ in range(b)], dtype=torch.int32, device="cuda")
    return q, kc, vc, torch.tensor(lengths, dtype=torch.int32, device="cuda"), k, v, parents


def check_tree(args, scale=None):
    out, lse = skv.tree_attention(*args, scale=scale)
    want, wl, eo, el = R.tree(*args, scale=scale)
    close(out, want, eo)
    close(lse, wl, el)
    return out, lse


TREES = [
    (dict(lengths=[0, 1, 63, 64, 65], n=1, hq=4, hkv=1, d=256, t=65), "tree"),
    (dict(lengths=[127, 128, 129, 0], n=5, hq=6, hkv=2, d=128, t=129), "tree"),
    (dict(lengths=[300, 7], n=64, hq=4, hkv=2, d=64, t=301), "tree"),
    (dict(lengths=[1000], n=64, hq=16, hkv=4, d=256, t=1000), "chain"),
    (dict(lengths=[513, 3], n=33, hq=16, hkv=2, d=256, t=517), "tree"),
    (dict(lengths=[700], n=17, hq=24, hkv=1, d=128, t=700), "tree"),
    (dict(lengths=[1], n=2, hq=1, hkv=1, d=64, t=1), "roots"),
    (dict(lengths=[20, 0, 70, 64], n=31, hq=4, hkv=1, d=256, t=80), "padded"),
    (dict(lengths=[20, 200], n=64, hq=2, hkv=2, d=128, t=200), "padded"),
]


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("c,kind", TREES)
def test_tree_attention(c, kind, dtype):
    check_tree(tree_case(5, dtype=dtype, kind=kind, **c))


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("sharp", [0.05, 30.0])
def test_tree_attention_flat_and_sharp_scores(sharp, dtype):
    """Scores that leave all weights alike, and scores of hundreds: the running
    maximum moves inside a CTA and between CTAs."""
    check_tree(tree_case(6, [2500, 900], 9, 8, 2, 256, 2500, dtype=dtype, sharp=sharp))
    args = list(tree_case(7, [2000], 3, 4, 1, 128, 2000, dtype=dtype, sharp=4.0))
    # keys that grow along the cache: the maximum moves all the way
    ramp = torch.linspace(0.1, 2.0, 2000, device="cuda")[:, None]
    kc = (args[1].float() * ramp).to(dtype)
    args[1] = kc
    check_tree(args)
    check_tree(args, scale=0.5)


def test_tree_attention_lengths_are_clamped():
    args = list(tree_case(8, [40, 40], 2, 4, 2, 64, 40))
    full = skv.tree_attention(*args)
    args[3] = torch.tensor([1000, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    assert all(torch.equal(a, b) for a, b in zip(skv.tree_attention(*args), full))
    args[3] = torch.tensor([-1, -(2 ** 31)], dtype=torch.int32, device="cuda")
    check_tree(args)


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("poison", [NAN, INF, -INF])
def test_tree_attention_what_is_not_seen_does_not_count(poison, dtype):
    """Garbage behind the length, in unused nodes, and in nodes that a row does not see."""
    if dtype is F8 and poison != poison:
        pass  # e4m3 has no infinity: only NaN fits behind the length there
    args = list(tree_case(9, [70, 0, 130], 6, 8, 2, 128, 140, dtype=dtype))
    parents = [[-1, 0, 0, 1, -2, 4]] * 3
    args[6] = torch.tensor(parents, dtype=torch.int32, device="cuda")
    clean = skv.tree_attention(*args)
    kc, vc, k, v = (x.clone() for x in (args[1], args[2], args[4], args[5]))
    for i, m in enumerate((70, 0, 130)):
        bad = poison if dtype is BF else NAN
        kc[i, :, m:] = bad
        vc[i, :, m:] = bad
    for x in (k, v):
        x[:, :, 4:] = poison
    got = skv.tree_attention(args[0], kc, vc, args[3], k, v, args[6])
    assert all(torch.equal(a, b) for a, b in zip(got, clean))
    # node 2's own value: only row 2 sees it
    v[:, :, 2, 5] = poison
    out, lse = skv.tree_attention(args[0], kc, vc, args[3], k, v, args[6])
    other = torch.ones(6, 128, dtype=torch.bool, device="cuda")
    other[2, 5] = False
    assert torch.equal(out.transpose(1, 2)[:, :, other], clean[0].transpose(1, 2)[:, :, other])
    assert torch.equal(lse, clean[1])
    seen = out[:, 2, :, 5].double()
    assert (seen == poison).all() if poison == poison else torch.isnan(seen).all()
    # a key that is not a number reaches exactly the rows that see it
    k[:, :, 1, 0] = NAN
    out, lse = skv.tree_attention(args[0], kc, vc, args[3], k, args[5], args[6])
    assert torch.isnan(lse[:, [1, 3]]).all() and torch.equal(lse[:, [0, 2, 4, 5]], clean[1][:, [0, 2, 4, 5]])
    assert torch.equal(out[:, [0, 2, 4, 5]], clean[0][:, [0, 2, 4, 5]])


@pytest.mark.parametrize("dtype", [BF, F8])
def test_tree_attention_non_finite_cache_and_query(dtype):
    """A visible NaN value makes its dimension NaN in every row; a NaN query its own row alone."""
    args = list(tree_case(10, [200], 4, 4, 1, 64, 200, dtype=dtype))
    clean = skv.tree_attention(*args)
    args[0][:, 2] = NAN
    out, lse = skv.tree_attention(*args)
    assert torch.isnan(out[:, 2]).all() and torch.isnan(lse[:, 2]).all()
    keep = [0, 1, 3]
    assert torch.equal(out[:, keep], clean[0][:, keep])
    vc = args[2].clone()
    vc[0, 0, 100, 9] = NAN
    out, _ = skv.tree_attention(args[0], args[1], vc, *args[3:])
    assert torch.isnan(out[..., 9]).all()
    rest = [x for x in range(64) if x != 9]
    assert torch.equal(out[:, keep][..., rest], clean[0][:, keep][..., rest])


@pytest.mark.parametrize("dtype", [BF, F8])
def test_tree_attention_layouts(dtype):
    """Token-major caches, a cache that all sequences share, strided q and nodes, strided lengths and parents."""
    q, kc, vc, lengths, k, v, parents = tree_case(11, [100, 37, 64], 5, 8, 2, 128, 111, dtype=dtype)
    want = skv.tree_attention(q, kc, vc, lengths, k, v, parents)
    token_major = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc)]
    wide = torch.zeros(3, 5, 3, 8, 128, device="cuda", dtype=BF)
    wide[:, :, 1] = q
    nodes = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    l2 = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    l2[:, 1] = lengths
    p2 = parents.t().contiguous().t()
    got = skv.tree_attention(wide[:, :, 1], *token_major, l2[:, 1], *nodes, p2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    shared = [x[:1].expand(3, -1, -1, -1) for x in (kc, vc)]
    lone = torch.tensor([100, 37, 64], dtype=torch.int32, device="cuda")
    got = skv.tree_attention(q, *shared, lone, k, v, parents)
    full = skv.tree_attention(q, *(x.contiguous() for x in shared), lone, k, v, parents)
    assert all(torch.equal(a, b) for a, b in zip(got, full))
    heads = [x[:, :1].expand(-1, 2, -1, -1) for x in (kc, vc)]
    got = skv.tree_attention(q, *heads, lengths, k, v, parents)
    full = skv.tree_attention(q, *(x.contiguous() for x in heads), lengths, k, v, parents)
    assert all(torch.equal(a, b) for a, b in zip(got, full))


def test_tree_attention_more_sequences_than_a_launch_and_repeatability():
    g = gen(12)
    b = 700
    kc, vc = normal(g, b, 1, 70, 64), normal(g, b, 1, 70, 64)
    q, k, v = normal(g, b, 2, 2, 64), normal(g, b, 1, 2, 64), normal(g, b, 1, 2, 64)
    lengths = (torch.arange(b, device="cuda") % 71).int()
    parents = torch.tensor([[-1, 0]] * b, dtype=torch.int32, device="cuda")
    out, lse = check_tree((q, kc, vc, lengths, k, v, parents))
    again = skv.tree_attention(q, kc, vc, lengths, k, v, parents)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
    assert skv.tree_attention(q[:0], kc[:0], vc[:0], lengths[:0], k[:0], v[:0], parents[:0])[0].shape == (0, 2, 2, 64)


def test_tree_attention_offsets_beyond_32_bits():
    """The last sequence of a cache of more than 2^31 elements."""
    b, hkv, t, d = 5, 4, 1 << 19, 256
    kc = torch.empty(b, hkv, t, d, device="cuda", dtype=BF)
    vc = torch.empty_like(kc)
    assert kc.numel() > 2 ** 31
    g = gen(13)
    kc[-1, :, -300:] = normal(g, hkv, 300, d)
    vc[-1, :, -300:] = normal(g, hkv, 300, d)
    kc[-1, :, :-300] = 0
    vc[-1, :, :-300] = 1
    q, k, v = normal(g, b, 1, 4, d), normal(g, b, hkv, 1, d), normal(g, b, hkv, 1, d)
    lengths = torch.tensor([0] * (b - 1) + [t], dtype=torch.int32, device="cuda")
    parents = torch.full((b, 1), -1, dtype=torch.int32, device="cuda")
    check_tree((q, kc, vc, lengths, k, v, parents))
    w = torch.zeros(b, hkv, t, device="cuda")
    lse = skv.tree_attention(q, kc, vc, lengths, k, v, parents)[1]
    y = skv.accumulate_weights(q, kc, lengths, lse, w)
    close(y[-1:], *R.weights(q[-1:], kc[-1:], lengths[-1:], lse[-1:], w[-1:]))
    assert (y[:-1] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("b,n,hkv,t", [(3, 5, 1, 511), (3, 5, 1, 513), (70, 2, 2, 900), (129, 1, 1, 800), (129, 40, 1, 700),
                                       (148, 1, 1, 130), (149, 1, 1, 130), (9, 64, 4, 640)])
def test_tree_attention_whole_and_cut_units(b, n, hkv, t, dtype):
    """Both sides of the rule that leaves units whole, and launches of one call on different sides of it."""
    rng = random.Random(t)
    check_tree(tree_case(17, [rng.choice([0, 1, t // 2, t - 1, t]) for _ in range(b)], n, 4 * hkv, hkv, 64, t, dtype=dtype,
                         kind="padded"))


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("lengths,n,hq,hkv,d", [([0, 1, 63, 64, 65], 1, 4, 1, 256), ([127, 128, 129, 0], 5, 6, 2, 128),
                                                ([300, 7], 64, 4, 2, 64), ([20, 0, 70, 2600], 31, 4, 1, 256),
                                                ([0], 64, 16, 4, 256), ([1], 1, 1, 1, 64)])
def test_tree_attention_short_lengths_in_a_long_cache(lengths, n, hq, hkv, d, dtype):
    check_tree(tree_case(18, lengths, n, hq, hkv, d, 2700, dtype=dtype, kind="padded"))


@pytest.mark.parametrize("dtype", [BF, F8])
def test_tree_attention_cut_between_units(dtype):
    """Two units for every SM, cut where they end: every row is written by the first of the two kernels, and what
    follows the second must find it there."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    args = tree_case(16, [1000] * (sms // 2), 3, 8, 4, 128, 1000, dtype=dtype)
    copies = []
    for _ in range(8):
        out, lse = skv.tree_attention(*args)
        copies.append((out.clone(), lse.clone()))
        out.zero_()
    for out, lse in copies[1:]:
        assert torch.equal(out, copies[0][0]) and torch.equal(lse, copies[0][1])
    want, wl, eo, el = R.tree(*args)
    close(copies[0][0], want, eo)
    close(copies[0][1], wl, el)


def test_tree_attention_graph_follows_the_cache():
    """A captured call replayed after lengths, queries and the cache changed; two graphs of one program."""
    args = list(tree_case(14, [50, 200], 4, 8, 2, 128, 400))
    skv.tree_attention(*args)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(skv.tree_attention(*args))
        graphs.append(graph)
    args[3].copy_(torch.tensor([400, 1], dtype=torch.int32))
    args[0].mul_(0.5)
    args[1].mul_(1.25)
    want = skv.tree_attention(*args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for graph, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tree_attention_streams_overlap():
    """Calls on several streams at once give what they give alone."""
    cases = [tree_case(20 + i, [300 * (i + 1)], 8, 8, 2, 128, 1300, dtype=(BF, F8)[i % 2]) for i in range(4)]
    want = [skv.tree_attention(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(5):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(skv.tree_attention(*c))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for x in g:
            assert torch.equal(x[0], w[0]) and torch.equal(x[1], w[1])


def test_tree_attention_refuses():
    q, kc, vc, lengths, k, v, parents = tree_case(15, [10], 3, 4, 2, 64, 16)
    kc, vc = kc.contiguous(), vc.contiguous()

    def call(**kw):
        a = dict(q=q, k_cache=kc, v_cache=vc, lengths=lengths, k=k, v=v, parents=parents)
        a.update(kw)
        return skv.tree_attention(**a)

    call()
    odd = torch.zeros(kc.numel() + 8, device="cuda", dtype=BF)[4:4 + kc.numel()].view(kc.shape)
    for bad in (dict(q=q[:, :, :3]), dict(q=q.float()), dict(k_cache=kc.half()), dict(v_cache=vc.to(F8)),
                dict(lengths=lengths.long()), dict(lengths=lengths.cpu()), dict(k=k[:, :, :2]), dict(parents=parents.long()),
                dict(parents=parents[:, :2]), dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(k_cache=odd),
                dict(k_cache=kc[:, :, :1].expand(-1, -1, 16, -1)), dict(k_cache=kc[..., :32], v_cache=vc[..., :32]),
                dict(v_cache=vc[:, :, :15]), dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)),
                dict(q=q.clone().requires_grad_())):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError, match="nodes"):
        call(q=q.repeat(1, 22, 1, 1), k=k.repeat(1, 1, 22, 1), v=v.repeat(1, 1, 22, 1), parents=parents.repeat(1, 22))


# ---------------------------------------------------------------- accumulated weights


WEIGHTS = [
    dict(lengths=[0, 1, 127, 128, 129], n=1, hq=4, hkv=1, d=256, t=129),
    dict(lengths=[300, 5], n=33, hq=16, hkv=4, d=256, t=333),
    dict(lengths=[1000], n=70, hq=16, hkv=4, d=128, t=1001),
    dict(lengths=[260, 0, 70], n=100, hq=8, hkv=1, d=64, t=260),
    dict(lengths=[50], n=300, hq=2, hkv=1, d=256, t=50),
    dict(lengths=[1], n=1, hq=3, hkv=3, d=64, t=1),
]


def weights_case(seed, lengths, n, hq, hkv, d, t, dtype=BF):
    g = gen(seed)
    b = len(lengths)
    rec = normal(g, b, hkv, t, 2 * d).to(dtype)
    q = normal(g, b, n, hq, d) * 2
    lse = torch.randn(b, n, hq, device="cuda", generator=g) + 6.0
    w = torch.rand(b, hkv, t, device="cuda", generator=g)
    return q, rec[..., :d], torch.tensor(lengths, dtype=torch.int32, device="cuda"), lse, w


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("c", WEIGHTS)
def test_accumulate_weights(c, dtype):
    q, kc, lengths, lse, w = weights_case(31, dtype=dtype, **c)
    y = skv.accumulate_weights(q, kc, lengths, lse, w)
    close(y, *R.weights(q, kc, lengths, lse, w))
    rows = torch.rand(q.shape[:2], device="cuda", generator=gen(32)) < 0.5
    lse[:, ::3] = -INF
    want, bound = R.weights(q, kc, lengths, lse, w, rows, 0.05)
    got = skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows, scale=0.05)
    close(got, want, bound)
    assert torch.equal(got, skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows, scale=0.05))
    # in place, and into a strided part of another tensor
    big = torch.full((*w.shape, 2), 9.0, device="cuda")
    assert skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows, scale=0.05, out=big[..., 1]).data_ptr() == \
        big[..., 1].data_ptr()
    assert torch.equal(big[..., 1], got) and (big[..., 0] == 9).all()
    assert skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows, scale=0.05, out=w) is w
    assert torch.equal(w, got)


@pytest.mark.parametrize("dtype", [BF, F8])
def test_accumulate_weights_what_is_left_out_does_not_count(dtype):
    """Garbage behind the length, queries of rows that do not count, -inf rows."""
    q, kc, lengths, lse, w = weights_case(33, [100, 0], 6, 8, 2, 128, 140, dtype=dtype)
    rows = torch.tensor([[1, 0, 1, 1, 0, 1]] * 2, device="cuda", dtype=torch.bool)
    clean = skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows)
    kc = kc.clone()
    kc[0, :, 100:] = NAN
    kc[1] = NAN
    q[:, [1, 4]] = NAN
    lse[:, 1] = NAN
    lse[:, 4] = INF
    assert torch.equal(skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows), clean)
    lse[:, 5] = -INF
    q[:, 5] = INF
    rows[:, 5] = False
    want = skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows)
    rows[:, 5] = True
    assert torch.equal(skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows), want)
    rows[:] = False
    assert torch.equal(skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows), w)


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("n,rows", [(1, [1]), (1, [0]), (3, [0, 1, 0]), (7, [1] * 7), (40, [0, 1] * 20), (40, [0] * 40)])
def test_accumulate_weights_keys_that_are_not_finite(n, rows, dtype):
    """Only the rows that count meet such a key, each with what exp() gives."""
    q, kc, lengths, lse, w = weights_case(35, [300, 140], n, 8, 2, 128, 300, dtype=dtype)
    for i, value in enumerate([NAN] if dtype is F8 else [NAN, INF, -INF]):  # (e4m3 has no infinity)
        kc[:, :, 17 + 100 * i, 5 * i] = value
    rows = torch.tensor([rows] * 2, device="cuda", dtype=torch.bool)
    close(skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows), *R.weights(q, kc, lengths, lse, w, rows))


def test_accumulate_weights_sum_to_the_rows_over_the_cache():
    """With tree_attention's lse a row's weights over the cache and over its own line sum to one."""
    args = tree_case(34, [900, 300], 5, 8, 2, 128, 900, kind="chain")
    _, lse = skv.tree_attention(*args)
    y = skv.accumulate_weights(args[0], args[1], args[3], lse, torch.zeros(2, 2, 900, device="cuda"))
    want, _, _, _ = R.tree(*args)
    q, k = args[0].double(), args[4].double()
    for i in range(2):
        for h in range(2):
            z = torch.einsum("ngd,md->ngm", q[i, :, 4 * h:4 * h + 4], k[i, h]) / 128 ** 0.5
            own = torch.exp(z - lse[i, :, 4 * h:4 * h + 4].double()[..., None])
            own = own * torch.tril(torch.ones(5, 5, device="cuda"))[:, None]
            # 20 rows; scores of up to 60 in FP32 with D = 128: 24 * 2^-23 * 60, twice
            assert abs(float(y[i, h].double().sum() + own.sum()) - 20) < 20 * 4e-4


def test_accumulate_weights_refuses():
    q, kc, lengths, lse, w = weights_case(35, [10], 3, 4, 2, 64, 16)
    kc = kc.contiguous()

    def call(**kw):
        a = dict(q=q, k_cache=kc, lengths=lengths, lse=lse, weights=w)
        a.update(kw)
        return skv.accumulate_weights(**a)

    call()
    flat = torch.zeros(w.numel() + 4, device="cuda")
    for bad in (dict(lse=lse.double()), dict(lse=lse[:, :2]), dict(weights=w.double()), dict(weights=w[:, :, :15]),
                dict(rows=torch.ones(1, 3, device="cuda")), dict(rows=torch.ones(1, 2, dtype=torch.bool, device="cuda")),
                dict(scale=0.0), dict(weights=flat[:-4].view(w.shape), out=flat[4:].view(w.shape)),
                dict(out=w[:, :1].clone().expand(-1, 2, -1)), dict(q=q[:, :, :3]), dict(k_cache=kc.float()),
                dict(weights=w.clone().requires_grad_()), dict(q=q[:, :0], lse=lse[:, :0])):
        with pytest.raises(ValueError):
            call(**bad)


# ---------------------------------------------------------------- eviction


def check_evict(k, v, w, lengths, keep, sink, local):
    ko, vo, wo, ids, left = skv.evict(k, v, w, lengths, keep=keep, sink=sink, local=local)
    bits = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[k.element_size()]
    for i in range(k.shape[0]):
        n = max(0, min(int(lengths[i]), k.shape[2]))
        assert int(left[i]) == min(n, keep)
        for h in range(k.shape[1]):
            want = R.kept(w[i, h].tolist(), n, keep, sink, local)
            m = len(want)
            got = ids[i, h].tolist()
            assert got == want + [-1] * (keep - m), (i, h)
            at = torch.tensor(want, device="cuda", dtype=torch.int64)
            for x, y in ((k, ko), (v, vo), (w[..., None], wo[..., None])):
                b = bits if x.dtype != torch.float32 else torch.int32
                x, y = x[i, h].contiguous().view(b), y[i, h].view(b)
                assert torch.equal(y[:m], x[at]) and (y[m:] == 0).all()


EVICT = [
    dict(lengths=[1, 0], t=1, keep=1, sink=0, local=0),
    dict(lengths=[31, 32, 33, 12, 0], t=33, keep=13, sink=2, local=3),
    dict(lengths=[4096, 4000, 700], t=4096, keep=701, sink=0, local=0),
    dict(lengths=[4097, 4096], t=4097, keep=2000, sink=128, local=256),
    dict(lengths=[9000, 5], t=9001, keep=384, sink=128, local=256),
    dict(lengths=[30001], t=30001, keep=30000, sink=1, local=1),
    dict(lengths=[200001], t=200001, keep=77, sink=5, local=6),
]


@pytest.mark.parametrize("c", EVICT)
@pytest.mark.parametrize("values", ["spread", "ties", "special"])
def test_evict(c, values):
    g = gen(41)
    b, h, d, t = len(c["lengths"]), 2, 64, c["t"]
    k, v = normal(g, b, h, t, d), normal(g, b, h, t, d)
    w = torch.exp(3 * torch.randn(b, h, t, device="cuda", generator=g))
    if values == "ties":
        w = torch.randint(0, 3, (b, h, t), device="cuda", generator=g).float() - 1
        w[w == 0] *= -1  # -0
    elif values == "special":
        special = torch.tensor([NAN, INF, -INF, 0.0, -0.0, 1e-42, -1e-42, 3.0], device="cuda")
        pick = torch.randint(0, 16, (b, h, t), device="cuda", generator=g)
        w = torch.where(pick < 8, special[pick % 8], -w)
    lengths = torch.tensor(c["lengths"], dtype=torch.int32, device="cuda")
    check_evict(k, v, w, lengths, c["keep"], c["sink"], c["local"])


@pytest.mark.parametrize("dtype,d", [(F8, 3), (F8, 64), (BF, 1), (BF, 6), (torch.float16, 128), (torch.float32, 320)])
def test_evict_types_rows_and_strides(dtype, d):
    g = gen(42)
    k, v = (normal(g, 2, 50, 3, d).to(dtype).transpose(1, 2) for _ in range(2))
    w = torch.rand(2, 50, 3, 2, device="cuda", generator=g)[..., 1].transpose(1, 2)
    lengths = torch.tensor([50, 0, 41, 0], dtype=torch.int32, device="cuda")[::2]
    check_evict(k, v, w, lengths, 20, 3, 4)
    rec = normal(g, 2, 3, 50, 2 * d).to(dtype)
    check_evict(rec[..., :d], rec[..., d:], w, lengths, 20, 0, 0)


@pytest.mark.parametrize("t", [524288, 786432, 786433, 1000003])
def test_evict_long_rows(t):
    """Rows of sixteen CTAs whose keys just fit into shared memory, and longer ones."""
    g = gen(47)
    k, v = (torch.randint(0, 120, (1, 2, t, 1), device="cuda", generator=g, dtype=torch.uint8).view(F8) for _ in range(2))
    check_evict(k, v, torch.rand(1, 2, t, device="cuda", generator=g), torch.tensor([t - 3], dtype=torch.int32, device="cuda"),
                t // 3, 4, 100)


def test_evict_graph_and_offsets():
    g = gen(43)
    k, v, w = normal(g, 1, 2, 5000, 64), normal(g, 1, 2, 5000, 64), torch.rand(1, 2, 5000, device="cuda", generator=g)
    lengths = torch.tensor([5000], dtype=torch.int32, device="cuda")
    skv.evict(k, v, w, lengths, keep=100, sink=2, local=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = skv.evict(k, v, w, lengths, keep=100, sink=2, local=2)
    w.copy_(1 - w)
    lengths.fill_(4321)
    graph.replay()
    want = skv.evict(k, v, w, lengths, keep=100, sink=2, local=2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # rows behind 2^31 elements
    t = 1 << 20
    k = torch.empty(1, 9, t, 256, device="cuda", dtype=BF)
    w = torch.zeros(1, 9, t, device="cuda")
    pick = torch.arange(5, t, t // 40, device="cuda")
    k[:, :, pick] = normal(g, 1, 9, pick.numel(), 256)
    w[:, :, pick] = 1.0
    n = pick.numel()
    ko, vo, _, ids, _ = skv.evict(k, k, w, torch.tensor([t], dtype=torch.int32, device="cuda"), keep=n, sink=0, local=0)
    assert torch.equal(ids[0, 8], pick.int()) and torch.equal(ko, k[:, :, pick]) and torch.equal(vo, ko)


def test_evict_refuses():
    g = gen(44)
    k, w, n = normal(g, 1, 2, 40, 64), torch.rand(1, 2, 40, device="cuda"), torch.tensor([40], dtype=torch.int32, device="cuda")

    def call(**kw):
        a = dict(k_cache=k, v_cache=k, weights=w, lengths=n, keep=20, sink=2, local=2)
        a.update(kw)
        return skv.evict(**a)

    call()
    for bad in (dict(keep=0), dict(keep=41), dict(keep=3), dict(sink=-1), dict(local=19), dict(keep=20.0), dict(weights=w.half()),
                dict(weights=w[:, :1]), dict(v_cache=k.half()), dict(lengths=n.long()), dict(k_cache=k.int()),
                dict(k_cache=k.transpose(2, 3)), dict(weights=w.clone().requires_grad_())):
        with pytest.raises(ValueError):
            call(**bad)


# ---------------------------------------------------------------- together


@pytest.mark.parametrize("dtype", [BF, F8])
def test_draft_verify_accumulate_evict(dtype):
    """A drafting decode loop as a server runs it: rotate the drafts, attend,
    accept a line of the tree, weigh and append it, evict when the caches are
    full; every step against the definitions on what that step was given."""
    g, rng = gen(51), random.Random(51)
    b, n, hq, hkv, d, room, keep = 2, 6, 8, 2, 128, 150, 100
    cache = [torch.zeros(b, hkv, room, d, device="cuda", dtype=dtype) for _ in range(2)]
    weights = torch.zeros(b, hkv, room, device="cuda")
    lengths = torch.tensor([90, 140], dtype=torch.int32, device="cuda")
    position = torch.tensor([90, 140], device="cuda")
    for x in cache:
        x.copy_(normal(g, b, hkv, room, d).to(dtype))
    f, m = R.frequencies(d)
    evictions = 0
    for step in range(4):
        parents = torch.tensor([make_parents(rng, n, "tree") for _ in range(b)], dtype=torch.int32, device="cuda")
        depth = torch.tensor([[len(R.visible(p)[i].nonzero()) - 1 for i in range(n)] for p in parents.tolist()], device="cuda")
        q, k, v = normal(g, b, n, hq, d), normal(g, b, hkv, n, d), normal(g, b, hkv, n, d)
        pos = position[:, None] + depth
        qr, kr = skv.rotary(q, k, pos)
        close(qr, *R.rotated(q, pos, d, "half", f, m, 2))
        close(kr, *R.rotated(k, pos, d, "half", f, m, 1))
        out, lse = check_tree((qr, *cache, lengths, kr, v, parents))
        line = [R.visible(p)[rng.randrange(n)] for p in parents.tolist()]
        accepted = torch.stack(line).cuda()
        new = skv.accumulate_weights(qr, cache[0], lengths, lse, weights, rows=accepted)
        close(new, *R.weights(qr, cache[0], lengths, lse, weights, accepted))
        weights = new
        for i in range(b):
            m_new, at = int(accepted[i].sum()), int(lengths[i])
            cache[0][i, :, at:at + m_new] = kr[i][:, accepted[i]].to(dtype)
            cache[1][i, :, at:at + m_new] = v[i][:, accepted[i]].to(dtype)
            weights[i, :, at:at + m_new] = 0
            lengths[i] += m_new
            position[i] += m_new
        if int(lengths.max()) > room - n:
            check_evict(*cache, weights, lengths, keep, 4, 16)
            ko, vo, wo, _, lengths = skv.evict(*cache, weights, lengths, keep=keep, sink=4, local=16)
            for x, y in zip((*cache, weights), (ko, vo, wo)):
                x.zero_()
                x[:, :, :keep] = y
            evictions += 1
    assert evictions


CAPTURED = """
import torch
import seoulkv_b200 as skv

b, n, hq, hkv, d, room, keep = 2, 6, 8, 2, 128, 700, 300
g = torch.Generator(device="cuda").manual_seed(53)
normal = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
q, k, v = normal(b, n, hq, d), normal(b, hkv, n, d), normal(b, hkv, n, d)
caches = normal(b, hkv, room, d), normal(b, hkv, room, d)
lengths = torch.tensor([690, 100], dtype=torch.int32, device="cuda")
positions = lengths.long()[:, None] + torch.arange(n, device="cuda")
parents = torch.tensor([[-1, 0, 0, 2, -1, 9]] * b, dtype=torch.int32, device="cuda")
accepted = torch.ones(b, n, dtype=torch.bool, device="cuda")
weights = torch.zeros(b, hkv, room, device="cuda")


def step():
    skv.rotary(q, k, positions, out=(q, k))
    out, lse = skv.tree_attention(q, *caches, lengths, k, v, parents)
    skv.accumulate_weights(q, caches[0], lengths, lse, weights, rows=accepted, out=weights)
    return (out, lse, *skv.evict(*caches, weights, lengths, keep=keep, sink=4, local=16))


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
for turn in range(3):
    lengths.fill_(turn * 300 + 7)
    caches[0].mul_(0.75)
    start = [x.clone() for x in (q, k, weights)]
    graph.replay()
    got = [x.clone() for x in (*captured, q, k, weights)]
    for x, y in zip((q, k, weights), start):
        x.copy_(y)
    want = (*step(), q, k, weights)
    for i, (x, y) in enumerate(zip(got, want)):
        assert torch.equal(x.nan_to_num(nan=7.0), y.nan_to_num(nan=7.0)), (turn, i)
skv.check_operators("cuda:0")
"""


def test_first_calls_captured_together():
    """One graph of all operators, in place where they may be, as a process's first calls of them;
    replayed with other contents it gives what eager calls give."""
    done = subprocess.run([sys.executable, "-c", CAPTURED], capture_output=True, text=True, timeout=600,
                          cwd=pathlib.Path(__file__).parents[1])
    assert done.returncode == 0, done.stderr[-2000:]


# ---------------------------------------------------------------- the engine's own cache


@pytest.fixture(scope="module")
def grown():
    from tests.helpers import AppendCase

    return AppendCase()  # built on 8192 tokens, grows to 8892


def records(ac, t):
    """The engine's FP8 records of the first t tokens, [4, t, 256] each."""
    return [torch.stack([x[g][:t] for g in range(4)]).to(F8).cuda() for x in (ac.k_full, ac.v_full)]


def drafted(seed, slots, n):
    g, rng = gen(seed), random.Random(seed)
    q = normal(g, slots, n, 16, 256)
    k, v = normal(g, slots, 4, n, 256), normal(g, slots, 4, n, 256)
    parents = torch.tensor([make_parents(rng, n, "tree") for _ in range(slots)], dtype=torch.int32, device="cuda")
    return q, k, v, parents


def test_run_tree_sees_the_engines_cache(grown, cuda):
    """Exact attention over the FP8 records, before and after appends, on the
    device and captured; equal to tree_attention over the same records."""
    cfg = skv.SeoulKV4Config(max_context=grown.total)
    q, k, v, parents = drafted(61, 1, 7)
    with skv.SeoulKV4(device=cuda, k=grown.k, v=grown.v, index=grown.index,
                      config=cfg) as attn:
        t = grown.context

        def check(out, lse, t):
            kc, vc = records(grown, t)
            n = torch.tensor([t], dtype=torch.int32, device="cuda")
            want, wl, eo, el = R.tree(q, kc[None], vc[None], n, k, v, parents)
            close(out, want, eo)
            close(lse, wl, el)

        check(*attn.run_tree(q, k[0], v[0], parents[0]), t)
        host = attn.run_tree(q.cpu(), k[0].cpu(), v[0].cpu(), parents[0].cpu())
        assert torch.equal(host[0], attn.run_tree(q, k[0], v[0], parents[0])[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = attn.run_tree(q, k[0], v[0], parents[0])
        for m in (1, 300):
            attn.append(*grown.appended(t, t + m))
            t += m
            check(*attn.run_tree(q, k[0], v[0], parents[0]), t)
            graph.replay()
            check(out, lse, t)
        # run() and the tree share the cache without touching each other
        y = attn.run(grown.query(t, seed=3)).to_torch()
        attn.run_tree(q, k[0], v[0], parents[0])
        assert torch.equal(attn.run(grown.query(t, seed=3)).to_torch(), y)
        for bad in (dict(q=q[:, :, :4]), dict(q=q.float()), dict(k=k), dict(v=v[0, :, :3]), dict(parents=parents),
                    dict(parents=parents[0].long()), dict(q=q.clone().requires_grad_())):
            a = dict(q=q, k=k[0], v=v[0], parents=parents[0])
            a.update(bad)
            with pytest.raises(ValueError):
                attn.run_tree(**a)
    with pytest.raises(RuntimeError, match="closed"):
        attn.run_tree(q, k[0], v[0], parents[0])


def test_run_tree_batched(grown, cuda):
    """Every cache's own tree, equal to one instance per cache."""
    t = grown.context
    kv = [(grown.k, grown.v, grown.index)] * 3
    q, k, v, parents = drafted(62, 3, 5)
    with skv.SeoulKV4Batch(device=cuda, caches=kv) as batch:
        out, lse = batch.run_tree(q, k, v, parents)
    with skv.SeoulKV4(device=cuda, k=grown.k, v=grown.v, index=grown.index) as attn:
        for i in range(3):
            one, l1 = attn.run_tree(q[i:i + 1], k[i], v[i], parents[i])
            # (the same tiles joined at other places: three roundings of the weights apart)
            assert float((one.double() - out[i:i + 1].double()).abs().max()) <= 3 * 2.0 ** -8 * float(one.abs().max())
            assert float((l1 - lse[i:i + 1]).abs().max()) < 1e-4
