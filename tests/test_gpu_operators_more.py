"""Operators around a decode step on the B200: orders of execution, reports and
arguments beside those of tests/test_gpu_operators.py, against the same 64-bit
definitions and bounds."""

import math

import pytest
import torch

import seoulkv_b200 as skv
from tests import operator_reference as R
from tests.test_gpu_operators import BF, F8, INF, NAN, close, drafted, gen, grown, normal, records, tree_case  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_wait_gave_up(cuda):
    yield
    skv.check_operators(cuda)


# ---------------------------------------------------------------- tree attention


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("n", [1, 9, 32])
def test_tree_attention_maxima_of_the_two_halves_of_a_row(n, dtype):
    """Scores of hundreds whose maximum changes sides of a tile from tile to
    tile: both threads of a row need the same one, at every tile, every time."""
    args = list(tree_case(71, [3000, 1500], n, 16, 4, 256, 3000, dtype=dtype, sharp=8.0))
    t = torch.arange(3000, device="cuda")
    # keys of one half of a tile outweigh the other's, tile by tile in turn, and grow along the cache
    size = torch.where((t // 64 + t // 128) % 2 == 0, 1.0, 0.1) * (0.2 + t / 3000)
    args[1] = (args[1].float() * size[:, None]).to(dtype)
    out, lse = skv.tree_attention(*args)
    want, wl, eo, el = R.tree(*args)
    close(out, want, eo)
    close(lse, wl, el)
    for _ in range(20):
        again = skv.tree_attention(*args)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("poison", [NAN, INF, -INF])
def test_tree_attention_value_that_is_not_finite_in_a_part_of_no_weight(poison, dtype):
    """A visible value that is not finite reaches the output however small its
    weight is, also where the part of the cache that holds it was another CTA's:
    scores of -128 against 0 leave it a weight below FP32's smallest number."""
    if dtype is F8 and poison == poison:
        pytest.skip("e4m3 has no infinity")
    g, t, d = gen(75), 40000, 64
    q = torch.full((1, 1, 2, d), 4.0, device="cuda", dtype=BF)
    kc = torch.zeros(1, 1, t, d, device="cuda", dtype=BF)
    kc[:, :, :600] = -4.0  # 4 * 4 * 64 / 8 = 128
    vc = normal(g, 1, 1, t, d)
    vc[0, 0, 10, 5] = poison
    k, v = torch.zeros(1, 1, 1, d, device="cuda", dtype=BF), normal(g, 1, 1, 1, d)
    one = torch.full((1, 1), -1, dtype=torch.int32, device="cuda")
    out, lse = skv.tree_attention(q, kc.to(dtype), vc.to(dtype), torch.tensor([t], dtype=torch.int32, device="cuda"), k, v, one)
    assert not torch.isfinite(out[..., 5]).any()
    rest = [x for x in range(d) if x != 5]
    assert torch.isfinite(out[..., rest]).all() and torch.isfinite(lse).all()


# ---------------------------------------------------------------- the engine's own cache


def _tree_over_records(q, k, v, parents, ac, values, t):
    kc = torch.stack([ac.k_full[g][:t] for g in range(4)]).to(F8).cuda()
    n = torch.tensor([t], dtype=torch.int32, device="cuda")
    return R.tree(q, kc[None], values.to(F8).cuda()[None], n, k, v, parents)


def test_run_tree_of_engines_that_follow_one_another(grown, cuda):  # noqa: F811
    """Engines with other records in turn in one process: each one's tensor maps
    and records may lie where a closed one's lay, and each call sees its own."""
    q, k, v, parents = drafted(72, 1, 7)
    t = grown.context
    outs = []
    for turn in range(4):
        values = torch.roll(grown.v, 1000 * turn + 1, 1) * (1.0 + turn)
        room = t if turn % 2 else grown.total
        with skv.SeoulKV4(device=cuda, k=grown.k, v=values, index=grown.index,
                          config=skv.SeoulKV4Config(max_context=room)) as attn:
            out, lse = attn.run_tree(q, k[0], v[0], parents[0])
            want, wl, eo, el = _tree_over_records(q, k, v, parents, grown, values, t)
            close(out, want, eo)
            close(lse, wl, el)
            again = attn.run_tree(q, k[0], v[0], parents[0])
            assert torch.equal(again[0], out) and torch.equal(again[1], lse)
            outs.append(out)
    assert all(not torch.equal(outs[0], x) for x in outs[1:])


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2+ GPUs")
def test_run_tree_on_another_device_than_the_current_one(grown):  # noqa: F811
    q, k, v, parents = drafted(73, 1, 5)
    with skv.SeoulKV4(device="cuda:1", k=grown.k, v=grown.v, index=grown.index) as attn:
        attn.run(grown.query(grown.context, seed=3)).to_torch()
        torch.cuda.set_device(0)
        out, lse = attn.run_tree(q, k[0], v[0], parents[0])
        assert out.get_device() == 1 and torch.cuda.current_device() == 0
        want, wl, eo, el = _tree_over_records(q, k, v, parents, grown, grown.v, grown.context)
        close(out.cuda(0), want, eo)
        close(lse.cuda(0), wl, el)


# ---------------------------------------------------------------- rotary


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 6.5), ("ntk", 4.0)])
def test_rotary_values_at_far_positions(scaling, factor, layout):
    """Rotated values against angles of 60 digits, also where positions differ
    above bit 31 alone.  Beside R.rotated()'s bound: a position p is off by
    p 2^-65 turns, p 2^-65 2 pi of |a| + |b|."""
    r, g = 64, gen(74)
    positions = [7, 2 ** 24 + 1, 2 ** 31 + 5, 5, 2 ** 32 + 7, 2 ** 33 + 7, 2 ** 33 + 8, 2 ** 39 - 1, -7, -(2 ** 32) - 7, -(2 ** 38) - 3]
    q = normal(g, 1, len(positions), 3, 96, dtype=torch.float32)
    pos = torch.tensor(positions, device="cuda")
    y, _ = skv.rotary(q, None, pos, rotary_dim=r, layout=layout, scaling=scaling, factor=factor)
    turns = [[float(x) for x in row] for row in R.exact_turns(r, positions, 1e4, factor, scaling)]
    ang = 2 * math.pi * torch.tensor(turns, dtype=torch.float64, device="cuda")[None, :, None]
    ia = torch.arange(r // 2, device="cuda") * (1 if layout == "half" else 2)
    ib = ia + (r // 2 if layout == "half" else 1)
    x = q.double()
    u, w = x[..., ia], x[..., ib]
    size = u.abs() + w.abs()
    bound = size * (2.0 ** -20 + 2.0 ** -64 * math.pi * pos.abs()[None, :, None, None]) + 2.0 ** -120
    assert ((y[..., ia].double() - (u * ang.cos() - w * ang.sin())).abs() <= bound).all()
    assert ((y[..., ib].double() - (u * ang.sin() + w * ang.cos())).abs() <= bound).all()
    assert torch.equal(y[..., r:], q[..., r:])


def test_rotary_follows_the_value_of_its_settings():
    """A setting given as a tensor counts by its value at the call, not as the object that an earlier call had."""
    q, pos = normal(gen(81), 1, 5, 2, 64, dtype=torch.float32), torch.arange(5, device="cuda") + 9
    theta, factor = torch.tensor(1e4), torch.tensor(2.0)
    skv.rotary(q, None, pos, theta=theta, scaling="linear", factor=factor)
    theta.fill_(5e5)
    factor.fill_(4.0)
    got = skv.rotary(q, None, pos, theta=theta, scaling="linear", factor=factor)[0]
    assert torch.equal(got, skv.rotary(q, None, pos, theta=5e5, scaling="linear", factor=4.0)[0])


# ---------------------------------------------------------------- accumulated weights


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("n,hq", [(40003, 4), (8195, 48)])
def test_accumulate_weights_of_a_long_window(n, hq, dtype):
    """More than 2^17 rows a KV head: the number of nodes is not limited."""
    g, t, d = gen(76), 70, 64
    q, kc = normal(g, 1, n, hq, d), normal(g, 1, 1, t, d).to(dtype)
    lse = torch.randn(1, n, hq, device="cuda", generator=g) + 12.0
    rows = torch.rand(1, n, device="cuda", generator=g) < 0.5
    w, lengths = torch.rand(1, 1, t, device="cuda", generator=g), torch.tensor([t - 3], dtype=torch.int32, device="cuda")
    close(skv.accumulate_weights(q, kc, lengths, lse, w, rows=rows), *R.weights(q, kc, lengths, lse, w, rows))


# ---------------------------------------------------------------- autograd around the operators


def test_outputs_given_to_an_operator_count_as_changed():
    """A tensor that backward needs and that an operator then writes to: an error, not a wrong gradient."""
    pos = torch.arange(3, device="cuda")
    for name in ("q", "k", "w"):
        q, k = normal(gen(77), 1, 3, 4, 64, dtype=torch.float32), normal(gen(78), 1, 2, 3, 64, dtype=torch.float32)
        kc, w = normal(gen(79), 1, 2, 9, 64), torch.rand(1, 2, 9, device="cuda")
        x = dict(q=q, k=k, w=w)[name]
        factor = torch.ones_like(x, requires_grad=True)
        y = (factor * x).sum()
        before = x._version
        if name == "w":
            skv.accumulate_weights(q.to(BF), kc, torch.tensor([9], dtype=torch.int32, device="cuda"),
                                   torch.full((1, 3, 4), 5.0, device="cuda"), w, out=w)
        else:
            skv.rotary(q, k, pos, out=(q, k))
        assert x._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        q = torch.ones(1, 3, 4, 64, device="cuda")
        skv.rotary(q, None, pos, out=(q, None))


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    args = tree_case(80, [9], 3, 4, 2, 64, 16)
    q, kc, vc, lengths, k, v, parents = args
    lse, w = torch.zeros(1, 3, 4, device="cuda"), torch.zeros(1, 2, 16, device="cuda")
    with fwd.dual_level():
        def dual(x):
            return fwd.make_dual(x, torch.ones_like(x))

        skv.tree_attention(*args)  # (without a tangent)
        for call in (lambda: skv.rotary(dual(q), None, torch.arange(3, device="cuda")),
                     lambda: skv.rotary(q, dual(k), torch.arange(3, device="cuda")),
                     lambda: skv.tree_attention(dual(q), *args[1:]),
                     lambda: skv.tree_attention(q, kc, dual(vc), lengths, k, v, parents),
                     lambda: skv.tree_attention(q, kc, vc, lengths, k, dual(v), parents),
                     lambda: skv.accumulate_weights(q, kc, lengths, dual(lse), w),
                     lambda: skv.accumulate_weights(q, kc, lengths, lse, dual(w)),
                     lambda: skv.evict(kc, dual(vc), w, lengths, keep=4, sink=0, local=0)):
            with pytest.raises(ValueError, match="tangent"):
                call()


def test_rotary_in_place_refuses_q_and_k_that_share_places():
    """Each element would turn twice, in any order."""
    pos = torch.arange(6, device="cuda")
    x = normal(gen(82), 2, 6, 4, 64)
    before = x.clone()
    k = x.transpose(1, 2)
    with pytest.raises(ValueError, match="share places"):
        skv.rotary(x, k, pos, out=(x, k))
    with pytest.raises(ValueError, match="share places"):
        skv.rotary(x, k[:, 3:], pos, out=(x, k[:, 3:]))
    with pytest.raises(ValueError, match="share one place"):
        windows = torch.zeros(64 + 8 * 5, device="cuda", dtype=BF).unfold(0, 64, 8)[None, :, None]
        skv.rotary(windows, None, pos, out=(windows, None))
    assert torch.equal(x, before)
    # parts side by side in every head turn as copies of them do
    qkv = normal(gen(83), 2, 6, 4, 3, 64)
    want = skv.rotary(qkv[:, :, :, 0].contiguous(), qkv[:, :, :, 1].transpose(1, 2).contiguous(), pos)
    q, k, v = qkv[:, :, :, 0], qkv[:, :, :, 1].transpose(1, 2), qkv[:, :, :, 2].clone()
    skv.rotary(q, k, pos, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, :, :, 2], v)


def test_synchronize_waits_for_the_last_tree(grown, cuda):  # noqa: F811
    """Also for one on another stream than any run, before the first run and after it."""
    q, k, v, parents = drafted(84, 1, 3)
    side = torch.cuda.Stream()
    with skv.SeoulKV4(device=cuda, k=grown.k, v=grown.v, index=grown.index) as attn:
        attn.run_tree(q, k[0], v[0], parents[0])
        for turn in range(2):
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                torch.cuda._sleep(200_000_000)  # a tenth of a second
                out, _ = attn.run_tree(q, k[0], v[0], parents[0])
            assert not side.query()
            attn.synchronize()
            assert side.query()
            assert torch.isfinite(out).all()
            attn.run(grown.query(grown.context, seed=3)).to_torch()
