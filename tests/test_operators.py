"""Operators around a decode step, without a GPU: what they refuse, at the
Python functions and at the C ABI (before any CUDA call)."""

import ctypes
import struct

import pytest
import torch

import seoulkv_b200 as skv
from seoulkv_b200 import _native, operators
from tests import operator_reference as R

BF = torch.bfloat16


def q_k(b=1, n=2, hq=4, hkv=2, d=64, dtype=BF):
    return torch.zeros(b, n, hq, d, dtype=dtype), torch.zeros(b, hkv, n, d, dtype=dtype)


def test_cpu_tensors_are_refused():
    q, k = q_k()
    cache, n = torch.zeros(1, 2, 9, 64, dtype=BF), torch.ones(1, dtype=torch.int32)
    for call in (lambda: skv.rotary(q, k, torch.arange(2)),
                 lambda: skv.tree_attention(q, cache, cache, n, k, k, torch.full((1, 2), -1, dtype=torch.int32)),
                 lambda: skv.accumulate_weights(q, cache, n, torch.zeros(1, 2, 4), torch.zeros(1, 2, 9)),
                 lambda: skv.evict(cache, cache, torch.zeros(1, 2, 9), n, keep=4, sink=1, local=1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_wrong_types_and_shapes_are_refused():
    q, k = q_k()
    with pytest.raises(ValueError, match="q: expected"):
        skv.rotary(q.to(torch.float64), k, torch.arange(2))
    with pytest.raises(ValueError, match="shape"):
        skv.rotary(q[0], k, torch.arange(2))
    with pytest.raises(ValueError, match="k_cache: expected a"):
        skv.evict(q.to(torch.int8), q, q, q, keep=1)
    with pytest.raises(ValueError, match="k_cache"):
        skv.tree_attention(q, k.half(), k, None, k, k, None)


def test_rotary_table_refusals_and_values():
    t = operators._rotary_table.__wrapped__
    for bad in (dict(theta=-1.0), dict(theta=1.0), dict(factor=0.0), dict(scaling="other"),
                dict(scaling="yarn", original_context=None), dict(scaling="yarn", original_context=8, beta_fast=1.0),
                dict(attention_factor=float("inf"))):
        kw = dict(theta=1e4, scaling="none", factor=2.0, original_context=4096, beta_fast=32.0, beta_slow=1.0,
                  attention_factor=None)
        kw.update(bad)
        with pytest.raises(ValueError):
            t(64, **kw)
    # the fractions of a turn are the definition's, for every scaling
    for scaling in ("none", "linear", "ntk", "yarn"):
        buf, _, m = t(128, 1e4, scaling, 4.0, 8192, 32.0, 1.0, None)
        got = [x / 2.0 ** 64 * 2 * 3.141592653589793 for x in struct.unpack("64Q", buf.raw[:512])]
        want, wm = R.frequencies(128, scaling=scaling, factor=4.0, original=8192)
        assert m == wm and max(abs(a / b - 1) for a, b in zip(got, want)) < 1e-13


def test_descriptors_match_the_header():
    """The packed descriptors have the C structs' sizes (all fields are 8 bytes)."""
    import re
    from pathlib import Path

    text = (Path(__file__).resolve().parent.parent / "include" / "seoulkv_b200.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, layout in (("SkvRotary", operators._ROTARY), ("SkvTree", operators._TREE),
                         ("SkvWeights", operators._WEIGHTS), ("SkvEvict", operators._EVICT)):
        body = re.search(rf"typedef struct {name} \{{(.*?)\}} {name};", text, flags=re.S).group(1)
        n = 0
        for decl in filter(None, (x.strip() for x in body.split(";"))):
            for field in decl.split(","):
                size = re.search(r"\[(\d+)\]", field)
                n += int(size.group(1)) if size else 1
        assert layout.size == 8 * n, name


def _refused(name, packed):
    lib = _native.load()
    rc = getattr(lib, name)(packed, None)
    return rc, lib.skv_last_error().decode()


P = 4096  # any aligned non-null address: refused before it is used


def _tree(**kw):
    f = dict(scale=0.1, device=0, dtype=0, bytes=0, b=1, n=2, hq=4, hkv=2, d=64, t=9, ptr=P)
    f.update(kw)
    return operators._TREE.pack(*([f["ptr"]] * 10), f["scale"], f["device"], f["dtype"], f["bytes"], f["b"], f["n"],
                                f["hq"], f["hkv"], f["d"], f["t"], *([*([f.get("stride", 64)] * 3), f.get("inner", 1)] * 5), 64, 64, 1)


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=65), dict(d=96), dict(hq=5), dict(hkv=0), dict(t=0), dict(t=1 << 30),
                                 dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(dtype=2),
                                 dict(b=-1), dict(ptr=0), dict(ptr=P + 2), dict(stride=4), dict(stride=-64),
                                 dict(inner=2)])
def test_c_tree_attention_refuses(bad):
    rc, message = _refused("skv_tree_attention", _tree(**bad))
    assert rc == -1 and message


def _weights(**kw):
    f = dict(scale=0.1, device=0, dtype=0, b=1, n=2, hq=4, hkv=2, d=64, t=9, ptr=P)
    f.update(kw)
    return operators._WEIGHTS.pack(*([f["ptr"]] * 7), f["scale"], f["device"], f["dtype"], f["b"], f["n"], f["hq"],
                                   f["hkv"], f["d"], f["t"], *([*([f.get("stride", 64)] * 3), f.get("inner", 1)] * 2), *([64] * 12))


@pytest.mark.parametrize("bad", [dict(n=0), dict(d=63), dict(hq=5), dict(t=0), dict(scale=-1.0), dict(dtype=1), dict(ptr=0),
                                 dict(ptr=P + 8), dict(stride=12), dict(inner=0)])
def test_c_accumulate_weights_refuses(bad):
    rc, message = _refused("skv_accumulate_weights", _weights(**bad))
    assert rc == -1 and message


def _evict(**kw):
    f = dict(device=0, b=1, hkv=2, t=9, d=64, size=2, keep=4, sink=1, local=1, ptr=P)
    f.update(kw)
    return operators._EVICT.pack(*([f["ptr"]] * 9), f["device"], f["b"], f["hkv"], f["t"], f["d"], f["size"], f["keep"],
                                 f["sink"], f["local"], *([64, 64, 64, f.get("inner", 1)] * 2), *([64] * 4))


@pytest.mark.parametrize("bad", [dict(keep=0), dict(keep=10), dict(sink=4), dict(sink=-1), dict(local=-1), dict(hkv=0),
                                 dict(t=0), dict(d=0), dict(d=1 << 20), dict(size=3), dict(ptr=0), dict(b=-1), dict(inner=2)])
def test_c_evict_refuses(bad):
    rc, message = _refused("skv_evict", _evict(**bad))
    assert rc == -1 and message


def _rotary(**kw):
    f = dict(device=0, dtype=0, layout=0, b=1, n=2, hq=4, hkv=2, d=64, r=64, ptr=P, stride=64)
    f.update(kw)
    return operators._ROTARY.pack(*([f["ptr"]] * 6), 1.0, f["device"], f["dtype"], f["layout"], 0, f["b"], f["n"], f["hq"],
                                  f["hkv"], f["d"], f["r"], *([*([f["stride"]] * 3), f.get("inner", 1)] * 4), 64, 1)


@pytest.mark.parametrize("bad", [dict(r=0), dict(r=63), dict(r=66), dict(d=1), dict(hq=0), dict(hkv=-1), dict(dtype=3),
                                 dict(layout=2), dict(ptr=0), dict(b=-1), dict(d=1026, r=514), dict(inner=2)])
def test_c_rotary_refuses(bad):
    rc, message = _refused("skv_rotary", _rotary(**bad))
    assert rc == -1 and message


def test_null_descriptors_are_refused():
    lib = _native.load()
    for name in ("skv_rotary", "skv_tree_attention", "skv_accumulate_weights", "skv_evict"):
        assert getattr(lib, name)(None, None) == -1
    assert lib.skv_tree_workspace(_tree(), None) == -1
    assert lib.skv_operator_status(0, None) == -1
    assert lib.skv_run_tree(None, _tree(), None) == -1


@pytest.mark.parametrize("device", [-1, 64, 1 << 32, (1 << 32) + 1])
def test_devices_out_of_range_are_refused(device):
    for name, packed in (("skv_rotary", _rotary(device=device)), ("skv_tree_attention", _tree(device=device)),
                         ("skv_accumulate_weights", _weights(device=device)), ("skv_evict", _evict(device=device))):
        rc, message = _refused(name, packed)
        assert rc == -1 and "device" in message, name
    size = ctypes.c_int64()
    assert _native.load().skv_tree_workspace(_tree(device=device), ctypes.byref(size)) == -1


def test_empty_batches_need_no_gpu():
    for name, packed in (("skv_rotary", _rotary(b=0)), ("skv_tree_attention", _tree(b=0)),
                         ("skv_accumulate_weights", _weights(b=0)), ("skv_evict", _evict(b=0))):
        assert _refused(name, packed)[0] == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU error path")
def test_no_gpu_is_an_error_status():
    flags = ctypes.c_uint32()
    assert _native.load().skv_operator_status(0, ctypes.byref(flags)) == -2
    assert _refused("skv_evict", _evict())[0] == -2


def test_reference_visibility_and_eviction():
    """The tests' own definitions on cases that can be checked by hand."""
    see = R.visible([-1, 0, 0, 1, -2, 4, 7, -1])
    assert [see[i].nonzero().flatten().tolist() for i in range(8)] == [
        [0], [0, 1], [0, 2], [0, 1, 3], [], [], [], [7]]
    nan = float("nan")
    assert R.kept([5.0, nan, 1.0, 1.0, -0.0, 0.0, 9.0], 7, 4, 1, 1) == [0, 2, 3, 6]
    assert R.kept([0.0, nan, -1.0, -float("inf"), 3.0], 5, 4, 0, 1) == [0, 2, 3, 4]
    assert R.kept([1.0] * 9, 3, 4, 0, 0) == [0, 1, 2]
