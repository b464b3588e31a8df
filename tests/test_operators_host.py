"""Parts of the operators that can be checked without a GPU: the order of
accesses to shared memory, tables, refusals and reports."""

import random
import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest
import torch

from seoulkv_b200 import operators
from tests import operator_reference as R

CSRC = Path(__file__).resolve().parent.parent / "seoulkv_b200" / "csrc"


# ---------------------------------------------------------------- values that two threads exchange


def _slots(tmp_path, tiles):
    """exchange_slot(half, tile) of the kernel's own header: [half][tile]."""
    if not shutil.which("g++"):
        pytest.skip("g++ not found")
    src, exe = tmp_path / "slots.cc", tmp_path / "slots"
    src.write_text('#include <cstdio>\n#include "skv_exchange.cuh"\nint main() {\n'
                   f'  for (int h = 0; h < 2; ++h)\n    for (uint32_t g = 0; g < {tiles}; ++g)\n'
                   '      std::printf("%d ", skv::exchange_slot(h, g));\n}\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(src), "-o", str(exe)], check=True)
    flat = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    return [flat[:tiles], flat[tiles:]]


def _wrong_reads(slots, tiles):
    """Every order in which two threads can run write / barrier / read per tile;
    the set of tiles at which one of them reads anything but its partner's value."""
    wrong, seen, todo = set(), set(), [((0, 0), (None, None))]
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        at, held = state
        if all(x < 3 * tiles and x % 3 == 1 for x in at):  # both wait
            assert at[0] == at[1]
            todo.append(((at[0] + 1, at[1] + 1), held))
            continue
        for t in range(2):
            if at[t] >= 3 * tiles or at[t] % 3 == 1:
                continue
            g, now = at[t] // 3, list(held)
            if at[t] % 3 == 0:
                now[slots[t][g]] = (t, g)
            elif held[slots[1 - t][g]] != (1 - t, g):
                wrong.add(g)
            todo.append(((at[0] + (t == 0), at[1] + (t == 1)), tuple(now)))
    return wrong


def test_row_exchange_reads_the_partners_value_in_every_order(tmp_path):
    tiles = 5
    slots = _slots(tmp_path, tiles)
    assert all({slots[0][g], slots[1][g]} == {0, 1} for g in range(tiles))
    assert _wrong_reads(slots, tiles) == set()
    # (the model does see a value that is overwritten too early: slots that stay)
    assert _wrong_reads([[0] * tiles, [1] * tiles], tiles)


def test_row_exchange_is_the_kernels():
    """Every access to the exchanged values goes through exchange_slot (or a slot made with it)."""
    text = (CSRC / "skv_tree.cu").read_text()
    assert text.count("s.share[") == 5
    assert text.count("s.share[exchange_slot(") == 3 and "s.share[first][row] + s.share[first ^ 1][row]" in text


# ---------------------------------------------------------------- tensor maps in global memory


def test_maps_in_global_memory_are_acquired_before_their_first_load():
    """The loader takes a cell's map pair from global memory in one place, and
    acquires both there, before the segment's loop of loads."""
    text = (CSRC / "skv_tree.cu").read_text()
    kernel = text[text.index("k_tree_attention("):text.index("k_tree_combine(")]
    take = kernel.index("a.cell_maps + ")
    assert kernel.count("a.cell_maps + ") == 1
    loop = kernel.index("p < 2 * w.count", take)
    assert kernel[take:loop].count("tma_acquire_map(one, cell") == 2
    tensor = (CSRC / "skv_tensor.cuh").read_text()
    assert "fence.proxy.tensormap::generic.acquire.sys" in tensor


# ---------------------------------------------------------------- the engine's device


def test_run_tree_selects_the_engines_device_before_it_touches_the_stream():
    """(The null stream and an event record belong to the device that is current.)"""
    text = (CSRC / "skv_engine.cu").read_text()
    body = text[text.index("int skv_run_tree("):]
    body = body[:body.index("\n}\n")]
    scope = body.index("DeviceScope scope(e->desc.device)")
    assert all(body.index(x) > scope for x in ("tree_attention(", "cudaStreamIsCapturing(", "cudaEventRecord("))


# ---------------------------------------------------------------- rotary frequencies


@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 6.5), ("ntk", 4.0)])
@pytest.mark.parametrize("r,theta", [(64, 1e4), (128, 5e5), (256, 1e4), (2, 3.7)])
def test_rotary_fractions_are_right_to_their_last_place(r, theta, scaling, factor):
    """The 64-bit fractions of a turn per position, against 60 digits: the
    rounding to 2^-64 is all that they may be off by (half a unit)."""
    if scaling == "ntk" and r == 2:
        pytest.skip("one pair alone has no slowest pair to divide")
    buf, _, _ = operators._rotary_table(r, theta, scaling, factor, None, 32.0, 1.0, None)
    got = struct.unpack(f"{r // 2}Q", buf.raw[:4 * r])
    want = R.exact_turns(r, [1], theta, factor, scaling)[0]
    for i, (a, b) in enumerate(zip(got, want)):
        off = abs(a - b * 2 ** 64)
        assert min(off, 2 ** 64 - off) <= 0.5000001, (i, float(off))


def test_rotary_table_goes_by_the_values_of_its_settings():
    """A setting that is a tensor may change in place between two calls."""
    theta, factor = torch.tensor(1e4), torch.tensor(2.0)

    def fractions(*a):
        return operators._rotary_table(64, *a, 8192, 32.0, 1.0, None)[0].raw

    first = fractions(theta, "linear", factor)
    assert first == fractions(1e4, "linear", 2)
    theta.fill_(5e5)
    factor.fill_(4.0)
    assert fractions(theta, "linear", factor) == fractions(5e5, "linear", 4.0) != first
    context = torch.tensor(4096)
    first = operators._rotary_table(64, 1e4, "yarn", 4.0, context, 32.0, 1.0, None)[0].raw
    context.fill_(8192)
    assert operators._rotary_table(64, 1e4, "yarn", 4.0, context, 32.0, 1.0, None)[0].raw != first


# ---------------------------------------------------------------- derivatives


def test_a_wanted_derivative_is_seen_in_either_mode():
    import torch.autograd.forward_ad as fwd

    x, g = torch.ones(3), torch.ones(3, requires_grad=True)
    assert operators._recorded(x, g) and not operators._recorded(x)
    with torch.no_grad():
        assert not operators._recorded(x, g)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones(3))
        assert operators._recorded(x, d) and operators._recorded(d) and not operators._recorded(x)
        with torch.no_grad():  # (no_grad is about the backward pass alone)
            assert operators._recorded(x, d) and not operators._recorded(g)


# ---------------------------------------------------------------- outputs that share places


def _places(t):
    at = torch.zeros(t.shape, dtype=torch.int64)
    for i, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).reshape([-1 if j == i else 1 for j in range(t.ndim)])
    return (at + t.storage_offset()).flatten().tolist()


def test_shared_places_are_found_exactly():
    """Against the sets of places, over views of one buffer that nest, interleave, overlap and fold."""
    rng = random.Random(1)
    buffer = torch.zeros(4000)
    met = folded = 0
    for _ in range(1500):
        views = []
        for _ in range(2):
            shape = [rng.choice([1, 2, 3, 5]) for _ in range(3)] + [rng.choice([1, 2, 4])]
            stride = [rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 20, 24, 40, 120]) for _ in range(3)] + [1]
            views.append(torch.as_strided(buffer, shape, stride, rng.randrange(0, 60)))
        a, b = (_places(x) for x in views)
        assert operators._meet(*views) == bool(set(a) & set(b)), views
        for x, p in zip(views, (a, b)):
            assert operators._folded(x) == (len(set(p)) < len(p)), (x.shape, x.stride())
            folded += len(set(p)) < len(p)
        met += bool(set(a) & set(b))
    assert met > 100 and folded > 100


def test_query_and_key_parts_of_one_projection_do_not_meet():
    b, n, hq, hkv, d = 2, 9, 4, 2, 64
    blocks = torch.zeros(b, n, hq + 2 * hkv, d)
    q, k = blocks[:, :, :hq], blocks[:, :, hq:hq + hkv].transpose(1, 2)
    assert not operators._meet(q, k) and operators._meet(q, blocks[:, :, hq - 1:hq + 1].transpose(1, 2))
    by_head = torch.zeros(b, n, hq, 3, d)  # each head's q, k and v side by side
    q, k = by_head[:, :, :, 0], by_head[:, :, :, 1].transpose(1, 2)
    assert not operators._meet(q, k) and operators._meet(q, q.transpose(1, 2))
    assert not operators._folded(q) and not operators._folded(k)
    assert operators._folded(torch.zeros(200).unfold(0, 64, 8)[None, :, None])


# ---------------------------------------------------------------- reports of waits that gave up


def test_reports_of_waits_that_gave_up_reach_their_reader_once():
    """A tree of an engine writes the engine's word, which skv_sync reads on every way out and clears; the
    device's word is cleared when it is read.  (No wait is made to give up here: what is checked is who reads.)"""
    engine = (CSRC / "skv_engine.cu").read_text()
    assert re.search(r"tree_attention\(&d, e->record_maps, .*e->tree_status, st\)", engine)
    sync = engine[engine.index("int skv_sync("):]
    sync = sync[:sync.index("\n}\n")]
    assert sync.index("sync_trees(e)") < sync.index("e->ran") and sync.count("tree_error(e)") == 2
    error = engine[engine.index("int tree_error("):]
    assert "cudaMemset(e->tree_status" in error[:error.index("\n}\n")]
    tree = (CSRC / "skv_tree.cu").read_text()
    assert "cudaMemset(word" in tree[tree.index("int skv_operator_status("):]


# ---------------------------------------------------------------- limits


@pytest.mark.parametrize("counts,word", [(dict(hq=5), "4096"), (dict(hq=8192), "4096"), (dict(b=1 << 30), "2^31"),
                                         (dict(b=1 << 62), "2^31")])
def test_tree_attention_names_the_limit_that_a_call_passes(counts, word):
    """(b = 2^62 times 8 rows is 2^65: the product itself would wrap around to 0.)"""
    from tests.test_operators import _refused, _tree

    rc, message = _refused("skv_tree_attention", _tree(**counts))
    assert rc == -1 and word in message


@pytest.mark.parametrize("counts", [dict(sink=1 << 62, local=1 << 62), dict(sink=(1 << 63) - 1, local=1),
                                    dict(b=1 << 24, hkv=1 << 40), dict(b=2, hkv=1 << 63 - 1)])
def test_evict_refuses_counts_whose_sums_and_products_wrap_around(counts):
    from tests.test_operators import _evict, _refused

    rc, message = _refused("skv_evict", _evict(**counts))
    assert rc == -1 and message
