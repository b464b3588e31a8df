"""Operators around a decode step: rotary positions, attention of a tree of
drafted tokens over a cache, attention weights accumulated per cached key, and
eviction from the cache by those weights.

The reference takes rotated K and Q, decodes one token per step and never
drops one; these are what a decode loop that drafts several tokens ahead, or
that has to stay inside a memory budget, needs next to it::

    q, k = rotary(q, k, positions)                                     # drafted tokens
    y, lse = tree_attention(q, k_cache, v_cache, lengths, k, v, parents)
    weights = accumulate_weights(q, k_cache, lengths, lse, weights, rows=accepted)
    k_cache, v_cache, weights, ids, lengths = evict(k_cache, v_cache, weights, lengths, keep=budget)

Every operator is a function of CUDA tensors of one device and returns new
ones (``rotary`` and ``accumulate_weights`` also write into given ones).  The
work is enqueued on the current PyTorch stream of that device; nothing waits,
and every call may be captured into a CUDA graph.  Tensors may have any
strides as long as the innermost dimension is contiguous; for the attention
operators rows have to start on 16-byte boundaries (and there are at most 4096
query heads), and the pairs of an interleaved rotation on two elements.
ValueError otherwise.
They are for inference: a tensor that requires a gradient is refused while
gradients are recorded, and so is one with a forward-mode tangent.
"""

from __future__ import annotations

import ctypes
import decimal
import functools
import math
import struct

import torch
import torch.autograd.forward_ad as _forward

from seoulkv_b200 import _native
from seoulkv_b200.api import _current_stream

# Tells autograd that a tensor was written to (one that backward has saved is then an error there).
_changed = torch.autograd.graph.increment_version

TREE_MAX_NODES = 64
ROTARY_MAX_DIM = 512
_BF16, _F32, _I32, _FP8 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, torch.float8_e4m3fn: 3}
_NAMES = {torch.bfloat16: "BF16", torch.float16: "FP16", torch.float32: "FP32", torch.float8_e4m3fn: "FP8 e4m3",
          torch.int32: "int32", torch.int64: "int64", torch.bool: "bool"}

# Arguments are checked twice over: one expression that holds for every good
# call (these functions run once per decode step), and, where it does not
# hold, _check() on each argument, which says what is wrong.


def _check(name: str, t, shape, dtypes, device: int | None = None) -> None:
    """A CUDA tensor of one of the dtypes; ``shape`` entries of None are free."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError(f"{name}: expected a {' or '.join(_NAMES.get(x, str(x)) for x in dtypes)} tensor")
    got = t.shape
    if len(got) != len(shape) or any(w is not None and w != g for w, g in zip(shape, got)):
        raise ValueError(f"{name}: expected shape [{','.join('*' if w is None else str(w) for w in shape)}], "
                         f"got {list(got)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: the operators have no backward pass (detach it, or use no_grad)")
    if _tangent(t):
        raise ValueError(f"{name} carries a forward-mode tangent: the operators have no derivatives (detach it)")


def _tangent(t) -> bool:
    return _forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None


def _recorded(*tensors) -> bool:
    """Whether a derivative of one of them is wanted, in either mode."""
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            return True
    return _forward._current_level >= 0 and any(_tangent(t) for t in tensors)


def _span(t: torch.Tensor) -> tuple[int, int]:
    """First and last byte address (exclusive) that a tensor reaches."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def _reaches(total: int, terms: list) -> bool:
    """Whether sum(s * t) == total for some integers lo <= t <= hi of each term (s, lo, hi), s > 0.
    Largest s first: in a layout whose dimensions nest, one or two t are left for each."""
    if not terms:
        return total == 0
    (s, lo, hi), rest = terms[0], terms[1:]
    least, most = sum(x * a for x, a, _ in rest), sum(x * b for x, _, b in rest)
    first, last = max(lo, -((most - total) // s)), min(hi, (total - least) // s)
    return any(_reaches(total - s * t, rest) for t in range(first, last + 1))


@functools.lru_cache(maxsize=256)
def _layouts_meet(off: int, a: tuple, of_a: tuple, b: tuple, of_b: tuple) -> bool:
    """Whether layouts (strides, sizes) share a place, the second one ``off`` elements behind the first."""
    terms = {}
    for s, n in zip(a, of_a):
        lo, hi = terms.get(s, (0, 0))
        terms[s] = lo, hi + n - 1
    for s, n in zip(b, of_b):
        lo, hi = terms.get(s, (0, 0))
        terms[s] = lo - n + 1, hi
    return _reaches(off, sorted(((s, *x) for s, x in terms.items() if s), reverse=True))


@functools.lru_cache(maxsize=256)
def _layout_folds(strides: tuple, sizes: tuple) -> bool:
    """Whether two elements of a layout share one place."""
    dims = sorted(((s, n - 1) for s, n in zip(strides, sizes) if n > 1), reverse=True)
    if dims and dims[-1][0] == 0:
        return True
    terms = [(s, -n, n) for s, n in dims]
    return any(_reaches(-s * i, terms[at + 1:]) for at, (s, n) in enumerate(dims)
               for i in range(1, min(n, sum(x * m for x, m in dims[at + 1:]) // s) + 1))


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one element type share a place."""
    if not _overlap(a, b):
        return False
    off, size = b.data_ptr() - a.data_ptr(), a.element_size()
    return off % size != 0 or _layouts_meet(off // size, a.stride(), a.shape, b.stride(), b.shape)


def _folded(t: torch.Tensor) -> bool:
    """Whether two elements of a tensor share one place."""
    return not t.is_contiguous() and t.numel() > 0 and _layout_folds(t.stride(), t.shape)


def _run(entry, packed: bytes, device: int, what: str) -> None:
    rc = entry(packed, _current_stream(device))
    if rc:
        message = _native.load().skv_last_error().decode(errors="replace")
        if rc == -1:
            raise ValueError(f"{what}: {message}")
        raise _native.NativeError(rc, f"{what}: {message}")


def check_operators(device) -> None:
    """Wait for the device; RuntimeError if a bounded wait of an operator's kernel gave up on it
    since the last check (the outputs of that call are NaN).  One record per device, for all its
    users in the process; ``run_tree`` reports to its instance's ``synchronize()`` instead.  Not
    for the inner loop."""
    from seoulkv_b200.api import _cuda_index

    flags = ctypes.c_uint32()
    _native.check(_native.load().skv_operator_status(_cuda_index(device), ctypes.byref(flags)), "skv_operator_status")
    if flags.value:
        raise RuntimeError(f"an operator's kernel gave up waiting (status {flags.value:#x}); its results are invalid")


# ---------------------------------------------------------------- rotary positions


def _pi(digits: int) -> decimal.Decimal:
    """pi = 16 atan(1/5) - 4 atan(1/239) (Machin), in integers of 10^-(digits + 10)."""
    one = 10 ** (digits + 10)

    def atan_inverse(n):
        term, total, i = one // n, 0, 0
        while term:
            total += (-1) ** i * (term // (2 * i + 1))
            term, i = term // (n * n), i + 1
        return total

    return decimal.Decimal(16 * atan_inverse(5) - 4 * atan_inverse(239)).scaleb(-digits - 10)


def _by_value(table):
    """Caches a table of a few numbers by their values.  An object (a tensor) would be found again after its
    value has changed; nothing is kept of a call that raises, so no object ever enters the cache."""

    @functools.lru_cache(maxsize=64)
    def cached(*settings):
        if not all(x is None or isinstance(x, (int, float, str)) for x in settings):
            raise TypeError
        return table(*settings)

    @functools.wraps(table)
    def call(rotary_dim, theta, scaling, factor, original_context, beta_fast, beta_slow, attention_factor):
        try:
            return cached(rotary_dim, theta, scaling, factor, original_context, beta_fast, beta_slow, attention_factor)
        except TypeError:
            return cached(rotary_dim, float(theta), scaling, float(factor),
                          None if original_context is None else float(original_context), float(beta_fast),
                          float(beta_slow), None if attention_factor is None else float(attention_factor))

    return call


@_by_value
def _rotary_table(rotary_dim, theta, scaling, factor, original_context, beta_fast, beta_slow, attention_factor):
    """(turns per position * 2^64 of each pair as packed uint64, its address, factor on the rotated part)."""
    theta, factor, beta_fast, beta_slow = (float(x) for x in (theta, factor, beta_fast, beta_slow))
    if not theta > 0.0 or not math.isfinite(theta) or theta == 1.0:
        raise ValueError("theta must be positive, finite and not 1")
    if not factor > 0.0 or not math.isfinite(factor):
        raise ValueError("factor must be positive and finite")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError("scaling must be 'none', 'linear', 'ntk' or 'yarn'")
    pairs, r = rotary_dim // 2, float(rotary_dim)
    low = high = 0
    m = 1.0
    if scaling == "yarn":
        if original_context is None or original_context < 1:
            raise ValueError("yarn scaling needs original_context >= 1")
        if not beta_fast > beta_slow > 0.0:
            raise ValueError("yarn scaling needs beta_fast > beta_slow > 0")

        def pair_of(turns):  # the (real) pair that turns so often in the original context
            return r * math.log(original_context / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        m = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    if attention_factor is not None:
        m = float(attention_factor)
    if not math.isfinite(m):
        raise ValueError("attention_factor must be finite")
    # The fractions need 64 places behind the point, which is more than a
    # double has: 60 decimal digits, and as many more as the frequencies may
    # have before the point.
    with decimal.localcontext() as context:
        context.prec = digits = 60 + math.ceil(3 * (abs(math.log10(theta)) + abs(math.log10(factor))))
        base, stretch = decimal.Decimal(theta), decimal.Decimal(factor)
        if scaling == "ntk" and rotary_dim > 2:
            base *= stretch ** (decimal.Decimal(rotary_dim) / (rotary_dim - 2))
        step = base ** (decimal.Decimal(-2) / rotary_dim)
        places, f = 2 ** 64 / (2 * _pi(digits)), decimal.Decimal(1)
        turns = []
        for i in range(pairs):
            x = f
            if scaling == "linear":
                x = f / stretch
            elif scaling == "yarn":
                part = min(1, max(0, (i - low) / max(decimal.Decimal(high - low), decimal.Decimal(1e-3))))
                x = f * (1 - part) + f / stretch * part
            turns.append(int((x * places).to_integral_value()) & (2 ** 64 - 1))
            f *= step
    table = ctypes.create_string_buffer(struct.pack(f"{pairs}Q", *turns))
    return table, ctypes.addressof(table), m


_ROTARY = struct.Struct("6Qd" + 10 * "q" + 18 * "q")


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, *, rotary_dim: int | None = None,
           theta: float = 10000.0, layout: str = "half", scaling: str = "none", factor: float = 1.0,
           original_context: int | None = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
           attention_factor: float | None = None, out=None):
    """Rotary positions on queries [B, N, Hq, D] and keys [B, Hkv, N, D] (or None).

    BF16, FP16 or FP32, both alike, on one device.  ``positions`` int32 or
    int64, [N] or [B, N]; the angle of position p is off by p * 2^-65 turns,
    which is less than its FP32 rounding up to 2^39; negative positions turn
    back (the inverse rotation, and the gradient's, for a factor of 1).  The
    first ``rotary_dim`` (even, at most 512; all of D by default) dimensions
    turn, the others are copied.  ``layout``: "half" pairs dimension i with
    i + rotary_dim/2, "interleaved" 2i with 2i + 1.

    ``scaling`` for contexts beyond the trained one: "linear" divides every
    frequency by ``factor``; "ntk" raises theta so that the slowest pair is
    divided by it; "yarn" (Peng et al., 2023) divides the pairs that turn less
    than ``beta_slow`` times in ``original_context`` tokens, keeps those above
    ``beta_fast``, and multiplies the rotated part by 0.1 ln(factor) + 1
    (``attention_factor`` sets another multiplier).  Between the two corner
    pairs, rounded outwards to whole ones, the share of the division grows
    linearly with the pair's index, the form in use (the paper's text has it
    linear in the number of turns).  With "none" the factor and the settings of
    "yarn" are not used, except for ``attention_factor``.

    Returns (q, k) in new tensors, or in ``out=(q_out, k_out)``, which may be
    the inputs themselves (q and k may then be parts of one projection that
    share no place; otherwise the outputs must not overlap the inputs).
    """
    if not isinstance(q, torch.Tensor) or q.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError("q: expected a BF16 or FP16 or FP32 tensor")
    dtype, dev = q.dtype, q.get_device()
    if q.ndim != 4 or dev < 0:
        _check("q", q, (None,) * 4, (dtype,))
    b, n, hq, d = q.shape
    hkv = 0
    if k is not None:
        if not (isinstance(k, torch.Tensor) and k.ndim == 4 and k.dtype is dtype and k.get_device() == dev):
            _check("k", k, (b, None, n, d), (dtype,), dev)
        hkv = k.shape[1]
        if k.shape != (b, hkv, n, d):
            _check("k", k, (b, None, n, d), (dtype,), dev)
    if hq < 1 or (k is not None and hkv < 1):
        raise ValueError("q and k need at least one head")
    if not isinstance(positions, torch.Tensor) or positions.ndim not in (1, 2):
        raise ValueError("positions: expected an int32 or int64 tensor [N] or [B,N]")
    if not (positions.dtype in (torch.int64, _I32) and positions.get_device() == dev
            and positions.shape == ((n,) if positions.ndim == 1 else (b, n))):
        _check("positions", positions, (n,) if positions.ndim == 1 else (b, n), (_I32, torch.int64), dev)
    if _recorded(q, q if k is None else k):
        _check("q", q, (None,) * 4, (dtype,))
        _check("k", k, (None,) * 4, (dtype,))
    r = d if rotary_dim is None else rotary_dim
    if type(r) is not int or r < 2 or r % 2 or r > d or r > ROTARY_MAX_DIM:
        raise ValueError(f"rotary_dim must be an even integer in [2, min(D, {ROTARY_MAX_DIM})]")
    if layout not in ("half", "interleaved"):
        raise ValueError("layout must be 'half' or 'interleaved'")
    _, phase, m = _rotary_table(r, theta, scaling, factor, original_context, beta_fast, beta_slow, attention_factor)
    if out is None:
        qo = q.new_empty(b, n, hq, d)
        ko = None if k is None else k.new_empty(b, hkv, n, d)
    else:
        qo, ko = out
        _check_rotary_out(q, k, qo, ko, dev)
    if not b or not n:
        return qo, ko
    kk, kko = (q, qo) if k is None else (k, ko)
    pos = positions.stride()
    packed = _ROTARY.pack(
        q.data_ptr(), kk.data_ptr(), qo.data_ptr(), kko.data_ptr(), positions.data_ptr(), phase, m,
        dev, _DTYPE[dtype], layout == "interleaved", positions.dtype is torch.int64, b, n, hq, hkv, d, r,
        *q.stride(), *kk.stride(), *qo.stride(), *kko.stride(), *((0, *pos) if len(pos) == 1 else pos))
    _run(_native.load().skv_rotary, packed, dev, "rotary")
    if out is not None:
        _changed(qo)
        if ko is not None:
            _changed(ko)
    return qo, ko


def _check_rotary_out(q, k, qo, ko, dev: int) -> None:
    _check("out[0]", qo, tuple(q.shape), (q.dtype,), dev)
    pairs = [("out[0]", qo, q)]
    if k is None:
        if ko is not None:
            raise ValueError("out[1]: there is no k")
    else:
        _check("out[1]", ko, tuple(k.shape), (q.dtype,), dev)
        pairs.append(("out[1]", ko, k))
    for name, y, x in pairs:
        if _folded(y):
            raise ValueError(f"{name}: two elements share one place")
        same = y.data_ptr() == x.data_ptr() and y.stride() == x.stride()
        if not same and _overlap(y, x):
            raise ValueError(f"{name} overlaps its input without being it")
    if k is not None and qo.data_ptr() == q.data_ptr() and ko.data_ptr() == k.data_ptr():
        # (in place, q and k may be interleaved parts of one projection)
        if _meet(qo, ko):
            raise ValueError("out[1] overlaps out[0]: q and k share places")
    elif k is not None:
        for name, y, x in (("out[0]", qo, k), ("out[1]", ko, q), ("out[1]", ko, qo)):
            if _overlap(y, x):
                raise ValueError(f"{name} overlaps another tensor of the call")


# ---------------------------------------------------------------- attention of drafted trees


_TREE = struct.Struct("10Qd" + 9 * "q" + 23 * "q")


def _check_cache(k_cache, v_cache, lengths) -> None:
    """Says what is wrong with a cache."""
    _check("k_cache", k_cache, (None,) * 4, (_BF16, _FP8))
    b, h, t, d = k_cache.shape
    dev = k_cache.get_device()
    if d not in (64, 128, 256):
        raise ValueError("head size must be 64, 128 or 256")
    if t < 1 or h < 1:
        raise ValueError("k_cache: expected at least one head and one token of room")
    if v_cache is not None:
        _check("v_cache", v_cache, (b, h, t, d), (k_cache.dtype,), dev)
    _check("lengths", lengths, (b,), (_I32,), dev)


def _scale(scale) -> float:
    s = float(scale)
    if not (s > 0.0 and math.isfinite(s)):
        raise ValueError("scale must be positive and finite")
    return s


_ROOT = {64: 0.125, 128: 128 ** -0.5, 256: 0.0625}


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                   k: torch.Tensor, v: torch.Tensor, parents: torch.Tensor, *, scale: float | None = None):
    """Exact attention of N drafted tokens per sequence over a cache and their own ancestors.

    ``q`` BF16 [B, N, Hq, D] with N <= 64 and D 64, 128 or 256; ``k_cache``
    and ``v_cache`` BF16 or FP8 e4m3 [B, Hkv, T, D] with Hq a multiple of Hkv;
    ``lengths`` int32 [B], the valid tokens (clamped to [0, T]; what lies
    behind them is not read into any result); ``k`` and ``v`` BF16
    [B, Hkv, N, D], the drafted tokens' own; ``parents`` int32 [B, N]: the
    node before node i (below i), -1 for a node that follows the cache.  Any
    other value marks an unused node (padding of a smaller tree): it and the
    nodes below it get zeros and an lse of -inf, and nothing sees them.

    The weights are rounded to BF16 for the product with V (2^-8 of each at
    most; their sum is not).  Over an FP8 cache the scores take the queries as
    sums of two FP8 rows: an element is off by at most 2^-17 of its row's
    largest one, and a query with an infinity gives NaN.

    Returns the attention output, BF16 [B, N, Hq, D], and the natural
    log-sum-exp of each row's scaled scores, FP32 [B, N, Hq].  ``scale``
    defaults to D**-0.5.  N = 1 with parent -1 is exact decode of one token.
    """
    if not (isinstance(k_cache, torch.Tensor) and k_cache.ndim == 4 and isinstance(q, torch.Tensor) and q.ndim == 4):
        _check("k_cache", k_cache, (None,) * 4, (_BF16, _FP8))
        _check("q", q, (None,) * 4, (_BF16,))
    b, hkv, t, d = shape = k_cache.shape
    _, n, hq, _ = q.shape
    dev, kind = k_cache.get_device(), k_cache.dtype
    node = (b, hkv, n, d)
    try:
        good = (dev >= 0 and (kind is _BF16 or kind is _FP8) and v_cache.dtype is kind and v_cache.shape == shape
                and q.dtype is _BF16 and q.shape == (b, n, hq, d) and k.dtype is _BF16 and k.shape == node
                and v.dtype is _BF16 and v.shape == node and lengths.dtype is _I32 and lengths.shape == (b,)
                and parents.dtype is _I32 and parents.shape == (b, n) and v_cache.get_device() == dev
                and q.get_device() == dev and k.get_device() == dev and v.get_device() == dev
                and lengths.get_device() == dev and parents.get_device() == dev
                and d in _ROOT and t and hkv and 0 < n <= TREE_MAX_NODES and hq and not hq % hkv
                and not _recorded(q, k_cache, v_cache, k, v))
    except AttributeError:  # not a tensor
        good = False
    if not good:
        _check_cache(k_cache, v_cache, lengths)
        _check("q", q, (b, None, None, d), (_BF16,), dev)
        if not 1 <= n <= TREE_MAX_NODES:
            raise ValueError(f"the tree must have 1 to {TREE_MAX_NODES} nodes")
        if hq < 1 or hq % hkv:
            raise ValueError("query heads must be a multiple of the KV heads")
        _check("k", k, node, (_BF16,), dev)
        _check("v", v, node, (_BF16,), dev)
        _check("parents", parents, (b, n), (_I32,), dev)
    out = q.new_empty(b, n, hq, d)
    lse = q.new_empty(b, n, hq, dtype=_F32)
    if not b:
        return out, lse
    size = _tree_workspace(dev, b, n, hq, hkv, d, t)
    work = q.new_empty(size, dtype=torch.uint8) if size else None
    packed = _TREE.pack(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lengths.data_ptr(), k.data_ptr(), v.data_ptr(),
        parents.data_ptr(), out.data_ptr(), lse.data_ptr(), work.data_ptr() if size else 0,
        _ROOT[d] if scale is None else _scale(scale), dev, _DTYPE[kind], size, b, n, hq, hkv, d, t,
        *q.stride(), *k_cache.stride(), *v_cache.stride(), *k.stride(), *v.stride(), *parents.stride(), *lengths.stride())
    _run(_native.load().skv_tree_attention, packed, dev, "tree_attention")
    return out, lse


def run_tree(engine, lead: tuple, q, k, v, parents, device: int):
    """Tree attention over an engine's FP8 records (``SeoulKV4.run_tree`` and
    ``SeoulKV4Batch.run_tree``): K and V [*lead, 4, N, 256], parents [*lead, N]."""
    slots = engine.n_slots
    if not isinstance(q, torch.Tensor) or q.ndim != 4 or q.dtype is not _BF16 or q.shape[0] != slots \
            or q.shape[2:] != (16, 256) or not 1 <= q.shape[1] <= TREE_MAX_NODES:
        raise ValueError(f"expected BF16 Q [{slots},N,16,256] with 1 <= N <= {TREE_MAX_NODES}")
    n = q.shape[1]
    dims = "".join(f"{x}," for x in lead)
    for name, t in (("K", k), ("V", v)):
        if not isinstance(t, torch.Tensor) or t.dtype is not _BF16 or tuple(t.shape) != (*lead, 4, n, 256):
            raise ValueError(f"expected BF16 drafted {name} [{dims}4,{n},256]")
    if not isinstance(parents, torch.Tensor) or parents.dtype is not _I32 or tuple(parents.shape) != (*lead, n):
        raise ValueError(f"expected int32 parents [{dims}{n}]")
    if _recorded(q, k, v):
        raise ValueError("run_tree has no derivatives: an input requires a gradient or carries a tangent "
                         "(detach it, or use no_grad)")
    q, k, v, parents = (t if t.get_device() == device else t.to(f"cuda:{device}") for t in (q, k, v, parents))
    if not lead:
        k, v, parents = k[None], v[None], parents[None]
    out = q.new_empty(slots, n, 16, 256)
    lse = q.new_empty(slots, n, 16, dtype=_F32)
    size = _tree_workspace(device, slots, n, 16, 4, 256, engine.max_context)
    work = q.new_empty(size, dtype=torch.uint8) if size else None
    packed = _TREE.pack(
        q.data_ptr(), 0, 0, 0, k.data_ptr(), v.data_ptr(), parents.data_ptr(), out.data_ptr(), lse.data_ptr(),
        work.data_ptr() if size else 0, 0.0625, device, _DTYPE[_FP8], size, slots, n, 16, 4, 256, engine.max_context,
        *q.stride(), *(8 * (0,)), *k.stride(), *v.stride(), *parents.stride(), 0)
    rc = engine.lib.skv_run_tree(engine.handle, packed, _current_stream(device))
    if rc == -1:
        raise ValueError(f"run_tree: {engine.lib.skv_last_error().decode(errors='replace')}")
    _native.check(rc, "skv_run_tree")
    return out, lse


@functools.lru_cache(maxsize=1024)
def _tree_workspace(device: int, b: int, n: int, hq: int, hkv: int, d: int, t: int) -> int:
    """Bytes of scratch that one call needs (a function of the sizes; 0 for short caches)."""
    size = ctypes.c_int64()
    packed = _TREE.pack(*(10 * (0,)), 1.0, device, 0, 0, b, n, hq, hkv, d, t, *(23 * (0,)))
    _native.check(_native.load().skv_tree_workspace(packed, ctypes.byref(size)), "skv_tree_workspace")
    return size.value


# ---------------------------------------------------------------- accumulated weights


_WEIGHTS = struct.Struct("7Qd" + 8 * "q" + 20 * "q")


def accumulate_weights(q: torch.Tensor, k_cache: torch.Tensor, lengths: torch.Tensor, lse: torch.Tensor,
                       weights: torch.Tensor, *, rows: torch.Tensor | None = None, scale: float | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Add the attention that rows of queries pay to each cached key to the keys' weights.

    weights[b, h, t] + sum over nodes and the query heads of KV head h of
    exp(scale q.k_t - lse) for t < lengths[b]; later tokens keep their weight.
    ``q`` BF16 [B, N, Hq, D] and ``lse`` FP32 [B, N, Hq] as given to and
    returned by ``tree_attention`` (N is not limited here: a window of prompt
    tokens with their log-sum-exp works as well), ``k_cache`` and ``lengths``
    as there, ``weights`` FP32 [B, Hkv, T].  ``rows`` (bool [B, N]) names the
    nodes that count, the accepted ones; a row whose lse is -inf never counts.

    Returns a new tensor, or ``out``, which may be ``weights`` itself
    (otherwise it must not overlap it).
    """
    if not (isinstance(k_cache, torch.Tensor) and k_cache.ndim == 4 and isinstance(q, torch.Tensor) and q.ndim == 4):
        _check("k_cache", k_cache, (None,) * 4, (_BF16, _FP8))
        _check("q", q, (None,) * 4, (_BF16,))
    b, hkv, t, d = k_cache.shape
    _, n, hq, _ = q.shape
    dev, kind = k_cache.get_device(), k_cache.dtype
    held = (b, hkv, t)
    try:
        good = (dev >= 0 and (kind is _BF16 or kind is _FP8) and q.dtype is _BF16 and q.shape == (b, n, hq, d)
                and lse.dtype is _F32 and lse.shape == (b, n, hq) and weights.dtype is _F32 and weights.shape == held
                and lengths.dtype is _I32 and lengths.shape == (b,) and q.get_device() == dev
                and lse.get_device() == dev and weights.get_device() == dev and lengths.get_device() == dev
                and d in _ROOT and t and hkv and n and hq and not hq % hkv
                and not _recorded(q, k_cache, lse, weights))
    except AttributeError:  # not a tensor
        good = False
    if not good:
        _check_cache(k_cache, None, lengths)
        _check("q", q, (b, None, None, d), (_BF16,), dev)
        if n < 1 or hq < 1 or hq % hkv:
            raise ValueError("q: expected at least one node, and query heads a multiple of the KV heads")
        _check("lse", lse, (b, n, hq), (_F32,), dev)
        _check("weights", weights, held, (_F32,), dev)
    if rows is not None and not (isinstance(rows, torch.Tensor) and rows.dtype is torch.bool and rows.shape == (b, n)
                                 and rows.get_device() == dev):
        _check("rows", rows, (b, n), (torch.bool,), dev)
    given = out is not None
    if not given:
        out = weights.new_empty(b, hkv, t)
    else:
        _check("out", out, held, (_F32,), dev)
        if _folded(out):
            raise ValueError("out: two elements share one place")
        if not (out.data_ptr() == weights.data_ptr() and out.stride() == weights.stride()) and _overlap(out, weights):
            raise ValueError("out overlaps weights without being it")
    if not b:
        return out
    packed = _WEIGHTS.pack(
        q.data_ptr(), k_cache.data_ptr(), lengths.data_ptr(), lse.data_ptr(), 0 if rows is None else rows.data_ptr(),
        weights.data_ptr(), out.data_ptr(), _ROOT[d] if scale is None else _scale(scale), dev, _DTYPE[kind], b, n, hq,
        hkv, d, t, *q.stride(), *k_cache.stride(), *lse.stride(), *((0, 0) if rows is None else rows.stride()),
        *weights.stride(), *out.stride(), *lengths.stride())
    _run(_native.load().skv_accumulate_weights, packed, dev, "accumulate_weights")
    if given:
        _changed(out)
    return out


# ---------------------------------------------------------------- eviction


_EVICT = struct.Struct("9Q" + 9 * "q" + 12 * "q")
_EVICTED = frozenset(_DTYPE)


def evict(k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor, lengths: torch.Tensor, *, keep: int,
          sink: int = 128, local: int = 256):
    """Shrink caches to ``keep`` tokens per head by accumulated attention weight.

    ``k_cache`` and ``v_cache`` [B, Hkv, T, D] (BF16, FP16, FP32 or FP8),
    ``weights`` FP32 [B, Hkv, T], ``lengths`` int32 [B] (clamped to [0, T]).
    Per head the first ``sink`` and the last ``local`` tokens stay and, of the
    others, the keep - sink - local heaviest (equal weights: the lowest index;
    NaN counts below every number); a cache of at most ``keep`` tokens stays
    whole.  Kept tokens keep their order.

    Returns new tensors (k, v, weights, ids, lengths): K and V
    [B, Hkv, keep, D], FP32 weights and int32 ids (indices into the old cache)
    [B, Hkv, keep], lengths int32 [B]; past the kept tokens K, V and weights
    are zero and ids -1.
    """
    if not (isinstance(k_cache, torch.Tensor) and k_cache.ndim == 4):
        _check("k_cache", k_cache, (None,) * 4, tuple(_DTYPE))
    b, h, t, d = shape = k_cache.shape
    dev, kind = k_cache.get_device(), k_cache.dtype
    try:
        good = (dev >= 0 and kind in _EVICTED and v_cache.dtype is kind and v_cache.shape == shape
                and weights.dtype is _F32 and weights.shape == (b, h, t) and lengths.dtype is _I32
                and lengths.shape == (b,) and v_cache.get_device() == dev and weights.get_device() == dev
                and lengths.get_device() == dev and t and h and d and not _recorded(k_cache, v_cache, weights))
    except AttributeError:  # not a tensor
        good = False
    if not good:
        _check("k_cache", k_cache, (None,) * 4, tuple(_DTYPE))
        if h < 1 or t < 1 or d < 1:
            raise ValueError("k_cache: expected at least one head, token and dimension")
        _check("v_cache", v_cache, (b, h, t, d), (kind,), dev)
        _check("weights", weights, (b, h, t), (_F32,), dev)
        _check("lengths", lengths, (b,), (_I32,), dev)
    if type(keep) is not int or type(sink) is not int or type(local) is not int or not 1 <= keep <= t \
            or sink < 0 or local < 0 or sink + local > keep:
        raise ValueError(f"keep must be in [1, {t}] and hold the sink and local tokens")
    ko = k_cache.new_empty(b, h, keep, d)
    vo = torch.empty_like(ko)
    wo = weights.new_empty(b, h, keep)
    ids = torch.empty_like(wo, dtype=_I32)
    left = torch.empty_like(lengths)
    if not b:
        return ko, vo, wo, ids, left
    packed = _EVICT.pack(
        k_cache.data_ptr(), v_cache.data_ptr(), weights.data_ptr(), lengths.data_ptr(), ko.data_ptr(), vo.data_ptr(),
        wo.data_ptr(), ids.data_ptr(), left.data_ptr(), dev, b, h, t, d, k_cache.element_size(), keep, sink, local,
        *k_cache.stride(), *v_cache.stride(), *weights.stride(), *lengths.stride())
    _run(_native.load().skv_evict, packed, dev, "evict")
    return ko, vo, wo, ids, left
