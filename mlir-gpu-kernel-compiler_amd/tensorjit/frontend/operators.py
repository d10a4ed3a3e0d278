"""Operators of a decoder's serving step, for use inside traced functions.

    @tj.jit
    def step(x, wq, wk, wv, k_cache, v_cache, pages, starts, counts, positions):
        ...
        q, k = tj.rotary(q, positions), tj.rotary(k, positions)
        k_cache = tj.paged_write(k_cache, k, pages, starts, counts)
        v_cache = tj.paged_write(v_cache, v, pages, starts, counts)
        return tj.paged_attention(q, k_cache, v_cache, pages, starts, counts), k_cache, v_cache

A paged cache is one tensor ``[pages, page size, heads, dim]`` for every sequence; row ``b`` of
``pages`` (i32 ``[batch, pages per sequence]``) lists the pages of sequence ``b`` in order, so its
token ``t`` lies in page ``pages[b, t // page size]`` at ``t % page size``.  A call brings up to
``S`` new tokens per sequence, at positions ``starts[b] .. starts[b] + counts[b] - 1``; the
program is compiled for ``S``, and lengths are data.
"""
from __future__ import annotations

import math
import struct

from ..ir import Node
from .tracer import Tensor, _active

LARGEST = 1e30          # number parameters become fp32 constants
SMALLEST_FP32 = 2.0**-149


def _node(op: str, name: str, t) -> Node:
    if not isinstance(t, Tensor):
        raise TypeError(f"{op}: {name} must be a tensor of the traced function, got {type(t).__name__}")
    return t.node


def _zero(v) -> bool:
    """By its bits: where a library has the process flush denormals, they compare equal to 0."""
    return struct.pack("<d", abs(v)) == bytes(8)


def _number(op: str, name: str, v, low: float = -math.inf, above: float = -math.inf, high: float = math.inf,
            least: float = 0.0) -> float:
    """``v``, checked: from ``low`` (or past ``above``) to ``high``, and 0 or of at least the size ``least``."""
    if isinstance(v, bool) or not isinstance(v, (int, float)):
        raise TypeError(f"{op}: {name} must be a number, got {type(v).__name__}")
    if not (math.isfinite(v) and low <= v <= high and v > above and (abs(v) >= least or _zero(v))):
        raise ValueError(f"{op}: {name} = {v} is out of range")
    return float(v)


def _whole(op: str, name: str, v, low: int) -> int:
    if isinstance(v, bool) or not isinstance(v, int):
        raise TypeError(f"{op}: {name} must be an integer, got {type(v).__name__}")
    if not low <= v < 2**31:
        raise ValueError(f"{op}: {name} = {v} is out of range")
    return v


def rotary(x: Tensor, positions: Tensor, *, dims: int | None = None, interleaved: bool = False, base: float = 10000.0,
           factor: float = 1.0, original: int | None = None, ramp: tuple[float, float] = (1.0, 32.0),
           magnitude: float = 1.0, inverse: bool = False, heads_first: bool = False) -> Tensor:
    """Rotary positions: pair ``i`` of each head's first ``dims`` values (default all) is turned by
    ``positions * f_i``, ``f_i = base ** (-2 i / dims)``; the other values pass unchanged.

    ``x`` is ``[..., tokens, heads, dim]``, or ``[..., heads, tokens, dim]`` with ``heads_first``;
    ``positions`` (i32) broadcasts to its tokens ``[..., tokens]``.  Pairs are ``(i, i + dims/2)``,
    or ``(2 i, 2 i + 1)`` with ``interleaved``.

    Long contexts: ``factor`` divides every frequency.  With ``original``, the context length the
    model was trained for, it does so by parts: a pair that turns more than ``ramp[1]`` times over
    that length keeps its frequency, one that turns less than ``ramp[0]`` times has it divided, and
    those between blend linearly.  ``magnitude`` scales the turned values
    (0, or from 1e-30 to 1e30 in size).

    ``inverse`` turns back: with the same arguments it is the gradient, ``dx = rotary(dy, ...,
    inverse=True)``.  Angles are computed in 64 bits, so far positions keep their fraction of a
    turn; the turn itself is computed in fp32 and rounded once."""
    op = "rotary"
    xn, pn = _node(op, "x", x), _node(op, "positions", positions)
    dims = x.shape[-1] if dims is None and x.shape else dims
    dims = _whole(op, "dims", dims, 2)
    if dims % 2:
        raise ValueError(f"rotary: dims = {dims} is odd")
    if not (isinstance(ramp, (tuple, list)) and len(ramp) == 2):
        raise TypeError("rotary: ramp must be a pair of numbers")
    ramp = tuple(_number(op, "ramp", r) for r in ramp)
    if ramp[0] >= ramp[1]:
        raise ValueError(f"rotary: ramp {ramp} must rise")
    return Tensor(_active().create(
        op, [xn, pn], dims=dims, interleaved=bool(interleaved), base=_number(op, "base", base, low=1 / LARGEST, high=LARGEST),
        factor=_number(op, "factor", factor, low=1 / LARGEST, high=LARGEST), original=None if original is None else _whole(op, "original", original, 1),
        ramp=ramp, magnitude=_number(op, "magnitude", magnitude, low=-LARGEST, high=LARGEST, least=1 / LARGEST),
        inverse=bool(inverse), heads_first=bool(heads_first)))


def paged_write(cache: Tensor, x: Tensor, pages: Tensor, starts: Tensor, counts: Tensor | None = None) -> Tensor:
    """Write the new tokens' rows ``x`` (``[batch, S, heads, dim]``) into ``cache`` and return it.

    Token ``i < counts[b]`` (default: all ``S``) of sequence ``b`` goes to position
    ``starts[b] + i``.  A token whose position is negative or past the sequence's page table, or
    whose page is not one of the cache's, is left out.  No two tokens of a call may have the same
    place; every other row of the cache keeps its values.

    The write is in place: ``cache`` must be an argument of the traced function (or another
    write's result), contiguous and 16-byte aligned, in no other argument's memory, and the result
    is that very tensor.  Whatever reads the cache in the same function has to read the result, and
    the result has to be returned or read.  Autograd does not record the write; a call moves the
    tensor's version, as torch's own writes in place do (a captured graph's replays do not), so a
    backward pass that needs its former values is refused."""
    op = "paged_write"
    ins = [_node(op, "cache", cache), _node(op, "x", x), _node(op, "pages", pages), _node(op, "starts", starts)]
    if counts is not None:
        ins.append(_node(op, "counts", counts))
    return Tensor(_active().create(op, ins))


def paged_attention(q: Tensor, k: Tensor, v: Tensor, pages: Tensor, starts: Tensor, counts: Tensor | None = None, *,
                    scale: float | None = None, window: int | None = None) -> Tensor:
    """Causal attention of new tokens over a paged cache that already holds their keys and values.

    ``q`` is ``[batch, S, query heads, dim]``, the caches ``k`` and ``v`` ``[pages, page size, heads,
    dim]``; consecutive groups of ``query heads / heads`` query heads share a head of the caches.
    Query ``i < counts[b]`` (default: all ``S``) of sequence ``b`` stands at position ``t =
    starts[b] + i`` and sees the keys at positions ``0 .. t``, with ``window`` the last ``window`` of
    them (itself included).  ``scale`` (default ``dim ** -0.5``) must be from 1e-30 to 1e30.

    Keys past the page table, or in a page that is not one of the cache's, are left out.  A query
    that sees no key gives zeros, and so do one whose scores are all ``-inf`` and the rows
    ``i >= counts[b]``.  Rows of the caches that no
    query of a sequence sees are not read, and an infinity or a NaN in ``v`` reaches the queries that
    see its position, and no others.

    Scores and sums are fp32.  With 16-bit caches each weight is rounded to their type before it meets
    ``v``, as in dense attention, and the result once more: an error of 1.3 to 1.4 times that of fp32
    weights (relative to the output 2.3e-3 for 1.7e-3 in bf16, 2.9e-4 for 2.1e-4 in fp16, random data).
    fp16 holds no weight under 2^-32 of a row's largest."""
    op = "paged_attention"
    ins = [_node(op, n, t) for n, t in (("q", q), ("k", k), ("v", v), ("pages", pages), ("starts", starts))]
    if counts is not None:
        ins.append(_node(op, "counts", counts))
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.shape and q.shape[-1] else 1.0
    return Tensor(_active().create(op, ins, scale=_number(op, "scale", scale, low=1 / LARGEST, high=LARGEST),
                                   window=None if window is None else _whole(op, "window", window, 1)))


def sample(logits: Tensor, uniform: Tensor, *, temperature=1.0, top_k=None, top_p=None, min_p=None) -> Tensor:
    """One token per row of ``logits`` (``[..., rows, vocabulary]``) as i32 ``[..., rows]``.

    ``uniform`` (f32, ``[..., rows]``, values in [0, 1)) holds the random numbers: the same ones give
    the same tokens.  ``temperature``, ``top_k``, ``top_p`` and ``min_p`` are numbers, or tensors with
    one value per row (f32; ``top_k`` i32); None leaves a filter off.  With ``p = exp((logits - max)
    / temperature)`` and tokens ordered by logit, equal ones by index:

    * ``top_k`` keeps the first ``top_k`` tokens (a row's value of 0 or less: all);
    * ``top_p`` keeps, of those, each token before which less than ``top_p`` of their mass lies (a
      row's value of 1 or more: all), and always the first;
    * ``min_p`` keeps tokens with ``p >= min_p`` (the largest ``p`` is 1).

    The token is the one of the lowest index up to which the kept tokens' mass is more than
    ``uniform`` of all of it.  A temperature of 0 (in a tensor: or less) gives the first token of the
    order.  NaN logits count as ``-inf`` and such tokens are never chosen; infinite ones share the
    row.  A row with nothing but those gives -1.

    Masses are summed as integers (steps of ``2 ** -43`` of the largest), so the choice does not
    depend on any order of summation.  Of V tokens it is that of 64-bit arithmetic unless a threshold
    stands nearer to one of their cumulative masses than V ``2 ** -44`` of the largest mass and
    ``2 ** -38`` of the sum."""
    op = "sample"
    ins = [_node(op, "logits", logits), _node(op, "uniform", uniform)]
    tensors, numbers = [], []
    for name, v in (("temperature", temperature), ("top_k", top_k), ("top_p", top_p), ("min_p", min_p)):
        if isinstance(v, Tensor):
            tensors.append(name)
            ins.append(v.node)
        elif v is None and name == "temperature":
            raise TypeError("sample: temperature must be a number or a tensor")
        elif v is not None:
            low = 0.0 if name in ("temperature", "min_p") else -math.inf
            numbers.append((name, _whole(op, name, v, 1) if name == "top_k" else
                            _number(op, name, v, low=low, above=0.0 if name == "top_p" else -math.inf,
                                    high=LARGEST if name == "temperature" else 1.0,
                                    least=SMALLEST_FP32 if name == "temperature" else 0.0)))
    return Tensor(_active().create(op, ins, tensors=tuple(tensors), numbers=tuple(numbers)))
