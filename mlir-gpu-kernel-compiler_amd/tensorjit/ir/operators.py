"""Operators: nodes that one hand-written kernel family computes whole.

They stand beside the primitives of the op table: the fusion passes give each a kernel of its own
(kind ``operator``) and neither join pointwise work to it nor look inside.  This module holds what
the IR knows of them: result types with the checks of their operands, and which of them write into
an operand's storage.

An operator in ``IN_PLACE`` returns its operand's own storage, changed.  In the graph its result is
a new value, so that readers are ordered behind the write by their data dependence; ``check_writes``
refuses the graphs in which that order would not hold.
"""
from __future__ import annotations

from .graph import DType, Graph, Node, TensorType

# operator -> position of the operand whose storage the result is
IN_PLACE = {"paged_write": 0}

MAX_HEAD_DIM = 256      # paged_attention
MAX_VOCABULARY = 1 << 20

_FLOATS = (DType.f32, DType.f16, DType.bf16)


def _float(op: str, name: str, n: Node) -> None:
    if n.dtype not in _FLOATS:
        raise TypeError(f"{op}: {name} must be f32, f16 or bf16, got {n.dtype.value}")


def _ints(op: str, name: str, n: Node, shape: tuple) -> None:
    if n.dtype != DType.i32:
        raise TypeError(f"{op}: {name} must be i32, got {n.dtype.value}")
    if tuple(n.shape) != shape:
        raise ValueError(f"{op}: {name} must have shape {shape}, got {tuple(n.shape)}")


def position_shape(x: tuple, heads_first: bool) -> tuple:
    """The tokens of ``x``: ``[..., S]`` of ``[..., S, H, D]``, or of ``[..., H, S, D]``."""
    return x[:-3] + (x[-2],) if heads_first else x[:-2]


def _rotary(ins: list[Node], attrs: dict) -> TensorType:
    x, pos = ins
    _float("rotary", "x", x)
    if len(x.shape) < 3:
        raise ValueError(f"rotary: x must be [..., tokens, heads, dim] or [..., heads, tokens, dim], got {x.shape}")
    if pos.dtype != DType.i32:
        raise TypeError(f"rotary: positions must be i32, got {pos.dtype.value}")
    tokens = position_shape(x.shape, attrs["heads_first"])
    lead = len(tokens) - len(pos.shape)
    if lead < 0 or any(d not in (1, t) for d, t in zip(pos.shape, tokens[lead:])):
        raise ValueError(f"rotary: positions {pos.shape} do not broadcast to the tokens {tokens}")
    if attrs["dims"] > x.shape[-1]:
        raise ValueError(f"rotary: dims {attrs['dims']} of a head of {x.shape[-1]}")
    return x.type


def _cache(op: str, name: str, c: Node) -> None:
    _float(op, name, c)
    if len(c.shape) != 4:
        raise ValueError(f"{op}: {name} must be [pages, page size, heads, dim], got {c.shape}")


def _sequences(op: str, ins: list[Node], batch: int, page: int) -> None:
    """The page table, the first new position and (optional) the count of new tokens per sequence."""
    pages, starts = ins[0], ins[1]
    if pages.dtype != DType.i32:
        raise TypeError(f"{op}: pages must be i32, got {pages.dtype.value}")
    if len(pages.shape) != 2 or pages.shape[0] != batch:
        raise ValueError(f"{op}: pages must be [{batch}, pages per sequence], got {pages.shape}")
    if pages.shape[1] * page >= 2**31 - 2**16:
        raise ValueError(f"{op}: {pages.shape[1]} pages of {page} pass 32-bit positions")
    if batch * pages.shape[1] >= 2**31:
        raise ValueError(f"{op}: a page table of {batch} x {pages.shape[1]} passes 32-bit places")
    _ints(op, "starts", starts, (batch,))
    if len(ins) > 2:
        _ints(op, "counts", ins[2], (batch,))


def _paged_write(ins: list[Node], attrs: dict) -> TensorType:
    cache, x = ins[:2]
    _cache("paged_write", "cache", cache)
    if len(x.shape) != 4 or x.shape[2:] != cache.shape[2:]:
        raise ValueError(f"paged_write: x must be [batch, tokens, {cache.shape[2]}, {cache.shape[3]}] as the cache's rows, got {x.shape}")
    if x.dtype != cache.dtype:
        raise TypeError(f"paged_write: x is {x.dtype.value}, the cache {cache.dtype.value}")
    _sequences("paged_write", ins[2:], x.shape[0], cache.shape[1])
    return cache.type


def _paged_attention(ins: list[Node], attrs: dict) -> TensorType:
    q, k, v = ins[:3]
    op = "paged_attention"
    _float(op, "q", q)
    _cache(op, "k", k)
    if len(q.shape) != 4:
        raise ValueError(f"{op}: q must be [batch, tokens, heads, dim], got {q.shape}")
    if v.type != k.type:
        raise ValueError(f"{op}: k is {k.type}, v {v.type}: both caches must be alike")
    if q.dtype != k.dtype:
        raise TypeError(f"{op}: q is {q.dtype.value}, the caches {k.dtype.value}")
    B, S, H, D = q.shape
    if D != k.shape[3]:
        raise ValueError(f"{op}: q has heads of {D}, the caches of {k.shape[3]}")
    if k.shape[2] == 0 or H % k.shape[2]:
        raise ValueError(f"{op}: {H} query heads do not share {k.shape[2]} heads of the caches evenly")
    unit = 16 // q.dtype.itemsize
    if D % unit or not 0 < D <= MAX_HEAD_DIM:
        raise ValueError(f"{op}: the head dim must be a multiple of {unit} ({q.dtype.value}) up to {MAX_HEAD_DIM}, got {D}")
    _sequences(op, ins[3:], B, k.shape[1])
    return q.type


def _sample(ins: list[Node], attrs: dict) -> TensorType:
    logits, uniform = ins[:2]
    _float("sample", "logits", logits)
    if len(logits.shape) < 2:
        raise ValueError(f"sample: logits must be [..., rows, vocabulary], got {logits.shape}")
    rows = tuple(logits.shape[:-1])
    if logits.shape[-1] > MAX_VOCABULARY:
        raise ValueError(f"sample: a vocabulary of {logits.shape[-1]} is over {MAX_VOCABULARY}")
    if uniform.dtype != DType.f32 or tuple(uniform.shape) != rows:
        raise ValueError(f"sample: uniform must be f32 {rows}, got {uniform.type}")
    for name, n in zip(attrs["tensors"], ins[2:]):
        want = DType.i32 if name == "top_k" else DType.f32
        if n.dtype != want or tuple(n.shape) != rows:
            raise ValueError(f"sample: {name} must be a number or {want.value} {rows}, got {n.type}")
    return TensorType(rows, DType.i32)


INFER = {"rotary": _rotary, "paged_write": _paged_write, "paged_attention": _paged_attention, "sample": _sample}


def infer_operator(op: str, inputs: list[Node], attrs: dict) -> TensorType:
    return INFER[op](inputs, attrs)


# ---------------------------------------------------------------------------
# writes in place
# ---------------------------------------------------------------------------


def _unshaped(n: Node) -> Node:
    while n.op == "reshape":
        n = n.inputs[0]
    return n


def check_writes(g: Graph) -> None:
    """Refuse graphs whose in-place operators would be dropped, or race with other readers.

    Every write has to reach an output (a program computes what is returned), its operand has to
    be an argument of the program or an earlier write's result, and nothing else may read the
    operand, as it is or reshaped, nor may the write's other operands be it: a reader of the value
    before the write has no order with it."""
    writes = [n for n in g.nodes if n.op in IN_PLACE]
    if not writes:
        return
    live: set[int] = set()
    todo = list(g.outputs)
    while todo:
        n = todo.pop()
        if id(n) not in live:
            live.add(id(n))
            todo.extend(n.inputs)
    outs = {id(o) for o in g.outputs}
    for w in writes:
        if id(w) not in live:
            raise ValueError(f"{w.op}: the result must be returned, or read by what is returned")
        place = IN_PLACE[w.op]
        before = _unshaped(w.inputs[place])
        if before.op != "input" and before.op not in IN_PLACE:
            raise ValueError(f"{w.op} writes into its first operand: it must be an argument of the function or the "
                             f"result of another {w.op}, not of {before.op}")
        values, readers = [before], []
        while values:
            v = values.pop()
            if id(v) in outs:
                readers.append("the function's result")
            for u in v.users:
                if id(u) not in live:
                    continue
                if u.op == "reshape":
                    values.append(u)
                elif u is not w or any(i is v for j, i in enumerate(w.inputs) if j != place):
                    readers.append(u.op)
        if readers:
            raise ValueError(f"{w.op}: the cache is also read by {', '.join(sorted(set(readers)))} without the write: "
                             f"read the result of {w.op} instead")
