"""Kernels of the operators (``ir/operators.py``): rotary positions and writes into a paged cache
here, paged attention in ``hip_paged``, sampling in ``hip_sample``.

Like every kernel of the backend they are generated per shape: sizes, layouts and number
parameters are literals of the text, lengths and page tables are data, and every index that
comes from data is checked in the kernel before it is used.
"""
from __future__ import annotations

import math

from ..ir import DType
from ..ir.operators import position_shape
from ..runtime.autotune import CU_COUNT
from .common import broadcast_strides, offset_expr
from .hip_kernels import KernelGen, Launch, _index_type

THREADS = 256
# element type of vectors that are converted to and from fp32 whole
ETYPE = {DType.f32: "float", DType.f16: "_Float16", DType.bf16: "__bf16"}


def operator_name(g: KernelGen) -> str:
    n = g.k.anchor
    return f"tj{g.idx}_{n.op}_{'x'.join(str(d) for d in n.inputs[0].shape)}_{n.inputs[0].dtype.value}"


def operand(g: KernelGen, i: int) -> str:
    """The kernel parameter of the operator's operand ``i`` (operands may be one and the same)."""
    return g.names[id(g.k.anchor.inputs[i])] + "_p"


def gen_operator(g: KernelGen):
    op = g.k.anchor.op
    if op == "rotary":
        return gen_rotary(g)
    if op == "paged_write":
        return gen_paged_write(g)
    if op == "paged_attention":
        from .hip_paged import gen_paged_attention

        return gen_paged_attention(g)
    if op == "sample":
        from .hip_sample import gen_sample

        return gen_sample(g)
    raise NotImplementedError(op)


def pow2_divisor(n: int, most: int) -> int:
    return math.gcd(n, most)


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------


def rotary_turns(attrs: dict) -> list[float]:
    """Turns (of 2 pi) per position of each pair."""
    dims, factor, original = attrs["dims"], attrs["factor"], attrs["original"]
    out = []
    for i in range(dims // 2):
        f = attrs["base"] ** (-2.0 * i / dims)
        if original is None:
            f /= factor
        else:
            slow, fast = attrs["ramp"]
            keep = min(max((original * f / math.tau - slow) / (fast - slow), 0.0), 1.0)
            f *= keep + (1.0 - keep) / factor
        out.append(f / math.tau)
    return out


def rotary_heads_per_thread(units: int, heads: int, item: int) -> int:
    """Heads that a thread turns by the same sines and cosines, where threads remain to fill the
    card; two at most in fp32, where 16 bytes take half as many of them.  us with 1 / 2 / 4 / 8 heads, bf16
    of 32 heads of 128: 4 x 2048 tokens 23.9 / 21.0 / 20.5 / 23.2, 4 x 256 5.1 / 3.6 / 3.5 / 5.0, 4 x 64 2.7 /
    2.8 / 3.1 / 3.5; fp32 3 x 1501 x 12 x 80 6.9 / 5.5 / 6.0 / 6.3."""
    return next((h for h in (4, 2) if h <= heads and h * item <= 8 and units // h >= 256 * CU_COUNT * h), 1)


def gen_rotary(g: KernelGen) -> tuple[str, Launch]:
    """``(a, b) -> m (a cos - b sin, a sin + b cos)`` for each pair: bound by reading and writing
    ``x`` once (4 x 2048 x 32 x 128 bf16: 20.5 us, 6.5 TB/s).

    A thread owns up to 16 bytes of pairs of one token and walks over some of its heads, so its
    sines and cosines are computed once.  The angle is taken in turns: position times turns per
    position in fp64 (a far position in fp32 would lose the fraction), of which the nearest whole
    number is dropped, so the fp32 sine and cosine see half a turn at most."""
    n = g.k.anchor
    a, x = n.attrs, n.inputs[0]
    dt, D, dims = x.dtype, x.shape[-1], a["dims"]
    E, item = ETYPE[dt], dt.itemsize
    V, half = 16 // item, dims // 2
    tokens = position_shape(x.shape, a["heads_first"])
    H, S = (x.shape[-3], x.shape[-2]) if a["heads_first"] else (x.shape[-2], 0)
    T = math.prod(tokens)
    pw = pow2_divisor(half, V // 2 if a["interleaved"] else V)      # pairs of a thread
    cw = pow2_divisor(math.gcd(dims, D), V)                         # values of a thread past dims
    UR, UC = half // pw, (D - dims) // cw
    U = UR + UC
    hpt = rotary_heads_per_thread(T * H * U, H, item)
    HG = -(-H // hpt)
    total = T * HG * U
    idx_t = _index_type(max(x.type.numel, total + THREADS))
    fname = operator_name(g)
    xp, pp, op = operand(g, 0), operand(g, 1), "out0_p"
    w = 2 * pw if a["interleaved"] else pw
    base = f"(((t / {S}u) * {H}u + h) * {S}u + t % {S}u) * {D}u" if a["heads_first"] else f"(t * {H}u + h) * {D}u"
    pos = offset_expr("t", tokens, broadcast_strides(tuple(n.inputs[1].shape), tokens))
    sign = "-" if a["inverse"] else ""
    turns = ", ".join(repr(t) for t in rotary_turns(a))
    heads = [f"#pragma unroll", f"    for (int k = 0; k < {hpt}; ++k) {{",
             f"      const {idx_t} h = hg + k * {HG}u;", *([f"      if (h >= {H}u) break;"] if HG * hpt > H else []),
             f"      const {idx_t} at = {base} + "]
    L = [f"__device__ const double {fname}_turns[{half}] = {{{turns}}};",
         f"typedef {E} {fname}_e __attribute__((ext_vector_type({w}), aligned({item})));",
         f"typedef float {fname}_f __attribute__((ext_vector_type({w})));",
         f"typedef {E} {fname}_c __attribute__((ext_vector_type({cw}), aligned({item})));",
         f'extern "C" __global__ __launch_bounds__({THREADS}) void {fname}({g.params()}) {{',
         f"  const {idx_t} id = ({idx_t})blockIdx.x * {THREADS}u + threadIdx.x;",
         f"  if (id >= {total}u) return;",
         f"  const {idx_t} u = id % {U}u, hg = id / {U}u % {HG}u, t = id / {U * HG}u;",
         *([f"  if (u < {UR}u) {{"] if UC else ["  {"]),
         f"    const double pos = (double){pp}[{pos}];",
         f"    float c[{pw}], s[{pw}];",
         "#pragma unroll", f"    for (int j = 0; j < {pw}; ++j) {{",
         f"      const double turn = pos * {fname}_turns[u * {pw}u + j];",
         "      sincospif(2.0f * (float)(turn - __builtin_rint(turn)), &s[j], &c[j]);"]
    if a["magnitude"] != 1.0:
        L.append(f"      s[j] *= {a['magnitude']!r}f; c[j] *= {a['magnitude']!r}f;")
    if sign:
        L.append("      s[j] = -s[j];")
    L += ["    }", *heads[:-1]]
    if a["interleaved"]:
        L += [heads[-1] + f"u * {w}u;",
              f"      const {fname}_f v = __builtin_convertvector(*(const {fname}_e*)((const {E}*){xp} + at), {fname}_f);",
              f"      {fname}_f r;",
              "#pragma unroll", f"      for (int j = 0; j < {pw}; ++j) {{",
              "        r[2 * j] = v[2 * j] * c[j] - v[2 * j + 1] * s[j];",
              "        r[2 * j + 1] = v[2 * j] * s[j] + v[2 * j + 1] * c[j];", "      }",
              f"      __builtin_nontemporal_store(__builtin_convertvector(r, {fname}_e), ({fname}_e*)(({E}*){op} + at));"]
    else:
        L += [heads[-1] + f"u * {w}u;",
              f"      const {fname}_f v = __builtin_convertvector(*(const {fname}_e*)((const {E}*){xp} + at), {fname}_f);",
              f"      const {fname}_f w = __builtin_convertvector(*(const {fname}_e*)((const {E}*){xp} + at + {half}u), {fname}_f);",
              f"      {fname}_f p, q;",
              "#pragma unroll", f"      for (int j = 0; j < {pw}; ++j) {{",
              "        p[j] = v[j] * c[j] - w[j] * s[j];", "        q[j] = v[j] * s[j] + w[j] * c[j];", "      }",
              f"      __builtin_nontemporal_store(__builtin_convertvector(p, {fname}_e), ({fname}_e*)(({E}*){op} + at));",
              f"      __builtin_nontemporal_store(__builtin_convertvector(q, {fname}_e), ({fname}_e*)(({E}*){op} + at + {half}u));"]
    L += ["    }", "  }"]
    if UC:
        L += ["  else {", *heads[:-1], heads[-1] + f"{dims}u + (u - {UR}u) * {cw}u;",
              f"      __builtin_nontemporal_store(*(const {fname}_c*)((const {E}*){xp} + at), ({fname}_c*)(({E}*){op} + at));",
              "    }", "  }"]
    L.append("}")
    meta = {"family": "rotary", "dtype": dt.value, "pairs": pw, "heads_per_thread": hpt,
            "bytes": 2 * x.type.numel * item + 4 * n.inputs[1].type.numel}
    return "\n".join(L), Launch(fname, (-(-total // THREADS), 1, 1), (THREADS, 1, 1), 0, meta)


# ---------------------------------------------------------------------------
# writes into a paged cache
# ---------------------------------------------------------------------------


def slot_lines(starts: str, pages: str, P: int, page: int, npages: int, b: str, i: str) -> list[str]:
    """``pg`` and ``off``, the place of token ``i`` of sequence ``b``; ``pg`` is negative where the
    token has none.  Positions are 64-bit: starts + i may pass 32."""
    return [f"const long slot = (long){starts}[{b}] + (long)({i});",
            f"const bool inside = slot >= 0 && slot < {P * page};",
            f"const unsigned int at_ = inside ? (unsigned int)slot : 0u, off = at_ % {page}u;",
            f"int pg = {pages}[{b} * {P}u + at_ / {page}u];",
            f"if (!inside || pg >= {npages}) pg = -1;"]


def gen_paged_write(g: KernelGen) -> tuple[str, Launch]:
    """Copy each new token's row (heads x dim values, contiguous on both sides) to its place:
    bound by reading and writing the rows (16 x 1021 x 8 x 128 fp16: 10.4 us, 5.5 TB/s).

    A thread moves up to 16 bytes of a row, of the largest width that divides the row, so no
    vector crosses into another token's row."""
    n = g.k.anchor
    cache, x = n.inputs[:2]
    item = cache.dtype.itemsize
    N, page = cache.shape[:2]
    B, S, P = x.shape[0], x.shape[1], n.inputs[2].shape[1]
    row = math.prod(cache.shape[2:]) * item
    w = pow2_divisor(row, 16)
    C = row // w
    vec = {2: "unsigned short", 4: "unsigned int", 8: "tj_u32x2", 16: "tj_u32x4"}[w]
    total = B * S * C
    idx_t = _index_type(max(total + THREADS, N * page * C))
    fname = operator_name(g) + f"_{B}x{S}"
    counted = len(n.inputs) > 4
    xp, tp, sp = operand(g, 1), operand(g, 2), operand(g, 3)
    L = [f'extern "C" __global__ __launch_bounds__({THREADS}) void {fname}({g.params()}) {{',
         f"  const {idx_t} id = ({idx_t})blockIdx.x * {THREADS}u + threadIdx.x;",
         f"  if (id >= {total}u) return;",
         f"  const {idx_t} c = id % {C}u, tok = id / {C}u;",
         f"  const unsigned int i = (unsigned int)(tok % {S}u), b = (unsigned int)(tok / {S}u);",
         *([f"  if ((int)i >= {operand(g, 4)}[b]) return;"] if counted else []),
         *("  " + x_ for x_ in slot_lines(sp, tp, P, page, N, "b", "i")),
         "  if (pg < 0) return;",
         f"  (({vec}*)out0_p)[(({idx_t})pg * {page}u + off) * {C}u + c] = ((const {vec}*){xp})[id];", "}"]
    meta = {"family": "paged_write", "dtype": cache.dtype.value, "bytes_per_thread": w, "bytes": 2 * B * S * row}
    return "\n".join(L), Launch(fname, (-(-total // THREADS), 1, 1), (THREADS, 1, 1), 0, meta)
