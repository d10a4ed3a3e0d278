"""Attention of new tokens over a paged cache (``ir/operators.py``).

The query heads that share a head of the caches are rows of one matrix product: row ``r`` of
sequence ``b`` and cache head ``kv`` is query ``r / G``, head ``kv G + r % G``.  Scores are computed
transposed, ``S^T = K Q^T``, so a lane holds some keys of one row and the online softmax needs no
exchange but its maximum's and sum's; the probabilities then are, as they lie, the second operand of
``O^T += V^T P^T``.

Two work divisions of a 256-lane workgroup:

* few rows (``few_rows``): the four waves take blocks of keys in turn, each with its own running
  maximum and sum, and are joined through LDS.  Bound by reading the cache: 48 tokens over 4000 to 8000
  each, 32:8 heads of 128, bf16: 200 us, 5.9 TB/s; 64 over 5000 6.5 TB/s.  A single token over 1500 takes
  8.5 us, which is latency.
* a chunk: the four waves take 16 or 32 rows each and share every key block through LDS (fp32:
  through the L1, whose rate is enough at fp32's MFMA rate).  Bound by the MFMAs and the softmax,
  which two waves of a SIMD overlap: 4 x 1024 tokens behind 8000 0.92 PFLOP/s (pages of 16) and 0.95 (of 64),
  behind ragged 1500 to 3000 209 to 245 us by the box, 0.70 to 0.82; fp32 87 TFLOP/s.

Either is also split over the keys where there are too few workgroups; the last workgroup of a
tile to finish joins the parts.  Lengths are data, so a launch has as many parts as its page table
could need, and parts that a short sequence leaves empty end at once.
"""
from __future__ import annotations

from ..ir import DType
from ..runtime.autotune import CU_COUNT
from .hip_attention import QUAD_HELPERS, XCDS
from .hip_kernels import KernelGen, Launch, _index_type, _nt_loads
from .hip_operators import operand, operator_name
from .hip_prelude import CTYPE

LOG2E = 1.4426950408889634
FP16_SHIFT = 7.0        # see SOFTMAX
FEW_ROWS = 32
FEW_TILES = 3 * CU_COUNT // 2    # see few_rows()
WIDE_TILES = CU_COUNT            # see wide_tiles()
FEW_BLOCK = 32          # keys that a wave takes at a time
LEAST_CHUNK_KEYS = 256  # see chunk_parts()
# As many as are resident; of few rows with heads over 128 half of them, by their LDS and registers, so those
# run in two rounds (48 tokens over 4000 to 8000, 8 heads of 256, bf16: 393 us, 6.2 TB/s).
CHUNK_GROUPS = FEW_GROUPS = 2 * CU_COUNT
# Few rows: blocks that a workgroup takes at least, and the blocks' worth of time that a tile takes
# before its first.  us at 8, 8 / 4, 0, 32:8 heads of 128: 8 x 4000 keys 21.6 / 24.4, 1 x 8000 12.8 / 17-19.
FEW_LEAST = FEW_OVERHEAD = 8
# And its share of a long tile is the root of this times the tile's blocks.  us at 0, 0.2, 0.33, 0.5: 1 token of 8:1
# heads over 100000 keys 55 / 31 / 29 / 30, 30000 21 / 19 / 17 / 18, 8000 11 / 11 / 12 / 11
FEW_BY_JOIN = 0.33
MAX_PARTS = 32
MOST_CHUNK_PARTS = 4 * CHUNK_GROUPS             # bounds the workspace to 140 MB
# A join's loads in flight for each lane, 4 / 8 / 12, us: 64 tokens behind 8000 39.6 / 34.9 / 34.5, one behind 1500 8.6 /
# 8.2 / 8.6 (those past the last part are made too)
JOIN_LOADS = 8
# A chunk's LDS reads stand this many fragments before their MFMAs: 0, 0 230.6, 3, 2 222.8, 6, 4 222.5 us
# (4 x 1024 tokens behind 1500-3000)
K_AHEAD, V_AHEAD = 3, 2

HELPERS = r"""#ifndef TJ_SHFL64
#define TJ_SHFL64
template <int N> struct tj_int { static constexpr int v = N; };
__device__ __forceinline__ unsigned long tj_shfl64(unsigned long v, int lane) {
  const unsigned int lo = __builtin_amdgcn_ds_bpermute(lane * 4, (int)(unsigned int)v);
  const unsigned int hi = __builtin_amdgcn_ds_bpermute(lane * 4, (int)(unsigned int)(v >> 32));
  return (unsigned long)hi << 32 | lo;
}
// the halves of a word that are finite, and whether any is not
template <bool BF> __device__ __forceinline__ unsigned int tj_odd_halves(unsigned int w) {
  return ((w & 0x7fff7fffu) + (BF ? 0x00800080u : 0x04000400u)) & 0x80008000u;      // a half from inf on reaches its top bit
}
template <bool BF> __device__ __forceinline__ bool tj_make_finite(tj_u32x4& w) {
  unsigned int any = 0u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned int odd = tj_odd_halves<BF>(w[k]);
    any |= odd;
    w[k] &= ~((odd >> 15) * 0xffffu);
  }
  return any != 0u;
}
__device__ __forceinline__ unsigned long tj_lane64(unsigned long v, int lane) {
  return (unsigned long)(unsigned int)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (unsigned int)__builtin_amdgcn_readlane((int)v, lane);
}
#endif
"""

# What every form shares: which keys the rows of a tile see, in blocks of BK keys.  Positions are
# 64-bit until they are cut to the page table.
TILE = r"""
  auto cut = [](long p) -> int { return (int)(p < 0 ? 0 : p < (long)L ? p : (long)L); };
  unsigned int b = 0u, kvh = 0u, r0 = 0u;
  long start = 0, count = 0, i1 = 0;
  int lo_all = 0, hi_all = 0, lo_one = 0, hi_one = 0, kb0 = 0;
  // the blocks of the rows r0 .. r0 + RT - 1 of a sequence with `c` new tokens from position `p` on
  auto blocks = [&](long p, long c) -> int {
    start = p;
    count = c < (long)S ? c : (long)S;
    // its queries that stand somewhere: i0 <= i < i1 (i1 <= i0: none), positions start + i
    long i0 = (long)(r0 / G);
    i1 = (long)((r0 + RT - 1u < R - 1u ? r0 + RT - 1u : R - 1u) / G) + 1;
    if (i1 > count) i1 = count;
    if (i0 < -start) i0 = -start;
    hi_all = i1 > i0 ? cut(start + i1) : 0;                        // past the last key that a row sees
    lo_all = WINDOW ? cut(start + i0 - (long)(WINDOW - 1)) : 0;
    hi_one = cut(start + i0 + 1);                                  // the first query's, and the last one's first key
    lo_one = WINDOW ? cut(start + i1 - (long)WINDOW) : 0;
    kb0 = lo_all / (int)BK;
    return hi_all > lo_all ? (hi_all + (int)BK - 1) / (int)BK - kb0 : 0;
  };
  // Whether the tile's rows see different keys of block kb.  There a masked key's zero probability meets V
  // all the same, and zero times an infinity or NaN is NaN: these are zeros in the products with V, and
  // are added afterwards to the rows that see them.
  auto uneven = [&](int kb) -> bool { return R > G && (kb * (int)BK + (int)BK > hi_one || (WINDOW && kb * (int)BK < lo_one)); };
  // f(offset of the row in the caches, key) for the keys of this part's uneven blocks, from block kb on in steps of `by`
  auto uneven_keys = [&](int kb, int end_kb, int by, auto f) {
#pragma unroll 1
    for (; kb < end_kb; kb += by) {
      if (!uneven(kb)) continue;
#pragma unroll 1
      for (int key = kb * (int)BK; key < kb * (int)BK + (int)BK; ++key) {
        if (key < lo_all || key >= hi_all) continue;
        const int p = pages_p[b * P + (unsigned int)key / PAGE];
        if ((unsigned int)p < N) f((unsigned long)(unsigned int)p * ((row_t)PAGE * KV * D) + ((row_t)((unsigned int)key % PAGE) * KV + kvh) * D, key);
      }
    }
  };
  // keys that row r sees: lo <= key < hi
  auto bounds = [&](unsigned int r, int& lo, int& hi) -> bool {
    const long i = (long)(r / G), p = start + i;
    const bool real = r < R && i < count && p >= 0;
    hi = real ? cut(p + 1) : 0;
    lo = real && WINDOW ? cut(p - (long)(WINDOW - 1)) : 0;
    return hi > lo;
  };
"""

# A chunk: a workgroup per tile of rows, and per part of the tile's blocks where the tiles alone
# would leave CUs idle.
CHUNK_BEGIN = r"""
  b = vh / KV % BATCH; kvh = vh % KV; r0 = qt * RT;
  const unsigned int tile = (b * KV + kvh) * NQ + qt, part = vh / (BATCH * KV);
  {
    const int nb = blocks((long)starts_p[b], COUNT(b));
    const int share = (nb + (int)PARTS - 1) / (int)PARTS > LEAST ? (nb + (int)PARTS - 1) / (int)PARTS : LEAST;
    const unsigned int parts = nb > 0 ? (unsigned int)((nb + share - 1) / share) : 1u;   // those that have blocks
    if (part >= parts) return;
    const int first = kb0 + (int)part * share, last = first + share < kb0 + nb ? first + share : kb0 + nb;
    auto slot = [&](unsigned int p) -> unsigned int { return (tile * PARTS + p) * PART_BYTES; };
    const unsigned int p_first = 0u, mine = part;
"""
CHUNK_END = "  }"

# Few rows: a tile is a head of a sequence.  All blocks, tile after tile, are dealt to the workgroups
# in equal shares of consecutive ones: a workgroup ends one tile, runs others whole and begins a
# last one, whatever the lengths, and all of them end together.  Each wave finds its workgroup's
# first tile for itself, by a scan over the sequences.
FEW_BEGIN = r"""
  // a tile takes the time of OVERHEAD blocks before its first; one without keys is still written
  auto cost = [&](int n) -> pos_t { return OVERHEAD + (n > 0 ? n : 1); };
  constexpr unsigned int PER = (BATCH + 63u) / 64u;
  pos_t own = 0;
  long lane_start = 0, lane_count = 0;
  for (unsigned int k = 0; k < PER; ++k) {
    const unsigned int x = lane * PER + k;
    if (x >= BATCH) break;
    lane_start = (long)starts_p[x];
    lane_count = COUNT(x);
    own += KV * cost(blocks(lane_start, lane_count));
  }
  pos_t upto = own;
  if (BATCH > 1u) {
    for (int o = 1; o < 64; o *= 2) {
      const pos_t w = (pos_t)tj_shfl64((unsigned long)upto, (int)lane >= o ? (int)lane - o : (int)lane);
      upto += (int)lane >= o ? w : (pos_t)0;
    }
  }
  const pos_t all = (pos_t)tj_lane64((unsigned long)upto, BATCH > 1u ? 63 : 0);
  // a tile's blocks take time one after the other in a part, and its parts in the join: the least of both
  const unsigned int busy = (unsigned int)__builtin_popcountl(__builtin_amdgcn_ballot_w64(own > KV * cost(0) * PER));
  const float each = (float)all / (float)((busy ? busy : 1u) * KV);
  const pos_t even = (pos_t)__builtin_sqrtf(each * BY_JOIN), least = even > LEAST ? even : (pos_t)LEAST;
  const pos_t share = (all + GROUPS - 1u) / GROUPS > least ? (all + GROUPS - 1u) / GROUPS : least;
  const unsigned int me = blockIdx.x;
  pos_t pos = me * share;
  const pos_t end = pos + share < all ? pos + share : all;
  if (pos >= all) return;
  const int at = __builtin_ctzl(__builtin_amdgcn_ballot_w64(upto > pos));       // the lane that holds the tile
  pos_t tile_at = (pos_t)tj_lane64((unsigned long)(upto - own), at);
  b = at * PER;
  int nb;
  if (PER == 1u) {
    nb = blocks((long)tj_lane64((unsigned long)lane_start, at), (long)tj_lane64((unsigned long)lane_count, at));
  } else {
    while (nb = blocks((long)starts_p[b], COUNT(b)), tile_at + KV * cost(nb) <= pos) {
      tile_at += KV * cost(nb);
      ++b;
    }
  }
  kvh = (unsigned int)((pos - tile_at) / cost(nb));
  tile_at += kvh * cost(nb);
  for (;;) {
    const pos_t real_at = tile_at + OVERHEAD, next_at = tile_at + cost(nb), stop_at = end < next_at ? end : next_at;
    if (stop_at > real_at) {
    const pos_t k0 = real_at / share, k1 = (next_at - 1) / share;
    const unsigned int parts = (unsigned int)(k1 - k0) + 1u, tile = b * KV + kvh;
    const int first = kb0 + (pos > real_at ? (int)(pos - real_at) : 0), upto_kb = kb0 + (int)(stop_at - real_at);
    const int last = nb > 0 ? upto_kb : first;
    // a workgroup's first slot holds its part of the tile that it ends, the second that of the one it begins
    auto slot = [&](unsigned int k) -> unsigned int { return (k * 2u + (real_at < (pos_t)k * share ? 0u : 1u)) * PART_BYTES; };
    const unsigned int p_first = (unsigned int)k0, mine = me;
"""
FEW_END = r"""
    }
    pos = tile_at + cost(nb);
    if (pos >= end) break;
    tile_at = pos;
    if (++kvh == KV) {
      kvh = 0u;
      ++b;
      nb = blocks((long)starts_p[b], COUNT(b));
    }
    __syncthreads();
  }
"""

# The parts (RT x D floats, then RT pairs of reference and sum) go to the stream's workspace, agent-
# coherent, as they may come from different XCDs.  The last workgroup of a tile joins them, in order.
PART = r"""
    const __amdgpu_buffer_rsrc_t ws = __builtin_amdgcn_make_buffer_rsrc((void*)ws_p, (short)0, WS_BYTES, 0x00020000);
    const int to = __builtin_amdgcn_readfirstlane((int)slot(mine));
"""
JOIN = r"""
    if (parts > 1u) {
      __builtin_amdgcn_s_waitcnt(0x0F70);       // vmcnt(0): this wave's stores are done
      __syncthreads();
      __shared__ unsigned int last_one;
      if (tid == 0u) last_one = atomicInc(&cnt_p[tile], parts - 1u) == parts - 1u ? 1u : 0u;   // wraps to 0
      __syncthreads();
      if (last_one) {
        // JU x JK loads in flight: each trip to the other XCDs' data costs a microsecond or two.  Those past the
        // last part read its again, and those past the last row the first's, which are not used.
        constexpr unsigned int QUADS = (RT < R ? RT : R) * (D / 4u);
        for (unsigned int w0 = tid; w0 < QUADS; w0 += 256u * JU) {
          float m[JU], l[JU];
          tj_f32x4 acc[JU];
#pragma unroll
          for (unsigned int u = 0; u < JU; ++u) { m[u] = LOWEST; l[u] = 0.0f; acc[u] = (tj_f32x4)(0.0f); }
          for (unsigned int p0 = 0; p0 < parts; p0 += JK) {
            tj_u32x2 ml[JK][JU];
            tj_u32x4 o[JK][JU];
#pragma unroll
            for (unsigned int k = 0; k < JK; ++k) {
              const int at = __builtin_amdgcn_readfirstlane((int)slot(p_first + (p0 + k < parts ? p0 + k : parts - 1u)));
#pragma unroll
              for (unsigned int u = 0; u < JU; ++u) {
                const unsigned int t = w0 + u * 256u, w = t < QUADS && r0 + t / (D / 4u) < R ? t : 0u;
                ml[k][u] = __builtin_amdgcn_raw_buffer_load_b64(ws, (int)(RT * D + w / (D / 4u) * 2u) * 4, at, 16);
                o[k][u] = __builtin_amdgcn_raw_buffer_load_b128(ws, (int)w * 16, at, 16);
              }
            }
#pragma unroll
            for (unsigned int k = 0; k < JK; ++k) {
              // selects: behind a branch the loads would move to their use, one trip after the other
              const bool part = p0 + k < parts;
#pragma unroll
              for (unsigned int u = 0; u < JU; ++u) {
                const float mp = part ? __builtin_bit_cast(float, (unsigned int)ml[k][u][0]) : LOWEST;
                const float mn = fmaxf(m[u], mp), fa = __builtin_amdgcn_exp2f(m[u] - mn), fb = __builtin_amdgcn_exp2f(mp - mn);
                l[u] = l[u] * fa + (part ? __builtin_bit_cast(float, (unsigned int)ml[k][u][1]) * fb : 0.0f);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[u][e] = acc[u][e] * fa + (part ? __builtin_bit_cast(float, (unsigned int)o[k][u][e]) * fb : 0.0f);
                m[u] = mn;
              }
            }
          }
#pragma unroll
          for (unsigned int u = 0; u < JU; ++u) {
            const unsigned int w = w0 + u * 256u, r = r0 + w / (D / 4u);
            if (w < QUADS && r < R) finish(r, w % (D / 4u) * 4u, acc[u], l[u]);
          }
        }
      }
    }
"""

# 16-bit types, few rows.  A wave takes a block of 32 keys: whole rows of K and V from memory to
# registers, one block ahead, and on to the wave's own LDS tiles.
FEW16 = r"""
  __shared__ __attribute__((aligned(16))) T Ks[4][BK][KP];
  __shared__ __attribute__((aligned(16))) T Vs[4][BK][VP];
  __shared__ float ml[4][16][2];
  constexpr unsigned int DC = D / 8u, KC = (DC + 3u) / 4u, NC = (BK * DC + 63u) / 64u, NU = (D + 15u) / 16u;
  // columns between D and the MFMAs' width: zeros once
  if (D % 32u) {
    constexpr unsigned int PAD = KC * 4u > DC ? KC * 4u - DC : 1u;
    for (unsigned int t = lane; t < BK * PAD; t += 64u) *(tj_u32x4*)&Ks[wave][t / PAD][D + t % PAD * 8u] = (tj_u32x4)(0u);
  }
  tj_u32x4 kn[NC], vn[NC];
  int pn = -1;                 // lane: the page of key lane % 32 of the next block, -1: none that anybody sees
  auto page_of = [&](int kb) {
    const int key = kb * (int)BK + (int)(lane % BK);
    int p = -1;
    if (key >= lo_all && key < hi_all) p = pages_p[b * P + (unsigned int)key / PAGE];
    return (unsigned int)p < N ? p : -1;
  };
  auto fetch = [&](int kb) {
#pragma unroll
    for (unsigned int i = 0; i < NC; ++i) {
      const unsigned int c = i * 64u + lane, row = c / DC;
      const int p = __builtin_amdgcn_ds_bpermute((int)(row % BK) * 4, pn);
      const unsigned long at = (unsigned long)(unsigned int)p * ((row_t)PAGE * KV * D) +
                               ((row_t)((unsigned int)(kb * (int)BK + (int)row) % PAGE) * KV + kvh) * D + c % DC * 8u;
      kn[i] = vn[i] = (tj_u32x4)(0u);
      if (p >= 0 && (BK * DC % 64u == 0u || row < BK)) {
        kn[i] = LOAD16(&k_p[at]);
        vn[i] = LOAD16(&v_p[at]);
      }
    }
  };
  OPV qf[QT][KC];
  int lo[QT], hi[QT];
  bool sees[QT];
  float m_run[QT], l_run[QT];
  bool far = false;                  // see SOFTMAX
  tj_f32x4 o[QT][NU];
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const unsigned int r = r0 + x * 16u + r16;
    sees[x] = bounds(r, lo[x], hi[x]);
    m_run[x] = LOWEST;
    l_run[x] = 0.0f;
#pragma unroll
    for (unsigned int u = 0; u < NU; ++u) o[x][u] = (tj_f32x4)(0.0f);
#pragma unroll
    for (unsigned int c = 0; c < KC; ++c) {
      tj_u32x4 w = (tj_u32x4)(0u);
      if (sees[x] && (DC % 4u == 0u || c * 4u + g16 < DC)) w = *(const tj_u32x4*)&q_p[q_at(r) + (c * 4u + g16) * 8u];
      qf[x][c] = __builtin_bit_cast(OPV, w);
    }
    if (!sees[x]) { lo[x] = 0; hi[x] = 0x7fffffff; }      // its sums are not used: no reason to mask
  }
  int kb = first + (int)wave;
  bool odd = false;            // V held infinities or NaN among uneven keys
  int pnn = -1;                // of the block after
  if (kb < last) {
    pn = page_of(kb);
    pnn = page_of(kb + 4);
    fetch(kb);
  }
  for (; kb < last; kb += 4) {
    const unsigned int real = (unsigned int)__builtin_amdgcn_ballot_w64(pn >= 0);
    if (uneven(kb)) {
#pragma unroll
      for (unsigned int i = 0; i < NC; ++i) odd |= tj_make_finite<BF>(vn[i]);
    }
#pragma unroll
    for (unsigned int i = 0; i < NC; ++i) {
      const unsigned int c = i * 64u + lane;
      if (BK * DC % 64u && c >= BK * DC) continue;
      *(tj_u32x4*)&Ks[wave][c / DC][c % DC * 8u] = kn[i];
      *(tj_u32x4*)&Vs[wave][c / DC][c % DC * 8u] = vn[i];
    }
    if (kb + 4 < last) {
      pn = pnn;
      pnn = page_of(kb + 8);
      fetch(kb + 4);
    }
    WAVE_FENCE;
    tj_f32x4 sq[QT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int x = 0; x < QT; ++x) sq[x][t] = (tj_f32x4)(0.0f);
#pragma unroll
      for (unsigned int c = 0; c < KC; ++c) {
        const OPV kf = *(const OPV*)&Ks[wave][t * 16u + r16][c * 32u + g16 * 8u];
#pragma unroll
        for (int x = 0; x < QT; ++x) sq[x][t] = MFMA(kf, qf[x][c], sq[x][t], 0, 0, 0);
      }
    }
    OPV pf[QT];
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      tj_f32x4* s = sq[x];
      const int k0 = kb * (int)BK;
      if (__builtin_amdgcn_ballot_w64(k0 < lo[x] || k0 + (int)BK > hi[x]) || real != 0xffffffffu) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = e / 4 * 16 + (int)g16 * 4 + e % 4;
          if (!(real >> j & 1u) || k0 + j < lo[x] || k0 + j >= hi[x]) s[e / 4][e % 4] = -__builtin_inff();
        }
      }
      SOFTMAX(x, 2, NU)
      tj_u32x4 pw;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[w / 2][w % 2 * 2], CS, -ref));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[w / 2][w % 2 * 2 + 1], CS, -ref));
        pw[w] = PACK2(e0, e1);
        l_run[x] = PAIR_SUM(pw[w], l_run[x]);
      }
      pf[x] = __builtin_bit_cast(OPV, pw);
    }
#pragma unroll
    for (unsigned int u = 0; u < NU; ++u) {
      const tj_i16x4 va = TR_READ(&Vs[wave][g16 * 4u + r16 / 4u][u * 16u + r16 % 4u * 4u]);
      const tj_i16x4 vb = TR_READ(&Vs[wave][16u + g16 * 4u + r16 / 4u][u * 16u + r16 % 4u * 4u]);
      const OPV vf = __builtin_bit_cast(OPV, __builtin_shufflevector(va, vb, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int x = 0; x < QT; ++x) o[x][u] = MFMA(vf, pf[x], o[x][u], 0, 0, 0);
    }
    WAVE_FENCE;
  }
  if (__builtin_amdgcn_ballot_w64(odd)) {
    uneven_keys(first + (int)wave, last, 4, [&](unsigned long at, int key) {
#pragma unroll
      for (int x = 0; x < QT; ++x) {
        if (key < lo[x] || key >= hi[x]) continue;
#pragma unroll
        for (unsigned int u = 0; u < NU; ++u) {
          if (u * 16u + g16 * 4u >= D) continue;
          const tj_u32x2 w = *(const tj_u32x2*)&v_p[at + u * 16u + g16 * 4u];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned int h = w[k / 2] >> (k % 2 * 16) & 0xffffu;
            if (tj_odd_halves<BF>(h)) o[x][u][k] += TO_FLOAT(h);
          }
        }
      }
    });
  }
"""

# the four waves' rows of column tile x joined, in their V tiles' place
FEW_JOIN = r"""
  for (int x = 0; x < QT; ++x) {
    const float l_wave = tj_quad_sum(l_run[x]);
    __syncthreads();
    if (g16 == 0u) { ml[wave][r16][0] = m_run[x]; ml[wave][r16][1] = l_wave; }
    ROWS_TO_LDS
    __syncthreads();
    for (unsigned int t = tid; t < 16u * (D / 4u); t += 256u) {
      const unsigned int row = t / (D / 4u), d = t % (D / 4u) * 4u, r = x * 16u + row;
      if (r >= R) break;
      const float m = fmaxf(fmaxf(ml[0][row][0], ml[1][row][0]), fmaxf(ml[2][row][0], ml[3][row][0]));
      float l = 0.0f;
      tj_f32x4 acc = (tj_f32x4)(0.0f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(ml[w][row][0] - m);
        l += f * ml[w][row][1];
        acc += f * *(const tj_f32x4*)(WROWS(w) + row * D + d);
      }
      if (SINGLE) {
        finish(r, d, acc, l);
      } else {
        STORE_PART
      }
    }
  }
"""
STORE_FEW = r"""
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(tj_u32x4, acc), ws, (int)(r * D + d) * 4, to, 16);
        if (d == 0u) {
          tj_u32x2 p;
          p[0] = __builtin_bit_cast(unsigned int, m);
          p[1] = __builtin_bit_cast(unsigned int, l);
          __builtin_amdgcn_raw_buffer_store_b64(p, ws, (int)(RT * D + r * 2u) * 4, to, 16);
        }
"""

# Lazy rescale: the reference moves only where a score passes it by 2^8.  The 16-bit types round the
# probabilities to theirs, as the product with V on MFMAs takes them (half a step each); the sums are those of
# the rounded ones, so that the weights sum to one.  fp16 ones stand 2^SHIFT higher, up to 2^15: fp16 has steps
# of 2^-24 below 2^-14, and without SHIFT a weight under 2^-25 of the largest came to nothing, however many.
# An exponent is fma(s, CS, -ref), where the reference is a rounded product: together off by half a last place
# of the reference, the same for all keys of a row.  From 2^27 on that would be a power that no type holds, so
# far references take rounded products on both sides.
SOFTMAX = r"""
      float ref;
      {
#pragma clang fp contract(off)
        float mx = s[0][0];
#pragma unroll
        for (int e = 1; e < 4 * (TILES); ++e) mx = fmaxf(mx, s[e / 4][e % 4]);
        const float mb = mx * CS;
        if (__builtin_amdgcn_ballot_w64(mb - m_run[X] > 8.0f + SHIFT)) {
          const float mn = fmaxf(m_run[X], tj_quad_max(mb) - SHIFT), f = __builtin_amdgcn_exp2f(m_run[X] - mn);
          l_run[X] *= f;
#pragma unroll
          for (unsigned int u = 0; u < (UNITS); ++u) o[X][u] *= f;
          m_run[X] = mn;
          far |= __builtin_amdgcn_ballot_w64(__builtin_fabsf(mn) > 0x1p20f && mn != LOWEST) != 0ul;
        }
        ref = m_run[X];
        if (far) {
#pragma unroll
          for (int e = 0; e < 4 * (TILES); ++e) s[e / 4][e % 4] = (s[e / 4][e % 4] * CS - ref) * (1.0f / CS);
          ref = 0.0f;
        }
      }
"""

# 16-bit types, a chunk: 64 (32 past head dim 128) keys per block in LDS, two stages; the next
# block is on its way to registers while this one is computed.
CHUNK16 = r"""
  __shared__ __attribute__((aligned(16))) T Ks[2][BK][KP];
  __shared__ __attribute__((aligned(16))) T Vs[2][BK][VP];
  constexpr unsigned int DC = D / 8u, KC = (DC + 3u) / 4u, NC = (BK * DC + 255u) / 256u, NU = (D + 15u) / 16u, NT = BK / 16u;
  // columns between D and the MFMAs' width: zeros once
  if (D % 32u) {
    constexpr unsigned int PAD = KC * 4u > DC ? KC * 4u - DC : 1u;
    for (unsigned int t = tid; t < 2u * BK * PAD; t += 256u)
      *(tj_u32x4*)((unsigned short*)Ks + t / PAD * KP + D + t % PAD * 8u) = (tj_u32x4)(0u);
  }
  __shared__ int odd;                    // V held infinities or NaN among uneven keys
  if (tid == 0u) odd = 0;
  __syncthreads();
  tj_u32x4 kn[NC], vn[NC];
#pragma unroll
  for (unsigned int i = 0; i < NC; ++i) vn[i] = (tj_u32x4)(0u);       // lanes past the last row: finite
  unsigned long real_next = 0ul;
  auto page_of = [&](int kb) {
    const int key = kb * (int)BK + (int)(lane % BK);
    int p = -1;
    if (key >= lo_all && key < hi_all) p = pages_p[b * P + (unsigned int)key / PAGE];
    return (unsigned int)p < N ? p : -1;
  };
  auto fetch = [&](int kb, int pg) {
    real_next = __builtin_amdgcn_ballot_w64(pg >= 0);
#pragma unroll
    for (unsigned int i = 0; i < NC; ++i) {
      const unsigned int c = i * 256u + tid, row = c / DC;
      int p = __builtin_amdgcn_ds_bpermute((int)(row % BK) * 4, pg);
      p = p < 0 ? 0 : p;                       // not kept: see put
      const unsigned long at = (unsigned long)(unsigned int)p * ((row_t)PAGE * KV * D) +
                               ((row_t)((unsigned int)(kb * (int)BK + (int)row) % PAGE) * KV + kvh) * D + c % DC * 8u;
      if (BK * DC % 256u == 0u || row < BK) {
        kn[i] = *(const tj_u32x4*)&k_p[at];
        vn[i] = *(const tj_u32x4*)&v_p[at];
      }
    }
  };
  auto put = [&](auto st, int kb, unsigned long real) {
    if (real != ~0ul) {                        // rows that nobody sees: a zero probability times what lies there
#pragma unroll
      for (unsigned int i = 0; i < NC; ++i)
        if (!(real >> ((i * 256u + tid) / DC % BK) & 1ul)) vn[i] = (tj_u32x4)(0u);
    }
    if (uneven(kb)) {
#pragma unroll
      for (unsigned int i = 0; i < NC; ++i)
        if (tj_make_finite<BF>(vn[i])) odd = 1;
    }
#pragma unroll
    for (unsigned int i = 0; i < NC; ++i) {
      const unsigned int c = i * 256u + tid;
      if (BK * DC % 256u && c >= BK * DC) continue;
      *(tj_u32x4*)&Ks[st.v][c / DC][c % DC * 8u] = kn[i];
      *(tj_u32x4*)&Vs[st.v][c / DC][c % DC * 8u] = vn[i];
    }
  };
  OPV qf[QT][KC];
  int lo[QT], hi[QT];
  bool sees[QT];
  float m_run[QT], l_run[QT];
  bool far = false;                  // see SOFTMAX
  tj_f32x4 o[QT][NU];
  const unsigned int rw = r0 + wave * (16u * QT);
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const unsigned int r = rw + x * 16u + r16;
    sees[x] = bounds(r, lo[x], hi[x]);
    m_run[x] = LOWEST;
    l_run[x] = 0.0f;
#pragma unroll
    for (unsigned int u = 0; u < NU; ++u) o[x][u] = (tj_f32x4)(0.0f);
#pragma unroll
    for (unsigned int c = 0; c < KC; ++c) {
      tj_u32x4 w = (tj_u32x4)(0u);
      if (sees[x] && (DC % 4u == 0u || c * 4u + g16 < DC)) w = *(const tj_u32x4*)&q_p[q_at(r) + (c * 4u + g16) * 8u];
      qf[x][c] = __builtin_bit_cast(OPV, w);
    }
    if (!sees[x]) { lo[x] = 0; hi[x] = 0x7fffffff; }      // its sums are not used: no reason to mask
  }
  int pg = first < last ? page_of(first) : -1;
  if (first < last) fetch(first, pg);
  pg = first + 1 < last ? page_of(first + 1) : -1;
  auto block = [&](int kb, auto st) {
    const unsigned long real = real_next;
    put(st, kb, real);
    __syncthreads();
    if (kb + 1 < last) {
      fetch(kb + 1, pg);
      pg = kb + 2 < last ? page_of(kb + 2) : -1;
    }
    const int k0 = kb * (int)BK;
    OPV pf[QT][NT / 2];
    bool any = false;
    {
      tj_f32x4 sq[QT][NT];
#pragma unroll
      for (int x = 0; x < QT; ++x) any |= sees[x] && k0 < hi[x] && k0 + (int)BK > lo[x];
      if (__builtin_amdgcn_ballot_w64(any) == 0ul) return;
#pragma unroll
      for (unsigned int t = 0; t < NT; ++t) {
#pragma unroll
        for (int x = 0; x < QT; ++x) sq[x][t] = (tj_f32x4)(0.0f);
#pragma unroll
        for (unsigned int c = 0; c < KC; ++c) {
          const OPV kf = *(const OPV*)&Ks[st.v][t * 16u + r16][c * 32u + g16 * 8u];
#pragma unroll
          for (int x = 0; x < QT; ++x) sq[x][t] = MFMA(kf, qf[x][c], sq[x][t], 0, 0, 0);
        }
      }
QK_SCHED
      bool cut_off = real != ~0ul;
#pragma unroll
      for (int x = 0; x < QT; ++x) cut_off |= k0 < lo[x] || k0 + (int)BK > hi[x];
      if (__builtin_amdgcn_ballot_w64(cut_off)) {
        const unsigned long mine = real >> (g16 * 4u);
#pragma unroll
        for (unsigned int e = 0; e < 4u * NT; ++e) {
          const int j = k0 + (int)(e / 4u * 16u + g16 * 4u + e % 4u);
          const bool in = mine >> (e / 4u * 16u + e % 4u) & 1ul;
#pragma unroll
          for (int x = 0; x < QT; ++x)
            if (!in || j < lo[x] || j >= hi[x]) sq[x][e / 4u][e % 4u] = -__builtin_inff();
        }
      }
#pragma unroll
      for (int x = 0; x < QT; ++x) {
        tj_f32x4* s = sq[x];
        SOFTMAX(x, NT, NU)
#pragma unroll
        for (unsigned int h = 0; h < NT / 2u; ++h) {
          tj_u32x4 pw;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2u * h + w / 2][w % 2 * 2], CS, -ref));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2u * h + w / 2][w % 2 * 2 + 1], CS, -ref));
            pw[w] = PACK2(e0, e1);
            l_run[x] = PAIR_SUM(pw[w], l_run[x]);
          }
          pf[x][h] = __builtin_bit_cast(OPV, pw);
        }
      }
    }
#pragma unroll
    for (unsigned int h = 0; h < NT / 2u; ++h)
#pragma unroll
      for (unsigned int u = 0; u < NU; ++u) {
        const tj_i16x4 va = TR_READ(&Vs[st.v][h * 32u + g16 * 4u + r16 / 4u][u * 16u + r16 % 4u * 4u]);
        const tj_i16x4 vb = TR_READ(&Vs[st.v][h * 32u + 16u + g16 * 4u + r16 / 4u][u * 16u + r16 % 4u * 4u]);
        const OPV vf = __builtin_bit_cast(OPV, __builtin_shufflevector(va, vb, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int x = 0; x < QT; ++x) o[x][u] = MFMA(vf, pf[x][h], o[x][u], 0, 0, 0);
      }
PV_SCHED
  };
  // the stage is known in each of the two calls: its LDS addresses are offsets in the instructions
  for (int kb = first; kb < last; ++kb) {
    block(kb, tj_int<0>());
    if (++kb < last) block(kb, tj_int<1>());
  }
  __syncthreads();
  if (odd) {
    uneven_keys(first, last, 1, [&](unsigned long at, int key) {
#pragma unroll
      for (int x = 0; x < QT; ++x) {
        if (key < lo[x] || key >= hi[x]) continue;
#pragma unroll
        for (unsigned int u = 0; u < NU; ++u) {
          if (u * 16u + g16 * 4u >= D) continue;
          const tj_u32x2 w = *(const tj_u32x2*)&v_p[at + u * 16u + g16 * 4u];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned int h = w[k / 2] >> (k % 2 * 16) & 0xffffu;
            if (tj_odd_halves<BF>(h)) o[x][u][k] += TO_FLOAT(h);
          }
        }
      }
    });
  }
"""

# each wave's rows to the output or the part; quad (u, j) of lane group g16 holds dims DIM
CHUNK_STORE = r"""
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const unsigned int r = rw + x * 16u + r16;
    const float l = tj_quad_sum(l_run[x]);
    if (r >= R) continue;
    QUADS_BEGIN
      if (SINGLE) {
        finish(r, d, acc, l);
      } else {
        STORE_PART
      }
    QUADS_END
  }
"""
STORE_CHUNK = r"""
        const unsigned int row = r - r0;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(tj_u32x4, acc), ws, (int)(row * D + d) * 4, to, 16);
        if (d == 0u) {
          tj_u32x2 p;
          p[0] = __builtin_bit_cast(unsigned int, m_run[x]);
          p[1] = __builtin_bit_cast(unsigned int, l);
          __builtin_amdgcn_raw_buffer_store_b64(p, ws, (int)(RT * D + row * 2u) * 4, to, 16);
        }
"""

# fp32, both divisions: KW waves in turn over blocks of 16 keys, or KW = 1 and rows by wave.  Nothing
# is staged: K's fragments are 16 bytes of a row per lane, four 16x16x4 MFMAs of which element j
# feeds the j-th; V's are 16 bytes of a row too, of which element j is dim 4 r16 + j of the j-th MFMA.
DIRECT32 = r"""
  constexpr unsigned int DC = D / 4u, KC = (DC + 3u) / 4u, NV = (DC + 15u) / 16u, NU = NV * 4u;
  tj_f32x4 kn[KC], vn[4][NV];
  int pn = -1;
  auto page_of = [&](int kb) {
    const int key = kb * (int)BK + (int)r16;
    int p = -1;
    if (key >= lo_all && key < hi_all) p = pages_p[b * P + (unsigned int)key / PAGE];
    return (unsigned int)p < N ? p : -1;
  };
  auto row_at = [&](int p, int key) -> unsigned long {
    return (unsigned long)(unsigned int)p * ((row_t)PAGE * KV * D) + ((row_t)((unsigned int)key % PAGE) * KV + kvh) * D;
  };
  auto fetch_k = [&](int kb) {
    const unsigned long at = row_at(pn, kb * (int)BK + (int)r16);
#pragma unroll
    for (unsigned int c = 0; c < KC; ++c) {
      kn[c] = (tj_f32x4)(0.0f);
      if (pn >= 0 && (DC % 4u == 0u || c * 4u + g16 < DC)) kn[c] = *(const tj_f32x4*)&k_p[at + (c * 4u + g16) * 4u];
    }
  };
  bool odd = false;                  // V held infinities or NaN among uneven keys
  auto finite = [](float v) -> bool { return (__builtin_bit_cast(unsigned int, v) & 0x7f800000u) != 0x7f800000u; };
  auto fetch_v = [&](int kb) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = (int)g16 * 4 + e, p = __builtin_amdgcn_ds_bpermute(j * 4, pn);
      const unsigned long at = row_at(p, kb * (int)BK + j);
#pragma unroll
      for (unsigned int u = 0; u < NV; ++u) {
        vn[e][u] = (tj_f32x4)(0.0f);
        if (p >= 0 && (DC % 16u == 0u || u * 16u + r16 < DC)) vn[e][u] = *(const tj_f32x4*)&v_p[at + (u * 16u + r16) * 4u];
      }
    }
  };
  tj_f32x4 qf[QT][KC];
  int lo[QT], hi[QT];
  bool sees[QT];
  float m_run[QT], l_run[QT];
  bool far = false;                  // see SOFTMAX
  tj_f32x4 o[QT][NU];
  const unsigned int rw = r0 + (KW == 1 ? wave * (16u * QT) : 0u);
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const unsigned int r = rw + x * 16u + r16;
    sees[x] = bounds(r, lo[x], hi[x]);
    m_run[x] = LOWEST;
    l_run[x] = 0.0f;
#pragma unroll
    for (unsigned int u = 0; u < NU; ++u) o[x][u] = (tj_f32x4)(0.0f);
#pragma unroll
    for (unsigned int c = 0; c < KC; ++c) {
      qf[x][c] = (tj_f32x4)(0.0f);
      if (sees[x] && (DC % 4u == 0u || c * 4u + g16 < DC)) qf[x][c] = *(const tj_f32x4*)&q_p[q_at(r) + (c * 4u + g16) * 4u];
    }
    if (!sees[x]) { lo[x] = 0; hi[x] = 0x7fffffff; }        // its sums are not used: no reason to mask
  }
  int kb = first + (KW == 1 ? 0 : (int)wave), stop = last;
  if (KW == 1) {                     // a wave's own rows may end before the tile's
    long iw = (long)((rw + 16u * QT - 1u) / G) + 1;
    if (iw > i1) iw = i1;
    const int done = (cut(start + iw) + (int)BK - 1) / (int)BK;
    stop = done < stop ? done : stop;
  }
  int pnn = -1;                      // pages of the block after
  if (kb < stop) {
    pn = page_of(kb);
    pnn = page_of(kb + KW);
    fetch_k(kb);
  }
  for (; kb < stop; kb += KW) {
    const unsigned int real = (unsigned int)__builtin_amdgcn_ballot_w64(pn >= 0) & 0xffffu;
    fetch_v(kb);
    tj_f32x4 sq[QT][1];
#pragma unroll
    for (int x = 0; x < QT; ++x) sq[x][0] = (tj_f32x4)(0.0f);
#pragma unroll
    for (unsigned int c = 0; c < KC; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < QT; ++x) sq[x][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kn[c][j], qf[x][c][j], sq[x][0], 0, 0, 0);
    if (uneven(kb)) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (unsigned int u = 0; u < NU; ++u) {
          odd |= !finite(vn[e][u / 4u][u % 4u]);
          vn[e][u / 4u][u % 4u] = finite(vn[e][u / 4u][u % 4u]) ? vn[e][u / 4u][u % 4u] : 0.0f;
        }
    }
    if (kb + KW < stop) {
      pn = pnn;
      pnn = page_of(kb + 2 * KW);
      fetch_k(kb + KW);
    }
    const int k0 = kb * (int)BK;
#pragma unroll
    for (int x = 0; x < QT; ++x) {
      tj_f32x4* s = sq[x];
      if (__builtin_amdgcn_ballot_w64(k0 < lo[x] || k0 + (int)BK > hi[x]) || real != 0xffffu) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = (int)g16 * 4 + e;
          if (!(real >> j & 1u) || k0 + j < lo[x] || k0 + j >= hi[x]) s[0][e] = -__builtin_inff();
        }
      }
      SOFTMAX(x, 1, NU)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[0][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][e], CS, -ref));
        l_run[x] += s[0][e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (unsigned int u = 0; u < NU; ++u)
#pragma unroll
        for (int x = 0; x < QT; ++x)
          o[x][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(vn[e][u / 4u][u % 4u], sq[x][0][e], o[x][u], 0, 0, 0);
  }
  if (__builtin_amdgcn_ballot_w64(odd)) {
    uneven_keys(first + (KW == 1 ? 0 : (int)wave), stop, KW, [&](unsigned long at, int key) {
#pragma unroll
      for (int x = 0; x < QT; ++x) {
        if (key < lo[x] || key >= hi[x]) continue;
#pragma unroll
        for (unsigned int u = 0; u < NV; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned int d = u * 64u + g16 * 16u + i * 4u;
            if (d >= D) continue;
            const tj_f32x4 w = *(const tj_f32x4*)&v_p[at + d];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (!finite(w[j])) o[x][u * 4u + j][i] += w[j];
          }
      }
    });
  }
"""


def chunk_parts(tiles: int, blocks: int, rows: int, keys: int) -> int:
    """Parts that each tile's ``blocks`` blocks of ``keys`` keys are cut into, for the least time:
    rounds of workgroups over the card, by a round's blocks and two for its beginning and end.  A part
    also writes and reads again its rows' sums, which costs as much as 3 times as many keys; one of under
    256 keys is not worth it.

    us, parts by this rule / whole tiles, bf16 of 32:8 heads of 128: 64 tokens behind 8000 35 / 193,
    2 x 100 behind 3000 34 / 67, 2 x 512 behind 1500 60 / 65; 5 x 512 behind 1500 whole either way 127,
    in four parts 148.  At least 2, 4, 8 blocks: 100 tokens behind 700 16.5 / 14.8 / 21.2, 256 behind 1000 20 / 20 /
    23; heads of 256 with blocks of 32, 100 behind 3000, 4 / 8: 60 / 40."""
    join = 3 * rows // keys
    most = max(1, min(MAX_PARTS, blocks // (LEAST_CHUNK_KEYS // keys), MOST_CHUNK_PARTS // tiles))
    return min(range(1, most + 1),
               key=lambda n: -(-tiles * n // CHUNK_GROUPS) * (-(-blocks // n) + 2 + (join if n > 1 else 0)))


def few_rows(rows: int, D: int, tiles: int) -> bool:
    """Whether the waves of a workgroup take keys rather than rows.  Up to 16 rows always.  To 32
    it reads the caches with fewer barriers, but its join is long, which pays over many heads alone.
    us, few / chunk: 20 rows of 128 over 4000, 8 heads 20 / 17, 128 55 / 46, 256 105 / 100, 384 154 / 170,
    512 181 / 191; 30 rows of 64 over 2000, 32 heads 12 / 10, 512 47 / 55, 1024 97 / 131.  Heads over 128
    would need more registers for 32 rows than there are."""
    return rows <= 16 or D <= 128 and rows <= FEW_ROWS and tiles >= FEW_TILES


def wide_tiles(rows: int, D: int, tiles: int, f32: bool) -> bool:
    """Whether a wave of a chunk takes 32 rows: half the LDS reads for each MFMA, but half the
    workgroups.  us, 32 / 16 rows, 512 tokens behind 1500, by tiles of 128 rows: 128 39 / 39, 256 60 / 67, 384
    85 / 107, 512 91 / 123, 768 153 / 176; 384 without a token before 28 / 25.  Registers bound the head's size."""
    return D <= (64 if f32 else 128) and tiles * -(-rows // 128) >= WIDE_TILES


def _ahead(ahead: int, reads: int, fragments: int, tiles: int) -> str:
    """Scheduling hints: each fragment's LDS reads stand ``ahead`` fragments before its MFMAs."""
    if not ahead:
        return ""
    group = "__builtin_amdgcn_sched_group_barrier(%d, %d, 0);"
    out = [group % (0x100, reads * min(ahead, fragments))]
    for f in range(fragments):
        out.append(group % (0x008, tiles))
        if f + ahead < fragments:
            out.append(group % (0x100, reads))
    return " ".join(out)


def _text(src: str, **names) -> str:
    for k, v in names.items():
        src = src.replace(k, str(v))
    return src


def _softmax(src: str) -> str:
    """Expand ``SOFTMAX(x, tiles, units)``."""
    while "SOFTMAX(" in src:
        a = src.index("SOFTMAX(")
        b = src.index(")", a)
        x, tiles, units = (w.strip() for w in src[a + 8:b].split(","))
        src = src[:a] + _text(SOFTMAX, TILES=tiles, UNITS=units, X=x) + src[b + 1:]
    return src


def gen_paged_attention(g: KernelGen):
    n = g.k.anchor
    q, kc = n.inputs[:2]
    dt = q.dtype
    T = CTYPE[dt]
    f32, bf = dt == DType.f32, dt == DType.bf16
    window = n.attrs["window"] or 0
    B, S, H, D = q.shape
    N, page, KV, _ = kc.shape
    P, G = n.inputs[3].shape[1], H // KV
    R, L = S * G, P * page
    few = few_rows(R, D, B * KV)
    wide = wide_tiles(R, D, B * KV, f32)
    QT = (2 if R > 16 else 1) if few else 2 if wide else 1
    RT = 16 * QT * (1 if few else 4)
    BK = 16 if f32 else FEW_BLOCK if few else 64 if D <= 128 else 32
    nq = -(-R // RT)
    tiles = B * KV * nq
    reach = min(L, window + -(-RT // G)) if window else L       # keys that a tile's rows see at most
    blocks = -(-reach // BK) + (1 if window else 0)
    if few:
        parts, least = 1, FEW_LEAST
        places = tiles * (blocks + FEW_OVERHEAD)
        groups = max(1, min(FEW_GROUPS, -(-places // least)))
        grid, slots = groups, 2 * groups
    else:
        keys = 64 if f32 else BK                                # 16 in fp32 take as long as 64
        least = LEAST_CHUNK_KEYS // keys
        parts = chunk_parts(tiles, blocks, RT, keys)
        grid, slots = tiles * parts, tiles * parts
    split = few or parts > 1
    part_bytes = RT * (D + 2) * 4
    trips = -(-min(RT, R) * (D // 4) // 256)                    # of a join's workgroup over a part
    JK = min(JOIN_LOADS // min(2, trips), parts) if not few else JOIN_LOADS // min(2, trips)
    JU = max(1, min(JOIN_LOADS // JK, trips))
    DK, DV = -(-D // 32) * 32, -(-D // 16) * 16
    KP = DK + 8
    VP = DV + 16 if DV % 32 == 0 else DV        # an odd number of 32 bytes: see the transposing reads
    cs = n.attrs["scale"] * LOG2E
    fname = operator_name(g) + f"_{N}x{page}x{KV}"
    consts = dict(S=S, H=H, D=D, G=G, KV=KV, R=R, RT=RT, N=N, PAGE=page, P=P, L=L, BK=BK, BATCH=B, NQ=nq, PART_BYTES=part_bytes,
                  **(dict(GROUPS=grid, OVERHEAD=FEW_OVERHEAD) if few else dict(PARTS=parts)))
    if split:
        consts.update(JK=JK, JU=JU, WS_BYTES=slots * part_bytes)
    ints = dict(QT=QT, LEAST=least, KW=4 if few else 1, WINDOW=window)
    counted = len(n.inputs) > 5
    text = [f'extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu({1 if D > 128 and (f32 or few) else 2}))) '
            f"{fname}({g.params()}{', unsigned int* cnt_p, float* ws_p' if split else ''}) {{",
            "  constexpr unsigned int " + ", ".join(f"{k} = {v}u" for k, v in consts.items()) + ";",
            *([f"  constexpr float BY_JOIN = {FEW_BY_JOIN}f;"] if few else []),
            "  constexpr int " + ", ".join(f"{k} = {v}" for k, v in ints.items()) + ";",
            f"  typedef {_index_type(page * KV * D)} row_t;          // offsets within a page",
            *([f"  typedef {_index_type(2 * places)} pos_t;          // places in the list of all blocks"] if few else [])]
    if not f32:
        text.append(f"  constexpr unsigned int KP = {KP}u, VP = {VP}u; constexpr bool BF = {str(bf).lower()};")
    text += [f"  constexpr float CS = {cs!r}f, LOWEST = -3.402823466e+38f, SHIFT = {FP16_SHIFT if dt == DType.f16 else 0.0}f;",
             *(f"  const {T}* __restrict__ {nm} = {operand(g, i)};" for i, nm in enumerate(("q_p", "k_p", "v_p"))),
             f"  const int* __restrict__ pages_p = {operand(g, 3)};", f"  const int* __restrict__ starts_p = {operand(g, 4)};",
             "  const unsigned int tid = threadIdx.x, lane = tid % 64u, wave = __builtin_amdgcn_readfirstlane(tid / 64u);",
             "  const unsigned int r16 = lane % 16u, g16 = lane / 16u;",
             TILE,
             "  auto q_at = [&](unsigned int r) -> unsigned long { return (((unsigned long)b * S + r / G) * H + kvh * G + r % G) * D; };",
             "  auto finish = [&](unsigned int r, unsigned int d, tj_f32x4 acc, float l) {",
             "    int lo, hi;", "    const bool sees = bounds(r, lo, hi);",
             "    const float inv = l == 0.0f ? 0.0f : 1.0f / l;"]
    if f32:
        text += ["    tj_f32x4 y;", "    for (int e = 0; e < 4; ++e) y[e] = sees ? acc[e] * inv : 0.0f;",
                 "    *(tj_f32x4*)&out0_p[q_at(r) + d] = y;", "  };"]
    else:
        pack = "tj_f2bf2" if bf else "tj_f2h2"
        text += ["    tj_u32x2 y;", f"    y[0] = sees ? {pack}(acc[0] * inv, acc[1] * inv) : 0u;",
                 f"    y[1] = sees ? {pack}(acc[2] * inv, acc[3] * inv) : 0u;", "    *(tj_u32x2*)&out0_p[q_at(r) + d] = y;", "  };"]
    if f32:
        body = DIRECT32
        if few:
            body = "  __shared__ float rows[4][16 * D];\n  __shared__ float ml[4][16][2];\n" + body
            lds = "for (unsigned int u = 0; u < NV; ++u)\n      for (int i = 0; i < 4; ++i) {\n" \
                  "        const unsigned int d = u * 64u + g16 * 16u + i * 4u;\n        if (d >= D) continue;\n        tj_f32x4 w;\n" \
                  "        for (int j = 0; j < 4; ++j) w[j] = o[x][u * 4u + j][i];\n" \
                  "        *(tj_f32x4*)&rows[wave][r16 * D + d] = w;\n      }"
            body += _text(FEW_JOIN, ROWS_TO_LDS=lds, STORE_PART=STORE_FEW, SINGLE="parts == 1u").replace("WROWS(w)", "&rows[w][0]")
        else:
            begin = "for (unsigned int u = 0; u < NV; ++u)\n#pragma unroll\n    for (int i = 0; i < 4; ++i) {\n" \
                    "      const unsigned int d = u * 64u + g16 * 16u + i * 4u;\n      if (d >= D) continue;\n      tj_f32x4 acc;\n" \
                    "      for (int j = 0; j < 4; ++j) acc[j] = o[x][u * 4u + j][i];\n"
            body += _text(CHUNK_STORE, QUADS_BEGIN="#pragma unroll\n    " + begin, QUADS_END="}", STORE_PART=STORE_CHUNK if split else "", SINGLE="parts == 1u" if split else "true")
    else:
        body = FEW16 if few else CHUNK16
        if few:
            lds = "for (unsigned int u = 0; u < NU; ++u)\n      if (u * 16u + g16 * 4u < D) *(tj_f32x4*)((float*)&Vs[wave][0][0] + r16 * D + u * 16u + g16 * 4u) = o[x][u];"
            body += _text(FEW_JOIN, ROWS_TO_LDS=lds, STORE_PART=STORE_FEW, SINGLE="parts == 1u").replace("WROWS(w)", "(const float*)&Vs[w][0][0]")
        else:
            begin = "for (unsigned int u = 0; u < NU; ++u) {\n      const unsigned int d = u * 16u + g16 * 4u;\n" \
                    "      if (d >= D) continue;\n      const tj_f32x4 acc = o[x][u];\n"
            body += _text(CHUNK_STORE, QUADS_BEGIN="#pragma unroll\n    " + begin, QUADS_END="}", STORE_PART=STORE_CHUNK if split else "", SINGLE="parts == 1u" if split else "true")
            body = _text(body, QK_SCHED=_ahead(K_AHEAD, 1, DK // 32 * (BK // 16), QT), PV_SCHED=_ahead(V_AHEAD, 2, DV // 16 * (BK // 32), QT))
        load = "__builtin_nontemporal_load((const tj_u32x4*)" if _nt_loads(B * L * KV * D * 2 * dt.itemsize) else "*(const tj_u32x4*)("
        body = _text(body, OPV="tj_bf16x8" if bf else "tj_f16x8", PACK2="tj_f2bf2" if bf else "tj_f2h2",
                     PAIR_SUM="tj_pair_acc_bf16" if bf else "tj_pair_acc_f16", TO_FLOAT="tj_bf2f" if bf else "tj_h2f",
                     MFMA="__builtin_amdgcn_mfma_f32_16x16x32_" + ("bf16" if bf else "f16"),
                     WAVE_FENCE='__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier()')
        body = body.replace("TR_READ(", "__builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) tj_i16x4*)")
        body = body.replace("LOAD16(", load).replace(" T Vs[", f" {T} Vs[").replace(" T Ks[", f" {T} Ks[")
    if few:
        text.append(FEW_BEGIN)
    else:
        # the row tiles of one head and part run on one XCD (blockIdx % 8), whose L2 then serves its
        # keys once; the last rows, which see the most keys, begin first
        if B * KV * parts % XCDS == 0:
            text += [f"  const unsigned int grp = blockIdx.x / {XCDS * nq}u, rem = blockIdx.x % {XCDS * nq}u, vh = grp * {XCDS}u + rem % {XCDS}u;",
                     f"  const unsigned int qt = {nq - 1}u - rem / {XCDS}u;"]
        else:
            text.append(f"  const unsigned int vh = blockIdx.x / {nq}u, qt = {nq - 1}u - blockIdx.x % {nq}u;")
        text.append(CHUNK_BEGIN)
    text += [PART if split else "", _softmax(body), JOIN if split else "", FEW_END if few else CHUNK_END, "}"]
    source = "\n".join(text)
    for x in ("b", "x"):
        source = source.replace(f"COUNT({x})", f"(long){operand(g, 5)}[{x}]" if counted else "(long)S")
    meta = {"family": "paged_attention", "dtype": dt.value, "rows": R, "row_tile": RT, "keys_per_block": BK, "few": few,
            "parts": parts, "tiles": tiles}
    if split:
        meta["split_ws"] = (tiles * 4, slots * part_bytes)
    return HELPERS + QUAD_HELPERS + source, Launch(fname, (grid, 1, 1), (256, 1, 1), 0, meta)
