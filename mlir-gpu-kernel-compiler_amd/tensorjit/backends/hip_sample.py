"""Sampling one token per row of logits (``ir/operators.py``).

The tokens of a row that are kept form a prefix of their order (logit falling, index rising), held as
its last member: a value and the index behind the last kept token of that value.  ``top_k`` and
``top_p`` each move it: ``select`` finds the token at which the running weight (1, or the token's
mass) reaches a target, without sorting: a histogram of the weights over the distance from the
row's largest logit names the bucket, and the tokens of that bucket alone are ranked against each
other.  ``locate`` then walks the kept masses in index order.  Masses are integers (``2 ** 43`` for
the largest logit), so sums do not depend on their order and no two runs differ.  A sum of V masses is off by
V half steps, 2^-44 of the largest each (together 2^-28 of it for 2^16 tokens, 2^-24 for 2^20), and by the
exponential's 2^-38 of itself.
"""
from __future__ import annotations

import math

from ..runtime.autotune import CU_COUNT
from .hip_kernels import KernelGen, Launch
from .hip_operators import operand, operator_name
from .hip_prelude import CTYPE, vec_width

THREADS = 1024
SPLIT_SWEEPS, LONG_SWEEPS = 4, 12   # rows that are split: see slices()
MAX_SLICES = 64     # of a row: a wave combines them
MAX_SPLIT_ROWS = 4096   # 33 KB of workspace each, 135 MB
HELD_LOGITS = 16    # a lane's part of a slice that stays in registers

HELPERS = r"""#ifndef TJ_SAMPLE
#define TJ_SAMPLE
typedef unsigned long tj_u64;
#define TJ_WAVE_SYNC __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier()
// a key that orders as its value does; -0 and 0 have one
__device__ __forceinline__ unsigned int tj_key(float x) {
  const unsigned int u = __builtin_bit_cast(unsigned int, x + 0.0f);
  return u ^ ((unsigned int)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float tj_unkey(unsigned int k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ tj_u64 tj_shfl(tj_u64 v, int lane) {
  const unsigned int lo = __builtin_amdgcn_ds_bpermute(lane * 4, (int)(unsigned int)v);
  const unsigned int hi = __builtin_amdgcn_ds_bpermute(lane * 4, (int)(unsigned int)(v >> 32));
  return (tj_u64)hi << 32 | lo;
}
// the value of lane l, the same for the whole wave
__device__ __forceinline__ tj_u64 tj_lane(tj_u64 v, int l) {
  return (tj_u64)(unsigned int)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (unsigned int)__builtin_amdgcn_readlane((int)v, l);
}
// the value of the lane that C names, of the rows (16 lanes) of mask M; 0 where there is none
template <int C, int M> __device__ __forceinline__ tj_u64 tj_dpp(tj_u64 v) {
  const unsigned int lo = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)(unsigned int)v, C, M, 0xf, false);
  return (tj_u64)(unsigned int)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), C, M, 0xf, false) << 32 | lo;
}
// inclusive sums over the lanes 0 .. l of the wave; every lane is active
__device__ __forceinline__ tj_u64 tj_wave_scan(tj_u64 v) {
  v += tj_dpp<0x111, 0xf>(v);      // from 1, 2, 4, 8 lanes before in the row
  v += tj_dpp<0x112, 0xf>(v);
  v += tj_dpp<0x114, 0xf>(v);
  v += tj_dpp<0x118, 0xf>(v);
  v += tj_dpp<0x142, 0xa>(v);      // rows 1 and 3: the last lane of the row before
  return v + tj_dpp<0x143, 0xc>(v);      // rows 2 and 3: lane 31
}

// a token as a number that falls in the tokens' order (an index is under 2^32 - 1, so none is 0)
__device__ __forceinline__ tj_u64 tj_entry(float v, unsigned int i) { return (tj_u64)tj_key(v) << 32 | ~i; }
__device__ __forceinline__ float tj_entry_value(tj_u64 e) { return tj_unkey((unsigned int)(e >> 32)); }
__device__ __forceinline__ unsigned int tj_entry_index(tj_u64 e) { return ~(unsigned int)e; }

struct tj_sample_shared {
  static constexpr unsigned int TH = 1024, NB = 2048, LIST = 1024, SEG = TH / 64;
  tj_u64 hist[NB], seg[SEG], weight[LIST], wave[TH / 64];
  tj_u64 list[LIST];             // tokens as tj_entry
  float fmax[TH / 64], fmin[TH / 64], tv;
  unsigned int count, bucket, ti;
  tj_u64 before;
};

// Everything is inlined into the kernel: a function of its own would get registers of its own, and a
// workgroup of 1024 lanes has 128 for each.
// SW sweeps of the row, from `from` on; HELD: they stay in registers, loaded at once.
template <typename T, unsigned int V, unsigned int SW, bool HELD> struct tj_sampler {
  typedef tj_sample_shared Shared;
  static constexpr unsigned int TH = 1024, VEC = V < 16 / sizeof(T) ? 1 : 16 / sizeof(T);
  static constexpr unsigned int NB = Shared::NB, LIST = Shared::LIST, FEW = 256, SEG = Shared::SEG;
  // sweeps in flight together: where much is computed for each logit, and where little is
  static constexpr unsigned int LONG = VEC > 4u ? 1 : 2, SHORT = 4;
  Shared& sh;
  const T* __restrict__ x;
  const unsigned int tid;
  unsigned int from;
  float top, inv;   // largest logit, buckets per unit of logit
  double rate, shift;       // log2(e) / temperature, and -top times that
  float tv;                 // kept: values above tv, and those equal to it at indices below ti
  unsigned int ti;
  tj_u32x4 held[HELD ? SW : 1u];

  __device__ __forceinline__ tj_sampler(Shared& s, const T* p, unsigned int first) : sh(s), x(p), tid(threadIdx.x), from(first) {
    if (HELD) fetch<SW>(0u, held);
  }
  // each wave has consecutive chunks: its share of the row is a segment of it
  __device__ __forceinline__ unsigned int chunk(unsigned int s) const { return from * TH + tid / 64u * (SW * 64u) + s * 64u + tid % 64u; }

  // Chunk c holds the logits c VEC .. c VEC + VEC - 1.  The last one is read from VEC before the row's
  // end, whatever its length, and chunks past it too: what belongs to an earlier chunk is -inf.
  __device__ __forceinline__ unsigned int base(unsigned int c) const { return c < V / VEC ? c * VEC : V - VEC; }
  template <unsigned int U> __device__ __forceinline__ void fetch(unsigned int s, tj_u32x4* r) const {
#pragma unroll
    for (unsigned int k = 0; k < U; ++k) {
      const unsigned int i = base(chunk(s + k));
      if (VEC == 1) r[k][0] = __builtin_bit_cast(unsigned int, tj_ld(x[i]));
      else r[k] = *(const tj_u32x4a2*)(x + i);
    }
  }
  __device__ __forceinline__ void unpack(tj_u32x4 r, unsigned int c, float* v) const {
    if (VEC == 1) v[0] = __builtin_bit_cast(float, (unsigned int)r[0]);
    else tj_unpackv(r, (const T*)nullptr, v);
    const unsigned int i = base(c);
    if (i != c * VEC) {
#pragma unroll
      for (unsigned int e = 0; e < VEC; ++e) v[e] = i + e < c * VEC ? -__builtin_inff() : v[e];
    }
  }
  // f(values, index of the first) for each of this thread's chunks, in order, M of them while the
  // next M are on their way
  template <unsigned int M, typename F> __device__ __forceinline__ void sweep(F f) const {
    if (HELD) {
#pragma unroll
      for (unsigned int k = 0; k < SW; ++k) {
        float v[VEC];
        unpack(held[k], chunk(k), v);
        f(v, base(chunk(k)));
      }
      return;
    }
    constexpr unsigned int U = SW < M ? SW : M;
    tj_u32x4 r[U], next[U];
    fetch<U>(0u, next);
#pragma unroll 1
    for (unsigned int s = 0; s < SW; s += U) {
#pragma unroll
      for (unsigned int k = 0; k < U; ++k) r[k] = next[k];
      if (s + U < SW) fetch<U>(s + U, next);
#pragma unroll
      for (unsigned int k = 0; k < U; ++k) {
        if (s + k >= SW) break;
        float v[VEC];
        unpack(r[k], chunk(s + k), v);
        f(v, base(chunk(s + k)));
      }
    }
  }
  // exp((v - top) / temperature) in steps of 2^-43, to the nearest, and exactly 2^43 for v = top.  In
  // fp64, which costs as much per operation as fp32 here: a mass off by 2^-24 would move a border
  // between two tokens often enough to see (10^4 tokens: one row in 10^4).  2^y = 2^n 2^f, the latter 1 + f
  // times the polynomial that interpolates (2^f - 1) / f at the 8 Chebyshev points of |f| <= 1/2
  // (relative error under 2^-38; y itself is off by 2^-53 of top / temperature, as in any 64-bit form).
  __device__ __forceinline__ tj_u64 mass(float v) const {
    const double y = __builtin_fmax(__builtin_fma((double)v, rate, shift), -100.0);
    const double n = __builtin_rint(y), f = y - n;
    double p = 1.325080551750225e-06;
    p = __builtin_fma(p, f, 1.5303700711365693e-05);
    p = __builtin_fma(p, f, 0.00015403475186530786);
    p = __builtin_fma(p, f, 0.0013333478473685416);
    p = __builtin_fma(p, f, 0.00961812913523614);
    p = __builtin_fma(p, f, 0.055504109063258665);
    p = __builtin_fma(p, f, 0.24022650695888503);
    p = __builtin_fma(p, f, 0.6931471805568324);
    p = __builtin_fma(p, f, 1.0);
    const double w = __builtin_ldexp(p, 43 + (int)n) + 4503599627370496.0;    // 2^52: the fraction is rounded off
    return v == top ? 1ul << 43 : __builtin_bit_cast(tj_u64, w) & 0xffffffffffffful;
  }
  __device__ __forceinline__ unsigned int bucket(float v) const {
    const float d = v == top ? 0.0f : top - v;
    return (unsigned int)fminf(d * inv, (float)(NB - 1u));
  }
  __device__ __forceinline__ bool kept(float v, unsigned int i) const { return v > tv || (v == tv && i < ti); }

  // sums of v over the threads before this one; `all` gets the sum over every thread
  __device__ __forceinline__ tj_u64 scan(tj_u64 v, tj_u64& all) const {
    const tj_u64 mine = tj_wave_scan(v);
    __syncthreads();
    if (tid % 64u == 63u) sh.wave[tid / 64u] = mine;
    __syncthreads();
    tj_u64 before = 0ul;
    all = 0ul;
    for (unsigned int w = 0; w < TH / 64; ++w) {
      before += w < tid / 64u ? sh.wave[w] : 0ul;
      all += sh.wave[w];
    }
    return before + mine - v;
  }

  // largest and smallest logit (-inf, inf: none); NaN logits lose every comparison, here and later
  __device__ __forceinline__ void extremes(float& hi, float& lo) {
    hi = -__builtin_inff();
    lo = __builtin_inff();
    sweep<SHORT>([&](const float* v, unsigned int) {
#pragma unroll
      for (unsigned int e = 0; e < VEC; ++e) {
        hi = v[e] > hi ? v[e] : hi;
        lo = v[e] < lo && v[e] > -__builtin_inff() ? v[e] : lo;
      }
    });
    hi = tj_wave_max(hi);
    lo = -tj_wave_max(-lo);
    if (tid % 64u == 0u) { sh.fmax[tid / 64u] = hi; sh.fmin[tid / 64u] = lo; }
    __syncthreads();
    for (unsigned int w = 0; w < TH / 64; ++w) { hi = fmaxf(hi, sh.fmax[w]); lo = fminf(lo, sh.fmin[w]); }
  }
  // what the other steps need of them
  __device__ __forceinline__ void begin(float hi, float lo, float temp) {
    top = hi;
    tv = -__builtin_inff();
    ti = 0u;
    rate = 1.4426950408889634 / (double)temp;      // up to 2^150, in range; not used at 0 and below
    shift = -(double)hi * rate;
    // the buckets cover what has a mass (45 halvings), or the row where that is less
    inv = (float)NB / fmaxf(fminf(45.0f / (float)rate, hi - lo), 1e-30f);
  }

  // the weights of each wave's segment, in sh.seg
  template <typename W> __device__ __forceinline__ void segments(W weight) {
    tj_u64 sum = 0ul;
    sweep<LONG>([&](const float* v, unsigned int i) {
#pragma unroll
      for (unsigned int e = 0; e < VEC; ++e) sum += weight(v[e], i + e);
    });
    sum = tj_wave_scan(sum);
    if (tid % 64u == 63u) sh.seg[tid / 64u] = sum;
    __syncthreads();
  }
  // The same of the kept tokens' masses where few are kept: a wave gathers them, in the list's place,
  // and computes 64 masses at a time.
  __device__ __forceinline__ void sparse_segments(double least) {
    float* mine = (float*)sh.list + tid / 64u * 128u;           // 2048 words, 128 a wave
    const unsigned int lane = tid % 64u;
    unsigned int n = 0u;
    tj_u64 sum = 0ul;
    auto flush = [&](unsigned int m) {
      TJ_WAVE_SYNC;
      const tj_u64 w = lane < m ? mass(mine[lane]) : 0ul;
      sum += (double)w < least ? 0ul : w;
      const float rest = mine[64u + lane];
      TJ_WAVE_SYNC;
      mine[lane] = rest;
    };
    sweep<LONG>([&](const float* v, unsigned int i) {
#pragma unroll
      for (unsigned int e = 0; e < VEC; ++e) {
        const bool in = kept(v[e], i + e);
        const tj_u64 all = __builtin_amdgcn_ballot_w64(in);
        if (all == 0ul) continue;
        const unsigned int at = n + __builtin_amdgcn_mbcnt_hi((unsigned int)(all >> 32), __builtin_amdgcn_mbcnt_lo((unsigned int)all, 0u));
        if (in) mine[at] = v[e];
        n += (unsigned int)__builtin_popcountl(all);
        if (n >= 64u) { flush(64u); n -= 64u; }
      }
    });
    flush(n);
    sum = tj_wave_scan(sum);
    if (lane == 63u) sh.seg[tid / 64u] = sum;
    __syncthreads();
  }
  // index of the token at which the running weight, in index order, passes target(total)
  template <typename W, typename G> __device__ __forceinline__ unsigned int locate(W weight, G target) {
    segments(weight);
    tj_u64 all = 0ul, before = 0ul;
    for (unsigned int g = 0; g < SEG; ++g) all += sh.seg[g];
    const tj_u64 want = target(all);
    unsigned int g = 0u;
    while (before + sh.seg[g] <= want) before += sh.seg[g++];
    return within(weight, want, g, before);
  }
  // the same within segment g, before which the running weight is `before`
  template <typename W> __device__ __forceinline__ unsigned int within(W weight, tj_u64 want, unsigned int g, tj_u64 before) {
    if (tid < 64u) {
#pragma unroll 1
      for (unsigned int s = 0; s < SW; ++s) {
        const unsigned int c = from * TH + g * (SW * 64u) + s * 64u + tid, i = base(c);
        tj_u64 w[VEC], sum = 0ul;
        float v[VEC];
        tj_u32x4 r;
        if (VEC == 1) r[0] = __builtin_bit_cast(unsigned int, tj_ld(x[i]));
        else r = *(const tj_u32x4a2*)(x + i);
        unpack(r, c, v);
#pragma unroll
        for (unsigned int e = 0; e < VEC; ++e) sum += w[e] = weight(v[e], i + e);
        const tj_u64 upto = before + tj_wave_scan(sum);
        if (tj_shfl(upto, 63) <= want) {
          before = tj_shfl(upto, 63);
          continue;
        }
        tj_u64 at = upto - sum;
#pragma unroll
        for (unsigned int e = 0; e < VEC; ++e) {
          if (at <= want && want < at + w[e]) sh.ti = i + e;
          at += w[e];
        }
        break;
      }
    }
    __syncthreads();
    return sh.ti;
  }

  // the kept tokens' weights by bucket, in sh.hist
  template <bool ALL, typename W> __device__ __forceinline__ void histogram(W weight) {     // ALL: nothing is cut off yet
    for (unsigned int b = tid; b < NB; b += TH) sh.hist[b] = 0ul;
    __syncthreads();
    sweep<LONG>([&](const float* v, unsigned int i) {
#pragma unroll
      for (unsigned int e = 0; e < VEC; ++e) {
        if (ALL ? v[e] > -__builtin_inff() : kept(v[e], i + e)) atomicAdd(&sh.hist[bucket(v[e])], weight(v[e]));
      }
    });
    __syncthreads();
  }
  // The bucket at which the running weight, in order, reaches want = target(total) (>= 1): sh.bucket, and
  // sh.before for the weight before it.  False where it never does.  The list is empty then.
  template <typename G> __device__ __forceinline__ bool border(G target, tj_u64& want) {
    constexpr unsigned int PER = NB / TH;
    tj_u64 own = 0ul, all;
#pragma unroll
    for (unsigned int k = 0; k < PER; ++k) own += sh.hist[tid * PER + k];
    tj_u64 before = scan(own, all);
    want = target(all);
    if (tid == 0u) sh.count = 0u;
    if (want > all) return false;
    if (before < want && want <= before + own) {
      unsigned int b = tid * PER;
      while (before + sh.hist[b] < want) before += sh.hist[b++];
      sh.bucket = b;
      sh.before = before;
    }
    __syncthreads();
    return true;
  }
  // the kept tokens of the buckets lo .. hi into the list (what fits); sh.count is their number
  __device__ __forceinline__ void collect(unsigned int lo, unsigned int hi) {
    // most tokens fail a comparison with the buckets' edges, and one bucket more for their rounding
    const float edge = hi + 1u < NB ? top - (float)(hi + 2u) / inv : -__builtin_inff();
    const float rim = lo > 1u ? top - (float)(lo - 1u) / inv : __builtin_inff();
    sweep<SHORT>([&](const float* v, unsigned int i) {
#pragma unroll
      for (unsigned int e = 0; e < VEC; ++e) {
        if (!(v[e] >= edge && v[e] <= rim) || !kept(v[e], i + e)) continue;
        const unsigned int b = bucket(v[e]);
        if (b < lo || b > hi) continue;
        const unsigned int at = atomicAdd(&sh.count, 1u);
        if (at < LIST) sh.list[at] = tj_entry(v[e], i + e);
      }
    });
    __syncthreads();
  }

  // the same, where the bucket's n tokens are in the list and the running weight before them is `before`
  template <typename W> __device__ __forceinline__ void cut_list(W weight, tj_u64 want, tj_u64 before, unsigned int n) {
    const tj_u64 mine = tid < n ? sh.list[tid] : 0ul;
    const float v = tj_entry_value(mine);
    const tj_u64 w = tid < n ? weight(v) : 0ul;
    sh.list[tid] = mine;
    sh.weight[tid] = w;
    __syncthreads();
    if (tid < n) {
      tj_u64 at = before;
#pragma unroll 1
      for (unsigned int k0 = 0; k0 < n; k0 += 8u) {            // past the n-th: no weight
#pragma unroll
        for (unsigned int k = k0; k < k0 + 8u; ++k) {
          const tj_u64 e = sh.list[k], we = sh.weight[k];
          at += e > mine ? we : 0ul;
        }
      }
      if (at < want && want <= at + w) { sh.tv = v; sh.ti = tj_entry_index(mine) + 1u; }
    }
    __syncthreads();
    tv = sh.tv;
    ti = sh.ti;
  }
  // keep the tokens, in order, up to the one at which the running weight reaches `want`, in the border's bucket
  template <typename W> __device__ __forceinline__ void cut(W weight, tj_u64 want) {
    const unsigned int b = sh.bucket;
    tj_u64 before = sh.before;
    collect(b, b);
    const unsigned int n = sh.count;
    if (n <= LIST) return cut_list(weight, want, before, n);
    // a bucket of many tokens: its keys digit by digit, then the indices of the equal ones
    unsigned int key = 0u;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256u) sh.hist[tid] = 0ul;
      __syncthreads();
      sweep<LONG>([&](const float* v, unsigned int i) {
#pragma unroll
        for (unsigned int e = 0; e < VEC; ++e) {
          const unsigned int k = tj_key(v[e]);
          if (!kept(v[e], i + e) || bucket(v[e]) != b || ((tj_u64)(k ^ key) >> (shift + 8))) continue;
          const tj_u64 w = weight(v[e]);
          if (w) atomicAdd(&sh.hist[k >> shift & 255u], w);
        }
      });
      __syncthreads();
      unsigned int d = 255u;
      while (d > 0u && before + sh.hist[d] < want) before += sh.hist[d--];
      key |= d << shift;
    }
    const float v = tj_unkey(key);
    const tj_u64 w = weight(v), nth = (want - before + w - 1ul) / w;
    const tj_sampler& me = *this;
    __syncthreads();
    const unsigned int last = locate([&](float y, unsigned int i) -> tj_u64 { return y == v && me.kept(y, i) ? 1ul : 0ul; },
                                     [&](tj_u64) -> tj_u64 { return nth - 1ul; });
    tv = v;
    ti = last + 1u;
  }

  // The token among the list's n <= FEW, of which the first `want` in order are kept, by their masses.
  // Each wave compares 16 entries, as scalars, with all of them: reading both sides of n^2 comparisons
  // from LDS takes twice as long (192 entries: 15 thousand cycles / 7).
  template <typename G> __device__ __forceinline__ int among(unsigned int n, tj_u64 want, G target, double least, double part) {
    const unsigned int lane = tid % 64u, k0 = tid / 64u * 16u;
    unsigned int *in_order = (unsigned int*)sh.hist, *by_index = in_order + FEW;     // entries that precede each
    tj_u64* upto = sh.hist + FEW;
    if (tid >= n && tid < FEW) sh.list[tid] = 0ul;
    if (tid < 2u * FEW) in_order[tid] = 0u;
    __syncthreads();
    if (k0 < n) {
      const tj_u64 own = sh.list[k0 + lane % 16u];
#pragma unroll 1
      for (unsigned int m = lane; m - lane < n; m += 64u) {
        const tj_u64 e = sh.list[m];
        unsigned int above = 0u, before = 0u;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const tj_u64 other = tj_lane(own, k);
          above += other > e ? 1u : 0u;
          before += (unsigned int)other > (unsigned int)e ? 1u : 0u;
        }
        atomicAdd(&in_order[m], above);
        atomicAdd(&by_index[m], before);
      }
    }
    __syncthreads();
    const tj_u64 e = sh.list[tid % FEW];
    const unsigned int rank = in_order[tid % FEW], place = by_index[tid % FEW];
    if (tid < n) sh.weight[rank] = rank < want ? mass(tj_entry_value(e)) : 0ul;
    __syncthreads();
    tj_u64 all, w = tid < n ? sh.weight[tid] : 0ul;
    const tj_u64 before = scan(w, all);
    if (tid < n && (before >= target(all) || (double)w < least)) sh.weight[tid] = 0ul;
    __syncthreads();
    w = tid < n ? sh.weight[rank] : 0ul;
    if (tid < n) upto[place] = w;
    __syncthreads();
    const tj_u64 mine = tid < n ? upto[tid] : 0ul, at = scan(mine, all);
    if (tid < n) upto[tid] = at;
    __syncthreads();
    const tj_u64 pick = (tj_u64)(part * (double)all), from_it = upto[place % FEW];
    if (tid < n && from_it <= pick && pick < from_it + w) sh.ti = tj_entry_index(e);
    __syncthreads();
    return (int)sh.ti;
  }

  // the mass up to which tokens, in order, are kept; and the least one that is
  static __device__ __forceinline__ tj_u64 nucleus_of(float top_p, tj_u64 all) {
    if (!(top_p < 1.0f)) return ~0ul;
    const double t = __builtin_ceil((double)top_p * (double)all);
    return t >= 1.0 ? (tj_u64)t : 1ul;
  }
  static __device__ __forceinline__ double least_of(float min_p) {
    return min_p > 0.0f ? (double)fminf(min_p, 1.0f) * 8796093022208.0 : 0.0;
  }
  static __device__ __forceinline__ double part_of(float u) { return u > 0.0f ? (double)fminf(u, 0.99999994f) : 0.0; }

  // Filters by top_k (`by_count`) and the nucleus, with the histogram of the first of them that is on in
  // sh.hist: the token where few are left, else -1, and the cut in tv and ti.  LATER: -2 where few are
  // left, the buckets 0 .. sh.bucket, which others collect.
  template <bool LATER> __device__ __forceinline__ int filter(float u, int top_k, float top_p, float min_p, bool by_count) {
    const tj_sampler& me = *this;
    auto one = [](float) -> tj_u64 { return 1ul; };
    auto weight = [&](float v) -> tj_u64 { return me.mass(v); };
    auto nucleus = [&](tj_u64 all) -> tj_u64 { return nucleus_of(top_p, all); };
    tj_u64 want;
    if (by_count) {
      if (border([&](tj_u64) -> tj_u64 { return (tj_u64)top_k; }, want)) {
        const unsigned int n = (unsigned int)(sh.before + sh.hist[sh.bucket]);
        if (n <= FEW) {
          if (LATER) return -2;
          collect(0u, sh.bucket);
          return among(n, want, nucleus, least_of(min_p), part_of(u));
        }
        cut(one, want);
      }
      if (!(top_p < 1.0f)) return -1;
      __syncthreads();
      histogram<false>(weight);
    }
    if (border(nucleus, want)) cut(weight, want);
    return -1;
  }

  // a row that is this workgroup's alone; top_k <= 0 and !(top_p < 1): off
  __device__ __forceinline__ int run(float u, float temp, int top_k, float top_p, float min_p) {
    float hi, lo;
    extremes(hi, lo);
    if (!(hi > -__builtin_inff())) return -1;
    begin(hi, lo, temp);
    const tj_sampler& me = *this;
    if (!(temp > 0.0f))
      return (int)locate([&](float v, unsigned int) -> tj_u64 { return v == me.top ? 1ul : 0ul; },
                         [](tj_u64) -> tj_u64 { return 0ul; });
    const bool by_count = top_k > 0 && (unsigned int)top_k < V;
    if (by_count || top_p < 1.0f) {
      if (by_count) histogram<true>([](float) -> tj_u64 { return 1ul; });
      else histogram<true>([&](float v) -> tj_u64 { return me.mass(v); });
      const int token = filter<false>(u, top_k, top_p, min_p, by_count);
      if (token >= 0) return token;
    }
    const double least = least_of(min_p), part = part_of(u);
    return (int)locate([&](float v, unsigned int i) -> tj_u64 {
      if (!me.kept(v, i)) return 0ul;
      const tj_u64 w = me.mass(v);
      return (double)w < least ? 0ul : w;
    }, [&](tj_u64 all) -> tj_u64 { return (tj_u64)(part * (double)all); });
  }
};

// Rows split over workgroups: SL slices of N sweeps, in three launches.
//   a: each slice's largest and smallest logit
//   b: each slice's histogram (counts for top-k, masses for the nucleus); the row's last workgroup
//      adds them and finds the border's bucket.  Where few tokens are left the slices collect them in
//      launch c; else it decides between the tokens of that bucket, over the whole row
//   c: each slice's tokens, or its kept mass; the row's last workgroup finds the token
// What one launch leaves for the next lies in the row's state; what workgroups of one launch
// exchange is agent-coherent.
struct tj_sample_state {
  unsigned int mode, ti;
  float tv;
  unsigned int bucket;
};
enum { TJ_ALL = 0, TJ_LIST = 1, TJ_CUT = 2 };      // kept: all tokens; top_k of those up to bucket; tv and ti

template <typename T, unsigned int V, unsigned int N, unsigned int SL, bool HELD> struct tj_sample_split {
  typedef tj_sampler<T, V, N, HELD> Slice;
  typedef tj_sampler<T, V, N * SL, false> Row;
  static constexpr unsigned int TH = 1024, NB = Slice::NB, SEG = Slice::SEG;
  tj_sample_state* st;
  tj_u64 *ext, *hist, *total, *seg;
  unsigned int* cnt;
  unsigned int slice;

  static constexpr unsigned int BYTES = sizeof(tj_sample_state) + 8u * SL * (1u + NB + 1u + SEG);
  __device__ __forceinline__ tj_sample_split(void* ws, unsigned int* c, unsigned int row, unsigned int s) : slice(s) {
    char* p = (char*)ws + (unsigned long)row * BYTES;
    st = (tj_sample_state*)p;
    ext = (tj_u64*)(p + sizeof(tj_sample_state));
    hist = ext + SL;
    total = hist + SL * NB;
    seg = total + SL;
    cnt = c + row;
  }
  static __device__ __forceinline__ void put(tj_u64* p, tj_u64 v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
  static __device__ __forceinline__ tj_u64 get(const tj_u64* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
  // true in the row's workgroup that comes here last, for all its lanes; the counter wraps to zero
  __device__ __forceinline__ bool last() {
    __builtin_amdgcn_s_waitcnt(0x0F70);       // vmcnt(0): this wave's stores are done
    __shared__ unsigned int is_last;
    __syncthreads();
    if (threadIdx.x == 0u) is_last = atomicInc(cnt, SL - 1u) == SL - 1u ? 1u : 0u;
    __syncthreads();
    return is_last != 0u;
  }
  // the row's extremes, from its slices'
  __device__ __forceinline__ void extremes(float& hi, float& lo) const {
    const unsigned int lane = threadIdx.x % 64u;
    const tj_u64 e = lane < SL ? ext[lane] : 0x7f800000ff800000ul;       // inf, -inf
    hi = tj_wave_max(__builtin_bit_cast(float, (unsigned int)e));
    lo = -tj_wave_max(-__builtin_bit_cast(float, (unsigned int)(e >> 32)));
  }
  static __device__ __forceinline__ bool by_count(float temp, int top_k) { return temp > 0.0f && top_k > 0 && (unsigned int)top_k < V; }
  static __device__ __forceinline__ bool by_mass(float temp, int top_k, float top_p) {
    return temp > 0.0f && !by_count(temp, top_k) && top_p < 1.0f;
  }

  __device__ __forceinline__ void a(Slice& s) {
    float hi, lo;
    s.extremes(hi, lo);
    if (threadIdx.x == 0u) ext[slice] = (tj_u64)__builtin_bit_cast(unsigned int, lo) << 32 | __builtin_bit_cast(unsigned int, hi);
  }
  __device__ __forceinline__ void b(Slice& s, float u, float temp, int top_k, float top_p, float min_p) {
    const unsigned int tid = threadIdx.x;
    const bool count = by_count(temp, top_k), mass = by_mass(temp, top_k, top_p);
    float hi, lo;
    extremes(hi, lo);
    if (!(hi > -__builtin_inff()) || !(count || mass)) {
      if (slice == 0u && tid == 0u) st->mode = TJ_ALL;
      return;
    }
    s.begin(hi, lo, temp);
    if (count) s.template histogram<true>([](float) -> tj_u64 { return 1ul; });
    else s.template histogram<true>([&](float v) -> tj_u64 { return s.mass(v); });
    for (unsigned int k = tid; k < NB; k += TH) put(&hist[slice * NB + k], s.sh.hist[k]);
    if (!last()) return;
    for (unsigned int k = tid; k < NB; k += TH) {
      tj_u64 sum = 0ul;
#pragma unroll 8
      for (unsigned int j = 0; j < SL; ++j) sum += get(&hist[j * NB + k]);
      s.sh.hist[k] = sum;
    }
    __syncthreads();
    Row r(s.sh, s.x, 0u);
    r.begin(hi, lo, temp);
    const int token = r.template filter<true>(u, top_k, top_p, min_p, count);
    if (tid == 0u) {
      st->tv = r.tv;
      st->ti = r.ti;
      st->bucket = s.sh.bucket;
      st->mode = token == -2 ? TJ_LIST : TJ_CUT;
    }
  }
  // the row's tokens up to a bucket, FEW at most: each slice's, in its histogram's place, then all of them
  __device__ __forceinline__ int list(Slice& s, unsigned int bucket, float u, unsigned int top_k, float top_p, float min_p) {
    const unsigned int tid = threadIdx.x;
    if (tid == 0u) s.sh.count = 0u;
    __syncthreads();
    s.collect(0u, bucket);
    const unsigned int n = s.sh.count;
    if (tid < n) put(&hist[slice * NB + tid], s.sh.list[tid]);
    if (tid == 0u) put(&total[slice], n);
    if (!last()) return -1;
    if (tid < 64u) {
      const tj_u64 own = tid < SL ? get(&total[tid]) : 0ul, upto = tj_wave_scan(own);
      s.sh.hist[tid] = upto - own;
      if (tid == 63u) s.sh.count = (unsigned int)upto;
    }
    __syncthreads();
    const unsigned int all = s.sh.count;
    if (tid < all) {
      unsigned int j = 0u;                   // the slice of entry tid
      for (unsigned int k = 32u; k > 0u; k /= 2u) j += s.sh.hist[j + k] <= tid ? k : 0u;
      s.sh.list[tid] = get(&hist[j * NB + tid - (unsigned int)s.sh.hist[j]]);
    }
    __syncthreads();
    return s.among(all, top_k, [&](tj_u64 mass) -> tj_u64 { return Slice::nucleus_of(top_p, mass); }, Slice::least_of(min_p), Slice::part_of(u));
  }
  // `filtered`: launch b came before
  __device__ __forceinline__ void c(Slice& s, bool filtered, float u, float temp, int top_k, float top_p, float min_p, int* out) {
    const unsigned int tid = threadIdx.x, mode = filtered ? st->mode : TJ_ALL;
    float hi, lo;
    extremes(hi, lo);
    if (!(hi > -__builtin_inff())) {
      if (slice == 0u && tid == 0u) *out = -1;
      return;
    }
    s.begin(hi, lo, temp);
    if (mode == TJ_LIST) {
      const int token = list(s, st->bucket, u, (unsigned int)top_k, top_p, min_p);
      if (token >= 0 && tid == 0u) *out = token;
      return;
    }
    if (mode == TJ_CUT) { s.tv = st->tv; s.ti = st->ti; }
    const bool greedy = !(temp > 0.0f);
    const double least = Slice::least_of(min_p), part = Slice::part_of(u);
    auto weight = [&](float v, unsigned int i) -> tj_u64 {
      if (greedy) return v == hi ? 1ul : 0ul;
      if (!s.kept(v, i)) return 0ul;
      const tj_u64 w = s.mass(v);
      return (double)w < least ? 0ul : w;
    };
    if (mode == TJ_CUT) s.sparse_segments(least);
    else s.segments(weight);
    if (tid < 64u) {
      if (tid < SEG) put(&seg[slice * SEG + tid], s.sh.seg[tid]);
      const tj_u64 sum = tj_wave_scan(tid < SEG ? s.sh.seg[tid] : 0ul);
      if (tid == 63u) put(&total[slice], sum);
    }
    if (!last()) return;
    // one wave: the slice, its segment, then the token
    if (tid < 64u) {
      tj_u64 own = tid < SL ? get(&total[tid]) : 0ul, upto = tj_wave_scan(own);
      const tj_u64 all = tj_shfl(upto, 63), want = greedy ? 0ul : (tj_u64)(part * (double)all);
      const unsigned int from = __builtin_ctzl(__builtin_amdgcn_ballot_w64(upto > want));
      const tj_u64 before = tj_shfl(upto - own, (int)from);
      own = tid < SEG ? get(&seg[from * SEG + tid]) : 0ul;
      upto = before + tj_wave_scan(own);
      const unsigned int g = __builtin_ctzl(__builtin_amdgcn_ballot_w64(upto > want));
      upto = tj_shfl(upto - own, (int)g);
      s.from = from * N;
      if (tid == 0u) { s.sh.bucket = g; s.sh.before = upto; s.sh.wave[0] = want; }
    }
    __syncthreads();
    const unsigned int token = s.within(weight, s.sh.wave[0], s.sh.bucket, s.sh.before);
    if (tid == 0u) *out = (int)token;
  }
};
#endif
"""


def sweeps_of(V: int, vec: int) -> int:
    return -(-(-(-V // (1 if V < vec else vec))) // THREADS)


def slices(rows: int, sweeps: int, top_k: bool) -> tuple[int, int]:
    """(slices of a row, sweeps of a slice); one slice: the row is a single workgroup's, in one launch.

    Splitting takes up to two launches more; those of histograms and of masses are joined by a row's last
    workgroup.  us, split / one workgroup
    per row: without top-k (masses of every logit) bf16 1 x 32000 19 / 23, 1 x 128000 30 / 73, 64 x 32000
    26 / 34, 64 x 128000 52 / 113, 384 x 128000 162 / 205, 2048 x 128000 721 / 826, fp32 128 x 50257 44 / 55, 300 x 100000
    148 / 178, but 256 x 20000 48 / 31.  Past 128 rows fp32 gains nothing where the rows alone fill the CUs evenly: 512 x 100000
    206 / 204, 1024 x 100000 388 / 385, and 50257 loses, 256 rows 69 / 61, 512 120 / 114, 1024 214 / 207, 4096 862 / 777;
    300 x 100000 in three slices took 140.  With top-k (counts, then
    few masses) bf16 1 x 128000 22 / 37, fp32 16 x 50257 22 / 23, 64 x 100003 32 / 47, 128 x 100003 48 / 51, but 64 x 32000
    24 / 18.  A workgroup for each CU: 256, 512, 768 of them 32, 38, 39 (64 x 100003, top-k); a slice
    of 1, 2, 4 sweeps 25, 22, 23 (16 x 50257, top-k) and 30, 32, 37 (1 x 128000, no top-k)."""
    if sweeps < (LONG_SWEEPS if top_k else SPLIT_SWEEPS) or rows > (128 if top_k or sweeps < LONG_SWEEPS else MAX_SPLIT_ROWS):
        return 1, sweeps
    per = max(2 if top_k else 1, -(-sweeps // min(MAX_SLICES, max(2, CU_COUNT // rows))))
    return -(-sweeps // per), per


def gen_sample(g: KernelGen):
    """A workgroup per row, or a row split over workgroups; see the module's docstring for the method."""
    n = g.k.anchor
    x = n.inputs[0]
    V, R = x.shape[-1], math.prod(x.shape[:-1])
    T, item = CTYPE[x.dtype], x.dtype.itemsize
    fname = operator_name(g)
    numbers, tensors = dict(n.attrs["numbers"]), list(n.attrs["tensors"])

    def param(name: str, off: str) -> str:
        if name in tensors:
            return f"{operand(g, 2 + tensors.index(name))}[row]"
        return (repr(numbers[name]) + ("" if name == "top_k" else "f")) if name in numbers else off

    u = f"{operand(g, 1)}[row]"
    temp, top_k, top_p, min_p = param("temperature", "1.0f"), param("top_k", "0"), param("top_p", "1.0f"), param("min_p", "0.0f")
    SW = sweeps_of(V, vec_width(x.dtype))
    has = (*numbers, *tensors)
    SL, N = slices(R, SW, "top_k" in has)
    x_row = f"{operand(g, 0)} + (unsigned long)row * {V}u"
    meta = {"family": "sample", "dtype": x.dtype.value, "rows": R, "V": V, "slices": SL, "sweeps": N, "bytes": R * (V * item + 8)}
    if SL == 1:
        sampler = f"tj_sampler<{T}, {V}u, {SW}u, {str(SW * vec_width(x.dtype) <= HELD_LOGITS // 2).lower()}>"
        L = [f'extern "C" __global__ __launch_bounds__({THREADS}) void {fname}({g.params()}) {{',
             "  const unsigned int row = blockIdx.x;", "  __shared__ tj_sample_shared sh;",
             f"  {sampler} s(sh, {x_row}, 0u);", f"  const int token = s.run({u}, {temp}, {top_k}, {top_p}, {min_p});",
             "  if (threadIdx.x == 0u) out0_p[row] = token;", "}"]
        return HELPERS + "\n".join(L), Launch(fname, (R, 1, 1), (THREADS, 1, 1), 0, meta)
    filtered = "top_k" in has or "top_p" in has
    split = f"tj_sample_split<{T}, {V}u, {N}u, {SL}u, {str(N * vec_width(x.dtype) <= HELD_LOGITS).lower()}>"
    row_bytes = 16 + 8 * SL * (1 + 2048 + 1 + THREADS // 64)
    calls = {"a": "p.a(s);"}
    if filtered:
        calls["b"] = f"p.b(s, {u}, {temp}, {top_k}, {top_p}, {min_p});"
    calls["c"] = f"p.c(s, {str(filtered).lower()}, {u}, {temp}, {top_k}, {top_p}, {min_p}, out0_p + row);"
    L, launches = [f"static_assert({split}::BYTES == {row_bytes}u, \"workspace\");"], []
    for i, (which, call) in enumerate(calls.items()):
        L += [f'extern "C" __global__ __launch_bounds__({THREADS}, 8) void {fname}_{which}({g.params()}, unsigned int* cnt_p, float* ws_p) {{',
              f"  const unsigned int row = blockIdx.x / {SL}u, slice = blockIdx.x % {SL}u;",
              "  __shared__ tj_sample_shared sh;",
              f"  {split}::Slice s(sh, {x_row}, slice * {N}u);",
              f"  {split} p(ws_p, cnt_p + {i * R}u, row, slice);",
              f"  {call}", "}"]
        launches.append(Launch(f"{fname}_{which}", (R * SL, 1, 1), (THREADS, 1, 1), 0, dict(meta, split_ws=(12 * R, R * row_bytes))))
    return HELPERS + "\n".join(L), launches
