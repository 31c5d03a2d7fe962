// What the paged-attention kernels share: how the work of a launch is cut into CTAs, and how the parts of a (sequence, head
// group) pair that several CTAs worked on are added.
//
//   * The kUnit-token units of all pairs form one list, and CTA c takes units [c S, (c + 1) S) of it, whatever the lengths of
//     the sequences.  The lengths are read on the device (no host step).
//   * A pair that spans CTAs leaves partial states in the workspace; the CTA that finishes last adds them in list order (the
//     result does not depend on arrival order) -- no second launch.
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "internal.h"

namespace ib200 {

// Up to so many sequences the pairs are cut evenly.  More balance by themselves, and every CTA searches all
// lengths: 1030 to 4000 sequences, 3 % of them sixteen times as long as the rest or all equal, were 0.7 to 1.07
// times as fast when cut.
constexpr int kMaxBatchCut = 1024;
constexpr int kAlignMost = 2;         // units that a share grows by at most to end with the pairs
constexpr int kAttnRows = 8;          // query heads per CTA at most
constexpr int kAttnSms = 148;         // of a B200: the CTAs that workspace, weights and counters are laid out for

struct AttnWork {
  const int32_t* seq_lens;
  float* partial;      // [CTA][2] parts
  int* counters;       // [CTA], zero at the start, this launch's alone
  int batch, block_size, max_blocks;
  int gt, groups;      // query heads per CTA, head groups per sequence
  int whole;           // 1: no workspace, CTA i takes the whole of pair i
};

// What exponents are taken relative to: 0 as long as every score was -inf (their p is 0, not NaN).
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

// A capped or biased score in base 2.  x: the product in units of the cap, or in base 2 without one.  tanh(x): up to 1/4 the
// first terms of its series (off by 62/2835 x^8, 2^-21 relative, at most), beyond it 1 - 2 / (1 + e^2x), off by some 2^-22.  Either
// way a score is good to 2^-20 of itself, however large the cap (the second form alone: 2^-22 of the cap).
__device__ __forceinline__ float scored(float x, float cap_log2e, float slope_log2e, int distance) {
  if (cap_log2e > 0.0f) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * 2.885390081777927f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    const float z = x * x, series = x * fmaf(z, fmaf(z, fmaf(z, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
    x = cap_log2e * (fabsf(x) <= 0.25f ? series : fmaf(-2.0f, r, 1.0f));
  }
  return fmaf(-slope_log2e, static_cast<float>(distance), x);
}

__device__ __forceinline__ int clamped_len(const AttnWork& p, int b) {
  const int len = __ldg(p.seq_lens + b);
  const int cap = p.max_blocks * p.block_size;
  return len < 0 ? 0 : (len > cap ? cap : len);
}

template <int kUnit>
struct UnitList {
  // an empty sequence counts one unit: its zeros have to be written by somebody
  static __device__ __forceinline__ int units_of(int len) { return len <= 0 ? 1 : (len + kUnit - 1) / kUnit; }

  // A place in the CTA's run of units: pair (b, gi), first token of the unit, end of the sequence.
  struct Cursor {
    int b, gi, t, len;
    int left;   // units of the CTA from here on
    __device__ __forceinline__ void next(const AttnWork& p) {
      --left;
      t += kUnit;
      if (t >= len && left > 0) {
        t = 0;
        if (++gi == p.groups) {
          gi = 0;
          ++b;
          len = clamped_len(p, b);
        }
      }
    }
  };

  // This CTA's run: its first place, the units per CTA and the index of its first unit (both unused where whole).  False:
  // there is none (the whole CTA).  Every warp on its own, no barrier: the lengths are a few cache lines, and
  // the first of them stay in registers between the sum and the search.
  // The CTA that merges a pair reads its parts one batch after another, so a pair of U units goes to no more than
  // about sqrt(U / balance) CTAs, where a unit's time and a part's balance.
  // kAligned: where a little larger share lets every CTA end with a pair or before, it is taken: a pair is then as many CTAs'
  // worth of units (the last one's partly void), and no CTA pays for the end of one pair and the start of another (E4M3, 32
  // heads over 8 of 128, one cache as K and V: 16 x 1000 23.4 -> 16.8 us, 48 x 1000 31.7 -> 26.4, 8 x 4096 26.6 -> 24.7; calls
  // that are cut the same either way pay 0.2 to 0.6 us for the decision).
  template <bool kAligned>
  static __device__ __forceinline__ bool begin(const AttnWork& p, float balance, Cursor& use, long long& share, long long& u0) {
    const int lane = threadIdx.x & 31;
    share = u0 = 0;
    if (p.whole) {
      use.b = blockIdx.x / p.groups;
      use.gi = blockIdx.x % p.groups;
      use.t = 0;
      use.len = clamped_len(p, use.b);
      use.left = units_of(use.len);
      return true;
    }
    const int mine0 = lane < p.batch ? units_of(clamped_len(p, lane)) : 0;
    long long sum = mine0;
    int longest = mine0;
    for (int b = lane + 32; b < p.batch; b += 32) {
      const int ub = units_of(clamped_len(p, b));
      sum += ub;
      longest = max(longest, ub);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      longest = max(longest, __shfl_xor_sync(0xFFFFFFFFu, longest, o));
    }
    long long total = sum * p.groups;
    share = (total + gridDim.x - 1) / gridDim.x;
    share = max(share, static_cast<long long>(ceilf(sqrtf(balance * static_cast<float>(longest)))));
    int pad = 1;   // the list's units of a pair are a multiple of it
    const long long pairs = static_cast<long long>(p.batch) * p.groups;
    if (kAligned && share > 1 && pairs > 1 && pairs <= gridDim.x) {
      for (int s = static_cast<int>(share); s <= share + kAlignMost; ++s) {
        int parts = (mine0 + s - 1) / s;
        for (int b = lane + 32; b < p.batch; b += 32) parts += (units_of(clamped_len(p, b)) + s - 1) / s;
        const long long ctas = static_cast<long long>(__reduce_add_sync(0xFFFFFFFFu, parts)) * p.groups;
        if (ctas <= gridDim.x) {
          share = pad = s;
          total = ctas * s;
          break;
        }
      }
    }
    const auto padded = [&](int units) { return kAligned && pad > 1 ? (units + pad - 1) / pad * pad : units; };
    u0 = share * blockIdx.x;
    if (u0 >= total) return false;
    // the sequence that unit u0 belongs to: an inclusive scan over the lengths, 32 at a time
    long long before = 0;
    for (int b0 = 0;; b0 += 32) {
      const int b = b0 + lane;
      const int ub = b0 == 0 ? mine0 : (b < p.batch ? units_of(clamped_len(p, b)) : 0);
      const long long mine = static_cast<long long>(padded(ub)) * p.groups;
      long long inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, u0 < before + inc);
      if (hit != 0u) {
        const int src = __ffs(hit) - 1;
        const int r = static_cast<int>(u0 - before - __shfl_sync(0xFFFFFFFFu, inc - mine, src));
        const int units = __shfl_sync(0xFFFFFFFFu, ub, src), list_units = padded(units);
        use.b = b0 + src;
        use.gi = r / list_units;
        use.t = (r - use.gi * list_units) * kUnit;
        use.left = static_cast<int>(pad > 1 ? min(share, static_cast<long long>(units - use.t / kUnit)) : min(share, total - u0));
        break;
      }
      before += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
    use.len = clamped_len(p, use.b);
    return true;
  }
};

// The states of a CTA's warps -> the pair's result or, where several CTAs work on the pair, a part of it; the CTA that finishes
// last adds the parts.  states: [warp][rows][D + 2] (sums, maximum in base 2, denominator), gt x CTAs floats at least;
// out: the pair's first row; t_first, t_last: first and last unit's first token; left: units of the CTA behind this pair;
// seg_u: list index of the first unit.  kZeroIfNone: a pair without any weight gives zeros (else 0 / 0).
template <int kWarps, int D, int kUnit, bool kZeroIfNone, typename T, typename Narrow>
__device__ __forceinline__ void finish_pair(const AttnWork& p, float* states, int rows, int& sh_last, T* out, int len, int t_first,
                                            int t_last, int left, long long share, long long seg_u, Narrow narrow) {
  constexpr int kThreads = 32 * kWarps, kRec = D + 2, kPart = kAttnRows * (D + 2);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
  const bool before = t_first > 0;                             // the pair began in an earlier CTA
  const bool after = left == 0 && t_last + kUnit < len;        // ... goes on in a later one
  const bool split = before || after;
  float* rec = p.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (before ? 0 : 1)) * kPart;
  for (int idx = threadIdx.x; idx < p.gt * D; idx += kThreads) {
    const int g = idx / D, d = idx % D;
    const float* st = states + g * kRec;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, st[w * rows * kRec + D]);
    float a = 0.0f, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float mw = st[w * rows * kRec + D];
      const float f = mw == -INFINITY ? 0.0f : exp2f(mw - mm);
      a = fmaf(st[w * rows * kRec + d], f, a);
      ll = fmaf(st[w * rows * kRec + D + 1], f, ll);
    }
    if (!split) {
      out[idx] = narrow(len <= 0 || (kZeroIfNone && ll == 0.0f) ? 0.0f : a / ll);
    } else {
      __stcg(rec + idx, a);
      if (d == 0) __stcg(reinterpret_cast<float2*>(rec + kAttnRows * D) + g, make_float2(mm, ll));
    }
  }
  if (!split) return;
  // the pair's CTAs: c_lo (its last segment, record 1) ... c_hi (its first, record 0 like those between)
  const long long pair_u = seg_u - t_first / kUnit;
  const int c_lo = static_cast<int>(pair_u / share);
  const int c_hi = static_cast<int>((pair_u + UnitList<kUnit>::units_of(len) - 1) / share);
  const int parts = c_hi - c_lo + 1;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) sh_last = atomicAdd(p.counters + c_lo, 1) == parts - 1;
  __syncthreads();
  if (!sh_last) return;
  __threadfence();
  const float* first = p.partial + (static_cast<int64_t>(c_lo) * 2 + 1) * kPart;   // part i > 0: 2 i - 1 records on
  auto part = [&](int i) { return first + (i == 0 ? 0 : 2 * i - 1) * kPart; };
  // weights of the parts, so many heads per warp: states[head * parts + part]
  constexpr int kHeads = kWarps < kAttnRows ? kAttnRows / kWarps : 1;
  if (warp < kAttnRows) {
    float mm[kHeads], ll[kHeads];
#pragma unroll
    for (int e = 0; e < kHeads; ++e) mm[e] = -INFINITY, ll[e] = 0.0f;
    for (int i = lane; i < parts; i += 32) {
      float2 v[kHeads];
#pragma unroll
      for (int e = 0; e < kHeads; ++e)
        if (warp + e * kWarps < p.gt)
          v[e] = __ldcg(reinterpret_cast<const float2*>(part(i) + kAttnRows * D) + warp + e * kWarps);
#pragma unroll
      for (int e = 0; e < kHeads; ++e) {
        if (warp + e * kWarps >= p.gt) break;
        const float m_new = fmaxf(mm[e], v[e].x), ref = finite_max(m_new);
        ll[e] = fmaf(ll[e], exp2f(mm[e] - ref), v[e].y * exp2f(v[e].x - ref));
        mm[e] = m_new;
        states[(warp + e * kWarps) * parts + i] = v[e].x;
      }
    }
#pragma unroll
    for (int e = 0; e < kHeads; ++e) {
      const int g = warp + e * kWarps;
      if (g >= p.gt) break;
      float m_all = mm[e];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m_all = fmaxf(m_all, __shfl_xor_sync(0xFFFFFFFFu, m_all, o));
      m_all = finite_max(m_all);
      float l_all = ll[e] * exp2f(mm[e] - m_all);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l_all += __shfl_xor_sync(0xFFFFFFFFu, l_all, o);
      const float inv = kZeroIfNone && l_all == 0.0f ? 0.0f : 1.0f / l_all;
      for (int i = lane; i < parts; i += 32) states[g * parts + i] = exp2f(states[g * parts + i] - m_all) * inv;
    }
  }
  __syncthreads();
  // the sums: a thread's four-element columns side by side, eight loads in flight (sixteen make the stream spill)
  constexpr int kCols = kAttnRows * D / 4 < kThreads ? 1 : kAttnRows * D / 4 / kThreads;
  constexpr int kBatch = 8 / kCols;
  float4 a[kCols], v[kCols][kBatch];
#pragma unroll
  for (int j = 0; j < kCols; ++j) a[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto fetch = [&](float4 (&to)[kCols][kBatch], int i0) {
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const int idx = threadIdx.x + j * kThreads;
      if (idx >= p.gt * D / 4) break;
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(to[j][e].x), "=f"(to[j][e].y), "=f"(to[j][e].z), "=f"(to[j][e].w)
                     : "l"(part(min(i0 + e, parts - 1)) + idx * 4));
      }
    }
  };
  auto add = [&](const float4 (&from)[kCols][kBatch], int i0) {
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      const int idx = threadIdx.x + j * kThreads;
      if (idx >= p.gt * D / 4) break;
      const float* wg = states + idx / (D / 4) * parts;
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        if (i0 + e >= parts) break;   // (not a weight of zero: the sum may be infinite)
        const float w = wg[i0 + e];
        a[j].x = fmaf(from[j][e].x, w, a[j].x);
        a[j].y = fmaf(from[j][e].y, w, a[j].y);
        a[j].z = fmaf(from[j][e].z, w, a[j].z);
        a[j].w = fmaf(from[j][e].w, w, a[j].w);
      }
    }
  };
  if constexpr (D == 64) {   // (small states: a second batch is on its way meanwhile)
    float4 u[kCols][kBatch];
    fetch(v, 0);
    for (int i0 = 0; i0 < parts; i0 += 2 * kBatch) {
      if (i0 + kBatch < parts) fetch(u, i0 + kBatch);
      add(v, i0);
      if (i0 + 2 * kBatch < parts) fetch(v, i0 + 2 * kBatch);
      if (i0 + kBatch < parts) add(u, i0 + kBatch);
    }
  } else {
    for (int i0 = 0; i0 < parts; i0 += kBatch) {
      fetch(v, i0);
      add(v, i0);
    }
  }
#pragma unroll
  for (int j = 0; j < kCols; ++j) {
    const int idx = threadIdx.x + j * kThreads;
    if (idx >= p.gt * D / 4) break;
    T* dst = out + idx * 4;
    dst[0] = narrow(a[j].x);
    dst[1] = narrow(a[j].y);
    dst[2] = narrow(a[j].z);
    dst[3] = narrow(a[j].w);
  }
}

// the largest divisor of the group that fits the rows
inline int heads_per_pair(int group) {
  int gt = kAttnRows;
  while (group % gt != 0) --gt;
  return gt;
}

}  // namespace ib200
