// Rotation of queries and keys and the store of keys and values into a paged cache, one launch (no counterpart in the
// reference, whose caller rotates with rope_neox and copies rows into the cache by itself).
//
//   q [tokens, heads, dim], k / v [tokens, kv_heads, dim]: rows of a token contiguous, tokens at any stride (the three parts
//   of a fused projection's output); caches [blocks, block_size, kv_heads, dim] in the operands' type or in E4M3.
//
// Token i of a sequence whose n new tokens end at length len has position p = len - n + i; pairs (x_j, x_{j + r/2}) are
// turned by p base^(-2j/r) yarn, and K and V go to row p % block_size of block block_tables[b][p / block_size].
//
// Bound by HBM for many tokens (every byte is read once and written once), by latency for few.  So the loads of a thread's
// items are issued before anything is known about the token (its sequence, its angles), and both are worked out while they
// are on their way.  Angles: p times the frequency in turns, in fp64, of which only the fraction is kept: p f in fp32 has
// lost 6e-3 rad by position 1e5.  One fp64 product per token and pair, shared by all heads through shared memory.
//
// E4M3: a scale belongs to a cache block and a KV head, so the unit of work is a block, and all of a call's tokens in it
// belong to one CTA, a warp per head and kind (K, V).  The rows are staged in shared memory and gone through twice, for the
// maximum and for the bytes: with the rows or the rotated values in registers instead, half as many warps fit an SM, and
// 16384 tokens, half of the head rotated, took 105 to 116 us for 91.  Scales are powers of two: a floating format loses nothing by them
// (a scale that fits closer would move the values inside a binade), and when a later token needs a larger one, the
// tokens already there move to it without another rounding (but for E4M3's subnormals).  The values that are quantised
// are the rotated ones in fp32.
//
// Measured (B200, launches in a graph): 16384 tokens of 32 + 2 x 8 heads of 128, bf16, with k_out: 76 us = 5.7 TB/s, into E4M3
// caches 86 us = 4.7 TB/s (half of the head rotated 91 us = 4.4); 8192 tokens in fp32 76 us = 5.7 TB/s; E4M3 blocks of 32, 8192 tokens
// 59 us; one token each of 8 sequences 3.3 us, of 128 sequences into E4M3 caches 5.6 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "internal.h"
#include "quant_math.cuh"
#include "ragged.cuh"

namespace ib200 {
namespace {

constexpr int kThreads = 128;      // 16-bit and fp32 caches: a warp per token
constexpr int kWarps = kThreads / 32;
constexpr int kItems = 2;          // vector pairs of a lane in flight (1, 3, 4 or two sets of 1 to 3 were up to a quarter slower)
constexpr int kWarpsWanted = 148 * 16;
constexpr int kFp8Threads = 256;   // E4M3 caches: a CTA per block
constexpr int kFp8Warps = kFp8Threads / 32;
constexpr int kMaxHalf = 128;      // rotary_dim up to 256, the largest head
constexpr int kMaxTile = 16;       // tokens of a block that are handled at a time
constexpr int kMaxJobBytes = 8192; // ... and bytes of a head of theirs
constexpr float kMinScale = 7.888609052210118e-31f;   // 2^-100: the scale of a block without a non-zero value

struct AppendParams {
  const void *q, *k, *v;
  void *q_out, *k_out;             // k_out may be null
  void *k_cache, *v_cache;
  float *k_scales, *v_scales;      // E4M3 caches only
  const int32_t *block_tables, *seq_lens, *cu;   // cu null: token i is sequence i's only one
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;   // of a token, in elements
  int64_t tokens;
  int batch, heads, kv_heads, dim, half, block_size, max_blocks, num_blocks;
  int pairs_log2;                  // log2 of the vector pairs of a head
  int parts;                       // warps that share a token's heads
  int chunk;                       // E4M3: tokens that are handled at a time
  uint32_t kv_ctas;                // E4M3: CTAs of the block role
  double turns[kMaxHalf];          // frequency of pair j in turns per position
};

// V elements that are read and written together: 16 bytes, or one element where alignment or the rotary size ask for it
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T e[V];
};
template <int V>
struct alignas(V) Bytes {
  uint8_t e[V];
};

// A vector as floats and back, rounded once; 16-bit elements two at a time.
template <typename T, int V>
__device__ __forceinline__ void widen(const Vec<T, V>& v, float (&x)[V]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = v.e[e];
  } else if constexpr (V % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      const float2 f = widen2<T>(w[e / 2]);
      x[e] = f.x;
      x[e + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = static_cast<float>(v.e[e]);
  }
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> narrow(const float (&x)[V]) {
  Vec<T, V> v;
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int e = 0; e < V; e += 2) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(x[e], x[e + 1]);
        w[e / 2] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[e], x[e + 1]);
        w[e / 2] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v.e[e] = static_cast<T>(x[e]);
  }
  return v;
}

// where a token lies: its position (-1: nobody's token) and its cache row (-1: none)
struct Place {
  int pos;
  int64_t row;
};
__device__ __forceinline__ int64_t cache_row(const AppendParams& p, int b, int pos) {
  const int j = pos / p.block_size;
  if (j >= p.max_blocks) return -1;
  const int blk = __ldg(p.block_tables + static_cast<int64_t>(b) * p.max_blocks + j);
  return blk < 0 || blk >= p.num_blocks ? -1 : static_cast<int64_t>(blk) * p.block_size + (pos - j * p.block_size);
}
// (the whole warp)
__device__ __forceinline__ Place place_of(const AppendParams& p, int64_t t) {
  Place out = {-1, -1};
  int b;
  if (p.cu == nullptr) {
    b = static_cast<int>(t);
    out.pos = max(0, __ldg(p.seq_lens + b)) - 1;
  } else {
    b = last_at_or_below(t, p.batch, [&](int i) { return static_cast<int64_t>(__ldg(p.cu + i)); });
    if (b < 0) return out;
    const int64_t behind = __ldg(p.cu + b + 1) - t;
    if (behind <= 0) return out;
    out.pos = static_cast<int>(max(static_cast<int64_t>(-1), __ldg(p.seq_lens + b) - behind));
  }
  if (out.pos >= 0) out.row = cache_row(p, b, out.pos);
  return out;
}

// (cos, sin) of pair j at a position
__device__ __forceinline__ float2 turn_of(const AppendParams& p, int pos, int j) {
  const double turns = static_cast<double>(pos) * p.turns[j];
  float s, c;
  sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
  return make_float2(c, s);
}

// Pair i of a head of dim / (2 V): the vectors it consists of (in units of V elements) and whether it is turned.
// The first half / V pairs are (j, j + half / V); what lies behind the rotary part goes two by two.
struct PairOf {
  int a, b;
  bool turned;
};
template <int V>
__device__ __forceinline__ PairOf pair_of(const AppendParams& p, int i) {
  const int h = p.half / V;
  if (i < h) return {i, i + h, true};
  return {2 * i, 2 * i + 1, false};
}

// a pair of vectors turned (which product is rounded by itself is spelled out: the same bits whatever the form of the call)
template <int V>
__device__ __forceinline__ void turn(const float2 (&cs)[V], float (&x0)[V], float (&x1)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float f0 = x0[e], f1 = x1[e];
    x0[e] = __fmaf_rn(f0, cs[e].x, -__fmul_rn(f1, cs[e].y));
    x1[e] = __fmaf_rn(f0, cs[e].y, __fmul_rn(f1, cs[e].x));
  }
}

// ---- a warp with one token, or with one of p.parts shares of its heads: heads [0, heads) are q's, then kv_heads of k, then
// kv_heads of v (kStore; else q alone).  Every head has the same pairs, so a lane has one pair (V > 1: a head has at most 32),
// and with it the angles of its V elements in registers, for all the heads that it sees.  (A CTA of a few tokens with one
// table in shared memory, read for every head, took 57 us for 8192 tokens of 28 + 2 x 4 heads of 128, fp16; this form 32.)
template <typename T, int V, bool kStore>
__device__ __forceinline__ void token_role(const AppendParams& p, int64_t unit, float2* cs) {
  const int lane = threadIdx.x & 31;
  const int64_t t = unit / p.parts;
  if (t >= p.tokens) return;
  const int part = static_cast<int>(unit - t * p.parts);
  const int all = p.heads + (kStore ? 2 * p.kv_heads : 0), share = (all + p.parts - 1) / p.parts;
  const int first = part * share, last = min(all, first + share);
  const int pairs = 1 << p.pairs_log2;
  // item i of the share: pair i % pairs of head first + i / pairs
  const int total = (last - first) << p.pairs_log2;

  Vec<T, V> a[kItems], b[kItems];
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int it = base + i * 32 + lane;
      if (it < total) {
        int h = first + (it >> p.pairs_log2);
        const T* src = static_cast<const T*>(p.q) + t * p.q_stride;
        if (kStore && h >= p.heads) {
          h -= p.heads;
          src = static_cast<const T*>(p.k) + t * p.k_stride;
          if (h >= p.kv_heads) {
            h -= p.kv_heads;
            src = static_cast<const T*>(p.v) + t * p.v_stride;
          }
        }
        const PairOf pr = pair_of<V>(p, it & (pairs - 1));
        const Vec<T, V>* row = reinterpret_cast<const Vec<T, V>*>(src + h * p.dim);
        a[i] = row[pr.a];
        b[i] = row[pr.b];
      }
    }
  };
  load(0);
  const Place at = place_of(p, t);
  if (at.pos < 0) return;
  for (int j = lane; j < p.half; j += 32) cs[j] = turn_of(p, at.pos, j);
  __syncwarp();
  float2 turns[V];
  const PairOf mine = pair_of<V>(p, lane & (pairs - 1));
  if (V > 1 && mine.turned) {
#pragma unroll
    for (int e = 0; e < V; ++e) turns[e] = cs[(lane & (pairs - 1)) * V + e];
  }
  for (int base = 0; base < total; base += kItems * 32) {
    if (base > 0) load(base);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int it = base + i * 32 + lane;
      if (it >= total) break;
      int h = first + (it >> p.pairs_log2);
      const int j = it & (pairs - 1);
      const PairOf pr = V > 1 ? mine : pair_of<V>(p, j);
      T *to = static_cast<T*>(p.q_out) + t * p.q_out_stride, *also = nullptr;
      bool turned = pr.turned;
      if (kStore && h >= p.heads) {
        h -= p.heads;
        to = at.row < 0 ? nullptr : static_cast<T*>(p.k_cache) + at.row * p.kv_heads * p.dim;
        also = p.k_out ? static_cast<T*>(p.k_out) + t * p.k_out_stride : nullptr;
        if (h >= p.kv_heads) {
          h -= p.kv_heads;
          to = at.row < 0 ? nullptr : static_cast<T*>(p.v_cache) + at.row * p.kv_heads * p.dim;
          also = nullptr;
          turned = false;
        }
      }
      if (turned) {
        if (V == 1) turns[0] = cs[j];
        float x0[V], x1[V];
        widen<T, V>(a[i], x0);
        widen<T, V>(b[i], x1);
        turn<V>(turns, x0, x1);
        a[i] = narrow<T, V>(x0);
        b[i] = narrow<T, V>(x1);
      }
      if (to) {
        Vec<T, V>* d = reinterpret_cast<Vec<T, V>*>(to + h * p.dim);
        d[pr.a] = a[i];
        d[pr.b] = b[i];
      }
      if (also) {
        Vec<T, V>* d = reinterpret_cast<Vec<T, V>*>(also + h * p.dim);
        d[pr.a] = a[i];
        d[pr.b] = b[i];
      }
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 8)
append_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5;
  token_role<T, V, true>(p, static_cast<int64_t>(blockIdx.x) * kWarps + warp, reinterpret_cast<float2*>(smem) + warp * p.half);
}

// ------------------------------------------------------------------------------------------------ E4M3 caches
// the smallest power of two s with amax <= 448 s (448 = 1.75 2^8), no less than kMinScale
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax) + 0x1FFFFFu;   // a mantissa above 1.75 carries into the exponent
  const int e = static_cast<int>(u >> 23) - 8;
  return fmaxf(e > 0 ? __uint_as_float(static_cast<uint32_t>(e) << 23) : 0.0f, kMinScale);
}
// x / s as E4M3 bytes (1 / s is exact): infinities become +-448, NaN stays NaN
template <int V>
__device__ __forceinline__ Bytes<V> quantised(const float (&x)[V], float inv) {
  Bytes<V> y;
  if constexpr (V % 4 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
    for (int e = 0; e < V; e += 4) w[e / 4] = cvt2(x[e] * inv, x[e + 1] * inv) | (cvt2(x[e + 2] * inv, x[e + 3] * inv) << 16);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) y.e[e] = static_cast<uint8_t>(__nv_cvt_float_to_fp8(x[e] * inv, __NV_SATFINITE, __NV_E4M3));
  }
  return y;
}
__device__ __forceinline__ float value_of(uint8_t byte) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(byte, __NV_E4M3)));
}

// ---- a CTA of one cache block of one sequence: its new tokens, rows [off, off + n) of the block, every KV head.
// Sequence b owns items [cu[b] / block_size + 2 b, cu[b + 1] / block_size + 2 (b + 1)): n tokens touch no more than
// floor(n / block_size) + 2 blocks, and the bound needs no sum over the sequences before.
template <typename T, int V>
__device__ __forceinline__ void block_role(const AppendParams& p, int64_t item, float2* cs) {
  __shared__ float amax_of[2][64];   // several chunks of tokens: maximum so far of (kind, head) of this set of heads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int b, first_pos, last_pos, j;     // the sequence's new positions [first_pos, last_pos], the block among its own
  int64_t t_first;
  if (p.cu == nullptr) {
    b = static_cast<int>(item);
    last_pos = first_pos = max(0, __ldg(p.seq_lens + b)) - 1;
    if (first_pos < 0) return;
    j = first_pos / p.block_size;
    t_first = item;
  } else {
    b = last_at_or_below(item, p.batch, [&](int i) { return static_cast<int64_t>(__ldg(p.cu + i) / p.block_size) + 2 * i; });
    if (b < 0) return;
    const int c0 = __ldg(p.cu + b), c1 = __ldg(p.cu + b + 1);
    if (c0 < 0 || c1 <= c0 || c1 > p.tokens) return;
    const int n = c1 - c0, len = max(0, __ldg(p.seq_lens + b));
    last_pos = len - 1;
    first_pos = len - n;
    t_first = c0;
    if (first_pos < 0) {   // more new tokens than the sequence is long: the first of them have no position
      t_first -= first_pos;
      first_pos = 0;
    }
    if (last_pos < 0) return;
    j = first_pos / p.block_size + static_cast<int>(item - (c0 / p.block_size + 2 * b));
    if (static_cast<int64_t>(j) * p.block_size > last_pos) return;
  }
  const int pos0 = max(first_pos, j * p.block_size);
  const int n = static_cast<int>(min(static_cast<int64_t>(last_pos), static_cast<int64_t>(j + 1) * p.block_size - 1)) - pos0 + 1;
  const int64_t t0 = t_first + (pos0 - first_pos);
  const int64_t row0 = cache_row(p, b, pos0);
  if (row0 < 0 && p.k_out == nullptr) return;
  const int off = pos0 - j * p.block_size;
  const int64_t blk = row0 < 0 ? 0 : row0 / p.block_size;
  const int pairs = 1 << p.pairs_log2, mask = pairs - 1;
  const int chunks = (n + p.chunk - 1) / p.chunk;

  // Angles of a chunk's tokens, one token's behind the other: element e of pair j at e half / V + j, and `pairs` places between
  // tokens, so that the lanes of a warp (pairs of one to eight tokens) find theirs in different banks.
  const int turned_pairs = p.half / V, token_turns = p.half + pairs;
  auto table = [&](int c) {
    const int rows = min(p.chunk, n - c * p.chunk);
    for (int i = threadIdx.x; i < rows * p.half; i += kFp8Threads) {
      const int r = i / p.half, x = i - r * p.half;
      cs[r * token_turns + x % V * turned_pairs + x / V] = turn_of(p, pos0 + c * p.chunk + r, x);
    }
  };
  // a head's rows of a chunk, dense, on their way into this warp's part of shared memory
  T* const mine = reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(cs + p.chunk * token_turns) + warp * (p.chunk * p.dim * sizeof(T)));
  auto fetch = [&](int job, int h0, int c) {
    const int rows = min(p.chunk, n - c * p.chunk), h = h0 + (job >> 1);
    const int64_t stride = (job & 1) == 0 ? p.k_stride : p.v_stride;
    const T* src = static_cast<const T*>((job & 1) == 0 ? p.k : p.v) + (t0 + c * p.chunk) * stride + static_cast<int64_t>(h) * p.dim;
    if (V > 1) {
      const int per_row = p.dim / V;
      for (int i = lane; i < rows * per_row; i += 32) {
        const int r = i / per_row;
        const T* from = src + r * stride + (i - r * per_row) * V;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(mine + i * V)), "l"(from) : "memory");
      }
    } else {
      for (int i = lane; i < rows * p.dim; i += 32) {
        const int r = i / p.dim;
        mine[i] = src[r * stride + (i - r * p.dim)];
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // pair j of row r, turned where it is to be
  auto pair_at = [&](int r, int j, bool is_k, PairOf* pr, float (&x0)[V], float (&x1)[V]) {
    *pr = pair_of<V>(p, j);
    const Vec<T, V>* row = reinterpret_cast<const Vec<T, V>*>(mine + r * p.dim);
    widen<T, V>(row[pr->a], x0);
    widen<T, V>(row[pr->b], x1);
    if (is_k && pr->turned) {
      float2 t[V];
#pragma unroll
      for (int e = 0; e < V; ++e) t[e] = cs[r * token_turns + e * turned_pairs + j];
      turn<V>(t, x0, x1);
    }
  };
  // (64 heads at a time, so that the maxima have a place whatever the number of heads)
  for (int h0 = 0; h0 < p.kv_heads; h0 += 64) {
    const int jobs = 2 * min(64, p.kv_heads - h0);
    for (int step = 0; step < (chunks == 1 ? 1 : 2 * chunks); ++step) {
      const bool measure = step < chunks, store = chunks == 1 || step >= chunks;
      const int c = step < chunks ? step : step - chunks;
      const int rows = min(p.chunk, n - c * p.chunk), total = rows << p.pairs_log2;
      const int64_t tc = t0 + c * p.chunk;
      __syncwarp();   // every lane is done with this warp's rows before
      if (warp < jobs) fetch(warp, h0, c);
      if (step > 0 || h0 > 0) __syncthreads();   // everybody is done with the table before
      table(c);
      __syncthreads();
      for (int job = warp; job < jobs; job += kFp8Warps) {
        const bool is_k = (job & 1) == 0;
        const int hr = job >> 1, h = h0 + hr;
        float* scales = is_k ? p.k_scales : p.v_scales;
        const int64_t at = blk * p.kv_heads + h;
        const float old = off > 0 && row0 >= 0 ? scales[at] : 0.0f;
        if (job != warp) {
          __syncwarp();
          fetch(job, h0, c);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();
        float amax = 0.0f;
        if (measure) {
          // (NaN sets no scale: fmaxf drops it.  Nor does an infinity: then the finite values are gone through by themselves)
          for (bool finite_only = false;; finite_only = true) {
            amax = 0.0f;
            for (int it = lane; it < total; it += 32) {
              PairOf pr;
              float x0[V], x1[V];
              pair_at(it >> p.pairs_log2, it & mask, is_k, &pr, x0, x1);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const float f0 = fabsf(x0[e]), f1 = fabsf(x1[e]);
                if (!finite_only || f0 < INFINITY) amax = fmaxf(amax, f0);
                if (!finite_only || f1 < INFINITY) amax = fmaxf(amax, f1);
              }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
            if (finite_only || amax < INFINITY) break;
          }
          if (chunks > 1) {
            if (lane == 0) amax_of[is_k ? 0 : 1][hr] = step == 0 ? amax : fmaxf(amax_of[is_k ? 0 : 1][hr], amax);
            __syncwarp();
          }
        }
        if (!store) continue;
        if (chunks > 1) amax = amax_of[is_k ? 0 : 1][hr];
        const float scale = fmaxf(old, scale_for(amax)), inv = 1.0f / scale;
        uint8_t* cache = static_cast<uint8_t*>(is_k ? p.k_cache : p.v_cache);
        const int64_t row_bytes = static_cast<int64_t>(p.kv_heads) * p.dim;
        uint8_t* head = cache + row0 * row_bytes + static_cast<int64_t>(h) * p.dim;   // (row0 < 0: not written)
        if (row0 >= 0 && c == 0) {
          if (off > 0 && scale > old) {   // the tokens before move to the larger scale
            const float ratio = old / scale;
            constexpr int W = 8;
            const int per_row = p.dim / W;
            for (int it = lane; it < off * per_row; it += 32) {
              const int r = it / per_row;
              Bytes<W>* d = reinterpret_cast<Bytes<W>*>(head - (r + 1) * row_bytes) + (it - r * per_row);
              const Bytes<W> y = *d;
              float x[W];
#pragma unroll
              for (int e = 0; e < W; ++e) x[e] = value_of(y.e[e]);
              *d = quantised<W>(x, ratio);
            }
          }
          if (off == 0 || scale > old) {
            __syncwarp();   // every lane has read the old one
            if (lane == 0) scales[at] = scale;
          }
        }
        for (int it = lane; it < total; it += 32) {
          const int r = it >> p.pairs_log2;
          PairOf pr;
          float x0[V], x1[V];
          pair_at(r, it & mask, is_k, &pr, x0, x1);
          if (row0 >= 0) {
            Bytes<V>* d = reinterpret_cast<Bytes<V>*>(head + (c * p.chunk + r) * row_bytes);
            d[pr.a] = quantised<V>(x0, inv);
            d[pr.b] = quantised<V>(x1, inv);
          }
          if (is_k && p.k_out) {
            Vec<T, V>* d = reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.k_out) + (tc + r) * p.k_out_stride +
                                                        static_cast<int64_t>(h) * p.dim);
            d[pr.a] = narrow<T, V>(x0);
            d[pr.b] = narrow<T, V>(x1);
          }
        }
      }
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kFp8Threads, 4)
append_fp8_kernel(const __grid_constant__ AppendParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  float2* cs = reinterpret_cast<float2*>(smem);
  const int warp = threadIdx.x >> 5;
  // (the blocks first: their chain of waits is the longer one; CTAs of the two kinds alternating were 2 to 10 % slower)
  if (blockIdx.x < p.kv_ctas) block_role<T, V>(p, blockIdx.x, cs);
  else token_role<T, V, false>(p, static_cast<int64_t>(blockIdx.x - p.kv_ctas) * kFp8Warps + warp, cs + warp * p.half);
}

template <typename T, int V>
int launch_tv(AppendParams p, bool fp8, cudaStream_t stream) {
  p.pairs_log2 = 0;
  while ((2 * V) << p.pairs_log2 < p.dim) ++p.pairs_log2;
  // few tokens: as many warps for each as fill the GPU, with a pass of 32 pairs or more for every one of them
  const int64_t passes = (((static_cast<int64_t>(p.heads) + (fp8 ? 0 : 2 * p.kv_heads)) << p.pairs_log2) + 31) / 32;
  const int64_t parts = kWarpsWanted / p.tokens;
  p.parts = static_cast<int>(parts < 1 ? 1 : (parts > passes ? passes : parts));
  const int warps = fp8 ? kFp8Warps : kWarps;
  int64_t ctas = (p.tokens * p.parts + warps - 1) / warps;
  size_t smem = static_cast<size_t>(warps) * p.half * sizeof(float2);
  if (fp8) {
    const int64_t kv = p.cu ? p.tokens / p.block_size + 2 * static_cast<int64_t>(p.batch) : p.tokens;
    if (kv > 0x3FFFFFFF) return INFEROP_ERR_LIMIT;
    p.kv_ctas = static_cast<uint32_t>(kv);
    ctas += kv;
    const int row = p.dim * static_cast<int>(sizeof(T));
    p.chunk = kMaxJobBytes / row < kMaxTile ? kMaxJobBytes / row : kMaxTile;
    const size_t need = static_cast<size_t>(p.chunk) * ((p.half + (1 << p.pairs_log2)) * sizeof(float2) + kFp8Warps * row);
    smem = need > smem ? need : smem;
    static bool attr_done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    // (by the first call, whatever it needs: the 48 KB that come by themselves hold the kernel's static arrays as well)
    if (dev >= 0 && dev < 64 && !attr_done[dev]) {
      const cudaError_t e = cudaFuncSetAttribute(append_fp8_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
      if (e != cudaSuccess) return note_cuda_error(e);
      attr_done[dev] = true;
    }
  }
  if (ctas > 0x7FFFFFFF) return INFEROP_ERR_LIMIT;
  const unsigned grid = static_cast<unsigned>(ctas);
  if (fp8) append_fp8_kernel<T, V><<<grid, kFp8Threads, smem, stream>>>(p);
  else append_kernel<T, V><<<grid, kThreads, smem, stream>>>(p);
  return check_launch();
}

template <typename T>
int launch_t(const AppendParams& p, bool fp8, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                       reinterpret_cast<uintptr_t>(p.q_out) | reinterpret_cast<uintptr_t>(p.k_out) |
                       reinterpret_cast<uintptr_t>(p.k_cache) | reinterpret_cast<uintptr_t>(p.v_cache);
  const int64_t strides = p.q_stride | p.k_stride | p.v_stride | p.q_out_stride | (p.k_out ? p.k_out_stride : 0);
  if ((at & 15u) == 0 && strides % V == 0 && p.half % V == 0) return launch_tv<T, V>(p, fp8, stream);
  return launch_tv<T, 1>(p, fp8, stream);
}

}  // namespace

int launch_kv_append(const KvAppendArgs& a, cudaStream_t stream) {
  AppendParams p;
  p.q = a.q, p.k = a.k, p.v = a.v;
  p.q_out = a.q_out, p.k_out = a.k_out;
  p.k_cache = a.k_cache, p.v_cache = a.v_cache;
  p.k_scales = a.k_scales, p.v_scales = a.v_scales;
  p.block_tables = a.block_tables, p.seq_lens = a.seq_lens, p.cu = a.cu_seqlens;
  p.q_stride = a.q_stride, p.k_stride = a.k_stride, p.v_stride = a.v_stride;
  p.q_out_stride = a.q_out_stride, p.k_out_stride = a.k_out_stride;
  p.tokens = a.tokens;
  p.batch = a.batch, p.heads = a.heads, p.kv_heads = a.kv_heads, p.dim = a.dim, p.half = a.rotary_dim / 2;
  p.block_size = a.block_size, p.max_blocks = a.max_blocks, p.num_blocks = a.num_blocks;
  p.kv_ctas = 0;
  // base^(-2 j / rotary_dim) as powers of one root: the product of 128 of them is off by 2e-14 at most, 2e-8 rad at 1e6
  const double root = p.half > 0 ? pow(a.base, -1.0 / p.half) : 1.0;
  double f = a.yarn_factor / 6.283185307179586476925;
  for (int j = 0; j < kMaxHalf; ++j, f *= root) p.turns[j] = j < p.half ? f : 0.0;
  switch (a.dt) {
    case 0: return launch_t<float>(p, a.k_scales != nullptr, stream);
    case 1: return launch_t<__half>(p, a.k_scales != nullptr, stream);
    case 2: return launch_t<__nv_bfloat16>(p, a.k_scales != nullptr, stream);
    default: return INFEROP_ERR_DTYPE;
  }
}

}  // namespace ib200
