// Paged attention, single-token decode with grouped-query heads, 16-bit types, on the tensor cores
// (same contract as attention.cu; reference kernels/attention/paged_attn_decode.cu:26-118).
//
// The step is a stream of the sequences' K and V rows from HBM; what has to be kept small is
// everything else that an SM does per row.
//   * Scores and the weighted sum are matrix products (mma.sync m16n8k16): up to eight query heads
//     that share a KV head are rows 0-7 of the A operand, 16 tokens at a time the other side.  The
//     CUDA-core form of this step spent 4 x 2 FMAs per element of K and V and a shuffle tree per
//     token and was bound by instruction issue (72 % of the slots at 4.6 TB/s).
//   * The probabilities keep their fp32 value: p = hi + lo + rest in the 16-bit type, hi in rows 0-7 and
//     the remainders in rows 8-15 of two MMAs (rows 8-15 would be idle otherwise): 24 bits, in fp16 of
//     p 2^15, so that they hold from 1 down to 2^-15 and an absolute step of 2^-39 remains below.  Their sums
//     over the steps are fp32 additions, of hi by itself: an infinity of V is an infinity of that sum (join_parts).
//   * Every warp streams 16-token blocks of its own through a cp.async ring in shared memory
//     (16-byte chunks, chunk index xor row, so that ldmatrix is free of bank conflicts); no
//     block-wide synchronisation inside a sequence.
//   * The work is cut evenly into units of 64 tokens of a (sequence, head group) pair: attention_split.cuh.
//
// Bound by HBM for large batches.  Measured (bf16, 32 heads over 8 KV heads of 128, blocks of 16 in
// random order; the CUDA-core form in brackets): 64 x 4096 tokens 173.5 us = 6.2 TB/s (224 us), 128
// sequences of 500-2000 tokens 120 us = 5.5 TB/s (176 us), one sequence of 65536 58 us (75 us), 3 of
// 5000-20000 36.5 us (60 us); 28 heads over 4 KV heads, 64 x 2048: 55 us (232 us).  ncu on the first: DRAM bytes =
// the cache, issue slots 37 % busy (72 % in the CUDA-core form), tensor pipe 28 %.  Calls that it does not
// gain on take the other form: paged_attn_on_tensor_cores.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "attention_split.cuh"
#include "internal.h"

namespace ib200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTok = 16;              // tokens of a warp per step
constexpr int kUnit = kWarps * kTok;  // tokens of the CTA per step: the unit the work is cut in
constexpr int kRows = kAttnRows;
constexpr int kSms = kAttnSms;
using Units = UnitList<kUnit>;
using Cursor = Units::Cursor;

template <int D>
struct MCfg {
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kChunks = D / 8;                 // 16-byte chunks of a row
  static constexpr int kTileBytes = kTok * kRowBytes;   // a warp step's K (or V) rows
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kCtasPerSm = D == 256 ? 1 : 2;
  static constexpr int kRec = D + 2;                    // a warp's state of a head: accumulator, maximum (base 2), denominator
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kStateFloats = kWarps * kRows * kRec;
  static constexpr int kWeightFloats = kRows * kSms * kCtasPerSm;
  static constexpr int kMergeBytes = 4 * (kStateFloats > kWeightFloats ? kStateFloats : kWeightFloats);
  static constexpr int kSmemBytes = kRingBytes + kMergeBytes;
};
// (1 KiB per CTA is the system's; the kernel's static variables take less than 256 bytes)
static_assert(2 * (MCfg<64>::kSmemBytes + 1280) <= 233472 && 2 * (MCfg<128>::kSmemBytes + 1280) <= 233472, "two CTAs per SM");
static_assert(kSms * MCfg<64>::kCtasPerSm <= AttnSet::kCounters && kSms * MCfg<128>::kCtasPerSm <= AttnSet::kCounters,
              "a counter per CTA");
static_assert(MCfg<256>::kSmemBytes + 256 <= 232448, "one CTA per SM");

struct MmaAttnParams : AttnWork {
  void* out;
  const void* q;
  const void* k_cache;
  const void* v_cache;
  const int32_t* block_tables;
  int num_heads, num_kv_heads, block_shift;   // block_shift: log2(block_size) or -1
  int q_words;         // q may be read in 32-bit words
  float scale_log2e;   // what a product is multiplied by: to base 2 or, capped, to the cap's units
  float cap_log2e;     // kMod: the cap (0: none), to base 2
  const float* slopes; // kMod: a head's loss per token of distance, or null
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The sum of a head's leading parts and that of the remainders.  An infinite V makes the second
// NaN (a remainder is often zero or negative) while the first has the infinity that p V has.
__device__ __forceinline__ float join_parts(float lead, float remainder) {
  return fabsf(lead) < INFINITY ? lead + remainder : lead;
}

// a += b, two sums per instruction where kPairs
template <bool kPairs>
__device__ __forceinline__ void add4(float (&a)[4], const float (&b)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    if (kPairs) {
      asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
          : "+f"(a[i]), "+f"(a[i + 1])
          : "f"(b[i]), "f"(b[i + 1]));
    } else {
      a[i] += b[i];
      a[i + 1] += b[i + 1];
    }
  }
}

template <typename T>
struct Ops16;
template <>
struct Ops16<__nv_bfloat16> {
  static constexpr float kScale = 1.0f;   // the exponent range of fp32
  static __device__ __forceinline__ float floor_of(float p) { return p; }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  }
  static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
  // (the product alone)
  static __device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Ops16<__half> {
  // p <= 1 is summed as p 2^15: the parts have steps of 2^-39 then.  Without it the steps are 2^-24, and tokens
  // of 2^-25 and less are lost from the sum while the denominator has them.
  static constexpr float kScale = 32768.0f;
  // no leading part of a positive p is zero (2 x 2^-24; the remainder takes the difference back)
  static __device__ __forceinline__ float floor_of(float p) { return p > 0.0f ? fmaxf(p, 1.1920929e-7f) : p; }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
  // (the product alone)
  static __device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                   uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// kMod: scores may be capped and / or fall with distance
template <typename T, int D, bool kMod>
__global__ void __launch_bounds__(kThreads, MCfg<D>::kCtasPerSm)
paged_attn_mma_kernel(const MmaAttnParams p) {
  using C = MCfg<D>;
  using O = Ops16<T>;
  extern __shared__ __align__(128) uint8_t smem[];
  float* states = reinterpret_cast<float*>(smem + C::kRingBytes);
  __shared__ int sh_last;
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x >> 5), 0);
  const int row = lane >> 2;        // head row of this lane's accumulators
  const int quad = lane & 3;

  // q, the cache, the tables and the lengths may come from the kernel queued before this one; dependents are
  // not signalled early: the outputs are whole when a kernel behind this one starts, however it is launched
  pdl_wait();

  // ---- this CTA's run of units.  Balance of a unit's time and a part's: one sequence of 16384 tokens, 8 heads over one KV
  // head of 128: 118 us on 256 CTAs, 20 us on 32; 65536 tokens: 115 us on 256, 33 us on 69.  sqrt(2 U) CTAs were up to a
  // third slower, sqrt(10 U) between 30 % faster and 25 % slower.  With a dozen pairs and more the even share is the larger.
  long long share, u0;
  Cursor use;
  if (!Units::template begin<false>(p, 0.2f, use, share, u0)) return;

  const int my_units = use.left;

  // ---- producer: rows of one step of this warp, 16 tokens of K and of V
  const uint32_t ring = smem_u32(smem) + warp * (C::kStages * C::kStageBytes);
  const int gpk = (p.num_heads / p.num_kv_heads) / p.gt;   // head groups per KV head
  const int64_t row_elems = static_cast<int64_t>(p.num_kv_heads) * D;
  Cursor pre = use;
  // lane l looks up the row of token l (mod 16) of a step, one step before its copies are issued
  auto lookup = [&](const Cursor& c) -> uint32_t {
    const int t = c.t + warp * kTok + (lane & (kTok - 1));
    if (c.left <= 0 || t >= c.len) return 0xFFFFFFFFu;
    const int bi = p.block_shift >= 0 ? t >> p.block_shift : t / p.block_size;
    const int off = t - bi * p.block_size;
    return static_cast<uint32_t>(__ldg(p.block_tables + static_cast<int64_t>(c.b) * p.max_blocks + bi)) *
               static_cast<uint32_t>(p.block_size) + static_cast<uint32_t>(off);
  };
  uint32_t rows = lookup(pre);
  auto issue = [&](int slot) {
    const uint32_t dst = ring + slot * C::kStageBytes;
    const int kvh = pre.gi / gpk;
    const T* kb = static_cast<const T*>(p.k_cache) + kvh * D;
    const T* vb = static_cast<const T*>(p.v_cache) + kvh * D;
    const bool any = pre.left > 0 && pre.t + warp * kTok < pre.len;   // warp-uniform
    const uint32_t now = rows;
    if (pre.left > 0) {
      pre.next(p);
      rows = lookup(pre);
    }
    if (any) {
#pragma unroll
      for (int i = 0; i < kTok * C::kChunks / 32; ++i) {
        const int c = i * 32 + lane;
        const int r = c / C::kChunks, col = c % C::kChunks;
        const uint32_t token = __shfl_sync(0xFFFFFFFFu, now, r);
        // tokens beyond the sequence are zeros (never stale bytes: 0 x NaN would reach the sums)
        const int bytes = token == 0xFFFFFFFFu ? 0 : 16;
        const int64_t at = static_cast<int64_t>(bytes ? token : 0u) * row_elems + col * 8;
        const uint32_t d = dst + r * C::kRowBytes + ((col ^ (r & 7)) << 4);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(kb + at), "r"(bytes) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d + C::kTileBytes), "l"(vb + at), "r"(bytes)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the query rows of a pair as A fragments; requested before anything waits for them
  uint32_t qa[D / 16][2];
  float slope = 0.0f;
  auto load_q = [&](const Cursor& c) {
    const int kvh = c.gi / gpk;
    const int head0 = kvh * (p.num_heads / p.num_kv_heads) + (c.gi - kvh * gpk) * p.gt;
    const uint16_t* qrow = static_cast<const uint16_t*>(p.q) + (static_cast<int64_t>(c.b) * p.num_heads + head0 + row) * D;
    if constexpr (kMod) slope = p.slopes && row < p.gt ? __ldg(p.slopes + head0 + row) * 1.4426950408889634f : 0.0f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = kk * 16 + h * 8 + quad * 2;
        uint32_t w = 0;
        if (row < p.gt) {
          if (p.q_words) w = __ldg(reinterpret_cast<const uint32_t*>(qrow + e));
          else w = static_cast<uint32_t>(qrow[e]) | (static_cast<uint32_t>(qrow[e + 1]) << 16);
        }
        qa[kk][h] = w;
      }
    }
  };
  load_q(use);
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) issue(s);

  // ldmatrix addresses inside a tile: K rows as they are (n = token), V transposed (k = token)
  const int mi = lane >> 3, mr = lane & 7;
  const uint32_t k_row = ((mi >> 1) * 8 + mr) * C::kRowBytes;
  const uint32_t v_row = C::kTileBytes + ((mi & 1) * 8 + mr) * C::kRowBytes;

  int slot = 0;
  while (use.left > 0) {
    // ---- a pair (or the part of it that is this CTA's)
    const int b = use.b, gi = use.gi, len = use.len, t_first = use.t;
    const int kvh = gi / gpk;
    const int head0 = kvh * (p.num_heads / p.num_kv_heads) + (gi - kvh * gpk) * p.gt;
    float acc[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const long long seg_u = u0 + (my_units - use.left);   // unit index of this segment's first unit
    int t_last;
    bool end;
    do {
      __syncwarp();   // every lane has read the slot that is filled next
      {
        int ahead = slot + C::kStages - 1;
        if (ahead >= C::kStages) ahead -= C::kStages;
        issue(ahead);
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(C::kStages - 1) : "memory");
      __syncwarp();   // the other lanes' copies of this step are there too
      const int tw = use.t + warp * kTok;
      if (tw < len) {
        const uint32_t base = ring + slot * C::kStageBytes;
        float sc[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t kf[4];
          ldsm4(base + k_row + (((2 * kk + (mi & 1)) ^ mr) << 4), kf);
          O::mma(sc[0], qa[kk][0], 0u, qa[kk][1], 0u, kf[0], kf[1]);
          O::mma(sc[1], qa[kk][0], 0u, qa[kk][1], 0u, kf[2], kf[3]);
        }
        // scores of head `row` for tokens 2 quad, + 1 of either half of the block
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = tw + (i >> 1) * 8 + quad * 2 + (i & 1);
          float x = sc[i >> 1][i & 1] * p.scale_log2e;
          if constexpr (kMod) x = scored(x, p.cap_log2e, slope, len - 1 - t);
          s[i] = t < len ? x : -INFINITY;
        }
        float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
        if (__any_sync(0xFFFFFFFFu, mx > m)) {
          // a new maximum (always in the first step, rare later): the state is rescaled
          const float m_new = fmaxf(m, mx);
          const float alpha = ex2(m - finite_max(m_new));
          m = m_new;
          l *= alpha;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            acc[j][0] *= alpha;
            acc[j][1] *= alpha;
            acc[j][2] *= alpha;
            acc[j][3] *= alpha;
          }
        }
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] = ex2(s[i] - finite_max(m));   // 0 for a missing token
        l += (pr[0] + pr[1]) + (pr[2] + pr[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) pr[i] *= O::kScale;
        // rows 0-7 take the leading part of p, half of it in either MMA (zeros in the second would be 0 x inf
        // under an infinite V), rows 8-15 the two remainders
        uint32_t hi[2], lo[2], rest[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          hi[h] = O::pack(0.5f * O::floor_of(pr[2 * h]), 0.5f * O::floor_of(pr[2 * h + 1]));
          const float2 a = O::unpack(hi[h]);
          const float r0 = fmaf(a.x, -2.0f, pr[2 * h]), r1 = fmaf(a.y, -2.0f, pr[2 * h + 1]);   // exact
          lo[h] = O::pack(r0, r1);
          const float2 c = O::unpack(lo[h]);
          rest[h] = O::pack(r0 - c.x, r1 - c.y);
        }
#pragma unroll
        for (int j = 0; j < D / 8; j += 2) {
          uint32_t vf[4];
          ldsm4_trans(base + v_row + (((j + (mi >> 1)) ^ mr) << 4), vf);
          // The tensor cores truncate their sums, fp32 additions round: products of a step are summed there, the
          // steps by additions (a chain of MMAs left 6e-6 of a sum of 20000 tokens, 40 times the error of fp32
          // additions; 171.5 -> 173.5 us at 64 x 4096 tokens).
          float p0[4], p1[4];
          O::mma_first(p0, hi[0], lo[0], hi[1], lo[1], vf[0], vf[1]);
          O::mma_first(p1, hi[0], lo[0], hi[1], lo[1], vf[2], vf[3]);
          O::mma(p0, hi[0], rest[0], hi[1], rest[1], vf[0], vf[1]);
          O::mma(p1, hi[0], rest[0], hi[1], rest[1], vf[2], vf[3]);
          add4<D <= 128>(acc[j], p0);   // (size 256 has no registers for the pairs: 97 us for 88)
          add4<D <= 128>(acc[j + 1], p1);
        }
      }
      if (++slot == C::kStages) slot = 0;
      t_last = use.t;
      end = use.t + kUnit >= len || use.left == 1;
      use.next(p);
    } while (!end);

    if (use.left > 0) load_q(use);

    // ---- the four warps' states -> one
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
    l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
    if (row < p.gt) {
      float* st = states + (warp * kRows + row) * C::kRec;
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(st + j * 8 + quad * 2) =
            make_float2(join_parts(acc[j][0], acc[j][2]) * (1.0f / O::kScale), join_parts(acc[j][1], acc[j][3]) * (1.0f / O::kScale));
      if (quad == 0) {
        st[D] = m;
        st[D + 1] = l;
      }
    }
    T* out = static_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.num_heads + head0) * D;
    finish_pair<kWarps, D, kUnit, false>(p, states, kRows, sh_last, out, len, t_first, t_last, use.left, share, seg_u,
                                         [](float v) { return O::narrow(v); });
    __syncthreads();   // the states may be overwritten now
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T, int D, bool kMod>
int launch_d(MmaAttnParams p, int sm_count, bool pdl, cudaStream_t stream) {
  using C = MCfg<D>;
  const auto kernel = paged_attn_mma_kernel<T, D, kMod>;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return note_cuda_error(e);
    attr_done[dev] = true;
  }
  const int64_t pairs = static_cast<int64_t>(p.batch) * p.groups;
  int64_t ctas = pairs;
  if (!p.whole) {
    // as many CTAs as are resident at once, but no more than the tables could fill
    const int64_t most = pairs * ((static_cast<int64_t>(p.max_blocks) * p.block_size + kUnit - 1) / kUnit);
    ctas = static_cast<int64_t>(sm_count < kSms ? sm_count : kSms) * C::kCtasPerSm;
    if (ctas > most) ctas = most;   // (two units per CTA at least: 7.8 instead of 5.2 us for one sequence of 64 tokens)
  }
  if (ctas > 0x7FFFFFFF) return INFEROP_ERR_LIMIT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return note_cuda_error(e);
  return check_launch();
}

template <typename T, bool kMod>
int launch_t(const MmaAttnParams& p, int head_dim, int sm_count, bool pdl, cudaStream_t stream) {
  switch (head_dim) {
    case 64: return launch_d<T, 64, kMod>(p, sm_count, pdl, stream);
    case 128: return launch_d<T, 128, kMod>(p, sm_count, pdl, stream);
    case 256: return launch_d<T, 256, kMod>(p, sm_count, pdl, stream);
    default: return INFEROP_ERR_SHAPE;
  }
}

}  // namespace

// Which 16-bit calls come here; the others take attention.cu.  Both forms were timed on 550 shapes per type: head
// sizes 64, 128 and 256, one to eight query heads per KV head, 1 to 4000 sequences of 64 to 65536 tokens, all
// equal or ragged down to a quarter.  The figures are the other form's time over this one's, equal / ragged.  A pair
// costs this form about 5 us whatever its length, with two in flight per SM (one at head size 256) where the
// other has four; its gain is that a K / V row is read and multiplied once for up to eight heads.  So:
//   * where the other form (4, 2 or 1 heads per CTA) would fetch rows more than once: from 256 pairs or 1024
//     units on, 1.1 to 2.5 / 0.9 to 2.4 (below: 0.6 to 1.4); at head size 256 from 1024 tokens and 2048 units on,
//     1.4 to 1.9 / 1.3 to 1.9 (below: 0.5 to 1.4);
//   * four heads in either form: at head size 128 from 512 tokens and 2048 units on, or 1024 with 32 pairs and
//     more, 1.0 to 1.6 / 0.9 to 1.5 (the lower figures below 2048 units, and there the other form's second launch
//     comes on top: 8 x 1024 tokens called one by one 22.8 us, 13.4 / 16.3 here; with fewer pairs down to 0.7; 256
//     tokens and many pairs 0.8 to 1.1); at 64 from 512 tokens and 4096 units on, 1.0 to 1.35; at 256 from 4096
//     tokens and 4096 units on, 1.02 to 1.2;
//   * two heads, or one with 32 to 256 pairs: at head size 128 from 4096 tokens and 4096 units on, 1.0 to 1.3;
//     at 64 the other form is as fast or faster (0.5 to 1.1), at 256 faster (0.2 to 0.95).
bool paged_attn_on_tensor_cores(int batch, int num_heads, int num_kv_heads, int head_dim, int64_t tokens) {
  const Options& opt = options();
  if (opt.attn_path != 0) return opt.attn_path == 2;
  if (opt.attn_splits > 0 || opt.attn_heads_per_cta > 0) return false;
  const int group = num_heads / num_kv_heads;
  const int gt = heads_per_pair(group);
  const int other = group % 4 == 0 ? 4 : (group % 2 == 0 ? 2 : 1);
  const int64_t pairs = static_cast<int64_t>(batch) * (num_heads / gt);
  const int64_t units = pairs * ((tokens + kUnit - 1) / kUnit);
  if (2 * gt >= 3 * other) return head_dim <= 128 ? pairs >= 256 || units >= 1024 : tokens >= 1024 && units >= 2048;
  if (gt >= 4) {
    if (head_dim == 64) return tokens >= 512 && units >= 4096 && batch <= kMaxBatchCut;   // (uncut: 0.96 / 0.94)
    return head_dim == 128 ? tokens >= 512 && units >= (pairs >= 32 ? 1024 : 2048) : tokens >= 4096 && units >= 4096;
  }
  return head_dim == 128 && tokens >= 4096 && units >= 4096 && (gt > 1 || (pairs >= 32 && pairs <= 256));
}

size_t paged_attn_mma_workspace_bytes() {
  const size_t c = paged_attn_fp8_workspace_bytes();
  const size_t a = static_cast<size_t>(kSms) * MCfg<128>::kCtasPerSm * 2 * kRows * MCfg<128>::kRec * sizeof(float);
  const size_t b = static_cast<size_t>(kSms) * MCfg<256>::kCtasPerSm * 2 * kRows * MCfg<256>::kRec * sizeof(float);
  const size_t most = a > b ? a : b;
  return most > c ? most : c;
}

int launch_paged_attn_mma(void* out, const void* q, const void* k_cache, const void* v_cache, const int32_t* block_tables,
                          const int32_t* seq_lens, int32_t dt, int batch, int num_heads, int num_kv_heads, int head_dim,
                          int block_size, int max_blocks_per_seq, float scale, const ScoreMod& mod, int sm_count, float* workspace,
                          int* counters, bool pdl, cudaStream_t stream) {
  MmaAttnParams p;
  p.out = out;
  p.q = q;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.block_tables = block_tables;
  p.seq_lens = seq_lens;
  p.partial = workspace;
  p.counters = counters;
  p.batch = batch;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.block_size = block_size;
  p.block_shift = -1;
  for (int sh = 0; sh < 31; ++sh)
    if ((1 << sh) == block_size) p.block_shift = sh;
  p.max_blocks = max_blocks_per_seq;
  const int group = num_heads / num_kv_heads;
  p.gt = heads_per_pair(group);
  p.groups = num_heads / p.gt;

  p.whole = workspace == nullptr || batch > kMaxBatchCut ? 1 : 0;
  p.q_words = (reinterpret_cast<uintptr_t>(q) & 3u) == 0 ? 1 : 0;
  p.scale_log2e = mod.softcap > 0.0f ? scale / mod.softcap : scale * 1.4426950408889634f;
  p.cap_log2e = mod.softcap * 1.4426950408889634f;
  p.slopes = mod.slopes;
  if (dt == 1)
    return mod.any() ? launch_t<__half, true>(p, head_dim, sm_count, pdl, stream)
                     : launch_t<__half, false>(p, head_dim, sm_count, pdl, stream);
  return mod.any() ? launch_t<__nv_bfloat16, true>(p, head_dim, sm_count, pdl, stream)
                   : launch_t<__nv_bfloat16, false>(p, head_dim, sm_count, pdl, stream);
}

}  // namespace ib200
