// Attention of whole prompts, packed one behind the other, on the 5th-generation tensor cores (no counterpart in the
// reference, whose attention is single-token decode).
//
//   out[i] = softmax_j(f(scale q_i.k_j)) v_j  over the tokens j < max(i + 1, prefix) of i's own prompt,
//   f(s) = cap tanh(s / cap) - slope |i - j|
//
// One pass over the keys with a running maximum and sum per query row.
//   * A CTA has two tiles of 128 query rows (two heads of one KV head where the group is even, else 256 rows of a head; one
//     tile at head size 256), so that the tensor cores work on one while the other's scores are exponentiated.
//   * S = Q K^T and O += P V are tcgen05.mma with accumulators in tensor memory; P goes back into tensor memory and is the A
//     operand from there.  A thread has a row of S: neither maximum nor sum needs a shuffle.
//   * P lies beside the scores, in a place of its own: MMAs are promised to run in the order of their issue only where accumulator
//     and shape are the same, so scores must not be written over the P that an earlier product may still read.  At head size 128
//     tensor memory has room for that with one score buffer, which the tiles use in turn: a tile's scores are in registers
//     soon after they are there.
//   * Where there are few tiles, a CTA has one, and its two warpgroups take the even and the odd blocks of keys, each with a
//     maximum, a denominator and sums of its own; they are added at the end.  A long row's chain is half as long.
//   * A V block and the next K block are one stage of a ring that TMA fills: one wait and one release per block for the
//     warp that issues the MMAs, whose own time between two products is the tensor cores' idle time (2 % of the call below).
//     V lies as it is (tokens outside): operand B with N contiguous.
//   * O is rescaled only where a row's maximum grew by more than 2^8 since the last time (the exponentials stay below
//     that), which is rare behind the first blocks; the row's thread does it in tensor memory.
//   * Rows of a V block behind the prompt's end are set to zero in shared memory: they are another prompt's, and 0 x NaN
//     would be NaN.  Their scores are masked.
// P is rounded to the operands' type for the second product: 2^-9 (bf16) or 2^-12 relative per term, of random sign, where
// the sum is rounded to the same type at the end anyway; row sums are of the unrounded values, in fp32.
//
// Bound by the tensor cores and the special-function units, each busy 56 % of the time, and in long runs by the power cap: 8192
// tokens, 32 heads over 8 KV heads of 128, bf16, causal: 467 us = 1177 TFLOP/s after a pause, 538 us = 1022 in long runs.  Of a
// pair of blocks (256 rows, 128 keys) the products are 2048 cycles and the softmax of a tile, which the other tile's products run
// beside, 1850; capped scores 700 us, 16 heads over 8 of 256 510 to 580.  With P over the scores, behind a wait for the product that
// reads it: 527 to 533 in long runs, capped 755 to 761.  Not faster (P over the scores, without that wait: 525 in long runs):
// blocks of 64 keys with two score buffers per tile (products of 64 columns run at half the rate: 640 us), a quarter of the
// exponentials by polynomials (558), P handed over in halves (546), two threads per row (564), an MMA warp per tile (600).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "internal.h"
#include "ragged.cuh"

namespace ib200 {
namespace {

constexpr int kTile = 128;                // query rows of a tile: the lanes of tensor memory
// two warpgroups with a row per thread; the issuer of MMAs, the TMA producer and two warps that only give up their registers:
// 168 per thread at launch, 208 for the first two groups and 88 for the last make the same sum
constexpr int kThreads = 384;
constexpr int kSoftmaxWarps = 8;
constexpr int kSms = 148;
constexpr int kMaxSorted = 32;            // prompts, a lane each
constexpr int kMaxSortedCtas = 4;         // per SM
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleAbove = 8.0f;     // powers of two that a maximum may lag behind

template <int D>
struct PCfg {
  static constexpr int kTiles = D == 256 ? 1 : 2;
  static constexpr int kBlock = D == 256 ? 64 : 128;              // keys of a block
  static constexpr int kBoxes = D / 64;                           // 128-byte columns of a row
  static constexpr int kQBytes = kTile * D * 2;                   // of one tile
  static constexpr int kBlockBytes = kBlock * D * 2;              // of K or V
  static constexpr int kStageBytes = 2 * kBlockBytes;             // V of a block, then K of the next
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kBarOffset = kTiles * kQBytes + kStages * kStageBytes;
  static constexpr int kSmemBytes = kBarOffset + 256 + 1024 + kTile * 8;      // (the base is rounded up to 1024)
  // tensor memory: score buffers (one per tile, or of alternate blocks; head size 128: one for all), two places for P, the sums
  static constexpr int kScoreBufs = D == 128 ? 1 : 2;
  static constexpr int kSCol = 0, kPCol = kScoreBufs * kBlock, kOCol = kPCol + 2 * (kBlock / 2);
  static_assert(kOCol + kTiles * D <= 512, "tensor memory");
  static_assert(kSmemBytes <= 232448, "shared memory");
};

struct PrefillParams {
  void* out;
  const int32_t* cu;
  const int32_t* prefix;   // or null
  const float* slopes;     // or null
  int64_t out_stride;
  int64_t tokens;
  int batch, heads, kv_heads;
  int by_heads;            // the two tiles are two heads, not 256 rows of one
  int groups;              // CTAs side by side over the heads
  int rows;                // query rows of a head per CTA
  int slots;               // CTAs over the tokens
  int sorted;              // pieces by falling index
  float scale_log2e;       // what a product is multiplied by: to base 2 or, capped, to the cap's units
  float cap_log2e;
  int no_loads;            // test hook: the producer issues no load
  DeviceStatus* status;
};

enum : uint32_t {
  kSiteAProducerEmpty = 0x141,
  kSiteAProducerEdge = 0x142,
  kSiteAMmaQ = 0x241,
  kSiteAMmaFull = 0x242,
  kSiteAMmaP = 0x243,
  kSiteAMmaS = 0x244,
  kSiteASoftmaxS = 0x341,
  kSiteASoftmaxO = 0x342,
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (NaN is dropped, as by fmaxf)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float d;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <typename T>
struct Num;
template <>
struct Num<__nv_bfloat16> {
  static constexpr uint32_t kFormat = 1;
  static constexpr float kUp = 0.0f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Num<__half> {
  static constexpr uint32_t kFormat = 0;
  // exponentials are of x + 7: with the maximum's lag they stay below 2^15, and those down to 2^-21 of the maximum's have
  // all bits of fp16
  static constexpr float kUp = 7.0f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// A wait of a whole warp: every lane goes on, or none.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, DeviceStatus* status,
                                          uint32_t site) {
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, status, site));
}

// A row's products of a block -> its scores in base 2: capped, less the distance bias.  ahead: the row's position from the
// block's first key; behind: no key that counts lies behind the row; sees: how many of the block's keys count, the first of them.
// tanh: where every score of the row is within the cap, an odd polynomial of degree 11 (off by 2.4e-7 on [-1, 1], least maximum of
// the error) on the FMA units; else 1 - 2 / (1 + e^2x), whose two special functions are the bound of the kernel then (8192
// tokens, 32 heads of 128: 1000 us against 700).  A row decides for itself: what it does not see, and what other rows see, has
// no say in its bits.
template <int kChunks>
__device__ __forceinline__ void change_scores(uint32_t (&s)[kChunks][32], const PrefillParams& p, float slope, int ahead, bool behind,
                                              int sees) {
  const auto twice = [](float v) { return make_float2(v, v); };
  const float2 f2 = twice(p.scale_log2e);
  if (p.cap_log2e > 0.0f) {
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
      for (int e = 0; e < 32; e += 2) top = max3_abs(top, __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
    }
    if (sees < kChunks * 32 && top * fabsf(p.scale_log2e) > 1.0f) {   // it may be one that does not count
      top = 0.0f;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (sees > c * 32 + e) top = fmaxf(top, fabsf(__uint_as_float(s[c][e])));
      }
    }
    if (top * fabsf(p.scale_log2e) <= 1.0f) {   // (NaN is no hindrance: it stays NaN)
      const float2 cap2 = twice(p.cap_log2e);
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 y = __fmul2_rn(make_float2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), f2), z = __fmul2_rn(y, y);
          float2 t = __ffma2_rn(twice(-0.00283946399576962f), z, twice(0.01611417718231678f));
          t = __ffma2_rn(t, z, twice(-0.05097286030650139f));
          t = __ffma2_rn(t, z, twice(0.13253524899482727f));
          t = __ffma2_rn(t, z, twice(-0.3332400321960449f));
          t = __ffma2_rn(t, z, twice(0.9999968409538269f));
          t = __fmul2_rn(t, __fmul2_rn(y, cap2));
          s[c][e] = __float_as_uint(t.x);
          s[c][e + 1] = __float_as_uint(t.y);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float r;
          asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + ex2(__uint_as_float(s[c][e]) * p.scale_log2e * (2.0f * kLog2e))));
          s[c][e] = __float_as_uint(p.cap_log2e * fmaf(-2.0f, r, 1.0f));
        }
      }
    }
    __syncwarp();
  } else {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 y = __fmul2_rn(make_float2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), f2);
        s[c][e] = __float_as_uint(y.x);
        s[c][e + 1] = __float_as_uint(y.y);
      }
    }
  }
  if (p.slopes == nullptr) return;
  if (behind) {
    float2 d = make_float2(static_cast<float>(-ahead), static_cast<float>(1 - ahead));   // minus the distance
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 y = __ffma2_rn(twice(slope), d, make_float2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])));
        s[c][e] = __float_as_uint(y.x);
        s[c][e + 1] = __float_as_uint(y.y);
        d = __fadd2_rn(d, twice(2.0f));   // (whole numbers)
      }
    }
  } else {
    float2 d = make_float2(static_cast<float>(ahead), static_cast<float>(ahead - 1));
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        s[c][e] = __float_as_uint(fmaf(-slope, fabsf(d.x), __uint_as_float(s[c][e])));
        s[c][e + 1] = __float_as_uint(fmaf(-slope, fabsf(d.y), __uint_as_float(s[c][e + 1])));
        d = __fadd2_rn(d, twice(-2.0f));
      }
    }
  }
}

// ---- piece `index` of prompt b, which is rows [c0, c0 + n) (b < 0: none); the whole warp
struct Piece {
  int b, c0, n, index;
};
// (offsets out of order or out of range: an empty prompt)
__device__ __forceinline__ int rows_of(const PrefillParams& p, int b, int* c0) {
  const int from = __ldg(p.cu + b), to = __ldg(p.cu + b + 1);
  *c0 = from;
  return from < 0 || to <= from || to > p.tokens ? 0 : to - from;
}
// Prompt b owns slots from cu[b] / rows + b on: floor(n / rows) + 1 at least, and no sum over the prompts before.
__device__ __forceinline__ Piece piece_by_slot(const PrefillParams& p, int slot) {
  Piece at;
  at.b = last_at_or_below(slot, p.batch, [&](int i) { return static_cast<int64_t>(__ldg(p.cu + i) / p.rows) + i; });
  if (at.b < 0) return at;
  at.n = rows_of(p, at.b, &at.c0);
  at.index = slot - (at.c0 / p.rows + at.b);
  if (at.index < 0 || static_cast<int64_t>(at.index) * p.rows >= at.n) at.b = -1;
  return at;
}
// All prompts' pieces by falling index: what takes longest is begun first, whatever the order of the prompts (seven of 77 to
// 1642 tokens, 16 heads of 64, cap and bias: 74 us, 88 in the prompts' order, without the turns below).  A piece of index t or
// more exists sum max(0, pieces - t) times; t is found by bisection.
__device__ __forceinline__ Piece piece_by_rank(const PrefillParams& p, int rank) {
  const int lane = threadIdx.x & 31;
  int c0 = 0;
  const int n = lane < p.batch ? rows_of(p, lane, &c0) : 0;
  const int mine = static_cast<int>((static_cast<uint32_t>(n) + p.rows - 1) / p.rows);
  int lo = 0, hi = __reduce_max_sync(0xFFFFFFFFu, mine);   // pieces of an index >= lo: more than rank, >= hi: no more
  int behind = 0;                                          // pieces of an index >= hi
  while (hi - lo > 1) {
    const int t = (lo + hi) / 2, f = __reduce_add_sync(0xFFFFFFFFu, max(0, mine - t));
    if (f > rank) {
      lo = t;
    } else {
      hi = t;
      behind = f;
    }
  }
  // (there may be no such piece: then rank - behind is no less than the prompts with more than lo pieces)
  const uint32_t has = __ballot_sync(0xFFFFFFFFu, mine > lo);
  const bool it = (has >> lane & 1u) && __popc(has & ((1u << lane) - 1u)) == rank - behind;
  Piece at;
  at.b = __ffs(__ballot_sync(0xFFFFFFFFu, it)) - 1;
  at.c0 = __shfl_sync(0xFFFFFFFFu, c0, max(0, at.b));
  at.n = __shfl_sync(0xFFFFFFFFu, n, max(0, at.b));
  at.index = lo;
  return at;
}

// where a CTA's tile i lies
struct TileAt {
  int head, q0, blocks;
};

// kHalves: a CTA has one tile, and warpgroup and sums i take the blocks of keys j with j % 2 = i
template <typename T, int D, bool kMod, bool kHalves>
__global__ void __launch_bounds__(kThreads, 1)
prefill_attn_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const PrefillParams p) {
  using C = PCfg<D>;
  constexpr int NT = C::kTiles, BN = C::kBlock;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + NT * C::kQBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
  uint64_t* q_full = bars;                     // [1]  TMA -> MMA
  uint64_t* edge = bars + 1;                   // [1]  TMA -> producer: a V block whose tail is set to zero
  uint64_t* s_full = bars + 2;                 // [2]  MMA -> softmax
  uint64_t* p_full = bars + 4;                 // [2]  softmax -> MMA (a warp each)
  uint64_t* o_done = bars + 6;                 // [2]  MMA -> softmax: a product into the sums, but for the last
  uint64_t* o_last = bars + 8;                 // [2]  ... the last
  uint64_t* s_free = bars + 10;                // [2]  softmax -> MMA (a warp each; pairs, or one buffer): the scores have been read
  uint64_t* turn = bars + 12;                  // [2]  softmax -> the other tile's: its exponentials are done
  uint64_t* full = bars + 14;                  // [kStages]  TMA -> MMA
  uint64_t* empty = full + C::kStages;         // [kStages]  MMA -> TMA
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(empty + C::kStages);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  float2* merge_at = reinterpret_cast<float2*>(bars + 32);   // [row]: maximum and denominator of the odd blocks

  const int warp = __shfl_sync(0xFFFFFFFFu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;

  // ---- this CTA's rows, a piece of p.rows of a prompt.  The last rows first: causal ones have the most keys.
  const int group_at = blockIdx.x % p.groups;
  const int slot = static_cast<int>(blockIdx.x / p.groups);
  const Piece at = p.sorted ? piece_by_rank(p, slot) : piece_by_slot(p, p.slots - 1 - slot);
  if (at.b < 0) return;
  const int b = at.b, c0 = at.c0, n = at.n, first_row = at.index * p.rows;
  const int prefix = p.prefix ? min(n, max(0, __ldg(p.prefix + b))) : 0;
  const auto tile_at = [&](int i) {
    TileAt t;
    t.head = p.by_heads ? 2 * group_at + i : group_at;
    t.q0 = first_row + (p.by_heads ? 0 : i * kTile);
    t.blocks = t.q0 >= n ? 0 : (min(n, max(t.q0 + kTile, prefix)) + BN - 1) / BN;
    return t;
  };
  static_assert(NT == 2 || !kHalves, "two warpgroups");
  constexpr bool kPairs = NT == 2 && !kHalves;    // two tiles
  constexpr bool kOneBuf = C::kScoreBufs == 1;    // both warpgroups' scores come into one buffer
  constexpr int kStep = kHalves ? 2 : 1;       // from one block of a warpgroup to its next
  const TileAt t0 = tile_at(0), t1 = NT == 1 ? TileAt{0, 0, 0} : kHalves ? t0 : tile_at(1);
  const int blocks = max(t0.blocks, t1.blocks);
  const int kv_col = t0.head / (p.heads / p.kv_heads) * D;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(edge, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&s_free[i], 4);
      mbar_init(&turn[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&o_last[i], 1);
    }
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    *abort_flag = 0u;
    mbar_init_fence();
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == kSoftmaxWarps) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);

  if (warp >= kSoftmaxWarps) {
    reg_dealloc<88>();
    if (warp == kSoftmaxWarps + 1) {
      // ------------------------------ TMA producer ------------------------
      bool ok = true;
      if (!p.no_loads) {
        if (lane == 0) {
          constexpr int tiles = kHalves ? 1 : NT;
          mbar_arrive_expect_tx(q_full, tiles * C::kQBytes);   // (a tile without rows is loaded too: nothing of it is stored)
          for (int i = 0; i < tiles; ++i) {
            const TileAt t = i == 0 ? t0 : t1;
            for (int x = 0; x < C::kBoxes; ++x)
              tma_load_2d(smem + i * C::kQBytes + x * (kTile * 128), &map_q, q_full, t.head * D + x * 64, c0 + t.q0);
          }
        }
        int stage = 0;
        uint32_t phase = 0;
        for (int j = -1; j < blocks; ++j) {                // K 0 alone, then V j with K j + 1
          if (!warp_wait(&empty[stage], phase ^ 1u, abort_flag, p.status, kSiteAProducerEmpty)) {
            ok = false;
            break;
          }
          uint8_t* dst = ring + stage * C::kStageBytes;
          const bool v = j >= 0, k = j + 1 < blocks;
          const bool tail = v && (j + 1) * BN > n;         // (once, in the last block of the prompt: there is no K behind it)
          uint64_t* bar = tail ? edge : &full[stage];
          if (lane == 0) {
            mbar_arrive_expect_tx(bar, (v ? C::kBlockBytes : 0) + (k ? C::kBlockBytes : 0));
            for (int x = 0; k && x < C::kBoxes; ++x)
              tma_load_2d(dst + C::kBlockBytes + x * (BN * 128), &map_k, bar, kv_col + x * 64, c0 + (j + 1) * BN);
            for (int x = 0; v && x < C::kBoxes; ++x) tma_load_2d(dst + x * (BN * 128), &map_v, bar, kv_col + x * 64, c0 + j * BN);
          }
          __syncwarp();
          if (tail) {
            if (!warp_wait(edge, 0u, abort_flag, p.status, kSiteAProducerEdge)) {
              ok = false;
              break;
            }
            const int r0 = n - j * BN;                       // the swizzle moves 16-byte pieces inside a row only
            for (int x = 0; x < C::kBoxes; ++x)
              for (int i = r0 * 8 + lane; i < BN * 8; i += 32)
                reinterpret_cast<uint4*>(dst + x * (BN * 128))[i] = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
          }
          if (++stage == C::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {
        // copies that this warp started may still be on their way: give them time to land before the CTA ends
        const long long w0 = clock64();
        while (clock64() - w0 < (1LL << 22)) {
        }
      }
    } else if (warp == kSoftmaxWarps) {
      // ------------------------------ MMA issuer --------------------------
      constexpr uint32_t idesc_s = umma_idesc_16bit_f32(Num<T>::kFormat, kTile, BN, false);
      constexpr uint32_t idesc_o = umma_idesc_16bit_f32(Num<T>::kFormat, kTile, D, true);
      const uint32_t q_addr = smem_u32(smem), ring_addr = smem_u32(ring);
      int stage = 0;
      uint32_t phase = 0;
      auto scores = [&](int i, int buf) {     // S = Q_i K^T
        const uint32_t d = tmem + C::kSCol + (kOneBuf ? 0 : buf * BN);
        const uint32_t k = ring_addr + stage * C::kStageBytes + C::kBlockBytes, q = q_addr + i * C::kQBytes;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t in_box = (kk % 4) * 32;
            umma_16bit_ss(d, umma_desc_k_sw128(q + (kk / 4) * (kTile * 128) + in_box),
                          umma_desc_k_sw128(k + (kk / 4) * (BN * 128) + in_box), idesc_s, kk > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[buf]);
        }
        __syncwarp();
      };
      auto sums = [&](int i, int buf, bool first, bool last) {   // O_i += P V
        const uint32_t a = tmem + C::kPCol + buf * (BN / 2);
        const uint32_t v = ring_addr + stage * C::kStageBytes;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            umma_16bit_ts(tmem + C::kOCol + i * D, a + kk * 8, umma_desc_mn_sw128(v + kk * 2048, BN * 128), idesc_o,
                          !first || kk > 0 ? 1u : 0u);
          umma_commit(last ? &o_last[i] : &o_done[i]);
        }
        __syncwarp();
      };
      const int tile_blocks[2] = {t0.blocks, t1.blocks};
      bool ok = warp_wait(q_full, 0u, abort_flag, p.status, kSiteAMmaQ);
      // What a product overwrites has been read: scores by s_free or, where they alternate between two buffers, by the P of the
      // block before last.  One tile per CTA: the scores of the next block are there before P is waited for.
      for (int j = -1; ok && j < blocks; ++j) {
        ok = warp_wait(&full[stage], phase, abort_flag, p.status, kSiteAMmaFull);
        if (!ok) break;
        tc_fence_after_sync();
        // (a pair) those of tile i's next block, once the scores before in the same buffer have been read, block `block` of tile `by`
        const auto next_scores = [&](int i) {
          if (j + 1 >= tile_blocks[i]) return;
          int by = i, block = j;
          if (kOneBuf && i == 0 && j < tile_blocks[1]) by = 1;
          if (kOneBuf && i == 1 && j + 1 < tile_blocks[0]) by = 0, block = j + 1;
          if (block >= 0) ok = ok && warp_wait(&s_free[by], block & 1, abort_flag, p.status, kSiteAMmaS);
          if (!ok) return;
          tc_fence_after_sync();
          scores(i, i);
        };
        if constexpr (!kPairs) {
          if (j + 1 < blocks) {
            if (kOneBuf && j >= 0) ok = warp_wait(&s_free[j & 1], (j >> 1) & 1, abort_flag, p.status, kSiteAMmaS);
            if (!ok) break;
            tc_fence_after_sync();
            scores(0, (j + 1) & 1);
          }
        } else if (!kOneBuf) {
#pragma unroll
          for (int i = 0; i < NT; ++i) next_scores(i);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if (kPairs && kOneBuf) next_scores(i);
          if (j >= 0 && j < tile_blocks[i] && (!kHalves || (j & 1) == i)) {
            const int buf = NT == 2 ? i : j & 1;
            ok = ok && warp_wait(&p_full[buf], (kPairs ? j : j >> 1) & 1, abort_flag, p.status, kSiteAMmaP);
            if (!ok) break;
            tc_fence_after_sync();
            sums(i, buf, j < kStep, j + kStep >= tile_blocks[i]);
          }
        }
        if (elect_one()) umma_commit(&empty[stage]);
        __syncwarp();
        if (++stage == C::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else {
    reg_alloc<208>();
    if (warp < 4 * NT) {
      // ------------------------------ softmax: a thread per row -----------
      const int i = warp >> 2;
      const TileAt t = i == 0 ? t0 : t1;
      const int pos = t.q0 + (warp & 3) * 32 + lane;
      const int lim = min(n, max(pos + 1, prefix));          // keys from here on are masked (rows behind the prompt: any)
      const int lim_warp = __shfl_sync(0xFFFFFFFFu, lim, 0), pos_warp = __shfl_sync(0xFFFFFFFFu, pos, 0);
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t o_at = tmem + lanes + C::kOCol + i * D;
      const float slope = kMod && p.slopes ? __ldg(p.slopes + t.head) * kLog2e : 0.0f;
      float m = -INFINITY, l = 0.0f;                         // m: what the row's exponentials are relative to, base 2
      bool ok = true;
      int done = 0;                                          // blocks so far
      // Changed scores: the tiles take turns at their exponentials, so that one changes scores on the FMA units while the other
      // keeps the special-function units busy (without turns they drift into step: 8192 tokens, 16 heads of 64,
      // cap and bias 437 us, 410 with turns; plain scores 200 and 218; at head size 128, where the tiles share a score
      // buffer, capped 702 and 713).
      constexpr bool kTurns = D == 64 && kPairs && kMod;
      const int both = min(t0.blocks, t1.blocks);            // blocks that both tiles have
      for (int j = kHalves ? i : 0; j < t.blocks; j += kStep, ++done) {
        const int buf = NT == 2 ? i : j & 1;
        const uint32_t s_at = tmem + lanes + C::kSCol + (kOneBuf ? 0 : buf * BN);
        const uint32_t p_at = tmem + lanes + C::kPCol + buf * (BN / 2);
        ok = warp_wait(&s_full[buf], (NT == 2 ? done : done >> 1) & 1, abort_flag, p.status, kSiteASoftmaxS);
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t s[BN / 32][32];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) tmem_ld_32x32(s_at + c * 32, s[c]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) pin32(s[c]);
        if constexpr (kPairs || kOneBuf) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[i]);
        }
        if constexpr (kMod)
          change_scores<BN / 32>(s, p, slope, pos - j * BN, (j + 1) * BN <= pos_warp + 1 || prefix == 0, lim - j * BN);
        if ((j + 1) * BN > lim_warp) {
#pragma unroll
          for (int c = 0; c < BN / 32; ++c) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (j * BN + c * 32 + e >= lim) s[c][e] = 0xFF800000u;   // -inf
          }
        }
        const float f = kMod ? 1.0f : p.scale_log2e;
        float mx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = -INFINITY;
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
#pragma unroll
          for (int e = 0; e < 32; e += 2)
            mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
        }
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * f;
        // The product that reads the P before in the same place has to be over.  One tile per CTA: it is that of the block before
        // last, issued before the scores above were, whose arrival says that everything before them is done.
        if (kPairs && done > 0) {   // (and it is the last one on these sums)
          ok = warp_wait(&o_done[i], (done - 1) & 1, abort_flag, p.status, kSiteASoftmaxO);
          if (!ok) break;
          tc_fence_after_sync();
        }
        // (rows behind the prompt have no say: a prompt's bits do not depend on its neighbours; the rows of a warp are one
        // another's, though, so which of them moved its maximum may show in the others' last bit)
        if (__any_sync(0xFFFFFFFFu, pos < n && (top > m + kRescaleAbove || m == -INFINITY))) {
          const float m_new = fmaxf(m, top);
          const float alpha = m_new == -INFINITY ? 1.0f : ex2(m - m_new);   // (every score so far -inf: no weight, not NaN)
          l *= alpha;
          m = m_new;
          if (done > 0) {
            // The product before is the last one on these sums until this warp's next arrival.  (The phase before it is over: its
            // product was issued before the scores above were.  The warps of a tile may be a block apart, so the
            // end has a barrier of its own: there a warp may be two phases ahead, where a parity says nothing.)
            if constexpr (!kPairs) {
              ok = warp_wait(&o_done[i], (done - 1) & 1, abort_flag, p.status, kSiteASoftmaxO);
              if (!ok) break;
              tc_fence_after_sync();
            }
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32(o_at + c, o);
              tmem_ld_wait();
              pin32(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st_32x32(o_at + c, o);
            }
          }
        }
        if (kTurns && done < both && (i == 1 || done > 0)) {
          ok = warp_wait(&turn[i], (i == 1 ? done : done - 1) & 1, abort_flag, p.status, kSiteASoftmaxS);
          if (!ok) break;
        }
        const float ref = (m == -INFINITY ? 0.0f : m) - Num<T>::kUp;
        const float2 f2 = make_float2(f, f), ref2 = make_float2(-ref, -ref);
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float2 x = make_float2(__uint_as_float(s[c][2 * e]), __uint_as_float(s[c][2 * e + 1]));
            x = kMod ? __fadd2_rn(x, ref2) : __ffma2_rn(x, f2, ref2);
            x.x = ex2(x.x);
            x.y = ex2(x.y);
            sum[e & 1] = __fadd2_rn(sum[e & 1], x);
            w[e] = Num<T>::pack(x.x, x.y);
          }
          tmem_st_32x16(p_at + c * 16, w);
        }
        if (kTurns && done < both) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&turn[1 - i]);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[buf]);
      }
      // ---- the row's sums / l
      if (done > 0) {
        ok = ok && warp_wait(&o_last[i], 0u, abort_flag, p.status, kSiteASoftmaxO);
        tc_fence_after_sync();
      }
      // The odd blocks' sums and the even ones', through the place of Q (of which every product is done: scores are asked for a
      // block ahead of sums): [dim][row], then the maxima and the denominators.
      float mine = 1.0f, theirs = 0.0f;                      // weights of this thread's sums and of the others'
      float* other = reinterpret_cast<float*>(smem) + (warp & 3) * 32 + lane;
      if (kHalves && t.blocks > 1) {
        if (i == 1 && ok) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32(o_at + c, o);
            tmem_ld_wait();
            pin32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) other[(c + e) * kTile] = __uint_as_float(o[e]);
          }
          merge_at[pos - t.q0] = make_float2(m, l);
        }
        ok = !named_bar_or(1, 256, !ok) && ok;
        if (i == 0 && ok) {
          const float2 ml = merge_at[pos - t.q0];
          const float m_all = fmaxf(m, ml.x);
          mine = m == m_all ? 1.0f : ex2(m - m_all);
          theirs = ml.x == m_all ? 1.0f : ex2(ml.x - m_all);
          l = l * mine + ml.y * theirs;
        }
      }
      if (done > 0 && ok && !(kHalves && i == 1)) {
        const float inv = 1.0f / l;
        T* dst = static_cast<T*>(p.out) + (static_cast<int64_t>(c0) + pos) * p.out_stride + static_cast<int64_t>(t.head) * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32(o_at + c, o);
          tmem_ld_wait();
          pin32(o);
          if (kHalves && t.blocks > 1) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(fmaf(__uint_as_float(o[e]), mine, other[(c + e) * kTile] * theirs));
          }
          if (pos < n) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint4 w;
              w.x = Num<T>::pack(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
              w.y = Num<T>::pack(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
              w.z = Num<T>::pack(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
              w.w = Num<T>::pack(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
              *reinterpret_cast<uint4*>(dst + c + e) = w;
            }
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (warp == kSoftmaxWarps) tmem_dealloc(tmem, 512);
}

template <typename T, int D, bool kMod, bool kHalves>
int launch_h(const PrefillArgs& a, PrefillParams p, cudaStream_t stream) {
  using C = PCfg<D>;
  const auto kernel = prefill_attn_kernel<T, D, kMod, kHalves>;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !attr_done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmemBytes);
    if (e != cudaSuccess) return note_cuda_error(e);
    attr_done[dev] = true;
  }
  p.by_heads = C::kTiles == 2 && !kHalves && a.heads / a.kv_heads % 2 == 0 ? 1 : 0;
  p.groups = p.by_heads ? a.heads / 2 : a.heads;
  p.rows = p.by_heads || kHalves ? kTile : C::kTiles * kTile;
  const int64_t slots = a.tokens / p.rows + a.batch;
  if (slots * p.groups > 0x7FFFFFFF) return INFEROP_ERR_LIMIT;
  p.slots = static_cast<int>(slots);
  // In the prompts' order where all CTAs run at once, and from some four per SM on, which are balanced by themselves.  Times
  // sorted / in order, ragged batches of 7 to 30: 0.85 to 1.01 between 1 and 4.3 CTAs per SM, 0.97 to 1.05 above.
  p.sorted = a.batch > 1 && a.batch <= kMaxSorted && slots * p.groups > kSms && slots * p.groups <= kMaxSortedCtas * kSms ? 1 : 0;
  CUtensorMap mq, mk, mv;
  int rc = make_tensor_map_2d(&mq, a.q, 2, a.tokens, static_cast<uint64_t>(a.heads) * D, a.q_stride * 2, kTile, 64, true);
  const uint64_t kv_cols = static_cast<uint64_t>(a.kv_heads) * D;
  if (rc == INFEROP_OK) rc = make_tensor_map_2d(&mk, a.k, 2, a.tokens, kv_cols, a.k_stride * 2, C::kBlock, 64, true);
  if (rc == INFEROP_OK) rc = make_tensor_map_2d(&mv, a.v, 2, a.tokens, kv_cols, a.v_stride * 2, C::kBlock, 64, true);
  if (rc != INFEROP_OK) return rc;
  kernel<<<static_cast<unsigned>(slots * p.groups), kThreads, C::kSmemBytes, stream>>>(mq, mk, mv, p);
  return check_launch();
}

template <typename T, int D, bool kMod>
int launch_d(const PrefillArgs& a, const PrefillParams& p, cudaStream_t stream) {
  if constexpr (PCfg<D>::kTiles == 2) {
    // A tile per CTA where the longest chain decides, not the sum of the work: all CTAs at once, or, the longer the prompts, up to
    // two to three per SM.  Two tiles and one, causal, heads of 128 (of 64 in brackets): 512 tokens and 32 heads 14.1 and 12.2 us (13.0
    // and 10.6), 1000 and 8 21.1 and 16.3 (19.4 and 13.8), 4096 and 3 65 and 42 (56 and 35); two CTAs per SM: 4096 and 8 65 and 45
    // (57 and 38), 2000 and 16 36 and 30 (32 and 25), but 1000 and 32 22.1 and 23.2 (19.8 and 19.2), 4 x 1200 and 8 25 and 33 (23 and
    // 28), 8 x 400 and 8 13.4 and 19.0 (12.5 and 15.8); more: 8192 and 6 126 and 120 (108 and 99), 4096 and 12 67 and 72 (59 and 59),
    // 2000 and 24 37 and 48 (33 and 39), 8192 and 8 124 and 145 (107 and 120).  Cap and bias: 4096 and 8 110 and 76 (112 and 71),
    // 512 and 32 20.1 and 16.9, 4 x 1200 and 8 (40 and 42).  Ragged, 1500 + 300 + 800 and 12: 30 and 26, two tiles are taken.
    const int64_t pieces = (a.tokens + static_cast<int64_t>(a.batch) * (kTile - 1)) / kTile;   // at most
    const int64_t mean = a.tokens / a.batch / kTile;
    const int half_ctas = mean >= 64 ? 6 : mean >= 32 ? 5 : mean >= 9 ? 4 : 2;                 // per SM
    if (pieces * a.heads * 2 <= half_ctas * kSms) return launch_h<T, D, kMod, true>(a, p, stream);
  }
  return launch_h<T, D, kMod, false>(a, p, stream);
}

template <typename T, bool kMod>
int launch_t(const PrefillArgs& a, const PrefillParams& p, cudaStream_t stream) {
  switch (a.dim) {
    case 64: return launch_d<T, 64, kMod>(a, p, stream);
    case 128: return launch_d<T, 128, kMod>(a, p, stream);
    case 256: return launch_d<T, 256, kMod>(a, p, stream);
    default: return INFEROP_ERR_SHAPE;
  }
}

}  // namespace

int launch_prefill_attn(DeviceCtx* ctx, const PrefillArgs& a, cudaStream_t stream) {
  PrefillParams p = {};
  p.out = a.out;
  p.cu = a.cu_seqlens;
  p.prefix = a.prefix_lens;
  p.slopes = a.mod.slopes;
  p.out_stride = a.out_stride;
  p.tokens = a.tokens;
  p.batch = a.batch, p.heads = a.heads, p.kv_heads = a.kv_heads;
  p.scale_log2e = a.mod.softcap > 0.0f ? a.scale / a.mod.softcap : a.scale * kLog2e;
  p.cap_log2e = a.mod.softcap * kLog2e;
  p.no_loads = options().debug_no_loads;
  p.status = ctx->status;
  // (the plain form takes the maximum of the products and scales it, so it needs a positive scale)
  const bool mod = a.mod.any() || !(a.scale > 0.0f);
  if (a.dt == 1) return mod ? launch_t<__half, true>(a, p, stream) : launch_t<__half, false>(a, p, stream);
  return mod ? launch_t<__nv_bfloat16, true>(a, p, stream) : launch_t<__nv_bfloat16, false>(a, p, stream);
}

}  // namespace ib200
