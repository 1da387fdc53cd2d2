// Attention with a sliding window and visible first tokens (sinks), forward: one CTA works on two 128-row
// tiles of queries against the keys they can see.
//
//   S = scale Q K^T over the visible keys, m = max S, P = exp(S - m), l = sum P, O = P V / l, lse = m + log l
//
// Query i of a sequence is at position p = i + kv_length - q_length and sees keys j <= p with p - j < window
// or j < sinks.  Key tiles that no row of the pair of tiles sees are not visited: the sinks' tiles come first,
// then the window's.
//
// A tile's 128 rows are `pack` query heads that share a KV head times 128 / pack tokens (heads fastest):
// the tensor map's box brings them in that order.  A group of heads then reads each key tile once, and a few
// new tokens of many heads still fill rows.
//
// Roles (12 warps): warp 0 loads (TMA: both Q tiles, then K and V tiles through two rings), warps 1 and 3 issue the
// UMMAs of one tile each, warp 2 allocates TMEM, warps 4-7 and 8-11 are one softmax group per tile, one thread per row.
// TMEM (512 columns): S of either tile (128 FP32 columns each; P overwrites the first 64 of its own S as
// packed BF16 and is the A operand of P V straight from there) and O of either tile.  With heads of 64 O takes half as
// much, and P has columns of its own.
//
// The UMMAs of a tile are issued in the order P V, S of the next keys: while one tile's softmax runs, the tensor cores
// work for the other.  They execute in issue order, so S may overwrite the P that the UMMA before it reads, and "S of
// the next keys is complete" implies "O holds all keys before", which is what a softmax group needs to rescale O in place.
// With heads of 64 S of the next keys is issued first, as soon as the softmax group has read this one's, and P V's completion
// is waited for by itself.
//
// Few queries (one tile of them) against many keys: the keys are split over blocks, and within a block both tiles hold
// the same queries and take every other key tile, so that one's softmax overlaps the other's products and the loads keep
// coming.  Every part leaves its normalised O and its lse, and a second kernel joins them.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last time (the weights then
// stay below 2^8 in BF16 and the sums below 2^8 kv_len in FP32; the result is divided by the same sum, so
// this changes no value beyond rounding).  S, the statistics and O are FP32; P is rounded to BF16 for the
// second product and summed before that rounding.
#pragma once

#include "host.cuh"
#include "sync.cuh"

namespace fuse_b200 {
namespace attn {

constexpr int kTile = 128;  // rows of a query tile, keys of a key tile
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  WaitContext wait;
  const int32_t *q_starts, *q_lengths, *kv_starts, *kv_lengths;
  int64_t q_rows, kv_rows;  // extents of the tensors
  int32_t batch, q_len, kv_len, q_heads, kv_heads;
  int32_t pack;        // query heads in a tile: a power of two that divides the group
  int32_t pack_shift;
  int32_t causal, window, sinks;
  float scale, scale_log2;
  uint16_t* out;
  int8_t* rest;  // [q_rows][q_heads * head_dim] what rounding takes off out, or nullptr
  int64_t out_stride;
  float* lse;  // [q_heads][q_rows] or nullptr
  // split over keys: partial results per (part, batch, token, head), joined by a second kernel
  int32_t splits;  // blocks along the keys
  int32_t paired;  // one query tile a block: both of its tiles work on it, on every other key tile
  int32_t parts;   // splits, times two when paired
  float *partial, *partial_lse;
};

// What is the same for a whole warp, said so: values that come from memory are not known to be, and the UMMA
// warp's operands would take the long way through vector registers (measured: 850 cycles for the eight
// instructions of a 128 x 128 x 128 product that the tensor cores do in 512).
__device__ __forceinline__ int32_t uniform(int32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

struct Sequence {
  int32_t q0, k0;  // first rows
  int32_t ql, kl;  // lengths
  int32_t off;     // position of query 0
};

// Lengths and starts come from device memory: whatever they hold, no row outside the tensors is touched.
__device__ __forceinline__ void clamp_rows(int64_t start, int32_t length, int32_t most, int64_t rows, int32_t* first,
                                           int32_t* count) {
  int64_t n = length < most ? length : most;
  if (start < 0 || start > rows) n = start = 0;
  if (n > rows - start) n = rows - start;
  *first = int32_t(start);
  *count = n < 0 ? 0 : int32_t(n);
}
// (By whole warps.)
__device__ __forceinline__ Sequence sequence(const Args& a, int32_t b) {
  Sequence s;
  clamp_rows(a.q_starts ? a.q_starts[b] : int64_t(b) * a.q_len, a.q_lengths ? a.q_lengths[b] : a.q_len, a.q_len, a.q_rows,
             &s.q0, &s.ql);
  clamp_rows(a.kv_starts ? a.kv_starts[b] : int64_t(b) * a.kv_len, a.kv_lengths ? a.kv_lengths[b] : a.kv_len, a.kv_len,
             a.kv_rows, &s.k0, &s.kl);
  s.q0 = uniform(s.q0);
  s.k0 = uniform(s.k0);
  s.ql = uniform(s.ql);
  s.kl = uniform(s.kl);
  s.off = s.kl - s.ql;
  return s;
}

// What the tokens [first, last) of a sequence see: keys [lo, end) and [0, sinks).
struct KeyRange {
  int32_t lo, end, sinks;
  __device__ __forceinline__ KeyRange(const Args& a, const Sequence& s, int32_t first, int32_t last) {
    lo = 0;
    end = s.kl;
    if (a.causal) {
      if (last + s.off < end) end = last + s.off;
      if (a.window > 0 && first + s.off - a.window + 1 > 0) lo = first + s.off - a.window + 1;
    }
    if (first >= last || end < 0) end = 0;
    sinks = a.window > 0 && a.sinks > 0 ? (a.sinks < end ? a.sinks : end) : 0;
  }
  // Whether any of the `keys` keys from k0 on is seen.
  __device__ __forceinline__ bool sees(int32_t k0, int32_t keys) const { return k0 < end && (k0 + keys > lo || k0 < sinks); }
};
// Tiles of a range in the order they are visited.
struct TileList {
  int32_t sink_tiles, first, count;
  __device__ __forceinline__ explicit TileList(const KeyRange& r) {
    first = r.lo / kTile;
    sink_tiles = (r.sinks + kTile - 1) / kTile;
    if (sink_tiles > first) sink_tiles = first;
    count = r.end > 0 ? sink_tiles + (r.end + kTile - 1) / kTile - first : 0;
  }
  __device__ __forceinline__ int32_t tile(int32_t i) const { return i < sink_tiles ? i : first + i - sink_tiles; }
};
// Whether some row among tokens [first, last) does not see all of the `keys` keys from k0 on.
__device__ __forceinline__ bool needs_mask(const Args& a, const Sequence& s, int32_t first, int32_t last, int32_t k0,
                                           int32_t keys) {
  if (k0 + keys > s.kl) return true;
  if (!a.causal) return false;
  if (k0 + keys - 1 > first + s.off) return true;
  return a.window > 0 && k0 < last - 1 + s.off - a.window + 1 && k0 + keys > a.sinks;
}

// The low n of 32 bits (n may be anything).
__device__ __forceinline__ uint32_t low_bits(int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// Of the 32 keys from k0 on, those a row sees: keys <= hi that are >= lo or < sinks.
__device__ __forceinline__ uint32_t visible_keys(int32_t k0, int32_t hi, int32_t lo, int32_t sinks) {
  return low_bits(hi + 1 - k0) & (~low_bits(lo - k0) | low_bits(sinks - k0));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two FP32 values in a 64-bit register, for the packed FP32 instructions.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16_pair(uint64_t v) {
  float a, b;
  unpair(v, a, b);
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
// max(a, b, c), NaN if any is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float as_float(uint32_t v) { return __uint_as_float(v); }
// A whole warp waits together (the common case, a barrier that is through or about to be, is one vote).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const WaitContext& w, uint32_t site) {
  if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  const uint64_t start = ptx::globaltimer();
  for (uint32_t spin = 1;; ++spin) {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
    if ((spin & 31u) == 0u) {
      bool over = aborted(w);
      if (!over && ptx::globaltimer() - start > w.budget_ns) {
        write_timeout(w, kStatusMbarrierTimeout, site, bar, parity, 0);
        over = true;
      }
      if (__any_sync(0xffffffffu, over)) return false;
    }
  }
}

// A warp arrives with one lane.  tcgen05.ld, .st, .wait and the named barriers are .sync.aligned: behind every branch that
// lanes take apart (this one, a row's store, zeroed rows) the warp is brought together before it comes to the next of them.
__device__ __forceinline__ void warp_arrive(uint32_t bar, int lane) {
  __syncwarp();
  if (lane == 0) ptx::mbar_arrive(bar);
  __syncwarp();
}

// A [128 x kDim] BF16 tile in shared memory: kDim / 64 blocks of 128 rows x 128 bytes, 128-byte swizzle.
template <int kDim>
struct TileShape {
  static constexpr uint32_t kBlockBytes = kTile * 128;
  static constexpr uint32_t kBlocks = kDim / 64;
  static constexpr uint32_t kBytes = kBlocks * kBlockBytes;
};
template <int kDim>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t head, int32_t row) {
#pragma unroll
  for (uint32_t b = 0; b < TileShape<kDim>::kBlocks; ++b)
    ptx::tma_load_3d(dst + b * TileShape<kDim>::kBlockBytes, map, bar, int32_t(b * 64), head, row);
}
// Rows [valid, 128) of a tile become zeros (a row is 128 bytes in every block, whatever the swizzle): what lies
// behind a sequence's end may be anything, and 0 times that need not be 0.  One row per thread.
template <int kDim>
__device__ __forceinline__ void zero_rows(uint32_t tile, int32_t row, int32_t valid) {
  if (row >= valid) {
#pragma unroll
    for (uint32_t b = 0; b < TileShape<kDim>::kBlocks; ++b)
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i)
        ptx::st_shared_v4(tile + b * TileShape<kDim>::kBlockBytes + uint32_t(row) * 128u + i * 16u, make_uint4(0u, 0u, 0u, 0u));
  }
  ptx::fence_proxy_async_shared();
  __syncwarp();
}

// D[128 x 128] = A B^T over kDim: both operands K-major tiles.  A converged warp.
template <int kDim>
__device__ __forceinline__ void mma_rows(uint32_t issue, uint32_t d, uint32_t a_tile, uint32_t b_tile) {
  constexpr uint32_t kIdesc = ptx::idesc_bf16_f32(kTile, kTile, 0, 0);
  const uint64_t a_desc = ptx::smem_desc_k_sw128(a_tile), b_desc = ptx::smem_desc_k_sw128(b_tile);
#pragma unroll
  for (uint32_t k = 0; k < kDim / 16; ++k) {
    const uint64_t at = ((k / 4) * TileShape<kDim>::kBlockBytes + (k % 4) * 32) >> 4;
    ptx::umma_f16_if(issue, d, a_desc + at, b_desc + at, kIdesc, k != 0 ? 1u : 0u);
  }
}
// D[128 x kDim] (+)= A[128 x 128] B: A in TMEM (K values 16 k .. 16 k + 15 at column a_column(k)), B a tile whose rows are
// the K axis.
template <int kDim, class Column>
__device__ __forceinline__ void mma_weights(uint32_t issue, uint32_t d, Column a_column, uint32_t b_tile, bool accumulate) {
  constexpr uint32_t kIdesc = ptx::idesc_bf16_f32(kTile, kDim, 0, 1);
  const uint64_t b_desc = ptx::smem_desc_mn_sw128(b_tile, TileShape<kDim>::kBlockBytes);
#pragma unroll
  for (uint32_t k = 0; k < kTile / 16; ++k)
    ptx::umma_f16_a_tmem_if(issue, d, a_column(k), b_desc + uint64_t(k * 128u), kIdesc, k != 0 || accumulate ? 1u : 0u);
}

// An operand in TMEM whose K values lie in consecutive columns.
struct Columns {
  uint32_t base;
  __device__ __forceinline__ uint32_t operator()(uint32_t k) const { return base + k * 8u; }
};

// What rounding to BF16 takes off an FP32 value, as a byte: the difference of the bit patterns in units of 2^8 (half a step of BF16 is
// 2^15), so that value and byte together keep 16 bits of the fraction.  Infinities and NaN stay what they are.
__device__ __forceinline__ int32_t rounded_off(float v, uint32_t bf16_bits) {
  const int32_t difference = int32_t(__float_as_uint(v) - (bf16_bits << 16));
  return max(min((difference + 128) >> 8, 127), -128);
}
__device__ __forceinline__ float with_rest(uint32_t bf16_bits, int32_t rest) {
  return __uint_as_float((bf16_bits << 16) + uint32_t(rest * 256));
}
__device__ __forceinline__ uint32_t rest_of_pair(uint32_t pair, float lo, float hi) {  // two bytes
  return (uint32_t(rounded_off(lo, pair & 0xffffu)) & 0xffu) | ((uint32_t(rounded_off(hi, pair >> 16)) & 0xffu) << 8);
}

template <int kDim>
struct ForwardLayout {
  static constexpr int kStages = kDim == 128 ? 2 : 4;  // of either ring
  static constexpr uint32_t kTileBytes = TileShape<kDim>::kBytes;
  static constexpr uint32_t kK = 2 * kTileBytes;
  static constexpr uint32_t kV = kK + kStages * kTileBytes;
  static constexpr uint32_t kBarriers = kV + kStages * kTileBytes;
  // q_full[2], s_full[2], p_ready[2], drain[2], s_read[2], o_done[2], o_full, then k_full, k_empty, v_full, v_empty [kStages]
  static constexpr uint32_t kNumBarriers = 13 + 4 * kStages;
  // Heads of 64 leave TMEM for P beside S: S of the next keys is then issued as soon as this one's is in registers.
  static constexpr bool kOwnP = kDim == 64;
  static constexpr uint32_t kSlot = kBarriers + kNumBarriers * 8;
  static constexpr uint32_t kDynamicBytes = kSlot + 16;
  static_assert(kDynamicBytes <= 227 * 1024, "shared memory budget");
  static_assert(kDynamicBytes > 114 * 1024, "must force one CTA per SM (all of TMEM is allocated)");
};
constexpr int kForwardThreads = 384;

template <int kDim>
__global__ void __launch_bounds__(kForwardThreads, 1)
attention_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a) {
  using Layout = ForwardLayout<kDim>;
  constexpr int kStages = Layout::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = ptx::smem_u32(smem_raw);
  const int warp = uniform(int32_t(threadIdx.x >> 5)), lane = threadIdx.x & 31;

  // block -> (tokens, head pack, batch, split); the last tokens, which see the most keys, come first
  const int32_t tile_tokens = kTile >> a.pack_shift, packs = a.q_heads >> a.pack_shift;
  int32_t at = int32_t(blockIdx.x);
  const int32_t split = at % a.splits;
  at /= a.splits;
  const int32_t pack = at % packs;
  at /= packs;
  const int32_t b = at % a.batch;
  const int32_t second = a.paired ? 0 : tile_tokens;  // from the first tile's tokens to the other's
  const int32_t token_blocks = (a.q_len + tile_tokens + second - 1) / (tile_tokens + second);
  const int32_t t0 = (token_blocks - 1 - at / a.batch) * (tile_tokens + second);
  const Sequence seq = sequence(a, b);
  if (t0 >= seq.ql) return;  // (the whole block, before anything is set up)
  const int32_t head0 = pack << a.pack_shift, kv_head = head0 / (a.q_heads / a.kv_heads);
  const KeyRange range(a, seq, t0, min(t0 + second + tile_tokens, seq.ql));
  // whether tile t, which sees the keys `own`, works on the key tile of iteration `it`
  auto works = [&](int t, const KeyRange& own, const TileList& list, int32_t it, int32_t first_it) {
    return own.sees(list.tile(it) * kTile, kTile) && (!a.paired || ((it - first_it) & 1) == t);
  };
  const TileList tiles(range);
  const int32_t per_split = (tiles.count + a.splits - 1) / a.splits;
  const int32_t it0 = min(split * per_split, tiles.count), it1 = min(it0 + per_split, tiles.count);

  const uint32_t bars = base + Layout::kBarriers;
  auto q_full = [&](int t) { return bars + 8u * t; };
  auto s_full = [&](int t) { return bars + 8u * (2 + t); };
  auto p_ready = [&](int t) { return bars + 8u * (4 + t); };
  auto drain = [&](int t) { return bars + 8u * (6 + t); };
  auto s_read = [&](int t) { return bars + 8u * (8 + t); };
  auto o_done = [&](int t) { return bars + 8u * (10 + t); };
  const uint32_t o_full = bars + 8u * 12;
  auto k_full = [&](int s) { return bars + 8u * (13 + s); };
  auto k_empty = [&](int s) { return bars + 8u * (13 + kStages + s); };
  auto v_full = [&](int s) { return bars + 8u * (13 + 2 * kStages + s); };
  auto v_empty = [&](int s) { return bars + 8u * (13 + 3 * kStages + s); };
  auto k_tile = [&](int s) { return base + Layout::kK + s * Layout::kTileBytes; };
  auto v_tile = [&](int s) { return base + Layout::kV + s * Layout::kTileBytes; };

  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(q_full(t), 1);
      ptx::mbar_init(s_full(t), 1);
      ptx::mbar_init(drain(t), 1);
      ptx::mbar_init(p_ready(t), 4);  // one arrival per warp of the softmax group
      ptx::mbar_init(s_read(t), 4);
      ptx::mbar_init(o_done(t), 1);
    }
    ptx::mbar_init(o_full, 2);  // from here on 2: a commit of either issuing warp
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(k_full(s), 1);
      ptx::mbar_init(k_empty(s), 2);
      ptx::mbar_init(v_full(s), 1);
      ptx::mbar_init(v_empty(s), 2);
    }
    ptx::fence_mbar_init();
  }
  __syncwarp();
  if (warp == 2) {
    ptx::tmem_alloc(base + Layout::kSlot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns are this block's
  auto s_tmem = [&](int t) { return tmem + uint32_t(t) * 128u; };
  auto o_tmem = [&](int t) { return tmem + 256u + uint32_t(t) * kDim; };
  auto p_tmem = [&](int t) { return Layout::kOwnP ? tmem + 384u + uint32_t(t) * 64u : s_tmem(t); };

  bool unwound = false;
  // 168 registers a thread at launch, 64,512 in all: 88 for the first four warps and 208 for the eight softmax warps
  // are as many
  if (warp < 4) ptx::setmaxnreg_dec<88>();
  if (warp == 0) {
    if (lane == 0 && it0 < it1) {
      bool ok = true;
      auto load_q = [&](int t) {
        if (t0 + t * second >= seq.ql) return;
        ptx::mbar_expect_tx(q_full(t), Layout::kTileBytes);
        load_tile<kDim>(base + t * Layout::kTileBytes, &map_q, q_full(t), head0, seq.q0 + t0 + t * second);
      };
      load_q(0);
      for (int32_t it = it0; ok && it < it1; ++it) {
        const int s = (it - it0) % kStages;
        const uint32_t phase = ((it - it0) / kStages) & 1;
        const int32_t row = seq.k0 + tiles.tile(it) * kTile;
        if (!(ok = mbar_wait<false>(k_empty(s), phase ^ 1u, a.wait, kSiteSmemEmpty))) break;
        ptx::mbar_expect_tx(k_full(s), Layout::kTileBytes);
        load_tile<kDim>(k_tile(s), &map_k, k_full(s), kv_head, row);
        if (it == it0) load_q(1);
        if (!(ok = mbar_wait<false>(v_empty(s), phase ^ 1u, a.wait, kSiteSmemEmpty))) break;
        ptx::mbar_expect_tx(v_full(s), Layout::kTileBytes);
        load_tile<kDim>(v_tile(s), &map_v, v_full(s), kv_head, row);
      }
      unwound = !ok;
    }
  } else if (warp == 1 || warp == 3) {
    // One warp per tile, on two quarters of the SM: beside the softmax warps a warp gets an instruction through every
    // ten cycles or so, and the waits and commits of both tiles would be more than one warp's time.  The whole warp walks
    // the schedule and one lane issues: the operands of the instructions stay uniform.
    const int t = warp >> 1;
    if (it0 < it1) {
      const uint32_t issue = ptx::elect_one();
      const int32_t my_first = t0 + t * second;
      const KeyRange own(a, seq, my_first, min(my_first + tile_tokens, seq.ql));
      const uint32_t q_tile = base + t * Layout::kTileBytes;
      auto seen = [&](int32_t it) { return it < it1 && works(t, own, tiles, it, it0); };
      bool ok = my_first >= seq.ql || warp_wait(q_full(t), 0, a.wait, kSiteSmemFull);
      uint32_t p_phase = 0, has_o = 0;
      uint32_t s = 0, s_next = 0, v_phase = 0, k_phase = 0;  // stages of V of tile `it` and of K of tile it + 1
      bool now = false, next = seen(it0);
      uint32_t read_phase = 0, issued = 0;
      auto scores = [&]() __attribute__((always_inline)) {
        mma_rows<kDim>(issue, s_tmem(t), q_tile, k_tile(s_next));
        ptx::umma_commit_if(issue, s_full(t));
      };
      for (int32_t it = it0 - 1; ok && it < it1; ++it) {
        if (it + 1 < it1 && !(ok = warp_wait(k_full(s_next), k_phase, a.wait, kSiteSmemFull))) break;
        if constexpr (Layout::kOwnP) {
          if (next) {  // behind P V of the keys before, ahead of P V of these
            if (issued && !(ok = warp_wait(s_read(t), read_phase, a.wait, kSiteTmemEmpty))) break;
            read_phase ^= issued;
            issued = 1;
            ptx::tc_fence_after();
            scores();
          }
        }
        if (it >= it0 && !(ok = warp_wait(v_full(s), v_phase, a.wait, kSiteSmemFull))) break;
        if (now) {
          if (!(ok = warp_wait(p_ready(t), p_phase, a.wait, kSiteTmemEmpty))) break;
          ptx::tc_fence_after();
          mma_weights<kDim>(issue, o_tmem(t), Columns{p_tmem(t)}, v_tile(s), has_o);
          if constexpr (Layout::kOwnP) ptx::umma_commit_if(issue, o_done(t));
          has_o = 1;
          p_phase ^= 1u;
        }
        if constexpr (!Layout::kOwnP) {
          if (next) scores();
        }
        if (it >= it0) ptx::umma_commit_if(issue, v_empty(s));
        if (it + 1 < it1) ptx::umma_commit_if(issue, k_empty(s_next));
        now = next;
        next = seen(it + 2);
        s = s_next;
        v_phase = k_phase;
        if (++s_next == kStages) { s_next = 0; k_phase ^= 1u; }
      }
      ptx::umma_commit_if(issue, ok ? o_full : drain(t));
      if (!ok) mbar_wait<false>(drain(t), 0u, a.wait, kSiteDrain, false);  // UMMAs already issued retire before TMEM is released
      unwound = !ok;
    }
  } else if (warp >= 4) {
    ptx::setmaxnreg_inc<208>();
    const int t = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const int32_t my_first = t ? t0 + second : t0, my_last = min(my_first + tile_tokens, seq.ql);
    const KeyRange my_range(a, seq, my_first, my_last);
    const uint32_t o_at = o_tmem(t) + lanes;
    const int32_t token = my_first + (row >> a.pack_shift), head = head0 + (row & (a.pack - 1));
    const int32_t pos = token + seq.off;
    const int32_t hi = a.causal ? min(pos, seq.kl - 1) : seq.kl - 1;
    const int32_t lo = a.causal && a.window > 0 ? pos - a.window + 1 : 0;
    const int32_t sinks = a.window > 0 ? a.sinks : 0;
    const bool live = my_first < my_last;
    const uint32_t s_at = s_tmem(t) + lanes;
    float m = -INFINITY, l = 0.0f;  // m: the reference of the exponent, in units of the scaled score's log2
    bool ok = true, begun = false;
    uint32_t phase = 0;
    for (int32_t it = it0; ok && it < it1; ++it) {
      const int32_t k0 = tiles.tile(it) * kTile;
      if (!works(t, my_range, tiles, it, it0)) continue;
      if (!(ok = warp_wait(s_full(t), phase, a.wait, kSiteTmemFull))) break;
      phase ^= 1u;
      ptx::tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int i = 0; i < 4; ++i) ptx::tmem_ld_32x32b_x32(s_at + i * 32, s[i]);
      ptx::tmem_wait_ld();
      if constexpr (Layout::kOwnP) {
        ptx::tc_fence_before();
        warp_arrive(s_read(t), lane);
      }
      if (needs_mask(a, seq, my_first, my_last, k0, kTile)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t seen = visible_keys(k0 + i * 32, hi, lo, sinks);
#pragma unroll
          for (int c = 0; c < 32; ++c) s[i][c] = seen & (1u << c) ? s[i][c] : 0xff800000u;
        }
      }
      float top[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        top[i] = max3(as_float(s[i][0]), as_float(s[i][1]), as_float(s[i][2]));
#pragma unroll
        for (int c = 3; c < 31; c += 2) top[i] = max3(top[i], as_float(s[i][c]), as_float(s[i][c + 1]));
        top[i] = max3(top[i], as_float(s[i][31]), as_float(s[i][31]));
      }
      const float largest = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * a.scale_log2;
      l = largest != largest ? largest : l;  // a score that is no number: so is the row
      if constexpr (Layout::kOwnP) {  // P V of the keys before: O is complete, and P may be written again
        if (begun && !(ok = warp_wait(o_done(t), phase, a.wait, kSiteTmemFull))) break;
        ptx::tc_fence_after();
      }
      if (__any_sync(0xffffffffu, largest > m + 8.0f)) {
        const float to = fmaxf(m, largest);
        const float factor = m == -INFINITY ? 0.0f : exp2_approx(m - to);
        l *= factor;
        m = to;
        if (begun) {
          // O of the keys before is complete: S of this tile was issued behind it (or it has been waited for above)
#pragma unroll
          for (int c = 0; c < kDim; c += 32) {
            uint32_t o[32];
            ptx::tmem_ld_32x32b_x32(o_at + c, o);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(as_float(o[i]) * factor);
            ptx::tmem_st_32x32b_x32(o_at + c, o);
          }
        }
      }
      begun = true;
      const float ref = m == -INFINITY ? 0.0f : m;
      const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), ref2 = pair(-ref, -ref);
      const int valid = seq.kl - k0;
      if (valid < kTile) {  // values behind the last key (the same for the whole group)
        const int s_v = (it - it0) % kStages;
        if (!(ok = warp_wait(v_full(s_v), ((it - it0) / kStages) & 1, a.wait, kSiteSmemFull))) break;
        zero_rows<kDim>(v_tile(s_v), row, valid);
      }
      uint64_t sum[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t p[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          float x, y;
          unpair(fma2(pair(as_float(s[i][2 * c]), as_float(s[i][2 * c + 1])), scale2, ref2), x, y);
          x = exp2_approx(x);
          y = exp2_approx(y);
          sum[i] = c ? add2(sum[i], pair(x, y)) : pair(x, y);
          p[c] = pack_bf16(x, y);
        }
        ptx::tmem_st_32x32b_x16(p_tmem(t) + lanes + i * 16, p);
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      warp_arrive(p_ready(t), lane);
      float l0, l1;
      unpair(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), l0, l1);
      l += l0 + l1;
    }
    if (ok && live) {
      const bool any = it0 < it1;
      if (any) ok = warp_wait(o_full, 0, a.wait, kSiteTmemFull);
      ptx::tc_fence_after();
      const bool mine = token < my_last;
      const bool seen = any && l != 0.0f;  // else a row with no visible key (of this split): zeros, -inf
      const float inverse = 1.0f / l;
      const float lse = seen ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
      const int64_t out_row = int64_t(seq.q0) + token;
      if (ok) {
        const int32_t part = a.paired ? 2 * split + t : split;
        const int64_t cell = ((int64_t(part) * a.batch + b) * a.q_len + token) * a.q_heads + head;
        if (mine) {
          if (a.parts > 1) a.partial_lse[cell] = lse;
          else if (a.lse != nullptr) a.lse[int64_t(head) * a.q_rows + out_row] = lse;
        }
#pragma unroll
        for (int c = 0; c < kDim; c += 32) {
          uint32_t o[32];
          __syncwarp();
          ptx::tmem_ld_32x32b_x32(o_at + c, o);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = seen ? __float_as_uint(as_float(o[i]) * inverse) : 0u;
          if (!mine) continue;
          if (a.parts > 1) {
            uint4* to = reinterpret_cast<uint4*>(a.partial + cell * kDim + c);
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          } else {
            uint4* to = reinterpret_cast<uint4*>(a.out + out_row * a.out_stride + int64_t(head) * kDim + c);
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = pack_bf16(as_float(o[2 * i]), as_float(o[2 * i + 1]));
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            if (a.rest != nullptr) {
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = rest_of_pair(w[i], as_float(o[2 * i]), as_float(o[2 * i + 1]));
              uint4* rest = reinterpret_cast<uint4*>(a.rest + (out_row * a.q_heads + head) * kDim + c);
#pragma unroll
              for (int i = 0; i < 2; ++i)
                rest[i] = make_uint4(w[8 * i] | (w[8 * i + 1] << 16), w[8 * i + 2] | (w[8 * i + 3] << 16),
                                     w[8 * i + 4] | (w[8 * i + 5] << 16), w[8 * i + 6] | (w[8 * i + 7] << 16));
            }
          }
        }
      }
    }
    unwound = !ok;
  }
  if (unwound) {  // a wait gave up: loads in flight get their time to land before shared memory goes away
    const uint64_t start = ptx::globaltimer();
    while (ptx::globaltimer() - start < 200000ull) __nanosleep(1000);
  }
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// Joins the parts: one warp per (token, head).
//   m = max lse_s, w_s = exp(lse_s - m), O = sum w_s O_s / sum w_s, lse = m + log sum w_s
template <int kDim>
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ Args a) {
  constexpr int kEach = kDim / 32;
  const int lane = threadIdx.x & 31;
  const int64_t cells = int64_t(a.batch) * a.q_len * a.q_heads;
  const int64_t cell = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (cell >= cells) return;
  const int32_t head = int32_t(cell % a.q_heads), token = int32_t(cell / a.q_heads % a.q_len);
  const Sequence seq = sequence(a, int32_t(cell / a.q_heads / a.q_len));
  if (token >= seq.ql) return;
  float m = -INFINITY;
  for (int32_t s = lane; s < a.parts; s += 32) m = fmaxf(m, a.partial_lse[s * cells + cell]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float sum = 0.0f, acc[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) acc[i] = 0.0f;
  const float ref = m == -INFINITY ? 0.0f : m;
  for (int32_t s = 0; s < a.parts; ++s) {
    const float w = exp2_approx((a.partial_lse[s * cells + cell] - ref) * kLog2e);
    if (w == 0.0f) continue;  // (the same for the whole warp)
    sum += w;
    const float* from = a.partial + (s * cells + cell) * kDim + lane * kEach;
#pragma unroll
    for (int i = 0; i < kEach; ++i) acc[i] = fmaf(w, from[i], acc[i]);
  }
  const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;
  const int64_t row = int64_t(seq.q0) + token;
  uint16_t* to = a.out + row * a.out_stride + int64_t(head) * kDim + lane * kEach;
  int8_t* rest = a.rest + (row * a.q_heads + head) * kDim + lane * kEach;
#pragma unroll
  for (int i = 0; i < kEach; i += 2) {
    const float x = acc[i] * inverse, y = acc[i + 1] * inverse;
    const uint32_t w = pack_bf16(x, y);
    *reinterpret_cast<uint32_t*>(to + i) = w;
    if (a.rest != nullptr) *reinterpret_cast<uint16_t*>(rest + i) = uint16_t(rest_of_pair(w, x, y));
  }
  if (lane == 0 && a.lse != nullptr)
    a.lse[int64_t(head) * a.q_rows + row] = sum != 0.0f ? m + logf(sum) : -INFINITY;
}

}  // namespace attn
}  // namespace fuse_b200
