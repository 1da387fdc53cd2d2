// Attention with a sliding window and sinks, backward: two kernels that recompute the weights from the forward's
// lse.
//
//   D = rowsum(dO (O + rest)),  P = exp(scale S - lse),  dP = dO V^T,  dS = P (dP - D)
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K
//
// The first kernel walks the key tiles of one query tile (D, which it leaves for the second, and dQ), the second the
// query tiles of one key tile (dK and dV, summed over the query heads that share the KV head).  S and dP
// are computed in both: seven products instead of the five of a single pass, but every sum stays in TMEM in a fixed
// order -- no atomics, the same bits every time, no FP32 copy of dQ in memory.
//
// Roles as in the forward kernel: loads, UMMA issue, TMEM, and eight warps of elementwise work, four per half of the
// columns, one thread per row and half.  The first kernel's dQ has an issuing warp of its own (192 -> 187 us at
// 8192 x 8 heads); the second kernel's four products keep one order, dV, S of the next tile, dK, dP of the next (two
// warps: 245 -> 319 us).  P and dS are rounded to BF16 for their products, as every operand of
// the tensor cores is; they are made from FP32 scores and dP and accumulated in FP32.  D is taken from the output and
// what its rounding took off: dS = P (dP - D) is small beside D where a row's weight lies on few keys, and D of the rounded output alone
// put dQ's relative error at 0.0046 for sequences of two tokens and at 0.0060 for scores of standard deviation 16 at any length,
// against 0.0027 and 0.0025 with the rest (0.0017 is the rounding of dQ itself).  Many keys of like weight hide it: 0.0024 and 0.0024.
#pragma once

#include "attention.cuh"

namespace fuse_b200 {
namespace attn {

struct BackwardArgs {
  Args f;
  const uint16_t *o, *d_o;
  int64_t o_stride, do_stride;
  const float* lse;
  float* delta;  // [q_heads][q_rows]
  uint16_t *dq, *dk, *dv;
  int64_t dq_stride, dk_stride, dv_stride;
  // The key gradients of a key tile that more than `chunk` query tiles see are made by several blocks.  The first
  // `long_tiles` key tiles of a sequence (all, or those with sinks where a window limits the others) have room for
  // `long_chunks` of them, the others for `short_chunks`.
  int32_t chunk, key_tiles, long_tiles, long_chunks, short_chunks;
  int32_t partial_chunks;  // of one sequence: all of its chunks, or none behind the long tiles' where those are alone
  float* partial;          // [batch][kv head][partial_chunks][dV, dK][128][head_dim]
  // chunk 0 of a key tile among the sequence's, and from one chunk to the next
  __device__ __forceinline__ int32_t first_chunk(int32_t tile) const {
    return tile < long_tiles ? tile : long_tiles * long_chunks + tile - long_tiles;
  }
  __device__ __forceinline__ int32_t chunk_step(int32_t tile) const { return tile < long_tiles ? long_tiles : key_tiles - long_tiles; }
};

constexpr int kBackwardThreads = 384, kElementwiseThreads = 256;

// The two halves of an operand in TMEM: K values 0..63 at `base`, 64..127 sixty-four columns on, so that
// each half of the warps writes over columns that it alone has read.
struct Halves {
  uint32_t base;
  __device__ __forceinline__ uint32_t operator()(uint32_t k) const { return base + (k / 4) * 64u + (k % 4) * 8u; }
};

// 32 accumulator columns of one row, scaled, as BF16.
__device__ __forceinline__ void store_row32(uint16_t* to, const uint32_t (&v)[32], float scale) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    reinterpret_cast<uint4*>(to)[i] = make_uint4(pack_bf16(as_float(v[8 * i]) * scale, as_float(v[8 * i + 1]) * scale),
                                                 pack_bf16(as_float(v[8 * i + 2]) * scale, as_float(v[8 * i + 3]) * scale),
                                                 pack_bf16(as_float(v[8 * i + 4]) * scale, as_float(v[8 * i + 5]) * scale),
                                                 pack_bf16(as_float(v[8 * i + 6]) * scale, as_float(v[8 * i + 7]) * scale));
}

template <int kDim>
struct QueryGradLayout {
  static constexpr int kKStages = kDim == 128 ? 3 : 4, kVStages = kDim == 128 ? 2 : 4;
  static constexpr uint32_t kTileBytes = TileShape<kDim>::kBytes;
  static constexpr uint32_t kQ = 0, kDo = kTileBytes, kK = 2 * kTileBytes, kV = kK + kKStages * kTileBytes;
  static constexpr uint32_t kBarriers = kV + kVStages * kTileBytes;
  // q_full, s_full, s_read, dp_full[2], ds_ready[2], ds_read[2], dq_full, drain[2], then k_full, k_empty, v_full, v_empty
  static constexpr uint32_t kNumBarriers = 12 + 2 * kKStages + 2 * kVStages;
  static constexpr uint32_t kSlot = kBarriers + kNumBarriers * 8;
  static constexpr uint32_t kDelta = (kSlot + 16 + 15) / 16 * 16;  // [2][128] partial sums
  static constexpr uint32_t kDynamicBytes = kDelta + 1024 + 1024;
  static_assert(kDynamicBytes <= 227 * 1024, "shared memory budget");
  static_assert(kDynamicBytes > 114 * 1024, "must force one CTA per SM (all of TMEM is allocated)");
};

template <int kDim>
__global__ void __launch_bounds__(kBackwardThreads, 1)
attention_query_grad_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                            const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                            const __grid_constant__ BackwardArgs ba) {
  using Layout = QueryGradLayout<kDim>;
  constexpr int kKStages = Layout::kKStages, kVStages = Layout::kVStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const Args& a = ba.f;
  const uint32_t base = ptx::smem_u32(smem_raw);
  const int warp = uniform(int32_t(threadIdx.x >> 5)), lane = threadIdx.x & 31;

  const int32_t tile_tokens = kTile >> a.pack_shift, packs = a.q_heads >> a.pack_shift;
  int32_t at = int32_t(blockIdx.x);
  const int32_t pack = at % packs;
  at /= packs;
  const int32_t b = at % a.batch;
  const int32_t token_blocks = (a.q_len + tile_tokens - 1) / tile_tokens;
  const int32_t first = (token_blocks - 1 - at / a.batch) * tile_tokens;
  const Sequence seq = sequence(a, b);
  if (first >= seq.ql) return;
  const int32_t last = min(first + tile_tokens, seq.ql);
  const int32_t head0 = pack << a.pack_shift, kv_head = head0 / (a.q_heads / a.kv_heads);
  const TileList tiles(KeyRange(a, seq, first, last));

  const uint32_t bars = base + Layout::kBarriers;
  const uint32_t q_full = bars, s_full = bars + 8, s_read = bars + 16, dq_full = bars + 72;
  auto dp_full = [&](uint32_t i) { return bars + 8u * (3 + i); };
  auto ds_ready = [&](uint32_t i) { return bars + 8u * (5 + i); };
  auto ds_read = [&](uint32_t i) { return bars + 8u * (7 + i); };
  auto drain = [&](uint32_t i) { return bars + 8u * (10 + i); };
  auto k_full = [&](uint32_t s) { return bars + 8u * (12 + s); };
  auto k_empty = [&](uint32_t s) { return bars + 8u * (12 + kKStages + s); };
  auto v_full = [&](uint32_t s) { return bars + 8u * (12 + 2 * kKStages + s); };
  auto v_empty = [&](uint32_t s) { return bars + 8u * (12 + 2 * kKStages + kVStages + s); };
  auto k_tile = [&](uint32_t s) { return base + Layout::kK + s * Layout::kTileBytes; };
  auto v_tile = [&](uint32_t s) { return base + Layout::kV + s * Layout::kTileBytes; };

  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_do);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(s_full, 1);
    ptx::mbar_init(s_read, 8);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(dp_full(i), 1);
      ptx::mbar_init(ds_ready(i), 8);
      ptx::mbar_init(ds_read(i), 1);
      ptx::mbar_init(drain(i), 1);
    }
    ptx::mbar_init(dq_full, 1);
    for (int s = 0; s < kKStages; ++s) {
      ptx::mbar_init(k_full(s), 1);
      ptx::mbar_init(k_empty(s), 1);
    }
    for (int s = 0; s < kVStages; ++s) {
      ptx::mbar_init(v_full(s), 1);
      ptx::mbar_init(v_empty(s), 1);
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
  const uint32_t s_tmem = tmem, dq_tmem = tmem + 384u;
  auto dp_tmem = [&](uint32_t i) { return tmem + 128u + i * 128u; };

  bool unwound = false;
  if (warp == 0) {
    if (lane == 0 && tiles.count > 0) {
      bool ok = true;
      ptx::mbar_expect_tx(q_full, 2 * Layout::kTileBytes);
      load_tile<kDim>(base + Layout::kQ, &map_q, q_full, head0, seq.q0 + first);
      load_tile<kDim>(base + Layout::kDo, &map_do, q_full, head0, seq.q0 + first);
      for (int32_t it = 0; it < tiles.count; ++it) {
        const uint32_t ks = it % kKStages, vs = it % kVStages;
        const int32_t row = seq.k0 + tiles.tile(it) * kTile;
        if (!(ok = mbar_wait<false>(k_empty(ks), ((it / kKStages) & 1) ^ 1u, a.wait, kSiteSmemEmpty))) break;
        ptx::mbar_expect_tx(k_full(ks), Layout::kTileBytes);
        load_tile<kDim>(k_tile(ks), &map_k, k_full(ks), kv_head, row);
        if (!(ok = mbar_wait<false>(v_empty(vs), ((it / kVStages) & 1) ^ 1u, a.wait, kSiteSmemEmpty))) break;
        ptx::mbar_expect_tx(v_full(vs), Layout::kTileBytes);
        load_tile<kDim>(v_tile(vs), &map_v, v_full(vs), kv_head, row);
      }
      unwound = !ok;
    }
  } else if (warp == 1) {
    // S and dP; the products that wait for the elementwise warps are another warp's, so neither holds the other up
    if (tiles.count > 0) {
      const uint32_t issue = ptx::elect_one();
      bool ok = warp_wait(q_full, 0, a.wait, kSiteSmemFull);
      uint32_t ks = 0, k_phase = 0, vs = 0, v_phase = 0;
      for (int32_t it = 0; ok && it < tiles.count; ++it) {
        if (!(ok = warp_wait(k_full(ks), k_phase, a.wait, kSiteSmemFull))) break;
        // the last tile's S is in registers
        if (it > 0 && !(ok = warp_wait(s_read, (it - 1) & 1, a.wait, kSiteTmemEmpty))) break;
        ptx::tc_fence_after();
        mma_rows<kDim>(issue, s_tmem, base + Layout::kQ, k_tile(ks));
        ptx::umma_commit_if(issue, s_full);
        if (++ks == kKStages) { ks = 0; k_phase ^= 1u; }
        if (!(ok = warp_wait(v_full(vs), v_phase, a.wait, kSiteSmemFull))) break;
        // dP alternates between two slots, whose dS the product two tiles ago has read
        if (it > 1 && !(ok = warp_wait(ds_read(it & 1), ((it >> 1) - 1) & 1, a.wait, kSiteTmemEmpty))) break;
        mma_rows<kDim>(issue, dp_tmem(it & 1), base + Layout::kDo, v_tile(vs));
        ptx::umma_commit_if(issue, dp_full(it & 1));
        ptx::umma_commit_if(issue, v_empty(vs));
        if (++vs == kVStages) { vs = 0; v_phase ^= 1u; }
      }
      if (!ok) {  // UMMAs already issued retire before TMEM is released
        ptx::umma_commit_if(issue, drain(0));
        mbar_wait<false>(drain(0), 0u, a.wait, kSiteDrain, false);
      }
      unwound = !ok;
    }
  } else if (warp == 2) {
    if (tiles.count > 0) {  // dQ
      const uint32_t issue = ptx::elect_one();
      bool ok = true;
      uint32_t ks = 0;
      for (int32_t it = 0; it < tiles.count; ++it) {
        if (!(ok = warp_wait(ds_ready(it & 1), (it >> 1) & 1, a.wait, kSiteTmemEmpty))) break;
        ptx::tc_fence_after();
        mma_weights<kDim>(issue, dq_tmem, Halves{dp_tmem(it & 1)}, k_tile(ks), it > 0);
        ptx::umma_commit_if(issue, ds_read(it & 1));
        ptx::umma_commit_if(issue, k_empty(ks));
        if (++ks == kKStages) ks = 0;
      }
      ptx::umma_commit_if(issue, ok ? dq_full : drain(1));
      if (!ok) mbar_wait<false>(drain(1), 0u, a.wait, kSiteDrain, false);
      unwound = !ok;
    }
  } else if (warp >= 4) {
    const int half = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16, columns = uint32_t(half) * 64u;
    const int32_t token = first + (row >> a.pack_shift), head = head0 + (row & (a.pack - 1));
    const bool mine = token < last;
    const int64_t q_row = int64_t(seq.q0) + token;
    // D of this row: each half sums its part of the columns
    float part = 0.0f;
    if (mine) {
      const uint4* o = reinterpret_cast<const uint4*>(ba.o + q_row * ba.o_stride + int64_t(head) * kDim + half * (kDim / 2));
      const uint4* g = reinterpret_cast<const uint4*>(ba.d_o + q_row * ba.do_stride + int64_t(head) * kDim + half * (kDim / 2));
      const uint2* r = a.rest ? reinterpret_cast<const uint2*>(a.rest + (q_row * a.q_heads + head) * kDim + half * (kDim / 2)) : nullptr;
#pragma unroll
      for (int i = 0; i < kDim / 16; ++i) {
        const uint4 x = o[i], y = g[i];
        const uint2 z = r != nullptr ? r[i] : make_uint2(0u, 0u);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[2] = {z.x, z.y};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int32_t bytes = int32_t(zs[j >> 1] << (j & 1 ? 0 : 16));  // of this pair, the upper half word
          part = fmaf(with_rest(xs[j] & 0xffffu, (bytes << 8) >> 24), as_float(ys[j] << 16), part);
          part = fmaf(with_rest(xs[j] >> 16, bytes >> 24), as_float(ys[j] & 0xffff0000u), part);
        }
      }
    }
    float* parts = reinterpret_cast<float*>(smem_raw + Layout::kDelta);
    parts[half * kTile + row] = part;
    __syncwarp();
    ptx::named_bar_sync(1, kElementwiseThreads);
    const float delta = parts[row] + parts[kTile + row];
    const int64_t stat = int64_t(head) * a.q_rows + q_row;
    float lse = INFINITY;  // rows that see nothing: every weight is exp(-inf)
    if (mine) {
      if (half == 0) ba.delta[stat] = delta;
      lse = ba.lse[stat] * kLog2e;
      if (lse == -INFINITY) lse = INFINITY;
    }
    __syncwarp();
    const int32_t pos = token + seq.off;
    const int32_t hi = a.causal ? min(pos, seq.kl - 1) : seq.kl - 1;
    const int32_t lo = a.causal && a.window > 0 ? pos - a.window + 1 : 0;
    const int32_t sinks = a.window > 0 ? a.sinks : 0;
    const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), minus_lse = pair(-lse, -lse), minus_delta = pair(-delta, -delta);
    bool ok = true;
    for (int32_t it = 0; it < tiles.count; ++it) {
      const int32_t tile = tiles.tile(it), k0 = tile * kTile;
      const uint32_t slot = it & 1;
      if (!(ok = warp_wait(s_full, it & 1, a.wait, kSiteTmemFull))) break;
      ptx::tc_fence_after();
      uint32_t s[2][32];
      ptx::tmem_ld_32x32b_x32(s_tmem + lanes + columns, s[0]);
      ptx::tmem_ld_32x32b_x32(s_tmem + lanes + columns + 32, s[1]);
      ptx::tmem_wait_ld();
      ptx::tc_fence_before();
      warp_arrive(s_read, lane);
      const bool masked = needs_mask(a, seq, first, last, k0, kTile);
      if (masked) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t seen = visible_keys(k0 + int32_t(columns) + i * 32, hi, lo, sinks);
#pragma unroll
          for (int c = 0; c < 32; ++c) s[i][c] = seen & (1u << c) ? s[i][c] : 0xff800000u;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          float x, y;
          unpair(fma2(pair(as_float(s[i][c]), as_float(s[i][c + 1])), scale2, minus_lse), x, y);
          s[i][c] = __float_as_uint(exp2_approx(x));
          s[i][c + 1] = __float_as_uint(exp2_approx(y));
        }
      if (k0 + kTile > seq.kl && half == 0) zero_rows<kDim>(k_tile(it % kKStages), row, seq.kl - k0);  // S has read it
      if (!(ok = warp_wait(dp_full(slot), (it >> 1) & 1, a.wait, kSiteTmemFull))) break;
      ptx::tc_fence_after();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t dp[32], ds[16];
        ptx::tmem_ld_32x32b_x32(dp_tmem(slot) + lanes + columns + i * 32, dp);
        ptx::tmem_wait_ld();
        if (masked) {  // dP of a key nobody may see can be anything
#pragma unroll
          for (int c = 0; c < 32; ++c) dp[c] = s[i][c] != 0u ? dp[c] : __float_as_uint(delta);
        }
#pragma unroll
        for (int c = 0; c < 16; ++c)
          ds[c] = pack_bf16_pair(mul2(pair(as_float(s[i][2 * c]), as_float(s[i][2 * c + 1])),
                                      add2(pair(as_float(dp[2 * c]), as_float(dp[2 * c + 1])), minus_delta)));
        ptx::tmem_st_32x32b_x16(dp_tmem(slot) + lanes + columns + i * 16, ds);
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      warp_arrive(ds_ready(slot), lane);
    }
    if (ok) {
      if (tiles.count > 0) ok = warp_wait(dq_full, 0, a.wait, kSiteTmemFull);
      ptx::tc_fence_after();
      if (ok) {
#pragma unroll
        for (int c = 0; c < kDim / 2; c += 32) {
          uint32_t v[32];
          const int32_t column = half * (kDim / 2) + c;
          __syncwarp();
          ptx::tmem_ld_32x32b_x32(dq_tmem + lanes + uint32_t(column), v);
          ptx::tmem_wait_ld();
          if (tiles.count == 0) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
          }
          if (mine) store_row32(ba.dq + q_row * ba.dq_stride + int64_t(head) * kDim + column, v, a.scale);
        }
      }
    }
    unwound = !ok;
  }
  if (unwound) {
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

// ------------------------------------------------------------------------------------------------ dK, dV
template <int kDim>
struct KeyGradLayout {
  static constexpr int kStages = kDim == 128 ? 2 : 4;  // of Q and of dO
  static constexpr uint32_t kTileBytes = TileShape<kDim>::kBytes;
  static constexpr uint32_t kK = 0, kV = kTileBytes, kQ = 2 * kTileBytes, kDo = kQ + kStages * kTileBytes;
  static constexpr uint32_t kStats = kDo + kStages * kTileBytes;  // [2][-lse, -D][128]
  static constexpr uint32_t kBarriers = kStats + 2 * 2 * kTile * 4;
  // kv_full, s_full, dp_full, p_ready, ds_ready, grads_full, drain, stat_full[2], stat_empty[2],
  // then q_full, q_empty, do_full, do_empty
  static constexpr uint32_t kNumBarriers = 11 + 4 * kStages;
  static constexpr uint32_t kSlot = kBarriers + kNumBarriers * 8;
  static constexpr uint32_t kDynamicBytes = kSlot + 16 + 1024;
  static_assert(kDynamicBytes <= 227 * 1024, "shared memory budget");
  static_assert(kDynamicBytes > 114 * 1024, "must force one CTA per SM (all of TMEM is allocated)");
};

// The query tiles that see a key tile: token tiles [first, first + count) of every head pack of the group.
struct QueryTiles {
  int32_t first, count;
  __device__ __forceinline__ QueryTiles(const Args& a, const Sequence& s, int32_t key_tile, int32_t tile_tokens) {
    const int32_t k0 = key_tile * kTile, k1 = min(k0 + kTile, s.kl);
    int32_t from = 0, to = s.ql;
    if (a.causal) {
      from = max(0, k0 - s.off);
      if (a.window > 0 && k0 >= a.sinks) to = min(to, k1 - 1 + a.window - s.off);
    }
    first = from / tile_tokens;
    count = to > from ? (to + tile_tokens - 1) / tile_tokens - first : 0;
  }
};

template <int kDim>
__global__ void __launch_bounds__(kBackwardThreads, 1)
attention_key_grad_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_do,
                          const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const __grid_constant__ BackwardArgs ba) {
  using Layout = KeyGradLayout<kDim>;
  constexpr int kStages = Layout::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const Args& a = ba.f;
  const uint32_t base = ptx::smem_u32(smem_raw);
  const int warp = uniform(int32_t(threadIdx.x >> 5)), lane = threadIdx.x & 31;

  // first chunks come first, last chunks, which few key tiles have, last
  const int32_t tile_tokens = kTile >> a.pack_shift;
  int32_t at = int32_t(blockIdx.x);
  const int32_t kv_head = at % a.kv_heads;
  at /= a.kv_heads;
  const int32_t b = at % a.batch, slot = at / a.batch;
  const bool is_long = slot < ba.long_tiles * ba.long_chunks;
  const int32_t among = is_long ? slot : slot - ba.long_tiles * ba.long_chunks, tiles_alike = is_long ? ba.long_tiles : ba.key_tiles - ba.long_tiles;
  const int32_t chunk = among / tiles_alike, key_tile = among - chunk * tiles_alike + (is_long ? 0 : ba.long_tiles), k0 = key_tile * kTile;
  const Sequence seq = sequence(a, b);
  if (k0 >= seq.kl) return;
  const QueryTiles tiles(a, seq, key_tile, tile_tokens);
  const int32_t group = a.q_heads / a.kv_heads, packs = group >> a.pack_shift, head_base = kv_head * group;
  const int32_t all = tiles.count * packs, chunks = (all + ba.chunk - 1) / ba.chunk;
  if (chunk > 0 && chunk >= chunks) return;
  // this block's part: query tiles [j0, j0 + total) of the list (token tiles of one head pack after another)
  const int32_t j0 = chunk * ba.chunk, total = min(all - j0, ba.chunk);
  auto first_token = [&](int32_t j) { return (tiles.first + (j0 + j) % tiles.count) * tile_tokens; };
  auto first_head = [&](int32_t j) { return head_base + (((j0 + j) / tiles.count) << a.pack_shift); };

  const uint32_t bars = base + Layout::kBarriers;
  const uint32_t kv_full = bars, s_full = bars + 8, dp_full = bars + 16, p_ready = bars + 24, ds_ready = bars + 32;
  const uint32_t grads_full = bars + 40, drain = bars + 48;
  auto stat_full = [&](uint32_t i) { return bars + 56u + 8u * i; };
  auto stat_empty = [&](uint32_t i) { return bars + 72u + 8u * i; };
  auto q_full = [&](uint32_t s) { return bars + 8u * (11 + s); };
  auto q_empty = [&](uint32_t s) { return bars + 8u * (11 + kStages + s); };
  auto do_full = [&](uint32_t s) { return bars + 8u * (11 + 2 * kStages + s); };
  auto do_empty = [&](uint32_t s) { return bars + 8u * (11 + 3 * kStages + s); };
  float* stats = reinterpret_cast<float*>(smem_raw + Layout::kStats);
  auto q_tile = [&](uint32_t s) { return base + Layout::kQ + s * Layout::kTileBytes; };
  auto do_tile = [&](uint32_t s) { return base + Layout::kDo + s * Layout::kTileBytes; };

  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&map_q);
    ptx::prefetch_tensormap(&map_do);
    ptx::prefetch_tensormap(&map_k);
    ptx::prefetch_tensormap(&map_v);
    ptx::mbar_init(kv_full, 1);
    ptx::mbar_init(s_full, 1);
    ptx::mbar_init(dp_full, 1);
    ptx::mbar_init(p_ready, 8);
    ptx::mbar_init(ds_ready, 8);
    ptx::mbar_init(grads_full, 1);
    ptx::mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(stat_full(i), 1);
      ptx::mbar_init(stat_empty(i), 8);
    }
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(q_full(s), 1);
      ptx::mbar_init(q_empty(s), 1);
      ptx::mbar_init(do_full(s), 1);
      ptx::mbar_init(do_empty(s), 1);
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
  const uint32_t s_tmem = tmem, dp_tmem = tmem + 128u, dv_tmem = tmem + 256u, dk_tmem = tmem + 384u;

  bool unwound = false;
  if (warp == 0) {
    if (lane == 0 && total > 0) {
      bool ok = true;
      ptx::mbar_expect_tx(kv_full, 2 * Layout::kTileBytes);
      load_tile<kDim>(base + Layout::kK, &map_k, kv_full, kv_head, seq.k0 + k0);
      load_tile<kDim>(base + Layout::kV, &map_v, kv_full, kv_head, seq.k0 + k0);
      for (int32_t j = 0; j < total; ++j) {
        const uint32_t s = j % kStages, phase = ((j / kStages) & 1) ^ 1u;
        const int32_t row = seq.q0 + first_token(j), head = first_head(j);
        if (!(ok = mbar_wait<false>(q_empty(s), phase, a.wait, kSiteSmemEmpty))) break;
        ptx::mbar_expect_tx(q_full(s), Layout::kTileBytes);
        load_tile<kDim>(q_tile(s), &map_q, q_full(s), head, row);
        if (!(ok = mbar_wait<false>(do_empty(s), phase, a.wait, kSiteSmemEmpty))) break;
        ptx::mbar_expect_tx(do_full(s), Layout::kTileBytes);
        load_tile<kDim>(do_tile(s), &map_do, do_full(s), head, row);
      }
      unwound = !ok;
    }
  } else if (warp == 1) {
    if (total > 0) {
      // P overwrites S and dS overwrites dP; the UMMAs' issue order keeps each from being overwritten too early
      const uint32_t issue = ptx::elect_one();
      bool ok = warp_wait(kv_full, 0, a.wait, kSiteSmemFull);
      uint32_t s = 0, s_next = 0, phase = 0;  // stages of tiles j and j + 1, phase of the latter
      for (int32_t j = -1; ok && j < total; ++j) {
        const bool now = j >= 0, next = j + 1 < total;
        if (now) {
          if (!(ok = warp_wait(p_ready, j & 1, a.wait, kSiteTmemEmpty))) break;
          ptx::tc_fence_after();
          mma_weights<kDim>(issue, dv_tmem, Halves{s_tmem}, do_tile(s), j > 0);
          ptx::umma_commit_if(issue, do_empty(s));
        }
        if (next) {
          if (!(ok = warp_wait(q_full(s_next), phase, a.wait, kSiteSmemFull))) break;
          mma_rows<kDim>(issue, s_tmem, base + Layout::kK, q_tile(s_next));
          ptx::umma_commit_if(issue, s_full);
        }
        if (now) {
          if (!(ok = warp_wait(ds_ready, j & 1, a.wait, kSiteTmemEmpty))) break;
          ptx::tc_fence_after();
          mma_weights<kDim>(issue, dk_tmem, Halves{dp_tmem}, q_tile(s), j > 0);
          ptx::umma_commit_if(issue, q_empty(s));
        }
        if (next) {
          if (!(ok = warp_wait(do_full(s_next), phase, a.wait, kSiteSmemFull))) break;
          mma_rows<kDim>(issue, dp_tmem, base + Layout::kV, do_tile(s_next));
          ptx::umma_commit_if(issue, dp_full);
        }
        s = s_next;
        if (++s_next == kStages) { s_next = 0; phase ^= 1u; }
      }
      ptx::umma_commit_if(issue, ok ? grads_full : drain);
      if (!ok) mbar_wait<false>(drain, 0u, a.wait, kSiteDrain, false);
      unwound = !ok;
    }
  } else if (warp == 3) {
    // -lse (in log2 units) and -D of the rows of every query tile, two tiles ahead at most
    bool ok = true;
    for (int32_t j = 0; j < total; ++j) {
      const int32_t t0 = first_token(j), head = first_head(j);
      float lse[4], delta[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t r = i * 32 + lane, token = t0 + (r >> a.pack_shift);
        const int64_t stat = int64_t(head + (r & (a.pack - 1))) * a.q_rows + seq.q0 + token;
        const bool there = token < seq.ql;
        lse[i] = there ? -ba.lse[stat] * kLog2e : -INFINITY;
        delta[i] = there ? -ba.delta[stat] : 0.0f;
        if (lse[i] == INFINITY) lse[i] = -INFINITY;  // a row that sees nothing: every weight is exp(-inf)
      }
      if (!(ok = warp_wait(stat_empty(j & 1), ((j >> 1) & 1) ^ 1u, a.wait, kSiteSmemEmpty))) break;
      float* mine = stats + (j & 1) * 2 * kTile;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mine[i * 32 + lane] = lse[i];
        mine[kTile + i * 32 + lane] = delta[i];
      }
      warp_arrive(stat_full(j & 1), lane);
    }
    unwound = !ok;
  } else if (warp >= 4) {
    const int half = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16, columns = uint32_t(half) * 64u;
    const int32_t key = k0 + row;
    // the tokens that see this key: [from, to)
    const int32_t from = a.causal ? key - seq.off : 0;
    const int32_t to = key >= seq.kl ? 0 : a.causal && a.window > 0 && key >= a.sinks ? min(seq.ql, key + a.window - seq.off) : seq.ql;
    const uint64_t scale2 = pair(a.scale_log2, a.scale_log2);
    bool ok = true;
    for (int32_t j = 0; j < total; ++j) {
      const uint32_t stage = j % kStages;
      const float* mine = stats + (j & 1) * 2 * kTile;
      const int32_t t0 = first_token(j);
      const bool tail = t0 + tile_tokens > seq.ql;
      // every (key, query) pair visible: the tile's last key is seen by its first query and its first key by its last
      const bool masked = tail || k0 + kTile > seq.kl ||
                          (a.causal && (t0 + seq.off < k0 + kTile - 1 ||
                                        (a.window > 0 && k0 + kTile > a.sinks && t0 + tile_tokens - 1 + seq.off - k0 >= a.window)));
      if (!(ok = warp_wait(stat_full(j & 1), (j >> 1) & 1, a.wait, kSiteSmemFull))) break;
      if (!(ok = warp_wait(s_full, j & 1, a.wait, kSiteTmemFull))) break;
      ptx::tc_fence_after();
      uint32_t p[2][32];
      ptx::tmem_ld_32x32b_x32(s_tmem + lanes + columns, p[0]);
      ptx::tmem_ld_32x32b_x32(s_tmem + lanes + columns + 32, p[1]);
      ptx::tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const ulonglong2* lse = reinterpret_cast<const ulonglong2*>(mine + columns + i * 32);
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const ulonglong2 v = lse[c / 4];
          float x, y;
          unpair(fma2(pair(as_float(p[i][c]), as_float(p[i][c + 1])), scale2, v.x), x, y);
          p[i][c] = __float_as_uint(exp2_approx(x));
          p[i][c + 1] = __float_as_uint(exp2_approx(y));
          unpair(fma2(pair(as_float(p[i][c + 2]), as_float(p[i][c + 3])), scale2, v.y), x, y);
          p[i][c + 2] = __float_as_uint(exp2_approx(x));
          p[i][c + 3] = __float_as_uint(exp2_approx(y));
        }
      }
      if (masked) {
        // the columns of tokens [from, to): those in [low, high).  Tokens are brought into the tile before they are multiplied by its
        // heads: in a tile with sinks `to` can lie a whole context away, and that times 128 heads is past 31 bits
        const int32_t low = min(max(from - t0, 0), tile_tokens) << a.pack_shift, high = min(max(to - t0, 0), tile_tokens) << a.pack_shift;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int32_t at = int32_t(columns) + i * 32;
          const uint32_t seen = low_bits(high - at) & ~low_bits(low - at);
#pragma unroll
          for (int c = 0; c < 32; ++c) p[i][c] = seen & (1u << c) ? p[i][c] : 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t w[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) w[c] = pack_bf16(as_float(p[i][2 * c]), as_float(p[i][2 * c + 1]));
        ptx::tmem_st_32x32b_x16(s_tmem + lanes + columns + i * 16, w);
      }
      if (tail) {  // rows behind the last query take part in dV and dK as zeros
        if (!(ok = warp_wait(do_full(stage), (j / kStages) & 1, a.wait, kSiteSmemFull))) break;
        const int32_t valid = (seq.ql - t0) << a.pack_shift;
        zero_rows<kDim>(half == 0 ? do_tile(stage) : q_tile(stage), row, valid);
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      warp_arrive(p_ready, lane);
      if (!(ok = warp_wait(dp_full, j & 1, a.wait, kSiteTmemFull))) break;
      ptx::tc_fence_after();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t dp[32], ds[16];
        ptx::tmem_ld_32x32b_x32(dp_tmem + lanes + columns + i * 32, dp);
        ptx::tmem_wait_ld();
        const ulonglong2* delta = reinterpret_cast<const ulonglong2*>(mine + kTile + columns + i * 32);
        uint64_t d[16];
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const ulonglong2 v = delta[c / 2];
          d[c] = add2(pair(as_float(dp[2 * c]), as_float(dp[2 * c + 1])), v.x);
          d[c + 1] = add2(pair(as_float(dp[2 * c + 2]), as_float(dp[2 * c + 3])), v.y);
        }
        if (masked) {  // dP of a pair that does not count can be anything
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float x, y;
            unpair(d[c], x, y);
            d[c] = pair(p[i][2 * c] != 0u ? x : 0.0f, p[i][2 * c + 1] != 0u ? y : 0.0f);
          }
        }
#pragma unroll
        for (int c = 0; c < 16; ++c) ds[c] = pack_bf16_pair(mul2(pair(as_float(p[i][2 * c]), as_float(p[i][2 * c + 1])), d[c]));
        ptx::tmem_st_32x32b_x16(dp_tmem + lanes + columns + i * 16, ds);
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        ptx::mbar_arrive(stat_empty(j & 1));
        ptx::mbar_arrive(ds_ready);
      }
      __syncwarp();
    }
    if (ok) {
      if (total > 0) ok = warp_wait(grads_full, 0, a.wait, kSiteTmemFull);
      ptx::tc_fence_after();
      if (ok) {
        const bool mine = key < seq.kl;
        const int64_t kv_row = int64_t(seq.k0) + key;
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
          for (int c = 0; c < kDim / 2; c += 32) {
            uint32_t v[32];
            const int32_t column = half * (kDim / 2) + c;
            __syncwarp();
            ptx::tmem_ld_32x32b_x32((which ? dk_tmem : dv_tmem) + lanes + uint32_t(column), v);
            ptx::tmem_wait_ld();
            if (total == 0) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0u;
            }
            if (!mine) continue;
            if (chunks > 1) {
              const int64_t place = (int64_t(b) * a.kv_heads + kv_head) * ba.partial_chunks + slot;
              uint4* to4 = reinterpret_cast<uint4*>(ba.partial + ((place * 2 + which) * kTile + row) * kDim + column);
#pragma unroll
              for (int i = 0; i < 8; ++i) to4[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            } else {
              store_row32((which ? ba.dk + kv_row * ba.dk_stride : ba.dv + kv_row * ba.dv_stride) + int64_t(kv_head) * kDim + column,
                          v, which ? a.scale : 1.0f);
            }
          }
      }
    }
    unwound = !ok;
  }
  if (unwound) {
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

// Sums the chunks of a key tile in their order.  A block per key tile, four columns per thread and step.
template <int kDim>
__global__ void __launch_bounds__(256) attention_key_grad_join_kernel(const __grid_constant__ BackwardArgs ba) {
  const Args& a = ba.f;
  int32_t at = int32_t(blockIdx.x);
  const int32_t kv_head = at % a.kv_heads;
  at /= a.kv_heads;
  const int32_t b = at % a.batch, key_tile = at / a.batch, k0 = key_tile * kTile;
  const Sequence seq = sequence(a, b);
  if (k0 >= seq.kl) return;
  const int32_t all = QueryTiles(a, seq, key_tile, kTile >> a.pack_shift).count * ((a.q_heads / a.kv_heads) >> a.pack_shift);
  const int32_t chunks = (all + ba.chunk - 1) / ba.chunk;
  if (chunks <= 1) return;
  const int64_t place = (int64_t(b) * a.kv_heads + kv_head) * ba.partial_chunks + ba.first_chunk(key_tile);
  const int64_t step = int64_t(ba.chunk_step(key_tile)) * 2 * kTile * kDim;
  const int32_t rows = min(kTile, seq.kl - k0);
  constexpr int kVectors = kDim / 4;
  for (int32_t i = int32_t(blockIdx.y) * 256 + threadIdx.x; i < 2 * rows * kVectors; i += int32_t(gridDim.y) * 256) {
    const int32_t which = i / (rows * kVectors), rest = i - which * rows * kVectors, row = rest / kVectors, column = rest % kVectors * 4;
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float* from = ba.partial + ((place * 2 + which) * kTile + row) * kDim + column;
    for (int32_t c = 0; c < chunks; ++c) {
      const float4 v = *reinterpret_cast<const float4*>(from + c * step);
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
    const float scale = which ? a.scale : 1.0f;
    const int64_t kv_row = int64_t(seq.k0) + k0 + row;
    uint16_t* to = (which ? ba.dk + kv_row * ba.dk_stride : ba.dv + kv_row * ba.dv_stride) + int64_t(kv_head) * kDim + column;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(sum.x * scale, sum.y * scale), pack_bf16(sum.z * scale, sum.w * scale));
  }
}

}  // namespace attn
}  // namespace fuse_b200
