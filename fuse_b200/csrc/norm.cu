// Root-mean-square norm with the residual's addition, BF16 or MXFP8 out, and its backward.
//
//   h = bf16(x + res);  r = (mean(h^2) + eps)^(-1/2);  y = h r g
//   n = h r;  dn = dy g;  dx = dh + r (dn - n mean(dn n));  dg = sum over rows of dy n
//
// The norm is that of the ROUNDED stream h: the backward reads h and so differentiates exactly what
// the forward computed.  Sums and means are FP32; every output is rounded once, except the MXFP8 form,
// which is by definition the quantisation of the BF16 output (so that a caller may mix the two).
//
// Bound by HBM: the forward moves 8 bytes per element (7.03 with MXFP8 out), the backward 8.  A row
// stays in registers between its sum and its scaling, so every element is read once; it belongs to a warp
// or to a block (16-byte vectors, two to four per thread: with four in the forward the registers thin
// the SM out, 16384 x 4096 to MXFP8 100 us against 91).  The backward of wide rows stages them in shared memory instead.
// Blocks walk the rows with the grid's stride and keep gamma in registers.  Measured: forward 8191 x 8192 80 us (6.7 TB/s), backward
// 82 us (6.6) and 6 for the join of dgamma; 16384 x 4096 to MXFP8 91 us (5.2 TB/s: conversions and scale words share the issue slots).
#include "launch.cuh"

namespace fuse_b200 {
namespace {

using host::DeviceInfo;

struct NormArgs {
  const uint16_t *x, *res, *gamma;
  uint16_t *h, *y;
  uint8_t *data, *scales;
  int64_t x_stride, res_stride, h_stride, y_stride, rows;
  int32_t hidden;
  float eps;
};

struct NormGradArgs {
  const uint16_t *dy, *h, *gamma, *dh;
  uint16_t* dx;
  float* partial;  // [row groups of the grid][hidden], or nullptr
  WaitContext wait;
  int64_t dy_stride, h_stride, dh_stride, dx_stride, rows;
  int32_t hidden;
  float eps;
};

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
}
__device__ __forceinline__ uint4 load16(const uint16_t* p) { return *reinterpret_cast<const uint4*>(p); }

constexpr int kVectors = 2;                // of a thread in a block per row
constexpr int kMaxWarps = 64 / kVectors;  // of a block, which has one row

// Sum over the threads of one row, a warp or the block; `slot` alternates from row to row, so that one barrier per
// row is enough (a slot is written again only after the barrier of the row in between).
template <bool kWarpRow, int kValues>
__device__ __forceinline__ void row_sum(float (&v)[kValues], float* scratch, int slot) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < kValues; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if constexpr (!kWarpRow) {
    const int warps = int(blockDim.x) >> 5;
    float* mine = scratch + slot * kMaxWarps * kValues;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < kValues; ++i) mine[(threadIdx.x >> 5) * kValues + i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kValues; ++i) v[i] = 0.0f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
      for (int i = 0; i < kValues; ++i) v[i] += mine[w * kValues + i];
  }
}

// Squares of values past 2^64 leave FP32's range although the values and the result lie within BF16's: a row
// whose sum did is summed again with its values scaled by 2^-72 (2^56 at most, 2^126 the sum of 16384 squares).
constexpr float kTooLarge = 1.7014118e38f;           // 2^127
constexpr float kDown = 2.1175823681357508e-22f;     // 2^-72
constexpr float kMinEpsilon = 1e-30f;

// A warp per row (four rows to a block), or a block.
template <bool kWarpRow, int kVec, bool kMx>
__global__ void __launch_bounds__(kWarpRow ? 128 : 32 * kMaxWarps) rms_norm_kernel(const NormArgs a) {
  __shared__ float scratch[2 * kMaxWarps];
  const int threads = kWarpRow ? 32 : int(blockDim.x), rows_of_block = kWarpRow ? 4 : 1;
  const int t = kWarpRow ? threadIdx.x & 31 : threadIdx.x;
  uint4 gamma[kVec];
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int32_t c = (j * threads + t) * 8;
    gamma[j] = c < a.hidden ? load16(a.gamma + c) : make_uint4(0u, 0u, 0u, 0u);
  }
  const float inv = 1.0f / float(a.hidden);
  // with MXFP8 out the rows up to the next multiple of 128 get neutral scales
  const int64_t last = kMx ? (a.rows + 127) & ~int64_t(127) : a.rows;
  const int64_t k_atoms = (int64_t(a.hidden) + 127) >> 7;
  int slot = 0;
  for (int64_t row = int64_t(blockIdx.x) * rows_of_block + (kWarpRow ? threadIdx.x >> 5 : 0); row < last;
       row += int64_t(gridDim.x) * rows_of_block) {
    if (kMx && row >= a.rows) {  // (the same for all threads of the row)
      for (int64_t atom = t; atom < k_atoms; atom += threads)
        *reinterpret_cast<uint32_t*>(a.scales + mxfp8_scale_offset(row, atom << 7, k_atoms)) = 0x7f7f7f7fu;
      continue;
    }
    uint4 h[kVec], res[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * threads + t) * 8;
      h[j] = res[j] = make_uint4(0u, 0u, 0u, 0u);
      if (c < a.hidden) {
        h[j] = load16(a.x + row * a.x_stride + c);
        if (a.res != nullptr) res[j] = load16(a.res + row * a.res_stride + c);
      }
    }
    float sum[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * threads + t) * 8;
      float f[8];
      if (a.res != nullptr) {
        float g[8];
        unpack8(h[j], f);
        unpack8(res[j], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += g[i];
        h[j] = pack8(f);
      }
      if (a.h != nullptr && c < a.hidden) *reinterpret_cast<uint4*>(a.h + row * a.h_stride + c) = h[j];
      unpack8(h[j], f);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[0] = fmaf(f[i], f[i], sum[0]);
    }
    row_sum<kWarpRow, 1>(sum, scratch, slot);
    slot ^= 1;
    float r = rsqrtf(fmaf(sum[0], inv, a.eps));
    if (!(sum[0] < kTooLarge)) {  // (the same for all threads of the row)
      sum[0] = 0.0f;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        float f[8];
        unpack8(h[j], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[0] = fmaf(f[i] * kDown, f[i] * kDown, sum[0]);
      }
      row_sum<kWarpRow, 1>(sum, scratch, slot);
      slot ^= 1;
      r = rsqrtf(sum[0] * inv) * kDown;  // epsilon is far below the last bit
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * threads + t) * 8;
      float f[8], g[8];
      unpack8(h[j], f);
      unpack8(gamma[j], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * r * g[i];
      const uint4 y = pack8(f);
      if (a.y != nullptr && c < a.hidden) *reinterpret_cast<uint4*>(a.y + row * a.y_stride + c) = y;
      if constexpr (kMx) {
        // four neighbouring threads hold one group of 32; sixteen hold one K atom of the row, whose
        // four scale bytes are one aligned word (threads past the row bring zeros: 2^0)
        unpack8(y, f);
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(f[i]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int exponent = mxfp8_scale_exponent(amax);
        const float inverse = mxfp8_inverse_scale(exponent);
        if (c < a.hidden) {
          const uint2 bytes = make_uint2(pack_e4m3x4(f[0] * inverse, f[1] * inverse, f[2] * inverse, f[3] * inverse),
                                         pack_e4m3x4(f[4] * inverse, f[5] * inverse, f[6] * inverse, f[7] * inverse));
          *reinterpret_cast<uint2*>(a.data + row * a.hidden + c) = bytes;
        }
        uint32_t word = uint32_t(exponent + 127) << (8 * ((t >> 2) & 3));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if ((t & 15) == 0 && c < a.hidden)
          *reinterpret_cast<uint32_t*>(a.scales + mxfp8_scale_offset(row, c, k_atoms)) = word;
      }
    }
  }
}

// The row's share of both outputs, from one vector of its elements.
__device__ __forceinline__ void grad_vector(const uint4& h, const uint4& dy, const uint4& gamma, const uint4& dh, float r, float mean,
                                            float (&acc)[8], uint16_t* to) {
  float fh[8], fd[8], fg[8], out[8];
  unpack8(h, fh);
  unpack8(dy, fd);
  unpack8(gamma, fg);
  unpack8(dh, out);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float n = fh[i] * r;
    acc[i] = fmaf(fd[i], n, acc[i]);
    out[i] = fmaf(r, fmaf(fd[i], fg[i], -n * mean), out[i]);
  }
  *reinterpret_cast<uint4*>(to) = pack8(out);
}
// What a vector adds to the sums of h^2 and of dy g h, h scaled by `down`.
__device__ __forceinline__ void grad_sums(const uint4& h, const uint4& dy, const uint4& gamma, float down, float (&sum)[2]) {
  float fh[8], fd[8], fg[8];
  unpack8(h, fh);
  unpack8(dy, fd);
  unpack8(gamma, fg);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = fh[i] * down;
    sum[0] = fmaf(x, x, sum[0]);
    sum[1] = fmaf(fd[i] * fg[i], x, sum[1]);
  }
}
__device__ __forceinline__ void store_share(const float (&acc)[8], float* to) {
  reinterpret_cast<float4*>(to)[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
  reinterpret_cast<float4*>(to)[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
}

// Backward, a warp per row (hidden up to 512): the row stays in registers, as does the warp's share of the gamma
// gradient, which it writes as one row of `partial`.
template <int kVec>
__global__ void __launch_bounds__(128) rms_norm_backward_warp_kernel(const NormGradArgs a) {
  const int t = threadIdx.x & 31;
  uint4 gamma[kVec];
  float acc[kVec][8];
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int32_t c = (j * 32 + t) * 8;
    gamma[j] = c < a.hidden ? load16(a.gamma + c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[j][i] = 0.0f;
  }
  const float inv = 1.0f / float(a.hidden);
  const int64_t group = int64_t(blockIdx.x) * 4 + threadIdx.x / 32;
  for (int64_t row = group; row < a.rows; row += int64_t(gridDim.x) * 4) {
    uint4 h[kVec], dy[kVec], dh[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * 32 + t) * 8;
      h[j] = dy[j] = dh[j] = make_uint4(0u, 0u, 0u, 0u);
      if (c < a.hidden) {
        h[j] = load16(a.h + row * a.h_stride + c);
        dy[j] = load16(a.dy + row * a.dy_stride + c);
        if (a.dh != nullptr) dh[j] = load16(a.dh + row * a.dh_stride + c);
      }
    }
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kVec; ++j) grad_sums(h[j], dy[j], gamma[j], 1.0f, sum);
    row_sum<true, 2>(sum, nullptr, 0);
    float r = rsqrtf(fmaf(sum[0], inv, a.eps)), mean = sum[1] * inv * r;  // mean(dn n)
    if (!(sum[0] < kTooLarge)) {
      sum[0] = sum[1] = 0.0f;
#pragma unroll
      for (int j = 0; j < kVec; ++j) grad_sums(h[j], dy[j], gamma[j], kDown, sum);
      row_sum<true, 2>(sum, nullptr, 0);
      r = rsqrtf(sum[0] * inv);
      mean = sum[1] * inv * r;
      r *= kDown;
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * 32 + t) * 8;
      if (c < a.hidden) grad_vector(h[j], dy[j], gamma[j], dh[j], r, mean, acc[j], a.dx + row * a.dx_stride + c);
    }
  }
  if (a.partial != nullptr) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * 32 + t) * 8;
      if (c < a.hidden) store_share(acc[j], a.partial + group * a.hidden + c);
    }
  }
}

// Backward, a block per row: the three input rows arrive in shared memory by bulk copies, two rows of the block's walk
// in flight, so that loads go on across the row's two barriers.
__global__ void __launch_bounds__(512) rms_norm_backward_kernel(const NormGradArgs a) {
  constexpr int kVec = 4, kStages = 2;
  extern __shared__ __align__(128) uint8_t rows_shared[];  // [kStages][h, dy, dh][hidden]
  __shared__ float scratch[2 * kMaxWarps * 2];
  __shared__ __align__(8) uint64_t bars[kStages];
  const int t = threadIdx.x, threads = blockDim.x;
  const uint32_t row_bytes = uint32_t(a.hidden) * 2, inputs = a.dh != nullptr ? 3u : 2u;
  const uint32_t base = ptx::smem_u32(rows_shared);
  auto bar = [&](int s) { return ptx::smem_u32(bars + s); };
  auto fetch = [&](int s, int64_t row) {  // one thread
    const uint32_t to = base + uint32_t(s) * 3 * row_bytes;
    ptx::mbar_expect_tx(bar(s), inputs * row_bytes);
    ptx::bulk_load(to, a.h + row * a.h_stride, row_bytes, bar(s));
    ptx::bulk_load(to + row_bytes, a.dy + row * a.dy_stride, row_bytes, bar(s));
    if (a.dh != nullptr) ptx::bulk_load(to + 2 * row_bytes, a.dh + row * a.dh_stride, row_bytes, bar(s));
  };
  if (t == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(bar(s), 1);
    ptx::fence_mbar_init();
    for (int s = 0; s < kStages; ++s)
      if (blockIdx.x + int64_t(s) * gridDim.x < a.rows) fetch(s, blockIdx.x + int64_t(s) * gridDim.x);
  }
  uint4 gamma[kVec];
  float acc[kVec][8];
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    const int32_t c = (j * threads + t) * 8;
    gamma[j] = c < a.hidden ? load16(a.gamma + c) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[j][i] = 0.0f;
  }
  __syncthreads();
  const float inv = 1.0f / float(a.hidden);
  int slot = 0, stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    // the block decides together whether the row has come
    ok = __syncthreads_and(mbar_wait(bar(stage), phase, a.wait, kSiteSmemFull)) != 0;
    if (!ok) break;
    const uint16_t* h = reinterpret_cast<const uint16_t*>(rows_shared) + int64_t(stage) * 3 * a.hidden;
    const uint16_t *dy = h + a.hidden, *dh = dy + a.hidden;
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * threads + t) * 8;
      if (c < a.hidden) grad_sums(load16(h + c), load16(dy + c), gamma[j], 1.0f, sum);
    }
    row_sum<false, 2>(sum, scratch, slot);
    slot ^= 1;
    float r = rsqrtf(fmaf(sum[0], inv, a.eps)), mean = sum[1] * inv * r;  // mean(dn n)
    if (!(sum[0] < kTooLarge)) {
      sum[0] = sum[1] = 0.0f;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const int32_t c = (j * threads + t) * 8;
        if (c < a.hidden) grad_sums(load16(h + c), load16(dy + c), gamma[j], kDown, sum);
      }
      row_sum<false, 2>(sum, scratch, slot);
      slot ^= 1;
      r = rsqrtf(sum[0] * inv);
      mean = sum[1] * inv * r;
      r *= kDown;
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * threads + t) * 8;
      if (c < a.hidden)
        grad_vector(load16(h + c), load16(dy + c), gamma[j], a.dh != nullptr ? load16(dh + c) : make_uint4(0u, 0u, 0u, 0u), r, mean,
                    acc[j], a.dx + row * a.dx_stride + c);
    }
    __syncthreads();  // the stage is read
    if (t == 0 && row + int64_t(kStages) * gridDim.x < a.rows) fetch(stage, row + int64_t(kStages) * gridDim.x);
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1u;
    }
  }
  if (!ok) {  // a wait gave up: copies in flight get their time to land before shared memory goes away
    const uint64_t start = ptx::globaltimer();
    while (ptx::globaltimer() - start < 200000ull) __nanosleep(1000);
    return;
  }
  if (a.partial != nullptr) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int32_t c = (j * threads + t) * 8;
      if (c < a.hidden) store_share(acc[j], a.partial + int64_t(blockIdx.x) * a.hidden + c);
    }
  }
}

// grad_gamma[c] = sum of the partial rows, 32 columns per block, 32 row lanes in a fixed order.
__global__ void __launch_bounds__(1024) rms_norm_gamma_kernel(const float* partial, int32_t groups, int32_t hidden,
                                                              uint16_t* grad_gamma) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int32_t c = int32_t(blockIdx.x) * 32 + lane;
  float sum = 0.0f;
  if (c < hidden)
    for (int32_t g = part; g < groups; g += 32) sum += partial[int64_t(g) * hidden + c];
  sums[part][lane] = sum;
  __syncthreads();
  if (part == 0 && c < hidden) {
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += sums[i][lane];
    grad_gamma[c] = uint16_t(pack2(sum, 0.0f));
  }
}

constexpr int32_t kMaxHidden = 16384;

// Threads of a row: a warp with up to four vectors each (no block barrier, four rows to a block), or a block of as
// few as hold it in kVectors each.
int row_threads(int32_t hidden) {
  const int threads = (hidden + 256 * kVectors - 1) / (256 * kVectors) * 32;
  return hidden <= 1024 ? 32 : threads < 128 ? 128 : threads;
}
// The backward's: a warp as far as its registers hold the row and its gradients without thinning the SM out (with the join
// of dgamma, 65536 x 256 takes 40 us and 65536 x 512 54 by warps, 110 and 114 by blocks), else a block of four
// warps or of as many as take the row in four vectors each.  Narrow rows leave most of such a block idle and its two stages
// small: 65536 x 544 takes 120 us, 65536 x 1024 127, 32768 x 2048 90, 16384 x 4096 92 (43, 82, 82 and 82 by their bytes).
int grad_threads(int32_t hidden) { return hidden <= 512 ? 32 : hidden <= 4096 ? 128 : (hidden + 1023) / 1024 * 32; }
// Row groups of the backward grid (rows of `partial`): whole blocks, as many as stay resident.  A block per row keeps two
// rows of three inputs in shared memory (6 bytes per element and row) and 512 threads fill an SM's registers.
int backward_groups(int64_t rows, int32_t hidden, int sm_count) {
  const int threads = grad_threads(hidden), block = threads < 128 ? 128 : threads, per_block = block / threads;
  int64_t per_sm = 512 / block;
  if (threads >= 128 && per_sm * 12 * hidden > 200 * 1024) per_sm = 200 * 1024 / (12 * hidden);
  const int64_t resident = int64_t(sm_count) * (per_sm > 0 ? per_sm : 1);
  const int64_t wanted = (rows + per_block - 1) / per_block;
  return int((wanted < resident ? wanted : resident) * per_block);
}

bool aligned_row(const void* p, int64_t stride, int32_t hidden) {
  return host::aligned16(p) && stride >= hidden && stride % 8 == 0;
}

template <bool kMx>
void launch_forward(const NormArgs& a, int sm_count, cudaStream_t stream) {
  const int threads = row_threads(a.hidden), block = threads < 128 ? 128 : threads, per_block = block / threads;
  const int64_t rows = kMx ? (a.rows + 127) / 128 * 128 : a.rows;
  const int64_t wanted = (rows + per_block - 1) / per_block, resident = int64_t(sm_count) * (2048 / block);
  const unsigned grid = unsigned(wanted < resident ? wanted : resident);
  const int vec = (a.hidden + threads * 8 - 1) / (threads * 8);
  if (threads > 32) rms_norm_kernel<false, kVectors, kMx><<<grid, block, 0, stream>>>(a);
  else if (vec == 1) rms_norm_kernel<true, 1, kMx><<<grid, block, 0, stream>>>(a);
  else if (vec == 2) rms_norm_kernel<true, 2, kMx><<<grid, block, 0, stream>>>(a);
  else rms_norm_kernel<true, 4, kMx><<<grid, block, 0, stream>>>(a);
}

cudaError_t rms_norm(const fuse_b200_rms_norm_params& p, cudaStream_t stream) {
  NormArgs a{};
  a.hidden = p.hidden;
  a.rows = p.rows;
  a.eps = p.epsilon;
  a.x_stride = launch::packed_or(p.input_stride, p.hidden);
  a.res_stride = launch::packed_or(p.residual_stride, p.hidden);
  a.h_stride = launch::packed_or(p.residual_output_stride, p.hidden);
  a.y_stride = launch::packed_or(p.output_stride, p.hidden);
  const bool mx = p.quantized.data != nullptr;
  if (p.rows < 0 || p.hidden <= 0 || p.hidden > kMaxHidden || p.hidden % (mx ? 32 : 8) != 0 ||
      !(p.epsilon >= kMinEpsilon) || std::isinf(p.epsilon) || (p.output == nullptr && !mx))
    return cudaErrorInvalidValue;
  if (p.rows == 0) return cudaSuccess;
  if (!aligned_row(p.input, a.x_stride, p.hidden) || !host::aligned16(p.gamma) ||
      (p.residual != nullptr && !aligned_row(p.residual, a.res_stride, p.hidden)) ||
      (p.residual_output != nullptr && !aligned_row(p.residual_output, a.h_stride, p.hidden)) ||
      (p.output != nullptr && !aligned_row(p.output, a.y_stride, p.hidden)))
    return cudaErrorInvalidValue;
  const size_t atoms = size_t((p.rows + 127) / 128) * size_t((p.hidden + 127) / 128);
  if (mx && (!host::aligned16(p.quantized.data) || !host::aligned16(p.quantized.scales) ||
             p.quantized.data_bytes < size_t(p.rows) * size_t(p.hidden) || p.quantized.scale_bytes < atoms * 512))
    return cudaErrorInvalidValue;
  DeviceInfo info;
  cudaError_t status = launch::check_device(&info);
  if (status != cudaSuccess) return status;
  a.x = p.input;
  a.res = p.residual;
  a.gamma = p.gamma;
  a.h = p.residual_output;
  a.y = p.output;
  a.data = const_cast<uint8_t*>(p.quantized.data);
  a.scales = const_cast<uint8_t*>(p.quantized.scales);
  if (mx) launch_forward<true>(a, info.sm_count, stream);
  else launch_forward<false>(a, info.sm_count, stream);
  status = cudaGetLastError();
  if (status == cudaSuccess) host::count_launch();
  return status;
}

cudaError_t backward_workspace(int64_t rows, int32_t hidden, size_t* bytes) {
  if (bytes == nullptr || rows < 0 || hidden <= 0 || hidden > kMaxHidden || hidden % 8 != 0) return cudaErrorInvalidValue;
  DeviceInfo info;
  const cudaError_t status = launch::check_device(&info);
  if (status != cudaSuccess) return status;
  *bytes = size_t(backward_groups(rows, hidden, info.sm_count)) * size_t(hidden) * sizeof(float);
  return cudaSuccess;
}

cudaError_t rms_norm_backward(const fuse_b200_rms_norm_backward_params& p, cudaStream_t stream) {
  NormGradArgs a{};
  a.hidden = p.hidden;
  a.rows = p.rows;
  a.eps = p.epsilon;
  a.dy_stride = launch::packed_or(p.grad_output_stride, p.hidden);
  a.h_stride = launch::packed_or(p.stream_input_stride, p.hidden);
  a.dh_stride = launch::packed_or(p.grad_stream_stride, p.hidden);
  a.dx_stride = launch::packed_or(p.grad_input_stride, p.hidden);
  if (p.rows < 0 || p.hidden <= 0 || p.hidden > kMaxHidden || p.hidden % 8 != 0 || !(p.epsilon >= kMinEpsilon) ||
      std::isinf(p.epsilon))
    return cudaErrorInvalidValue;
  if (p.rows > 0 && (!aligned_row(p.grad_output, a.dy_stride, p.hidden) || !host::aligned16(p.gamma) ||
                     !aligned_row(p.stream_input, a.h_stride, p.hidden) ||
                     !aligned_row(p.grad_input, a.dx_stride, p.hidden) ||
                     (p.grad_stream != nullptr && !aligned_row(p.grad_stream, a.dh_stride, p.hidden))))
    return cudaErrorInvalidValue;
  if (p.grad_gamma != nullptr && reinterpret_cast<uintptr_t>(p.grad_gamma) % 2 != 0) return cudaErrorInvalidValue;
  if (p.rows == 0 && p.grad_gamma == nullptr) return cudaSuccess;
  DeviceInfo info;
  cudaError_t status = launch::check_device(&info);
  if (status != cudaSuccess) return status;
  const int threads = grad_threads(p.hidden), block = threads < 128 ? 128 : threads;
  const int groups = backward_groups(p.rows, p.hidden, info.sm_count);
  const unsigned grid = unsigned(groups / (block / threads));
  if (p.grad_gamma != nullptr && groups > 0 &&
      (p.workspace == nullptr || reinterpret_cast<uintptr_t>(p.workspace) % 256 != 0 ||
       p.workspace_bytes < size_t(groups) * size_t(p.hidden) * sizeof(float)))
    return cudaErrorInvalidValue;
  a.dy = p.grad_output;
  a.h = p.stream_input;
  a.gamma = p.gamma;
  a.dh = p.grad_stream;
  a.dx = p.grad_input;
  a.partial = p.grad_gamma != nullptr ? static_cast<float*>(p.workspace) : nullptr;
  a.wait = host::make_wait(info, 0, 0);
  if (grid > 0) {
    const int vec = (p.hidden + threads * 8 - 1) / (threads * 8);
    constexpr uint32_t kElementBytes = 2 * 3 * 2;  // of shared memory: two stages of three BF16 rows
    if (threads > 32) {
      status = host::launch_kernel_sized(rms_norm_backward_kernel, int(grid), threads, kElementBytes * uint32_t(p.hidden),
                                         kElementBytes * uint32_t(kMaxHidden), false, stream, a);
    } else {
      if (vec == 1) rms_norm_backward_warp_kernel<1><<<grid, 128, 0, stream>>>(a);
      else rms_norm_backward_warp_kernel<2><<<grid, 128, 0, stream>>>(a);
      status = cudaGetLastError();
      if (status == cudaSuccess) host::count_launch();
    }
    if (status != cudaSuccess) return status;
  }
  if (p.grad_gamma != nullptr) {
    rms_norm_gamma_kernel<<<unsigned((p.hidden + 31) / 32), 1024, 0, stream>>>(a.partial, groups, p.hidden, p.grad_gamma);
    if ((status = cudaGetLastError()) != cudaSuccess) return status;
    host::count_launch();
  }
  return cudaSuccess;
}

}  // namespace
}  // namespace fuse_b200

extern "C" {

int fuse_b200_launch_rms_norm(const fuse_b200_rms_norm_params* params, fuse_stream stream) {
  if (params == nullptr) return int(cudaErrorInvalidValue);
  return int(fuse_b200::rms_norm(*params, stream));
}
int fuse_b200_rms_norm_backward_workspace_size(int64_t rows, int32_t hidden, size_t* bytes) {
  return int(fuse_b200::backward_workspace(rows, hidden, bytes));
}
int fuse_b200_launch_rms_norm_backward(const fuse_b200_rms_norm_backward_params* params, fuse_stream stream) {
  if (params == nullptr) return int(cudaErrorInvalidValue);
  return int(fuse_b200::rms_norm_backward(*params, stream));
}

}  // extern "C"
