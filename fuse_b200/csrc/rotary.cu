// Rotary positions on the heads of Q and K: pair i of a head at position p is turned by p f_i,
//
//   (a, b) -> m (a cos - b sin, a sin + b cos),
//
// and its adjoint, the same with the angle negated.
//
// The angle of a far position needs more than FP32: p f_i may be 10^5 turns, of which only the
// fraction matters.  Positions are whole numbers, so the fraction of p f_i / 2 pi is p times the
// 64-bit fraction of f_i / 2 pi modulo 2^64: one integer product.  What it is off by is p times the error of
// the fraction: 2^-63 turns from the quotient's 64 bits and the cut, and, against the formula, up to 2^-55 from f_i, which pow and
// the scalings give in FP64 (half a last place of f_i <= 1).  Up to 2^31 positions the latter is 2^-24 turns, 2^-21.3 of a radian, no
// more than the hardware's sine below is off.  The product's high word is the angle as a signed fraction of a half turn.
//
// Bound by HBM: 2 bytes read and 2 written per element.  A block takes a few rows at a time, computes
// their cosines and sines once into shared memory (they serve every head) and then walks the rows'
// heads in items of sixteen elements, two 16-byte loads and stores each.
#include "launch.cuh"

namespace fuse_b200 {
namespace {

using host::DeviceInfo;

constexpr int kMaxPairs = 128;
constexpr double kTwoPi = 6.28318530717958647692;

struct RotaryArgs {
  const uint16_t *q, *k;
  uint16_t *qo, *ko;
  int64_t q_stride, k_stride, qo_stride, ko_stride;
  const void* positions;
  int64_t start, rows, seq_len;
  int32_t q_heads, kv_heads, head_dim, rotary_dim, position_bytes;
  float magnitude;  // of the cosine
  float sine;       // of the sine: the magnitude, negative for the adjoint
  uint64_t turns[kMaxPairs];  // fraction of a turn per position, in 2^-64
};

// `within`: the row's place in its sequence, counted on from a row that lies in it (one division for
// all rows of a block; only rows behind the sequence's end divide again).
__device__ __forceinline__ float2 pair_rotation(const RotaryArgs& a, int64_t row, int64_t within, uint64_t per_position) {
  int64_t p;
  if (a.positions == nullptr) p = a.start + (within < a.seq_len ? within : within % a.seq_len);
  else if (a.position_bytes == 4) p = static_cast<const int32_t*>(a.positions)[row];
  else p = static_cast<const int64_t*>(a.positions)[row];
  const uint64_t turn = uint64_t(p) * per_position;
  // |angle| <= pi, where the hardware's sine and cosine are within 2^-21.1 (absolute): far below the
  // BF16 step of what they multiply (2^-9 of it)
  const float angle = float(int32_t(turn >> 32)) * 1.46291807926715968e-9f /* pi 2^-31 */;
  return make_float2(__cosf(angle) * a.magnitude, __sinf(angle) * a.sine);
}

__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// An item is 16 elements of one head: with the half layout eight of the first half and the eight they
// pair with, with the interleaved layout (and in the part that is only copied) sixteen neighbours.
// A thread keeps one item of the row and goes from row to row, kBatch rows' loads in flight at a time.
constexpr int kBlock = 256, kBatch = 2, kResident = 4;
template <bool kInterleaved>
__global__ void __launch_bounds__(kBlock, kResident) rotary_kernel(const __grid_constant__ RotaryArgs a, int32_t tokens) {
  // [tokens][4][rotated items]: cosine and sine of pairs 2j and 2j + 1 of an item, neighbouring items side by side
  extern __shared__ float4 turn[];
  // lanes that index the kernel's parameters apart from one another are served one by one (77 us against 70 for 128K rows of five heads of 128)
  __shared__ uint64_t per_position[kMaxPairs];
  if (threadIdx.x < kMaxPairs) per_position[threadIdx.x] = a.turns[threadIdx.x];
  __syncthreads();
  const int32_t pairs = a.rotary_dim >> 1, heads = a.q_heads + a.kv_heads;
  const int32_t rotated = a.rotary_dim >> 4;                  // items of a head that turn
  const int32_t items = a.head_dim >> 4, slots = heads * items;
  const int32_t rows_at_once = slots < kBlock ? kBlock / slots : 1;
  const int32_t first_row = slots < kBlock ? int32_t(threadIdx.x) / slots : 0;
  const int32_t first_slot = int32_t(threadIdx.x) - first_row * (slots < kBlock ? slots : 0);
  // a thread's pair, and the first and further rows whose angles it computes
  const int32_t turns_at_once = kBlock / pairs, first_turn = int32_t(threadIdx.x) / pairs, pair = int32_t(threadIdx.x) - first_turn * pairs;
  const int32_t turn_at = ((pair & 7) >> 1) * (2 * rotated) + (pair >> 3) * 2 + (pair & 1);
  const uint64_t mine = per_position[pair];
  const int64_t chunks = (a.rows + tokens - 1) / tokens;
  for (int64_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int64_t row0 = chunk * tokens;
    const int32_t n = int32_t(a.rows - row0 < tokens ? a.rows - row0 : tokens);
    const int64_t within0 = a.positions == nullptr ? row0 % a.seq_len : 0;
    for (int32_t token = first_turn; token < n; token += turns_at_once)
      if (first_turn < turns_at_once)
        reinterpret_cast<float2*>(turn)[token * pairs + turn_at] = pair_rotation(a, row0 + token, within0 + token, mine);
    __syncthreads();
    for (int32_t slot = first_row < rows_at_once ? first_slot : slots; slot < slots; slot += kBlock) {
      const int32_t head = slot / items, item = slot - head * items;
      const bool is_q = head < a.q_heads, turned = item < rotated;
      const int64_t in_stride = is_q ? a.q_stride : a.k_stride, out_stride = is_q ? a.qo_stride : a.ko_stride;
      const int64_t column = int64_t(is_q ? head : head - a.q_heads) * a.head_dim;
      const int32_t first = kInterleaved || !turned ? item * 16 : item * 8;
      const int32_t second = kInterleaved || !turned ? first + 8 : first + pairs;
      const uint16_t* in = (is_q ? a.q : a.k) + (row0 + first_row) * in_stride + column + first;
      uint16_t* out = (is_q ? a.qo : a.ko) + (row0 + first_row) * out_stride + column + first;
      const int64_t in_step = rows_at_once * in_stride, out_step = rows_at_once * out_stride;
      const int32_t apart = second - first;
      for (int32_t token0 = first_row; token0 < n; token0 += kBatch * rows_at_once) {
        uint4 us[kBatch], vs[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int32_t token = token0 + k * rows_at_once;
          if (token < n) {
            us[k] = *reinterpret_cast<const uint4*>(in);
            vs[k] = *reinterpret_cast<const uint4*>(in + apart);
          }
          in += in_step;
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int32_t token = token0 + k * rows_at_once;
          if (token >= n) break;
          uint4 &u = us[k], &v = vs[k];
          if (turned) {
            uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
            const float4* cs = turn + token * (pairs >> 1) + item;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 t = cs[j * rotated];  // cosine and sine of pairs 2j and 2j + 1 of this item
              if constexpr (kInterleaved) {
                uint32_t& w0 = j < 2 ? uw[2 * j] : vw[2 * j - 4];
                uint32_t& w1 = j < 2 ? uw[2 * j + 1] : vw[2 * j - 3];
                const float a0 = low(w0), b0 = high(w0), a1 = low(w1), b1 = high(w1);
                w0 = pack(a0 * t.x - b0 * t.y, a0 * t.y + b0 * t.x);
                w1 = pack(a1 * t.z - b1 * t.w, a1 * t.w + b1 * t.z);
              } else {
                const float a0 = low(uw[j]), a1 = high(uw[j]), b0 = low(vw[j]), b1 = high(vw[j]);
                uw[j] = pack(a0 * t.x - b0 * t.y, a1 * t.z - b1 * t.w);
                vw[j] = pack(a0 * t.y + b0 * t.x, a1 * t.w + b1 * t.z);
              }
            }
            u = make_uint4(uw[0], uw[1], uw[2], uw[3]);
            v = make_uint4(vw[0], vw[1], vw[2], vw[3]);
          }
          *reinterpret_cast<uint4*>(out) = u;
          *reinterpret_cast<uint4*>(out + apart) = v;
          out += out_step;
        }
      }
    }
    __syncthreads();
  }
}

// Any even rotary_dim, any stride: one thread per pair (or per two copied elements).
__global__ void __launch_bounds__(256) rotary_pairs_kernel(const __grid_constant__ RotaryArgs a, int32_t interleaved) {
  const int32_t pairs = a.rotary_dim >> 1, heads = a.q_heads + a.kv_heads;
  const int32_t rest = a.head_dim - a.rotary_dim, slots = pairs + rest;
  const int64_t total = a.rows * slots;
  for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += int64_t(gridDim.x) * blockDim.x) {
    const int64_t row = i / slots;
    const int32_t slot = int32_t(i - row * slots);
    const bool turned = slot < pairs;
    const float2 t = turned ? pair_rotation(a, row, row, a.turns[slot]) : make_float2(1.0f, 0.0f);
    const int32_t first = !turned ? a.rotary_dim + slot - pairs : interleaved ? 2 * slot : slot;
    const int32_t second = interleaved ? first + 1 : first + pairs;
    for (int32_t head = 0; head < heads; ++head) {
      const bool is_q = head < a.q_heads;
      const uint16_t* in = is_q ? a.q + row * a.q_stride + int64_t(head) * a.head_dim
                                : a.k + row * a.k_stride + int64_t(head - a.q_heads) * a.head_dim;
      uint16_t* out = is_q ? a.qo + row * a.qo_stride + int64_t(head) * a.head_dim
                           : a.ko + row * a.ko_stride + int64_t(head - a.q_heads) * a.head_dim;
      if (turned) {
        const float x = low(in[first]), y = low(in[second]);
        const uint32_t w = pack(x * t.x - y * t.y, x * t.y + y * t.x);
        out[first] = uint16_t(w);
        out[second] = uint16_t(w >> 16);
      } else {
        out[first] = in[first];
      }
    }
  }
}

cudaError_t frequencies(const fuse_b200_rotary_spec& s, double* f, double* magnitude) {
  const int32_t n = s.rotary_dim;
  if (n <= 0 || n % 2 != 0 || n > 2 * kMaxPairs || !(s.theta > 0.0) || !std::isfinite(s.theta) ||
      s.scaling < FUSE_B200_ROTARY_NONE || s.scaling > FUSE_B200_ROTARY_YARN || !std::isfinite(s.magnitude) ||
      s.magnitude < 0.0)
    return cudaErrorInvalidValue;
  double theta = s.theta, scale = 1.0;
  if (s.scaling != FUSE_B200_ROTARY_NONE && (!(s.factor > 0.0) || !std::isfinite(s.factor))) return cudaErrorInvalidValue;
  if (s.scaling >= FUSE_B200_ROTARY_WAVELENGTH && s.original_context <= 0) return cudaErrorInvalidValue;
  if (s.scaling == FUSE_B200_ROTARY_NTK) {
    if (n <= 2) return cudaErrorInvalidValue;
    theta *= std::pow(s.factor, double(n) / (n - 2));
  }
  if (s.scaling == FUSE_B200_ROTARY_WAVELENGTH && !(s.high_freq_factor > s.low_freq_factor)) return cudaErrorInvalidValue;
  double ramp_low = 0.0, ramp_high = 0.0;
  if (s.scaling == FUSE_B200_ROTARY_YARN) {
    if (!(s.beta_fast > s.beta_slow) || !(s.beta_slow > 0.0) || !(theta > 1.0)) return cudaErrorInvalidValue;
    // the (real) index of the pair that turns b times within the original context
    auto pair = [&](double b) { return n * std::log(double(s.original_context) / (b * kTwoPi)) / (2.0 * std::log(theta)); };
    ramp_low = std::fmax(std::floor(pair(s.beta_fast)), 0.0);
    ramp_high = std::fmin(std::ceil(pair(s.beta_slow)), double(n - 1));
    scale = 0.1 * std::log(s.factor) + 1.0;
  }
  for (int32_t i = 0; i < n / 2; ++i) {
    double v = std::pow(theta, -2.0 * i / n);
    if (s.scaling == FUSE_B200_ROTARY_LINEAR) {
      v /= s.factor;
    } else if (s.scaling == FUSE_B200_ROTARY_WAVELENGTH) {
      const double turns = double(s.original_context) * v / kTwoPi;
      const double keep = std::fmin(std::fmax((turns - s.low_freq_factor) / (s.high_freq_factor - s.low_freq_factor), 0.0), 1.0);
      v = (1.0 - keep) * v / s.factor + keep * v;
    } else if (s.scaling == FUSE_B200_ROTARY_YARN) {
      const double ramp = std::fmin(std::fmax((i - ramp_low) / std::fmax(ramp_high - ramp_low, 1e-3), 0.0), 1.0);
      v = v * (1.0 - ramp) + v / s.factor * ramp;
    }
    f[i] = v;
  }
  *magnitude = s.magnitude > 0.0 ? s.magnitude : scale;
  return cudaSuccess;
}

bool row_fits(const void* p, int64_t stride, int64_t width) {
  return p != nullptr && reinterpret_cast<uintptr_t>(p) % 2 == 0 && stride >= width;
}

cudaError_t rotary(const fuse_b200_rotary_params& p, cudaStream_t stream) {
  const int32_t d = p.head_dim, n = p.spec.rotary_dim;
  RotaryArgs a;
  double f[kMaxPairs], magnitude = 1.0;
  cudaError_t status = frequencies(p.spec, f, &magnitude);
  if (status != cudaSuccess) return status;
  if (d <= 0 || n > d || p.q_heads < 0 || p.kv_heads < 0 || p.q_heads + int64_t(p.kv_heads) <= 0 ||
      p.q_heads + int64_t(p.kv_heads) > 65536 || d > 4096 || p.rows < 0 || p.rows > (int64_t(1) << 40) ||
      (p.positions == nullptr ? p.seq_len <= 0 : p.position_bytes != 4 && p.position_bytes != 8))
    return cudaErrorInvalidValue;
  a.q_stride = launch::packed_or(p.q_stride, int64_t(p.q_heads) * d);
  a.k_stride = launch::packed_or(p.k_stride, int64_t(p.kv_heads) * d);
  a.qo_stride = launch::packed_or(p.q_output_stride, int64_t(p.q_heads) * d);
  a.ko_stride = launch::packed_or(p.k_output_stride, int64_t(p.kv_heads) * d);
  if (p.rows == 0) return cudaSuccess;
  if ((p.q_heads > 0 && (!row_fits(p.q, a.q_stride, int64_t(p.q_heads) * d) ||
                         !row_fits(p.q_output, a.qo_stride, int64_t(p.q_heads) * d) ||
                         (p.q == p.q_output && a.q_stride != a.qo_stride))) ||
      (p.kv_heads > 0 && (!row_fits(p.k, a.k_stride, int64_t(p.kv_heads) * d) ||
                          !row_fits(p.k_output, a.ko_stride, int64_t(p.kv_heads) * d) ||
                          (p.k == p.k_output && a.k_stride != a.ko_stride))) ||
      (p.positions != nullptr && reinterpret_cast<uintptr_t>(p.positions) % p.position_bytes != 0))
    return cudaErrorInvalidValue;
  DeviceInfo info;
  if ((status = launch::check_device(&info)) != cudaSuccess) return status;
  a.q = p.q;
  a.k = p.k;
  a.qo = p.q_output;
  a.ko = p.k_output;
  a.positions = p.positions;
  a.start = p.position_start;
  a.rows = p.rows;
  a.seq_len = p.positions == nullptr ? p.seq_len : 1;
  a.q_heads = p.q_heads;
  a.kv_heads = p.kv_heads;
  a.head_dim = d;
  a.rotary_dim = n;
  a.position_bytes = p.position_bytes;
  a.magnitude = float(magnitude);
  a.sine = p.adjoint ? -float(magnitude) : float(magnitude);
  for (int32_t i = 0; i < kMaxPairs; ++i) {
    // whole turns drop out; the fraction scaled by 2^64 stays below it
    const long double turns = i < n / 2 ? (long double)f[i] / 6.283185307179586476925286766559L : 0.0L;
    a.turns[i] = uint64_t((turns - floorl(turns)) * 18446744073709551616.0L);
  }
  bool vectors = d % 16 == 0 && n % 16 == 0;
  if (p.q_heads > 0)
    vectors = vectors && host::aligned16(p.q) && host::aligned16(p.q_output) && a.q_stride % 8 == 0 && a.qo_stride % 8 == 0;
  if (p.kv_heads > 0)
    vectors = vectors && host::aligned16(p.k) && host::aligned16(p.k_output) && a.k_stride % 8 == 0 && a.ko_stride % 8 == 0;
  if (vectors) {
    // rows per block: one batch of every thread, while the angles stay within 24 KiB
    const int64_t slots = int64_t(p.q_heads + p.kv_heads) * (d / 16);
    int64_t tokens = slots < kBlock ? kBatch * (kBlock / slots) : kBatch;
    constexpr int64_t kTurns = 24 * 1024 / sizeof(float2);
    if (tokens * (n / 2) > kTurns) tokens = kTurns / (n / 2);
    const int64_t chunks = (p.rows + tokens - 1) / tokens, resident = int64_t(info.sm_count) * 8;
    const unsigned grid = unsigned(chunks < resident ? chunks : resident);
    const size_t shared = size_t(tokens) * (n / 2) * sizeof(float2);
    if (p.spec.interleaved) rotary_kernel<true><<<grid, kBlock, shared, stream>>>(a, int32_t(tokens));
    else rotary_kernel<false><<<grid, kBlock, shared, stream>>>(a, int32_t(tokens));
  } else {
    const int64_t threads = p.rows * (n / 2 + (d - n));
    const int64_t blocks = (threads + 255) / 256, resident = int64_t(info.sm_count) * 8;
    rotary_pairs_kernel<<<unsigned(blocks < resident ? blocks : resident), 256, 0, stream>>>(a, p.spec.interleaved ? 1 : 0);
  }
  status = cudaGetLastError();
  if (status == cudaSuccess) host::count_launch();
  return status;
}

}  // namespace
}  // namespace fuse_b200

extern "C" {

int fuse_b200_rotary_frequencies(const fuse_b200_rotary_spec* spec, double* out, double* magnitude) {
  if (spec == nullptr || out == nullptr || magnitude == nullptr) return int(cudaErrorInvalidValue);
  return int(fuse_b200::frequencies(*spec, out, magnitude));
}
int fuse_b200_launch_rotary(const fuse_b200_rotary_params* params, fuse_stream stream) {
  if (params == nullptr) return int(cudaErrorInvalidValue);
  return int(fuse_b200::rotary(*params, stream));
}

}  // extern "C"
