// Attention between the projections: argument checks, the split over keys and the launches (kernels: attention.cuh).
#include "attention_backward.cuh"
#include "launch.cuh"

namespace fuse_b200 {
namespace {

using host::DeviceInfo;

bool aligned_rows(const void* p, int64_t stride, int64_t width) {
  return host::aligned16(p) && stride >= width && stride % 8 == 0;
}

cudaError_t check_shape(const fuse_b200_attention_params& p) {
  if (p.head_dim != 64 && p.head_dim != 128) return cudaErrorNotSupported;
  if (p.batch < 0 || p.q_len < 0 || p.kv_len < 0 || p.q_heads <= 0 || p.kv_heads <= 0 || p.q_heads % p.kv_heads != 0 ||
      p.q_heads > 65536 || p.q_rows < 0 || p.kv_rows < 0 || p.q_rows > INT32_MAX - 1024 || p.kv_rows > INT32_MAX - 1024 ||
      p.window < 0 || p.sinks < 0 || (!p.causal && p.window > 0) || !(p.scale > 0.0f) || std::isinf(p.scale) ||
      // positions and products of sizes stay within 31 bits
      p.q_len > (1 << 29) || p.kv_len > (1 << 29) || p.batch > (1 << 24))
    return cudaErrorInvalidValue;
  // without starts sequence b begins at row b * len
  if ((p.q_starts == nullptr && int64_t(p.batch) * p.q_len > p.q_rows) ||
      (p.kv_starts == nullptr && int64_t(p.batch) * p.kv_len > p.kv_rows))
    return cudaErrorInvalidValue;
  return cudaSuccess;
}

// Query heads that share a tile: the largest power of two that divides the group, at most 128.
int32_t packed_heads(const fuse_b200_attention_params& p) {
  const int32_t group = p.q_heads / p.kv_heads;
  int32_t pack = 1;
  while (pack < attn::kTile && group % (2 * pack) == 0) pack *= 2;
  return pack;
}
int64_t query_blocks(const fuse_b200_attention_params& p) {
  const int32_t pack = packed_heads(p), tokens = 2 * attn::kTile / pack;
  return int64_t((p.q_len + tokens - 1) / tokens) * (p.q_heads / pack) * p.batch;
}

// Splits over keys: when the query blocks do not fill the SMs, the number of splits whose waves of blocks
// take the least time, in units of one key tile per block.  kFixed is what a block costs besides its tiles
// (set-up, first loads, its partial result); a further split has to win by the joining kernel's cost.  From one block per SM on
// nothing is weighed and nothing split; what that costs is the last wave: 144 blocks of 16384 keys (18 sequences of one token, 32 / 8
// heads of 128) take 218 us, 160 of them 428.
int32_t plan_splits(const fuse_b200_attention_params& p, int sm_count) {
  const int64_t blocks = query_blocks(p);
  int64_t keys = p.kv_len;
  const int64_t seen = int64_t(p.window) + p.q_len;
  const bool limited = p.window > 0 && p.window < p.kv_len;  // as the kernels take it: a longer window is none
  if (limited && seen < keys) keys = seen + (p.sinks < keys - seen ? p.sinks : keys - seen);
  const int64_t tiles = (keys + attn::kTile - 1) / attn::kTile + (limited ? 1 : 0);
  if (blocks == 0 || blocks >= sm_count || tiles < 4) return 1;
  constexpr double kFixed = 5.0, kJoin = 2.0;
  double best = double(tiles) + kFixed;
  int32_t splits = 1;
  for (int64_t s = 2; s <= tiles && s <= 256; ++s) {
    const int64_t waves = (blocks * s + sm_count - 1) / sm_count;
    const double cost = double(waves) * (double((tiles + s - 1) / s) + kFixed) + kJoin;
    if (cost < best - 1e-9) {
      best = cost;
      splits = int32_t(s);
    }
  }
  return splits;
}
// The whole of the queries is one tile per head pack and batch item: both tiles of a block work on it.
bool pair_tiles(const fuse_b200_attention_params& p, int32_t splits) {
  return splits > 1 && p.q_len <= attn::kTile / packed_heads(p);
}
size_t cells(const fuse_b200_attention_params& p) { return size_t(p.batch) * size_t(p.q_len) * size_t(p.q_heads); }
size_t split_bytes(const fuse_b200_attention_params& p, int32_t splits) {
  const size_t parts = size_t(splits) * (pair_tiles(p, splits) ? 2 : 1);
  return splits > 1 ? parts * cells(p) * size_t(p.head_dim + 1) * sizeof(float) : 0;
}

cudaError_t workspace_size(const fuse_b200_attention_params& p, size_t* bytes) {
  cudaError_t status = check_shape(p);
  if (status != cudaSuccess) return status;
  DeviceInfo info;
  if ((status = launch::check_device(&info)) != cudaSuccess) return status;
  *bytes = split_bytes(p, plan_splits(p, info.sm_count));
  return cudaSuccess;
}

attn::Args fill_args(const fuse_b200_attention_params& p) {
  attn::Args a{};
  a.q_starts = p.q_starts;
  a.q_lengths = p.q_lengths;
  a.kv_starts = p.kv_starts;
  a.kv_lengths = p.kv_lengths;
  a.q_rows = p.q_rows;
  a.kv_rows = p.kv_rows;
  a.batch = p.batch;
  a.q_len = p.q_len;
  a.kv_len = p.kv_len;
  a.q_heads = p.q_heads;
  a.kv_heads = p.kv_heads;
  a.pack = packed_heads(p);
  while ((1 << a.pack_shift) < a.pack) ++a.pack_shift;
  a.causal = p.causal ? 1 : 0;
  // a window as long as the keys limits nothing; both then stay within 29 bits
  a.window = p.window < p.kv_len ? p.window : 0;
  a.sinks = p.sinks < p.kv_len ? p.sinks : p.kv_len;
  a.scale = p.scale;
  a.scale_log2 = p.scale * attn::kLog2e;
  a.out = p.output;
  a.rest = p.output_rest;
  a.lse = p.lse;
  a.splits = a.parts = 1;
  return a;
}

template <int kDim>
cudaError_t launch_forward(const fuse_b200_attention_params& p, const attn::Args& a, int64_t q_stride, int64_t k_stride,
                           int64_t v_stride, cudaStream_t stream) {
  CUtensorMap q, k, v;
  cudaError_t status;
  // a tensor without key rows (all its queries see nothing) still needs a valid map: it is never loaded from
  const uint64_t kv_rows = p.kv_rows > 0 ? uint64_t(p.kv_rows) : 1;
  const void* kp = p.kv_rows > 0 ? p.k : p.q;
  const void* vp = p.kv_rows > 0 ? p.v : p.q;
  if ((status = host::encode_tensor_map_heads(&q, p.q, uint64_t(p.q_rows), uint64_t(p.q_heads), kDim, uint64_t(q_stride) * 2,
                                              uint32_t(attn::kTile / a.pack), uint32_t(a.pack))) != cudaSuccess ||
      (status = host::encode_tensor_map_heads(&k, kp, kv_rows, uint64_t(p.kv_heads), kDim, uint64_t(k_stride) * 2,
                                              attn::kTile, 1)) != cudaSuccess ||
      (status = host::encode_tensor_map_heads(&v, vp, kv_rows, uint64_t(p.kv_heads), kDim, uint64_t(v_stride) * 2,
                                              attn::kTile, 1)) != cudaSuccess)
    return status;
  const int64_t blocks = query_blocks(p) * a.splits;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  status = host::launch_kernel(attn::attention_forward_kernel<kDim>, int(blocks), attn::kForwardThreads,
                               attn::ForwardLayout<kDim>::kDynamicBytes, false, stream, q, k, v, a);
  if (status != cudaSuccess || a.splits == 1) return status;
  return host::launch_kernel(attn::attention_join_kernel<kDim>, int((cells(p) + 3) / 4), 128, 0, false, stream, a);
}

cudaError_t attention(const fuse_b200_attention_params& p, const fuse_b200_options* options, cudaStream_t stream) {
  cudaError_t status = check_shape(p);
  if (status != cudaSuccess) return status;
  const int64_t q_width = int64_t(p.q_heads) * p.head_dim, kv_width = int64_t(p.kv_heads) * p.head_dim;
  const int64_t q_stride = launch::packed_or(p.q_stride, q_width), out_stride = launch::packed_or(p.output_stride, q_width);
  const int64_t k_stride = launch::packed_or(p.k_stride, kv_width), v_stride = launch::packed_or(p.v_stride, kv_width);
  if (p.batch == 0 || p.q_len == 0 || p.q_rows == 0) return cudaSuccess;
  if (!aligned_rows(p.q, q_stride, q_width) || !aligned_rows(p.output, out_stride, q_width) ||
      (p.kv_rows > 0 && (!aligned_rows(p.k, k_stride, kv_width) || !aligned_rows(p.v, v_stride, kv_width))) ||
      (p.output_rest != nullptr && !host::aligned16(p.output_rest)) || (p.lse != nullptr && !host::aligned4(p.lse)))
    return cudaErrorInvalidValue;
  DeviceInfo info;
  if ((status = launch::check_device(&info)) != cudaSuccess) return status;
  attn::Args a = fill_args(p);
  a.out_stride = out_stride;
  a.splits = plan_splits(p, info.sm_count);
  a.paired = pair_tiles(p, a.splits) ? 1 : 0;
  a.parts = a.paired ? 2 * a.splits : a.splits;
  if (a.splits > 1) {
    if (p.workspace == nullptr || reinterpret_cast<uintptr_t>(p.workspace) % 256 != 0 ||
        p.workspace_bytes < split_bytes(p, a.splits))
      return cudaErrorInvalidValue;
    a.partial = static_cast<float*>(p.workspace);
    a.partial_lse = a.partial + size_t(a.parts) * cells(p) * p.head_dim;
  }
  a.wait = host::make_wait(info, 0, options ? options->wait_budget_ns : 0);
  return p.head_dim == 128 ? launch_forward<128>(p, a, q_stride, k_stride, v_stride, stream)
                           : launch_forward<64>(p, a, q_stride, k_stride, v_stride, stream);
}

size_t delta_bytes(const fuse_b200_attention_params& p) {
  return (size_t(p.q_heads) * size_t(p.q_rows) * sizeof(float) + 255) & ~size_t{255};
}

// Query tiles that one block of the key gradients takes at most.  Key tiles see very unequal numbers of them (the first
// key of a causal sequence all, the last one; a sink all, any other key a window's), and with few KV heads there
// are fewer key tiles than SMs.  About two blocks per SM of equal size (measured: 450 us for a backward of 8192 x 8 / 2 heads, 478 with three, 502 with six), as every
// further block costs its FP32 partial sums (128 KiB written and read with heads of 128); shorter than eight
// tiles, a block's set-up shows.
struct ChunkPlan {
  int32_t chunk, key_tiles, long_tiles, long_chunks, short_chunks;
  int64_t sequence_chunks, partial_chunks;
  size_t partial_bytes;
};
ChunkPlan plan_chunks(const fuse_b200_attention_params& p, int sm_count) {
  const int32_t pack = packed_heads(p), tokens = attn::kTile / pack, packs = p.q_heads / p.kv_heads / pack;
  ChunkPlan plan{};
  plan.key_tiles = (p.kv_len + attn::kTile - 1) / attn::kTile;
  plan.long_tiles = plan.key_tiles;
  const int64_t token_tiles = (int64_t(p.q_len) + tokens - 1) / tokens, longest = token_tiles * packs;  // every query tile
  int64_t usual = longest;  // of a key tile without sinks, at most
  double total = double(longest) * plan.key_tiles;
  if (p.causal && p.window > 0 && p.window < p.kv_len) {
    // its queries' positions span 127 + window at most
    const int64_t near = (int64_t(p.window) + attn::kTile - 1 + tokens - 1) / tokens + 1;
    if (near < token_tiles) usual = near * packs;
    const int64_t sinks = (int64_t(p.sinks) + attn::kTile - 1) / attn::kTile;
    plan.long_tiles = int32_t(sinks < plan.key_tiles ? sinks : plan.key_tiles);
    total = double(longest) * plan.long_tiles + double(usual) * (plan.key_tiles - plan.long_tiles);
  } else if (p.causal && p.kv_len < 2 * int64_t(p.q_len)) {
    total *= 0.5;  // (of the keys that are queries' own; those before are seen by all)
  }
  total *= double(p.kv_heads) * p.batch;
  int64_t chunk = int64_t(std::ceil(total / (2.0 * sm_count)));
  if (chunk < 8) chunk = 8;
  if (chunk > longest) chunk = longest > 0 ? longest : 1;
  plan.chunk = int32_t(chunk);
  plan.long_chunks = int32_t(longest > chunk ? (longest + chunk - 1) / chunk : 1);
  plan.short_chunks = int32_t(usual > chunk ? (usual + chunk - 1) / chunk : 1);
  const int64_t of_long = int64_t(plan.long_tiles) * plan.long_chunks;
  plan.sequence_chunks = of_long + int64_t(plan.key_tiles - plan.long_tiles) * plan.short_chunks;
  plan.partial_chunks = plan.short_chunks > 1 ? plan.sequence_chunks : plan.long_chunks > 1 ? of_long : 0;
  plan.partial_bytes = size_t(plan.partial_chunks) * p.kv_heads * p.batch * 2 * attn::kTile * p.head_dim * sizeof(float);
  return plan;
}

cudaError_t backward_workspace_size(const fuse_b200_attention_backward_params& p, size_t* bytes) {
  cudaError_t status = check_shape(p.forward);
  if (status != cudaSuccess) return status;
  DeviceInfo info;
  if ((status = launch::check_device(&info)) != cudaSuccess) return status;
  *bytes = delta_bytes(p.forward) + plan_chunks(p.forward, info.sm_count).partial_bytes;
  return cudaSuccess;
}

template <int kDim>
cudaError_t launch_backward(const fuse_b200_attention_params& p, const attn::BackwardArgs& b, int64_t q_stride,
                            int64_t k_stride, int64_t v_stride, int64_t sequence_chunks, cudaStream_t stream) {
  CUtensorMap q, d_o, k, v;
  cudaError_t status;
  const attn::Args& a = b.f;
  const uint64_t kv_rows = p.kv_rows > 0 ? uint64_t(p.kv_rows) : 1;
  const void* kp = p.kv_rows > 0 ? p.k : p.q;
  const void* vp = p.kv_rows > 0 ? p.v : p.q;
  const uint32_t tokens = uint32_t(attn::kTile / a.pack), pack = uint32_t(a.pack);
  if ((status = host::encode_tensor_map_heads(&q, p.q, uint64_t(p.q_rows), uint64_t(p.q_heads), kDim, uint64_t(q_stride) * 2,
                                              tokens, pack)) != cudaSuccess ||
      (status = host::encode_tensor_map_heads(&d_o, b.d_o, uint64_t(p.q_rows), uint64_t(p.q_heads), kDim,
                                              uint64_t(b.do_stride) * 2, tokens, pack)) != cudaSuccess ||
      (status = host::encode_tensor_map_heads(&k, kp, kv_rows, uint64_t(p.kv_heads), kDim, uint64_t(k_stride) * 2,
                                              attn::kTile, 1)) != cudaSuccess ||
      (status = host::encode_tensor_map_heads(&v, vp, kv_rows, uint64_t(p.kv_heads), kDim, uint64_t(v_stride) * 2,
                                              attn::kTile, 1)) != cudaSuccess)
    return status;
  const int64_t query_tiles = (int64_t(p.q_len) + tokens - 1) / tokens * (p.q_heads / a.pack) * p.batch;
  const int64_t key_tiles = int64_t(b.key_tiles) * p.kv_heads * p.batch;
  const int64_t key_blocks = sequence_chunks * p.kv_heads * p.batch;
  if (query_tiles > INT32_MAX || key_blocks > INT32_MAX) return cudaErrorInvalidValue;
  if (query_tiles > 0 &&
      (status = host::launch_kernel(attn::attention_query_grad_kernel<kDim>, int(query_tiles), attn::kBackwardThreads,
                                    attn::QueryGradLayout<kDim>::kDynamicBytes, false, stream, q, d_o, k, v, b)) != cudaSuccess)
    return status;
  if (key_tiles == 0) return cudaSuccess;
  status = host::launch_kernel(attn::attention_key_grad_kernel<kDim>, int(key_blocks), attn::kBackwardThreads,
                               attn::KeyGradLayout<kDim>::kDynamicBytes, false, stream, q, d_o, k, v, b);
  if (status != cudaSuccess || b.partial_chunks == 0) return status;
  // eight blocks a key tile: against two, a forward and backward of 8192 x 8 / 2 heads takes 546 us instead of 555, of 16384 x 4 / 4
  // with a window of 512 and sinks 209 instead of 227; with 1024 key tiles, of which the sinks' alone has chunks, 1404 and 1390
  attn::attention_key_grad_join_kernel<kDim><<<dim3(unsigned(key_tiles), 8), 256, 0, stream>>>(b);
  status = cudaGetLastError();
  if (status == cudaSuccess) host::count_launch();
  return status;
}

cudaError_t attention_backward(const fuse_b200_attention_backward_params& g, const fuse_b200_options* options,
                               cudaStream_t stream) {
  const fuse_b200_attention_params& p = g.forward;
  cudaError_t status = check_shape(p);
  if (status != cudaSuccess) return status;
  const int64_t q_width = int64_t(p.q_heads) * p.head_dim, kv_width = int64_t(p.kv_heads) * p.head_dim;
  const int64_t q_stride = launch::packed_or(p.q_stride, q_width);
  const int64_t k_stride = launch::packed_or(p.k_stride, kv_width), v_stride = launch::packed_or(p.v_stride, kv_width);
  attn::BackwardArgs b{};
  b.f = fill_args(p);
  b.o_stride = launch::packed_or(p.output_stride, q_width);
  b.do_stride = launch::packed_or(g.grad_output_stride, q_width);
  b.dq_stride = launch::packed_or(g.grad_q_stride, q_width);
  b.dk_stride = launch::packed_or(g.grad_k_stride, kv_width);
  b.dv_stride = launch::packed_or(g.grad_v_stride, kv_width);
  if (p.batch == 0 || (p.q_rows == 0 && p.kv_rows == 0)) return cudaSuccess;
  if (p.q_rows == 0) return cudaErrorInvalidValue;  // key gradients of no query: the caller's zeros
  if (!aligned_rows(p.q, q_stride, q_width) || !aligned_rows(p.output, b.o_stride, q_width) ||
      !aligned_rows(g.grad_output, b.do_stride, q_width) || !aligned_rows(g.grad_q, b.dq_stride, q_width) ||
      !host::aligned4(p.lse) || (p.output_rest != nullptr && !host::aligned16(p.output_rest)) ||
      (p.kv_rows > 0 && (!aligned_rows(p.k, k_stride, kv_width) || !aligned_rows(p.v, v_stride, kv_width) ||
                         !aligned_rows(g.grad_k, b.dk_stride, kv_width) || !aligned_rows(g.grad_v, b.dv_stride, kv_width))) ||
      g.workspace == nullptr || reinterpret_cast<uintptr_t>(g.workspace) % 256 != 0 || g.workspace_bytes < delta_bytes(p))
    return cudaErrorInvalidValue;
  DeviceInfo info;
  if ((status = launch::check_device(&info)) != cudaSuccess) return status;
  const ChunkPlan plan = plan_chunks(p, info.sm_count);
  if (g.workspace_bytes < delta_bytes(p) + plan.partial_bytes) return cudaErrorInvalidValue;
  b.chunk = plan.chunk;
  b.key_tiles = plan.key_tiles;
  b.long_tiles = plan.long_tiles;
  b.long_chunks = plan.long_chunks;
  b.short_chunks = plan.short_chunks;
  if (plan.sequence_chunks > INT32_MAX) return cudaErrorInvalidValue;
  b.partial_chunks = int32_t(plan.partial_chunks);
  b.partial = reinterpret_cast<float*>(static_cast<uint8_t*>(g.workspace) + delta_bytes(p));
  b.o = p.output;
  b.d_o = g.grad_output;
  b.lse = p.lse;
  b.delta = static_cast<float*>(g.workspace);
  b.dq = g.grad_q;
  b.dk = g.grad_k;
  b.dv = g.grad_v;
  b.f.wait = host::make_wait(info, 0, options ? options->wait_budget_ns : 0);
  return p.head_dim == 128 ? launch_backward<128>(p, b, q_stride, k_stride, v_stride, plan.sequence_chunks, stream)
                           : launch_backward<64>(p, b, q_stride, k_stride, v_stride, plan.sequence_chunks, stream);
}

}  // namespace
}  // namespace fuse_b200

extern "C" {

int fuse_b200_attention_workspace_size(const fuse_b200_attention_params* params, size_t* bytes) {
  if (params == nullptr || bytes == nullptr) return int(cudaErrorInvalidValue);
  return int(fuse_b200::workspace_size(*params, bytes));
}
int fuse_b200_launch_attention(const fuse_b200_attention_params* params, const fuse_b200_options* options,
                               fuse_stream stream) {
  if (params == nullptr) return int(cudaErrorInvalidValue);
  return int(fuse_b200::attention(*params, options, stream));
}
int fuse_b200_attention_backward_workspace_size(const fuse_b200_attention_backward_params* params, size_t* bytes) {
  if (params == nullptr || bytes == nullptr) return int(cudaErrorInvalidValue);
  return int(fuse_b200::backward_workspace_size(*params, bytes));
}
int fuse_b200_launch_attention_backward(const fuse_b200_attention_backward_params* params, const fuse_b200_options* options,
                                        fuse_stream stream) {
  if (params == nullptr) return int(cudaErrorInvalidValue);
  return int(fuse_b200::attention_backward(*params, options, stream));
}

}  // extern "C"
