// The paged decode that also accounts for where its attention goes (kernels of the attention: paged_decode.h):
//   weights[b, kv, t] += sum over the query heads h of KV head kv of softmax(scale * q[b, h] K^T)[t],  t < seqlen[b].
//
// A weight needs its head's maximum and sum over the whole row, which are known when the last split ends. Reading K
// again for it would double the bytes; the split kernel's scores are written instead, 4 bytes per
// (token, query head) beside the 4 D (16-bit types) of its K and V, and the launch that merges the splits
// reads them back: some of its workgroups fold the splits of a (row, head), as the plain
// form's second launch does, the others turn the scores of a (row, KV head, stretch of tokens)
// into weights. Each weight is read, added to and written once, by one lane, in a fixed order of heads. Bound by the reads of
// K and V: 32 rows of 128 to 2048 tokens, H 16 / H_kv 8 / D 128 bf16, 145 MB a layer: 21 us + 4.8; a row of 300 5.6 + 3.7.
// A batch of short rows takes the one-launch kernel, whose scores never leave LDS.
#include "paged_decode.h"

namespace miattn {
namespace {

constexpr int kWeighThreads = 256;
constexpr int kStretch = 4 * kWeighThreads;  // tokens a workgroup weighs per round

template <typename T, int D, int GB>
__global__ __launch_bounds__(kWeighThreads) void paged_decode_weigh_kernel(
    const int32_t* __restrict__ seqlen, const int32_t* __restrict__ ws_rows, const float* __restrict__ ws_ml,
    const float* __restrict__ ws_acc, T* __restrict__ out, DecodeArgs a, Weighed ext, int n_stretch) {
  const int b = blockIdx.y;
  const int x = int(blockIdx.x) - a.H_kv * n_stretch;
  const int tid = threadIdx.x;
  if (x >= 0) {  // the merge of head x; whole waves
    if (tid < (D > 64 ? D : 64)) merge_row<T, D>(seqlen, ws_rows, ws_ml, ws_acc, out, a, x, b);
    return;
  }
  extern __shared__ float sm[];  // [G] maximum and 1 / sum of each query head of the group
  const int kvh = int(blockIdx.x) / n_stretch, stretch = int(blockIdx.x) - kvh * n_stretch;
  const int capacity = a.max_blocks << a.bs_log2;
  const int len = clamp_len(seqlen[b], capacity);
  if (stretch * kStretch >= len) return;
  const int first = ws_rows[2 * b], n_split = ws_rows[2 * b + 1];
  const int lane = tid & 63, wave = tid >> 6;
  for (int g = wave; g < a.G; g += kWeighThreads / 64) {
    const float2* ml = reinterpret_cast<const float2*>(ws_ml) + int64_t(kvh * a.G + g) * a.slots + first;
    float M = -INFINITY, L = 0.0f;
    for (int j = lane; j < n_split; j += 64) {
      const float2 p = ml[j];
      const float m = fmaxf(M, p.x);
      const float u = m == -INFINITY ? 0.0f : m;
      L = fmaf(L, fast_exp2(M - u), p.y * fast_exp2(p.x - u));
      M = m;
    }
    const float m = group_allreduce<64, MaxOp>(M);
    const float u = m == -INFINITY ? 0.0f : m;
    const float l = group_allreduce<64, SumOp>(L * fast_exp2(M - u));
    if (lane == 0) {
      sm[2 * g] = u;
      sm[2 * g + 1] = 1.0f / (l < 1.0f ? 1.0f : l);  // the sum holds the maximum's own 1; NaN stays
    }
  }
  __syncthreads();
  const float* scores = ext.scores + (int64_t(b) * a.H_kv + kvh) * capacity * a.G;
  float* weights = ext.weights + b * ext.ws0 + kvh * ext.ws1;
  typedef float vec_t __attribute__((ext_vector_type(GB)));
  for (int t0 = stretch * kStretch; t0 < len; t0 += n_stretch * kStretch) {
#pragma unroll
    for (int i = 0; i < kStretch / kWeighThreads; ++i) {
      const int t = t0 + i * kWeighThreads + tid;
      if (t >= len) break;
      float w = weights[t];
      for (int g0 = 0; g0 < a.G; g0 += GB) {
        const vec_t s = *reinterpret_cast<const vec_t*>(scores + int64_t(t) * a.G + g0);
#pragma unroll
        for (int g = 0; g < GB; ++g) {
          w = fmaf(fast_exp2(s[g] - sm[2 * (g0 + g)]), sm[2 * (g0 + g) + 1], w);
        }
      }
      weights[t] = w;
    }
  }
}

template <typename T, int D, int GB>
int finish_weighed(const int32_t* seqlen, void* out, const int32_t* ws_rows, const float* ws_ml, const float* ws_acc,
                   const DecodeArgs& a, const Weighed& ext, hipStream_t stream) {
  const int64_t capacity = int64_t(a.max_blocks) << a.bs_log2;
  // a workgroup per stretch, fewer where the tables are wide for their rows' lengths (they go round then)
  const int64_t want = (capacity + kStretch - 1) / kStretch, most = std::max<int64_t>(1, 8192 / (int64_t(a.H_kv) * a.B));
  const int n = int(std::min(want, most));
  hipLaunchKernelGGL((paged_decode_weigh_kernel<T, D, GB>), dim3(a.H_kv * n + a.H, a.B), dim3(kWeighThreads),
                     a.G * 2 * sizeof(float), stream, seqlen, ws_rows, ws_ml, ws_acc, static_cast<T*>(out), a, ext, n);
  return launch_status("mi_paged_decode_weigh (merge and weights)");
}

size_t scores_bytes(int B, int H, int block_size, int max_blocks) {
  return size_t(B) * H * size_t(max_blocks) * block_size * sizeof(float);
}

}  // namespace
}  // namespace miattn

extern "C" size_t mi_paged_decode_weigh_workspace_size(int B, int H, int H_kv, int D, int block_size, int max_blocks,
                                                       int dtype) {
  using namespace miattn;
  if (!shape_ok(B, H, H_kv, D, block_size, max_blocks, dtype)) return 0;
  const Plan p = make_plan(B, H, H_kv, D, block_size, max_blocks, dtype);
  return p.rows_bytes + p.ml_bytes + p.acc_bytes + scores_bytes(B, H, block_size, max_blocks);
}

extern "C" int mi_paged_decode_weigh(const void* q, const void* k_cache, const void* v_cache,
                                     const int32_t* block_table, const int32_t* seqlen, void* out, int B, int H,
                                     int H_kv, int D, int block_size, int max_blocks, const int64_t* strides,
                                     float scale, int dtype, float* weights, int64_t weights_s0, int64_t weights_s1,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace miattn;
  if (weights == nullptr && B > 0) return fail(MI_ERR_INVALID, "mi_paged_decode_weigh: weights is NULL");
  Weighed w{};
  w.weights = weights;
  w.ws0 = weights_s0;
  w.ws1 = weights_s1;
  size_t inner = workspace_bytes;
  if (shape_ok(B, H, H_kv, D, block_size, max_blocks, dtype)) {
    if (D == 16) return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_weigh: head_dim 16 is not supported (32, 64, 128, 256)");
    if (H / H_kv > 4096) return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_weigh: at most 4096 query heads per KV head");
    const size_t base = mi_paged_decode_workspace_size(B, H, H_kv, D, block_size, max_blocks, dtype);
    const size_t need = base + scores_bytes(B, H, block_size, max_blocks);
    if (workspace == nullptr || workspace_bytes < need) {
      return fail(MI_ERR_WORKSPACE, "mi_paged_decode_weigh: workspace of %zu bytes < %zu needed", workspace_bytes, need);
    }
    w.scores = reinterpret_cast<float*>(static_cast<char*>(workspace) + base);
    inner = base;
  }
  return paged_decode_entry(q, k_cache, v_cache, block_table, seqlen, out, B, H, H_kv, D, block_size, max_blocks,
                            strides, scale, dtype, workspace, inner, stream, w);
}
