// Block-table paged-decode attention over the 4-bit cache (format in fp4.h): one query token per row,
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q[b, h] . k_t - max),  t < seqlen[b],
// with k_t, v_t the rows of KV head h / (H / H_kv); a row of length 0 gives zeros.
#include <type_traits>

#include "fp4.h"

namespace miattn {
namespace {

struct Fp4DecodeArgs {
  int B, H, H_kv, G, bs_log2, max_blocks;
  int64_t qs0, qs1, ks0, ks1, vs0, vs1, os0, os1, bts0;
  float scale_log2;
};

// One workgroup per (query head, row): D / 8 lanes per token, an online softmax per lane group.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_decode_fp4_kernel(const T* __restrict__ q, const uint8_t* __restrict__ kc,
                                                               const uint8_t* __restrict__ vc,
                                                               const int32_t* __restrict__ block_table,
                                                               const int32_t* __restrict__ seqlen, T* __restrict__ out,
                                                               Fp4DecodeArgs a) {
  constexpr int LPR = D / 8, NG = 256 / LPR;  // lanes per token, tokens at a time
  __shared__ float sm_ml[NG][2];
  __shared__ float sm_acc[NG][D];
  const int h = blockIdx.x, b = blockIdx.y;
  const int c = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int kvh = h / a.G;
  const int bs = 1 << a.bs_log2;
  const int cap = a.max_blocks << a.bs_log2;
  int len = seqlen[b];
  len = len < cap ? len : cap;
  float qv[8];
  load8<T, false>(q + b * a.qs0 + h * a.qs1 + c * 8, 1, qv);
  float m = -INFINITY, l = 0.0f, acc[8] = {};
  for (int t = grp; t < len; t += NG) {
    const int64_t page = block_table[b * a.bts0 + (t >> a.bs_log2)];
    const int at = t & (bs - 1);
    const int64_t code = int64_t(at) * (D / 2) + c * 4, sc = int64_t(bs) * (D / 2) + int64_t(c >> 2) * bs + at;
    const uint8_t* kp = kc + page * a.ks0 + kvh * a.ks1;
    const uint8_t* vp = vc + page * a.vs0 + kvh * a.vs1;
    float kv[8], vv[8];
    fp4_decode(*reinterpret_cast<const uint32_t*>(kp + code), fp4_scale(kp[sc]), kv);
    fp4_decode(*reinterpret_cast<const uint32_t*>(vp + code), fp4_scale(vp[sc]), vv);
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) dot = fmaf(qv[j], kv[j], dot);
    const float s = group_allreduce<LPR, SumOp>(dot) * a.scale_log2;
    const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.0f : mn;
    const float alpha = fast_exp2(m - mu), p = fast_exp2(s - mu);
    m = mn;
    l = l * alpha + p;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = fmaf(p, vv[j], acc[j] * alpha);
  }
  if (c == 0) {
    sm_ml[grp][0] = m;
    sm_ml[grp][1] = l;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sm_acc[grp][c * 8 + j] = acc[j];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 256) {
    float M = -INFINITY, L = 0.0f, A = 0.0f;
    for (int g = 0; g < NG; ++g) M = fmaxf(M, sm_ml[g][0]);
    const float mu = M == -INFINITY ? 0.0f : M;
    for (int g = 0; g < NG; ++g) {
      const float w = fast_exp2(sm_ml[g][0] - mu);
      L = fmaf(sm_ml[g][1], w, L);
      A = fmaf(sm_acc[g][d], w, A);
    }
    out[b * a.os0 + h * a.os1 + d] = from_f32<T>(fp4_saturate<T>(len > 0 ? A / L : 0.0f));
  }
}

int esize_of(int dtype) { return dtype == MI_F32 ? 4 : dtype == MI_F16 || dtype == MI_BF16 ? 2 : 0; }

bool fp4_dim(int D) { return D == 64 || D == 128 || D == 256; }

bool fp4_block(int bs) { return bs >= 16 && (bs & (bs - 1)) == 0; }

template <typename T, int D>
int launch_d(const void* q, const void* k, const void* v, const int32_t* bt, const int32_t* seqlen, void* out,
             const Fp4DecodeArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((paged_decode_fp4_kernel<T, D>), dim3(a.H, a.B), dim3(256), 0, s, static_cast<const T*>(q),
                     static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), bt, seqlen, static_cast<T*>(out), a);
  return launch_status("mi_paged_decode_fp4");
}

template <typename T>
int launch_t(int D, const void* q, const void* k, const void* v, const int32_t* bt, const int32_t* seqlen, void* out,
             const Fp4DecodeArgs& a, hipStream_t s) {
  switch (D) {
    case 64: return launch_d<T, 64>(q, k, v, bt, seqlen, out, a, s);
    case 128: return launch_d<T, 128>(q, k, v, bt, seqlen, out, a, s);
    default: return launch_d<T, 256>(q, k, v, bt, seqlen, out, a, s);
  }
}

}  // namespace
}  // namespace miattn

extern "C" size_t mi_paged_decode_fp4_workspace_size(int B, int H, int H_kv, int D, int block_size, int max_blocks,
                                                     int dtype) {
  (void)B, (void)H, (void)H_kv, (void)D, (void)block_size, (void)max_blocks, (void)dtype;
  return 0;
}

extern "C" int mi_paged_decode_fp4(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                   const int32_t* seqlen, void* out, int B, int H, int H_kv, int D, int block_size,
                                   int max_blocks, const int64_t* strides, float scale, int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  using namespace miattn;
  (void)workspace, (void)workspace_bytes;
  if (esize_of(dtype) == 0) return fail(MI_ERR_INVALID, "mi_paged_decode_fp4: unknown dtype %d", dtype);
  if (B < 0 || H < 1 || H_kv < 1 || H % H_kv != 0) {
    return fail(MI_ERR_INVALID, "mi_paged_decode_fp4: n_head (%d) must be a multiple of n_kv_head (%d)", H, H_kv);
  }
  if (!fp4_dim(D)) {
    return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_fp4: head_dim %d is not supported by the 4-bit cache (64, 128, 256)", D);
  }
  if (!fp4_block(block_size)) {
    return fail(MI_ERR_UNSUPPORTED,
                "mi_paged_decode_fp4: the 4-bit cache needs a power-of-two block_size of at least 16, got %d", block_size);
  }
  if (max_blocks < 1) return fail(MI_ERR_INVALID, "mi_paged_decode_fp4: max_blocks must be >= 1");
  if (strides == nullptr) return fail(MI_ERR_INVALID, "mi_paged_decode_fp4: strides is NULL");
  if (B == 0) return MI_OK;
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || block_table == nullptr || seqlen == nullptr ||
      out == nullptr) {
    return fail(MI_ERR_INVALID, "mi_paged_decode_fp4: NULL tensor pointer");
  }
  if ((long long)max_blocks * block_size * B > 2147483647LL) {
    return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_fp4: B * max_blocks * block_size must stay below 2^31 tokens");
  }
  if (B > 65535 || H > 65535) {
    return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_fp4: grid too large (B=%d, H=%d)", B, H);
  }
  const int64_t* st = strides;
  const int es = esize_of(dtype);
  bool ok = true;
  for (const void* p : {q, k_cache, v_cache, static_cast<const void*>(out)}) ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i : {0, 1, 6, 7}) ok = ok && (st[i] * es) % 16 == 0;
  for (int i : {2, 3, 4, 5}) ok = ok && st[i] % 16 == 0;
  if (!ok) {
    return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_fp4: q, out, k_cache and v_cache need 16-byte aligned rows and heads");
  }
  Fp4DecodeArgs a;
  a.B = B; a.H = H; a.H_kv = H_kv; a.G = H / H_kv; a.max_blocks = max_blocks;
  a.bs_log2 = __builtin_ctz(unsigned(block_size));
  a.qs0 = st[0]; a.qs1 = st[1]; a.ks0 = st[2]; a.ks1 = st[3]; a.vs0 = st[4]; a.vs1 = st[5];
  a.os0 = st[6]; a.os1 = st[7]; a.bts0 = st[8];
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MI_BF16: return launch_t<bf16_t>(D, q, k_cache, v_cache, block_table, seqlen, out, a, s);
    case MI_F16: return launch_t<f16_t>(D, q, k_cache, v_cache, block_table, seqlen, out, a, s);
    default: return launch_t<float>(D, q, k_cache, v_cache, block_table, seqlen, out, a, s);
  }
}
