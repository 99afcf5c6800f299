// Where the last queries of each prompt look: for every key j of a packed prompt,
//   w[kv, j] = sum over the query heads h of KV head kv and the prompt's last `observe` queries i >= j of
//              softmax(scale * q[i, h] K^T)[j]   (causal).
//
// A weight needs its query's maximum and sum over all keys, so the scores are computed twice, on the matrix cores, and
// stored never (in fp32 they would be 4 bytes per pair, more time in memory than the product takes):
//   1. sums: (m, l) of every observed (query, head) over its keys. The G heads of a KV head and its queries are
//      the rows r = (query - first) * G + head of one matrix, 64 rows to a workgroup, so a K row
//      read serves all of them; S^T = K Q^T puts a query's scores in one lane (and lane ^ 32), so the running
//      maximum and sum need no exchange until the end. Long key ranges are cut into pieces
//      whose (m, l) the second launch joins.
//   2. weights: S = Q K^T for 64 keys per workgroup over all rows that see them; a key's weights lie in one
//      lane, summed in registers in the order of the rows, then over the waves. No atomics: the same sums
//      in the same order on every run.
// Operands go straight from memory to registers in both: in the first every wave has keys of its own, in the second rows
// of its own, so nothing is loaded twice by a workgroup and no barrier stands in the loops; the next tile's loads
// are issued when the matrix instructions have taken the last one's registers and land behind its exponentials. Bound by
// those: per 32 x 32 scores of a wave 16 v_exp_f32 (16 cycles each) and 3 vector operations per
// register beside 8 matrix instructions of 32 cycles (head_dim 128).
#include <algorithm>
#include <vector>

#include "common.h"

namespace miattn {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));

template <typename T>
__device__ __forceinline__ floatx16 mfma32(const uint4& a, const uint4& b, const floatx16& c) {
  if constexpr (std::is_same<T, bf16_t>::value) {
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

constexpr int kHeader = 4;      // {pieces of launch 1, key blocks of launch 2, row blocks, partial slots}
constexpr int kPieceWords = 8;  // {seq0, L, observed queries, row block, first step, end step, partial slot, 0}
constexpr int kBlockWords = 8;  // {seq0, L, observed queries, key block, the segment's first row block, segment, 0, 0}
constexpr int kRowWords = 2;    // a row block: {first partial slot, pieces}
constexpr int kRows = 64;       // rows of a row block
constexpr int kStep = 128;      // keys of a step of launch 1, 32 per wave
constexpr int kKeys = 64;       // keys of a workgroup of launch 2
constexpr int kMaxPieces = 32;  // of a row block

struct WeightArgs {
  const int32_t* sched;
  float2* ml;  // [partial slot][H_kv][kRows]
  float* out;
  int64_t os0, os1;
  int H, H_kv, G, n_pieces, n_blocks, width;
  float scale_log2;
};

// Row r of a segment's observed rows: its query, and the q row's element offset at head kv * G.
__device__ __forceinline__ int64_t q_offset(int seq0, int first, int r, int kv, int D, const WeightArgs& a) {
  const int i = r / a.G;
  return (int64_t(seq0 + first + i) * a.H + kv * a.G + (r - i * a.G)) * D;
}

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void prompt_sums_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                                            WeightArgs a) {
  constexpr int KS = D / 16;
  __shared__ float2 sm[4][kRows];
  const int kv = int(blockIdx.x) % a.H_kv;  // a KV head's workgroups on one XCD where H_kv is the XCDs' multiple
  const int32_t* it = a.sched + kHeader + kPieceWords * (int(blockIdx.x) / a.H_kv);
  const int seq0 = it[0], L = it[1], observed = it[2], row0 = it[3] * kRows, step0 = it[4], step1 = it[5], slot = it[6];
  const int first = L - observed, rows = observed * a.G;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, g = lane >> 5;
  uint4 qf[2][KS];
  int see[2];  // last key that this lane's rows see
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const int r = min(row0 + rb * 32 + col, rows - 1);
    const T* p = q + q_offset(seq0, first, r, kv, D, a) + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[rb][ks] = load16(p + ks * 16);
    see[rb] = first + r / a.G;
  }
  const int least = first + row0 / a.G;                               // last key of the block's first row
  const int most = first + (min(row0 + kRows, rows) - 1) / a.G;       // and of its last
  const int64_t k_row = int64_t(a.H_kv) * D;
  const T* kbase = k + int64_t(seq0) * k_row + kv * D + g * 8;
  uint4 kf[KS];
  auto load = [&](int key0) {
    const T* p = kbase + min(key0 + col, L - 1) * k_row;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = load16(p + ks * 16);
  };
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  int key0 = step0 * kStep + wave * 32;
  load(key0);
  for (int s = step0; s < step1; ++s, key0 += kStep) {
    floatx16 sc[2];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[rb][e] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sc[rb] = mfma32<T>(kf[ks], qf[rb][ks], sc[rb]);
    }
    if (s + 1 < step1) load(key0 + kStep);
    if (key0 > most) continue;  // no row of the block sees a key of this wave's
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      if (key0 + 31 > least) {
        const int lim = see[rb] - key0 - g * 4;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if ((e >> 2) * 8 + (e & 3) > lim) sc[rb][e] = -INFINITY;
        }
      }
      float t = sc[rb][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) t = fmaxf(t, sc[rb][e]);
      t *= a.scale_log2;
      // the reference maximum moves only when it is passed by 2^8: the sum is exact against any reference
      const float to = t > m[rb] + 8.0f ? t : m[rb];
      const float u = to == -INFINITY ? 0.0f : to;
      float sum = l[rb] * fast_exp2(m[rb] - u);
#pragma unroll
      for (int e = 0; e < 16; ++e) sum += fast_exp2(fmaf(sc[rb][e], a.scale_log2, -u));
      l[rb] = sum;
      m[rb] = to;
    }
  }
  // the two halves of the wave, then the four waves
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const float M = max_halves(m[rb]), u = M == -INFINITY ? 0.0f : M;
    const float sum = sum_halves(l[rb] * fast_exp2(m[rb] - u));
    if (g == 0) sm[wave][rb * 32 + col] = make_float2(M, sum);
  }
  __syncthreads();
  if (tid < kRows) {
    float M = sm[0][tid].x;
#pragma unroll
    for (int w = 1; w < 4; ++w) M = fmaxf(M, sm[w][tid].x);
    const float u = M == -INFINITY ? 0.0f : M;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum = fmaf(sm[w][tid].y, fast_exp2(sm[w][tid].x - u), sum);
    a.ml[(int64_t(slot) * a.H_kv + kv) * kRows + tid] = make_float2(M, sum);
  }
}

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void prompt_weights_kernel(const T* __restrict__ q,
                                                                               const T* __restrict__ k, WeightArgs a) {
  constexpr int KS = D / 16;
  __shared__ float sums[4][kKeys];
  __shared__ __align__(16) float ref[4][32], inv[4][32];
  __shared__ __align__(16) int sees[4][32];
  const int kv = int(blockIdx.x) % a.H_kv;
  const int32_t* it = a.sched + kHeader + kPieceWords * a.n_pieces + kBlockWords * (int(blockIdx.x) / a.H_kv);
  const int32_t* row_blocks = a.sched + kHeader + kPieceWords * a.n_pieces + kBlockWords * a.n_blocks;
  const int seq0 = it[0], L = it[1], observed = it[2], key0 = it[3] * kKeys, rb0 = it[4], seg = it[5];
  const int first = L - observed, rows = observed * a.G;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, g = lane >> 5;
  const int64_t k_row = int64_t(a.H_kv) * D;
  uint4 kf[2][KS];
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const T* p = k + (int64_t(seq0) + min(key0 + kb * 32 + col, L - 1)) * k_row + kv * D + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[kb][ks] = load16(p + ks * 16);
  }
  const int n32 = (rows + 31) / 32;
  int rb = (key0 > first ? (key0 - first) * a.G / 32 : 0) + wave;  // 32-row blocks that see the first key, shared out
  uint4 qf[KS];
  float2 part = make_float2(0.0f, 1.0f);
  int2 rec = make_int2(0, 1);
  auto load = [&](int x) {
    const int r = min(x * 32 + col, rows - 1);
    const T* p = q + q_offset(seq0, first, r, kv, D, a) + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load16(p + ks * 16);
    rec = *reinterpret_cast<const int2*>(row_blocks + kRowWords * (rb0 + x / 2));
    part = a.ml[(int64_t(rec.x) * a.H_kv + kv) * kRows + (x & 1) * 32 + col];
  };
  float w[2] = {0.0f, 0.0f};  // long sums: the 16 weights of a tile are added up before they join (1.8e-7 -> see below)
  if (rb < n32) load(rb);
  for (; rb < n32; rb += 4) {
    // The rows' maxima and 1 / sums, and the last key each sees, where every lane of the wave can read them. A weight
    // is exp2(s - m) / l, not exp2(s - log2 of both): m + log2 l would be rounded at its own size, 2^-19 from 16 on.
    {
      float M = part.x, sum = part.y;
      for (int c0 = 1; c0 < rec.y; c0 += 8) {  // eight pieces per round trip
        float2 p[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          p[c] = a.ml[(int64_t(rec.x + min(c0 + c, rec.y - 1)) * a.H_kv + kv) * kRows + (rb & 1) * 32 + col];
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c0 + c >= rec.y) break;
          const float to = fmaxf(M, p[c].x), u = to == -INFINITY ? 0.0f : to;
          sum = fmaf(sum, fast_exp2(M - u), p[c].y * fast_exp2(p[c].x - u));
          M = to;
        }
      }
      const int r = rb * 32 + col;
      const bool none = r >= rows || M == -INFINITY;  // rows past the last one, and ones whose scores are all -inf
      if (g == 0) {
        ref[wave][col] = none ? INFINITY : M;
        inv[wave][col] = none ? 0.0f : 1.0f / sum;
        sees[wave][col] = first + min(r, rows - 1) / a.G;
      }
    }
    floatx16 sc[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[kb][e] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) sc[kb] = mfma32<T>(qf[ks], kf[kb][ks], sc[kb]);
    }
    const bool partial = key0 + kKeys - 1 > first + rb * 32 / a.G;  // some row does not see every key
    if (rb + 4 < n32) load(rb + 4);
    asm volatile("" ::: "memory");  // a wave's LDS operations complete in order
    float t16[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 m4 = *reinterpret_cast<const float4*>(&ref[wave][8 * j + 4 * g]);
      const float4 i4 = *reinterpret_cast<const float4*>(&inv[wave][8 * j + 4 * g]);
      const float m[4] = {m4.x, m4.y, m4.z, m4.w}, by[4] = {i4.x, i4.y, i4.z, i4.w};
      int4 last = make_int4(0, 0, 0, 0);
      if (partial) last = *reinterpret_cast<const int4*>(&sees[wave][8 * j + 4 * g]);
      const int t[4] = {last.x, last.y, last.z, last.w};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float p = fast_exp2(fmaf(sc[kb][4 * j + e], a.scale_log2, -m[e]));
          if (partial && key0 + kb * 32 + col > t[e]) p = 0.0f;
          t16[kb] = fmaf(p, by[e], t16[kb]);
        }
      }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) w[kb] += t16[kb];
    asm volatile("" ::: "memory");
  }
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const float x = sum_halves(w[kb]);
    if (g == 0) sums[wave][kb * 32 + col] = x;
  }
  __syncthreads();
  float* out = a.out + seg * a.os0 + kv * a.os1;
  if (tid < kKeys && key0 + tid < L) out[key0 + tid] = (sums[0][tid] + sums[1][tid]) + (sums[2][tid] + sums[3][tid]);
  if (key0 + kKeys >= L) {  // the segment's last keys: zeros behind them
    for (int i = L + tid; i < a.width; i += 256) out[i] = 0.0f;
  }
}

template <typename T, int D>
int launch(const void* q, const void* k, const WeightArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((prompt_sums_kernel<T, D>), dim3(a.n_pieces * a.H_kv), dim3(256), 0, s, static_cast<const T*>(q),
                     static_cast<const T*>(k), a);
  const int rc = launch_status("mi_prompt_weights (sums)");
  if (rc != MI_OK) return rc;
  hipLaunchKernelGGL((prompt_weights_kernel<T, D>), dim3(a.n_blocks * a.H_kv), dim3(256), 0, s, static_cast<const T*>(q),
                     static_cast<const T*>(k), a);
  return launch_status("mi_prompt_weights (weights)");
}

}  // namespace
}  // namespace miattn

extern "C" int mi_prompt_weights_schedule(const int32_t* host_cu_seqlens, int n_seqs, int H, int H_kv, int observe,
                                          int32_t* host_schedule, int capacity) {
  using namespace miattn;
  if (host_cu_seqlens == nullptr || n_seqs < 1) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: need at least 1 segment, got %d", n_seqs);
  }
  if (H < 1 || H_kv < 1 || H % H_kv != 0) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: n_head (%d) must be a multiple of n_kv_head (%d)", H, H_kv);
  }
  if (observe < 1) return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: observe must be >= 1, got %d", observe);
  const int G = H / H_kv;
  struct Piece { int seq, obs, rb, s0, s1, slot; };
  struct Block { int seq, obs, kb, rb0, rows; };
  int64_t steps = 0, n_rows = 0, n_keys = 0;
  auto last_key = [&](int L, int obs, int rb) {  // of a row block
    return L - obs + int((std::min(int64_t(rb + 1) * kRows, int64_t(obs) * G) - 1) / G);
  };
  auto row_blocks = [&](int obs) { return (int64_t(obs) * G + kRows - 1) / kRows; };
  for (int s = 0; s < n_seqs; ++s) {
    const int L = host_cu_seqlens[s + 1] - host_cu_seqlens[s];
    if (L <= 0) return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: segment %d is empty", s);
    const int obs = std::min(observe, L);
    if (int64_t(obs) * G > (int64_t(1) << 30)) return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights_schedule: segment %d too long", s);
    n_rows += row_blocks(obs);
    n_keys += (L + kKeys - 1) / kKeys;
    for (int rb = 0; rb < row_blocks(obs); ++rb) steps += last_key(L, obs, rb) / kStep + 1;
  }
  if (n_rows > (1 << 24) || n_keys * H_kv > INT32_MAX) {
    return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights_schedule: too many rows or keys");
  }
  // pieces of at most an even share of the work over 1024 workgroups (two to four per CU), at most kMaxPieces per row block
  const int share = int(std::max<int64_t>(1, (steps * H_kv + 1023) / 1024));
  std::vector<Piece> pieces;
  std::vector<Block> blocks;
  std::vector<int32_t> rows;
  int slot = 0;
  for (int s = 0; s < n_seqs; ++s) {
    const int L = host_cu_seqlens[s + 1] - host_cu_seqlens[s], obs = std::min(observe, L);
    const int rb0 = int(rows.size()) / kRowWords;
    for (int rb = 0; rb < row_blocks(obs); ++rb) {
      const int n = last_key(L, obs, rb) / kStep + 1;
      const int cuts = std::min(kMaxPieces, (n + share - 1) / share);
      rows.push_back(slot);
      rows.push_back(cuts);
      for (int c = 0; c < cuts; ++c) {
        pieces.push_back({s, obs, rb, int(int64_t(c) * n / cuts), int(int64_t(c + 1) * n / cuts), slot++});
      }
    }
    for (int kb = 0; kb * kKeys < L; ++kb) {
      const int64_t hidden = std::max<int64_t>(0, int64_t(kb) * kKeys - (L - obs)) * G;
      blocks.push_back({s, obs, kb, rb0, int(int64_t(obs) * G - hidden)});
    }
  }
  const int64_t words64 = kHeader + int64_t(kPieceWords) * pieces.size() + int64_t(kBlockWords) * blocks.size() + rows.size();
  if (words64 > INT32_MAX || int64_t(pieces.size()) * H_kv > INT32_MAX) {
    return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights_schedule: schedule too large");
  }
  const int words = int(words64);
  if (host_schedule == nullptr) return words;
  if (capacity < words) return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: capacity %d < %d words", capacity, words);
  // longest first
  std::stable_sort(pieces.begin(), pieces.end(), [](const Piece& x, const Piece& y) { return x.s1 - x.s0 > y.s1 - y.s0; });
  std::stable_sort(blocks.begin(), blocks.end(), [](const Block& x, const Block& y) { return x.rows > y.rows; });
  int32_t* w = host_schedule;
  *w++ = int(pieces.size());
  *w++ = int(blocks.size());
  *w++ = int(rows.size()) / kRowWords;
  *w++ = slot;
  for (const Piece& p : pieces) {
    const int32_t x[kPieceWords] = {host_cu_seqlens[p.seq], host_cu_seqlens[p.seq + 1] - host_cu_seqlens[p.seq], p.obs,
                                    p.rb, p.s0, p.s1, p.slot, 0};
    w = std::copy(x, x + kPieceWords, w);
  }
  for (const Block& b : blocks) {
    const int32_t x[kBlockWords] = {host_cu_seqlens[b.seq], host_cu_seqlens[b.seq + 1] - host_cu_seqlens[b.seq], b.obs,
                                    b.kb, b.rb0, b.seq, 0, 0};
    w = std::copy(x, x + kBlockWords, w);
  }
  std::copy(rows.begin(), rows.end(), w);
  return words;
}

extern "C" size_t mi_prompt_weights_workspace_size(const int32_t* host_schedule, int H_kv) {
  if (host_schedule == nullptr || H_kv < 1) return 0;
  return size_t(host_schedule[3]) * H_kv * miattn::kRows * sizeof(float2);
}

extern "C" int mi_prompt_weights(const void* q, const void* k, const int32_t* schedule, const int32_t* host_header, int H,
                                 int H_kv, int D, float scale, int dtype, float* out, int64_t out_s0, int64_t out_s1,
                                 int width, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace miattn;
  if (dtype != MI_BF16 && dtype != MI_F16) {
    return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights: fp16/bf16 only (dtype code %d)", dtype);
  }
  if (D != 64 && D != 128 && D != 256) return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights: head_dim 64, 128 or 256, got %d", D);
  if (H < 1 || H_kv < 1 || H % H_kv != 0) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights: n_head (%d) must be a multiple of n_kv_head (%d)", H, H_kv);
  }
  if (!(scale > 0.0f)) return fail(MI_ERR_INVALID, "mi_prompt_weights: scale must be positive, got %g", double(scale));
  if (q == nullptr || k == nullptr || schedule == nullptr || host_header == nullptr || out == nullptr) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights: NULL pointer argument");
  }
  if (host_header[0] < 1 || host_header[1] < 1 || host_header[2] < 1 || host_header[3] < 1 || width < 1) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights: bad schedule header or width %d", width);
  }
  auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const size_t need = mi_prompt_weights_workspace_size(host_header, H_kv);
  if (workspace == nullptr || workspace_bytes < need || !al(workspace)) {
    return fail(MI_ERR_WORKSPACE, "mi_prompt_weights: a 16-byte aligned workspace of %zu bytes is needed, got %zu", need,
                workspace_bytes);
  }
  if (!al(q) || !al(k)) return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights: q and k must be 16-byte aligned");
  WeightArgs a{};
  a.sched = schedule;
  a.ml = static_cast<float2*>(workspace);
  a.out = out;
  a.os0 = out_s0;
  a.os1 = out_s1;
  a.H = H;
  a.H_kv = H_kv;
  a.G = H / H_kv;
  a.n_pieces = host_header[0];
  a.n_blocks = host_header[1];
  a.width = width;
  a.scale_log2 = float(double(scale) * 1.4426950408889634);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MI_BF16) {
    return D == 64 ? launch<bf16_t, 64>(q, k, a, s) : D == 128 ? launch<bf16_t, 128>(q, k, a, s) : launch<bf16_t, 256>(q, k, a, s);
  }
  return D == 64 ? launch<f16_t, 64>(q, k, a, s) : D == 128 ? launch<f16_t, 128>(q, k, a, s) : launch<f16_t, 256>(q, k, a, s);
}
