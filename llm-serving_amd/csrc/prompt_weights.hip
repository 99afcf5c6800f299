// Where the last queries of each prompt look: for every key j of a packed prompt,
//   w[kv, j] = sum over the query heads h of KV head kv and the prompt's last `observe` queries i >= j of
//              softmax(scale * q[i, h] K^T)[j]   (causal).
//
// A weight needs its query's maximum and sum over all keys, so the scores are computed twice, on the matrix cores, and
// stored never (in fp32 they would be 4 bytes per pair, more time in memory than the product takes):
//   1. sums: (m, l) of every observed (query, head) over its keys, 64 rows (two units of 32 queries of a head) to a
//      workgroup, so that a K row read serves all of them; S^T = K Q^T puts a query's scores in one lane (and
//      lane ^ 32), so the running maximum and sum need no exchange until the end. Few rows over many keys are cut into
//      pieces of the keys, whose (m, l) a launch between the two joins.
//   2. weights: S = Q K^T for 64 keys per workgroup over all rows that see them; a key's weights lie in one
//      lane, summed in registers in the order of the rows, then over the waves. No atomics: the same sums
//      in the same order on every run.
// In the first every wave has keys of its own, in the second rows of its own: nothing is loaded twice by a workgroup, and no
// barrier stands in the loops. Bound by the vector pipe: per 32 x 32 scores of a wave 16 v_exp_f32 (16 cycles each)
// and 3 other operations per register, beside 8 matrix instructions of 32 cycles (head_dim 128). Prompts of 4096, 2048,
// 1742 and 306 tokens, H 16 / H_kv 8 / D 128, all queries (49 GFLOP counted once): 68 + 69 us, of which the exponentials
// alone are 21 each; 8 prompts of 4311 tokens, last 32 queries: 8.6 + 3.0 (join) + 8.2 us under a profiler, 16.8 in all in
// a replayed graph, launches and round trips.
#include <algorithm>
#include <new>
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

constexpr int kHeader = 8;      // {pieces, joins, key blocks, partial slots, units, H, H_kv, longest segment}
constexpr int kPieceWords = 8;  // {seq0, L, observed queries, row block, first step, end step, partial slot or -1, first unit}
constexpr int kJoinWords = 8;   // {first partial slot, pieces, the segment's first unit, row block, observed queries, 0, 0, 0}
constexpr int kBlockWords = 8;  // {seq0, L, observed queries, key block, the segment's first unit, segment, 0, 0}
constexpr int kStep = 128;      // keys of a step of launch 1, 32 per wave
constexpr int kMaxPieces = 32;  // of a row block
// Units of 32 rows in a row block (launch 1), 32s of keys in a key block (launch 2): what a wave holds as operands. With 4 a
// wave streams half as much past them, 20 registers more leave two waves per SIMD, and no time is gained (72 us).
constexpr int kHeld = 2, kRows = 32 * kHeld, kKeys = 32 * kHeld;
constexpr int kWaves = 4;

struct WeightArgs {
  const int32_t* sched;
  float2* ml;    // [partial slot][H_kv][kRows]: (m, l) of the pieces of row blocks that are cut
  float2* rows;  // [H_kv][units][32]: (m, 1 / l) of every row
  float* out;
  int64_t os0, os1;
  int H, H_kv, G, n_pieces, n_joins, n_blocks, units, width;
  float scale_log2;
};

// A division leaves a uniform value in vector registers, where an address made from it would be taken lane by lane.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

typedef __attribute__((address_space(3))) void lds_void_t;

// 16 bytes per lane from a buffer straight into LDS, lane l to bytes 16 l .. of `dst`.
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t rs, uint8_t* dst, int offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)((__attribute__((address_space(3))) uint8_t*)dst), 16, offset, 0, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00020000);
}

// A wave's own 32 rows of D elements in LDS, filled from memory without registers between: a wave-wide load writes 1 KiB, RPS
// whole rows, 16-byte chunk c of row r at slot c ^ sw(r). Loaded straight into operand registers each lane would fetch its own
// row, 32 lines per instruction (here 8), 16 bytes of each at a time: 119 and 133 us against 79 and 101 (as above). No
// other wave reads the buffer, so there is no barrier: a wave waits for its own loads, reads its operands and fills the buffer
// again at once, and the next tile lands behind the products and exponentials of this one (a second buffer: two waves
// per SIMD in place of three in launch 1, 78 us against 72).
template <int D>
struct Tile32 {
  static constexpr int ROWB = D * 2, NCH = D / 8, RPS = 1024 / ROWB, LOADS = 32 / RPS, BYTES = 32 * ROWB;
  // rows whose chunk c share a bank fall on 16 (8 at head_dim 64, two rows to the 64 banks) different slots
  static __device__ __forceinline__ int sw(int r) { return D == 64 ? (r >> 1) & 7 : r & 15; }
  static constexpr int PERIOD = (16 + RPS - 1) / RPS < LOADS ? 16 / RPS : LOADS;  // loads after which sw repeats

  int off[PERIOD], step;
  // stride: bytes from a row to the next
  __device__ __forceinline__ void init(int stride) {
    const int lane = __lane_id();
#pragma unroll
    for (int j = 0; j < PERIOD; ++j) {
      const int r = j * RPS + lane / NCH;
      off[j] = r * stride + (((lane % NCH) ^ sw(r)) << 4);
    }
    step = PERIOD * RPS * stride;
  }
  // rows past `rows` read as zeros
  __device__ __forceinline__ void load(const void* base, int rows, int stride, uint8_t* dst) const {
    const auto rs = resource(base, rows * stride);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      load_lds16(rs, dst + j * 1024, off[j % PERIOD] + (j / PERIOD) * step);
    }
  }
  // the matrix operand of k-step ks: row lane & 31, elements 16 ks + 8 (lane >> 5) ..
  __device__ __forceinline__ static uint4 operand(const uint8_t* buf, int ks) {
    const int lane = __lane_id(), r = lane & 31;
    return *reinterpret_cast<const uint4*>(buf + r * ROWB + (((ks * 2 + (lane >> 5)) ^ sw(r)) << 4));
  }
};

// Waits for the wave's loads; LDS reads stay behind it.
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0 | (7 << 4) | (15 << 8));  // vmcnt 0
  asm volatile("" ::: "memory");
}
// Waits until the operands are in their registers: the buffer that they came from may be filled again.
template <int KS>
__device__ __forceinline__ void wait_operands(uint4 (&f)[KS]) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(f[ks].x), "+v"(f[ks].y), "+v"(f[ks].z), "+v"(f[ks].w) : : "memory");
}

// 32 x 32 scores: a's rows against b's.
template <typename T, int KS>
__device__ __forceinline__ floatx16 product(const uint4 (&a)[KS], const uint4 (&b)[KS]) {
  floatx16 c;
#pragma unroll
  for (int e = 0; e < 16; ++e) c[e] = 0.0f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) c = mfma32<T>(a[ks], b[ks], c);
  return c;
}

// Each of the KS matrix instructions of the next 32 x 32 scores among N vector instructions on the last ones: the two or three
// waves of a SIMD do not hide each other's by themselves (launch 1: 72 us against 78 with all products first).
template <int KS, int N>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x0008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x0002, N, 0);
  }
}

// A segment's rows in units of 32: unit u is head kv * G + u % G at queries first + 32 (u / G) .. (fewer at the end),
// so a unit's rows lie H * D apart and the units of a row block see about the same keys.
struct Unit {
  int i0, head, rows;
};
__device__ __forceinline__ Unit unit_at(int qb, int g, int first, int L, int kv, int G) {
  Unit x;
  x.i0 = first + qb * 32;
  x.head = kv * G + g;
  x.rows = uniform(min(32, L - x.i0));
  return x;
}
__device__ __forceinline__ Unit unit_of(int u, int first, int L, int kv, int G) {
  const int qb = uniform(u / G);
  return unit_at(qb, u - qb * G, first, L, kv, G);
}

// What launch 2 takes of a row: its maximum and 1 / sum; nothing of one that is not there or whose scores are all -inf.
__device__ __forceinline__ float2 row_record(bool there, float M, float sum) {
  return there && M != -INFINITY ? make_float2(M, 1.0f / sum) : make_float2(INFINITY, 0.0f);
}

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 3) void prompt_sums_kernel(const T* __restrict__ q, const T* __restrict__ k,
                                                                            WeightArgs a) {
  using Tl = Tile32<D>;
  constexpr int KS = D / 16;
  __shared__ float2 sm[4][kRows];
  __shared__ __align__(512) uint8_t tiles[4][Tl::BYTES];
  const int item = uniform(int(blockIdx.x) / a.H_kv), kv = int(blockIdx.x) - item * a.H_kv;  // a KV head's workgroups on one XCD where H_kv is the XCDs' multiple
  const int32_t* it = a.sched + kHeader + kPieceWords * item;
  const int seq0 = uniform(it[0]), L = uniform(it[1]), observed = uniform(it[2]), rb0 = uniform(it[3]);
  const int step0 = uniform(it[4]), step1 = uniform(it[5]), slot = uniform(it[6]), unit0 = uniform(it[7]);
  const int first = L - observed, units = (observed + 31) / 32 * a.G;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, g = lane >> 5;
  const int k_stride = a.H_kv * D * 2;
  const char* kbase = reinterpret_cast<const char*>(k + int64_t(seq0) * a.H_kv * D + kv * D);
  Tl tile;
  tile.init(k_stride);
  uint8_t* buf = tiles[wave];
  auto issue = [&](int key0) {
    tile.load(kbase + int64_t(key0) * k_stride, uniform(min(32, max(0, L - key0))), k_stride, buf);
  };
  const int key_first = step0 * kStep + wave * 32;
  issue(key_first);
  uint4 qf[kHeld][KS];
  int see[kHeld], least = 0, most = 0;  // last key that this lane's rows see; that the block's first and last row see
#pragma unroll
  for (int rb = 0; rb < kHeld; ++rb) {
    const Unit u = unit_of(min(rb0 * kHeld + rb, units - 1), first, L, kv, a.G);
    const T* p = q + (int64_t(seq0 + u.i0 + min(col, u.rows - 1)) * a.H + u.head) * D + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[rb][ks] = load16(p + ks * 16);
    see[rb] = u.i0 + min(col, u.rows - 1);
    if (rb == 0) least = u.i0;
    most = u.i0 + u.rows - 1;
  }
  float m[kHeld], l[kHeld];
#pragma unroll
  for (int rb = 0; rb < kHeld; ++rb) {
    m[rb] = -INFINITY;
    l[rb] = 0.0f;
  }
  int key0 = key_first;
  for (int s = step0; s < step1; ++s, key0 += kStep) {
    if (key0 > most) break;  // no row of the block sees a key of this wave's, here or later
    uint4 kf[KS];
    wait_loads();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = Tl::operand(buf, ks);
    wait_operands(kf);
    issue(key0 + kStep);  // (a tile past the segment reads nothing)
    auto fold_all = [&](auto masked) {
      floatx16 cur = product<T>(kf, qf[0]);
#pragma unroll
      for (int rb = 0; rb < kHeld; ++rb) {
        floatx16 sc = cur;
        if (rb + 1 < kHeld) cur = product<T>(kf, qf[rb + 1]);
        if constexpr (decltype(masked)::value) {
          const int lim = see[rb] - key0 - g * 4;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if ((e >> 2) * 8 + (e & 3) > lim) sc[e] = -INFINITY;
          }
        }
        float t = sc[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) t = fmaxf(t, sc[e]);
        t *= a.scale_log2;
        // the reference maximum moves only when it is passed by 2^8: the sum is exact against any reference
        const float to = t > m[rb] + 8.0f ? t : m[rb];
        const float u = to == -INFINITY ? 0.0f : to;
        float sum[4];  // four chains: one of 16 dependent additions is longer than the exponentials take
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = fast_exp2(fmaf(sc[e], a.scale_log2, -u));
          sum[e & 3] = e < 4 ? p : sum[e & 3] + p;
        }
        l[rb] = fmaf(l[rb], fast_exp2(m[rb] - u), (sum[0] + sum[1]) + (sum[2] + sum[3]));
        m[rb] = to;
        if (rb + 1 < kHeld) interleave<KS, decltype(masked)::value ? 13 : 9>();
      }
    };
    if (key0 + 31 > least) {
      fold_all(std::true_type{});
    } else {
      fold_all(std::false_type{});
    }
  }
  wait_loads();
  // the two halves of the wave, then the four waves
#pragma unroll
  for (int rb = 0; rb < kHeld; ++rb) {
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
    if (slot >= 0) {
      a.ml[(int64_t(slot) * a.H_kv + kv) * kRows + tid] = make_float2(M, sum);
    } else {  // the whole key range: nothing to join
      const int u = rb0 * kHeld + tid / 32;
      if (u < units) {
        a.rows[(int64_t(kv) * a.units + unit0 + u) * 32 + tid % 32] = row_record(u / a.G * 32 + tid % 32 < observed, M, sum);
      }
    }
  }
}

// Row blocks whose keys were cut: the pieces' (m, l) joined, a thread per row, 16 pieces per round trip. (Joined by launch
// 2 itself, a wave waited for the record, then the pieces, in each of its steps: 99 us for what took 81 then. By its workgroups
// before their first step, where there are few rows: 11.3 us for 6.8 and the join's 2.0.)
__global__ __launch_bounds__(kRows) void prompt_join_kernel(WeightArgs a) {
  constexpr int N = 16;
  const int item = uniform(int(blockIdx.x) / a.H_kv), kv = int(blockIdx.x) - item * a.H_kv, tid = threadIdx.x;
  const int32_t* it = a.sched + kHeader + kPieceWords * a.n_pieces + kJoinWords * item;
  const int slot = it[0], pieces = it[1], unit0 = it[2], u = it[3] * kHeld + tid / 32, observed = it[4];
  float M = -INFINITY, sum = 0.0f;
  for (int c0 = 0; c0 < pieces; c0 += N) {
    float2 p[N];
#pragma unroll
    for (int c = 0; c < N; ++c) p[c] = a.ml[(int64_t(slot + min(c0 + c, pieces - 1)) * a.H_kv + kv) * kRows + tid];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const bool there = c0 + c < pieces;  // (a break here would index p at run time, in scratch)
      const float to = there ? fmaxf(M, p[c].x) : M, z = to == -INFINITY ? 0.0f : to;
      sum = fmaf(sum, fast_exp2(M - z), there ? p[c].y * fast_exp2(p[c].x - z) : 0.0f);
      M = to;
    }
  }
  if (u < (observed + 31) / 32 * a.G) {
    a.rows[(int64_t(kv) * a.units + unit0 + u) * 32 + tid % 32] = row_record(u / a.G * 32 + tid % 32 < observed, M, sum);
  }
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 1 : 2) void prompt_weights_kernel(const T* __restrict__ q,
                                                                                    const T* __restrict__ k, WeightArgs a) {
  using Tl = Tile32<D>;
  constexpr int KS = D / 16;
  __shared__ float sums[kWaves][kKeys];
  __shared__ __align__(16) float ref[kWaves][32], inv[kWaves][32];
  __shared__ __align__(512) uint8_t tiles[kWaves][Tl::BYTES];
  const int item = uniform(int(blockIdx.x) / a.H_kv), kv = int(blockIdx.x) - item * a.H_kv;
  const int32_t* it = a.sched + kHeader + kPieceWords * a.n_pieces + kJoinWords * a.n_joins + kBlockWords * item;
  const int seq0 = uniform(it[0]), L = uniform(it[1]), observed = uniform(it[2]), key0 = uniform(it[3]) * kKeys;
  const int unit0 = uniform(it[4]), seg = uniform(it[5]);
  const int first = L - observed, units = (observed + 31) / 32 * a.G;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, g = lane >> 5;
  const int q_stride = a.H * D * 2;
  Tl tile;
  tile.init(q_stride);
  uint8_t* buf = tiles[wave];
  auto issue = [&](const Unit& x) {
    tile.load(q + (int64_t(seq0 + x.i0) * a.H + x.head) * D, x.rows, q_stride, buf);
  };
  // units that see the first key, every kWaves-th of them; the next one's place is counted on (a division per step would not be
  // hidden)
  int u = (key0 > first ? (key0 - first) / 32 * a.G : 0) + wave;
  int qb = uniform(u / a.G), hd = u - qb * a.G;
  const int dq = uniform(kWaves / a.G), dr = kWaves - dq * a.G, last_qb = (observed - 1) / 32;
  const float2* records = a.rows + (int64_t(kv) * a.units + unit0) * 32 + col;
  Unit x = unit_at(min(qb, last_qb), hd, first, L, kv, a.G);  // (past the last unit, some other one: loaded and not used)
  float2 part = records[min(u, units - 1) * 32];
  issue(x);
  uint4 kf[kHeld][KS];
#pragma unroll
  for (int kb = 0; kb < kHeld; ++kb) {
    const T* p = k + (int64_t(seq0) + min(key0 + kb * 32 + col, L - 1)) * (a.H_kv * D) + kv * D + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[kb][ks] = load16(p + ks * 16);
  }
  float w[kHeld] = {};
  for (; u < units; u += kWaves) {
    // the next unit's rows and record go out here, this unit's have had a step to land
    const Unit now = x;
    if (g == 0) {  // where every lane of the wave can read it
      ref[wave][col] = part.x;
      inv[wave][col] = part.y;
    }
    qb += dq;
    hd += dr;
    if (hd >= a.G) {
      hd -= a.G;
      ++qb;
    }
    x = unit_at(min(qb, last_qb), hd, first, L, kv, a.G);
    uint4 qf[KS];
    wait_loads();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = Tl::operand(buf, ks);
    wait_operands(qf);
    part = records[min(u + kWaves, units - 1) * 32];
    issue(x);
    auto add = [&](auto masked) {
      float m[16], by[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 m4 = *reinterpret_cast<const float4*>(&ref[wave][8 * j + 4 * g]);
        const float4 i4 = *reinterpret_cast<const float4*>(&inv[wave][8 * j + 4 * g]);
        m[4 * j] = m4.x, m[4 * j + 1] = m4.y, m[4 * j + 2] = m4.z, m[4 * j + 3] = m4.w;
        by[4 * j] = i4.x, by[4 * j + 1] = i4.y, by[4 * j + 2] = i4.z, by[4 * j + 3] = i4.w;
      }
      floatx16 cur = product<T>(qf, kf[0]);
#pragma unroll
      for (int kb = 0; kb < kHeld; ++kb) {
        const floatx16 sc = cur;
        if (kb + 1 < kHeld) cur = product<T>(qf, kf[kb + 1]);
        // rows below lim do not see the key, those from `there` on are none: zeros, whose product with an infinite key is NaN
        const int lim = key0 + kb * 32 + col - now.i0 - 4 * g, there = now.rows - 4 * g;
        float t[4];  // long sums: a unit's weights are added up (in four chains) before they join the others
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p = fast_exp2(fmaf(sc[e], a.scale_log2, -m[e]));
          const float to = e < 4 ? p * by[e] : fmaf(p, by[e], t[e & 3]);
          // (a row's 1 / sum may be NaN: what does not see the key adds nothing, not 0 times that)
          const int r = (e >> 2) * 8 + (e & 3);
          const bool hidden = decltype(masked)::value && (r < lim || r >= there);
          t[e & 3] = hidden ? (e < 4 ? 0.0f : t[e & 3]) : to;
        }
        w[kb] += (t[0] + t[1]) + (t[2] + t[3]);
        if (kb + 1 < kHeld) interleave<KS, decltype(masked)::value ? 10 : 6>();
      }
    };
    if (key0 + kKeys - 1 > now.i0 || now.rows < 32) {  // some row does not see every key, or is none
      add(std::true_type{});
    } else {
      add(std::false_type{});
    }
    asm volatile("" ::: "memory");  // a wave's LDS operations complete in order
  }
  wait_loads();
#pragma unroll
  for (int kb = 0; kb < kHeld; ++kb) {
    const float s = sum_halves(w[kb]);
    if (g == 0) sums[wave][kb * 32 + col] = s;
  }
  __syncthreads();
  float* out = a.out + seg * a.os0 + kv * a.os1;
  if (tid < kKeys && key0 + tid < L) {
    float x = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; i += 4) x += (sums[i][tid] + sums[i + 1][tid]) + (sums[i + 2][tid] + sums[i + 3][tid]);
    out[key0 + tid] = x;
  }
  if (key0 + kKeys >= L) {  // the segment's last keys: zeros behind them
    for (int i = L + tid; i < a.width; i += 64 * kWaves) out[i] = 0.0f;
  }
}

template <typename T, int D>
int launch(const void* q, const void* k, const WeightArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((prompt_sums_kernel<T, D>), dim3(a.n_pieces * a.H_kv), dim3(64 * kWaves), 0, s,
                     static_cast<const T*>(q), static_cast<const T*>(k), a);
  int rc = launch_status("mi_prompt_weights (sums)");
  if (rc != MI_OK) return rc;
  if (a.n_joins > 0) {
    hipLaunchKernelGGL(prompt_join_kernel, dim3(a.n_joins * a.H_kv), dim3(kRows), 0, s, a);
    rc = launch_status("mi_prompt_weights (join)");
    if (rc != MI_OK) return rc;
  }
  hipLaunchKernelGGL((prompt_weights_kernel<T, D>), dim3(a.n_blocks * a.H_kv), dim3(64 * kWaves), 0, s,
                     static_cast<const T*>(q), static_cast<const T*>(k), a);
  return launch_status("mi_prompt_weights (weights)");
}

template <typename T>
int launch_any(const void* q, const void* k, int D, const WeightArgs& a, hipStream_t s) {
  return D == 64 ? launch<T, 64>(q, k, a, s) : D == 128 ? launch<T, 128>(q, k, a, s) : launch<T, 256>(q, k, a, s);
}

int schedule_weights(const int32_t* host_cu_seqlens, int n_seqs, int H, int H_kv, int D, int observe,
                     int32_t* host_schedule, int capacity) {
  if (host_cu_seqlens == nullptr || n_seqs < 1) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: need at least 1 segment, got %d", n_seqs);
  }
  if (H < 1 || H_kv < 1 || H % H_kv != 0) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: n_head (%d) must be a multiple of n_kv_head (%d)", H, H_kv);
  }
  if (observe < 1) return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: observe must be >= 1, got %d", observe);
  if (D != 64 && D != 128 && D != 256) {
    return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights_schedule: head_dim 64, 128 or 256, got %d", D);
  }
  const int G = H / H_kv;
  struct Piece { int seq, obs, rb, s0, s1, slot, unit0; };
  struct Join { int slot, pieces, unit0, rb, obs; };
  struct Block { int seq, obs, kb, unit0, units; };
  int64_t steps = 0, n_units = 0, n_keys = 0;
  auto units = [&](int obs) { return int64_t((obs + 31) / 32) * G; };
  auto row_blocks = [&](int obs) { return (units(obs) + kHeld - 1) / kHeld; };
  auto last_key = [&](int L, int obs, int64_t rb) {  // of a row block
    const int64_t u = std::min((rb + 1) * kHeld, units(obs)) - 1;
    return int(std::min<int64_t>(L, L - obs + (u / G + 1) * 32) - 1);
  };
  for (int s = 0; s < n_seqs; ++s) {
    const int L = host_cu_seqlens[s + 1] - host_cu_seqlens[s];
    if (L <= 0) return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: segment %d is empty", s);
    const int obs = std::min(observe, L);
    if (int64_t(obs) * G > (int64_t(1) << 30)) return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights_schedule: segment %d too long", s);
    n_units += units(obs);
    n_keys += (L + kKeys - 1) / kKeys;
    for (int rb = 0; rb < row_blocks(obs); ++rb) steps += last_key(L, obs, rb) / kStep + 1;
  }
  if (n_units * H_kv > (1 << 26) || n_keys * H_kv >= (1 << 24)) {
    return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights_schedule: too many rows or keys");
  }
  // pieces of at most an even share of the work over 512 workgroups (two per CU), at most kMaxPieces per row block: many
  // row blocks are not cut at all, and launch 2 has nothing to join
  const int share = int(std::max<int64_t>(1, (steps * H_kv + 511) / 512));
  std::vector<Piece> pieces;
  std::vector<Join> joins;
  std::vector<Block> blocks;
  int slot = 0, unit0 = 0, longest = 0;
  for (int s = 0; s < n_seqs; ++s) {
    const int L = host_cu_seqlens[s + 1] - host_cu_seqlens[s], obs = std::min(observe, L);
    longest = std::max(longest, L);
    for (int rb = 0; rb < row_blocks(obs); ++rb) {
      const int n = last_key(L, obs, rb) / kStep + 1;
      const int cuts = std::min(kMaxPieces, (n + share - 1) / share);
      if (cuts > 1) joins.push_back({slot, cuts, unit0, rb, obs});
      for (int c = 0; c < cuts; ++c) {
        pieces.push_back({s, obs, rb, int(int64_t(c) * n / cuts), int(int64_t(c + 1) * n / cuts), cuts > 1 ? slot++ : -1, unit0});
      }
    }
    for (int kb = 0; kb * kKeys < L; ++kb) {
      blocks.push_back({s, obs, kb, unit0, int(units(obs) - std::max(0, kb * kKeys - (L - obs)) / 32 * G)});
    }
    unit0 += int(units(obs));
  }
  const int64_t words64 = kHeader + int64_t(kPieceWords) * pieces.size() + int64_t(kJoinWords) * joins.size() +
                          int64_t(kBlockWords) * blocks.size();
  if (words64 > INT32_MAX || int64_t(pieces.size()) * H_kv >= (1 << 24)  /* 2^32 threads */) {
    return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights_schedule: schedule too large");
  }
  const int words = int(words64);
  if (host_schedule == nullptr) return words;
  if (capacity < words) return fail(MI_ERR_INVALID, "mi_prompt_weights_schedule: capacity %d < %d words", capacity, words);
  // longest first
  std::stable_sort(pieces.begin(), pieces.end(), [](const Piece& x, const Piece& y) { return x.s1 - x.s0 > y.s1 - y.s0; });
  std::stable_sort(blocks.begin(), blocks.end(), [](const Block& x, const Block& y) { return x.units > y.units; });
  const int32_t head[kHeader] = {int(pieces.size()), int(joins.size()), int(blocks.size()), slot, unit0, H, H_kv, longest};
  int32_t* w = std::copy(head, head + kHeader, host_schedule);
  for (const Piece& p : pieces) {
    const int32_t x[kPieceWords] = {host_cu_seqlens[p.seq], host_cu_seqlens[p.seq + 1] - host_cu_seqlens[p.seq], p.obs,
                                    p.rb, p.s0, p.s1, p.slot, p.unit0};
    w = std::copy(x, x + kPieceWords, w);
  }
  for (const Join& j : joins) {
    const int32_t x[kJoinWords] = {j.slot, j.pieces, j.unit0, j.rb, j.obs, 0, 0, 0};
    w = std::copy(x, x + kJoinWords, w);
  }
  for (const Block& b : blocks) {
    const int32_t x[kBlockWords] = {host_cu_seqlens[b.seq], host_cu_seqlens[b.seq + 1] - host_cu_seqlens[b.seq], b.obs,
                                    b.kb, b.unit0, b.seq, 0, 0};
    w = std::copy(x, x + kBlockWords, w);
  }
  return words;
}

}  // namespace
}  // namespace miattn

extern "C" int mi_prompt_weights_schedule(const int32_t* host_cu_seqlens, int n_seqs, int H, int H_kv, int D,
                                          int observe, int32_t* host_schedule, int capacity) {
  using namespace miattn;
  try {
    return schedule_weights(host_cu_seqlens, n_seqs, H, H_kv, D, observe, host_schedule, capacity);
  } catch (const std::bad_alloc&) {
    return fail(MI_ERR_UNSUPPORTED, "mi_prompt_weights_schedule: out of host memory");
  }
}

extern "C" size_t mi_prompt_weights_workspace_size(const int32_t* host_schedule, int H_kv) {
  if (host_schedule == nullptr || H_kv < 1) return 0;
  // a row's record each, then the pieces
  return (size_t(host_schedule[4]) * 32 + size_t(host_schedule[3]) * miattn::kRows) * H_kv * sizeof(float2);
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
  if (host_header[0] < 1 || host_header[1] < 0 || host_header[2] < 1 || host_header[3] < 0 || host_header[4] < 1 || width < 1) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights: bad schedule header or width %d", width);
  }
  // units, pieces and their records are counted by the heads of a group, and every key of a segment is written
  if (host_header[5] != H || host_header[6] != H_kv || width < host_header[7]) {
    return fail(MI_ERR_INVALID, "mi_prompt_weights: a schedule of %d heads over %d and segments of up to %d tokens does not fit %d "
                "over %d and width %d", host_header[5], host_header[6], host_header[7], H, H_kv, width);
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
  a.rows = static_cast<float2*>(workspace);
  a.ml = a.rows + int64_t(host_header[4]) * H_kv * 32;
  a.out = out;
  a.os0 = out_s0;
  a.os1 = out_s1;
  a.H = H;
  a.H_kv = H_kv;
  a.G = H / H_kv;
  a.n_pieces = host_header[0];
  a.n_joins = host_header[1];
  a.n_blocks = host_header[2];
  a.units = host_header[4];
  a.width = width;
  a.scale_log2 = float(double(scale) * 1.4426950408889634);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == MI_BF16 ? launch_any<bf16_t>(q, k, D, a, s) : launch_any<f16_t>(q, k, D, a, s);
}
