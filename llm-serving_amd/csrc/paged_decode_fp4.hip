// Block-table paged-decode attention over the 4-bit cache (format in fp4.h): one query token per row,
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q[b, h] . k_t - max),  t < seqlen[b],
// with k_t, v_t the rows of KV head h / (H / H_kv); a row of length 0 gives zeros.
//
// A token of one KV head is 17 D / 32 bytes each of K and V for 4 D operations per query head, and turning a 4-bit
// element into an operand costs vector instructions that a 16-bit cache does not pay, at a quarter
// of its bytes: with the products on the vector unit too, that unit would bound the kernel and not the
// memory. So both products run on the matrix cores, and the elements are converted once for all
// query heads of their KV head:
//   * a wave works on tiles of 32 tokens of one KV head. The columns of both products are the query heads,
//     each in NC columns (below);
//   * S = K Q^T: 16 tokens are the rows of a 16x16x32 product. A lane holds D / 8 bytes of one token's row
//     (D / 4 elements under one or two scales), and v_cvt_scalef32_pk_bf16_fp4 turns two elements, scale applied,
//     into a bf16 pair in one instruction: exact, E2M1 has two significant bits. The order of the D
//     elements in the products' depth is free, so a lane's elements are in memory order and Q is laid out to match;
//   * O^T = V^T P^T: the rows are 16 elements of D, the depth 32 tokens. A lane holds D / 16 elements of each of 8
//     tokens; converted pairs lie along D and are exchanged between two tokens by v_perm_b32 (one
//     instruction per pair), so a register holds one element of two tokens. The 8 tokens are those whose scores
//     the same lane holds of S, so P needs no exchange between lanes;
//   * exactness: q of a 16-bit type in one bf16 operand (bf16) or a high and a low one (fp16), fp32 in three, all exact.
//     p is in fp32; for fp32 outputs it is cut into three bf16 parts, its 24 bits. For 16-bit outputs it is the nearest
//     bf16 and the nearest one to what that leaves: off by at most 2^-17 of p, to either side, so the errors of a row's tokens
//     average out. One output in 82 (fp16, 16 ragged rows at D 256) or 420 (bf16, 32 at D 128) is not its type's nearest
//     value to the 64-bit result; one in 27 or 160 with the second part cut (2^-14, always towards zero), one in 580 or 3400
//     with fp32 tensor operations. A third part would be exact, for 16 more instructions a tile and half the heads a pass.
//     The parts are columns of the same product that would be empty otherwise: NC = 2 columns per query head (4 for
//     fp32), 8 (4) heads at a time;
//   * the running maximum is raised only when a tile's is past it by 2^4, so the accumulators are rarely rescaled. p is
//     taken against a reference 2^4 above that maximum: never more than 1, as against the row's own largest, so the fp32 sums of
//     p v overflow only where those do (the format holds values to 1.5 * 2^127). Terms below 2^-122 of the largest are lost. The
//     reference shifts the exponents, and with 2^8 their fp32 rounding was coarser (fp32 outputs, 4 rows of 500 at D 256, off by
//     2.1e-7 of their norm against 1.5e-7; fp32 tensor operations 4.4e-7); with 2^2, 2^4 and 2^8 the times are the same.
// Rows are cut into splits of whole rounds (one tile per wave of the workgroup), planned on the device from the row
// lengths so that the splits of all rows fill the chip however ragged the batch is; the waves of a
// workgroup take a split's tiles in turn and are merged through LDS; the last workgroup of a row to finish
// folds its splits.
//
// Measured (H 16 / H_kv 8 / D 128 bf16, us per layer in a graph; an empty launch is 1.8 there): one row of 300 tokens 5.6, 8
// of 512 6.9, 32 of 128-2048 14.2, 32 of 8192 54 (285 MB: 5.3 TB/s; a large copy reaches 5.15), one of 100003 27.6. fp32:
// 5.8, 15.4 and 61 for the first, third and fourth; D 64 (H 16 / H_kv 16): 5.0 for one of 300, 60 for 32 of 8192. A 16-bit cache
// reads 3.8 times the bytes (32 of 8192: 162 us). Bound by memory in the long cases; in the short ones by dependent round
// trips (row lengths with the page ids beside them, then K and V; rows behind a split one load the page ids in between) and, per
// round of 8 tiles on a CU, 0.75 us of vector instructions (220 a tile and wave: 64 conversions, 32 exchanges, 8
// exponentials at a quarter of the rate). Tried and left: a workgroup for all KV heads at once, so that
// whole pages are swept (32 of 8192 53.3 against 51.0, more splits to fold elsewhere); 16 waves per workgroup
// (as 8 in long rows, 1 us slower in short ones); two register sets, loads two tiles ahead (half the waves, 8 of
// 512 8.0 against 6.8).
#include <type_traits>

#include "fp4.h"

namespace miattn {
namespace {

struct Fp4DecodeArgs {
  int B, H, H_kv, G, n_hchunks, bs_log2, max_blocks, target, cols, cols_log2;
  int64_t qs0, qs1, ks0, ks1, vs0, vs1, os0, os1, bts0;
  float scale_log2;
};

constexpr int kTile = 32;       // tokens per wave and step
constexpr float kRaise = 4.0f;  // log2 units a tile's maximum may be past the running one, and p's reference above that

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// columns per query head (parts of q and p), query heads per pass
template <typename T> constexpr int kCols = sizeof(T) == 4 ? 4 : 2;
template <typename T> constexpr int kHeads = 16 / kCols<T>;

__device__ __forceinline__ int clamp_len(int len, int capacity) {
  len = len < capacity ? len : capacity;
  return len > 0 ? len : 0;
}

__device__ __forceinline__ float hi_bf16(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// the high halves of two floats as a bf16 pair (cut, not rounded)
__device__ __forceinline__ uint32_t pack_hi(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// two floats rounded to the nearest bf16, as a pair
__device__ __forceinline__ uint32_t pack_near(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, bf16x2_t{(__bf16)lo, (__bf16)hi});
}
__device__ __forceinline__ bf16x8_t operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_bit_cast(bf16x8_t, make_uint4(a, b, c, d));
}
// max / sum over lanes i, i ^ 16, i ^ 32 and i ^ 48 (the four lane groups of a column)
template <typename Op>
__device__ __forceinline__ float over_groups(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = Op::op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return Op::op(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
// sum over the NC columns of a query head
template <int NC>
__device__ __forceinline__ float over_parts(float x) {
  x += dpp<kDppQuadXor1>(x);
  if constexpr (NC == 4) x += dpp<kDppQuadXor2>(x);
  return x;
}

// ceil(x / y) for quotients of at most a few hundred, exact: the product is off by less than one either way.
__device__ __forceinline__ int ceil_div(int x, int y) {
  const uint32_t v = uint32_t(x) + uint32_t(y) - 1u;
  const int n = int(float(v) * __builtin_amdgcn_rcpf(float(y)));
  const int r = int(v - uint32_t(n) * uint32_t(y));
  return n + (r < 0 ? -1 : r >= y ? 1 : 0);
}

struct Fp4Split {
  int b, split, n_split, first, len, begin, end;
};
// This workgroup's (row, split) and its tokens, derived by every wave from the row lengths, 64 rows at a time. Tokens
// per split: the share, total / target in whole rounds, or kLeast if that is more; as long as the splits of the first 64 rows
// (one per row at least, an empty row's writes its zeros) are more than target the share grows, up to kFitSteps times. A
// row's tokens are then shared out evenly over its splits, again in whole rounds.
// A merge of splits costs about 2 us (a partial's way to memory, the count's there and back, the partials' way back) and more
// with their number, a round of tiles 0.75 (D 256: about 2) where others hide its loads, up to 2 where nothing does. So
// no split is shorter than kLeast, or half of it in rows of up to kShortRow, and rows of up to kWhole tokens stay whole,
// kWholeAlone where the share says that the chip is far from full. Measured, us per layer, H 16 / H_kv 8 / D 128: 4 rows of
// 600 whole 6.9, cut at 256 8.3; one of 1000 whole 8.8, cut at 512 8.5, at 256 7.7; 4 of 1000 9.1 and 8.3 (256); 4 of 2048
// cut at 512 9.4, at 256 9.7; one of 8000 at 512 10.2, at 768 10.7. D 256, 8 / 2 heads: one of 500 whole 9.6, cut at 128
// 7.6; 16 rows of 128-2048 cut at 256 10.0, at 128 10.9, at 128 only up to 1024 tokens 10.0. D 64, 16 / 16 heads, takes D 128's
// figures: with D 256's instead one row of 600 is 7.2 for 6.3 and 4 of 600 7.6 for 6.6, the longer ones equal; at twice D 128's 16
// rows of 128-2048 are 16.7 for 12.9, 4 of 1000 8.0 for 8.3, one of 8000 11.1 for 11.7.
constexpr int kFitSteps = 8;
template <int D> constexpr int kLeast = D == 256 ? 256 : 512;
template <int D> constexpr int kWhole = D == 256 ? 512 : 1024;
template <int D> constexpr int kWholeAlone = D == 256 ? 256 : 768;
constexpr int kShortRow = 1024;
template <int kRound, int D>
__device__ __forceinline__ bool plan_split(const int32_t* __restrict__ seqlen, const Fp4DecodeArgs& a, int w,
                                           Fp4Split& si) {
  const int lane = __lane_id();
  const int capacity = a.max_blocks << a.bs_log2;
  const int len_first = lane < a.B ? clamp_len(seqlen[lane], capacity) : 0;
  int total = __builtin_amdgcn_readlane(wave_inclusive_scan(len_first), 63);
  for (int r0 = 64; r0 < a.B; r0 += 64) {
    const int row = r0 + lane;
    total += __builtin_amdgcn_readlane(wave_inclusive_scan(row < a.B ? clamp_len(seqlen[row], capacity) : 0), 63);
  }
  // total / target rounded up to whole rounds: the share of one split
  int share = (int((uint32_t(total) + uint32_t(a.target) * kRound - 1u) / (uint32_t(a.target) * kRound))) * kRound;
  auto count = [&](int len, int row) {
    const int chunk = len > kShortRow ? max(share, kLeast<D>) : max(share, kLeast<D> / 2);
    const int n = ceil_div(len, chunk);
    return row < a.B ? (len > (share > kLeast<D> / 2 ? kWhole<D> : kWholeAlone<D>) ? n : 1) : 0;
  };
  int n = count(len_first, lane), incl = wave_inclusive_scan(n);
  if (2 * a.B <= a.target) {
    const int step = (share / 16 + kRound) / kRound * kRound;
#pragma unroll 1
    for (int i = 0; i < kFitSteps && __builtin_amdgcn_readlane(incl, 63) > a.target; ++i) {
      share += step;
      n = count(len_first, lane);
      incl = wave_inclusive_scan(n);
    }
  }
  int len = len_first, base = 0;
  for (int r0 = 0;;) {
    const uint64_t owner = __ballot(w >= base + incl - n && w < base + incl);
    if (owner != 0) {
      const int o = __ffsll(static_cast<unsigned long long>(owner)) - 1;
      const int excl = __builtin_amdgcn_readlane(incl - n, o);
      const int of_row = __builtin_amdgcn_readlane(n, o);
      si.len = __builtin_amdgcn_readlane(len, o);
      const int each = ((si.len + of_row - 1) / of_row + kRound - 1) & -kRound;
      si.b = r0 + o;
      si.split = w - base - excl;
      si.first = base + excl;
      si.n_split = si.len > 0 ? (si.len + each - 1) / each : 1;
      si.begin = si.split * each;
      si.end = min(si.len, si.begin + each);
      return si.split < si.n_split;  // rounding up may leave the last split nothing
    }
    r0 += 64;
    if (r0 >= a.B) return false;
    base += __builtin_amdgcn_readlane(incl, 63);
    const int row = r0 + lane;
    len = row < a.B ? clamp_len(seqlen[row], capacity) : 0;
    n = count(len, row);
    incl = wave_inclusive_scan(n);
  }
}

// One split's partial of one column: sums of nh heads, then (reference, l) of each; whole 16 bytes.
__host__ __device__ constexpr int partial_floats(int nh, int D) { return nh * D + (2 * nh + 3) / 4 * 4; }

// Device-scope 16- and 8-byte accesses of the partials: written through to, and read from, the level that all XCDs share,
// so no cache has to be written back or dropped for them.
constexpr int kSc1 = 16;
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ auto partial_rsrc(float* p, int64_t floats) {
  return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, int(floats * 4), 0x00020000);
}

template <typename T, int D, int kW>
__global__ __launch_bounds__(64 * kW, 2) void paged_decode_fp4_kernel(
    const T* __restrict__ q, const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
    const int32_t* __restrict__ block_table, const int32_t* __restrict__ seqlen, T* __restrict__ out,
    unsigned* __restrict__ counters, float* __restrict__ partials, Fp4DecodeArgs a) {
  constexpr int kRound = kW * kTile;
  constexpr int KW = D / 32;                // code dwords of K per lane and 16 tokens
  constexpr int KS = D == 256 ? 2 : 1;      // scales of those
  constexpr int VE = D / 16;                // V elements per lane and token
  constexpr int VW = VE >= 8 ? VE / 8 : 1;  // dwords they take (D 64: half of one)
  constexpr int NC = kCols<T>, HB = kHeads<T>;
  extern __shared__ __align__(16) float smem[];  // per wave: (reference, l) of HB heads, then nh x D sums

  Fp4Split si;
  // Columns (KV head and chunk of its query heads) are the fast index, so the workgroups that have a split come first and
  // are dealt out evenly over the CUs; those without one come last.
  const int slot = a.cols_log2 >= 0 ? int(blockIdx.x) >> a.cols_log2 : int(blockIdx.x / unsigned(a.cols));
  const int column = int(blockIdx.x) - slot * a.cols;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The pages of this wave's first two tiles if no row before this one is split, loaded beside the row lengths: one memory
  // round trip less for such batches, the short ones. Entries inside the table, used only if the plan says so.
  int page0, pg[2], pn[2];
  {
    const int32_t* row = block_table + int64_t(min(slot, a.B - 1)) * a.bts0;
    page0 = row[0];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      pg[u] = row[min((wave * kTile + 16 * u) >> a.bs_log2, a.max_blocks - 1)];
      pn[u] = row[min((wave * kTile + kRound + 16 * u) >> a.bs_log2, a.max_blocks - 1)];
    }
  }
  if (!plan_split<kRound, D>(seqlen, a, slot, si)) return;  // uniform
  const int b = si.b;
  const int t_begin = si.begin, t_end = si.end;
  const int kvh = a.n_hchunks == 1 ? column : column / a.n_hchunks;
  const int hch = column - kvh * a.n_hchunks;
  const int nh = min(HB, a.G - hch * HB);  // query heads of this workgroup
  const int h0 = kvh * a.G + hch * HB;
  const int lane = threadIdx.x & 63;
  const int col = lane & 15, lg = lane >> 4;  // of the products: row or column, and depth group
  const int part = col % NC;
  const int bs = 1 << a.bs_log2;

  if (si.len == 0) {  // uniform: the row has no tokens, and its table may name no page
    for (int i = threadIdx.x; i < nh * D; i += 64 * kW) out[b * a.os0 + (h0 + i / D) * a.os1 + i % D] = from_f32<T>(0.0f);
    return;
  }

  // Q as the depth x column operand: column `col`, elements lg D / 4 + 8 kk + j of depth step kk. Each wave loads
  // some of the KW steps here, and converts them into LDS once its first K and V loads are out.
  constexpr int QW = (KW + kW - 1) / kW;      // steps per wave
  constexpr int QN = sizeof(T) == 4 ? 2 : 1;  // 16-byte loads per 8 elements
  const bool there = col / NC < nh;
  uint4 q_raw[QW][QN];
#pragma unroll
  for (int i = 0; i < QW; ++i) {
    const int kk = min(wave + i * kW, KW - 1);
    const T* src = q + b * a.qs0 + (h0 + (there ? col / NC : 0)) * a.qs1 + lg * (D / 4) + 8 * kk;
#pragma unroll
    for (int n = 0; n < QN; ++n) q_raw[i][n] = load16(src + 4 * n);
  }

  const int32_t* bt_row = block_table + b * a.bts0;
  const int k_lane = col * (D / 2) + lg * (D / 8);
  const int ks_lane = bs * (D / 2) + (lg * (D / 4) / kFp4Group) * bs + col;
  const int v_lane = lg * 4 * (D / 2) + col * (D / 32);
  const int vs_lane = bs * (D / 2) + (col * VE / kFp4Group) * bs + lg * 4;

  // First token of 16-token half u of the tile at t0; a half past the end repeats the first (masked out), a
  // tile past the end the split's first.
  auto half_at = [&](int t0, int u) {
    t0 = t0 < t_end ? t0 : t_begin;
    return t0 + 16 * u < t_end ? t0 + 16 * u : t0;
  };
  auto load_pages = [&](int t0, int (&pg)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) pg[u] = bt_row[half_at(t0, u) >> a.bs_log2];
  };
  uint32_t tk[2][KW], tks[2][KS], tv[2][4][VW], tvs[2];  // one tile: codes and scales of K, of V
  auto issue_k = [&](int t0, const int (&pg)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int at = half_at(t0, u) & (bs - 1);
      const uint8_t* kp = kc + (int64_t(pg[u]) * a.ks0 + kvh * a.ks1);
      const uint8_t* kr = kp + (at * (D / 2) + k_lane);
#pragma unroll
      for (int i = 0; i < KW; i += 4) {
        if constexpr (KW >= 4) {
          const uint4 w = load16_nt(kr + 4 * i);
          tk[u][i] = w.x; tk[u][i + 1] = w.y; tk[u][i + 2] = w.z; tk[u][i + 3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(kr);
          tk[u][0] = w.x; tk[u][1] = w.y;
        }
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) tks[u][i] = kp[at + ks_lane + i * bs];
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto issue_v = [&](int t0, const int (&pg)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int at = half_at(t0, u) & (bs - 1);
      const uint8_t* vp = vc + (int64_t(pg[u]) * a.vs0 + kvh * a.vs1);
      const uint8_t* vr = vp + (at * (D / 2) + v_lane);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (VE == 4) {
          tv[u][j][0] = *reinterpret_cast<const uint16_t*>(vr + j * (D / 2));
        } else if constexpr (VE == 8) {
          tv[u][j][0] = *reinterpret_cast<const uint32_t*>(vr + j * (D / 2));
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(vr + j * (D / 2));
          tv[u][j][0] = w.x; tv[u][j][1] = w.y;
        }
      }
      tvs[u] = *reinterpret_cast<const uint32_t*>(vp + at + vs_lane);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  int t0 = t_begin + wave * kTile;
  if (si.b != slot || t_begin != 0) {
    load_pages(t0, pg);
    load_pages(t0 + kRound, pn);
  } else {  // as load_pages gives them
    auto settle = [&](int t, int (&x)[2]) {
      x[0] = t < t_end ? x[0] : page0;
      x[1] = t + 16 < t_end ? x[1] : x[0];
    };
    settle(t0, pg);
    settle(t0 + kRound, pn);
  }
  issue_k(t0, pg);
  issue_v(t0, pg);
  // A negative scale is moved into q, so that the largest score is the largest product.
  const float flip = a.scale_log2 < 0.0f ? -1.0f : 1.0f;
  const float c2 = a.scale_log2 * flip;
  uint4* sm_q = reinterpret_cast<uint4*>(smem + kW * (HB * 2 + min(HB, a.G) * (D + 16)));  // [KW][64 lanes]
#pragma unroll
  for (int i = 0; i < QW; ++i) {
    const int kk = wave + i * kW;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = Vec16<T>::get(q_raw[i][j / Vec16<T>::N], j % Vec16<T>::N);
      x[j] = there ? x[j] * flip : 0.0f;
      if constexpr (!std::is_same<T, bf16_t>::value) {
        // part i holds the bits left by the parts before it; past the last part nothing is left
        for (int n = 0; n < NC - 1; ++n) x[j] = n < part ? x[j] - hi_bf16(x[j]) : x[j];
        if (NC == 4 && part == 3) x[j] = 0.0f;
      }
    }
    if (kk < KW) {
      sm_q[kk * 64 + lane] =
          make_uint4(pack_hi(x[0], x[1]), pack_hi(x[2], x[3]), pack_hi(x[4], x[5]), pack_hi(x[6], x[7]));
    }
  }
  // a barrier that does not wait for the loads on their way
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");

  f32x4_t o[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) o[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, mc = 0.0f, l = 0.0f;  // the running maximum (of q . k), p's reference in log2 units, the sum of p
  const float raise = fminf(kRaise / c2, 3.0e38f);
  // of p, what the parts before this column's hold: by pairs with two parts, by value with three
  const uint32_t cut1 = part >= 1 ? (NC == 4 ? 0xffff0000u : 0xffffffffu) : 0u, cut2 = part >= 2 ? 0xffff0000u : 0u;

  // One tile: the scores from K, the running maximum, the sums from V; `next` issues the loads that come into K's, then
  // into V's registers.
  auto compute = [&](int t0, auto masked, auto&& next_k, auto&& next_v) {
    constexpr bool kMasked = decltype(masked)::value;
    __builtin_amdgcn_sched_barrier(0);
    uint4 qf[KW];
#pragma unroll
    for (int kk = 0; kk < KW; ++kk) qf[kk] = sm_q[kk * 64 + lane];
    f32x4_t s[2];
    uint4 kf[2][KW];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int kk = 0; kk < KW; ++kk) {
        const float sc = fp4_scale(tks[u][kk * 8 * KS / (D / 4)]);
        const uint32_t w = tk[u][kk];
        kf[u][kk] = make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0)),
                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1)),
                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2)),
                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3)));
      }
    }
    next_k();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kk = 0; kk < KW; ++kk) {
        s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kf[u][kk]),
                                                       __builtin_bit_cast(bf16x8_t, qf[kk]), s[u], 0, 0, 0);
      }
    }
    // this lane's 8 tokens: t0 + 16 u + 4 lg + i
    float most = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (!std::is_same<T, bf16_t>::value) s[u][i] = over_parts<NC>(s[u][i]);
        if constexpr (kMasked) {
          if (t0 + 16 * u + 4 * lg + i >= t_end) s[u][i] = -INFINITY;
        }
        most = fmaxf(most, s[u][i]);
      }
    }
    most = over_groups<MaxOp>(most);
    if (__any(!(most - m <= raise))) {  // also the first tile
      const float up = fmaxf(m, most);
      const float ref = up == -INFINITY ? 0.0f : fmaf(up, c2, kRaise);
      const float alpha = m == -INFINITY ? 0.0f : fast_exp2(mc - ref);
      m = up;
      mc = ref;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < VE; ++i) o[i] *= alpha;
    }
    float p[8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = fast_exp2(fmaf(s[u][i], c2, -mc));
        if constexpr (kMasked) x = t0 + 16 * u + 4 * lg + i < t_end ? x : 0.0f;
        l += x;
        if constexpr (NC == 4) {
          x -= __uint_as_float(__float_as_uint(x) & cut1);
          x -= __uint_as_float(__float_as_uint(x) & cut2);
          if (part == 3) x = 0.0f;
        }
        p[4 * u + i] = x;
      }
    }
    uint32_t pw[4];  // this column's part of two p each
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (NC == 4) {
        pw[j] = pack_hi(p[2 * j], p[2 * j + 1]);
      } else {
        const uint32_t near = pack_near(p[2 * j], p[2 * j + 1]) & cut1;  // part 0 takes nothing away
        pw[j] = pack_near(p[2 * j] - __uint_as_float(near << 16), p[2 * j + 1] - __uint_as_float(near & 0xffff0000u));
      }
    }
    const bf16x8_t pf = operand(pw[0], pw[1], pw[2], pw[3]);
    if constexpr (kMasked) {
      // past the end: zero codes, and scales of 1 (garbage may be a NaN scale, which 0 * NaN would keep)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int n = t_end - (t0 + 16 * u + 4 * lg);  // tokens of this lane's four that are there
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int k = 0; k < VW; ++k) tv[u][i][k] = i < n ? tv[u][i][k] : 0u;
        }
        const uint32_t keep = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
        tvs[u] = (tvs[u] & keep) | (0x7f7f7f7fu & ~keep);
      }
    }
    // the scale of token i of a half is byte i of its dword, shifted under the exponent (the conversion
    // reads no other bit of it)
    float vsc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      vsc[j] = __uint_as_float((j & 3) == 3 ? tvs[j >> 2] >> 1 : tvs[j >> 2] << (23 - 8 * (j & 3)));
    }
    // One dword of codes at a time: all its elements converted, then, the codes' registers being free, the next tile's
    // loads, then the products.
    constexpr int kBytes = VE >= 8 ? 4 : 2;
#pragma unroll
    for (int k = 0; k < VW; ++k) {
      uint32_t x[4][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = tv[j >> 2][j & 3][k];
        x[0][j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vsc[j], 0));
        x[1][j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vsc[j], 1));
        if constexpr (kBytes == 4) {
          x[2][j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vsc[j], 2));
          x[3][j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, vsc[j], 3));
        }
      }
      if (k == VW - 1) next_v();
#pragma unroll
      for (int y = 0; y < kBytes; ++y) {
        uint32_t lo[4], hi[4];  // elements 2 y and 2 y + 1 of two tokens each
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = __builtin_amdgcn_perm(x[y][2 * j + 1], x[y][2 * j], 0x05040100u);
          hi[j] = __builtin_amdgcn_perm(x[y][2 * j + 1], x[y][2 * j], 0x07060302u);
        }
        const int e = 8 * k + 2 * y;
        o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(lo[0], lo[1], lo[2], lo[3]), pf, o[e], 0, 0, 0);
        o[e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(hi[0], hi[1], hi[2], hi[3]), pf, o[e + 1], 0, 0, 0);
      }
    }
  };

  // Loads stay one tile ahead of their use: the next tile's K is on its way from when this tile's scores are made, its
  // V from when the sums are, and its pages are known a tile earlier. Every load of the loop is unconditional.
  if (t0 < t_end) {
    auto none = [] {};
    for (; t0 + kRound < t_end; t0 += kRound) {  // a tile with another behind it is whole
      const int t1 = t0 + kRound;
      compute(t0, std::false_type{}, [&] { issue_k(t1, pn); pg[0] = pn[0]; pg[1] = pn[1]; load_pages(t1 + kRound, pn); },
              [&] { issue_v(t1, pg); });
    }
    compute(t0, std::true_type{}, none, none);
  }

  // ---- the waves' states through LDS (not q's part of it, which other waves may still read): (reference, l) per head, then the
  // sums, parts added up, four elements at a time. Piece x of a head is rows 4 lg + r of the products, elements
  // 4 n .. 4 n + 3 of each, x = (r VE / 4 + n) 4 + lg: the lane groups of a column and, heads being 16 words apart
  // modulo the banks, its heads write side by side.
  l = over_groups<SumOp>(l);
  constexpr int kHeadWords = D + 16;
  auto element_of = [](int x) { return (4 * (x & 3) + (x >> 2) / (VE / 4)) * VE + (x >> 2) % (VE / 4) * 4; };
  float* sm_ml = smem;                // [wave][HB][2]
  float* sm_o = smem + kW * HB * 2;   // [wave][nh][kHeadWords]
  const int g = col / NC;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
#pragma unroll
    for (int r = 0; r < 4; ++r) o[i][r] = over_parts<NC>(o[i][r]);
  }
  if (part == 0 && g < nh) {
    if (lg == 0) *reinterpret_cast<float2*>(sm_ml + (wave * HB + g) * 2) = make_float2(m == -INFINITY ? m : mc, l);
    float* dst = sm_o + (wave * nh + g) * kHeadWords + lg * 4;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int i = 0; i < VE; i += 4) {
        *reinterpret_cast<float4*>(dst + (r * (VE / 4) + i / 4) * 16) = make_float4(o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]);
      }
    }
  }
  __syncthreads();
  auto finish = [&](int gg, int x, const float4& acc, float L) {
    const float inv = 1.0f / L;
    const float y[4] = {fp4_saturate<T>(acc.x * inv), fp4_saturate<T>(acc.y * inv), fp4_saturate<T>(acc.z * inv),
                        fp4_saturate<T>(acc.w * inv)};
    T* row = out + b * a.os0 + (h0 + gg) * a.os1 + element_of(x);
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(row) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
      const uint32_t w0 = uint32_t(from_f32<T>(y[0]).bits) | uint32_t(from_f32<T>(y[1]).bits) << 16;
      const uint32_t w1 = uint32_t(from_f32<T>(y[2]).bits) | uint32_t(from_f32<T>(y[3]).bits) << 16;
      *reinterpret_cast<uint2*>(row) = make_uint2(w0, w1);
    }
  };
  const int part_floats = partial_floats(min(HB, a.G), D);
  const auto mine = partial_rsrc(partials + int64_t(blockIdx.x) * part_floats, part_floats);
  for (int i = threadIdx.x; i < nh * (D / 4); i += 64 * kW) {
    const int gg = i / (D / 4), x = i - gg * (D / 4);
    float2 ml[kW];
    float4 v[kW];
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      ml[w] = *reinterpret_cast<const float2*>(sm_ml + (w * HB + gg) * 2);
      v[w] = *reinterpret_cast<const float4*>(sm_o + (w * nh + gg) * kHeadWords + x * 4);
      M = fmaxf(M, ml[w].x);
    }
    float L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const float wt = ml[w].x == -INFINITY ? 0.0f : fast_exp2(ml[w].x - M);
      L = fmaf(ml[w].y, wt, L);
      acc.x = fmaf(v[w].x, wt, acc.x);
      acc.y = fmaf(v[w].y, wt, acc.y);
      acc.z = fmaf(v[w].z, wt, acc.z);
      acc.w = fmaf(v[w].w, wt, acc.w);
    }
    if (si.n_split == 1) {
      finish(gg, x, acc, L);
    } else {
      const u32x4_nt val = {__float_as_uint(acc.x), __float_as_uint(acc.y), __float_as_uint(acc.z), __float_as_uint(acc.w)};
      __builtin_amdgcn_raw_buffer_store_b128(val, mine, (gg * D + x * 4) * 4, 0, kSc1);
      if (x == 0) {
        const u32x2_t mine_ml = {__float_as_uint(M), __float_as_uint(L)};
        __builtin_amdgcn_raw_buffer_store_b64(mine_ml, mine, (nh * D + gg * 2) * 4, 0, kSc1);
      }
    }
  }
  if (si.n_split == 1) return;

  // ---- the last of the row's workgroups to get here folds their partials: each has its own at the shared level
  // before it counts itself, and the last one reads them from there
  int* sm_last = reinterpret_cast<int*>(smem);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    // It counts modulo n_split, so it is 0 again by itself: launches of the same row lengths that overlapped on one
    // workspace by mistake leave it at 0 too (counted up and then cleared, it stayed off for every later launch).
    const unsigned last = unsigned(si.n_split - 1);
    *sm_last = atomicInc(counters + int64_t(b) * a.cols + column, last) == last;
  }
  __syncthreads();
  if (!*sm_last) return;  // uniform
  __syncthreads();        // sm_last has been read by every wave; its words are used again below
  const auto row_parts = partial_rsrc(partials + (int64_t(si.first) * a.cols + column) * part_floats,
                                      (int64_t(si.n_split - 1) * a.cols + 1) * part_floats);
  // ng groups of threads take the splits in turn and are folded through LDS, in the groups' order
  const int lanes = nh * (D / 4);                       // threads that hold one split's sums, 4 each
  const int ng = max(1, 64 * kW / lanes);               // 64 kW threads, lanes a multiple of 16
  float* sm_f = smem;                                   // [group][lanes] sums, then [group][lanes] (reference, l)
  float* sm_g = smem + ng * lanes * 4;
  // splits loaded at once by a group: 2, 1 or 8 are within 2% of 4 either way, 1 up to 10% slower with many splits; with the
  // few groups of D 256 in 4 waves 8 are faster (one row of 8000 13.0 -> 12.1 us)
  constexpr int kFold = D == 256 && kW == 4 ? 8 : 4;
  for (int i0 = 0; i0 < lanes; i0 += 64 * kW) {  // more than one pass where a column has more sums than threads
    const int grp = ng > 1 ? threadIdx.x / lanes : 0;
    const int i = ng > 1 ? threadIdx.x - grp * lanes : i0 + threadIdx.x;
    const bool mine_too = grp < ng && i < lanes;
    const int gg = mine_too ? i / (D / 4) : 0, x0 = mine_too ? i - gg * (D / 4) : 0;
    float M = -INFINITY, L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = grp; s0 < si.n_split; s0 += kFold * ng) {
      u32x2_t ml[kFold];
      u32x4_nt x[kFold];
#pragma unroll
      for (int j = 0; j < kFold; ++j) {
        const int s = min(s0 + j * ng, si.n_split - 1);
        const int at = (s * a.cols * part_floats + gg * D + x0 * 4) * 4;
        const int at_ml = (s * a.cols * part_floats + nh * D + gg * 2) * 4;
        ml[j] = __builtin_amdgcn_raw_buffer_load_b64(row_parts, at_ml, 0, kSc1);
        x[j] = __builtin_amdgcn_raw_buffer_load_b128(row_parts, at, 0, kSc1);
      }
      float mj[kFold], top = M;
#pragma unroll
      for (int j = 0; j < kFold; ++j) {
        mj[j] = s0 + j * ng < si.n_split ? __uint_as_float(ml[j].x) : -INFINITY;
        top = fmaxf(top, mj[j]);
      }
      const float again = M == -INFINITY ? 0.0f : fast_exp2(M - top);
      M = top;
      L *= again;
      acc.x *= again; acc.y *= again; acc.z *= again; acc.w *= again;
#pragma unroll
      for (int j = 0; j < kFold; ++j) {
        if (s0 + j * ng < si.n_split) {
          const float wt = mj[j] == -INFINITY ? 0.0f : fast_exp2(mj[j] - top);
          L = fmaf(__uint_as_float(ml[j].y), wt, L);
          acc.x = fmaf(__uint_as_float(x[j].x), wt, acc.x);
          acc.y = fmaf(__uint_as_float(x[j].y), wt, acc.y);
          acc.z = fmaf(__uint_as_float(x[j].z), wt, acc.z);
          acc.w = fmaf(__uint_as_float(x[j].w), wt, acc.w);
        }
      }
    }
    if (ng > 1) {
      if (mine_too) {
        *reinterpret_cast<float4*>(sm_f + (grp * lanes + i) * 4) = acc;
        *reinterpret_cast<float2*>(sm_g + (grp * lanes + i) * 2) = make_float2(M, L);
      }
      __syncthreads();
      if (grp > 0) return;
      for (int w = 1; w < min(ng, si.n_split); ++w) {
        const float4 x = *reinterpret_cast<const float4*>(sm_f + (w * lanes + i) * 4);
        const float2 ml = *reinterpret_cast<const float2*>(sm_g + (w * lanes + i) * 2);
        const float top = fmaxf(M, ml.x);
        const float w0 = M == -INFINITY ? 0.0f : fast_exp2(M - top), w1 = ml.x == -INFINITY ? 0.0f : fast_exp2(ml.x - top);
        M = top;
        L = L * w0 + ml.y * w1;
        acc.x = acc.x * w0 + x.x * w1;
        acc.y = acc.y * w0 + x.y * w1;
        acc.z = acc.z * w0 + x.z * w1;
        acc.w = acc.w * w0 + x.w * w1;
      }
    }
    if (mine_too) finish(gg, x0, acc, L);
  }
}

int esize_of(int dtype) { return dtype == MI_F32 ? 4 : dtype == MI_F16 || dtype == MI_BF16 ? 2 : 0; }

bool fp4_dim(int D) { return D == 64 || D == 128 || D == 256; }

bool fp4_block(int bs) { return bs >= 16 && (bs & (bs - 1)) == 0; }

// The kernel's offsets inside a page of one KV head are 32 bits.
bool fp4_page_fits(int bs, int D) { return fp4_page_bytes(bs, D) <= 0x7fffffff; }

struct Fp4Plan {
  int n_hchunks, cols, waves, target, slots, nh;
  size_t counter_bytes, partial_bytes;
  size_t bytes() const { return counter_bytes + partial_bytes; }
};

Fp4Plan make_plan(int B, int H, int H_kv, int D, int dtype) {
  Fp4Plan p;
  const int heads = dtype == MI_F32 ? kHeads<float> : kHeads<bf16_t>;
  p.n_hchunks = (H / H_kv + heads - 1) / heads;
  p.cols = H_kv * p.n_hchunks;
  p.nh = H / H_kv < heads ? H / H_kv : heads;
  // One workgroup of 8 waves per CU, or two of 4: the latter where the rows times columns are more than half the
  // CUs and at most all of them, too few splits per row for 256 workgroups to be dealt out evenly. The host knows the number of
  // rows but not their lengths, so this gives some of the even batches' time for more of the ragged ones'. us per layer
  // with 8 and 4 waves, D 128, 32 rows (256 in all): ragged 128-2048 16.8 and 14.6, 4000-8000 56.5 and 47.3; all of 500 8.1 and
  // 8.5, of 2000 16.9 and 18.8, of 8192 52.2 and 54.4. 17 rows (136): ragged 13.2 and 12.8, of 500 7.4 and 8.1, of 8192 44.6
  // and 37.3. D 64, 16 rows (256): ragged 13.5 and 12.9, of 500 6.5 and 7.0, of 8192 40.2 and 41.8. D 256, 100 rows (200): ragged
  // 29.3 and 21.8, of 4000 58.6 and 55.9. Outside: 16 rows (128) of 4000-8000 28.9 and 27.8, 8 of 512 (64) 7.4 and 7.9, 64 ragged
  // ones (512) 22.6 and 23.4, one of 8000 equal.
  // At D 256 a round of 8 waves is two tiles per SIMD, so up to 32 rows times columns, which leave CUs idle, take 4 as well:
  // 16 rows of 2 columns (32), ragged 11.3 and 10.2, of 512 10.5 and 8.9, but of 4000 14.6 and 17.1; 8 of 512 (16) 10.2 and 8.7,
  // one of 500 9.9 and 7.9; 32 ragged ones (64) 13.2 and 13.5.
  const int64_t items = int64_t(B) * p.cols;
  p.waves = (D == 256 && items <= 32) || (items > 128 && items <= 256) ? 4 : 8;
  const int groups = p.waves == 8 ? 256 : 512;
  p.target = groups / p.cols > 1 ? groups / p.cols : 1;
  p.slots = p.target + B;
  p.counter_bytes = (size_t(B) * p.cols * sizeof(unsigned) + 255) / 256 * 256;
  p.partial_bytes = size_t(p.slots) * p.cols * partial_floats(p.nh, D) * sizeof(float);
  return p;
}

template <typename T, int D>
int launch_d(const void* q, const void* k, const void* v, const int32_t* bt, const int32_t* seqlen, void* out,
             void* workspace, const Fp4DecodeArgs& a, const Fp4Plan& p, hipStream_t s) {
  unsigned* counters = static_cast<unsigned*>(workspace);
  float* partials = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.counter_bytes);
  auto go = [&](auto waves) {
    constexpr int kW = decltype(waves)::value;
    // the waves' states; the fold of the splits needs 6 floats per thread at most
    const size_t states = size_t(kW) * (kHeads<T> * 2 + p.nh * (D + 16)), fold = size_t(64 * kW) * 6;
    const size_t lds = (states + D * 8 > fold ? states + D * 8 : fold) * sizeof(float);  // 32 D bytes of q
    hipLaunchKernelGGL((paged_decode_fp4_kernel<T, D, kW>), dim3(unsigned(p.slots) * unsigned(p.cols)), dim3(64 * kW), lds, s,
                       static_cast<const T*>(q), static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), bt, seqlen,
                       static_cast<T*>(out), counters, partials, a);
  };
  if (p.waves == 8) go(std::integral_constant<int, 8>{}); else go(std::integral_constant<int, 4>{});
  return launch_status("mi_paged_decode_fp4");
}

template <typename T>
int launch_t(int D, const void* q, const void* k, const void* v, const int32_t* bt, const int32_t* seqlen, void* out,
             void* workspace, const Fp4DecodeArgs& a, const Fp4Plan& p, hipStream_t s) {
  switch (D) {
    case 64: return launch_d<T, 64>(q, k, v, bt, seqlen, out, workspace, a, p, s);
    case 128: return launch_d<T, 128>(q, k, v, bt, seqlen, out, workspace, a, p, s);
    default: return launch_d<T, 256>(q, k, v, bt, seqlen, out, workspace, a, p, s);
  }
}

}  // namespace
}  // namespace miattn

extern "C" size_t mi_paged_decode_fp4_workspace_size(int B, int H, int H_kv, int D, int block_size, int max_blocks,
                                                     int dtype) {
  using namespace miattn;
  if (B < 1 || H < 1 || H_kv < 1 || H % H_kv != 0 || !fp4_dim(D) || !fp4_block(block_size) ||
      !fp4_page_fits(block_size, D) || max_blocks < 1 || esize_of(dtype) == 0) {
    return 0;
  }
  return make_plan(B, H, H_kv, D, dtype).bytes();
}

extern "C" int mi_paged_decode_fp4(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                   const int32_t* seqlen, void* out, int B, int H, int H_kv, int D, int block_size,
                                   int max_blocks, const int64_t* strides, float scale, int dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  using namespace miattn;
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
  if (!fp4_page_fits(block_size, D)) {
    return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_fp4: a page of one KV head must stay below 2^31 bytes, got block_size %d",
                block_size);
  }
  if (max_blocks < 1) return fail(MI_ERR_INVALID, "mi_paged_decode_fp4: max_blocks must be >= 1");
  if (strides == nullptr) return fail(MI_ERR_INVALID, "mi_paged_decode_fp4: strides is NULL");
  if (B == 0) return MI_OK;
  if (q == nullptr || k_cache == nullptr || v_cache == nullptr || block_table == nullptr || seqlen == nullptr ||
      out == nullptr) {
    return fail(MI_ERR_INVALID, "mi_paged_decode_fp4: NULL tensor pointer");
  }
  // token counts and their rounding up to whole rounds stay in 32 bits
  const int64_t row_tokens = int64_t(max_blocks) * block_size;  // below 2^57
  if (row_tokens > (1LL << 30) || row_tokens * B > (1LL << 30)) {
    return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_fp4: B * max_blocks * block_size must stay within 2^30 tokens");
  }
  const Fp4Plan p = make_plan(B, H, H_kv, D, dtype);
  if (int64_t(p.slots) * p.cols > 0x7fffffff / (64 * 8)) {  // threads of the grid in 32 bits
    return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_fp4: grid too large (B=%d, H=%d)", B, H);
  }
  const int64_t* st = strides;
  const int es = esize_of(dtype);
  bool ok = true;
  for (const void* p : {q, k_cache, v_cache, static_cast<const void*>(out)}) ok = ok && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  // the stride of a dimension of one is never used
  for (int i : {0, 6}) ok = ok && (B == 1 || (st[i] * es) % 16 == 0);
  for (int i : {1, 7}) ok = ok && (H == 1 || (st[i] * es) % 16 == 0);
  for (int i : {2, 4}) ok = ok && st[i] % 16 == 0;
  for (int i : {3, 5}) ok = ok && (H_kv == 1 || st[i] % 16 == 0);
  if (!ok) {
    return fail(MI_ERR_UNSUPPORTED, "mi_paged_decode_fp4: q, out, k_cache and v_cache need 16-byte aligned rows and heads");
  }
  if (workspace == nullptr || workspace_bytes < p.bytes()) {
    return fail(MI_ERR_WORKSPACE, "mi_paged_decode_fp4: workspace of %zu bytes < %zu needed", workspace_bytes, p.bytes());
  }
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
    return fail(MI_ERR_WORKSPACE, "mi_paged_decode_fp4: workspace must be 16-byte aligned");
  }
  Fp4DecodeArgs a;
  a.n_hchunks = p.n_hchunks; a.target = p.target; a.cols = p.cols;
  a.cols_log2 = (p.cols & (p.cols - 1)) == 0 ? __builtin_ctz(unsigned(p.cols)) : -1;
  a.B = B; a.H = H; a.H_kv = H_kv; a.G = H / H_kv; a.max_blocks = max_blocks;
  a.bs_log2 = __builtin_ctz(unsigned(block_size));
  a.qs0 = st[0]; a.qs1 = st[1]; a.ks0 = st[2]; a.ks1 = st[3]; a.vs0 = st[4]; a.vs1 = st[5];
  a.os0 = st[6]; a.os1 = st[7]; a.bts0 = st[8];
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MI_BF16: return launch_t<bf16_t>(D, q, k_cache, v_cache, block_table, seqlen, out, workspace, a, p, s);
    case MI_F16: return launch_t<f16_t>(D, q, k_cache, v_cache, block_table, seqlen, out, workspace, a, p, s);
    default: return launch_t<float>(D, q, k_cache, v_cache, block_table, seqlen, out, workspace, a, p, s);
  }
}
