// Rows into and out of the 4-bit paged cache (the format is in fp4.h): the slot write, the slot
// read, and the attention epilogue (q/k norm + RoPE + K/V write) in one launch.
//
// All three move memory: a row of D elements is D * esize bytes on the one side and 17 D / 32 on the other.
// A lane holds 8 consecutive elements (one code dword), a group of 32 is an aligned quad of
// lanes, a row D / 8 lanes, so a group's largest value is two DPP moves away and there is no
// LDS. A lane takes its elements as 16-byte loads where the source allows it.
#include <initializer_list>
#include <type_traits>

#include "fp4.h"

namespace miattn {
namespace {

struct Fp4Pool {
  uint8_t* k;  // n_blocks pages of H_kv heads each
  uint8_t* v;
  int64_t n_slots, head_bytes, block_bytes;
  int bs_log2;
};

// Where a lane's code dword and its group's scale byte of one row live.
struct Fp4Place {
  int64_t code, scale;
};
template <int D>
__device__ __forceinline__ Fp4Place fp4_place(const Fp4Pool& p, int64_t slot, int head, int c) {
  const int64_t page = (slot >> p.bs_log2) * p.block_bytes + head * p.head_bytes;
  const int at = int(slot & ((int64_t(1) << p.bs_log2) - 1));
  return {page + int64_t(at) * (D / 2) + c * 4,
          page + ((int64_t(D / 2)) << p.bs_log2) + (int64_t(c >> 2) << p.bs_log2) + at};
}

// Eight elements as they are loaded: 16-bit types stay packed.
template <typename T, bool kVec>
struct Raw8 {
  float x[8];
  __device__ __forceinline__ void load(const T* p, int64_t stride) { load8<T, kVec, true>(p, stride, x); }
  __device__ __forceinline__ int byte() const { return fp4_scale_byte(fp4_group_max(x)); }
  __device__ __forceinline__ uint32_t code(int b) const { return fp4_encode(x, b); }
};
template <typename T>
struct Packed8 {
  uint4 w;
  __device__ __forceinline__ void load(const T* p, int64_t) { w = load16_nt(p); }
  __device__ __forceinline__ int byte() const { return fp4_scale_byte(fp4_group_max16<T>(w)); }
  __device__ __forceinline__ uint32_t code(int b) const { return fp4_encode16<T>(w, b); }
};

template <typename T, bool kVec>
using Loaded8 = std::conditional_t<kVec && sizeof(T) == 2, Packed8<T>, Raw8<T, kVec>>;

template <typename R>
__device__ __forceinline__ void fp4_put_raw(uint8_t* pool, const Fp4Place& at, int c, const R& x) {
  const int byte = x.byte();
  *reinterpret_cast<uint32_t*>(pool + at.code) = x.code(byte);
  if ((c & 3) == 0) pool[at.scale] = uint8_t(byte);
}

template <int D>
__device__ __forceinline__ void fp4_put(uint8_t* pool, const Fp4Place& at, int c, const float (&x)[8]) {
  const int byte = fp4_scale_byte(fp4_group_max(x));
  *reinterpret_cast<uint32_t*>(pool + at.code) = fp4_encode(x, byte);
  if ((c & 3) == 0) pool[at.scale] = uint8_t(byte);
}

// 1 / sqrt(x), rounded once for a normal x: the instruction's result (within an ulp) and one Newton step on its exact residual
// 1 - x r^2.
__device__ __forceinline__ float exact_rsqrt(float x) {
  const float r = __builtin_amdgcn_rsqf(x);
  const float h = x * r;
  const float e = fmaf(-fmaf(x, r, -h), r, fmaf(-h, r, 1.0f));
  const float y = fmaf(0.5f * r, e, r);
  return x >= 0x1p-100f && x <= 0x1p100f ? y : r;  // the others: zero, infinity, NaN, or a residual out of range
}

__device__ __forceinline__ void report(int32_t* err, int64_t row) {
  if (err != nullptr) atomicCAS(err, 0, int32_t(row + 1));
}

// Eight elements of K and of V per lane and row. Work is ordered (group of tokens, head, token, lane) with as many tokens
// per group as rows fit kRows rounds of a wave: a wave writes consecutive tokens of one head, which are consecutive in
// the page when the slots are. kRows: rows per lane, all their loads issued before the first is used.
template <typename T, int D, typename IdxT, bool kVec, int kRows>
__global__ __launch_bounds__(256) void fp4_write_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                        const IdxT* __restrict__ slots, Fp4Pool pool, int64_t n_tokens,
                                                        int H_kv, int64_t ks0, int64_t ks1, int64_t ks2, int64_t vs0,
                                                        int64_t vs1, int64_t vs2, int32_t* err) {
  constexpr int LPR = D / 8, TPW = 64 / LPR;
  const int lane = threadIdx.x & 63, c = lane % LPR;
  const uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 6);  // this wave's (group, head), the same for its lanes
  const uint32_t grp = i / uint32_t(H_kv);
  const int head = int(i - grp * uint32_t(H_kv));
  const int64_t first = int64_t(grp) * (TPW * kRows) + lane / LPR;
  if (first >= n_tokens) return;  // whole quads leave together
  Loaded8<T, kVec> x[kRows], y[kRows];
  int64_t slot[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t token = first + r * TPW < n_tokens ? first + r * TPW : first;  // past the end: not stored
    x[r].load(k + token * ks0 + head * ks1 + c * 8 * ks2, ks2);
    y[r].load(v + token * vs0 + head * vs1 + c * 8 * vs2, vs2);
    slot[r] = int64_t(slots[token]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t token = first + r * TPW;
    if (token >= n_tokens) return;
    if (slot[r] < 0 || slot[r] >= pool.n_slots) {
      report(err, token);
      continue;
    }
    const Fp4Place at = fp4_place<D>(pool, slot[r], head, c);
    fp4_put_raw(pool.k, at, c, x[r]);
    fp4_put_raw(pool.v, at, c, y[r]);
  }
}

// The way back, in the same order. The rows go past the caches (a group of 4311 tokens at H_kv 8 / D 128, with the write
// before it: 15.2 -> 14.2 us).
template <typename T, int D, typename IdxT, int kRows>
__global__ __launch_bounds__(256) void fp4_read_kernel(Fp4Pool pool, const IdxT* __restrict__ slots,
                                                       T* __restrict__ k, T* __restrict__ v, int64_t n_tokens, int H_kv,
                                                       int32_t* err) {
  constexpr int LPR = D / 8, TPW = 64 / LPR;
  const int lane = threadIdx.x & 63, c = lane % LPR;
  const uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t grp = i / uint32_t(H_kv);
  const int head = int(i - grp * uint32_t(H_kv));
  const int64_t first = int64_t(grp) * (TPW * kRows) + lane / LPR;
  if (first >= n_tokens) return;
  int64_t slot[kRows];
  bool in[kRows];
  uint32_t wk[kRows] = {}, wv[kRows] = {}, sk[kRows] = {}, sv[kRows] = {};
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t token = first + r * TPW < n_tokens ? first + r * TPW : first;
    slot[r] = int64_t(slots[token]);
    in[r] = slot[r] >= 0 && slot[r] < pool.n_slots;
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (in[r]) {
      const Fp4Place at = fp4_place<D>(pool, slot[r], head, c);
      wk[r] = *reinterpret_cast<const uint32_t*>(pool.k + at.code);
      wv[r] = *reinterpret_cast<const uint32_t*>(pool.v + at.code);
      sk[r] = pool.k[at.scale];
      sv[r] = pool.v[at.scale];
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t token = first + r * TPW;
    if (token >= n_tokens) return;
    if (!in[r]) report(err, token);  // its rows come back as zeros: codes and scale of zero
    float x[8], y[8];
    fp4_decode(wk[r], fp4_scale(sk[r]), x);
    fp4_decode(wv[r], fp4_scale(sv[r]), y);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = fp4_saturate<T>(x[j]);
      y[j] = fp4_saturate<T>(y[j]);
    }
    const int64_t dst = (token * H_kv + head) * D + c * 8;
    store8<T, true>(k + dst, x);
    store8<T, true>(v + dst, y);
  }
}

struct EpilogueArgs {
  const void* qkv; int64_t row_stride; int parts; int64_t plane; const void* q_w; const void* k_w; const void* cos_tab;
  const void* sin_tab; int64_t n_pos; int rotary; const int64_t* pos; const void* slots; void* q_out; void* k_out;
  void* v_out; int B; int H; int H_kv; float eps; int zero_centred; int32_t* err;
};

// The attention epilogue. For each row (token): q and k heads are normalised, y = x / sqrt(mean(x^2) +
// eps) * w (or * (1 + w)), rotated, (a, b) -> (a cos - b sin, a sin + b cos) over the halves of the
// first `rotary` elements, and rounded to T once: everything up to there is fp32, so a value carries one
// rounding where the op-by-op chain of the 16-bit pool's epilogue carries seven. k is stored in 4 bits from
// the rounded T values, so the pool holds what fp4_write_kernel of k_out would have stored. A
// projection given as split-K partial sums is summed in split order and rounded to T first, the value
// that the projection's own output would hold. mean(x^2) is a lane's 8 squares, then a
// butterfly over the head's lanes; the rotation partner of a lane's elements is a lane too (c ^ rotary / 16).
template <typename T, int D, typename IdxT, bool kVec, bool kParts>
__global__ __launch_bounds__(256) void fp4_epilogue_kernel(EpilogueArgs a, Fp4Pool pool) {
  constexpr int LPR = D / 8, HPW = 256 / LPR;  // lanes per head, heads per workgroup pass
  const int c = threadIdx.x % LPR;
  const int64_t b = blockIdx.x;
  const int n_heads = a.H + 2 * a.H_kv;
  const int step = HPW * gridDim.y;
  const int head0 = blockIdx.y * HPW + threadIdx.x / LPR;
  const int64_t pb = a.pos[b];
  const IdxT slot_in = static_cast<const IdxT*>(a.slots)[b];
  const int64_t slot = int64_t(slot_in);
  const int e0 = c * 8;
  auto packed_row = [&](int head) -> T* {
    if (head < a.H) return static_cast<T*>(a.q_out) + (b * a.H + head) * D + e0;
    T* out = static_cast<T*>(head < a.H + a.H_kv ? a.k_out : a.v_out);
    return out == nullptr ? nullptr : out + (b * a.H_kv + (head - a.H) % a.H_kv) * D + e0;
  };
  const bool idle = slot == -1;
  if (idle || pb < 0 || pb >= a.n_pos || slot < 0 || slot >= pool.n_slots) {  // uniform
    if (!idle && blockIdx.y == 0 && threadIdx.x == 0) report(a.err, b);
    const float zero[8] = {};
    for (int head = head0; head < n_heads; head += step) {
      T* row = packed_row(head);
      if (row != nullptr) store8(row, zero);
    }
    return;
  }
  const int half = a.rotary >> 1;  // 32, 64 or 128: a lane's 8 elements are on one side of it
  const int a0 = e0 < half ? e0 : (e0 < a.rotary ? e0 - half : 0);
  float cs[8], sn[8], wq[8], wk[8];
  load8<T, kVec>(static_cast<const T*>(a.cos_tab) + pb * half + a0, 1, cs);
  load8<T, kVec>(static_cast<const T*>(a.sin_tab) + pb * half + a0, 1, sn);
  load8<T, kVec>(static_cast<const T*>(a.q_w) + e0, 1, wq);
  load8<T, kVec>(static_cast<const T*>(a.k_w) + e0, 1, wk);
  const int64_t src = b * a.row_stride + e0;
  for (int head = head0; head < n_heads; head += step) {
    float x[8];
    if constexpr (kParts) {
      const float* f = static_cast<const float*>(a.qkv) + src + int64_t(head) * D;
      load8<float, kVec, true>(f, 1, x);
      for (int s = 1; s < a.parts; ++s) {
        float y[8];
        load8<float, kVec, true>(f + s * a.plane, 1, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += y[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = rt<T>(x[j]);
    } else {
      load8<T, kVec, true>(static_cast<const T*>(a.qkv) + src + int64_t(head) * D, 1, x);
    }
    if (head < a.H + a.H_kv) {  // uniform over a head's lanes
      // Each operation rounded by itself and the squares added in the order of a tensor reduction (fours in turn from
      // D 128 on, then pairs): the result is the one that fp32 tensor operations give, so a k next to a border of
      // its 4-bit levels falls to the same side as theirs.
#pragma clang fp contract(off)
      float sq[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) sq[j] = x[j] * x[j];
      const float low = D == 64 ? (sq[0] + sq[1]) + (sq[2] + sq[3]) : ((sq[0] + sq[1]) + sq[2]) + sq[3];
      const float high = D == 64 ? (sq[4] + sq[5]) + (sq[6] + sq[7]) : ((sq[4] + sq[5]) + sq[6]) + sq[7];
      const float r = exact_rsqrt(group_allreduce<LPR, SumOp>(low + high) * (1.0f / D) + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = head < a.H ? wq[j] : wk[j];
        x[j] = (x[j] * r) * (a.zero_centred ? 1.0f + w : w);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = half == 64 ? dpp<kDppRowRor8>(x[j]) : half == 32 ? swap4(x[j]) : swap16(x[j]);
        const float own = x[j] * cs[j], other = p * sn[j];
        if (e0 < a.rotary) x[j] = e0 < half ? own - other : own + other;
        x[j] = to_f32(from_f32<T>(x[j]));
      }
    }
    T* row = packed_row(head);
    if (row != nullptr) store8(row, x);
    if (head >= a.H) {
      fp4_put<D>(head < a.H + a.H_kv ? pool.k : pool.v, fp4_place<D>(pool, slot, (head - a.H) % a.H_kv, c), c, x);
    }
  }
}

// ------------------------------------------------------------------ host side
int esize_of(int dtype) { return dtype == MI_F32 ? 4 : dtype == MI_F16 || dtype == MI_BF16 ? 2 : 0; }

int log2_of(int64_t x) {
  int n = 0;
  while ((int64_t(1) << n) < x) ++n;
  return n;
}

// The checks that all three entry points share; fills the pool's geometry.
int make_pool(const char* what, void* k, void* v, int64_t n_blocks, int block_size, int H_kv, int D, int dtype,
              int slot_bits, Fp4Pool& pool) {
  if (esize_of(dtype) == 0) return fail(MI_ERR_INVALID, "%s: unknown dtype code %d", what, dtype);
  if (slot_bits != 32 && slot_bits != 64) {
    return fail(MI_ERR_INVALID, "%s: slot_bits must be 32 or 64, got %d", what, slot_bits);
  }
  if (D != 64 && D != 128 && D != 256) {
    return fail(MI_ERR_UNSUPPORTED, "%s: head_dim %d is not supported by the 4-bit cache (64, 128, 256)", what, D);
  }
  if (block_size < 16 || (block_size & (block_size - 1)) != 0) {
    return fail(MI_ERR_UNSUPPORTED, "%s: the 4-bit cache needs a power-of-two block_size of at least 16, got %d", what,
                block_size);
  }
  if (H_kv < 1 || n_blocks < 0) {
    return fail(MI_ERR_INVALID, "%s: bad sizes n_blocks=%lld H_kv=%d", what, (long long)n_blocks, H_kv);
  }
  pool.k = static_cast<uint8_t*>(k);
  pool.v = static_cast<uint8_t*>(v);
  pool.head_bytes = fp4_page_bytes(block_size, D);
  pool.block_bytes = pool.head_bytes * H_kv;
  pool.n_slots = n_blocks * block_size;
  pool.bs_log2 = log2_of(block_size);
  return MI_OK;
}

bool aligned16(std::initializer_list<const void*> all) {
  uintptr_t x = 0;
  for (const void* p : all) x |= reinterpret_cast<uintptr_t>(p);
  return x % 16 == 0;
}

// Rows per lane: two once one per lane fills the chip's 4096 wave slots at 16 per CU (4311 tokens of H_kv 8 / D 128: a write
// 8.1 -> 7.5 us; 32 tokens 2.3 against 2.6).
int rows_per_lane(int64_t n_tokens, int H_kv, int D) { return n_tokens * H_kv * (D / 8) >= 4096 * 64 ? 2 : 1; }

// Workgroups of four waves that give every (token, head) row its own lanes; 0 where the threads of the grid
// would not count in 32 bits.
unsigned row_grid(int64_t n_tokens, int H_kv, int D) {
  const int64_t per_wave = 64 / (D / 8) * rows_per_lane(n_tokens, H_kv, D);
  const int64_t groups = ((n_tokens + per_wave - 1) / per_wave * H_kv + 3) / 4;
  return groups < (1 << 23) ? unsigned(groups) : 0u;
}

template <typename F>
int by_type(int dtype, F&& f) {
  switch (dtype) {
    case MI_BF16: return f(bf16_t{});
    case MI_F16: return f(f16_t{});
    default: return f(float{});
  }
}
template <typename F>
int by_dim(int D, F&& f) {
  switch (D) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    default: return f(std::integral_constant<int, 256>{});
  }
}
template <typename F>
int by_flag(bool x, F&& f) {
  return x ? f(std::true_type{}) : f(std::false_type{});
}

}  // namespace
}  // namespace miattn

extern "C" int64_t mi_fp4_page_bytes(int block_size, int D) {
  if (block_size < 1 || D < 32 || D % 32 != 0) return 0;
  return miattn::fp4_page_bytes(block_size, D);
}

extern "C" int mi_kv_slot_write_fp4(const void* k, const void* v, const void* slot_ids, int slot_bits, void* k_pool,
                                    void* v_pool, int64_t n_tokens, int H_kv, int D, int64_t n_blocks, int block_size,
                                    const int64_t* src_strides, int dtype, int32_t* error_word, void* stream) {
  using namespace miattn;
  Fp4Pool pool;
  const int rc = make_pool("mi_kv_slot_write_fp4", k_pool, v_pool, n_blocks, block_size, H_kv, D, dtype, slot_bits, pool);
  if (rc != MI_OK) return rc;
  if (n_tokens < 0) return fail(MI_ERR_INVALID, "mi_kv_slot_write_fp4: n_tokens %lld < 0", (long long)n_tokens);
  if (src_strides == nullptr) return fail(MI_ERR_INVALID, "mi_kv_slot_write_fp4: src_strides is NULL");
  if (n_tokens == 0) return MI_OK;
  if (k == nullptr || v == nullptr || slot_ids == nullptr || k_pool == nullptr || v_pool == nullptr) {
    return fail(MI_ERR_INVALID, "mi_kv_slot_write_fp4: NULL tensor pointer");
  }
  if (!aligned16({k_pool, v_pool})) {
    return fail(MI_ERR_UNSUPPORTED, "mi_kv_slot_write_fp4: the pools must be 16-byte aligned");
  }
  const int64_t* st = src_strides;
  const int es = esize_of(dtype);
  bool vec = aligned16({k, v}) && st[2] == 1 && st[5] == 1;
  for (int i : {0, 1, 3, 4}) vec = vec && (st[i] * es) % 16 == 0;
  const unsigned grid = row_grid(n_tokens, H_kv, D);
  if (grid == 0) {
    return fail(MI_ERR_UNSUPPORTED, "mi_kv_slot_write_fp4: %lld tokens in one call", (long long)n_tokens);
  }
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_dim(D, [&](auto d) {
      return by_flag(slot_bits == 32, [&](auto narrow) {
        return by_flag(vec, [&](auto is_vec) {
          return by_flag(rows_per_lane(n_tokens, H_kv, D) == 2, [&](auto two) {
            using IdxT = std::conditional_t<decltype(narrow)::value, int32_t, int64_t>;
            constexpr int kRows = decltype(two)::value ? 2 : 1;
            hipLaunchKernelGGL((fp4_write_kernel<T, decltype(d)::value, IdxT, decltype(is_vec)::value, kRows>),
                               dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream),
                               static_cast<const T*>(k), static_cast<const T*>(v), static_cast<const IdxT*>(slot_ids),
                               pool, n_tokens, H_kv, st[0], st[1], st[2], st[3], st[4], st[5], error_word);
            return launch_status("mi_kv_slot_write_fp4");
          });
        });
      });
    });
  });
}

extern "C" int mi_kv_slot_read_fp4(const void* k_pool, const void* v_pool, const void* slot_ids, int slot_bits, void* k,
                                   void* v, int64_t n_tokens, int H_kv, int D, int64_t n_blocks, int block_size,
                                   int dtype, int32_t* error_word, void* stream) {
  using namespace miattn;
  Fp4Pool pool;
  const int rc = make_pool("mi_kv_slot_read_fp4", const_cast<void*>(k_pool), const_cast<void*>(v_pool), n_blocks,
                           block_size, H_kv, D, dtype, slot_bits, pool);
  if (rc != MI_OK) return rc;
  if (n_tokens < 0) return fail(MI_ERR_INVALID, "mi_kv_slot_read_fp4: n_tokens %lld < 0", (long long)n_tokens);
  if (n_tokens == 0) return MI_OK;
  if (k == nullptr || v == nullptr || slot_ids == nullptr || k_pool == nullptr || v_pool == nullptr) {
    return fail(MI_ERR_INVALID, "mi_kv_slot_read_fp4: NULL tensor pointer");
  }
  if (!aligned16({k_pool, v_pool, k, v})) {
    return fail(MI_ERR_UNSUPPORTED, "mi_kv_slot_read_fp4: the pools and outputs must be 16-byte aligned");
  }
  const unsigned grid = row_grid(n_tokens, H_kv, D);
  if (grid == 0) {
    return fail(MI_ERR_UNSUPPORTED, "mi_kv_slot_read_fp4: %lld tokens in one call", (long long)n_tokens);
  }
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_dim(D, [&](auto d) {
      return by_flag(slot_bits == 32, [&](auto narrow) {
        return by_flag(rows_per_lane(n_tokens, H_kv, D) == 2, [&](auto two) {
          using IdxT = std::conditional_t<decltype(narrow)::value, int32_t, int64_t>;
          constexpr int kRows = decltype(two)::value ? 2 : 1;
          hipLaunchKernelGGL((fp4_read_kernel<T, decltype(d)::value, IdxT, kRows>), dim3(grid), dim3(256), 0,
                             static_cast<hipStream_t>(stream), pool, static_cast<const IdxT*>(slot_ids),
                             static_cast<T*>(k), static_cast<T*>(v), n_tokens, H_kv, error_word);
          return launch_status("mi_kv_slot_read_fp4");
        });
      });
    });
  });
}

extern "C" int mi_qk_norm_rope_write_fp4(const void* qkv, int64_t row_stride, int qkv_parts, const void* q_norm_w,
                                         const void* k_norm_w, const void* cos_tab, const void* sin_tab, int64_t n_pos,
                                         int rotary_dim, const int64_t* pos, const void* slot_ids, int slot_bits,
                                         void* q_out, void* k_pool, void* v_pool, void* k_out, void* v_out, int B, int H,
                                         int H_kv, int D, int64_t n_blocks, int block_size, float eps, int norm_mode,
                                         int dtype, int32_t* error_word, void* stream) {
  using namespace miattn;
  Fp4Pool pool;
  const int rc =
      make_pool("mi_qk_norm_rope_write_fp4", k_pool, v_pool, n_blocks, block_size, H_kv, D, dtype, slot_bits, pool);
  if (rc != MI_OK) return rc;
  if (B < 0 || H < 1 || H % H_kv != 0) {
    return fail(MI_ERR_INVALID, "mi_qk_norm_rope_write_fp4: n_head (%d) must be a multiple of n_kv_head (%d)", H, H_kv);
  }
  if (n_pos < 1) return fail(MI_ERR_INVALID, "mi_qk_norm_rope_write_fp4: the RoPE table is empty");
  if (qkv_parts < 0) return fail(MI_ERR_INVALID, "mi_qk_norm_rope_write_fp4: qkv_parts %d < 0", qkv_parts);
  if (row_stride < int64_t(H + 2 * H_kv) * D) {
    return fail(MI_ERR_INVALID, "mi_qk_norm_rope_write_fp4: row stride %lld < %d packed q/k/v elements",
                (long long)row_stride, (H + 2 * H_kv) * D);
  }
  if (!(rotary_dim == 64 || rotary_dim == 128 || rotary_dim == 256) || rotary_dim > D) {
    return fail(MI_ERR_UNSUPPORTED, "mi_qk_norm_rope_write_fp4: rotary_dim %d must be 64, 128 or 256 and <= head_dim %d",
                rotary_dim, D);
  }
  if (norm_mode != 0 && norm_mode != 1) {
    return fail(MI_ERR_INVALID, "mi_qk_norm_rope_write_fp4: norm_mode %d is not 0 or 1", norm_mode);
  }
  if (B == 0) return MI_OK;
  if (qkv == nullptr || q_norm_w == nullptr || k_norm_w == nullptr || cos_tab == nullptr || sin_tab == nullptr ||
      pos == nullptr || slot_ids == nullptr || q_out == nullptr || k_pool == nullptr || v_pool == nullptr) {
    return fail(MI_ERR_INVALID, "mi_qk_norm_rope_write_fp4: NULL pointer argument");
  }
  if (!aligned16({k_pool, v_pool, q_out, k_out, v_out})) {
    return fail(MI_ERR_UNSUPPORTED, "mi_qk_norm_rope_write_fp4: the pools and outputs must be 16-byte aligned");
  }
  const EpilogueArgs a{qkv, row_stride, qkv_parts, int64_t(B) * row_stride, q_norm_w, k_norm_w, cos_tab, sin_tab, n_pos,
                       rotary_dim, pos, slot_ids, q_out, k_out, v_out, B, H, H_kv, eps, norm_mode, error_word};
  const int in_size = qkv_parts > 0 ? 4 : esize_of(dtype);
  const bool vec = aligned16({qkv, q_norm_w, k_norm_w, cos_tab, sin_tab}) && (row_stride * in_size) % 16 == 0;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_dim(D, [&](auto d) {
      return by_flag(slot_bits == 32, [&](auto narrow) {
        return by_flag(vec, [&](auto is_vec) {
          return by_flag(qkv_parts > 0, [&](auto is_parts) {
            using IdxT = std::conditional_t<decltype(narrow)::value, int32_t, int64_t>;
            constexpr int Dv = decltype(d)::value, HPW = 256 / (Dv / 8);
            const unsigned groups = (H + 2 * H_kv + HPW - 1) / HPW;
            // From kRowPerGroup rows one workgroup walks all heads of a row, so position, slot, rotation and norm
            // weights are loaded once (8192 rows of H 16 / H_kv 8 / D 128: 34.5 -> 30.7 us, 4.7 TB/s); below, the heads are
            // shared out so that a small batch still spreads over the chip.
            constexpr int kRowPerGroup = 1024;
            hipLaunchKernelGGL(
                (fp4_epilogue_kernel<T, Dv, IdxT, decltype(is_vec)::value, decltype(is_parts)::value>),
                dim3(B, B >= kRowPerGroup ? 1 : groups), dim3(256), 0, static_cast<hipStream_t>(stream), a, pool);
            return launch_status("mi_qk_norm_rope_write_fp4");
          });
        });
      });
    });
  });
}
