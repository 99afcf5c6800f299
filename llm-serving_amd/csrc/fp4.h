// The 4-bit cache row format and its conversions (gfx950 converts FP4 pairs natively).
//
// A row is the D elements of one (token, KV head). Groups of 32 elements share a scale 2^e; each
// element is a 4-bit float (sign, then 0, 0.5, 1, 1.5, 2, 3, 4 or 6) times it. e is the smallest
// integer with max|x| <= 7 * 2^e, so no element is off by more than 2^e and none of a group's
// range is left unused (max / 2^e is in (3.5, 7]; past 6 an element is stored as 6, which is off
// by at most 1, what the gap between 4 and 6 costs too). e is held to [-120, 125]: below, 0.5 *
// 2^e would leave bf16's normal range, above, 6 * 2^e would overflow fp32 and bf16. A power of two
// because the conversion instructions apply it for nothing: no multiplication per element, and a row's
// values are exact in bf16 (two significant bits), which is what the attention's matrix products read.
// A group with a value that is not finite gets the scale byte 255 (codes 0), which those instructions
// turn into NaN for the whole group.
//
// A page (block_size tokens of one KV head, one of K or V): block_size rows of D / 2 code bytes
// (element 2i in the low half of byte i), then D / 32 rows of block_size scale bytes (e + 127). One head's
// tokens are contiguous, so a wave streams whole lines for one head, and the scales of four
// consecutive tokens of a group are one aligned dword.
#pragma once

#include "common.h"

namespace miattn {

constexpr int kFp4Group = 32;

// bytes of one page of one KV head
__host__ __device__ constexpr int64_t fp4_page_bytes(int64_t block_size, int D) {
  return block_size * (D / 2 + D / kFp4Group);
}

__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Largest |x| of 8 elements per lane over the 4 lanes (an aligned quad) of a group, as bits: as
// unsigned integers the absolute values order as the floats do, with infinity and NaN on top.
__device__ __forceinline__ uint32_t fp4_group_max(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max_u32(m, __float_as_uint(x[j]) & 0x7fffffffu);
  m = max_u32(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), kDppQuadXor1, 0xf, 0xf, false)));
  return max_u32(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), kDppQuadXor2, 0xf, 0xf, false)));
}

// Scale byte of a group whose largest |x| has these bits. 7 * 2^e = 1.75 * 2^(e + 2): e is the exponent
// less 2, one more where the significand is past 1.75 (the sum carries into the exponent).
__device__ __forceinline__ int fp4_scale_byte(uint32_t most) {
  const int e = int((most + 0x1fffffu) >> 23) - 2;
  const int byte = e < 7 ? 7 : e > 252 ? 252 : e;
  return most >= 0x7f800000u ? 255 : byte;
}

// The float whose exponent field is a scale byte (the conversions read nothing else of it).
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight elements as a code dword: nearest level, ties to the even code, past 6 to 6.
__device__ __forceinline__ uint32_t fp4_encode(const float (&x)[8], int scale_byte) {
  const float s = fp4_scale(uint32_t(scale_byte));
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  return scale_byte == 255 ? 0u : w;
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

// The same for eight 16-bit elements as they are in memory: the largest |x| as 16-bit integers, two at a time, and the
// conversions that read 16-bit pairs (a third of the instructions; a write of 4311 tokens at H_kv 8 / D 128 7.2 -> 6.9 us).
template <typename T>
__device__ __forceinline__ uint32_t fp4_group_max16(const uint4& w) {
  auto bits = [](uint32_t x) { return __builtin_bit_cast(u16x2_t, x & 0x7fff7fffu); };
  const u16x2_t a = __builtin_elementwise_max(bits(w.x), bits(w.y)), b = __builtin_elementwise_max(bits(w.z), bits(w.w));
  const u16x2_t c = __builtin_elementwise_max(a, b);
  uint32_t m = max_u32(c.x, c.y);
  m = max_u32(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), kDppQuadXor1, 0xf, 0xf, false)));
  m = max_u32(m, uint32_t(__builtin_amdgcn_update_dpp(0, int(m), kDppQuadXor2, 0xf, 0xf, false)));
  return __float_as_uint(to_f32(T{uint16_t(m)}));  // infinity and NaN stay what they are
}
template <typename T>
__device__ __forceinline__ uint32_t fp4_encode16(const uint4& x, int scale_byte) {
  const float s = fp4_scale(uint32_t(scale_byte));
  uint32_t w = 0;
  if constexpr (std::is_same<T, bf16_t>::value) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x.x), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x.y), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x.z), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x.w), s, 3);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2_t, x.x), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2_t, x.y), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2_t, x.z), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2_t, x.w), s, 3);
  }
  return scale_byte == 255 ? 0u : w;
}

// The eight values of a code dword.
__device__ __forceinline__ void fp4_decode(uint32_t w, float scale, float (&x)[8]) {
  const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
  const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
  const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
  const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}

// x as a T, values past fp16's largest as that (a stored 65504 reads as 65536: its group's grid
// has no level nearer); NaN stays.
template <typename T>
__device__ __forceinline__ float fp4_saturate(float x) {
  if constexpr (std::is_same<T, f16_t>::value) {
    x = x > 65504.0f ? 65504.0f : x;
    x = x < -65504.0f ? -65504.0f : x;
  }
  return x;
}

// Eight consecutive elements of T as fp32: 16-byte loads (kVec: p is 16-byte aligned and the stride 1)
// or one by one with a stride. kOnce: read here and not again soon, so past the caches (the slot write of 4311
// tokens at H_kv 8 / D 128 9.6 -> 7.3 us, the epilogue of 8192 37.7 -> 35.8).
template <typename T, bool kVec, bool kOnce = false>
__device__ __forceinline__ void load8(const T* p, int64_t stride, float (&x)[8]) {
  if constexpr (kVec) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      const uint4 w = kOnce ? load16_nt(p + i) : load16(p + i);
#pragma unroll
      for (int j = 0; j < N; ++j) x[i + j] = Vec16<T>::get(w, j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = to_f32(p[j * stride]);
  }
}

// Eight values as T, 16-byte aligned; kPast: past the caches.
template <typename T, bool kPast = false>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  constexpr int N = Vec16<T>::N;
#pragma unroll
  for (int i = 0; i < 8; i += N) {
    if constexpr (kPast) store16_nt(p + i, pack16<T>(x + i));
    else store16(p + i, pack16<T>(x + i));
  }
}

}  // namespace miattn
