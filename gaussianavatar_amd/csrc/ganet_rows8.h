// ganet_rows8.h — element types, 8-bit conversions and row access shared by the row-wise operators (internal).
#pragma once
#include <cstdint>

#include <hip/hip_runtime.h>

#include "ganet.h"
#include "ganet_common.h"

namespace ganet {
namespace rows8 {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int BLOCK = 128;                 // columns that share a power of two

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t pad16(int64_t c) { return (c + 15) / 16 * 16; }
inline int type_size(int32_t type) { return type == GANET_F32 ? 4 : 2; }
inline bool type_ok(int32_t type) { return type >= GANET_F32 && type <= GANET_F16; }

// N consecutive elements from `p`, of which the first n exist (the others read as zero): one or two 16-byte loads where
// all exist, whatever the alignment (the copy tells the compiler nothing beyond the element's own alignment, and the
// hardware takes unaligned vector accesses).
template <int N, typename T>
__device__ __forceinline__ void load_n(const T* __restrict__ p, int64_t n, float (&v)[N]) {
  if (n >= N) {
    T t[N];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
  }
}

template <int N, typename T>
__device__ __forceinline__ void store_n(T* __restrict__ p, int64_t n, const float (&v)[N]) {
  if (n >= N) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)v[i];
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

// The same past the caches, 16 bytes at a time: for what this operator does not touch again.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_loose __attribute__((aligned(2)));
template <typename T>
__device__ __forceinline__ u32x4 load_stream(const T* p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4_loose*>(p)); }
template <int N, typename T>
__device__ __forceinline__ void store_stream(T* __restrict__ p, int64_t n, const float (&v)[N]) {
  static_assert(N * sizeof(T) == 16, "one 16-byte store");
  if (n >= N) {
    T t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = (T)v[i];
    u32x4 q;
    __builtin_memcpy(&q, t, 16);
    __builtin_nontemporal_store(q, reinterpret_cast<u32x4_loose*>(p));
  } else store_n(p, n, v);
}

// one parameter of a type known at run time (a uniform branch)
__device__ __forceinline__ float load_param(const void* p, int32_t type, int64_t i) {
  return type == GANET_F32 ? static_cast<const float*>(p)[i]
         : type == GANET_BF16 ? (float)static_cast<const __bf16*>(p)[i]
                              : (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void store_param(void* p, int32_t type, int64_t i, float v) {
  if (type == GANET_F32) static_cast<float*>(p)[i] = v;
  else if (type == GANET_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
  else static_cast<_Float16*>(p)[i] = (_Float16)v;
}

// N consecutive parameters from element c on, `fill` where there are none (no tensor, or past its n elements)
template <int N>
__device__ __forceinline__ void load_params(const void* p, int32_t type, int c, int n, float fill, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = fill;
  if (!p || n <= 0) return;
  if (n >= N) {
    if (type == GANET_F32) load_n(static_cast<const float*>(p) + c, n, v);
    else if (type == GANET_BF16) load_n(static_cast<const __bf16*>(p) + c, n, v);
    else load_n(static_cast<const _Float16*>(p) + c, n, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) v[i] = load_param(p, type, c + i);
  }
}

// four values -> four codes, round to nearest, ties to even
template <int FMT>
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
  int r = 0;
  if (FMT == GANET_E4M3) {
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  } else {
    r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false);
    r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
  }
  return (unsigned)r;
}
template <int FMT>
__device__ __forceinline__ void unpack4(unsigned codes, float (&v)[4]) {
  f32x2 lo, hi;
  if (FMT == GANET_E4M3) {
    lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
    hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  } else {
    lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)codes, false);
    hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)codes, true);
  }
  v[0] = lo[0]; v[1] = lo[1]; v[2] = hi[0]; v[3] = hi[1];
}

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (e + 127) << 23); }

// Half of a block's scale, from its biased exponent e + 127 >= 1. The largest numbers of fp32 and bf16 are rounded to 2^128 by their codes (256 2^120), which
// bf16 has not: their halves it has. What is multiplied on bf16 instructions is decoded at half its size and doubled in the result.
// (For e = -126 the bits are those of zero; the conversions read the exponent field alone, 2^-127.)
__device__ __forceinline__ float half_scale(int biased) { return __builtin_bit_cast(float, (biased - 1) << 23); }

// The block exponent: with a = 1.m 2^p, F = 1.75 2^q (448: q = 8; 57344: q = 15) the smallest e with a <= F 2^e is p - q, or p - q + 1
// where 1.m > 1.75. Adding 0x1fffff to the bits carries into the exponent field exactly there. a is finite and >= 0;
// below 2^-118 the exponent stays at -126 and the codes lose bits, as numbers that small do in the type itself.
template <int FMT>
__device__ __forceinline__ int block_exponent(float a) {
  constexpr int q = FMT == GANET_E4M3 ? 8 : 15;
  const int p = (int)((__builtin_bit_cast(unsigned, a) + 0x1fffffu) >> 23) - 127;
  return a > 0.f ? max(p - q, -126) : 0;
}

// the magnitude that counts for a block's exponent: a NaN or an infinity does not
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < __builtin_huge_valf() ? a : 0.f;
}

// ctypes callers hand sizes over as they are: refuse what the kernels' grids and indices do not cover
inline bool rows_ok(int64_t M, int64_t C) { return M >= 0 && C >= 1 && M < (1ll << 31) && C < (1ll << 24); }

#define GANET_BY_TYPE(type, T, ...)                          \
  do {                                                       \
    if ((type) == GANET_F32) { using T = float; __VA_ARGS__; } \
    else if ((type) == GANET_BF16) { using T = __bf16; __VA_ARGS__; } \
    else { using T = _Float16; __VA_ARGS__; }                \
  } while (0)

}  // namespace rows8
}  // namespace ganet
