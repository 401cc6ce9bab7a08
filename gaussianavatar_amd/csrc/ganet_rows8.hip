// ganet_rows8.hip — activations and weights to 8-bit floating point and back (include/ganet.h: ganet_rows8_*, ganet_weight8_pack).
//
// A block of 128 values x shares a power of two: a = max |x|, e = the smallest integer with a <= F 2^e, code = RNE(x 2^-e).
// The scale being a power of two, x 2^-e is exact and the only rounding is the one to the format: at most 2^-4 (e4m3) or
// 2^-3 (e5m2) of the value, or half of the smallest step 2^(e-9) (2^(e-16)) for values far below the block's largest.
// The exponent byte e + 127 is what the matrix instructions take as their operand scale.
//
// Bound: HBM. Sixteen lanes hold a block, eight values each (one 16-byte load of a 16-bit type, two of fp32), the maximum is
// four shuffles, the codes leave as 8 bytes per lane: consecutive lanes write consecutive bytes.
#include "ganet_rows8.h"

namespace ganet {
using namespace rows8;

namespace {

constexpr int WG = 256;
constexpr int GROUPS = WG / 16;            // blocks of 128 values that a workgroup takes at a time

// How blocks map to workgroups: a row of KB blocks takes 2^log2p groups (the workgroup covers GROUPS >> log2p rows), or, where
// KB >= GROUPS, a workgroup takes GROUPS consecutive blocks of one row: no division per lane either way.
struct Map { int log2p; int64_t segs; int64_t grid; };
Map make_map(int64_t M, int64_t KB) {
  Map m;
  m.log2p = 0;
  while ((1 << m.log2p) < KB && m.log2p < 4) ++m.log2p;
  m.segs = cdiv(KB, GROUPS);
  m.grid = KB > GROUPS ? M * m.segs : cdiv(M, GROUPS >> m.log2p);
  return m;
}

__device__ __forceinline__ void my_block(int64_t KB, const Map& m, int64_t& row, int64_t& kb) {
  const int grp = threadIdx.x >> 4;
  if (KB > GROUPS) {
    row = blockIdx.x / (unsigned)m.segs;
    kb = (int64_t)(blockIdx.x % (unsigned)m.segs) * GROUPS + grp;
  } else {
    row = (int64_t)blockIdx.x * (GROUPS >> m.log2p) + (grp >> m.log2p);
    kb = grp & ((1 << m.log2p) - 1);
  }
}

template <typename T, int FMT>
__global__ void __launch_bounds__(WG)
rows8_pack_kernel(int64_t M, int64_t C, const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ codes, int64_t ldc,
                  uint8_t* __restrict__ exps, int64_t lde, int64_t KB, Map map) {
  int64_t row, kb;
  my_block(KB, map, row, kb);
  if (row >= M || kb >= KB) return;                       // whole groups of 16 lanes: the shuffles below stay inside a group
  const int l = threadIdx.x & 15;
  const int64_t c0 = kb * BLOCK + l * 8;
  float v[8];
  load_n(x + row * ldx + c0, C - c0, v);
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(v[i]));
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor(a, off, 16));
  const int e = block_exponent<FMT>(a);
  const float s = pow2(-e);                               // e <= 120: a normal number
  uint2 out;
  out.x = pack4<FMT>(v[0] * s, v[1] * s, v[2] * s, v[3] * s);
  out.y = pack4<FMT>(v[4] * s, v[5] * s, v[6] * s, v[7] * s);
  if (c0 < (C + 15) / 16 * 16) *reinterpret_cast<uint2*>(codes + row * ldc + c0) = out;
  if (l == 0) exps[row * lde + kb] = (uint8_t)(e + 127);
}

template <typename T>
__device__ __forceinline__ float largest();
template <> __device__ __forceinline__ float largest<float>() { return 3.402823466e38f; }
template <> __device__ __forceinline__ float largest<__bf16>() { return 3.3895313892515355e38f; }
template <> __device__ __forceinline__ float largest<_Float16>() { return 65504.f; }

template <typename T, int FMT>
__global__ void __launch_bounds__(WG)
rows8_unpack_kernel(int64_t M, int64_t C, const uint8_t* __restrict__ codes, int64_t ldc, const uint8_t* __restrict__ exps,
                    int64_t lde, T* __restrict__ y, int64_t KB, Map map) {
  int64_t row, kb;
  my_block(KB, map, row, kb);
  if (row >= M || kb >= KB) return;
  const int64_t c0 = kb * BLOCK + (threadIdx.x & 15) * 8;
  if (c0 >= C) return;
  const uint2 in = *reinterpret_cast<const uint2*>(codes + row * ldc + c0);
  const float s = pow2((int)exps[row * lde + kb] - 127);
  float lo[4], hi[4], v[8];
  unpack4<FMT>(in.x, lo);
  unpack4<FMT>(in.y, hi);
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[i] = lo[i]; v[4 + i] = hi[i]; }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float r = v[i] * s;                             // exact, or beyond the type's range
    const float b = fminf(fmaxf(r, -largest<T>()), largest<T>());
    v[i] = fabsf(v[i]) < __builtin_huge_valf() ? b : r;   // (a NaN and an e5m2 infinity stay what they are)
  }
  store_n(y + row * C + c0, C - c0, v);
}

// 4 x 4 bytes transposed: r[i] holds row i; afterwards column i
__device__ __forceinline__ void transpose4(unsigned (&r)[4]) {
  const unsigned a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
  const unsigned c = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), d = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
  r[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  r[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  r[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  r[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// One workgroup per 128 x 128 block: a thread holds 8 rows of 8 columns in registers, so that the weight is read once, 256 bytes (bf16) of a
// row by 16 lanes. The transposed codes are turned in registers, 4 x 4 bytes at a time, and change lanes through LDS, so that
// their rows leave as 128 bytes each. 8192 x 4096 bf16 with both orders: 88 us with the bytes turned in LDS one by one.
template <typename T>
__global__ void __launch_bounds__(WG)
weight8_pack_kernel(int64_t N, int64_t K, const T* __restrict__ w, int64_t ldw, uint8_t* __restrict__ codes, int64_t ldc,
                    uint8_t* __restrict__ exps, int64_t lde, uint8_t* __restrict__ tcodes, int64_t ldtc,
                    uint8_t* __restrict__ texps, int64_t ldte) {
  constexpr int PITCH = BLOCK + 8;
  __shared__ float s_max[WG / 64];
  __shared__ __align__(16) uint8_t s_t[BLOCK * PITCH];          // [column][row]
  const int64_t kb = blockIdx.x, nb = blockIdx.y;
  const int r0 = (threadIdx.x >> 4) * 8, c0 = (threadIdx.x & 15) * 8;
  const int64_t n0 = nb * BLOCK + r0, k0 = kb * BLOCK + c0;
  float v[8][8];
  float a = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) load_n(w + (n0 + j) * ldw + k0, n0 + j < N ? K - k0 : 0, v[j]);
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(v[j][i]));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) a = fmaxf(a, __shfl_xor(a, off));
  if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = a;
  __syncthreads();
  a = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  const int e = block_exponent<GANET_E4M3>(a);
  const float s = pow2(-e);
  const int64_t kpad = (K + 15) / 16 * 16;
  unsigned c[8][2];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    c[j][0] = pack4<GANET_E4M3>(v[j][0] * s, v[j][1] * s, v[j][2] * s, v[j][3] * s);
    c[j][1] = pack4<GANET_E4M3>(v[j][4] * s, v[j][5] * s, v[j][6] * s, v[j][7] * s);
    if (n0 + j < N && k0 < kpad) *reinterpret_cast<uint2*>(codes + (n0 + j) * ldc + k0) = make_uint2(c[j][0], c[j][1]);
  }
  if (threadIdx.x == 0) {
    exps[nb * lde + kb] = (uint8_t)(e + 127);
    if (tcodes) texps[kb * ldte + nb] = (uint8_t)(e + 127);
  }
  if (!tcodes) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {                 // columns 4 h .. 4 h + 3: rows 0 .. 3 and 4 .. 7
    unsigned lo[4] = {c[0][h], c[1][h], c[2][h], c[3][h]}, hi[4] = {c[4][h], c[5][h], c[6][h], c[7][h]};
    transpose4(lo);
    transpose4(hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint2*>(s_t + (c0 + 4 * h + i) * PITCH + r0) = make_uint2(lo[i], hi[i]);
  }
  __syncthreads();
  const int64_t npad = (N + 15) / 16 * 16, nn = nb * BLOCK + (threadIdx.x & 7) * 16;
  if (nn >= npad) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = j * 32 + (threadIdx.x >> 3);
    const int64_t k = kb * BLOCK + col;
    if (k >= K) continue;
    const uint2* src = reinterpret_cast<const uint2*>(s_t + col * PITCH + (threadIdx.x & 7) * 16);
    const uint2 x = src[0], y = src[1];
    *reinterpret_cast<uint4*>(tcodes + k * ldtc + nn) = make_uint4(x.x, x.y, y.x, y.y);
  }
}

// The rows of one launch: a grid has fewer than 2^32 threads in all
int64_t rows_per_launch(const Map& m, int64_t KB) {
  constexpr int64_t most = (1ll << 23);
  return KB > GROUPS ? most / m.segs : most * (GROUPS >> m.log2p);
}

bool codes_ok(const void* codes, int64_t ldc, int64_t C, const uint8_t* exps, int64_t lde) {
  return codes && exps && ldc % 16 == 0 && ldc >= pad16(C) && (reinterpret_cast<uintptr_t>(codes) & 15) == 0 && lde % 4 == 0 &&
         lde >= cdiv(C, BLOCK) && (reinterpret_cast<uintptr_t>(exps) & 3) == 0;
}

}  // namespace
}  // namespace ganet

using namespace ganet;

extern "C" {

int ganet_rows8_pack(int64_t M, int64_t C, int32_t type, int32_t fmt, const void* x, int64_t ldx, void* codes, int64_t ldc,
                     uint8_t* exps, int64_t lde, void* stream_) {
  if (!rows_ok(M, C) || !type_ok(type) || (fmt != GANET_E4M3 && fmt != GANET_E5M2)) {
    set_error("ganet_rows8_pack: unsupported M=%lld C=%lld type=%d format=%d", (long long)M, (long long)C, type, fmt);
    return 4;
  }
  if (M == 0) return 0;
  if (!x || (ldx < C && M > 1) || !codes_ok(codes, ldc, C, exps, lde)) {
    set_error("ganet_rows8_pack: NULL or misaligned argument, or a row stride too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const int64_t KB = cdiv(C, BLOCK);
  const int64_t most = rows_per_launch(make_map(M, KB), KB);
  for (int64_t m = 0; m < M; m += most) {
    const int64_t rows = M - m < most ? M - m : most;
    const Map map = make_map(rows, KB);
    GANET_BY_TYPE(type, T, {
      auto k = fmt == GANET_E4M3 ? rows8_pack_kernel<T, GANET_E4M3> : rows8_pack_kernel<T, GANET_E5M2>;
      hipLaunchKernelGGL(k, dim3((unsigned)map.grid), dim3(WG), 0, stream, rows, C, static_cast<const T*>(x) + m * ldx, ldx,
                         static_cast<uint8_t*>(codes) + m * ldc, ldc, exps + m * lde, lde, KB, map);
    });
  }
  return check_hip(hipGetLastError(), "ganet_rows8_pack");
}

int ganet_rows8_unpack(int64_t M, int64_t C, int32_t type, int32_t fmt, const void* codes, int64_t ldc, const uint8_t* exps,
                       int64_t lde, void* y, void* stream_) {
  if (!rows_ok(M, C) || !type_ok(type) || (fmt != GANET_E4M3 && fmt != GANET_E5M2)) {
    set_error("ganet_rows8_unpack: unsupported M=%lld C=%lld type=%d format=%d", (long long)M, (long long)C, type, fmt);
    return 4;
  }
  if (M == 0) return 0;
  if (!y || !codes_ok(codes, ldc, C, exps, lde)) {
    set_error("ganet_rows8_unpack: NULL or misaligned argument, or a row stride too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const int64_t KB = cdiv(C, BLOCK);
  const int64_t most = rows_per_launch(make_map(M, KB), KB);
  for (int64_t m = 0; m < M; m += most) {
    const int64_t rows = M - m < most ? M - m : most;
    const Map map = make_map(rows, KB);
    GANET_BY_TYPE(type, T, {
      auto k = fmt == GANET_E4M3 ? rows8_unpack_kernel<T, GANET_E4M3> : rows8_unpack_kernel<T, GANET_E5M2>;
      hipLaunchKernelGGL(k, dim3((unsigned)map.grid), dim3(WG), 0, stream, rows, C, static_cast<const uint8_t*>(codes) + m * ldc, ldc,
                         exps + m * lde, lde, static_cast<T*>(y) + m * C, KB, map);
    });
  }
  return check_hip(hipGetLastError(), "ganet_rows8_unpack");
}

int ganet_weight8_pack(int64_t N, int64_t K, int32_t type, const void* w, int64_t ldw, void* codes, int64_t ldc, uint8_t* exps,
                       int64_t lde, void* tcodes, int64_t ldtc, uint8_t* texps, int64_t ldte, void* stream_) {
  if (!rows_ok(N, K) || N < 1 || N >= (1ll << 23) || !type_ok(type)) {
    set_error("ganet_weight8_pack: unsupported N=%lld K=%lld type=%d", (long long)N, (long long)K, type);
    return 4;
  }
  if (!w || (ldw < K && N > 1) || !codes_ok(codes, ldc, K, exps, lde) || (tcodes && !codes_ok(tcodes, ldtc, N, texps, ldte))) {
    set_error("ganet_weight8_pack: NULL or misaligned argument, or a row stride too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const dim3 grid((unsigned)cdiv(K, BLOCK), (unsigned)cdiv(N, BLOCK));
  if (grid.y > 65535u) { set_error("ganet_weight8_pack: too many rows"); return 4; }
  GANET_BY_TYPE(type, T,
                hipLaunchKernelGGL(weight8_pack_kernel<T>, grid, dim3(WG), 0, stream, N, K, static_cast<const T*>(w), ldw,
                                   static_cast<uint8_t*>(codes), ldc, exps, lde, static_cast<uint8_t*>(tcodes), ldtc, texps,
                                   ldte));
  return check_hip(hipGetLastError(), "ganet_weight8_pack");
}

}  // extern "C"
