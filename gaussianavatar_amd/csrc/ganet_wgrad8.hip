// ganet_wgrad8.hip — the weight gradient of a layer whose input is kept in 8 bits (include/ganet.h: ganet_wgrad8).
//
//   dW[n, k] = sum_m g[m, n] 2^(e[m, k / 128]) code[m, k],   db[n] = sum_m g[m, n]
//
// The sum runs over the rows, along which the powers of two change, so the 8-bit matrix instructions (one scale per 32 products of
// a lane) do not apply to it as it lies. Codes become bf16 instead: 4 significand bits and a power of two fit bf16 exactly, so the kept input
// enters with no further rounding. g enters with all its bits as 1 (bf16), 2 (fp16) or 3 (fp32) bf16 pieces; sums are fp32.
//
// Both operands need the row index as the matrix instruction's k: tiles lie in LDS as they lie in memory ([row][column], bf16) and
// ds_read_b64_tr_b16 hands each lane four rows of its column.
#include "ganet_rows8.h"

namespace ganet {
using namespace rows8;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int WG = 256, TN = 128, TK = 128, STEP = 32;
// LDS row: 128 columns and 64 bytes more, so that the four rows that a 16-lane group reads start in four different 64-byte columns
constexpr int PITCH = TK + 32;
constexpr int PLANE = STEP * PITCH;

template <typename G> constexpr int PIECES = 3;
template <> constexpr int PIECES<__bf16> = 1;
template <> constexpr int PIECES<_Float16> = 2;

__device__ __forceinline__ unsigned bits(float v) { return __builtin_bit_cast(unsigned, v); }
__device__ __forceinline__ float head(float v) { return __builtin_bit_cast(float, bits(v) & 0xffff0000u); }
// upper halves of two fp32 words: two bf16 in order
__device__ __forceinline__ unsigned pack_hi(float even, float odd) {
  return __builtin_amdgcn_perm(bits(odd), bits(even), 0x07060302u);
}

template <int FMT>
__device__ __forceinline__ unsigned decode2(unsigned codes, float scale, bool high) {
  bf16x2 r;
  if (FMT == GANET_E4M3) r = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true)
                                  : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false);
  else r = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(codes, scale, true)
                : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(codes, scale, false);
  return __builtin_bit_cast(unsigned, r);
}

// eight rows (8 (lane / 32) + 0..7 of the 16 that start at m0) of column c0 + lane % 32
__device__ __forceinline__ bf16x8 column8(const unsigned short* plane, int m0, int c0, int lane) {
  const int grp = lane >> 4, li = lane & 15;
  const unsigned short* p = plane + (m0 + (grp >> 1) * 8 + (li >> 2)) * PITCH + c0 + (grp & 1) * 16 + (li & 3) * 4;
  union { s16x4 h[2]; bf16x8 v; } r;
  r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
  r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * PITCH));
  return r.v;
}

struct Job {
  int64_t M, N, K;
  const void* g; int64_t ldg; const uint8_t* codes; int64_t ldc; const uint8_t* exps; int64_t lde;
  void* dW; void* db; int32_t otype; float* part; int splits; int64_t rows; int tiles_n, tiles_k;
};

template <int FMT, typename G>
__global__ void __launch_bounds__(WG)
wgrad8_kernel(Job o) {
  constexpr int P = PIECES<G>;
  extern __shared__ __align__(16) unsigned short s_mem[];      // P planes of g, one of x
  unsigned short* const s_x = s_mem + P * PLANE;
  const int tiles = o.tiles_n * o.tiles_k;
  const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
  const int64_t n0 = (int64_t)(tile / o.tiles_k) * TN, kb = tile % o.tiles_k, k0 = kb * TK;
  const int64_t m_lo = split * o.rows, m_hi = min(m_lo + o.rows, o.M);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wn = (wave & 1) * 64, wk = (wave >> 1) * 64;
  const int sr = threadIdx.x >> 3, sc = (threadIdx.x & 7) * 16;        // this thread's 16 columns of a staged row
  const int64_t kend = (o.K + 15) / 16 * 16;
  const G* g = static_cast<const G*>(o.g);

  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const bool sums = k0 == 0 && o.db;
  float bias[16] = {};

  float gv[16];
  uint4 xv;
  float scale;
  auto load = [&](int64_t m) {
    const int64_t row = m + sr;
    const bool live = row < m_hi;
    load_n(g + row * o.ldg + n0 + sc, live ? o.N - (n0 + sc) : 0, gv);
    const bool in = live && k0 + sc < kend;
    xv = in ? *reinterpret_cast<const uint4*>(o.codes + row * o.ldc + k0 + sc) : make_uint4(0, 0, 0, 0);
    scale = in ? pow2((int)o.exps[row * o.lde + kb] - 127) : 1.f;
  };
  if (m_lo < m_hi) load(m_lo);
  for (int64_t m = m_lo; m < m_hi; m += STEP) {
    __syncthreads();                                   // the tiles of the step before have been read
    {
      unsigned* d = reinterpret_cast<unsigned*>(s_x + sr * PITCH + sc);
      const unsigned c[4] = {xv.x, xv.y, xv.z, xv.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        d[2 * i] = decode2<FMT>(c[i], scale, false);
        d[2 * i + 1] = decode2<FMT>(c[i], scale, true);
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) bias[i] += gv[i];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      unsigned* d = reinterpret_cast<unsigned*>(s_mem + p * PLANE + sr * PITCH + sc);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = pack_hi(gv[2 * i], gv[2 * i + 1]);
      if (p + 1 < P) {
#pragma unroll
        for (int i = 0; i < 16; ++i) gv[i] -= head(gv[i]);
      }
    }
    __syncthreads();
    if (m + STEP < m_hi) load(m + STEP);
#pragma unroll
    for (int h = 0; h < STEP; h += 16) {
      bf16x8 x[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) x[j] = column8(s_x, h, wk + j * 32, lane);
#pragma unroll
      for (int p = P - 1; p >= 0; --p)                 // small pieces first
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bf16x8 a = column8(s_mem + p * PLANE, h, wn + i * 32, lane);
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, x[j], acc[i][j], 0, 0, 0);
        }
    }
  }
  // a lane holds one column k of 16 rows n of each 32 x 32 tile
  float* part = o.splits > 1 ? o.part + (int64_t)split * (o.N * o.K + o.N) : nullptr;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t k = k0 + wk + j * 32 + (lane & 31);
    if (k >= o.K) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t n = n0 + wn + i * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
        if (n >= o.N) continue;
        if (part) part[n * o.K + k] = acc[i][j][r];
        else store_param(o.dW, o.otype, n * o.K + k, acc[i][j][r]);
      }
  }
  if (!sums) return;
  __syncthreads();
  float* s_b = reinterpret_cast<float*>(s_mem);        // [32][128]: 16 KiB of the planes' 20 or more
#pragma unroll
  for (int i = 0; i < 16; ++i) s_b[sr * TN + sc + i] = bias[i];
  __syncthreads();
  if (threadIdx.x >= TN || n0 + threadIdx.x >= o.N) return;
  float t = 0.f;
  for (int i = 0; i < STEP; ++i) t += s_b[i * TN + threadIdx.x];
  if (part) part[o.N * o.K + n0 + threadIdx.x] = t;
  else store_param(o.db, o.otype, n0 + threadIdx.x, t);
}

__global__ void __launch_bounds__(WG)
wgrad8_reduce_kernel(int64_t NK, int64_t N, int splits, const float* __restrict__ part, void* __restrict__ dW,
                     void* __restrict__ db, int32_t otype) {
  const int64_t i = (int64_t)blockIdx.x * WG + threadIdx.x, total = NK + (db ? N : 0);
  if (i >= total) return;
  float t = 0.f;
  for (int s = 0; s < splits; ++s) t += part[(int64_t)s * (NK + N) + i];
  if (i < NK) store_param(dW, otype, i, t);
  else store_param(db, otype, i - NK, t);
}

// Row ranges: as many as give every CU two workgroups, none shorter than 128 rows
int split_count(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = cdiv(N, TN) * cdiv(K, TK);
  int64_t s = cdiv(512, tiles);
  if (s > cdiv(M, 128)) s = cdiv(M, 128);
  return (int)(s < 1 ? 1 : s);
}

bool wgrad_ok(int64_t M, int64_t N, int64_t K) { return rows_ok(M, K) && N >= 1 && N < (1ll << 24); }

template <int FMT, typename G>
int launch(Job& o, hipStream_t stream) {
  constexpr int lds = (PIECES<G> + 1) * PLANE * 2;
  const int64_t grid = (int64_t)o.tiles_n * o.tiles_k * o.splits;
  if (grid >= (1ll << 31)) { set_error("ganet_wgrad8: too many tiles"); return 4; }
  hipLaunchKernelGGL((wgrad8_kernel<FMT, G>), dim3((unsigned)grid), dim3(WG), lds, stream, o);
  if (o.splits > 1) {
    const int64_t total = o.N * o.K + (o.db ? o.N : 0);
    hipLaunchKernelGGL(wgrad8_reduce_kernel, dim3((unsigned)cdiv(total, WG)), dim3(WG), 0, stream, o.N * o.K, o.N, o.splits, o.part,
                       o.dW, o.db, o.otype);
  }
  return check_hip(hipGetLastError(), "ganet_wgrad8");
}

}  // namespace
}  // namespace ganet

using namespace ganet;

extern "C" {

size_t ganet_wgrad8_workspace(int64_t M, int64_t N, int64_t K, int32_t gtype) {
  if (!wgrad_ok(M, N, K) || !type_ok(gtype)) return 0;
  const int s = split_count(M, N, K);
  return s > 1 ? (size_t)s * (size_t)(N * K + N) * sizeof(float) : 0;
}

int ganet_wgrad8(int64_t M, int64_t N, int64_t K, int32_t fmt, int32_t gtype, const void* g, int64_t ldg, const void* codes,
                 int64_t ldc, const uint8_t* exps, int64_t lde, void* dW, void* db, int32_t otype, void* workspace,
                 size_t workspace_bytes, void* stream_) {
  if (!wgrad_ok(M, N, K) || (fmt != GANET_E4M3 && fmt != GANET_E5M2) || !type_ok(gtype) || !type_ok(otype)) {
    set_error("ganet_wgrad8: unsupported M=%lld N=%lld K=%lld format=%d types=%d,%d", (long long)M, (long long)N, (long long)K, fmt,
              gtype, otype);
    return 4;
  }
  if (!dW || (M > 0 && (!g || (ldg < N && M > 1) || !codes || !exps || ldc % 16 || ldc < pad16(K) || lde % 4 || lde < cdiv(K, BLOCK) ||
                        (reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(exps) & 3))) ||
      workspace_bytes < ganet_wgrad8_workspace(M, N, K, gtype) || (ganet_wgrad8_workspace(M, N, K, gtype) && !workspace)) {
    set_error("ganet_wgrad8: NULL or misaligned argument, a row stride or the workspace too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  Job o{M, N, K, g, ldg, static_cast<const uint8_t*>(codes), ldc, exps, lde, dW, db, otype, static_cast<float*>(workspace),
        split_count(M, N, K), 0, (int)cdiv(N, TN), (int)cdiv(K, TK)};
  o.rows = cdiv(cdiv(M, o.splits), STEP) * STEP;
  GANET_BY_TYPE(gtype, T, return fmt == GANET_E4M3 ? launch<GANET_E4M3, T>(o, stream) : launch<GANET_E5M2, T>(o, stream));
}

}  // extern "C"
