// ganet_gemm8.hip — matrix products of 8-bit floating point with a power of two for each block of 128 (include/ganet.h: ganet_gemm8).
//
//   y[m, n] = sum_kb 2^(ex[m, kb] + ew[n / 128, kb]) sum_{k in block kb} x[m, k] w[n, k] + bias[n]
//
// The scaled matrix instructions (v_mfma_scale_f32_*_f8f6f4) multiply 64 or 128 codes at a time and take a biased exponent per
// lane and operand: a power of two per block of 128 costs no vector instruction, where an arbitrary fp32 scale would cost an
// accumulator update per block. Products of codes are exact; sums are fp32; y is rounded once.
#include "ganet_rows8.h"

namespace ganet {
using namespace rows8;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ uint4 g_zeros[1];        // what lanes past the end of a row read

__device__ __forceinline__ i32x8 join(const uint4& a, const uint4& b) {
  i32x8 r;
  r[0] = (int)a.x; r[1] = (int)a.y; r[2] = (int)a.z; r[3] = (int)a.w;
  r[4] = (int)b.x; r[5] = (int)b.y; r[6] = (int)b.z; r[7] = (int)b.w;
  return r;
}

struct Operands {
  int64_t M, N, K;
  const uint8_t* x; int64_t ldx; const uint8_t* ex; int64_t ldex;
  const uint8_t* w; int64_t ldw; const uint8_t* ew; int64_t ldew;
  const void* bias; int32_t btype; void* y; int64_t ldy;
};

// ------------------------------------------------------------------------------------------------ tiles through LDS
// A workgroup of four waves computes 64 MT x 64 NT of y, a wave 32 MT x 32 NT. One step is one block of 128 codes: its rows go
// from global memory straight into LDS (16 bytes per lane, no registers), the next step's while this one is multiplied. A row is
// 128 bytes = 8 chunks of 16; chunk c of row r lies at position c ^ ((r >> 1) & 7), so that the 16 rows that a quarter of a wave
// reads at once lie in 16 different 16-byte columns of LDS. The instruction writes lanes in order, so the swizzle is
// in the global address that a lane fetches.
template <int ROWS>
__device__ __forceinline__ void stage(const uint8_t* __restrict__ src, int64_t ld, int64_t r0, int64_t rows, int64_t k0,
                                      int chunks, uint8_t* lds) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < ROWS / 32; ++i) {
    const int rb = (i * 4 + wave) * 8;                       // this instruction's eight rows
    const int r = rb + (lane >> 3);
    const int c = (lane & 7) ^ ((r >> 1) & 7);
    const int64_t row = r0 + r < rows ? r0 + r : rows - 1;   // rows past the end: results nobody stores
    const uint8_t* p = c < chunks ? src + row * ld + k0 + c * 16 : reinterpret_cast<const uint8_t*>(g_zeros);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)p,
                                     (__attribute__((address_space(3))) unsigned*)(lds + rb * 128), 16, 0, 0);
  }
}

__device__ __forceinline__ i32x8 fragment(const uint8_t* lds, int row0, int lane, int half) {
  const int r = row0 + (lane & 31), c = half * 4 + (lane >> 5) * 2, sw = (r >> 1) & 7;
  const uint4 a = *reinterpret_cast<const uint4*>(lds + r * 128 + ((c ^ sw) * 16));
  const uint4 b = *reinterpret_cast<const uint4*>(lds + r * 128 + (((c + 1) ^ sw) * 16));
  return join(a, b);
}

template <int FMT, int MT, int NT, typename Y>
__global__ void __launch_bounds__(256)
gemm8_tile_kernel(Operands o, int tiles_m, int tiles_n) {
  constexpr int TM = 64 * MT, TN = 64 * NT, BYTES = (TM + TN) * 128;
  extern __shared__ __align__(16) uint8_t s_tiles[];
  // Workgroups go round the 8 XCDs in turn: give each XCD one run of tiles (its own L2 sees neighbouring rows and columns), and
  // inside a run walk 8 tiles down before the next column.
  const int T = tiles_m * tiles_n, q = T / 8, rem = T % 8, xcd = blockIdx.x % 8;
  const int t = xcd * q + (xcd < rem ? xcd : rem) + blockIdx.x / 8;
  const int group = t / (8 * tiles_n), gm = min(8, tiles_m - group * 8), in = t - group * 8 * tiles_n;
  const int64_t m0 = (int64_t)(group * 8 + in % gm) * TM, n0 = (int64_t)(in / gm) * TN;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wm = (wave & 1) * 32 * MT, wn = (wave >> 1) * 32 * NT;
  const int64_t kend = (o.K + 15) / 16 * 16;
  const int KB = (int)((o.K + BLOCK - 1) / BLOCK);

  f32x16 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][i][r] = 0.f;

  auto fetch = [&](int kb) {
    uint8_t* lds = s_tiles + (kb & 1) * BYTES;
    const int64_t k0 = (int64_t)kb * BLOCK;
    const int chunks = (int)min((int64_t)8, (kend - k0) / 16);
    stage<TM>(o.x, o.ldx, m0, o.M, k0, chunks, lds);
    stage<TN>(o.w, o.ldw, n0, o.N, k0, chunks, lds + TM * 128);
  };
  const uint8_t* exr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) exr[i] = o.ex + min(m0 + wm + i * 32 + (lane & 31), o.M - 1) * o.ldex;
  const uint8_t* ewr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) ewr[j] = o.ew + min(n0 + wn + j * 32, o.N - 1) / BLOCK * o.ldew;

  fetch(0);
  for (int kb = 0; kb < KB; ++kb) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();                       // step kb has landed for every wave, and nobody reads the other buffer any more
    if (kb + 1 < KB) fetch(kb + 1);
    const uint8_t* lds = s_tiles + (kb & 1) * BYTES;
    int sx[MT], sw[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = exr[i][kb];
#pragma unroll
    for (int j = 0; j < NT; ++j) sw[j] = ewr[j][kb];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      i32x8 a[MT], b[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) a[i] = fragment(lds, wm + i * 32, lane, half);
#pragma unroll
      for (int j = 0; j < NT; ++j) b[j] = fragment(lds + TM * 128, wn + j * 32, lane, half);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
          acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a[i], acc[j][i], GANET_E4M3, FMT, 0, sw[j], 0, sx[i]);
    }
  }
  // a lane holds one row m and, four at a time, consecutive columns n
  Y* y = static_cast<Y*>(o.y);
#pragma unroll
  for (int j = 0; j < NT; ++j) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int64_t n = n0 + wn + j * 32 + g * 8 + (lane >> 5) * 4;
      float bias[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) bias[r] = (o.bias && n + r < o.N) ? load_param(o.bias, o.btype, n + r) : 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + wm + i * 32 + (lane & 31);
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = acc[j][i][g * 4 + r] + bias[r];
        if (m < o.M) store_n(y + m * o.ldy + n, o.N - n, v);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// The weight's codes are the traffic: every wave streams its share of the blocks of 16 weight rows straight from global memory
// into matrix operands (a lane: 32 codes of one row), the eight waves' sums meet in LDS.
constexpr int FEW_WAVES = 8, FEW_UNROLL = 4;

template <int FMT, int MT, typename Y>
__global__ void __launch_bounds__(64 * FEW_WAVES)
gemm8_few_kernel(Operands o) {
  __shared__ f32x4 s_acc[FEW_WAVES][MT][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t kend = (o.K + 15) / 16 * 16;
  const int KB = (int)((o.K + BLOCK - 1) / BLOCK);
  const uint8_t* wr = o.w + min(n0 + r, o.N - 1) * o.ldw + q * 32;
  const uint8_t* ew = o.ew + n0 / BLOCK * o.ldew;
  const uint8_t *xr[MT], *ex[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = min((int64_t)(i * 16 + r), o.M - 1);
    xr[i] = o.x + m * o.ldx + q * 32;
    ex[i] = o.ex + m * o.ldex;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint4 zero = make_uint4(0, 0, 0, 0);
  for (int kb0 = wave; kb0 < KB; kb0 += FEW_WAVES * FEW_UNROLL) {
    uint4 w[FEW_UNROLL][2], x[FEW_UNROLL][MT][2];
    int sw[FEW_UNROLL], sx[FEW_UNROLL][MT];
#pragma unroll
    for (int u = 0; u < FEW_UNROLL; ++u) {
      const int kb = kb0 + u * FEW_WAVES;
      const int64_t k = (int64_t)kb * BLOCK;
      const bool lo = kb < KB && k + q * 32 < kend, hi = kb < KB && k + q * 32 + 16 < kend;
      w[u][0] = lo ? *reinterpret_cast<const uint4*>(wr + k) : zero;
      w[u][1] = hi ? *reinterpret_cast<const uint4*>(wr + k + 16) : zero;
      sw[u] = kb < KB ? ew[kb] : 127;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        x[u][i][0] = lo ? *reinterpret_cast<const uint4*>(xr[i] + k) : zero;
        x[u][i][1] = hi ? *reinterpret_cast<const uint4*>(xr[i] + k + 16) : zero;
        sx[u][i] = kb < KB ? ex[i][kb] : 127;
      }
    }
#pragma unroll
    for (int u = 0; u < FEW_UNROLL; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(join(w[u][0], w[u][1]), join(x[u][i][0], x[u][i][1]), acc[i],
                                                                  GANET_E4M3, FMT, 0, sw[u], 0, sx[u][i]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) s_acc[wave][i][lane] = acc[i];
  __syncthreads();
  if (threadIdx.x >= MT * 64) return;
  const int i = threadIdx.x >> 6;
  f32x4 t = s_acc[0][i][lane];
#pragma unroll
  for (int v = 1; v < FEW_WAVES; ++v) t += s_acc[v][i][lane];
  const int64_t m = i * 16 + r, n = n0 + q * 4;
  if (m >= o.M) return;
  float v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = t[c] + ((o.bias && n + c < o.N) ? load_param(o.bias, o.btype, n + c) : 0.f);
  store_n(static_cast<Y*>(o.y) + m * o.ldy + n, o.N - n, v);
}

template <int FMT, int MT, int NT, typename Y>
int launch_tile(const Operands& o, hipStream_t stream) {
  static PerDeviceFlag ready;
  constexpr int lds = 2 * 64 * (MT + NT) * 128;
  auto k = gemm8_tile_kernel<FMT, MT, NT, Y>;
  if (!ready) {
    const int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                             "ganet_gemm8");
    if (rc) return rc;
    ready = true;
  }
  const int64_t tm = cdiv(o.M, 64 * MT), tn = cdiv(o.N, 64 * NT);
  if (tm * tn >= (1ll << 30)) { set_error("ganet_gemm8: too many tiles"); return 4; }
  hipLaunchKernelGGL(k, dim3((unsigned)(tm * tn)), dim3(256), lds, stream, o, (int)tm, (int)tn);
  return check_hip(hipGetLastError(), "ganet_gemm8");
}

template <int FMT, typename Y>
int launch(const Operands& o, hipStream_t stream) {
  if (o.M <= 32) {
    const dim3 grid((unsigned)cdiv(o.N, 16));
    if (o.M <= 16) hipLaunchKernelGGL((gemm8_few_kernel<FMT, 1, Y>), grid, dim3(64 * FEW_WAVES), 0, stream, o);
    else hipLaunchKernelGGL((gemm8_few_kernel<FMT, 2, Y>), grid, dim3(64 * FEW_WAVES), 0, stream, o);
    return check_hip(hipGetLastError(), "ganet_gemm8");
  }
  if (cdiv(o.M, 256) * cdiv(o.N, 256) >= 256) return launch_tile<FMT, 4, 4, Y>(o, stream);
  return launch_tile<FMT, 2, 2, Y>(o, stream);
}

}  // namespace
}  // namespace ganet

using namespace ganet;

extern "C" {

size_t ganet_gemm8_workspace(int64_t M, int64_t N, int64_t K) { return 0; }

int ganet_gemm8(int64_t M, int64_t N, int64_t K, int32_t fmt, const void* codes, int64_t ldc, const uint8_t* exps, int64_t lde,
                const void* wcodes, int64_t ldwc, const uint8_t* wexps, int64_t ldwe, const void* bias, int32_t btype, void* y,
                int64_t ldy, int32_t ytype, void* workspace, size_t workspace_bytes, void* stream_) {
  if (!rows_ok(M, K) || N < 1 || N >= (1ll << 24) || (fmt != GANET_E4M3 && fmt != GANET_E5M2) || !type_ok(ytype) || !type_ok(btype)) {
    set_error("ganet_gemm8: unsupported M=%lld N=%lld K=%lld format=%d types=%d,%d", (long long)M, (long long)N, (long long)K, fmt,
              ytype, btype);
    return 4;
  }
  if (M == 0) return 0;
  const auto ok = [&](const void* c, int64_t ld, const uint8_t* e, int64_t le) {
    return c && e && ld % 16 == 0 && ld >= pad16(K) && (reinterpret_cast<uintptr_t>(c) & 15) == 0 && le % 4 == 0 &&
           le >= cdiv(K, BLOCK) && (reinterpret_cast<uintptr_t>(e) & 3) == 0;
  };
  if (!y || (ldy < N && M > 1) || !ok(codes, ldc, exps, lde) || !ok(wcodes, ldwc, wexps, ldwe)) {
    set_error("ganet_gemm8: NULL or misaligned argument, or a row stride too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const Operands o{M, N, K, static_cast<const uint8_t*>(codes), ldc, exps, lde, static_cast<const uint8_t*>(wcodes), ldwc, wexps,
                   ldwe, bias, btype, y, ldy};
  GANET_BY_TYPE(ytype, T, return fmt == GANET_E4M3 ? launch<GANET_E4M3, T>(o, stream) : launch<GANET_E5M2, T>(o, stream));
}

}  // extern "C"
