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

constexpr int WG = 256, STEP = 32;
// LDS row of a plane: its columns and 64 bytes more, so that the four rows that a 16-lane group reads start in four different
// 64-byte columns
constexpr int pitch(int cols) { return cols + 32; }

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
template <int PITCH>
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

struct Where { int tn, tk, split; };

// A workgroup of four waves computes 64 T x 64 T of dW over its range of rows, a wave 32 T x 32 T. A step is 32 rows: thread t brings row
// t / 8, 8 T columns of g and of x, from global memory into registers two steps ahead, and as bf16 into one of two LDS buffers one
// step ahead. A step is multiplied in 2 P parts (16 rows, one piece of g); the fragments of the next part are read before a
// part is multiplied, those of the next step's first part behind the step's one barrier, which stands before its last part: neither
// memory nor LDS latency stands between two multiplications.
// INSIDE: the tile ends before column N of g (vectors of 8; else element by element).
template <int FMT, typename G, int T, bool INSIDE>
__device__ __forceinline__ void wgrad8_tile(const Job& o, const Where& w, unsigned short* s_mem) {
  constexpr int P = PIECES<G>, COLS = 64 * T, PITCH = pitch(COLS), PLANE = STEP * PITCH, BUF = (P + 1) * PLANE;
  constexpr int GV = 8, GC = COLS / 64;                        // g: GC vectors of 8 elements, 64 columns apart
  constexpr int XC = COLS / 128;                               // x: XC vectors of 16 codes, one per 128 columns
  const int64_t n0 = (int64_t)w.tn * COLS, k0 = (int64_t)w.tk * COLS;
  const int split = w.split;
  const int64_t m_lo = split * o.rows, m_hi = min(m_lo + o.rows, o.M);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wn = (wave & 1) * 32 * T, wk = (wave >> 1) * 32 * T;
  const int sr = threadIdx.x >> 3, st = threadIdx.x & 7;
  const int64_t kend = (o.K + 15) / 16 * 16;
  const G* g = static_cast<const G*>(o.g);

  f32x16 acc[T][T];
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const bool sums = k0 == 0 && o.db;
  float bias[GC][GV] = {};

  struct Raw { G g[GC][GV]; uint4 x[XC]; int e[XC]; bool live; };
  auto load = [&](Raw& v, int64_t m) {
    // rows past the range and columns past the matrix load the last ones instead and become zero when they are put (no branch: a
    // value that two paths may have loaded is waited for where they meet)
    const int left = (int)min(m_hi - m, (int64_t)STEP);
    v.live = sr < left;
    // a uniform base and 32-bit offsets (a step's rows span less than 2^31 bytes)
    const int64_t m_in = left > 0 ? m : m_hi - 1;
    const unsigned row = left > 0 ? min(sr, left - 1) : 0;
    const char* gb = reinterpret_cast<const char*>(g + m_in * o.ldg + n0);
    const unsigned go = (row * (unsigned)o.ldg + st * GV) * (unsigned)sizeof(G);
#pragma unroll
    for (int i = 0; i < GC; ++i) {
      if constexpr (INSIDE) __builtin_memcpy(v.g[i], gb + i * 64 * sizeof(G) + go, sizeof(v.g[i]));
      else {
        const int last = (int)(o.N - 1 - n0), n = st * GV + i * 64;
#pragma unroll
        for (int j = 0; j < GV; ++j)
          v.g[i][j] = *reinterpret_cast<const G*>(gb + (row * (unsigned)o.ldg + min(n + j, last)) * (unsigned)sizeof(G));
      }
    }
    const uint8_t *xb = o.codes + m_in * o.ldc + k0, *eb = o.exps + m_in * o.lde + k0 / BLOCK;
    const int kleft = (int)min(kend - k0, (int64_t)COLS);
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const int k = min(i * 128 + st * 16, kleft - 16);
      v.x[i] = *reinterpret_cast<const uint4*>(xb + (row * (unsigned)o.ldc + k));
      v.e[i] = eb[row * (unsigned)o.lde + k / BLOCK];
    }
  };
  auto put = [&](const Raw& v, int buf) {
    unsigned short* base = s_mem + buf * BUF;
#pragma unroll
    for (int i = 0; i < XC; ++i) {
      const unsigned in = v.live && k0 + i * 128 + st * 16 < kend ? ~0u : 0u;
      const float scale = pow2(v.e[i] - 127);
      const unsigned c[4] = {v.x[i].x & in, v.x[i].y & in, v.x[i].z & in, v.x[i].w & in};
      uint4* d = reinterpret_cast<uint4*>(base + P * PLANE + sr * PITCH + i * 128 + st * 16);
      d[0] = make_uint4(decode2<FMT>(c[0], scale, false), decode2<FMT>(c[0], scale, true), decode2<FMT>(c[1], scale, false),
                        decode2<FMT>(c[1], scale, true));
      d[1] = make_uint4(decode2<FMT>(c[2], scale, false), decode2<FMT>(c[2], scale, true), decode2<FMT>(c[3], scale, false),
                        decode2<FMT>(c[3], scale, true));
    }
#pragma unroll
    for (int i = 0; i < GC; ++i) {
      uint4* d = reinterpret_cast<uint4*>(base + sr * PITCH + i * 64 + st * GV);
      float f[GV];
#pragma unroll
      for (int j = 0; j < GV; ++j)
        f[j] = v.live && (INSIDE || n0 + st * GV + i * 64 + j < o.N) ? (float)v.g[i][j] : 0.f;
#pragma unroll
      for (int j = 0; j < GV; ++j) bias[i][j] += f[j];         // (used by the first column of tiles; a branch here costs more)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        *reinterpret_cast<uint4*>(reinterpret_cast<unsigned short*>(d) + p * PLANE) =
            make_uint4(pack_hi(f[0], f[1]), pack_hi(f[2], f[3]), pack_hi(f[4], f[5]), pack_hi(f[6], f[7]));
        if (p + 1 < P) {
#pragma unroll
          for (int j = 0; j < GV; ++j) f[j] -= head(f[j]);
        }
      }
    }
  };
  // part q of a step: rows 16 (q / P) .., piece P - 1 - q % P of g (small pieces first)
  bf16x8 a[2][T], x[2][T];
  auto read = [&](int buf, int q) {
    const unsigned short* base = s_mem + buf * BUF;
    const int h = q / P * 16, p = P - 1 - q % P;
#pragma unroll
    for (int i = 0; i < T; ++i) a[q & 1][i] = column8<PITCH>(base + p * PLANE, h, wn + i * 32, lane);
    if (q % P == 0) {
#pragma unroll
      for (int j = 0; j < T; ++j) x[q / P][j] = column8<PITCH>(base + P * PLANE, h, wk + j * 32, lane);
    }
  };
  auto multiply = [&](int q) {
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int j = 0; j < T; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[q & 1][i], x[q / P][j], acc[i][j], 0, 0, 0);
  };
  auto step = [&](Raw& there, Raw& far, int buf, int64_t m) {
    load(far, m + 2 * STEP);
#pragma unroll
    for (int q = 0; q < 2 * P; ++q) {
      if (q + 1 < 2 * P) read(buf, q + 1);
      else {
        __syncthreads();                     // the next step's tiles stand, and this step's have been read
        read(buf ^ 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      multiply(q);
      if (q == 0) {                          // (between the multiplications)
        put(there, buf ^ 1);
#pragma unroll
        for (int i = 0; i < T * T; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);             // a matrix instruction
          __builtin_amdgcn_sched_group_barrier(0x002, 48 * P / T, 0);    // vector instructions
          __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);             // an LDS write
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (m_lo < m_hi) {
    Raw va, vb;
    load(va, m_lo);
    load(vb, m_lo + STEP);
    put(va, 0);
    __syncthreads();
    read(0, 0);
    for (int64_t m = m_lo; m < m_hi; m += 2 * STEP) {          // (an odd last step multiplies zeros)
      step(vb, va, 0, m);
      step(va, vb, 1, m + STEP);
    }
    __syncthreads();
  }
  // A lane holds one column k of 16 rows n of each 32 x 32 tile: an instruction stores 32 adjacent columns of two rows. Offsets
  // inside the tile fit 32 bits (K < 2^22).
  float* part = o.splits > 1 ? o.part + (int64_t)split * (o.N * o.K + o.N) : nullptr;
  auto store = [&](auto* out) {
    out += n0 * o.K + k0;
    const unsigned K = (unsigned)o.K, rows = (unsigned)min((int64_t)COLS, o.N - n0), cols = (unsigned)min((int64_t)COLS, o.K - k0);
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const unsigned n = wn + i * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
        const unsigned at = n * K + wk + (lane & 31);
#pragma unroll
        for (int j = 0; j < T; ++j)
          if (n < rows && wk + j * 32 + (lane & 31) < cols) out[at + j * 32] = acc[i][j][r];
        __builtin_amdgcn_sched_barrier(0);                     // one row's results in registers at a time
      }
  };
  if (part) store(part);
  else GANET_BY_TYPE(o.otype, O, store(static_cast<O*>(o.dW)));
  if (!sums) return;
  float* s_b = reinterpret_cast<float*>(s_mem);                // [32][COLS]: the buffers are free behind the last barrier
#pragma unroll
  for (int i = 0; i < GC; ++i)
#pragma unroll
    for (int j = 0; j < GV; ++j) s_b[sr * COLS + i * 64 + st * GV + j] = bias[i][j];
  __syncthreads();
  if (threadIdx.x >= COLS || n0 + threadIdx.x >= o.N) return;
  float t = 0.f;
  for (int i = 0; i < STEP; ++i) t += s_b[i * COLS + threadIdx.x];
  if (part) part[o.N * o.K + n0 + threadIdx.x] = t;
  else store_param(o.db, o.otype, n0 + threadIdx.x, t);
}

template <int FMT, typename G, int T>
__global__ void __launch_bounds__(WG, T == 4 ? 1 : 2)
wgrad8_kernel(Job o) {
  extern __shared__ __align__(16) unsigned short s_mem[];      // two buffers: the planes of g, one of x
  // Workgroups go round the 8 XCDs in turn: give each XCD one run of tiles, walked 4 tiles of n before the next tile of k, so that its 32
  // CUs read 4 strips of g and 8 of x through their L2 (where workgroup i takes tile i: 16 strips of g and 2 of x).
  const int tiles = o.tiles_n * o.tiles_k, T0 = tiles * o.splits, q = T0 / 8, rem = T0 % 8, xcd = blockIdx.x % 8;
  const int t = xcd * q + (xcd < rem ? xcd : rem) + blockIdx.x / 8, in_split = t % tiles;
  const int group = in_split / (4 * o.tiles_k), gn = min(4, o.tiles_n - group * 4), in = in_split - group * 4 * o.tiles_k;
  // (in scalar registers: the divisions are done in vector ones)
  const Where w{__builtin_amdgcn_readfirstlane(group * 4 + in % gn), __builtin_amdgcn_readfirstlane(in / gn),
                __builtin_amdgcn_readfirstlane(t / tiles)};
  if ((int64_t)(w.tn + 1) * 64 * T <= o.N) wgrad8_tile<FMT, G, T, true>(o, w, s_mem);
  else wgrad8_tile<FMT, G, T, false>(o, w, s_mem);
}

// The ranges' partial sums, added in a fixed order: a workgroup takes 64 adjacent results, its four waves a quarter of the ranges each.
__global__ void __launch_bounds__(WG)
wgrad8_reduce_kernel(int64_t NK, int64_t N, int splits, const float* __restrict__ part, void* __restrict__ dW,
                     void* __restrict__ db, int32_t otype) {
  __shared__ float s_t[WG];
  const int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63), total = NK + (db ? N : 0);
  const int wave = threadIdx.x >> 6;
  float t = 0.f;
  if (i < total) {
    const float* p = part + i;
#pragma unroll 8
    for (int s = wave; s < splits; s += 4) t += p[(int64_t)s * (NK + N)];
  }
  s_t[threadIdx.x] = t;
  __syncthreads();
  if (wave || i >= total) return;
  t = (s_t[threadIdx.x] + s_t[threadIdx.x + 64]) + (s_t[threadIdx.x + 128] + s_t[threadIdx.x + 192]);
  if (i < NK) store_param(dW, otype, i, t);
  else store_param(db, otype, i - NK, t);
}

// The tile: 256 x 256 (one workgroup per CU) where that still gives every CU a tile and a range of at least 256 rows, else 128 x 128.
// The ranges: as many as give every CU a workgroup (two of the small ones), none shorter than 128 rows.
struct Plan { int T; int64_t tiles_n, tiles_k; int splits; int64_t rows; };
Plan make_plan(int64_t M, int64_t N, int64_t K) {
  Plan p;
  const int64_t big = cdiv(N, 256) * cdiv(K, 256);
  p.T = (N > 128 && K > 128 && big * cdiv(M, 256) >= 256) ? 4 : 2;
  p.tiles_n = cdiv(N, 64 * p.T);
  p.tiles_k = cdiv(K, 64 * p.T);
  const int64_t tiles = p.tiles_n * p.tiles_k, want = p.T == 4 ? 256 : 512;
  int64_t s = tiles >= want ? 1 : want / tiles;
  if (s > cdiv(M, 128)) s = cdiv(M, 128);
  p.splits = (int)(s < 1 ? 1 : s);
  p.rows = cdiv(cdiv(M, p.splits), STEP) * STEP;
  return p;
}

bool wgrad_ok(int64_t M, int64_t N, int64_t K) { return rows_ok(M, K) && K < (1ll << 22) && N >= 1 && N < (1ll << 24); }

template <int FMT, typename G, int T>
int launch_tile(const Job& o, hipStream_t stream) {
  static PerDeviceFlag ready;
  constexpr int lds = 2 * (PIECES<G> + 1) * STEP * pitch(64 * T) * 2;
  auto k = wgrad8_kernel<FMT, G, T>;
  if (!ready) {
    const int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                             "ganet_wgrad8");
    if (rc) return rc;
    ready = true;
  }
  const int64_t grid = (int64_t)o.tiles_n * o.tiles_k * o.splits;
  if (grid >= (1ll << 30)) { set_error("ganet_wgrad8: too many tiles"); return 4; }
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(WG), lds, stream, o);
  return check_hip(hipGetLastError(), "ganet_wgrad8");
}

template <int FMT, typename G>
int launch(const Job& o, int T, hipStream_t stream) {
  const int rc = T == 4 ? launch_tile<FMT, G, 4>(o, stream) : launch_tile<FMT, G, 2>(o, stream);
  if (rc || o.splits == 1) return rc;
  const int64_t total = o.N * o.K + (o.db ? o.N : 0);
  hipLaunchKernelGGL(wgrad8_reduce_kernel, dim3((unsigned)cdiv(total, 64)), dim3(WG), 0, stream, o.N * o.K, o.N, o.splits, o.part,
                     o.dW, o.db, o.otype);
  return check_hip(hipGetLastError(), "ganet_wgrad8");
}

}  // namespace
}  // namespace ganet

using namespace ganet;

extern "C" {

size_t ganet_wgrad8_workspace(int64_t M, int64_t N, int64_t K, int32_t gtype) {
  if (!wgrad_ok(M, N, K) || !type_ok(gtype)) return 0;
  const int s = make_plan(M, N, K).splits;
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
  const Plan p = make_plan(M, N, K);
  const Job o{M, N, K, g, ldg, static_cast<const uint8_t*>(codes), ldc, exps, lde, dW, db, otype, static_cast<float*>(workspace),
              p.splits, p.rows, (int)p.tiles_n, (int)p.tiles_k};
  GANET_BY_TYPE(gtype, T, return fmt == GANET_E4M3 ? launch<GANET_E4M3, T>(o, p.T, stream) : launch<GANET_E5M2, T>(o, p.T, stream));
}

}  // extern "C"
