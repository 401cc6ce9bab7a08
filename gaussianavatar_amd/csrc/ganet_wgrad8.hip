// ganet_wgrad8.hip — the weight gradient of a layer whose input is kept in 8 bits (include/ganet.h: ganet_wgrad8).
//
//   dW[n, k] = sum_m g[m, n] 2^(e[m, k / 128]) code[m, k],   db[n] = sum_m g[m, n]
//
// The sum runs over the rows, along which the powers of two change, so the 8-bit matrix instructions (one scale per 32 products of
// a lane) do not apply to it as it lies. Codes become bf16 instead: 4 significand bits and a power of two fit bf16 exactly, so the kept input
// enters with no further rounding (at half its size, halves below 2^-133 lost, and the results doubled: half_scale()). g enters with all its bits as 1 (bf16), 2 (fp16) or 3 (fp32) bf16 pieces, of
// which a piece below bf16's smallest number, 2^-133, is lost; sums are fp32.
//
// What bounds it: for wide layers the matrix instructions (P products per product of the layer), for the 128 columns of a point decoder
// the reads (262144 x 128 x 128 fp32, 169 MB: 45 us with the reduction, 33 of them at a copy's rate).
// Both operands need the row index as the matrix instruction's k: tiles lie in LDS as they lie in memory ([row][column], bf16) and
// ds_read_b64_tr_b16 hands each lane four rows of its column.
#include "ganet_rows8.h"

namespace ganet {
using namespace rows8;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int STEP = 32, REDUCE_WG = 256;
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
  void* dW; void* db; int32_t otype, btype; float* part; int splits; int64_t rows; int tiles_n, tiles_k;
};

struct Where { int tn, tk, split; };

// A workgroup computes a tile of dW, COLS x COLS, over its range of rows; a wave 32 TI x 32 TJ of it. A step is 32 rows: thread t brings row
// t / TPR, 16 (8) columns of g and of x, from global memory into registers two steps ahead, and as bf16 into one of two LDS buffers
// one step ahead, so that one barrier per step is enough and a load has two steps to arrive. Two waves stand on a SIMD: one converts,
// reads and writes LDS while the other one's matrix instructions run. 8192 x 4096 x 4096 bf16: 274 us, 1.0 PFLOP/s (a large library
// product reaches 1.13). With one wave on a SIMD, four of 128 x 128 in a workgroup, which have a third less to read from LDS, 320 us (262144 x 128 x 128 fp32 47 us against 45).
// INSIDE: no vector of 8 columns crosses column N of g (one behind it is read as the last one); else element by element
// (300000 x 64 x 64 bf16: 29 us against 48). In 256 x 256 tiles it is that form, run by the tiles past column N alone, that needs more registers than there are
// (fp32 56 spilled, fp16 44, bf16 2); the other one has none spilled.
template <int TILE> struct Form;
template <> struct Form<256> { static constexpr int TI = 4, TJ = 2, WN = 2, WAVES = 8; };
template <> struct Form<128> { static constexpr int TI = 2, TJ = 1, WN = 2, WAVES = 8; };
template <int FMT, typename G, int COLS, bool INSIDE>
__device__ __forceinline__ void wgrad8_tile(const Job& o, const Where& w, unsigned short* s_mem) {
  typedef Form<COLS> F;
  constexpr int TI = F::TI, TJ = F::TJ;
  constexpr int P = PIECES<G>, PITCH = pitch(COLS), PLANE = STEP * PITCH, BUF = (P + 1) * PLANE;
  constexpr int PER = STEP * COLS / (64 * F::WAVES), GV = 8, GC = PER / GV, TPR = COLS / PER;    // g: GC vectors of 8 elements, COLS / GC apart
  typedef unsigned codes_t __attribute__((ext_vector_type(PER / 4)));
  const int64_t n0 = (int64_t)w.tn * COLS, k0 = (int64_t)w.tk * COLS;
  const int split = w.split;
  const int64_t m_lo = split * o.rows, m_hi = min(m_lo + o.rows, o.M);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wn = wave % F::WN * 32 * TI, wk = wave / F::WN * 32 * TJ;
  const int sr = threadIdx.x / TPR, st = threadIdx.x % TPR;
  const int64_t kend = (o.K + 15) / 16 * 16;
  const G* g = static_cast<const G*>(o.g);

  f32x16 acc[TI][TJ];
#pragma unroll
  for (int i = 0; i < TI; ++i)
#pragma unroll
    for (int j = 0; j < TJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const bool sums = k0 == 0 && o.db;
  float bias[GC][GV] = {};

  // Columns past the matrix load its last ones and give results that nobody stores. The last step loads the range's last 32 rows and
  // counts those that no step before it had (a range of fewer rows: its last row again and again); what does not count is
  // zeroed in x and in g: db adds g up, and an infinity of g that counts once must not meet a zero of x. Offsets inside a step's rows
  // are the same for every step and fit 32 bits: no branch and no address arithmetic in vector registers (a value that two paths may
  // have loaded is waited for where they meet).
  // (vectors of g are values, not memory: copied to memory and on, the compiler loads them again where they are put)
  typedef G vec __attribute__((ext_vector_type(8)));
  typedef G loose __attribute__((ext_vector_type(8), aligned(sizeof(G))));
  struct Raw { vec g[GC]; codes_t x; int e; bool live; };
  const unsigned lrow = (unsigned)min((int64_t)sr, m_hi - m_lo - 1);
  unsigned go[INSIDE ? 1 : GC * GV];
  if constexpr (INSIDE) go[0] = (lrow * (unsigned)o.ldg + (GC == 1 ? min(st * GV, (int)(o.N - n0) - GV) : st * GV)) * (unsigned)sizeof(G);
  else {
#pragma unroll
    for (int i = 0; i < GC * GV; ++i)
      go[i] = (lrow * (unsigned)o.ldg + min((int)(o.N - 1 - n0), i / GV * (COLS / GC) + st * GV + i % GV)) * (unsigned)sizeof(G);
  }
  const int xk = min(st * PER, (int)min(kend - k0, (int64_t)COLS) - PER);
  const unsigned xo = lrow * (unsigned)o.ldc + xk, eo = lrow * (unsigned)o.lde + xk / BLOCK;
  auto load = [&](Raw& v, int64_t m) {
    const int64_t at = max(m_lo, min(m, m_hi - STEP));
    v.live = at + sr >= m && at + sr < m_hi;
    const char* gb = reinterpret_cast<const char*>(g + at * o.ldg + n0);
#pragma unroll
    for (int i = 0; i < GC; ++i) {
      if constexpr (INSIDE) v.g[i] = *reinterpret_cast<const loose*>(gb + i * (COLS / GC) * sizeof(G) + go[0]);
      else {
#pragma unroll
        for (int j = 0; j < GV; ++j) v.g[i][j] = *reinterpret_cast<const G*>(gb + go[i * GV + j]);
      }
    }
    v.x = *reinterpret_cast<const codes_t*>(o.codes + at * o.ldc + k0 + xo);
    v.e = (o.exps + at * o.lde + k0 / BLOCK)[eo];
  };
  auto put = [&](const Raw& v, int buf) {
    unsigned short* base = s_mem + buf * BUF + sr * PITCH;
    const unsigned in = v.live ? ~0u : 0u;
    const float scale = half_scale(v.e);                      // (the results are doubled: store)
    uint4* d = reinterpret_cast<uint4*>(base + P * PLANE + st * PER);
#pragma unroll
    for (int i = 0; i < PER / 8; ++i) {
      const unsigned a = v.x[2 * i] & in, b = v.x[2 * i + 1] & in;
      d[i] = make_uint4(decode2<FMT>(a, scale, false), decode2<FMT>(a, scale, true), decode2<FMT>(b, scale, false),
                        decode2<FMT>(b, scale, true));
    }
#pragma unroll
    for (int i = 0; i < GC; ++i) {
      d = reinterpret_cast<uint4*>(base + i * (COLS / GC) + st * GV);
      float f[GV];
      if constexpr (P == 1) {                                  // bf16
        uint4 raw = __builtin_bit_cast(uint4, v.g[i]);
        raw = make_uint4(raw.x & in, raw.y & in, raw.z & in, raw.w & in);
        *d = raw;
        const vec masked = __builtin_bit_cast(vec, raw);
#pragma unroll
        for (int j = 0; j < GV; ++j) f[j] = (float)masked[j];
      } else {
#pragma unroll
        for (int j = 0; j < GV; ++j) f[j] = v.live ? (float)v.g[i][j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < GV; ++j) bias[i][j] += f[j];         // (used by the first column of tiles; a branch here costs more)
      if constexpr (P > 1) {
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
    }
  };
  auto step = [&](Raw& there, Raw& far, int buf, int64_t m) {
    load(far, m + 2 * STEP);
    const unsigned short* base = s_mem + buf * BUF;
    // groups of two fragments of g and TJ of x; the next group's g is read before a group is multiplied
    constexpr int GROUPS = P * TI / 2;
    bf16x8 a[2][2], x[TJ];
    auto read = [&](int n) {
      const int h = n / GROUPS * 16, p = P - 1 - n % GROUPS / (TI / 2), i = n % (TI / 2) * 2;        // small pieces first
      a[n & 1][0] = column8<PITCH>(base + p * PLANE, h, wn + i * 32, lane);
      a[n & 1][1] = column8<PITCH>(base + p * PLANE, h, wn + i * 32 + 32, lane);
    };
    auto readx = [&](int h) {
#pragma unroll
      for (int j = 0; j < TJ; ++j) x[j] = column8<PITCH>(base + P * PLANE, h, wk + j * 32, lane);
    };
    readx(0);
    read(0);
#pragma unroll
    for (int n = 0; n < 2 * GROUPS; ++n) {
      if (n + 1 < 2 * GROUPS) read(n + 1);
      const int i = n % (TI / 2) * 2;
#pragma unroll
      for (int j = 0; j < TJ; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[n & 1][0], x[j], acc[i][j], 0, 0, 0);
        acc[i + 1][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[n & 1][1], x[j], acc[i + 1][j], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (n + 1 == GROUPS) {
        readx(16);
        put(there, buf ^ 1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();                         // the next step's tiles stand, and this step's have been read
  };
  if (m_lo < m_hi) {
    Raw va, vb;
    load(va, m_lo);
    load(vb, m_lo + STEP);
    put(va, 0);
    __syncthreads();
    for (int64_t m = m_lo; m < m_hi; m += 2 * STEP) {          // (an odd last step multiplies zeros)
      step(vb, va, 0, m);
      step(va, vb, 1, m + STEP);
    }
  }
  // A lane holds one column k of 16 rows n of each 32 x 32 tile: an instruction stores 32 adjacent columns of two rows. Offsets
  // inside the tile fit 32 bits (K < 2^22).
  float* part = o.splits > 1 ? o.part + (int64_t)split * (o.N * o.K + o.N) : nullptr;
  auto store = [&](auto* out) {
    out += n0 * o.K + k0;
    const unsigned K = (unsigned)o.K, rows = (unsigned)min((int64_t)COLS, o.N - n0), cols = (unsigned)min((int64_t)COLS, o.K - k0);
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const unsigned n = wn + i * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
        const unsigned at = n * K + wk + (lane & 31);
#pragma unroll
        for (int j = 0; j < TJ; ++j)
          if (n < rows && wk + j * 32 + (lane & 31) < cols) out[at + j * 32] = 2.f * acc[i][j][r];
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
    for (int j = 0; j < GV; ++j) s_b[sr * COLS + i * (COLS / GC) + st * GV + j] = bias[i][j];
  __syncthreads();
  if (threadIdx.x >= COLS || n0 + threadIdx.x >= o.N) return;
  float t = 0.f;
  for (int i = 0; i < STEP; ++i) t += s_b[i * COLS + threadIdx.x];
  if (part) part[o.N * o.K + n0 + threadIdx.x] = t;
  else store_param(o.db, o.btype, n0 + threadIdx.x, t);
}

template <int FMT, typename G, int COLS>
__global__ void __launch_bounds__(64 * Form<COLS>::WAVES, 2)
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
  if ((int64_t)(w.tn + 1) * COLS <= o.N || (COLS == 128 && o.N % 8 == 0)) wgrad8_tile<FMT, G, COLS, true>(o, w, s_mem);
  else wgrad8_tile<FMT, G, COLS, false>(o, w, s_mem);
}

// The ranges' partial sums, added in a fixed order: a workgroup takes 64 adjacent results, its four waves a quarter of the ranges each.
__global__ void __launch_bounds__(REDUCE_WG)
wgrad8_reduce_kernel(int64_t NK, int64_t N, int splits, const float* __restrict__ part, void* __restrict__ dW,
                     void* __restrict__ db, int32_t otype, int32_t btype) {
  __shared__ float s_t[REDUCE_WG];
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
  else store_param(db, btype, i - NK, t);
}

// The tile: 256 x 256 (one workgroup per CU) where that still gives every CU a tile and a range of at least 256 rows, else 128 x 128.
// 8192 x 4096 x 4096, fp32 / fp16 / bf16: 679 / 436 / 264 us against 873 / 587 / 366; 1024 rows: 96 / 69 / 53 against 114 / 85 / 63;
// 65536 x 512 x 512: 110 / 87 / 67 against 128 / 101 / 76.
// The ranges: as many as give every CU a workgroup, none shorter than 128 rows. (Two small ones per CU: 262144 x 128 x 128 bf16 33 us
// against 30, 4096 x 512 x 512 26 against 23. Ranges of 512 rows at least: 20000 x 128 x 128 17 against 18, 2000 x 128 x 128 15
// against 11; of 32: 25 and 13.)
struct Plan { int cols; int64_t tiles_n, tiles_k; int splits; int64_t rows; };
Plan make_plan(int64_t M, int64_t N, int64_t K) {
  Plan p;
  const int64_t big = cdiv(N, 256) * cdiv(K, 256);
  p.cols = (N > 128 && K > 128 && big * cdiv(M, 256) >= 256) ? 256 : 128;
  p.tiles_n = cdiv(N, p.cols);
  p.tiles_k = cdiv(K, p.cols);
  const int64_t tiles = p.tiles_n * p.tiles_k;
  int64_t s = tiles >= 256 ? 1 : 256 / tiles;
  if (s > cdiv(M, 128)) s = cdiv(M, 128);
  p.splits = (int)(s < 1 ? 1 : s);
  p.rows = cdiv(cdiv(M, p.splits), STEP) * STEP;
  return p;
}

bool wgrad_ok(int64_t M, int64_t N, int64_t K) { return rows_ok(M, K) && K < (1ll << 22) && N >= 1 && N < (1ll << 24); }

template <int FMT, typename G, int COLS>
int launch_tile(const Job& o, hipStream_t stream) {
  static PerDeviceFlag ready;
  constexpr int lds = 2 * (PIECES<G> + 1) * STEP * pitch(COLS) * 2;
  auto k = wgrad8_kernel<FMT, G, COLS>;
  if (!ready) {
    const int rc = check_hip(hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                             "ganet_wgrad8");
    if (rc) return rc;
    ready = true;
  }
  const int64_t grid = (int64_t)o.tiles_n * o.tiles_k * o.splits;
  if (grid >= (1ll << 30)) { set_error("ganet_wgrad8: too many tiles"); return 4; }
  hipLaunchKernelGGL(k, dim3((unsigned)grid), dim3(64 * Form<COLS>::WAVES), lds, stream, o);
  return check_hip(hipGetLastError(), "ganet_wgrad8");
}

template <int FMT, typename G>
int launch(const Job& o, int cols, hipStream_t stream) {
  const int rc = cols == 256 ? launch_tile<FMT, G, 256>(o, stream) : launch_tile<FMT, G, 128>(o, stream);
  if (rc || o.splits == 1) return rc;
  const int64_t total = o.N * o.K + (o.db ? o.N : 0);
  hipLaunchKernelGGL(wgrad8_reduce_kernel, dim3((unsigned)cdiv(total, 64)), dim3(REDUCE_WG), 0, stream, o.N * o.K, o.N, o.splits, o.part,
                     o.dW, o.db, o.otype, o.btype);
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
                 int64_t ldc, const uint8_t* exps, int64_t lde, void* dW, void* db, int32_t otypes, void* workspace,
                 size_t workspace_bytes, void* stream_) {
  const int32_t otype = otypes & 0xff, btype = otypes >> 8 ? (otypes >> 8) - 1 : otype;
  if (!wgrad_ok(M, N, K) || (fmt != GANET_E4M3 && fmt != GANET_E5M2) || !type_ok(gtype) || !type_ok(otype) || !type_ok(btype)) {
    set_error("ganet_wgrad8: unsupported M=%lld N=%lld K=%lld format=%d types=%d,%d", (long long)M, (long long)N, (long long)K, fmt,
              gtype, otypes);
    return 4;
  }
  // (offsets inside a step of 32 rows are 32 bits)
  if (!dW || ldg > (1 << 24) || ldc > (1 << 24) || lde > (1 << 24) || (M > 0 && (!g || (ldg < N && M > 1) || !codes || !exps || ldc % 16 || ldc < pad16(K) || lde % 4 || lde < cdiv(K, BLOCK) ||
                        (reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(exps) & 3))) ||
      workspace_bytes < ganet_wgrad8_workspace(M, N, K, gtype) || (ganet_wgrad8_workspace(M, N, K, gtype) && !workspace)) {
    set_error("ganet_wgrad8: NULL or misaligned argument, a row stride outside columns .. 2^24, or the workspace too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const Plan p = make_plan(M, N, K);
  const Job o{M, N, K, g, ldg, static_cast<const uint8_t*>(codes), ldc, exps, lde, dW, db, otype, btype, static_cast<float*>(workspace),
              p.splits, p.rows, (int)p.tiles_n, (int)p.tiles_k};
  GANET_BY_TYPE(gtype, T, return fmt == GANET_E4M3 ? launch<GANET_E4M3, T>(o, p.cols, stream) : launch<GANET_E5M2, T>(o, p.cols, stream));
}

}  // extern "C"
