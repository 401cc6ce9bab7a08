// ganet_norm.hip — layer norm over the columns of a row + activation, forward and backward (include/ganet.h: ganet_ln_*).
//
//   xh = (x - mean) rstd, u = w xh + b, y = act(u)
//   g = dy act'(u), dw = sum_rows g xh, db = sum_rows g, dx = rstd (g w - mean_c(g w) - xh mean_c(g w xh))
//
// Bound: HBM. Forward reads x and writes y once, backward reads x (or its 8-bit xh) and dy and writes dx once: a row stays in
// registers between its reduction and its use, the variance is taken about the mean (no E[x^2] - mean^2), with the mean's own rounding
// taken back: the deviations d = x - mean are summed beside their squares, delta = sum(d) / C is what the first mean was off by, xh =
// (d - delta) rstd, var = sum(d^2) / C - delta^2. (Rows of equal values far from zero: xh = 0 and not a few units of x over sqrt(eps).) A group of G lanes holds
// a row, NC vectors of 16 bytes each: G = 1 .. 64 lanes of a wave for rows up to 4 KiB (backward: 2), a workgroup of 256 .. 1024 threads
// up to 32 KiB, and a streaming form that reads the row three times (from cache) beyond. Groups stride over the rows, so
// a lane always sees the same columns: w and b are loaded once, dw and db are summed in registers and leave as ONE partial row pair per workgroup,
// added in a fixed order by a second kernel (no atomics: bit-reproducible).
//
// xh as 8-bit codes: |xh| <= sqrt(C) for every input (sum xh^2 <= C), so the power of two that makes sqrt(C) fit the format is
// known before a value is seen: no maximum to take and no exponents to store.
#include <cmath>

#include "ganet_rows8.h"

namespace ganet {
using namespace rows8;

namespace {

constexpr int ACT_NONE = 0, ACT_SOFTPLUS = 1, ACT_RELU = 2;
constexpr int LN_WG = 256;

// softplus = max(u, 0) + log1p(e), e = exp(-|u|) (torch's threshold of 20 differs by 2e-9 of the value). With s = e / (2 + e), log1p(e) =
// log((1 + s) / (1 - s)) = 2 s (1 + z / 3 + z^2 / 5 + ..), z = s^2 <= 1/9: one polynomial in z (Chebyshev interpolation, 4e-9 relative), relatively
// accurate on both sides. The hardware logarithm of 1 + e instead is good to 1e-7 absolute only, 50 units of fp32 at u = -3.4.
// FULL (fp32 results): exp's argument -|u| log2(e) is rounded at the size of |u|, 2^-17 of e at |u| = 86; what the rounding and the constant
// lost is put back to first order: 2^-20 of the value (8 2^-24 in fp32 numpy). 16-bit results, 2^-12 at best, do without: 2^-16.
constexpr float LOG2E = 1.44269504f, LOG2E_REST = 1.925963e-8f, LN2 = 0.693147181f;
template <bool FULL>
__device__ __forceinline__ float softplus(float u) {
  float e, top;
  if (FULL) {
    const float a = fminf(fabsf(u), 110.f);                // (beyond: 0, and the correction stays a number)
    const float t = a * -LOG2E, rest = fmaf(a, -LOG2E_REST, fmaf(a, -LOG2E, -t));
    e = __builtin_amdgcn_exp2f(t);
    e = fmaf(e, rest * LN2, e);
    top = u < 0.f ? 0.f : u;                               // (a NaN stays one)
  } else {
    e = __builtin_amdgcn_exp2f(-LOG2E * fabsf(u));
    top = fmaxf(u, 0.f);
  }
  const float s = e * __builtin_amdgcn_rcpf(2.f + e), z = s * s;
  return fmaf(s, fmaf(z, fmaf(z, fmaf(z, fmaf(z, 0.281577796f, 0.279651582f), 0.400245965f), 0.666663229f), 2.f), top);
}
// sigmoid(u) = 1 / (1 + exp(-u)); exp(-u) = infinity gives 0. The hardware reciprocal: 1 ulp.
__device__ __forceinline__ float sigmoid(float u) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * u)); }

// act of N values, and g times its derivative (the kind is uniform: one branch per vector)
template <bool FULL, int N>
__device__ __forceinline__ void act_fwd(float (&v)[N], int act) {
  if (act == ACT_SOFTPLUS) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = softplus<FULL>(v[i]);
  } else if (act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];
  }
}
template <int N>
__device__ __forceinline__ void act_bwd(float (&g)[N], const float (&xh)[N], const float (&w)[N], const float (&b)[N], int act) {
  if (act == ACT_SOFTPLUS) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] *= sigmoid(fmaf(xh[i], w[i], b[i]));
  } else if (act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float u = fmaf(xh[i], w[i], b[i]);
      g[i] = u > 0.f ? g[i] : (u != u ? u : 0.f);
    }
  }
}

template <typename T> constexpr int VEC = 16 / (int)sizeof(T);

// Sum over 2^k <= 64 adjacent lanes; every lane gets it. Up to 16 lanes by register permutations: once all lanes of a group of 4
// (8) hold their sum, the mirrored lane of the 8 (16) holds the other group's.
template <int CTRL>
__device__ __forceinline__ float permuted(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ void lane_sum(float (&v)[N], int lanes) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (lanes > 1) v[i] += permuted<0xB1>(v[i]);       // quad_perm [1,0,3,2]
    if (lanes > 2) v[i] += permuted<0x4E>(v[i]);       // quad_perm [2,3,0,1]
    if (lanes > 4) v[i] += permuted<0x141>(v[i]);      // row_half_mirror
    if (lanes > 8) v[i] += permuted<0x140>(v[i]);      // row_mirror
    if (lanes > 16) v[i] += __shfl_xor(v[i], 16);
    if (lanes > 32) v[i] += __shfl_xor(v[i], 32);
  }
}

// Sum over the lanes that hold a row. WIDE: over the workgroup, through LDS (two buffers in turn: a buffer is written again only
// after a barrier that every reader of its last content has passed).
template <bool WIDE, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int G, float* s_red, int& phase) {
  if (!WIDE) {
    lane_sum(v, G);
    return;
  }
  lane_sum(v, 64);
  const int nw = blockDim.x >> 6, wave = threadIdx.x >> 6;
  float* s = s_red + phase * 2 * 16;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i * 16 + wave] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float t = 0.f;
    for (int w = 0; w < nw; ++w) t += s[i * 16 + w];
    v[i] = t;
  }
  phase ^= 1;
}

// A vector of a row as it was loaded: elements past the row's end, and all of a row that does not exist, are zero.
template <typename T>
struct Vec { T e[VEC<T>]; };
template <bool STREAM, typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* __restrict__ p, int n) {
  Vec<T> v;
  if (n >= VEC<T>) {
    if (STREAM) {
      const u32x4 q = load_stream(p);
      __builtin_memcpy(&v, &q, sizeof(v));
    } else __builtin_memcpy(&v, p, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < VEC<T>; ++i) v.e[i] = i < n ? p[i] : (T)0.f;
  }
  return v;
}

// STREAM: no backward pass reads x again (it reads codes, or there is none), so x passes the caches by. y does in any case: 262144 x 128
// fp32 65 -> 49 us, its backward pass 76 -> 63, and what reads y next is no slower (with the packing of y: 89 -> 76 us, of 65536 rows 27 ->
// 24). 16384 x 4096 bf16 to codes 78 -> 55 us with both; x that is kept and read again at once costs 12 us more in the backward pass.
template <typename T, int NC, bool WIDE, int THREADS, bool STREAM>
__global__ void __launch_bounds__(THREADS)
ln_fwd_kernel(int64_t M, int C, int G, const T* __restrict__ x, int64_t ldx, const void* __restrict__ w,
              const void* __restrict__ b, int32_t wtype, float eps, int act, T* __restrict__ y, float* __restrict__ mean_out,
              float* __restrict__ rstd_out, uint8_t* __restrict__ codes, int64_t ldc, float code_scale) {
  constexpr int V = VEC<T>;
  __shared__ float s_red[2 * 2 * 16];
  int phase = 0;
  const int l = WIDE ? threadIdx.x : (threadIdx.x & (G - 1));
  const int groups = WIDE ? 1 : THREADS / G, grp = WIDE ? 0 : threadIdx.x / G;
  const float inv = 1.0f / (float)C;
  const bool full = C % V == 0;              // no vector ends past the row
  float wv[NC][V], bv[NC][V];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = (j * G + l) * V;
    load_params(w, wtype, c, C - c, 1.f, wv[j]);
    load_params(b, wtype, c, C - c, 0.f, bv[j]);
  }
  // every lane of a wave takes the same number of turns: the sums need whole groups, a turn without a row reads nothing. The next
  // turn's row is loaded before this one's sums.
  const int64_t turn = (int64_t)gridDim.x * groups;
  int64_t row = (int64_t)blockIdx.x * groups + grp;
  const int64_t turns = (M - (int64_t)blockIdx.x * groups + turn - 1) / turn;
  Vec<T> next[NC];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (j * G + l) * V;
      next[j] = load_vec<STREAM>(x + r * ldx + c, r < M ? C - c : 0);
    }
  };
  fetch(row);
  for (int64_t t = 0; t < turns; ++t, row += turn) {
    const bool live = row < M;
    float v[NC][V];
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NC; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) { v[j][i] = (float)next[j].e[i]; s[0] += v[j][i]; }
    }
    if (t + 1 < turns) fetch(row + turn);
    row_sum<WIDE>(s, G, s_red, phase);
    const float mean = s[0] * inv;
    float d[2] = {0.f, 0.f};                               // the deviations' sum, and their squares'
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int left = C - (j * G + l) * V;
      if (full) {
        const float m = left > 0 ? mean : 0.f;             // (a vector past the row is zero: it stays so)
#pragma unroll
        for (int i = 0; i < V; ++i) { v[j][i] -= m; d[0] += v[j][i]; d[1] = fmaf(v[j][i], v[j][i], d[1]); }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) { v[j][i] = i < left ? v[j][i] - mean : 0.f; d[0] += v[j][i]; d[1] = fmaf(v[j][i], v[j][i], d[1]); }
      }
    }
    row_sum<WIDE>(d, G, s_red, phase);
    const float delta = d[0] * inv;
    const float rstd = rsqrtf(fmaxf(fmaf(d[1], inv, -delta * delta), 0.f) + eps), shift = -delta * rstd;
    if (live && l == 0) {
      if (mean_out) mean_out[row] = mean + delta;
      if (rstd_out) rstd_out[row] = rstd;
    }
    if (!live) continue;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (j * G + l) * V;
      if (c >= C) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = fmaf(v[j][i], rstd, shift);
      if (!full) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = i < C - c ? v[j][i] : 0.f;
      }
      if (codes) {
        uint8_t* p = codes + row * ldc + c;                // c is a multiple of V: aligned to V bytes; ldc covers the last vector
#pragma unroll
        for (int q = 0; q < V / 4; ++q)
          reinterpret_cast<unsigned*>(p)[q] =
              pack4<GANET_E4M3>(v[j][4 * q] * code_scale, v[j][4 * q + 1] * code_scale, v[j][4 * q + 2] * code_scale,
                                v[j][4 * q + 3] * code_scale);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = fmaf(v[j][i], wv[j][i], bv[j][i]);
      act_fwd<sizeof(T) == 4>(v[j], act);
      store_stream(y + row * C + c, C - c, v[j]);
    }
  }
}

// Streaming form: rows beyond 2048 vectors. One workgroup per row, three reads of the row.
template <typename T>
__global__ void __launch_bounds__(1024)
ln_fwd_stream_kernel(int64_t M, int64_t C, const T* __restrict__ x, int64_t ldx, const void* __restrict__ w,
                     const void* __restrict__ b, int32_t wtype, float eps, int act, T* __restrict__ y,
                     float* __restrict__ mean_out, float* __restrict__ rstd_out, uint8_t* __restrict__ codes, int64_t ldc,
                     float code_scale) {
  constexpr int V = VEC<T>;
  __shared__ float s_red[2 * 2 * 16];
  int phase = 0;
  const double inv = 1.0 / (double)C;
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
    const T* xr = x + row * ldx;
    float v[V];
    float s[1] = {0.f};
    for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
      load_n(xr + c, C - c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += v[i];
    }
    row_sum<true>(s, 0, s_red, phase);
    const float mean = (float)(s[0] * inv);
    float sd[2] = {0.f, 0.f};                              // the deviations' sum, and their squares'
    for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
      load_n(xr + c, C - c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = c + i < C ? v[i] - mean : 0.f;
        sd[0] += d;
        sd[1] = fmaf(d, d, sd[1]);
      }
    }
    row_sum<true>(sd, 0, s_red, phase);
    const float delta = (float)(sd[0] * inv);
    const float rstd = rsqrtf(fmaxf((float)(sd[1] * inv) - delta * delta, 0.f) + eps);
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[row] = mean + delta;
      if (rstd_out) rstd_out[row] = rstd;
    }
    for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
      load_n(xr + c, C - c, v);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = c + i < C ? (v[i] - mean - delta) * rstd : 0.f;    // (the backward pass reads a row's last vector whole)
      if (codes) {
        uint8_t* p = codes + row * ldc + c;
#pragma unroll
        for (int q = 0; q < V / 4; ++q)
          reinterpret_cast<unsigned*>(p)[q] = pack4<GANET_E4M3>(v[4 * q] * code_scale, v[4 * q + 1] * code_scale,
                                                                v[4 * q + 2] * code_scale, v[4 * q + 3] * code_scale);
      }
      float wv[V], bv[V];
      load_params(w, wtype, (int)c, (int)(C - c), 1.f, wv);
      load_params(b, wtype, (int)c, (int)(C - c), 0.f, bv);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = fmaf(v[i], wv[i], bv[i]);
      act_fwd<sizeof(T) == 4>(v, act);
      store_n(y + row * C + c, C - c, v);
    }
  }
}

// What the backward pass loads of a vector, and xh from it. Columns past the row give -mean rstd or zero: their gradient is zero.
template <typename T, bool KEPT8>
struct Kept {
  Vec<T> x;
  unsigned c[VEC<T> / 4];
  __device__ __forceinline__ void load(const T* xr, const uint8_t* cr, int c0, int n) {
    if (KEPT8) {
#pragma unroll
      for (int q = 0; q < VEC<T> / 4; ++q) c[q] = 0u;
      if (n > 0) __builtin_memcpy(c, __builtin_assume_aligned(cr + c0, VEC<T>), VEC<T>);
    } else x = load_vec<false>(xr + c0, n);
  }
  __device__ __forceinline__ void values(float mean, float rstd, float code_unit, float (&xh)[VEC<T>]) const {
    if (KEPT8) {
#pragma unroll
      for (int q = 0; q < VEC<T> / 4; ++q) {
        float t[4];
        unpack4<GANET_E4M3>(c[q], t);
#pragma unroll
        for (int i = 0; i < 4; ++i) xh[4 * q + i] = t[i] * code_unit;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC<T>; ++i) xh[i] = ((float)x.e[i] - mean) * rstd;
    }
  }
};

template <typename T, int NC, bool WIDE, int THREADS, bool KEPT8>
__global__ void __launch_bounds__(THREADS)
ln_bwd_kernel(int64_t M, int C, int G, const T* __restrict__ x, int64_t ldx, const float* __restrict__ mean_in,
              const uint8_t* __restrict__ codes, int64_t ldc, float code_unit, const float* __restrict__ rstd_in,
              const void* __restrict__ w, const void* __restrict__ b, int32_t wtype, int act, const T* __restrict__ dy,
              int64_t lddy, T* __restrict__ dx, float* __restrict__ part) {
  constexpr int V = VEC<T>;
  extern __shared__ float s_mem[];             // the partial sums of the waves (not WIDE)
  __shared__ float s_red[2 * 2 * 16];
  int phase = 0;
  const int l = WIDE ? threadIdx.x : (threadIdx.x & (G - 1));
  const int groups = WIDE ? 1 : THREADS / G, grp = WIDE ? 0 : threadIdx.x / G;
  const float inv = 1.0f / (float)C;
  // 1024 threads have 128 registers each: the parameters are read again (from cache) with every row
  constexpr bool HOLD = THREADS < 1024;
  float wv[NC][V], bv[NC][V], aw[NC][V], ab[NC][V];
  auto params = [&](int j) {
    const int c = (j * G + l) * V;
    load_params(w, wtype, c, C - c, 1.f, wv[j]);
    if (act != ACT_NONE) load_params(b, wtype, c, C - c, 0.f, bv[j]);
  };
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    if (HOLD) params(j);
#pragma unroll
    for (int i = 0; i < V; ++i) aw[j][i] = ab[j][i] = 0.f;
  }
  const int64_t turn = (int64_t)gridDim.x * groups;
  int64_t row = (int64_t)blockIdx.x * groups + grp;
  const int64_t turns = (M - (int64_t)blockIdx.x * groups + turn - 1) / turn;
  Vec<T> gn[NC];
  Kept<T, KEPT8> xn[NC];
  float mean_n = 0.f, rstd_n = 0.f;
  auto fetch = [&](int64_t r) {                // (a row that does not exist: zeros, and rstd = 0)
    const bool live = r < M;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (j * G + l) * V, n = live ? C - c : 0;
      gn[j] = load_vec<false>(dy + r * lddy + c, n);
      xn[j].load(x + r * ldx, codes + r * ldc, c, n);
    }
    if (!KEPT8) mean_n = live ? mean_in[r] : 0.f;
    rstd_n = live ? rstd_in[r] : 0.f;
  };
  fetch(row);
  for (int64_t t = 0; t < turns; ++t, row += turn) {
    const float mean = mean_n, rstd = rstd_n;
    float xh[NC][V], g[NC][V];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      xn[j].values(mean, rstd, code_unit, xh[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) g[j][i] = (float)gn[j].e[i];
    }
    if (t + 1 < turns) fetch(row + turn);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      if (!HOLD) params(j);
      act_bwd(g[j], xh[j], wv[j], bv[j], act);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        aw[j][i] = fmaf(g[j][i], xh[j][i], aw[j][i]);
        ab[j][i] += g[j][i];
        g[j][i] *= wv[j][i];
        s[0] += g[j][i];
        s[1] = fmaf(g[j][i], xh[j][i], s[1]);
      }
    }
    row_sum<WIDE>(s, G, s_red, phase);
    if (dx && row < M) {
      const float m1 = s[0] * inv, m2 = s[1] * inv;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = (j * G + l) * V;
        if (c >= C) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) g[j][i] = rstd * (g[j][i] - fmaf(xh[j][i], m2, m1));
        store_stream(dx + row * C + c, C - c, g[j]);
      }
    }
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * C;
  if (WIDE) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = (j * G + l) * V;
      store_n(out + c, C - c, aw[j]);
      store_n(out + C + c, C - c, ab[j]);
    }
    return;
  }
  // groups of a wave by shuffles, then the waves through LDS (dw, then db, through the same)
  for (int off = G; off < 64; off <<= 1) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        aw[j][i] += __shfl_xor(aw[j][i], off);
        ab[j][i] += __shfl_xor(ab[j][i], off);
      }
    }
  }
  const int wave = threadIdx.x >> 6, cols = G * NC * V;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k) __syncthreads();
    if ((threadIdx.x & 63) < G) {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) s_mem[wave * cols + (j * G + l) * V + i] = k ? ab[j][i] : aw[j][i];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += THREADS) {
      float t = 0.f;
#pragma unroll
      for (int v = 0; v < THREADS / 64; ++v) t += s_mem[v * cols + c];
      out[k * C + c] = t;
    }
  }
}

// Streaming form of the input gradient (two reads of the row), and the column sums over slices of the rows.
template <typename T, bool KEPT8>
__global__ void __launch_bounds__(1024)
ln_bwd_stream_kernel(int64_t M, int64_t C, const T* __restrict__ x, int64_t ldx, const float* __restrict__ mean_in,
                     const uint8_t* __restrict__ codes, int64_t ldc, float code_unit, const float* __restrict__ rstd_in,
                     const void* __restrict__ w, const void* __restrict__ b, int32_t wtype, int act, const T* __restrict__ dy,
                     int64_t lddy, T* __restrict__ dx) {
  constexpr int V = VEC<T>;
  __shared__ float s_red[2 * 2 * 16];
  int phase = 0;
  const float inv = (float)(1.0 / (double)C);
  for (int64_t row = blockIdx.x; row < M; row += gridDim.x) {
    const float mean = KEPT8 ? 0.f : mean_in[row], rstd = rstd_in[row];
    float m1 = 0.f, m2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      float s[2] = {0.f, 0.f};
      for (int64_t c = (int64_t)threadIdx.x * V; c < C; c += 1024 * V) {
        float g[V], xh[V];
        load_n(dy + row * lddy + c, C - c, g);
        Kept<T, KEPT8> kept;
        kept.load(x + row * ldx, codes + row * ldc, (int)c, (int)(C - c));
        kept.values(mean, rstd, code_unit, xh);
        float wv[V], bv[V];
        load_params(w, wtype, (int)c, (int)(C - c), 1.f, wv);
        load_params(b, wtype, (int)c, (int)(C - c), 0.f, bv);
        act_bwd(g, xh, wv, bv, act);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          g[i] *= wv[i];
          s[0] += g[i];
          s[1] = fmaf(g[i], xh[i], s[1]);
          g[i] = rstd * (g[i] - m1 - xh[i] * m2);
        }
        if (pass) store_n(dx + row * C + c, C - c, g);
      }
      if (!pass) {
        row_sum<true>(s, 0, s_red, phase);
        m1 = s[0] * inv;
        m2 = s[1] * inv;
      }
    }
  }
}

template <typename T, bool KEPT8>
__global__ void __launch_bounds__(LN_WG)
ln_bwd_columns_kernel(int64_t M, int64_t C, const T* __restrict__ x, int64_t ldx, const float* __restrict__ mean_in,
                      const uint8_t* __restrict__ codes, int64_t ldc, float code_unit, const float* __restrict__ rstd_in,
                      const void* __restrict__ w, const void* __restrict__ b, int32_t wtype, int act,
                      const T* __restrict__ dy, int64_t lddy, float* __restrict__ part) {
  constexpr int V = VEC<T>;
  const int64_t c = ((int64_t)blockIdx.x * LN_WG + threadIdx.x) * V;
  if (c >= C) return;
  float aw[V] = {}, ab[V] = {}, wv[V], bv[V];
  load_params(w, wtype, (int)c, (int)(C - c), 1.f, wv);
  load_params(b, wtype, (int)c, (int)(C - c), 0.f, bv);
  for (int64_t row = blockIdx.y; row < M; row += gridDim.y) {
    float g[V], xh[V];
    load_n(dy + row * lddy + c, C - c, g);
    Kept<T, KEPT8> kept;
    kept.load(x + row * ldx, codes + row * ldc, (int)c, (int)(C - c));
    kept.values(KEPT8 ? 0.f : mean_in[row], rstd_in[row], code_unit, xh);
    act_bwd(g, xh, wv, bv, act);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      aw[i] = fmaf(g[i], xh[i], aw[i]);
      ab[i] += g[i];
    }
  }
  float* out = part + (int64_t)blockIdx.y * 2 * C;
  store_n(out + c, C - c, aw);
  store_n(out + C + c, C - c, ab);
}

// dw / db: the workgroups' partial rows, added in a fixed order: a workgroup takes 16 adjacent columns, 64 slices of the rows
__global__ void __launch_bounds__(1024)
ln_bwd_final_kernel(int64_t C, int parts, const float* __restrict__ part, void* __restrict__ dw, void* __restrict__ db,
                    int32_t wtype) {
  __shared__ float s[64][17];
  const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 16 + cl;
  float t = 0.f;
  if (c < 2 * C) {
#pragma unroll 8
    for (int p = sl; p < parts; p += 64) t += part[(int64_t)p * 2 * C + c];
  }
  s[sl][cl] = t;
  __syncthreads();
  if (sl == 0 && c < 2 * C) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 64; ++k) t += s[k][cl];
    if (c < C) { if (dw) store_param(dw, wtype, c, t); }
    else if (db) store_param(db, wtype, c - C, t);
  }
}

struct Shape { int form; int G; int NC; int threads; };        // form 0: lanes of a wave, 1: workgroup, 2: streaming
Shape make_shape(int64_t C, int32_t type) {
  const int64_t n = cdiv(C, 16 / type_size(type));             // 16-byte vectors of a row
  Shape s{0, 1, 1, LN_WG};
  if (n <= 256) {
    // two vectors per lane where the row gives them: half the shuffles, twice the loads in flight of one vector per lane (200000 x 256
    // bf16, forward / backward: 57 / 85 us against 62 / 103). A workgroup per row for these: 65536 x 1024 bf16 157 / 351 against 70 / 116.
    while (s.G < 64 && s.G * 2 < n) s.G *= 2;
    s.NC = n <= s.G ? 1 : n <= 2 * s.G ? 2 : 4;
  } else if (n <= 2048) {                                      // (streaming instead: 8192 x 8192 bf16 153 / 387 against 72 / 121)
    s.form = 1;
    s.NC = 2;
    s.threads = n <= 512 ? 256 : n <= 1024 ? 512 : 1024;
    s.G = s.threads;
  } else {
    s.form = 2;
    s.threads = 1024;
  }
  return s;
}

// Backward, four vectors per lane would take all registers: a workgroup per row, one vector per lane (32768 x 2048 bf16 143 -> 98 us).
Shape bwd_shape(int64_t C, int32_t type) {
  Shape s = make_shape(C, type);
  if (s.NC == 4) s = Shape{1, 256, 1, 256};
  return s;
}

// One round of workgroups strides over the rows: as many as are resident at a time (256 CUs; by the kernels' registers). (Fewer, where
// that evens out the last turn: 200000 x 256 bf16 forward 57 against 53, 16384 x 4096 backward 121 against 104.)
constexpr int CUS = 256, STREAM_SLICES = 64;
int64_t one_round(int64_t turns, int per_cu) { return turns < (int64_t)CUS * per_cu ? turns : (int64_t)CUS * per_cu; }
int64_t fwd_grid(const Shape& s, int32_t type, int64_t M) {
  if (s.form == 2) return M < 2 * CUS ? M : 2 * CUS;
  const int per_cu = s.threads == 1024 ? 1 : s.threads == 512 ? 2 : type == GANET_F32 ? 6 : 4;
  return one_round(cdiv(M, s.form ? 1 : s.threads / s.G), per_cu);
}
// (a workgroup per row leaves a row of partial sums: at least four rows each, where that gives half of the CUs one: 1000 x 2048 bf16
// 25 -> 16 us, 300 x 4096 20 -> 17)
int64_t bwd_grid(const Shape& s, int32_t type, int64_t M) {
  if (s.form == 2) return M < STREAM_SLICES ? M : STREAM_SLICES;
  const int per_cu = s.threads >= 512 ? (type == GANET_F32 && s.threads == 512 ? 2 : 1) : type == GANET_F32 || (s.form && s.NC == 1) ? 4 : s.form ? 3 : 2;
  const int64_t n = one_round(cdiv(M, s.form ? 1 : s.threads / s.G), per_cu), few = cdiv(M, 4) > CUS / 2 ? cdiv(M, 4) : CUS / 2;
  return s.form && few < n ? few : n;
}

bool ln_ok(int64_t M, int64_t C, int32_t type, int32_t wtype, int32_t act) {
  return rows_ok(M, C) && type_ok(type) && type_ok(wtype) && act >= 0 && act <= 2;
}

}  // namespace
}  // namespace ganet

using namespace ganet;

extern "C" {

int32_t ganet_ln_code_exponent(int64_t C) {
  // the smallest e with sqrt(C) <= 448 2^e
  int e = -8;
  while (e < 16 && (double)C > 200704.0 * std::pow(4.0, e)) ++e;
  return e;
}

int ganet_ln_fwd(int64_t M, int64_t C, int32_t type, int32_t wtype, const void* x, int64_t ldx, const void* w, const void* b,
                 float eps, int32_t act, void* y, float* mean, float* rstd, void* codes, int64_t ldc, void* stream_) {
  if (!ln_ok(M, C, type, wtype, act)) {
    set_error("ganet_ln_fwd: unsupported M=%lld C=%lld types=%d,%d act=%d", (long long)M, (long long)C, type, wtype, act);
    return 4;
  }
  if (M == 0) return 0;
  if (!x || !y || (ldx < C && M > 1) || (codes && (ldc % 16 || ldc < pad16(C) || (reinterpret_cast<uintptr_t>(codes) & 15)))) {
    set_error("ganet_ln_fwd: NULL or misaligned argument, or a row stride too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const Shape s = make_shape(C, type);
  const float cs = std::ldexp(1.0f, -ganet_ln_code_exponent(C));
  const dim3 grid((unsigned)fwd_grid(s, type, M));
  uint8_t* cd = static_cast<uint8_t*>(codes);
  const bool again = mean != nullptr;
#define LN_FWD(NC, WIDE, TH)                                                                                            \
  hipLaunchKernelGGL((again ? ln_fwd_kernel<T, NC, WIDE, TH, false> : ln_fwd_kernel<T, NC, WIDE, TH, true>), grid, dim3(TH), 0, stream, M, \
                     (int)C, s.G, static_cast<const T*>(x), ldx, w, b, wtype, eps, act, static_cast<T*>(y), mean, rstd, cd, ldc, cs)
  GANET_BY_TYPE(type, T, {
    if (s.form == 2)
      hipLaunchKernelGGL(ln_fwd_stream_kernel<T>, grid, dim3(1024), 0, stream, M, C, static_cast<const T*>(x), ldx, w, b,
                         wtype, eps, act, static_cast<T*>(y), mean, rstd, cd, ldc, cs);
    else if (s.form == 1) {
      if (s.threads == 256) LN_FWD(2, true, 256);
      else if (s.threads == 512) LN_FWD(2, true, 512);
      else LN_FWD(2, true, 1024);
    } else {
      if (s.NC == 1) LN_FWD(1, false, LN_WG);
      else if (s.NC == 2) LN_FWD(2, false, LN_WG);
      else LN_FWD(4, false, LN_WG);
    }
  });
#undef LN_FWD
  return check_hip(hipGetLastError(), "ganet_ln_fwd");
}

size_t ganet_ln_bwd_workspace(int64_t M, int64_t C, int32_t type) {
  if (!rows_ok(M, C) || !type_ok(type)) return 0;
  return (size_t)bwd_grid(bwd_shape(C, type), type, M < 1 ? 1 : M) * 2 * (size_t)C * sizeof(float);
}

int ganet_ln_bwd(int64_t M, int64_t C, int32_t type, int32_t wtype, const void* x, int64_t ldx, const float* mean,
                 const void* codes, int64_t ldc, const float* rstd, const void* w, const void* b, int32_t act,
                 const void* dy, int64_t lddy, void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes,
                 void* stream_) {
  if (!ln_ok(M, C, type, wtype, act)) {
    set_error("ganet_ln_bwd: unsupported M=%lld C=%lld types=%d,%d act=%d", (long long)M, (long long)C, type, wtype, act);
    return 4;
  }
  const bool sums = dw || db;
  if ((M > 0 && (!rstd || !dy || (!codes && (!x || !mean)) || (!codes && ldx < C && M > 1) || (lddy < C && M > 1))) ||
      (codes && (ldc % 16 || ldc < pad16(C) || (reinterpret_cast<uintptr_t>(codes) & 15))) ||
      (sums && (!workspace || workspace_bytes < ganet_ln_bwd_workspace(M, C, type)))) {
    set_error("ganet_ln_bwd: NULL or misaligned argument, a row stride or the workspace too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const Shape s = bwd_shape(C, type);
  const float cu = std::ldexp(1.0f, ganet_ln_code_exponent(C));
  float* part = sums ? static_cast<float*>(workspace) : nullptr;
  const uint8_t* cd = static_cast<const uint8_t*>(codes);
  const int64_t parts = M ? bwd_grid(s, type, M) : 0;
#define LN_BWD(NC, WIDE, TH, K8)                                                                                              \
  hipLaunchKernelGGL((ln_bwd_kernel<T, NC, WIDE, TH, K8>), dim3((unsigned)parts), dim3(TH),                                        \
                     WIDE ? 0 : (size_t)(TH / 64) * s.G * NC * VEC<T> * sizeof(float), stream, M, (int)C, s.G,                 \
                     static_cast<const T*>(x), ldx, mean, cd, ldc, cu, rstd, w, b, wtype, act, static_cast<const T*>(dy), lddy, \
                     static_cast<T*>(dx), part)
#define LN_BWD_FORMS(K8)                                                                                                      \
  do {                                                                                                                        \
    if (s.form == 2) {                                                                                                        \
      if (dx)                                                                                                                 \
        hipLaunchKernelGGL((ln_bwd_stream_kernel<T, K8>), dim3((unsigned)(M < 2 * CUS ? M : 2 * CUS)), dim3(1024), 0, stream, \
                           M, C, static_cast<const T*>(x), ldx, mean, cd, ldc, cu, rstd, w, b, wtype, act,                     \
                           static_cast<const T*>(dy), lddy, static_cast<T*>(dx));                                             \
      if (part)                                                                                                               \
        hipLaunchKernelGGL((ln_bwd_columns_kernel<T, K8>), dim3((unsigned)cdiv(C, LN_WG * VEC<T>), (unsigned)parts), dim3(LN_WG), \
                           0, stream, M, C, static_cast<const T*>(x), ldx, mean, cd, ldc, cu, rstd, w, b, wtype, act,          \
                           static_cast<const T*>(dy), lddy, part);                                                            \
    } else if (s.form == 1) {                                                                                                 \
      if (s.NC == 1) LN_BWD(1, true, 256, K8);                                                                                \
      else if (s.threads == 256) LN_BWD(2, true, 256, K8);                                                                    \
      else if (s.threads == 512) LN_BWD(2, true, 512, K8);                                                                    \
      else LN_BWD(2, true, 1024, K8);                                                                                         \
    } else {                                                                                                                  \
      if (s.NC == 1) LN_BWD(1, false, LN_WG, K8);                                                                             \
      else LN_BWD(2, false, LN_WG, K8);                                                                                       \
    }                                                                                                                         \
  } while (0)
  if (M > 0) {
    GANET_BY_TYPE(type, T, {
      if (codes) LN_BWD_FORMS(true);
      else LN_BWD_FORMS(false);
    });
  }
#undef LN_BWD_FORMS
#undef LN_BWD
  if (sums)       // (also for M = 0: the gradients of no rows are zero)
    hipLaunchKernelGGL(ln_bwd_final_kernel, dim3((unsigned)cdiv(2 * C, 16)), dim3(1024), 0, stream, C, (int)parts, part, dw, db, wtype);
  return check_hip(hipGetLastError(), "ganet_ln_bwd");
}

}  // extern "C"
