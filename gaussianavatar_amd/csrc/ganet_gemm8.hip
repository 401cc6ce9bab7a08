// ganet_gemm8.hip — matrix products of 8-bit floating point with a power of two for each block of 128 (include/ganet.h: ganet_gemm8).
//
//   y[m, n] = sum_kb 2^(ex[m, kb] + ew[n / 128, kb]) sum_{k in block kb} x[m, k] w[n, k] + bias[n]
//
// The scaled matrix instructions (v_mfma_scale_f32_*_f8f6f4) multiply 64 or 128 codes at a time and take a biased exponent per
// lane and operand: a power of two per block of 128 costs no vector instruction, where an arbitrary fp32 scale would cost an
// accumulator update per block. Products of codes are exact; sums are fp32 and y is rounded once. The 8-bit instructions do not add in fp32
// (see multiply()): sums run on bf16 instructions over decoded codes, which are exact there, unless the caller asks for the 8-bit ones (GANET_FAST).
#include "ganet_rows8.h"

namespace ganet {
using namespace rows8;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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
// A workgroup of four waves computes 64 MT x 64 NT of y, a wave 32 MT x 32 NT. One phase is half a block, 64 codes: its rows go
// from global memory straight into LDS (16 bytes per lane, no registers). A row of a phase is 64 bytes = 4 chunks of 16; chunk c of row r lies at
// position c ^ ((r >> 2) & 3), so that the 16 rows that a quarter of a wave reads at once lie in 16 different 16-byte columns of LDS.
// The instruction writes lanes in order, so the swizzle is in the global address that a lane fetches.
//
// Four LDS buffers and two register sets of fragments. Phase h:
//     phase h + 1 has landed; barrier (and everybody has read phase h)
//     multiply phase h and, between the multiplications, read phase h + 1 and fetch phase h + 4 into the buffer of phase h
// so that neither LDS nor memory latency stands between two multiplications, and a fetch has three phases to arrive (with whole blocks
// and two buffers it had two: 8192^3 2.28 PFLOP/s). A wave issues in order: what stands behind sixteen multiplications waits for
// fifteen of them and then runs beside the last one only. So every multiplication is followed by its share of the reads and
// fetches, and nothing crosses it (2.16 PFLOP/s with the reads and fetches in one go). These rates are of the 8-bit instructions; on bf16 ones,
// four times as many at twice the time together, there is more to hide behind: 8192^3 1.39 PFLOP/s.
//
// No branch in the loop: rows past the matrix fetch its last row (results nobody stores), chunks past a row's codes fetch its last
// chunk and are zeroed in x's fragments, which only the last block needs; phases past the end fetch the last block again.
//
// The fetches are issued from inline assembly: they have no register result, and the compiler, which cannot tell the buffers apart,
// would otherwise wait for the phases in flight before it reads the one that has landed. Every wait for them is the explicit one below,
// by their number; so nothing else may load to registers in the loop: the exponents lie in LDS, 64 blocks at a time.
__device__ __forceinline__ void fetch16(const uint8_t* base, unsigned off, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}

// Chunk 2 (lane / 32) + h of fragment i of a wave's rows: a lane holds 32 codes of one of 32 rows.
__device__ __forceinline__ void read_chunk(const uint8_t* lds, int lane, int i, int h, i32x8& f) {
  const int r = lane & 31, c = (lane >> 5) * 2 + h;
  const uint4 v = *reinterpret_cast<const uint4*>(lds + r * 64 + i * 2048 + (c ^ ((r >> 2) & 3)) * 16);
  f[4 * h] = (int)v.x; f[4 * h + 1] = (int)v.y; f[4 * h + 2] = (int)v.z; f[4 * h + 3] = (int)v.w;
}

// Eight codes (dwords d, d + 1) times a power of two as bf16: exact, if it is at least 2^-133.
template <int FMT>
__device__ __forceinline__ bf16x8 decode8(const i32x8& f, int d, float scale) {
  union { bf16x2 h[4]; bf16x8 v; } r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (FMT == GANET_E4M3) {
      r.h[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[d + i], scale, false);
      r.h[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[d + i], scale, true);
    } else {
      r.h[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(f[d + i], scale, false);
      r.h[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(f[d + i], scale, true);
    }
  }
  return r.v;
}

// acc += b a^T over one half block. EXACT: on bf16 instructions, codes times half their powers of two being bf16 numbers; sums in fp32, 4e-8 of a
// result's norm. Else on the 8-bit ones, which add products in groups of eight adjacent k, each cut to a multiple of 2^-13 of the group's
// largest power of two, before they go on in fp32 (the older 16-deep ones are the same): 3e-5 to 6e-5 of a result's norm, 1/30 of bf16's rounding and 1/4 of
// fp16's, but where large products of one group cancel, what is left is no better than 2^-13 of them. They are faster: 8192 x 4096 ->
// 8192 230 us (2.4 PFLOP/s) against 408 (1.35), 3000 x 4096 -> 4096 53 against 93, 262144 x 256 -> 256 50 against 59.
// between(q) is called behind multiplication q of MULTIPLICATIONS.
template <bool EXACT, int MT, int NT> constexpr int MULTIPLICATIONS = (EXACT ? 4 : 1) * MT * NT;
template <int FMT, int MT, int NT, bool EXACT, typename Between>
__device__ __forceinline__ void multiply(const i32x8 (&a)[MT], const i32x8 (&b)[NT], const int (&sx)[MT], int sw, f32x16 (&acc)[NT][MT],
                                         Between between) {
  if constexpr (!EXACT) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a[i], acc[j][i], GANET_E4M3, FMT, 0, sw, 0, sx[i]);
        between(j * MT + i);
      }
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d) {                            // 16 products per instruction: eight codes of a lane
      bf16x8 x[MT], w[NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) x[i] = decode8<FMT>(a[i], 2 * d, half_scale(sx[i]));
#pragma unroll
      for (int j = 0; j < NT; ++j) w[j] = decode8<GANET_E4M3>(b[j], 2 * d, half_scale(sw));
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[j], x[i], acc[j][i], 0, 0, 0);
          between((d * NT + j) * MT + i);
        }
    }
  }
}

template <int FMT, int MT, int NT, typename Y, bool EXACT>
__global__ void __launch_bounds__(256, 1)
gemm8_tile_kernel(Operands o, int tiles_m, int tiles_n) {
  constexpr int TM = 64 * MT, TN = 64 * NT, BYTES = (TM + TN) * 64, EXPS = 64, EPITCH = EXPS + 4;
  extern __shared__ __align__(16) uint8_t s_tiles[];          // four buffers, then the exponents of 64 blocks: TM rows, TN / 128 columns
  uint8_t* const s_ex = s_tiles + 4 * BYTES;
  uint8_t* const s_ew = s_ex + TM * EPITCH;
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)s_tiles;
  // Workgroups go round the 8 XCDs in turn: give each XCD one run of tiles (its own L2 sees neighbouring rows and columns), and
  // inside a run walk 8 tiles down before the next column.
  const int T = tiles_m * tiles_n, q = T / 8, rem = T % 8, xcd = blockIdx.x % 8;
  const int t = xcd * q + (xcd < rem ? xcd : rem) + blockIdx.x / 8;
  const int group = t / (8 * tiles_n), gm = min(8, tiles_m - group * 8), in = t - group * 8 * tiles_n;
  // (in scalar registers: the divisions are done in vector ones)
  const int64_t m0 = (int64_t)__builtin_amdgcn_readfirstlane(group * 8 + in % gm) * TM, n0 = (int64_t)__builtin_amdgcn_readfirstlane(in / gm) * TN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wm = (wave & 1) * 32 * MT, wn = (wave >> 1) * 32 * NT;
  const int64_t kend = (o.K + 15) / 16 * 16;
  const int KB = (int)((o.K + BLOCK - 1) / BLOCK);

  // Instruction i of a wave's fetches of an operand: rows 64 i + 16 wave + lane / 4, the lane's chunk. (The swizzle does not depend on i.)
  constexpr int FX = MT, FW = NT, FETCHES = FX + FW, READS = 2 * (MT + NT), MULS = MULTIPLICATIONS<EXACT, MT, NT>;
  const int fr = wave * 16 + (lane >> 2), fc = (lane & 3) ^ ((fr >> 2) & 3);
  const int last_chunks = (int)((kend - (int64_t)(KB - 1) * BLOCK) / 16);
  // from a lane's offset in a block to its chunk of the last block's halves (with the offset never below zero: it is unsigned)
  const unsigned shift0 = (unsigned)(min(fc, last_chunks - 1) - fc) * 16u, shift1 = (unsigned)(min(4 + fc, last_chunks - 1) - fc) * 16u;
  unsigned offx[FX], offw[FW];
#pragma unroll
  for (int i = 0; i < FX; ++i) offx[i] = (unsigned)min((int64_t)(fr + i * 64), o.M - 1 - m0) * (unsigned)o.ldx + fc * 16;
#pragma unroll
  for (int i = 0; i < FW; ++i) offw[i] = (unsigned)min((int64_t)(fr + i * 64), o.N - 1 - n0) * (unsigned)o.ldw + fc * 16;
  const uint8_t *xt = o.x + m0 * o.ldx, *wt = o.w + n0 * o.ldw;
  auto fetch = [&](int kb, int half, int buf, int p) {        // instruction p of FETCHES
    const unsigned lds = lds0 + buf * BYTES + wave * 1024;
    const unsigned shift = kb + 1 == KB ? (half ? shift1 : shift0) : half * 64u;
    const int64_t at = (int64_t)kb * BLOCK;
    if (p < FX) fetch16(xt + at, offx[p] + shift, lds + p * 4096);
    else fetch16(wt + at, offw[p - FX] + shift, lds + TM * 64 + (p - FX) * 4096);
  };
  auto read = [&](int buf, i32x8 (&a)[MT], i32x8 (&b)[NT], int p) {                  // instruction p of READS
    const uint8_t* lds = s_tiles + buf * BYTES;
    if (p < 2 * MT) read_chunk(lds + wm * 64, lane, p >> 1, p & 1, a[p >> 1]);
    else read_chunk(lds + (TM + wn) * 64, lane, (p - 2 * MT) >> 1, p & 1, b[(p - 2 * MT) >> 1]);
  };
  // the exponents of blocks kb .. kb + 63 (four at a time: their rows are multiples of four bytes)
  auto exponents = [&](int kb) {
    const int n4 = (min(KB - kb, EXPS) + 3) >> 2;
    for (int t = threadIdx.x; t < (TM + TN / BLOCK + 1) * n4; t += 256) {
      const int r = t / n4, c = t - r * n4;
      const uint8_t* e = r < TM ? o.ex + min(m0 + r, o.M - 1) * o.ldex : o.ew + min(n0 + (r - TM) * BLOCK, o.N - 1) / BLOCK * o.ldew;
      *reinterpret_cast<unsigned*>(s_ex + r * EPITCH + c * 4) = *reinterpret_cast<const unsigned*>(e + kb + c * 4);
    }
  };
  i32x8 a0[MT], b0[NT], a1[MT], b1[NT];
  int sx[MT], sw, sx_next[MT], sw_next;
  const uint8_t *exl = s_ex + (wm + (lane & 31)) * EPITCH, *ewl = s_ew + wn / BLOCK * EPITCH;
  auto scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < MT; ++i) sx_next[i] = exl[i * 32 * EPITCH + (kb & (EXPS - 1))];
    sw_next = ewl[kb & (EXPS - 1)];
  };
  auto take_scales = [&]() {
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = sx_next[i];
    sw = sw_next;
  };
  // this wave's fetches have arrived but for the two newest phases'; after the barrier, every wave's
  auto landed = [&]() {
    static_assert(FETCHES == 8 || FETCHES == 4, "the wait below counts two phases of fetches");
    if (FETCHES == 8) asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };

  exponents(0);
#pragma unroll
  for (int h = 0; h < 4; ++h)
#pragma unroll
    for (int p = 0; p < FETCHES; ++p) fetch(min(h >> 1, KB - 1), h & 1, h, p);
  // the sums start at the bias (its loads run beside the first fetch)
  f32x16 acc[NT][MT];
  auto start = [&](auto bias) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = bias(min(n0 + wn + j * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3), o.N - 1));
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i][r] = EXACT ? 0.25f * v : v;
      }
  };
  if (!o.bias) start([](int64_t) { return 0.f; });
  else GANET_BY_TYPE(o.btype, B, start([&](int64_t n) { return (float)static_cast<const B*>(o.bias)[n]; }));
  // phase 0 (all but the three newest) for its first reads; the loop waits for phase 1 itself
  if (FETCHES == 8) asm volatile("s_waitcnt vmcnt(24) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(12) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  scales(0);
#pragma unroll
  for (int p = 0; p < READS; ++p) read(0, a0, b0, p);
  for (int kb = 0; kb + 1 < KB; ++kb) {
    const int buf = (kb & 1) * 2, next = min(kb + 2, KB - 1);
    landed();
    take_scales();
    __builtin_amdgcn_sched_barrier(0);
    multiply<FMT, MT, NT, EXACT>(a0, b0, sx, sw, acc, [&](int q) {
#pragma unroll
      for (int p = READS * q / MULS; p < READS * (q + 1) / MULS; ++p) read(buf + 1, a1, b1, p);
#pragma unroll
      for (int p = FETCHES * q / MULS; p < FETCHES * (q + 1) / MULS; ++p) fetch(next, 0, buf, p);
      __builtin_amdgcn_sched_barrier(0);
    });
    landed();
    if ((kb + 1) % EXPS == 0) {              // the next 64 blocks' exponents (nobody reads the old ones any more)
      exponents(kb + 1);
      __syncthreads();
    }
    scales(kb + 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply<FMT, MT, NT, EXACT>(a1, b1, sx, sw, acc, [&](int q) {
#pragma unroll
      for (int p = READS * q / MULS; p < READS * (q + 1) / MULS; ++p) read(2 - buf, a0, b0, p);
#pragma unroll
      for (int p = FETCHES * q / MULS; p < FETCHES * (q + 1) / MULS; ++p) fetch(next, 1, buf + 1, p);
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  landed();
  take_scales();
#pragma unroll
  for (int p = 0; p < READS; ++p) read(((KB - 1) & 1) * 2 + 1, a1, b1, p);
  if (last_chunks < 8) {                     // what was fetched past the rows' codes
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in0 = (lane >> 5) * 2 + h < last_chunks, in1 = 4 + (lane >> 5) * 2 + h < last_chunks;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int d = 4 * h; d < 4 * h + 4; ++d) {
          a0[i][d] = in0 ? a0[i][d] : 0;
          a1[i][d] = in1 ? a1[i][d] : 0;
        }
    }
  }
  multiply<FMT, MT, NT, EXACT>(a0, b0, sx, sw, acc, [](int) {});
  multiply<FMT, MT, NT, EXACT>(a1, b1, sx, sw, acc, [](int) {});
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // (the fetches behind the last step)
  // A lane holds one row m and, four at a time, consecutive columns n. Stored from there, an instruction would touch 32 rows with 16
  // or 32 bytes each; through LDS (rows of 16 bytes more than the tile's: the 32 rows of a write fall into different banks) every
  // row leaves in full 16-byte pieces.
  constexpr int V = 16 / (int)sizeof(Y), PITCH = TN + V;
  Y* s_y = reinterpret_cast<Y*>(s_tiles);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        Y v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = (Y)(EXACT ? 4.f * acc[j][i][g * 4 + r] : acc[j][i][g * 4 + r]);
        Y* d = s_y + (wm + i * 32 + (lane & 31)) * PITCH + wn + j * 32 + g * 8 + (lane >> 5) * 4;
        __builtin_memcpy(__builtin_assume_aligned(d, 4 * sizeof(Y)), v, sizeof(v));
      }
  __syncthreads();
  constexpr int PER_ROW = TN / V, ROWS = 256 / PER_ROW;
  const int c = threadIdx.x % PER_ROW * V, r0 = threadIdx.x / PER_ROW;
  Y* y = static_cast<Y*>(o.y) + m0 * o.ldy + n0 + c;
  const int64_t left = o.N - n0 - c;
  const int rows = (int)min((int64_t)TM, o.M - m0);
  // A result of half the last-level cache and more is written past the caches: what it would drive out there (the inputs, that the
  // backward pass reads again) is worth more. fp32, 128 columns in and out, both directions alone / with a layer norm behind it, past the caches against through
  // them: 131072 rows (64 MiB) 125 against 124 / 194 against 192 us, 196608 (96 MiB) 128 against 142 / 218 against 223, 262144 161 against 188 / 278
  // against 292, 524288 330 against 395 / 551 against 594.
  const bool past = o.M * o.N * (int64_t)sizeof(Y) >= 1ll << 27;
  if (left >= V) {
#pragma unroll 8
    for (int r = r0; r < rows; r += ROWS) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(s_y + r * PITCH + c);
      if (past) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_loose*>(y + r * o.ldy));
      else __builtin_memcpy(y + r * o.ldy, &v, 16);
    }
  } else {
    for (int r = r0; r < rows; r += ROWS)
      for (int e = 0; e < left; ++e) y[r * o.ldy + e] = s_y[r * PITCH + c + e];
  }
}

// ------------------------------------------------------------------------------------------------ few rows
// The weight's codes are the traffic: every wave streams its share of the blocks of 16 weight rows straight from global memory into matrix
// operands (a lane: 32 codes of one row), the eight waves' sums meet in LDS. X: the rows' type. Rows that come as they are (not as
// codes) are packed in registers, by the rule of ganet_rows8_pack: the four lanes that hold a row's block take its maximum and
// convert; every workgroup repeats that (packs_inside() below tells where that costs less than a launch).
// What bounds it is latency: so everything that a wave needs of UNROLL blocks is asked for at once, without a branch between the
// loads (rows past the last read the last one, as do blocks); a last block that is not full comes behind them. From codes, bf16, twenty in
// a graph, one of them: 1 x 4096 x 4096 5.2 us, 16 rows 7.2, 1 x 16384 x 4096 15.9, 4.2 TB/s. (With the loads under conditions 4.5 and 10 us more for 1 and 16 rows.)
constexpr int FEW_WAVES = 8;
struct Codes;        // the rows' type where they are codes already

// 32 values of a row's block, held by the four lanes l, l ^ 16, l ^ 32, l ^ 48 -> operand and biased exponent
__device__ __forceinline__ void pack_block(const float (&v)[32], i32x8& f, int& e) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) a = fmaxf(a, finite_abs(v[i]));
  a = fmaxf(a, __shfl_xor(a, 16));
  a = fmaxf(a, __shfl_xor(a, 32));
  const int x = block_exponent<GANET_E4M3>(a);
  const float s = pow2(-x);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (int)pack4<GANET_E4M3>(v[4 * i] * s, v[4 * i + 1] * s, v[4 * i + 2] * s, v[4 * i + 3] * s);
  e = x + 127;
}

// A lane's 32 values of a row's block as they were loaded, and the operand that they become
template <typename X>
struct Few {
  X v[32];
  __device__ __forceinline__ void load(const Operands& o, int64_t m, int64_t k, int) {
    __builtin_memcpy(v, reinterpret_cast<const X*>(o.x) + m * o.ldx + k, sizeof(v));
  }
  __device__ __forceinline__ void operand(i32x8& f, int& e) const {
    float t[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) t[i] = (float)v[i];
    pack_block(t, f, e);
  }
};
template <>
struct Few<Codes> {
  uint4 v[2];
  int e;
  __device__ __forceinline__ void load(const Operands& o, int64_t m, int64_t k, int kb) {
    const uint4* p = reinterpret_cast<const uint4*>(o.x + m * o.ldx + k);
    v[0] = p[0];
    v[1] = p[1];
    e = o.ex[m * o.ldex + kb];
  }
  __device__ __forceinline__ void operand(i32x8& f, int& exponent) const {
    f = join(v[0], v[1]);
    exponent = e;
  }
};

template <int FMT, int MT, typename X, typename Y>
__global__ void __launch_bounds__(64 * FEW_WAVES)
gemm8_few_kernel(Operands o) {
  constexpr bool CODES = __is_same(X, Codes);
  constexpr int UNROLL = MT * sizeof(Few<X>) <= 128 ? 4 : 2;
  __shared__ f32x4 s_acc[FEW_WAVES][MT][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int full = (int)(o.K / BLOCK);
  const uint8_t* wr = o.w + min(n0 + r, o.N - 1) * o.ldw + q * 32;
  const uint8_t* ew = o.ew + n0 / BLOCK * o.ldew;
  int64_t m[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    m[i] = min((int64_t)(i * 16 + r), o.M - 1);
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto multiply = [&](const i32x8& w, int sw, const i32x8 (&x)[MT], const int (&sx)[MT]) {
    // bf16 instructions on decoded codes whatever the result's type (see multiply() above): what the 8-bit ones would save is not what
    // bounds these (1 x 4096 x 4096 bf16, packed inside: 7.3 us on the 8-bit ones against 7.8; 32 rows 16.2 against 16.4)
#pragma unroll
    for (int d = 0; d < 8; d += 2) {
      const bf16x8 wd = decode8<GANET_E4M3>(w, d, half_scale(sw));
#pragma unroll
      for (int i = 0; i < MT; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wd, decode8<FMT>(x[i], d, half_scale(sx[i])), acc[i], 0, 0, 0);
    }
  };
  for (int kb0 = wave; kb0 < full; kb0 += FEW_WAVES * UNROLL) {
    uint4 w[UNROLL][2];
    Few<X> raw[UNROLL][MT];
    int sw[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int kb = min(kb0 + u * FEW_WAVES, full - 1);
      const uint4* p = reinterpret_cast<const uint4*>(wr + (int64_t)kb * BLOCK);
      w[u][0] = p[0];
      w[u][1] = p[1];
      sw[u] = ew[kb];
#pragma unroll
      for (int i = 0; i < MT; ++i) raw[u][i].load(o, m[i], (int64_t)kb * BLOCK + q * 32, kb);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      if (kb0 + u * FEW_WAVES >= full) break;
      i32x8 x[MT];
      int sx[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) raw[u][i].operand(x[i], sx[i]);
      multiply(join(w[u][0], w[u][1]), sw[u], x, sx);
    }
  }
  if (o.K % BLOCK && wave == full % FEW_WAVES) {
    const int64_t k = (int64_t)full * BLOCK + q * 32, kend = (o.K + 15) / 16 * 16;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto codes = [&](const uint8_t* p) {                       // p: of column k
      return join(k < kend ? *reinterpret_cast<const uint4*>(p) : zero, k + 16 < kend ? *reinterpret_cast<const uint4*>(p + 16) : zero);
    };
    i32x8 x[MT];
    int sx[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (CODES) {
        x[i] = codes(o.x + m[i] * o.ldx + k);
        sx[i] = o.ex[m[i] * o.ldex + full];
      } else {
        float v[32];
        load_n(reinterpret_cast<const X*>(o.x) + m[i] * o.ldx + k, o.K - k, v);
        pack_block(v, x[i], sx[i]);
      }
    }
    multiply(codes(wr + (int64_t)full * BLOCK), ew[full], x, sx);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) s_acc[wave][i][lane] = acc[i];
  __syncthreads();
  if (threadIdx.x >= MT * 64) return;
  const int i = threadIdx.x >> 6;
  f32x4 t = s_acc[0][i][lane];
#pragma unroll
  for (int v = 1; v < FEW_WAVES; ++v) t += s_acc[v][i][lane];
  const int64_t row = i * 16 + r, n = n0 + q * 4;
  if (row >= o.M) return;
  float v[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = 4.f * t[c] + ((o.bias && n + c < o.N) ? load_param(o.bias, o.btype, n + c) : 0.f);
  store_n(static_cast<Y*>(o.y) + row * o.ldy + n, o.N - n, v);
}

// (32 x 4096 x 4096 from codes, bf16 / fp32: 9.9 / 10.0 us; 64 x 4096 x 4128 in tiles 30, fast 16)
constexpr int FEW_ROWS = 32;
template <int FMT, typename X, typename Y>
int launch_few(const Operands& o, hipStream_t stream) {
  const dim3 grid((unsigned)cdiv(o.N, 16));
  if (o.M <= 16) hipLaunchKernelGGL((gemm8_few_kernel<FMT, 1, X, Y>), grid, dim3(64 * FEW_WAVES), 0, stream, o);
  else hipLaunchKernelGGL((gemm8_few_kernel<FMT, 2, X, Y>), grid, dim3(64 * FEW_WAVES), 0, stream, o);
  return check_hip(hipGetLastError(), "ganet_gemm8");
}

template <int FMT, int MT, int NT, typename Y, bool EXACT>
int launch_tile(const Operands& o, hipStream_t stream) {
  static PerDeviceFlag ready;
  constexpr int steps = 4 * 64 * (MT + NT) * 64 + (64 * MT + NT / 2 + 1) * 68, out = 64 * MT * (64 * NT * (int)sizeof(Y) + 16), lds = steps > out ? steps : out;
  auto k = gemm8_tile_kernel<FMT, MT, NT, Y, EXACT>;
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

// The tile: 256 x 256 for 16-bit results (an fp32 tile of that size does not fit LDS on its way out) where three quarters of the CUs get
// one, else 128 x 128. 192 tiles (3000 x 4096 x 4096): 93.2 us against 93.7 (fast: 52 against 62), 256 (4096^3) 106 against 118; 128
// (4096 x 4096 x 2048): 89 against 67 (fast: 31 against 27).
template <int FMT, typename Y, bool EXACT>
int launch_tiles(const Operands& o, hipStream_t stream) {
  if constexpr (sizeof(Y) == 2)
    if (cdiv(o.M, 256) * cdiv(o.N, 256) >= 192) return launch_tile<FMT, 4, 4, Y, EXACT>(o, stream);
  return launch_tile<FMT, 2, 2, Y, EXACT>(o, stream);
}

template <int FMT, typename Y>
int launch(const Operands& o, bool fast, hipStream_t stream) {
  if (o.M <= FEW_ROWS) return launch_few<FMT, Codes, Y>(o, stream);
  if constexpr (sizeof(Y) == 2)
    if (fast) return launch_tiles<FMT, Y, false>(o, stream);
  return launch_tiles<FMT, Y, true>(o, stream);
}

// GANET_FAST beside a type
bool fast_of(int32_t type) { return type >= 0 && (type & GANET_FAST); }
int32_t type_of(int32_t type) { return type < 0 ? type : type & ~GANET_FAST; }

// Whether few rows are packed inside the product's kernel: by what a CU has to pack then (16 rows, 4096 columns of the result, 1024 of the
// rows: one unit, of fp32 two). Inside / with a launch of its own, twenty in a graph, bf16: 1 x 1024 x 1024 4.9 / 6.6 us, 1 x 4096 x 4096
// 7.4 / 7.5, 1 x 8192 x 4096 12.1 / 11.0, 32 x 4096 x 4096 14.8 / 12.4; fp32: 1 x 1024 x 1024 5.7 / 6.5, 32 x 1024 x 4096 9.8 / 10.3, 1 x 4096 x 4096
// 8.2 / 7.4, 16 x 4096 x 4096 12.8 / 9.7.
bool packs_inside(int64_t M, int64_t N, int64_t K, int32_t type) {
  return M <= FEW_ROWS && cdiv(M, 16) * cdiv(N, 4096) * cdiv(K, 1024) * (type == GANET_F32 ? 2 : 1) <= 4;
}

bool held_ok(int64_t N, int64_t K, const void* c, int64_t ld, const uint8_t* e, int64_t le) {
  // (offsets inside a tile of 256 rows are 32 bits)
  return c && e && ld % 16 == 0 && ld >= pad16(K) && ld <= (1 << 24) && (reinterpret_cast<uintptr_t>(c) & 15) == 0 && le % 4 == 0 &&
         le >= cdiv(K, BLOCK) && le <= (1 << 24) && (reinterpret_cast<uintptr_t>(e) & 3) == 0;
}

// Where a buffer of ganet_rows8_bytes / ganet_weight8_bytes keeps its codes and exponents
struct Packed { uint8_t* codes; int64_t ldc; uint8_t* exps; int64_t lde; };
Packed packed(void* buffer, int64_t rows, int64_t cols) {
  const int64_t ldc = pad16(cols);
  uint8_t* b = static_cast<uint8_t*>(buffer);
  return {b, ldc, b + rows * ldc, (cdiv(cols, BLOCK) + 3) / 4 * 4};
}

}  // namespace
}  // namespace ganet

using namespace ganet;

extern "C" {

int ganet_gemm8(int64_t M, int64_t N, int64_t K, int32_t fmt, const void* codes, int64_t ldc, const uint8_t* exps, int64_t lde,
                const void* wcodes, int64_t ldwc, const uint8_t* wexps, int64_t ldwe, const void* bias, int32_t btype, void* y,
                int64_t ldy, int32_t ytypes, void* stream_) {
  const int32_t ytype = type_of(ytypes);
  const bool fast = fast_of(ytypes);
  if (!rows_ok(M, K) || N < 1 || N >= (1ll << 24) || (fmt != GANET_E4M3 && fmt != GANET_E5M2) || !type_ok(ytype) || !type_ok(btype)) {
    set_error("ganet_gemm8: unsupported M=%lld N=%lld K=%lld format=%d types=%d,%d", (long long)M, (long long)N, (long long)K, fmt,
              ytypes, btype);
    return 4;
  }
  if (M == 0) return 0;
  if (!y || (ldy < N && M > 1) || !held_ok(M, K, codes, ldc, exps, lde) || !held_ok(N, K, wcodes, ldwc, wexps, ldwe)) {
    set_error("ganet_gemm8: NULL or misaligned argument, or a row stride outside columns .. 2^24");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  const Operands o{M, N, K, static_cast<const uint8_t*>(codes), ldc, exps, lde, static_cast<const uint8_t*>(wcodes), ldwc, wexps,
                   ldwe, bias, btype, y, ldy};
  GANET_BY_TYPE(ytype, T, return fmt == GANET_E4M3 ? launch<GANET_E4M3, T>(o, fast, stream) : launch<GANET_E5M2, T>(o, fast, stream));
}

size_t ganet_rows8_bytes(int64_t M, int64_t C) {
  return rows_ok(M, C) ? (size_t)(M * pad16(C) + M * ((cdiv(C, BLOCK) + 3) / 4 * 4)) : 0;
}

size_t ganet_weight8_bytes(int64_t N, int64_t K) {
  return rows_ok(N, K) ? (size_t)(N * pad16(K) + cdiv(N, BLOCK) * ((cdiv(K, BLOCK) + 3) / 4 * 4)) : 0;
}

size_t ganet_linear8_held_workspace(int64_t M, int64_t N, int64_t K, int32_t type) {
  return packs_inside(M, N, K, type_of(type)) ? 0 : ganet_rows8_bytes(M, K);
}

int ganet_linear8_held(int64_t M, int64_t N, int64_t K, int32_t types, const void* x, int64_t ldx, const void* wcodes, int64_t ldwc,
                       const uint8_t* wexps, int64_t ldwe, const void* bias, int32_t btype, void* y, void* workspace,
                       size_t workspace_bytes, void* stream_) {
  const int32_t type = type_of(types);
  if (!rows_ok(M, K) || N < 1 || N >= (1ll << 24) || !type_ok(type) || !type_ok(btype)) {
    set_error("ganet_linear8_held: unsupported M=%lld N=%lld K=%lld types=%d,%d", (long long)M, (long long)N, (long long)K, types, btype);
    return 4;
  }
  if (M == 0) return 0;
  if (!x || !y || (ldx < K && M > 1) || !held_ok(N, K, wcodes, ldwc, wexps, ldwe) ||
      workspace_bytes < ganet_linear8_held_workspace(M, N, K, type) || (!packs_inside(M, N, K, type) && !workspace)) {
    set_error("ganet_linear8_held: NULL or misaligned argument, a row stride or the workspace too small");
    return 1;
  }
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (packs_inside(M, N, K, type)) {
    const Operands o{M, N, K, static_cast<const uint8_t*>(x), ldx, nullptr, 0, static_cast<const uint8_t*>(wcodes), ldwc, wexps, ldwe,
                     bias, btype, y, N};
    GANET_BY_TYPE(type, T, return (launch_few<GANET_E4M3, T, T>(o, stream)));
  }
  const Packed r = packed(workspace, M, K);
  const int rc = ganet_rows8_pack(M, K, type, GANET_E4M3, x, ldx, r.codes, r.ldc, r.exps, r.lde, stream_);
  return rc ? rc : ganet_gemm8(M, N, K, GANET_E4M3, r.codes, r.ldc, r.exps, r.lde, wcodes, ldwc, wexps, ldwe, bias, btype, y, N, types,
                               stream_);
}

int ganet_linear8_fwd(int64_t M, int64_t N, int64_t K, int32_t types, const void* x, int64_t ldx, int32_t wtype, const void* w,
                      int64_t ldw, const void* bias, int32_t btype, void* y, void* rows8, void* weight8, void* tweight8,
                      void* stream_) {
  if (!rows_ok(M, K) || !rows_ok(N, K) || N < 1 || !rows8 || !weight8) {
    set_error("ganet_linear8_fwd: unsupported M=%lld N=%lld K=%lld, or a NULL buffer", (long long)M, (long long)N, (long long)K);
    return 4;
  }
  const Packed r = packed(rows8, M, K), p = packed(weight8, N, K), t = tweight8 ? packed(tweight8, K, N) : Packed{};
  int rc = ganet_rows8_pack(M, K, type_of(types), GANET_E4M3, x, ldx, r.codes, r.ldc, r.exps, r.lde, stream_);
  if (!rc) rc = ganet_weight8_pack(N, K, wtype, w, ldw, p.codes, p.ldc, p.exps, p.lde, t.codes, t.ldc, t.exps, t.lde, stream_);
  return rc ? rc : ganet_gemm8(M, N, K, GANET_E4M3, r.codes, r.ldc, r.exps, r.lde, p.codes, p.ldc, p.exps, p.lde, bias, btype, y, N,
                               types, stream_);
}

size_t ganet_linear8_bwd_workspace(int64_t M, int64_t N, int64_t K, int32_t type) {
  const size_t rows = (ganet_rows8_bytes(M, N) + 255) / 256 * 256;
  return rows + ganet_wgrad8_workspace(M, N, K, type_of(type));
}

int ganet_linear8_bwd(int64_t M, int64_t N, int64_t K, int32_t types, const void* g, int64_t ldg, const void* rows8,
                      const void* tweight8, void* dx, void* dW, void* db, int32_t wtype, void* workspace, size_t workspace_bytes,
                      void* stream_) {
  const int32_t type = type_of(types);
  if (!rows_ok(M, K) || !rows_ok(M, N) || N < 1 || workspace_bytes < ganet_linear8_bwd_workspace(M, N, K, type) || !workspace ||
      !rows8 || (dx && !tweight8)) {
    set_error("ganet_linear8_bwd: unsupported M=%lld N=%lld K=%lld, a NULL buffer, or the workspace too small", (long long)M,
              (long long)N, (long long)K);
    return 4;
  }
  int rc = 0;
  if (dx) {
    const Packed q = packed(workspace, M, N), t = packed(const_cast<void*>(tweight8), K, N);
    rc = ganet_rows8_pack(M, N, type, GANET_E4M3, g, ldg, q.codes, q.ldc, q.exps, q.lde, stream_);
    if (!rc)
      rc = ganet_gemm8(M, K, N, GANET_E4M3, q.codes, q.ldc, q.exps, q.lde, t.codes, t.ldc, t.exps, t.lde, nullptr, GANET_F32, dx, K, types,
                       stream_);
  }
  if (rc || !dW) return rc;
  const Packed r = packed(const_cast<void*>(rows8), M, K);
  uint8_t* ws = static_cast<uint8_t*>(workspace) + (ganet_rows8_bytes(M, N) + 255) / 256 * 256;
  return ganet_wgrad8(M, N, K, GANET_E4M3, type, g, ldg, r.codes, r.ldc, r.exps, r.lde, dW, db, wtype, ws,
                      ganet_wgrad8_workspace(M, N, K, type), stream_);
}

}  // extern "C"
