// int8 matrix product with a scale per token and per channel (gfx950):  C = act(alpha sA[m] sB[n] sum_k A[m][k] B[n][k] + bias[n]) + residual
// The products are summed exactly in int32 (v_mfma_i32_16x16x64_i8, 16 codes of A and of B per lane and instruction), so the result does not depend on
// which of the kernels below a call takes; scales and epilogue are fp32, one rounding to C.
// The accumulators are kept transposed (B is the first operand of the matrix instruction): a lane then owns four consecutive columns of one row.
// replaces model/modeling_t5.py:304-311,528-536,581,1714 (nn.Linear forward) where int8 operands are wanted
#include <math.h>
#include "v2s_common.h"

namespace {

typedef signed char i8;
typedef __attribute__((ext_vector_type(4))) int i32x4;

struct GemmQ8 {
  int M, N, K;
  const i8 *A, *B;
  long lda, ldb;
  const float *sA, *sB;
  void* C; long ldc; int c_f32;
  float alpha;
  const float* bias; int act;
  const bf16_t* residual; long ldr;
  int tilesM, tilesN;
};

typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
template <int W> struct Raw;                                              // W bf16 values as loaded and stored
template <> struct Raw<4> { typedef u32x2 T; };
template <> struct Raw<8> { typedef u32x4 T; };
// scales and biases of W consecutive columns of a lane (columns behind N take the last one's: they are not stored)
template <int W> struct Cols { float s[W], b[W]; };
template <int W> __device__ __forceinline__ Cols<W> cols(const GemmQ8& p, int n) {
  Cols<W> c;
#pragma unroll
  for (int r = 0; r < W; ++r) c.s[r] = p.sB[min(n + r, p.N - 1)];
#pragma unroll
  for (int r = 0; r < W; ++r) c.b[r] = 0.f;
  if (p.bias) {
#pragma unroll
    for (int r = 0; r < W; ++r) c.b[r] = p.bias[min(n + r, p.N - 1)];
  }
  return c;
}
template <int W> __device__ __forceinline__ typename Raw<W>::T residual_of(const GemmQ8& p, int m, int n) {
  typename Raw<W>::T z = {};
  if (m < p.M && n + W <= p.N) z = *reinterpret_cast<const typename Raw<W>::T*>(p.residual + (long)m * p.ldr + n);
  return z;
}
// elements e .. 7 of eight bf16 values, moved to the front
__device__ __forceinline__ u32x4 from_element(u32x4 r, int e) {
  const int d = e >> 1;
  const uint32_t a0 = d == 0 ? r[0] : d == 1 ? r[1] : d == 2 ? r[2] : r[3], a1 = d == 0 ? r[1] : d == 1 ? r[2] : d == 2 ? r[3] : 0;
  const uint32_t a2 = d == 0 ? r[2] : d == 1 ? r[3] : 0, a3 = d == 0 ? r[3] : 0;
  const uint32_t h = (e & 1) * 16;
  return u32x4{__builtin_amdgcn_alignbit(a1, a0, h), __builtin_amdgcn_alignbit(a2, a1, h), __builtin_amdgcn_alignbit(a3, a2, h), a3 >> h};
}
// 16 bytes, past the caches where a row is whole cache lines (12876 x 11520 x 240 to fp32: 132 instead of 144 us); pieces of a line that another tile completes
// go through them (8601 x 2696 x 1440: 57 instead of 69)
__device__ __forceinline__ void store16(u32x4 o, void* to, bool stream) {
  if (stream) {
    __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(to));
  } else {
    asm volatile("");                       // the two stay apart: merged into one store, they lose the hint
    *reinterpret_cast<u32x4*>(to) = o;
    asm volatile("");
  }
}
// exact-erf GELU v Phi(v), Phi(v) = 1 / (1 + exp(-L(v))), L(v) = log(Phi(v) / Phi(-v)) = v P(v^2).  P is a minimax polynomial on v^2 <= 36, held at its last value
// beyond; its coefficients carry the factor -log2 e.  Errors are relative to v, in half steps of fp32 (2^-24 |v|); far below zero, where v Phi(v) is small, they bound
// no digit of the result (at v = -6 it is -1.9e-10 instead of -5.9e-9).
// To bf16: degree six, 3.6 half steps at most, the 2^-14th part of the rounding that follows.  19 cycles' worth of instructions a value, a quarter less than a form with the
// two tails of erfc apart, four cycles less than the one below (26346 x 2488 x 400: 82 and 91 us).
__device__ __forceinline__ float gelu_bf16(float v) {
  const float s = fminf(v * v, 36.0f);
  float t = fmaf(-5.209905840e-9f, s, 3.850448422e-7f);
  t = fmaf(t, s, -1.145242732e-5f); t = fmaf(t, s, 1.593893976e-4f); t = fmaf(t, s, 9.559299360e-5f); t = fmaf(t, s, -0.1048385799f); t = fmaf(t, s, -2.302207232f);
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * t));
}
// To fp32, where they show: degree seven, weighted by the error relative to v (0.44), and the smaller one of Phi and 1 - Phi: max(v, 0) - |v| T, T = Phi(-|v|) = e / (1 + e).
// With every rounding and one unit each of the chip's exp2 and reciprocal 3.2 half steps at most, 1.8 where these two round correctly (0.5 v (1 + erf): 1.8).
__device__ __forceinline__ float gelu_f32(float v) {
  const float s = fminf(v * v, 36.0f);
  float t = fmaf(-3.890140360e-11f, s, -3.379016307e-09f);
  t = fmaf(t, s, 3.545590694e-07f); t = fmaf(t, s, -1.123694268e-05f); t = fmaf(t, s, 1.588383633e-04f); t = fmaf(t, s, 9.530487809e-05f);
  t = fmaf(t, s, -1.048359587e-01f); t = fmaf(t, s, -2.302209154e+00f);
  const float a = fabsf(v), e = __builtin_amdgcn_exp2f(a * t);
  const float g = fmaf(-a, e * __builtin_amdgcn_rcpf(1.0f + e), fmaxf(v, 0.f));
  return v > 8.f ? v : g;                    // infinity has no product with T = 0; -infinity gives NaN
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}
// W values v = alpha * sA[m] * sum with their columns' scales and biases: activation
template <int W, bool GELU> __device__ __forceinline__ void activate(const GemmQ8& p, float (&v)[W], const Cols<W>& c) {
#pragma unroll
  for (int r = 0; r < W; ++r) v[r] = v[r] * c.s[r] + c.b[r];
  if (GELU && p.act == V2S_ACT_GELU) {
    if (p.c_f32) {
#pragma unroll
      for (int r = 0; r < W; ++r) v[r] = gelu_f32(v[r]);
    } else {
#pragma unroll
      for (int r = 0; r < W; ++r) v[r] = gelu_bf16(v[r]);
    }
  }
  if (p.act == V2S_ACT_RELU) {
#pragma unroll
    for (int r = 0; r < W; ++r) v[r] = v[r] < 0.f ? 0.f : v[r];           // keeps NaN
  }
}
template <int W> __device__ __forceinline__ void add_residual(float (&v)[W], const typename Raw<W>::T& res) {
#pragma unroll
  for (int r = 0; r < W / 2; ++r) { v[2 * r] += __uint_as_float(res[r] << 16); v[2 * r + 1] += __uint_as_float(res[r] & 0xffff0000u); }
}
template <int W> __device__ __forceinline__ typename Raw<W>::T pack(const float (&v)[W]) {
  typename Raw<W>::T o;
#pragma unroll
  for (int r = 0; r < W / 2; ++r) o[r] = pack_bf16(v[2 * r], v[2 * r + 1]);
  return o;
}
// the rest of the epilogue of four columns n .. n + 3 of row m, cut by N; res: their residual where N does not cut them
__device__ __forceinline__ void finish4(const GemmQ8& p, float (&v)[4], const Cols<4>& c, u32x2 res, int m, int n) {
  activate<4, true>(p, v, c);
  const long at = (long)m * p.ldc + n;
  if (n + 4 <= p.N) {
    if (p.residual) add_residual<4>(v, res);
    if (p.c_f32) *reinterpret_cast<float4*>((float*)p.C + at) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<u32x2*>((bf16_t*)p.C + at) = pack<4>(v);
  } else {
#pragma unroll
    for (int r = 0; r < 3; ++r)
      if (n + r < p.N) {
        if (p.residual) v[r] += bf2f(p.residual[(long)m * p.ldr + n + r]);
        if (p.c_f32) ((float*)p.C)[at + r] = v[r];
        else ((bf16_t*)p.C)[at + r] = f2bf(v[r]);
      }
  }
}

// ---- tiles -------------------------------------------------------------------------------------------------------------------------------
// BM x BN tile, WM x WN waves; K in stages of 128 codes (a cache line per row: with 64-byte pieces the L2 served twice the requests and the 8192^3
// product ran at 1617 TOPS instead of 2363) through two LDS images [BM + BN rows][128 bytes] that the LDS-DMA fills (global_load_lds, 1 KiB = 8 rows
// per wave and instruction), one barrier per stage, D = 3 steps before its end: by then every fragment of the stage has been read (they run three steps ahead
// of their products), so its image is free for stage s + 2, and the first reads of stage s + 1 wait under the last products.
// A row's eight 16-byte groups are stored at group ^ f(row): the sixteen rows of a fragment read fall into different banks.
// Fragment j of B takes the rows (r >> 2) * 4 NI + 4 j + (r & 3) of the wave's 16 NI, so that a lane ends up with 4 NI consecutive columns of a row; the
// write-out passes them through LDS rows of the wave's own, without a barrier, so that its stores are whole cache lines.
// Blocks are persistent: the first two stages of the next tile are requested before the write-out of the current one and arrive under it; the counted
// waits let its stores drain under those two stages.  In the 256 x 256 kernels that holds in part only: the compiler spills 15 (plain) and 11 (residual) registers,
// and a reload waits for all that the wave has in flight, which here is requests of the next tile, and stores of the last one (the counted waits stay right: more
// operations in flight only make them longer).
// 8192^3: 402 us = 2739 TOPS, 16384 x 1024 x 4096 with residual 57 to 60 us = 2400 TOPS when the same operands come again, 67 to 75 when they change: MFMA rate at the clock
// that its power allows.  27501 x 2304 x 768: 62 to 69 us = 1400 to 1570 TOPS: six stages a tile, then a write-out that no products cover (a block fills its CU: the
// accumulators take half of its registers).
// K need not be a multiple of 128: in the last stage lanes whose group lies behind K load the row's first group again (in bounds), and A's fragments
// are zeroed there.
__device__ __forceinline__ uint32_t lds_off(const void* p) { return (uint32_t)(uintptr_t)(V2S_LDS const char*)p; }
// one instruction: 16 bytes per lane from base + off to LDS at dst + lane * 16
__device__ __forceinline__ void dma16(uint32_t off, const void* base, uint32_t dst) {
  uint32_t keep;
  asm volatile("s_mov_b32 %[keep], m0\n\ts_mov_b32 m0, %[dst]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[off], %[base]\n\ts_mov_b32 m0, %[keep]"
               : [keep] "=&s"(keep) : [dst] "s"(dst), [base] "s"(base), [off] "v"(off) : "memory");
}
// every DMA but the youngest N operations of this wave has landed and its LDS reads are done; then the same for the block
template <int N> __device__ __forceinline__ void wait_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// What lanes of a wave pass to each other through LDS needs no wait (a wave's LDS operations keep their order), but the compiler, which sees one lane, has to
// be told that the words may have changed
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int BM_, int BN_, int WM_, int WN_, int OCC_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, OCC = OCC_, BK = 128;      // OCC: blocks per CU
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int DA = BM / 8 / WAVES, DB = BN / 8 / WAVES;            // DMA instructions per wave and stage
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;                // 16 x 16 fragments per wave
  static constexpr int STORES = MI * NI / 2;                                // 16-byte stores per wave of a whole bf16 tile
  static constexpr int OUT = 16 * NI * 32;                                   // bytes of 16 bf16 rows of a wave
  static constexpr int STG = (BM + BN) * BK, LDS = 2 * STG + WAVES * OUT + (BM + 2 * BN) * 4;
  static __device__ __forceinline__ int swzA(int row) { return (row >> 1) & 7; }
  static __device__ __forceinline__ int swzB(int row) { return ((row >> 1) & 1) | ((row / (NI * 4) & 3) << 1); }
};

// what a kernel's write-out can do: bf16 with none / ReLU, the same with a residual, everything.  The 256 x 256 tile comes in the first two forms, whose spills are few;
// GELU and fp32 take 128 x 128 tiles
enum { EPI_PLAIN, EPI_RESIDUAL, EPI_ANY };

template <class G, int EPI>
__global__ __launch_bounds__(G::THREADS, G::WAVES * G::OCC / 4) void gemm_q8_tile_kernel(const GemmQ8 p) {
  const bool has_res = EPI == EPI_RESIDUAL || (EPI == EPI_ANY && p.residual), f32 = EPI == EPI_ANY && p.c_f32;
  constexpr int BM = G::BM, BN = G::BN, BK = G::BK, DA = G::DA, DB = G::DB, MI = G::MI, NI = G::NI, STG = G::STG, DD = DA + DB;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* const s_a = reinterpret_cast<float*>(smem + 2 * STG + G::WAVES * G::OUT);      // scales of the tile's rows, scales and bias of its columns
  float* const s_b = s_a + BM;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / G::WN * (MI * 16), wn = wave % G::WN * (NI * 16);
  const int nst = (p.K + BK - 1) / BK, krem = p.K - (nst - 1) * BK;
  const int ntiles = p.tilesM * p.tilesN, nwg = gridDim.x;
  const uint32_t sbase = lds_off(smem);
  const int rl = lane >> 3, pos = lane & 7;             // row within a 1 KiB piece, 16-byte position within the row
  const int fr = lane & 15, fg = lane >> 4;
  int aoff[2], boff[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    aoff[k] = (wm + fr) * BK + ((k * 4 + fg) ^ G::swzA(fr)) * 16;
    const int br = (fr >> 2) * (NI * 4) + (fr & 3);
    boff[k] = (BM + wn + br) * BK + ((k * 4 + fg) ^ G::swzB(br)) * 16;
  }

  int m0 = 0, n0 = 0;
  uint32_t oa[DA], ob[DB];
  const i8 *ga = nullptr, *gb = nullptr;
  // tile of this block in round r: blocks of one XCD work on neighbouring tiles, four tile rows deep
  auto place = [&](int r) {
    const int id = r * nwg + xcd_remap(blockIdx.x, min(nwg, ntiles - r * nwg));
    const int per = 4 * p.tilesN, grp = id / per, in = id - grp * per, deep = min(4, p.tilesM - grp * 4);
    m0 = (grp * 4 + in % deep) * BM;
    n0 = in / deep * BN;
#pragma unroll
    for (int i = 0; i < DA; ++i) {
      const int row = (wave * DA + i) * 8 + rl;
      oa[i] = (uint32_t)min(row, p.M - 1 - m0) * (uint32_t)p.lda + (pos ^ G::swzA(row)) * 16;
    }
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      const int row = (wave * DB + i) * 8 + rl;
      ob[i] = (uint32_t)min(row, p.N - 1 - n0) * (uint32_t)p.ldb + (pos ^ G::swzB(row)) * 16;
    }
    ga = p.A + (long)m0 * p.lda;
    gb = p.B + (long)n0 * p.ldb;
  };
  auto piece = [&](int s, int x) {          // one of the DA + DB DMA instructions of a stage
    const uint32_t slot = sbase + (s & 1) * STG;
    const int lim = s == nst - 1 ? krem : BK;
    if (x < DA) {
      const int g = (pos ^ G::swzA((wave * DA + x) * 8 + rl)) * 16;
      dma16(oa[x] - (g >= lim ? g : 0), ga + (long)s * BK, slot + (wave * DA + x) * 1024);
    } else {
      const int y = x - DA, g = (pos ^ G::swzB((wave * DB + y) * 8 + rl)) * 16;
      dma16(ob[y] - (g >= lim ? g : 0), gb + (long)s * BK, slot + BM * BK + (wave * DB + y) * 1024);
    }
  };
  auto issue = [&](int s) {
#pragma unroll
    for (int x = 0; x < DD; ++x) piece(s, x);
  };

  place(0);
  issue(0);
  if (nst > 1) issue(1);
  bool stored = false;                      // at least STORES stores of this wave are younger than the stages 0 and 1
  for (int r = 0; r * nwg + (int)blockIdx.x < ntiles; ++r) {
    i32x4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    constexpr int SPT = (BM + BN + G::THREADS - 1) / G::THREADS, BPT = (BN + G::THREADS - 1) / G::THREADS;
    float sc[SPT], bi[BPT];
    // fragments: A's run D steps ahead of their products through a ring of four, B's k groups alternate between two sets
    constexpr int D = MI < 3 ? MI : 3;
    i32x4 af[4], bf[2][NI];
    auto read = [&](int s, int u) {         // step u of a stage: fragment u % MI of A in k group u / MI (with its first one, B's of that group)
      const char* st = smem + (s & 1) * STG;
      const int k = u / MI;
      if (u % MI == 0) {
#pragma unroll
        for (int j = 0; j < NI; ++j) bf[k][j] = *reinterpret_cast<const i32x4*>(st + boff[k] + j * 4 * BK);
      }
      af[u % 4] = *reinterpret_cast<const i32x4*>(st + aoff[k] + u % MI * 16 * BK);
    };
    auto multiply = [&](int u) {
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[u % MI][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[u / MI][j], af[u % 4], acc[u % MI][j], 0, 0, 0);
    };
    if (nst > 1) { if (stored) wait_barrier<DD + G::STORES>(); else wait_barrier<DD>(); }
    else if (stored) wait_barrier<G::STORES>();
    else wait_barrier<0>();
#pragma unroll
    for (int u = 0; u < D; ++u) read(0, u);
    for (int s = 0; s < nst - 1; ++s) {
      const bool head = s >= 1, tail = s + 2 < nst;
#pragma unroll
      for (int u = 0; u < 2 * MI; ++u) {
        // the requests of a stage go out PER a step (all at once they queue up in front of the block's products): the first ones behind the barrier, the
        // rest in the first steps of the next stage
        constexpr int PER = MI == 8 ? 1 : 2;
        const int t = u - (2 * MI - D);     // steps behind the barrier
        if (t == 0) {                       // the reads of stage s are done, stage s + 1 has landed: the image of stage s is free
          if (s == 0 && stored) wait_barrier<G::STORES>(); else wait_barrier<0>();
        }
        if (u + D < 2 * MI) read(s, u + D); else read(s + 1, u + D - 2 * MI);
        if (t >= 0) {
          if (tail) {
#pragma unroll
            for (int x = t * PER; x < (t + 1) * PER && x < DD; ++x) piece(s + 2, x);
          }
        } else if ((u + D) * PER < DD) {
          if (head) {
#pragma unroll
            for (int x = (u + D) * PER; x < (u + D + 1) * PER && x < DD; ++x) piece(s + 1, x);
          }
        }
        multiply(u);
        if ((u + D) % MI == 0) __builtin_amdgcn_sched_group_barrier(0x100, NI + 1, 0); else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, NI, 0);
      }
    }
    // last stage, the scales of the write-out on their way under it
#pragma unroll
    for (int x = 0; x < SPT; ++x) {
      const int i = tid + x * G::THREADS;
      sc[x] = i < BM ? p.sA[min(m0 + i, p.M - 1)] * p.alpha : p.sB[min(n0 + i - BM, p.N - 1)];
    }
#pragma unroll
    for (int x = 0; x < BPT; ++x) bi[x] = p.bias ? p.bias[min(n0 + tid + x * G::THREADS, p.N - 1)] : 0.f;
#pragma unroll
    for (int u = 0; u < 2 * MI; ++u) {
      if (u + D < 2 * MI) read(nst - 1, u + D);
      if (krem < BK && (u / MI * 4 + fg) * 16 >= krem) af[u % 4] = i32x4{0, 0, 0, 0};
      multiply(u);
    }
#pragma unroll
    for (int x = 0; x < SPT; ++x) if (tid + x * G::THREADS < BM + BN) s_a[tid + x * G::THREADS] = sc[x];
#pragma unroll
    for (int x = 0; x < BPT; ++x) if (tid + x * G::THREADS < BN) s_b[BN + tid + x * G::THREADS] = bi[x];
    const int m0w = m0 + wm, n0w = n0 + wn, tm = m0w + fr, tn = n0w + fg * (NI * 4);
    const bool more = (r + 1) * nwg + (int)blockIdx.x < ntiles;
    wait_barrier<0>();                      // scales visible, both stage images free
    // the next tile's first stages are requested, then 16 rows of the wave at a time: a lane finishes its 4 NI columns of one row, and the rows pass
    // through LDS of the wave's own (fp32 ones in two halves) so that its stores write whole cache lines.  The residual is requested AHEAD steps early.  A
    // group of 8 columns that N cuts takes the row's last 8 residuals from the right one on, and is stored by elements
    constexpr int Q = NI / 2, CPL = NI * 2, AHEAD = MI < 4 ? MI : 4;      // groups of 8 columns of a lane, 16-byte chunks per row
    const bf16_t* rp = p.residual + (long)tm * p.ldr + tn;
    typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t U4;
    const bool odd = p.N & 7;
    int cut[Q];                             // columns of a lane's group behind N
#pragma unroll
    for (int q = 0; q < Q; ++q) cut[q] = max(0, tn + q * 8 + 8 - p.N);
    u32x4 res[AHEAD][Q];
    auto fetch = [&](int i) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        res[i % AHEAD][q] = u32x4{0, 0, 0, 0};
        if (tm + i * 16 < p.M && cut[q] < 8) res[i % AHEAD][q] = *reinterpret_cast<const U4*>(rp + (long)i * 16 * p.ldr + q * 8 - cut[q]);
      }
    };
    if (has_res) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) fetch(i);
    }
    const int mlim = p.M - m0w, nlim = p.N - n0w;
    stored = m0 + BM <= p.M && n0 + BN <= p.N;
    if (more) {
      place(r + 1);
      issue(0);
      if (nst > 1) issue(1);
    }
    char* const out = smem + 2 * STG + wave * G::OUT;
    const float *sb = s_b + wn + fg * (NI * 4), *sa = s_a + wm + fr;
    const int sw = fr & (CPL - 1);
    const int ch = lane % CPL, row0 = lane / CPL;      // what the lane stores: chunk ch of the rows row0 + q * 64 / CPL
    const bool stream = (p.ldc * (f32 ? 4 : 2) | (long)(uintptr_t)p.C) % 128 == 0;
    const int left = nlim - ch * (f32 ? 4 : 8);          // columns from the lane's chunk on
    const long at = (long)(m0w + row0) * p.ldc + n0w + ch * (f32 ? 4 : 8);
    Cols<8> c[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int x = 0; x < 8; ++x) { c[q].s[x] = sb[q * 8 + x]; c[q].b[x] = sb[BN + q * 8 + x]; }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const float a = sa[i * 16];
      float v[Q][8];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
#pragma unroll
        for (int x = 0; x < 8; ++x) v[q][x] = (float)acc[i][q * 2 + (x >> 2)][x & 3] * a;
        activate<8, EPI == EPI_ANY>(p, v[q], c[q]);
        if (has_res) add_residual<8>(v[q], odd ? from_element(res[i % AHEAD][q], cut[q]) : res[i % AHEAD][q]);
      }
      if (has_res && i + AHEAD < MI) fetch(i + AHEAD);
      if (!f32) {
#pragma unroll
        for (int q = 0; q < Q; ++q) *reinterpret_cast<u32x4*>(out + fr * (NI * 32) + ((fg * Q + q) ^ sw) * 16) = pack<8>(v[q]);
        wave_sync();
#pragma unroll
        for (int q = 0; q < Q; ++q) {
          const int row = row0 + q * (64 / CPL);
          const u32x4 o = *reinterpret_cast<const u32x4*>(out + row * (NI * 32) + (ch ^ (row & (CPL - 1))) * 16);
          bf16_t* const to = (bf16_t*)p.C + at + (long)(i * 16 + q * (64 / CPL)) * p.ldc;
          if (i * 16 + row < mlim) {
            if (left >= 8) store16(o, to, stream);
            else if (odd) {
#pragma unroll
              for (int x = 0; x < 7; ++x) if (x < left) to[x] = (bf16_t)(o[x >> 1] >> (x & 1) * 16);
            }
          }
        }
      } else {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (fg >> 1 == hf) {
#pragma unroll
            for (int x = 0; x < NI; ++x)
              *reinterpret_cast<u32x4*>(out + fr * (NI * 32) + (((fg & 1) * NI + x) ^ sw) * 16) =
                  u32x4{__float_as_uint(v[x >> 1][(x & 1) * 4]), __float_as_uint(v[x >> 1][(x & 1) * 4 + 1]), __float_as_uint(v[x >> 1][(x & 1) * 4 + 2]),
                        __float_as_uint(v[x >> 1][(x & 1) * 4 + 3])};
          }
          wave_sync();
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            const int row = row0 + q * (64 / CPL);
            const u32x4 o = *reinterpret_cast<const u32x4*>(out + row * (NI * 32) + (ch ^ (row & (CPL - 1))) * 16);
            uint32_t* const to = (uint32_t*)p.C + at + (long)(i * 16 + q * (64 / CPL)) * p.ldc + hf * (NI * 8);
            if (i * 16 + row < mlim) {
              if (left - hf * (NI * 8) >= 4) store16(o, to, stream);
              else if (odd) {
#pragma unroll
                for (int x = 0; x < 3; ++x) if (x < left - hf * (NI * 8)) to[x] = o[x];
              }
            }
          }
          wave_sync();
        }
      }
      wave_sync();
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------------
// Block = 16 MT rows x 16 columns; its waves split K (contiguous pieces: a wave uses whole cache lines of the weight) and load fragments straight
// from memory, every weight byte once per 16 MT rows; the partial sums meet in LDS as integers.
template <int WAVES, int MT>
__global__ __launch_bounds__(WAVES * 64) void gemm_q8_skinny_kernel(const GemmQ8 p) {
  constexpr int U = 3;                  // steps asked for together
  static_assert(MT <= WAVES, "one wave writes 16 rows");
  __shared__ i32x4 red[WAVES][MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int steps = (p.K + 63) >> 6, per = (steps + WAVES - 1) / WAVES;
  const int end = min(steps, (wave + 1) * per);
  // what wave w < MT needs to finish 16 rows, asked for in front of the operands
  const int m = m0 + wave * 16 + fr, n = n0 + fg * 4;
  float sa = 0.f;
  Cols<4> c = {};
  u32x2 res = {};
  if (wave < MT) {
    sa = p.sA[min(m, p.M - 1)];
    c = cols<4>(p, n);
    if (p.residual) res = residual_of<4>(p, m, n);
  }
  const i8* pa[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) pa[i] = p.A + (long)min(m0 + i * 16 + fr, p.M - 1) * p.lda;
  const i8* pb = p.B + (long)min(n0 + fr, p.N - 1) * p.ldb;
  i32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = i32x4{0, 0, 0, 0};
  for (int s = wave * per; s < end; s += U) {
    i32x4 a[U][MT], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s + u) * 64 + fg * 16;
      const bool ok = s + u < end && k < p.K;
      b[u] = i32x4{0, 0, 0, 0};
      if (ok) b[u] = *reinterpret_cast<const i32x4*>(pb + k);
#pragma unroll
      for (int i = 0; i < MT; ++i) { a[u][i] = i32x4{0, 0, 0, 0}; if (ok) a[u][i] = *reinterpret_cast<const i32x4*>(pa[i] + k); }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[u], a[u][i], acc[i], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  if (wave >= MT) return;
  i32x4 v = red[0][wave][lane];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v += red[w][wave][lane];
  if (m >= p.M || n >= p.N) return;
  sa *= p.alpha;
  float x[4] = {(float)v[0] * sa, (float)v[1] * sa, (float)v[2] * sa, (float)v[3] * sa};
  finish4(p, x, c, res, m, n);
}

template <class G, int EPI> int tile_launch(GemmQ8& p, hipStream_t s) {
  static bool attr = false;
  if (!attr) { (void)hipFuncSetAttribute((const void*)gemm_q8_tile_kernel<G, EPI>, hipFuncAttributeMaxDynamicSharedMemorySize, G::LDS); attr = true; }
  p.tilesM = (p.M + G::BM - 1) / G::BM; p.tilesN = (p.N + G::BN - 1) / G::BN;
  const int64_t tiles = (int64_t)p.tilesM * p.tilesN;
  V2S_CHECK(tiles <= 0x3fffffff, V2S_ERR_SHAPE, "v2s_gemm_q8: too many tiles for one launch");
  hipLaunchKernelGGL((gemm_q8_tile_kernel<G, EPI>), dim3((unsigned)(tiles < 256 * G::OCC ? tiles : 256 * G::OCC)), dim3(G::THREADS), G::LDS, s, p);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}
typedef Tile<256, 256, 2, 4, 1> Tile256;
typedef Tile<128, 128, 2, 2, 2> Tile128;
typedef Tile<64, 64, 2, 2, 4> Tile64;
template <class G> int tile_any(GemmQ8& p, bool plain, hipStream_t s) {
  if (!plain) return tile_launch<G, EPI_ANY>(p, s);
  return p.residual ? tile_launch<G, EPI_RESIDUAL>(p, s) : tile_launch<G, EPI_PLAIN>(p, s);
}
template <int WAVES, int MT> int skinny_launch(GemmQ8 p, hipStream_t s) {
  constexpr int MOST = 65535 * 16 * MT;     // rows of one launch: a grid's y
  for (int left = p.M; left > 0; left -= MOST) {
    p.M = left < MOST ? left : MOST;
    hipLaunchKernelGGL((gemm_q8_skinny_kernel<WAVES, MT>), dim3((p.N + 15) / 16, (p.M + 16 * MT - 1) / (16 * MT)), dim3(WAVES * 64), 0, s, p);
    V2S_LAUNCH_CHECK();
    p.A += p.M * p.lda; p.sA += p.M; p.C = (char*)p.C + p.M * p.ldc * (p.c_f32 ? 4 : 2);
    if (p.residual) p.residual += p.M * p.ldr;
  }
  return V2S_OK;
}

}  // namespace

extern "C" int v2s_gemm_q8(const v2s_gemm_q8_args* a, void* stream) {
  V2S_CHECK(a && a->A && a->B && a->sA && a->sB && a->C, V2S_ERR_ARG, "v2s_gemm_q8: NULL pointer");
  V2S_CHECK(a->M > 0 && a->N > 0 && a->M <= 0x7fffff00 && a->N <= 0x7fffff00 && a->K > 0 && a->K % 16 == 0 && a->K <= 131056, V2S_ERR_SHAPE,
            "v2s_gemm_q8: unsupported shape M=%d N=%d K=%d (M, N <= 2^31 - 256, K a multiple of 16, <= 131056)", a->M, a->N, a->K);
  V2S_CHECK(a->lda >= a->K && a->ldb >= a->K && a->ldc >= a->N && (!a->residual || a->ldr >= a->N), V2S_ERR_SHAPE, "v2s_gemm_q8: a row stride is shorter than the row");
  V2S_CHECK(a->lda <= (1 << 24) && a->ldb <= (1 << 24), V2S_ERR_SHAPE, "v2s_gemm_q8: lda and ldb must be at most 2^24");
  V2S_CHECK(a->c_dtype == V2S_BF16 || a->c_dtype == V2S_F32, V2S_ERR_DTYPE, "v2s_gemm_q8: C must be bf16 or fp32");
  V2S_CHECK(a->act == V2S_ACT_NONE || a->act == V2S_ACT_RELU || a->act == V2S_ACT_GELU, V2S_ERR_ARG, "v2s_gemm_q8: unknown activation %d", a->act);
  V2S_CHECK(((uintptr_t)a->A | (uintptr_t)a->B | (uintptr_t)a->C | (uintptr_t)a->residual) % 16 == 0 && (a->lda | a->ldb) % 16 == 0 && a->ldc % 8 == 0 &&
                (!a->residual || a->ldr % 8 == 0) && ((uintptr_t)a->sA | (uintptr_t)a->sB | (uintptr_t)a->bias) % 4 == 0,
            V2S_ERR_ALIGN, "v2s_gemm_q8: A, B, C and residual must be 16-byte aligned, lda / ldb multiples of 16, ldc / ldr multiples of 8");
  GemmQ8 p;
  p.M = a->M; p.N = a->N; p.K = a->K; p.A = (const i8*)a->A; p.B = (const i8*)a->B; p.lda = a->lda; p.ldb = a->ldb; p.sA = a->sA; p.sB = a->sB;
  p.C = a->C; p.ldc = a->ldc; p.c_f32 = a->c_dtype == V2S_F32; p.alpha = a->alpha; p.bias = a->bias; p.act = a->act;
  p.residual = (const bf16_t*)a->residual; p.ldr = a->ldr; p.tilesM = p.tilesN = 0;
  hipStream_t s = (hipStream_t)stream;
  // Rounds of the chip's blocks times the time of one (us, n = stages of 128): 256 x 256 tiles 6.5 + 1.5 n, 128 x 128 3.0 + 0.95 n, 64 x 64 1.9 + 0.66 n, fitted to
  // N = 2304, K = 16 .. 3200: at K = 768, M = 1000 / 2000 / 8000 / 27501 they take 14.4 / 14.5 / 32.1 / 64.9, 8.0 / 10.1 / 22.5 / 70.7 and 7.3 / 10.1 / 27.2 / 108 us.
  // Few rows: a launch is bound by the latency of its operands, and the few-row kernels ask for all of them at once (64 x 2304 x 768: 4.3 us, 64 x 64 tiles 4.6;
  // 16 x 6000 x 1024: 4.2 and 5.4), until the rows read again for every 16 columns outweigh that (64 x 5000 x 768: 6.1 and 5.1, 64 x 32228 x 768: 18.5 and 9.5).
  // With more rows that comes earlier (400 x 300 x 4096: 10.2 and 12.8, 1000 x 128 x 768: 4.6 and 5.2; 300 x 1000 x 2000: 9.3 and 8.4, 7581 x 64 x 3488: 23 and 11).
  auto rounds = [&](int t, int slots) { return (double)(((int64_t)((p.M + t - 1) / t) * ((p.N + t - 1) / t) + slots - 1) / slots); };
  const double n = (p.K + 127) / 128;
  const double t4 = rounds(256, 256) * (6.5 + 1.5 * n), t3 = rounds(128, 512) * (3.0 + 0.95 * n), t2 = rounds(64, 1024) * (1.9 + 0.66 * n);
  int kind = v2s_opt_gemm_q8();
  const bool plain = !p.c_f32 && p.act != V2S_ACT_GELU;
  if (kind == 0) kind = (int64_t)p.M * p.N <= (p.M <= 64 ? 1 << 18 : 1 << 17) ? 1 : (plain && t4 <= t3 && t4 <= t2 ? 4 : (t3 <= t2 ? 3 : 2));
  if (p.N < 8) kind = 1;                    // the tiles read a cut group's residual as a row's last eight
  if (kind == 4 && plain) return p.residual ? tile_launch<Tile256, EPI_RESIDUAL>(p, s) : tile_launch<Tile256, EPI_PLAIN>(p, s);
  if (kind >= 3) return tile_any<Tile128>(p, plain, s);
  if (kind == 2) return tile_any<Tile64>(p, plain, s);
  const bool deep = p.K > 1024;
  const int64_t mb = (p.M + 15) / 16, nb = (p.N + 15) / 16;
  // rows of one block: 16 as long as that leaves the chip under two blocks per CU (64 x 1024 x 4096: 6.2 us, 64 rows 11.7), as many as there are otherwise
  // (64 x 4096 x 4096: 17 and 12 us)
  if (mb == 1 || mb * nb < 512) return deep ? skinny_launch<8, 1>(p, s) : skinny_launch<4, 1>(p, s);
  if (mb == 2) return deep ? skinny_launch<8, 2>(p, s) : skinny_launch<4, 2>(p, s);
  return deep ? skinny_launch<8, 4>(p, s) : skinny_launch<4, 4>(p, s);
}
