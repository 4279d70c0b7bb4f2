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

// scales and biases of W consecutive columns of a lane (columns behind N: zero)
template <int W> struct Cols { float s[W], b[W]; };
template <int W> __device__ __forceinline__ Cols<W> cols(const GemmQ8& p, int n) {
  Cols<W> c;
#pragma unroll
  for (int r = 0; r < W; ++r) {
    c.s[r] = n + r < p.N ? p.sB[n + r] : 0.f;
    c.b[r] = p.bias && n + r < p.N ? p.bias[n + r] : 0.f;
  }
  return c;
}
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
template <int W> struct Raw;                                              // W bf16 values as loaded and stored
template <> struct Raw<4> { typedef u32x2 T; };
template <> struct Raw<8> { typedef u32x4 T; };
// epilogue and store of W columns n .. n + W - 1 of row m; v = alpha * sA[m] * sum; res = the residual there (all of them inside N)
template <int W> __device__ __forceinline__ void finish(const GemmQ8& p, float (&v)[W], const Cols<W>& c, const typename Raw<W>::T& res, int m, int n) {
#pragma unroll
  for (int r = 0; r < W; ++r) v[r] = v[r] * c.s[r] + c.b[r];
  if (p.act == V2S_ACT_RELU) {
#pragma unroll
    for (int r = 0; r < W; ++r) v[r] = v[r] < 0.f ? 0.f : v[r];           // keeps NaN
  } else if (p.act == V2S_ACT_GELU) {
#pragma unroll 1
    for (int r = 0; r < W; ++r) v[r] = gelu_f(v[r]);
  }
  const long at = (long)m * p.ldc + n;
  if (n + W <= p.N) {
    if (p.residual) {
#pragma unroll
      for (int r = 0; r < W / 2; ++r) { v[2 * r] += __uint_as_float(res[r] << 16); v[2 * r + 1] += __uint_as_float(res[r] & 0xffff0000u); }
    }
    if (p.c_f32) {
#pragma unroll
      for (int r = 0; r < W / 4; ++r) *reinterpret_cast<float4*>((float*)p.C + at + 4 * r) = make_float4(v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]);
    } else {
      typename Raw<W>::T o;
#pragma unroll
      for (int r = 0; r < W / 2; ++r) o[r] = pack2bf(v[2 * r], v[2 * r + 1]);
      *reinterpret_cast<typename Raw<W>::T*>((bf16_t*)p.C + at) = o;
    }
  } else {
#pragma unroll 1
    for (int r = 0; r < W && n + r < p.N; ++r) {
      float x = v[r];
      if (p.residual) x += bf2f(p.residual[(long)m * p.ldr + n + r]);
      if (p.c_f32) ((float*)p.C)[at + r] = x;
      else ((bf16_t*)p.C)[at + r] = f2bf(x);
    }
  }
}
template <int W> __device__ __forceinline__ typename Raw<W>::T residual_of(const GemmQ8& p, int m, int n) {
  typename Raw<W>::T z = {};
  if (p.residual && m < p.M && n + W <= p.N) z = *reinterpret_cast<const typename Raw<W>::T*>(p.residual + (long)m * p.ldr + n);
  return z;
}

// ---- tiles -------------------------------------------------------------------------------------------------------------------------------
// BM x BN tile, 4 waves of (BM / 2) x (BN / 2); K in stages of 64 codes through a ring of three LDS images [BM + BN rows][64 bytes] that the LDS-DMA
// fills (global_load_lds, 1 KiB = 16 rows per wave and instruction; two stages in flight, counted waits, one barrier per stage).
// A row's four 16-byte groups are stored at group ^ (((row >> 2) & 1) << 1), which spreads the eight rows that a fragment read serves at once.
// K need not be a multiple of 64: in the last stage lanes whose group lies behind K load the row's first group again (in bounds), and A's fragments
// are zeroed there.
__device__ __forceinline__ uint32_t lds_off(const void* p) { return (uint32_t)(uintptr_t)(V2S_LDS const char*)p; }
// one instruction: 16 bytes per lane from base + off to LDS at dst + lane * 16
__device__ __forceinline__ void dma16(uint32_t off, const void* base, uint32_t dst) {
  uint32_t keep;
  asm volatile("s_mov_b32 %[keep], m0\n\ts_mov_b32 m0, %[dst]\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %[off], %[base]\n\ts_mov_b32 m0, %[keep]"
               : [keep] "=&s"(keep) : [dst] "s"(dst), [base] "s"(base), [off] "v"(off) : "memory");
}

template <int BM, int BN>
struct Tile {
  static constexpr int DA = BM / 64, DB = BN / 64;          // DMA instructions per wave and stage
  static constexpr int MI = BM / 32, NI = BN / 32;          // 16 x 16 fragments per wave
  static constexpr int STG = (BM + BN) * 64, NST = 3;
};

template <int BM, int BN>
__global__ __launch_bounds__(256, 2) void gemm_q8_tile_kernel(const GemmQ8 p) {
  using G = Tile<BM, BN>;
  constexpr int DA = G::DA, DB = G::DB, MI = G::MI, NI = G::NI, STG = G::STG;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = xcd_remap(blockIdx.x, p.tilesM * p.tilesN);
  const int m0 = id / p.tilesN * BM, n0 = id % p.tilesN * BN;
  const int wm = (wave >> 1) * (BM / 2), wn = (wave & 1) * (BN / 2);
  const int nst = (p.K + 63) >> 6, krem = p.K - (nst - 1) * 64;
  const uint32_t sbase = lds_off(smem);

  uint32_t oa[DA], ob[DB];
  const int rl = lane >> 2, gl = (lane & 3) ^ (((rl >> 2) & 1) << 1);       // row within a 1 KiB piece, the group this lane loads
#pragma unroll
  for (int i = 0; i < DA; ++i) oa[i] = (uint32_t)min((wave * DA + i) * 16 + rl, p.M - 1 - m0) * (uint32_t)p.lda + gl * 16;
#pragma unroll
  for (int i = 0; i < DB; ++i) ob[i] = (uint32_t)min((wave * DB + i) * 16 + rl, p.N - 1 - n0) * (uint32_t)p.ldb + gl * 16;
  const i8* ga = p.A + (long)m0 * p.lda;
  const i8* gb = p.B + (long)n0 * p.ldb;
  auto issue = [&](int s) {
    const uint32_t slot = sbase + (s % 3) * STG;
    const uint32_t back = s == nst - 1 && gl * 16 >= krem ? gl * 16 : 0;
#pragma unroll
    for (int i = 0; i < DA; ++i) dma16(oa[i] - back, ga + (long)s * 64, slot + (wave * DA + i) * 1024);
#pragma unroll
    for (int i = 0; i < DB; ++i) dma16(ob[i] - back, gb + (long)s * 64, slot + BM * 64 + (wave * DB + i) * 1024);
  };
  i32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  const int fr = lane & 15, fg = lane >> 4;
  const int foff = fr * 64 + ((fg ^ (((fr >> 2) & 1) << 1)) * 16);          // fragment rows start at multiples of 16

  issue(0);
  if (nst > 1) issue(1);
  for (int s = 0; s < nst; ++s) {
    // stage s has landed for this wave (stage s + 1 may be in flight) and its reads of the stage before are done; then the same for the block
    if (s + 1 < nst) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(DA + DB) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + 2 < nst) issue(s + 2);
    const char* sa = smem + (s % 3) * STG + wm * 64 + foff;
    const char* sb = smem + (s % 3) * STG + BM * 64 + wn * 64 + foff;
    i32x4 af[MI], bf[NI];
#pragma unroll
    for (int i = 0; i < MI; ++i) af[i] = *reinterpret_cast<const i32x4*>(sa + i * 1024);
#pragma unroll
    for (int j = 0; j < NI; ++j) bf[j] = *reinterpret_cast<const i32x4*>(sb + j * 1024);
    if (s == nst - 1 && krem < 64) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
        if (fg * 16 >= krem) af[i] = i32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[j], af[i], acc[i][j], 0, 0, 0);
  }
  // write-out in passes of 64 rows (two fragment rows of every wave) through LDS: the accumulators become fp32 with the row's scale on the way in, and
  // leave as 8 consecutive columns per lane, whole cache lines per row.  A lane keeps its columns, so their scales are loaded once; the residual of a
  // pass is requested before its values are staged
  constexpr int PB = BN + 4, CPR = BN / 8, RPI = 256 / CPR, NIT = 64 / RPI;        // pitch (floats), chunks per row, rows per iteration, iterations
  static_assert(64 * PB * 4 <= G::NST * STG, "a pass fits the ring");
  float* cs = reinterpret_cast<float*>(smem);
  const int n = n0 + (threadIdx.x % CPR) * 8, lr = threadIdx.x / CPR;
  const Cols<8> c = cols<8>(p, n);
  float sa[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) sa[i] = p.alpha * p.sA[min(m0 + wm + i * 16 + fr, p.M - 1)];
#pragma unroll
  for (int ps = 0; ps < MI / 2; ++ps) {
    // staged row r of the pass is row (r >> 5) * BM / 2 + ps * 32 + (r & 31) of the tile
    auto row_of = [&](int r) { return m0 + (r >> 5) * (BM / 2) + ps * 32 + (r & 31); };
    u32x4 res[NIT];
#pragma unroll
    for (int it = 0; it < NIT; ++it) res[it] = residual_of<8>(p, row_of(it * RPI + lr), n);
    __syncthreads();
#pragma unroll
    for (int ii = 0; ii < 2; ++ii)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const i32x4 v = acc[ps * 2 + ii][j];
        const float x = sa[ps * 2 + ii];
        *reinterpret_cast<float4*>(cs + ((wave >> 1) * 32 + ii * 16 + fr) * PB + wn + j * 16 + fg * 4) =
            make_float4((float)v[0] * x, (float)v[1] * x, (float)v[2] * x, (float)v[3] * x);
      }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const int r = it * RPI + lr, m = row_of(r);
      if (m < p.M && n < p.N) {
        const float4 x = *reinterpret_cast<const float4*>(cs + r * PB + (threadIdx.x % CPR) * 8), y = *reinterpret_cast<const float4*>(cs + r * PB + (threadIdx.x % CPR) * 8 + 4);
        float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        finish<8>(p, v, c, res[it], m, n);
      }
    }
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------------
// Block = 16 MT rows x 16 NT columns; its waves split K (contiguous pieces: a wave uses whole cache lines of the weight) and load fragments straight
// from memory, every weight byte once per 16 MT rows; the partial sums meet in LDS as integers.
template <int WAVES, int MT, int NT>
__global__ __launch_bounds__(WAVES * 64) void gemm_q8_skinny_kernel(const GemmQ8 p) {
  constexpr int F = MT * NT, U = 3;
  __shared__ i32x4 red[WAVES][F][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const int steps = (p.K + 63) >> 6, per = (steps + WAVES - 1) / WAVES;
  const int end = min(steps, (wave + 1) * per);
  const i8 *pa[MT], *pb[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) pa[i] = p.A + (long)min(m0 + i * 16 + fr, p.M - 1) * p.lda;
#pragma unroll
  for (int j = 0; j < NT; ++j) pb[j] = p.B + (long)min(n0 + j * 16 + fr, p.N - 1) * p.ldb;
  i32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
  for (int s = wave * per; s < end; s += U) {
    i32x4 a[U][MT], b[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s + u) * 64 + fg * 16;
      const bool ok = s + u < end && k < p.K;
#pragma unroll
      for (int j = 0; j < NT; ++j) { b[u][j] = i32x4{0, 0, 0, 0}; if (ok) b[u][j] = *reinterpret_cast<const i32x4*>(pb[j] + k); }
#pragma unroll
      for (int i = 0; i < MT; ++i) { a[u][i] = i32x4{0, 0, 0, 0}; if (ok) a[u][i] = *reinterpret_cast<const i32x4*>(pa[i] + k); }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[u][j], a[u][i], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) red[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < (F + WAVES - 1) / WAVES; ++q) {
    const int f = q * WAVES + wave;
    if (f >= F) break;
    i32x4 v = red[0][f][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += red[w][f][lane];
    const int m = m0 + f / NT * 16 + fr, n = n0 + f % NT * 16 + fg * 4;
    if (m < p.M && n < p.N) {
      const float sa = p.alpha * p.sA[m];
      float x[4] = {(float)v[0] * sa, (float)v[1] * sa, (float)v[2] * sa, (float)v[3] * sa};
      finish<4>(p, x, cols<4>(p, n), residual_of<4>(p, m, n), m, n);
    }
  }
}

template <int BM, int BN> int tile_launch(GemmQ8& p, hipStream_t s) {
  constexpr int LDS = Tile<BM, BN>::STG * Tile<BM, BN>::NST;
  static bool attr = false;
  if (!attr) { (void)hipFuncSetAttribute((const void*)gemm_q8_tile_kernel<BM, BN>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS); attr = true; }
  p.tilesM = (p.M + BM - 1) / BM; p.tilesN = (p.N + BN - 1) / BN;
  V2S_CHECK((int64_t)p.tilesM * p.tilesN <= 0x7fffffff, V2S_ERR_SHAPE, "v2s_gemm_q8: too many tiles for one launch");
  hipLaunchKernelGGL((gemm_q8_tile_kernel<BM, BN>), dim3(p.tilesM * p.tilesN), dim3(256), LDS, s, p);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}
template <int WAVES, int MT, int NT> int skinny_launch(const GemmQ8& p, hipStream_t s) {
  hipLaunchKernelGGL((gemm_q8_skinny_kernel<WAVES, MT, NT>), dim3((p.N + 16 * NT - 1) / (16 * NT), (p.M + 16 * MT - 1) / (16 * MT)), dim3(WAVES * 64), 0, s, p);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}

}  // namespace

extern "C" int v2s_gemm_q8(const v2s_gemm_q8_args* a, void* stream) {
  V2S_CHECK(a && a->A && a->B && a->sA && a->sB && a->C, V2S_ERR_ARG, "v2s_gemm_q8: NULL pointer");
  V2S_CHECK(a->M > 0 && a->N > 0 && a->K > 0 && a->K % 16 == 0 && a->K <= 131056, V2S_ERR_SHAPE,
            "v2s_gemm_q8: unsupported shape M=%d N=%d K=%d (K a multiple of 16, <= 131056)", a->M, a->N, a->K);
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
  auto tiles = [&](int bm, int bn) { return (int64_t)((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
  int kind = v2s_opt_gemm_q8();
  if (kind == 0) kind = p.M <= 64 ? 1 : (tiles(128, 256) >= 512 ? 4 : (tiles(128, 128) >= 256 ? 3 : 2));
  if (kind == 4) return tile_launch<128, 256>(p, s);
  if (kind == 3) return tile_launch<128, 128>(p, s);
  if (kind == 2) return tile_launch<64, 64>(p, s);
  const bool wide = p.N >= 8192, deep = p.K > 1024;
  V2S_CHECK((p.M + 15) / 16 <= 65535, V2S_ERR_SHAPE, "v2s_gemm_q8: too many rows for the few-row kernels");
  if (p.M <= 16) return deep ? skinny_launch<8, 1, 1>(p, s) : (wide ? skinny_launch<4, 1, 4>(p, s) : skinny_launch<4, 1, 1>(p, s));
  if (p.M <= 32) return deep ? skinny_launch<8, 2, 1>(p, s) : (wide ? skinny_launch<4, 2, 4>(p, s) : skinny_launch<4, 2, 1>(p, s));
  return deep ? skinny_launch<8, 4, 1>(p, s) : (wide ? skinny_launch<4, 4, 4>(p, s) : skinny_launch<4, 4, 1>(p, s));
}
