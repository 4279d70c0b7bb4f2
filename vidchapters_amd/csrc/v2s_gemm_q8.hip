// int8 matrix product with a scale per token and per channel (gfx950):  C = act(alpha sA[m] sB[n] sum_k A[m][k] B[n][k] + bias[n]) + residual
// The products are summed exactly in int32 by v_mfma_i32_16x16x64_i8; scales and epilogue in fp32, one rounding to C.
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

// one value of the epilogue; everything after the exact integer sum is fp32
__device__ __forceinline__ float q8_epilogue(const GemmQ8& p, int acc, float sa, int m, int n) {
  float v = (float)acc * sa * p.sB[n];
  if (p.bias) v += p.bias[n];
  if (p.act == V2S_ACT_RELU) v = v < 0.f ? 0.f : v;          // keeps NaN
  else if (p.act == V2S_ACT_GELU) v = gelu_f(v);
  if (p.residual) v += bf2f(p.residual[(long)m * p.ldr + n]);
  return v;
}

// 64 x 64 tile, 4 waves of 32 x 32, K in steps of 64 through LDS (pitch 80 bytes); K is a multiple of 16, the rest of the last step is zero
constexpr int PITCH = 80;
__global__ __launch_bounds__(256) void gemm_q8_kernel(const GemmQ8 p) {
  __shared__ __attribute__((aligned(16))) char sa[64 * PITCH], sb[64 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int tm = blockIdx.x / p.tilesN, tn = blockIdx.x % p.tilesN;
  const int m0 = tm * 64, n0 = tn * 64;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  const int lr = tid >> 2, lk = (tid & 3) * 16;
  const i8* ga = p.A + (long)min(m0 + lr, p.M - 1) * p.lda;
  const i8* gb = p.B + (long)min(n0 + lr, p.N - 1) * p.ldb;
  i32x4 acc[2][2] = {};
  for (int k0 = 0; k0 < p.K; k0 += 64) {
    uint4 va = make_uint4(0, 0, 0, 0), vb = va;
    if (k0 + lk < p.K) {
      va = *reinterpret_cast<const uint4*>(ga + k0 + lk);
      vb = *reinterpret_cast<const uint4*>(gb + k0 + lk);
    }
    __syncthreads();
    *reinterpret_cast<uint4*>(sa + lr * PITCH + lk) = va;
    *reinterpret_cast<uint4*>(sb + lr * PITCH + lk) = vb;
    __syncthreads();
    i32x4 af[2], bf[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      af[i] = *reinterpret_cast<const i32x4*>(sa + (wm + i * 16 + (lane & 15)) * PITCH + (lane >> 4) * 16);
      bf[i] = *reinterpret_cast<const i32x4*>(sb + (wn + i * 16 + (lane & 15)) * PITCH + (lane >> 4) * 16);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(af[i], bf[j], acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = m0 + wm + i * 16 + (lane >> 4) * 4 + r;
      if (m >= p.M) continue;
      const float s = p.alpha * p.sA[m];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int n = n0 + wn + j * 16 + (lane & 15);
        if (n >= p.N) continue;
        const float v = q8_epilogue(p, acc[i][j][r], s, m, n);
        if (p.c_f32) ((float*)p.C)[(long)m * p.ldc + n] = v;
        else ((bf16_t*)p.C)[(long)m * p.ldc + n] = f2bf(v);
      }
    }
}

}  // namespace

extern "C" int v2s_gemm_q8(const v2s_gemm_q8_args* a, void* stream) {
  V2S_CHECK(a && a->A && a->B && a->sA && a->sB && a->C, V2S_ERR_ARG, "v2s_gemm_q8: NULL pointer");
  V2S_CHECK(a->M > 0 && a->N > 0 && a->K > 0 && a->K % 16 == 0 && a->K <= 131056, V2S_ERR_SHAPE,
            "v2s_gemm_q8: unsupported shape M=%d N=%d K=%d (K a multiple of 16, <= 131056)", a->M, a->N, a->K);
  V2S_CHECK(a->lda >= a->K && a->ldb >= a->K && a->ldc >= a->N && (!a->residual || a->ldr >= a->N), V2S_ERR_SHAPE, "v2s_gemm_q8: a row stride is shorter than the row");
  V2S_CHECK(a->c_dtype == V2S_BF16 || a->c_dtype == V2S_F32, V2S_ERR_DTYPE, "v2s_gemm_q8: C must be bf16 or fp32");
  V2S_CHECK(a->act == V2S_ACT_NONE || a->act == V2S_ACT_RELU || a->act == V2S_ACT_GELU, V2S_ERR_ARG, "v2s_gemm_q8: unknown activation %d", a->act);
  V2S_CHECK(((uintptr_t)a->A | (uintptr_t)a->B | (uintptr_t)a->C | (uintptr_t)a->residual) % 16 == 0 && (a->lda | a->ldb) % 16 == 0 && a->ldc % 8 == 0 &&
                (!a->residual || a->ldr % 8 == 0) && ((uintptr_t)a->sA | (uintptr_t)a->sB | (uintptr_t)a->bias) % 4 == 0,
            V2S_ERR_ALIGN, "v2s_gemm_q8: A, B, C and residual must be 16-byte aligned, lda / ldb multiples of 16, ldc / ldr multiples of 8");
  GemmQ8 p;
  p.M = a->M; p.N = a->N; p.K = a->K; p.A = (const i8*)a->A; p.B = (const i8*)a->B; p.lda = a->lda; p.ldb = a->ldb; p.sA = a->sA; p.sB = a->sB;
  p.C = a->C; p.ldc = a->ldc; p.c_f32 = a->c_dtype == V2S_F32; p.alpha = a->alpha; p.bias = a->bias; p.act = a->act;
  p.residual = (const bf16_t*)a->residual; p.ldr = a->ldr;
  p.tilesM = (a->M + 63) / 64; p.tilesN = (a->N + 63) / 64;
  V2S_CHECK((int64_t)p.tilesM * p.tilesN <= 0x7fffffff, V2S_ERR_SHAPE, "v2s_gemm_q8: too many tiles for one launch");
  hipLaunchKernelGGL(gemm_q8_kernel, dim3(p.tilesM * p.tilesN), dim3(256), 0, (hipStream_t)stream, p);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}
