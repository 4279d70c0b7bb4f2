// 8-bit decoding for gfx950: rows of activations to int8 codes with one fp32 scale per row (with the residual addition and the RMSNorm in
// front of it), the int8 key / value cache, and the single-query attention that reads it.
//   code q and scale s of a row y:  s = max(amax|y|, 127 * 2^-126) / 127,  q = round_to_even(y * (127 / amax)).  s, that factor and the product are rounded
//   once each to fp32, so that |y - s q| <= s / 2 (1 + 2^-14)
// The floor of s keeps 1 / s finite: rows below it (1.5e-36) keep the smallest normal scale and fewer codes.  A row that holds a NaN or an
// infinity gets s = NaN and zero codes: every value that is read back is NaN, none of them is a plausible number.
//   RMSNorm: model/modeling_t5.py:263-277 (T5LayerNorm.forward); the cache it replaces: model/modeling_t5.py:555-556
#include <math.h>
#include "v2s_common.h"

namespace {

typedef signed char i8;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
constexpr float Q8_TINY = 127.0f * 1.17549435e-38f;

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// Reductions on the vector unit: rotations and mirrors within rows of 16 lanes, swaps of half waves and of odd and even rows across them (a shuffle through
// LDS has over ten times the latency, which is what a call of a few rows consists of).  Every lane gets the result.
template <int CTRL, class T> __device__ __forceinline__ T dpp(T v) {
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <class T, class F> __device__ __forceinline__ T half_reduce(T v, F f) {      // lane and lane ^ 32
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return f(__builtin_bit_cast(T, (uint32_t)a[0]), __builtin_bit_cast(T, (uint32_t)a[1]));
}
template <class T, class F> __device__ __forceinline__ T pair_reduce(T v, F f) {      // lane and lane ^ 16
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return f(__builtin_bit_cast(T, (uint32_t)a[0]), __builtin_bit_cast(T, (uint32_t)a[1]));
}
template <class T, class F> __device__ __forceinline__ T rows_reduce(T v, F f) { return pair_reduce(half_reduce(v, f), f); }      // the lanes with the same lane & 15
// over groups of LPR lanes; 256: a block, through red[4]
template <int LPR, class T, class F> __device__ __forceinline__ T group_reduce(T v, F f, T* red) {
  v = f(v, dpp<0x128>(v)); v = f(v, dpp<0x124>(v)); v = f(v, dpp<0x122>(v)); v = f(v, dpp<0x121>(v));      // row_ror 8, 4, 2, 1
  if (LPR >= 32) v = pair_reduce(v, f);
  if (LPR >= 64) v = half_reduce(v, f);
  if (LPR == 256) {
    red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = f(f(red[0], red[1]), f(red[2], red[3]));
  }
  return v;
}
struct Add { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};
// scale of a row whose largest magnitude has these bits (the maximum is taken on the bits: infinities and NaN are the largest), and 1 / scale; the quotient by
// 127 is the correctly rounded one (product with 1 / 127, corrected by its remainder)
__device__ __forceinline__ void q8_scale(uint32_t amax, float& scale, float& inv) {
  const float a = fmaxf(__uint_as_float(amax), Q8_TINY);
  const bool ok = amax < 0x7f800000u;
  const float s = a * (1.0f / 127.0f);
  scale = ok ? fmaf(fmaf(-127.0f, s, a), 1.0f / 127.0f, s) : __uint_as_float(0x7fc00000u);
  inv = ok ? 127.0f / a : 0.f;
}
__device__ __forceinline__ uint32_t q8_pack4(const float* y, float inv, bool ok) {
  const int a = (int)rintf(y[0] * inv), b = (int)rintf(y[1] * inv), c = (int)rintf(y[2] * inv), d = (int)rintf(y[3] * inv);
  const uint32_t r = (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
  return ok ? r : 0u;
}
__device__ __forceinline__ void q8_unpack4(uint32_t u, float* f) {
  f[0] = (float)(i8)(u & 255u); f[1] = (float)(i8)((u >> 8) & 255u); f[2] = (float)(i8)((u >> 16) & 255u); f[3] = (float)(i8)(u >> 24);
}

// eight values rounded to bf16 by v_cvt_pk_bf16_f32
__device__ __forceinline__ uint4 round8(const float* f) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{f[2 * i], f[2 * i + 1]}), bf16x2));
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// ---- rows -> codes ----------------------------------------------------------------------------------------------------------------------
struct RowsQ8 {
  const void* x; long ldx;
  const bf16_t* delta; long ldd;
  const float* w;
  bf16_t* h; long ldh;
  i8* q; long ldq;
  float* scale;
  int rows, cols;
  float eps;
};

__device__ __forceinline__ void ld8(const bf16_t* p, float* f) { unpack8(*reinterpret_cast<const uint4*>(p), f); }
__device__ __forceinline__ void ld8(const float* p, float* f) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// LPR lanes per row (a wave; fewer for a row shorter than half of one, a block for one longer than two), NCH chunks of 8 LPR columns held in registers: every byte is read once and written
// once.  32000 x 768 with the residual: 34 us, 5.05 TB/s (7 bytes per value); without norm from bf16 15.9 us, 4.6 TB/s, from fp32 22.7 us, 5.4 TB/s; 64 x 768: 3.1 to 3.8 us, a
// launch and one chain of loads and reductions.  A wave per row, in us for norm with residual / norm / codes of bf16 / of fp32: 24017 x 48 9.5 / 7.7 / 6.0 / 5.7 instead of 4.3 /
// 3.7 / 3.2 / 3.5, 64 x 4096 7.1 / 5.2 / 4.3 / 3.6 instead of 3.8 / 3.7 / 3.5 / 3.7, 4000 x 8192 97 / 53 / 30 / 33 instead of 47.5 / 25 / 22 / 31; at 4000 x 2048 both are
// equal (11.0 and 11.4, 7.3 and 7.8, 6.3 and 6.2, 7.6 and 8.0).
template <typename T, int NCH, int LPR, bool NORM>
__global__ __launch_bounds__(256) void rows_q8_kernel(const RowsQ8 p) {
  __shared__ float s_sum[4];
  __shared__ uint32_t s_max[4];
  const int lane = threadIdx.x & (LPR - 1);
  const int row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (row >= p.rows) return;
  const int nch = p.cols >> 3;
  const T* x = (const T*)p.x + (long)row * p.ldx;
  float v[NCH][8];
  float ss = 0.f;
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = lane + i * LPR;
    if (c < nch) {
      ld8(x + c * 8, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  float w[NCH][8];
  if (NORM) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) if (lane + i * LPR < nch) ld8(p.w + (lane + i * LPR) * 8, w[i]);      // under the row's reduction
    if (p.delta) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = lane + i * LPR;
        if (c < nch) {
          float d[8];
          ld8(p.delta + (long)row * p.ldd + c * 8, d);
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] += v[i][j];
          const uint4 s = round8(d);           // the residual stream is bf16: the norm sees the value that the next layer will read
          unpack8(s, v[i]);
          if (p.h) *reinterpret_cast<uint4*>(p.h + (long)row * p.ldh + c * 8) = s;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
    const float rstd = rsqrtf(group_reduce<LPR>(ss, Add(), s_sum) / p.cols + p.eps);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = lane + i * LPR;
      if (c < nch) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = w[i][j] * (v[i][j] * rstd);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) { const uint32_t b = abs_bits(v[i][j]); amax = amax > b ? amax : b; }
  amax = group_reduce<LPR>(amax, Max(), s_max);
  float scale, inv;
  q8_scale(amax, scale, inv);
  const bool ok = amax < 0x7f800000u;
  if (lane == 0) p.scale[row] = scale;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = lane + i * LPR;
    if (c < nch) {
      uint2 o;
      o.x = q8_pack4(v[i], inv, ok); o.y = q8_pack4(v[i] + 4, inv, ok);
      *reinterpret_cast<uint2*>(p.q + (long)row * p.ldq + c * 8) = o;
    }
  }
}

// y[row][c] = scale[row] * q[row][c], 8 columns per lane: bytes in, bytes out (32000 x 768: 14.3 us, 5.1 TB/s; 12.4 us where a cache still holds the codes)
__global__ __launch_bounds__(256) void dequant_q8_kernel(const i8* __restrict__ q, long ldq, const float* __restrict__ scale, bf16_t* __restrict__ y,
                                                         long ldy, int rows, int nch) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const int row = (int)(i / nch), c = (int)(i - (long)row * nch);
  if (i >= (long)rows * nch) return;
  const uint2 u = *reinterpret_cast<const uint2*>(q + (long)row * ldq + c * 8);
  const float s = scale[row];
  float f[8];
  q8_unpack4(u.x, f); q8_unpack4(u.y, f + 4);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] *= s;
  *reinterpret_cast<uint4*>(y + (long)row * ldy + c * 8) = round8(f);
}

// ---- key / value cache --------------------------------------------------------------------------------------------------------------------
// codes [.][64] and scales [.], row of (entry, head, token) = entry * e_rows + head * h_rows + token: the keys of one head are contiguous, a
// (sequence, head) of the attention streams whole cache lines
struct KvQ8 {
  i8 *kq, *vq;
  float *ks, *vs;
  long e_rows, h_rows;
  int E, H, maxlen, T;
  bf16_t *k, *v;                     // [E][T] rows of the attention's layout, head h at column h * 64
  long bs, rs;
  const int *pos, *pos_dev, *count;
  int pos0;
};

// Bound by HBM: 32 entries x 12 heads x up to 1100 tokens 32 us in and 24 us back, 3.9 and 5.2 TB/s, when operands and cache change from call to call (23.5 and 21.6 us, 5.3 and
// 5.7 TB/s, when the same come again); a single token by its chain of loads (2.9 us).
// eight lanes per (entry, head, token); TOKENS: eight tokens of one head per wave (512 contiguous bytes of codes), else eight heads of one token
template <bool TOKENS>
__device__ __forceinline__ bool kv_unit(const KvQ8& p, int& e, int& h, int& t) {
  const uint32_t u = blockIdx.x * 32u + (threadIdx.x >> 3);
  if (TOKENS) {
    const uint32_t tp = (uint32_t)(p.T + 7) & ~7u;
    const uint32_t eh = u / tp;
    t = (int)(u - eh * tp); h = (int)(eh % (uint32_t)p.H); e = (int)(eh / (uint32_t)p.H);
  } else {
    const uint32_t hp = (uint32_t)(p.H + 7) & ~7u;
    const uint32_t et = u / hp;
    h = (int)(u - et * hp); t = (int)(et % (uint32_t)p.T); e = (int)(et / (uint32_t)p.T);
  }
  return e < p.E && h < p.H && t < p.T;
}
// cache row of a unit; false if it takes no part, or has no row: a token behind the cache's end
__device__ __forceinline__ bool kv_row(const KvQ8& p, int e, int h, int t, long& row) {
  const long at = (long)(p.pos ? p.pos[e] : p.pos0) + (p.pos_dev ? *p.pos_dev : 0) + t;
  row = (long)e * p.e_rows + (long)h * p.h_rows + at;
  return !(p.count && t >= p.count[e]) && at >= 0 && at < p.maxlen;
}

template <bool TOKENS>
__global__ __launch_bounds__(256) void kv_append_q8_kernel(const KvQ8 p) {
  int e = 0, h = 0, t = 0;
  long row;
  if (!kv_unit<TOKENS>(p, e, h, t)) return;          // whole groups of eight lanes
  if (TOKENS && !kv_row(p, e, h, t, row)) return;
  const int c = threadIdx.x & 7;
  const long src = (long)e * p.bs + (long)t * p.rs + h * 64 + c * 8;
  const uint4 kr = *reinterpret_cast<const uint4*>(p.k + src), vr = *reinterpret_cast<const uint4*>(p.v + src);
  if (!TOKENS && !kv_row(p, e, h, t, row)) return;   // few tokens: the position arrives together with them, not in front of them
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float f[8];
    unpack8(w ? vr : kr, f);
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { const uint32_t b = abs_bits(f[j]); amax = amax > b ? amax : b; }
    amax = Max()(amax, dpp<0xB1>(amax)); amax = Max()(amax, dpp<0x4E>(amax)); amax = Max()(amax, dpp<0x141>(amax));      // quad permutes, half mirror: eight lanes
    float scale, inv;
    q8_scale(amax, scale, inv);
    const bool ok = amax < 0x7f800000u;
    uint2 u;
    u.x = q8_pack4(f, inv, ok); u.y = q8_pack4(f + 4, inv, ok);
    *reinterpret_cast<uint2*>((w ? p.vq : p.kq) + row * 64 + c * 8) = u;
    if (c == 0) (w ? p.vs : p.ks)[row] = scale;
  }
}

template <bool TOKENS>
__global__ __launch_bounds__(256) void kv_read_q8_kernel(const KvQ8 p) {
  int e = 0, h = 0, t = 0;
  long row;
  if (!kv_unit<TOKENS>(p, e, h, t) || !kv_row(p, e, h, t, row)) return;
  const int c = threadIdx.x & 7;
  const long dst = (long)e * p.bs + (long)t * p.rs + h * 64 + c * 8;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint2 u = *reinterpret_cast<const uint2*>((w ? p.vq : p.kq) + row * 64 + c * 8);
    const float s = (w ? p.vs : p.ks)[row];
    float f[8];
    q8_unpack4(u.x, f); q8_unpack4(u.y, f + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= s;
    *reinterpret_cast<uint4*>((w ? p.v : p.k) + dst) = round8(f);
  }
}

// ---- single-query attention over the cache --------------------------------------------------------------------------------------------------
//   z_j = scale * ks_j <q, kq_j> + bias_j,   o = sum_j exp(z_j - m) vs_j vq_j / sum_j exp(z_j - m)
// A masked key is not part of the sums at all (whatever its codes and scale hold); a query that sees no key -- all masked, or a bias of
// -infinity everywhere -- gets the mean of its keys' values, as softmax over equal scores gives (modeling_t5.py:996,559), and a query without
// keys gets zeros.
constexpr int PIECE = 1280;           // keys per block; fixed, so that a sequence's result does not depend on its batch
constexpr float LOG2E = 1.44269504088896340736f;

struct AttnQ8 {
  int B, H, Nk, G, gchunks, np;
  const bf16_t* q; long q_bs;
  const i8 *kq, *vq;
  const float *ks, *vs;
  long e_rows, h_rows;
  bf16_t* o; long o_bs;
  const float* bias; long bias_ld;
  const int* pos_dev; int bias_maxlen;
  const int* klen;
  const uint8_t* mask; long mask_ld;
  float scale;
  float* ws;                          // [B][H][np][66]: 64 sums, maximum, sum of weights
};

__device__ __forceinline__ int attn_q8_keys(const AttnQ8& p, int e) {
  int n = p.Nk;
  if (p.pos_dev) n = *p.pos_dev + 1;
  if (p.klen) n = p.klen[e];
  return n < 0 ? 0 : (n > p.Nk ? p.Nk : n);
}
// exp(m - M) of a running maximum; the difference is taken first, so that scores of any finite size are told apart
__device__ __forceinline__ float rescale(float m, float M) { return m == M ? 1.f : __builtin_amdgcn_exp2f((m - M) * LOG2E); }

// mean of the values of n keys of one (entry, head) by the first 256 threads of a block; lds: 256 floats.  The rare row without a visible key.
__device__ float attn_q8_mean(const i8* vq, const float* vs, int n, float* lds) {
  const int d = threadIdx.x & 63, part = threadIdx.x >> 6;
  float s = 0.f;
  if (part < 4) {
#pragma unroll 16
    for (int k = part; k < n; k += 4) s = fmaf(vs[k], (float)vq[(long)k * 64 + d], s);
  }
  __syncthreads();
  if (part < 4) lds[threadIdx.x] = s;
  __syncthreads();
  s = lds[d] + lds[64 + d] + lds[128 + d] + lds[192 + d];
  __syncthreads();
  return n > 0 ? s / (float)n : 0.f;
}

// What lanes of a wave pass to each other through LDS needs no wait (a wave's LDS operations keep their order), but the compiler, which sees one lane, has to
// be told that the words may have changed
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// eight codes as bf16, exactly
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t lo, uint32_t hi) {
  float f[8];
  q8_unpack4(lo, f); q8_unpack4(hi, f + 4);
  uint4 r;
  r.x = __builtin_amdgcn_perm(__float_as_uint(f[1]), __float_as_uint(f[0]), 0x07060302u);
  r.y = __builtin_amdgcn_perm(__float_as_uint(f[3]), __float_as_uint(f[2]), 0x07060302u);
  r.z = __builtin_amdgcn_perm(__float_as_uint(f[5]), __float_as_uint(f[4]), 0x07060302u);
  r.w = __builtin_amdgcn_perm(__float_as_uint(f[7]), __float_as_uint(f[6]), 0x07060302u);
  return __builtin_bit_cast(bf16x8, r);
}

// Block = 4 waves = up to PIECE keys of one (entry, head) against up to 16 of its queries, on the matrix pipe; a wave takes 64 keys at a time.
//   loads    16 whole keys (1 KiB in a row) per instruction.  Keys loaded straight into the fragments' lanes (16 rows of 16 bytes per instruction) asked the
//            cache for every line four times: 348 MB in 94 us, through LDS in 66 (both with the same cache again).
//   scores   S^T[key][query] = K[key][d] . Q^T[d][query] by v_mfma_f32_16x16x32_bf16: codes are exact in bf16, so the products are exact and the sums
//            fp32.  Tile t of a group of 32 keys holds the keys 8 (row >> 2) + 4 t + (row & 3), so that the eight scores a lane gets of its query are
//            those of the consecutive keys 8 g .. 8 g + 7 (g = lane >> 4), which is the B operand of the second product without any movement.
//   output   O^T[d][query] += V^T[d][key] . P^T[key][query]: the value codes follow the keys in the wave's LDS tile, the transposing read
//            (ds_read_b64_tr_b8) returns the codes of eight keys for one d.  The weights carry the values' scales and are split into three bf16 parts
//            of eight bits each, which is all of fp32 (three products): every product is exact and the sums are fp32, as for a single query.
// The running maximum of a query is shared by its four lanes; scales and bias of the piece wait in LDS, where a key without a part has bias -infinity
// and scales of zero.  4 x 4 queries x 16 heads x 40000 keys: 73 to 75 us = 4.7 TB/s with the join (weights in two bf16 parts, 16 bits: 70 to 73).  A value-per-lane form without the matrix pipe was
// bound by VALU issue (127 us); eight waves per block or five blocks per CU were slower on large caches, requesting the next chunk ahead did not pay.
constexpr int WG = 4;                 // waves per block
// byte of the 16-byte chunk c of key k in a wave's tile: the rows of a fragment read and those of a transposing read fall into different banks
__device__ __forceinline__ int tile_at(int k, int c) { return k * 64 + (c ^ ((k >> 3) & 3) ^ ((k >> 2) & 1)) * 16; }
__global__ __launch_bounds__(WG * 64, 4) void attn_q8_kernel(const AttnQ8 p) {
  __shared__ __attribute__((aligned(16))) float s_ks[PIECE], s_vs[PIECE], s_b[PIECE];
  __shared__ __attribute__((aligned(16))) char s_v[WG][64 * 64];       // value tiles, then the waves' sums
  __shared__ float s_m[WG][16], s_l[WG][16];
  __shared__ uint32_t s_any;           // chunks of 64 keys that hold a visible one
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), qi = lane & 15, g = lane >> 4;
  const int gc = blockIdx.x % p.gchunks, eh = blockIdx.x / p.gchunks;
  const int h = eh % p.H, e = eh / p.H;
  const int piece = blockIdx.y, k0 = piece * PIECE;
  const int n = attn_q8_keys(p, e);
  if (k0 >= n && piece > 0) return;
  const int end = min(n - k0, PIECE), nch = (end + 63) >> 6;
  const int g0 = gc * 16, ng = min(16, p.G - g0);
  const long base = (long)e * p.e_rows + (long)h * p.h_rows + k0;
  const i8 *kq = p.kq + base * 64, *vq = p.vq + base * 64;
  const float *ks = p.ks + base, *vs = p.vs + base;
  const float* bias = nullptr;
  if (p.bias) bias = p.bias + (long)h * p.bias_ld + k0 + (p.pos_dev ? p.bias_maxlen - 1 - min(*p.pos_dev, p.bias_maxlen - 1) : 0);

  if (tid == 0) s_any = 0;
  __syncthreads();
  bf16x8 qf[2];
  {
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (qi < ng) {
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (long)(e * p.G + g0 + qi) * p.q_bs + h * 64 + g * 16);
      a = src[0]; b = src[1];
    }
    qf[0] = __builtin_bit_cast(bf16x8, a); qf[1] = __builtin_bit_cast(bf16x8, b);
  }
  if (nch > 0) {                        // every load in flight before the first is used
    constexpr int R = (PIECE + WG * 64 - 1) / (WG * 64);
    float sk[R], sv[R], b[R];
    uint8_t mk[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = min(r * (WG * 64) + tid, end - 1);
      sk[r] = ks[k]; sv[r] = vs[k];
      b[r] = bias ? bias[k] : 0.f;
      mk[r] = p.mask ? p.mask[(long)e * p.mask_ld + k0 + k] : 1;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int k = r * (WG * 64) + tid;
      const bool see = k < end && mk[r] != 0 && !(b[r] == -INFINITY);
      if (k < PIECE) { s_ks[k] = see ? sk[r] * p.scale : 0.f; s_vs[k] = see ? sv[r] : 0.f; s_b[k] = see ? b[r] : -INFINITY; }
      const unsigned long long any = __ballot(see);
      if (lane == 0 && any != 0) atomicOr(&s_any, 1u << (r * WG + wave));
    }
  }
  __syncthreads();

  f32x4 acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  char* const vt = s_v[wave];
  u32x4 kr[4], vr[4];
  auto load = [&](int ch) {             // codes of a chunk; keys behind the end load the last one: their scales are zero
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = (uint32_t)(min(ch * 64 + i * 16 + (lane >> 2), end - 1) * 64 + (lane & 3) * 16);
      kr[i] = *reinterpret_cast<const u32x4*>(kq + at);
      vr[i] = *reinterpret_cast<const u32x4*>(vq + at);
    }
  };
  for (uint32_t rest = __builtin_amdgcn_readfirstlane(s_any) & (0x11111111u << wave); rest; rest &= rest - 1) {
    const int ch = __builtin_ctz(rest);
    load(ch);
    // all of the chunk's LDS traffic but the values' scales in one go (a wave's LDS operations keep their order, so the values may follow the keys in place)
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(vt + tile_at(i * 16 + (lane >> 2), lane & 3)) = kr[i];
    wave_sync();
    u32x4 kf[4];
    float4 sk[4], sb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      kf[i] = *reinterpret_cast<const u32x4*>(vt + tile_at((i >> 1) * 32 + 8 * (qi >> 2) + 4 * (i & 1) + (qi & 3), g));
      const int at = ch * 64 + (i >> 1) * 32 + 8 * g + 4 * (i & 1);
      sk[i] = *reinterpret_cast<const float4*>(s_ks + at); sb[i] = *reinterpret_cast<const float4*>(s_b + at);
    }
    wave_sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(vt + tile_at(i * 16 + (lane >> 2), lane & 3)) = vr[i];
    wave_sync();
    i32x2 vc[2][4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
        vc[kb][dt] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((V2S_LDS i32x2*)(vt + tile_at(kb * 32 + 8 * g + (qi >> 1), dt) + (qi & 1) * 8));
    wave_sync();
    __builtin_amdgcn_sched_barrier(0);
    float sc[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_bf16(kf[i][0], kf[i][1]), qf[0], d, 0, 0, 0);
      d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_bf16(kf[i][2], kf[i][3]), qf[1], d, 0, 0, 0);
      const float ks4[4] = {sk[i].x, sk[i].y, sk[i].z, sk[i].w}, b4[4] = {sb[i].x, sb[i].y, sb[i].z, sb[i].w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float z = fmaf(d[r], ks4[r], b4[r]);
        sc[4 * i + r] = b4[r] == -INFINITY ? b4[r] : z;      // whatever a query holds
      }
    }
    float mn = sc[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mn = fmaxf(mn, sc[i]);
    mn = rows_reduce(mn, Max());
    mn = fmaxf(mn, m);
    const float a = rescale(m, mn);
    m = mn;
    l *= a;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= a;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      float w[8];
      const float4 v0 = *reinterpret_cast<const float4*>(s_vs + ch * 64 + kb * 32 + 8 * g), v1 = *reinterpret_cast<const float4*>(s_vs + ch * 64 + kb * 32 + 8 * g + 4);
      const float sv[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z = sc[kb * 8 + i];
        const float x = z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((z - m) * LOG2E);
        l += x;
        w[i] = x * sv[i];
      }
      bf16x8 part[3];                   // hi, mid, lo: 24 bits
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        const uint4 r = round8(w);
        part[x] = __builtin_bit_cast(bf16x8, r);
        if (x < 2) {
          float f[8];
          unpack8(r, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] -= f[i];
        }
      }
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        const bf16x8 vf = codes_bf16((uint32_t)vc[kb][dt][0], (uint32_t)vc[kb][dt][1]);
#pragma unroll
        for (int x = 0; x < 3; ++x) acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, part[x], acc[dt], 0, 0, 0);
      }
    }
  }
  // join the waves: [query][64] sums per wave in the wave's own tile
  l = rows_reduce(l, Add());
  float* const so = reinterpret_cast<float*>(vt);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) *reinterpret_cast<f32x4*>(so + qi * 64 + dt * 16 + g * 4) = acc[dt];
  if (g == 0) { s_m[wave][qi] = m; s_l[wave][qi] = l; }
  __syncthreads();
  const auto seen = [&](int q) {        // sum of a query's weights: zero if it sees no key
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < WG; ++w) l += s_l[w][q];
    return l != 0.f;
  };
  if (p.np == 1) {
    bool none = false;                  // a query of this block without a visible key
    for (int q = 0; q < ng; ++q) none |= !seen(q);
    if (none) {                         // the same for every thread of the block
      const float mean = attn_q8_mean(vq, vs, n, s_b);
      for (int t = tid; t < ng * 64; t += WG * 64)
        if (!seen(t >> 6)) p.o[((long)e * p.G + g0 + (t >> 6)) * p.o_bs + h * 64 + (t & 63)] = f2bf(mean);
    }
  }
  for (int t = tid; t < ng * 64; t += WG * 64) {
    const int q = t >> 6, d = t & 63;
    float M = s_m[0][q];
#pragma unroll
    for (int w = 1; w < WG; ++w) M = fmaxf(M, s_m[w][q]);
    float L = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < WG; ++w) {
      const float a = rescale(s_m[w][q], M);
      L += s_l[w][q] * a; O += reinterpret_cast<const float*>(s_v[w])[q * 64 + d] * a;
    }
    const long b = (long)e * p.G + g0 + q;
    if (p.np == 1) {
      if (L != 0.f) p.o[b * p.o_bs + h * 64 + d] = f2bf(O / L);
    } else {
      float* w = p.ws + ((b * p.H + h) * p.np + piece) * 66;
      w[d] = O;
      if (d == 0) { w[64] = M; w[65] = L; }
    }
  }
}

// One query per entry: block = 4 waves = up to PIECE keys of one (entry, head).  lane = (key slot lane >> 2, 16 dimensions lane & 3): a load of the wave is
// 16 whole keys (1 KiB).  On the matrix pipe fifteen of the sixteen query columns would be empty while every lane still converts the codes and
// computes a softmax, so the fp32 pipe needs a third fewer instructions here.
// 32 x 16 heads x 5000 keys: 65 us with the join, 5.3 TB/s; twice the waves per block: 8 x 12 heads x 1200 keys 7.7 instead of 8.7 us, but 64 x 12 x 300
// keys 11.1 instead of 9.6.
constexpr int W1 = 4;
__global__ __launch_bounds__(W1 * 64) void attn_q8_one_kernel(const AttnQ8 p) {
  __shared__ float s_m[W1], s_l[W1], s_o[W1][64], s_red[256];
  __shared__ unsigned long long s_bits[(PIECE / 64 + W1 - 1) / W1 * W1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), slot = lane >> 2, c = lane & 3;
  const int h = blockIdx.x % p.H, e = blockIdx.x / p.H;
  const int piece = blockIdx.y, k0 = piece * PIECE;
  const int n = attn_q8_keys(p, e);
  if (k0 >= n && piece > 0) return;
  const int end = min(n - k0, PIECE), nch = (end + 63) >> 6;
  const long base = (long)e * p.e_rows + (long)h * p.h_rows + k0;
  const i8 *kq = p.kq + base * 64, *vq = p.vq + base * 64;
  const float *ks = p.ks + base, *vs = p.vs + base;
  const float* bias = nullptr;
  if (p.bias) bias = p.bias + (long)h * p.bias_ld + k0 + (p.pos_dev ? p.bias_maxlen - 1 - min(*p.pos_dev, p.bias_maxlen - 1) : 0);
  float qv[16];
  const long qr = (long)e * p.q_bs + h * 64 + c * 16;
  ld8(p.q + qr, qv); ld8(p.q + qr + 8, qv + 8);
  if (p.mask) {                                      // visible keys, one bit each
    for (int r = 0; r < nch; r += W1) {
      const int k = r * 64 + tid;
      const unsigned long long b = __ballot(k < end && p.mask[(long)e * p.mask_ld + k0 + min(k, end - 1)] != 0);
      if (lane == 0) s_bits[r + wave] = b;
    }
    __syncthreads();
  }
  float m = -INFINITY, l = 0.f, acc[16];
#pragma unroll
  for (int d = 0; d < 16; ++d) acc[d] = 0.f;
  for (int ch = wave; ch < nch; ch += W1) {
    const int left = end - ch * 64;
    unsigned long long bits = left >= 64 ? ~0ull : (1ull << left) - 1;
    if (p.mask) bits = s_bits[ch];
    if (__builtin_amdgcn_readfirstlane((uint32_t)bits | (uint32_t)(bits >> 32)) == 0) continue;
    u32x4 kr[4], vr[4];
    float sk[4], sv[4], bz[4], sc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t k = (uint32_t)min(ch * 64 + j * 16 + slot, end - 1);
      kr[j] = *reinterpret_cast<const u32x4*>(kq + k * 64 + c * 16);
      vr[j] = *reinterpret_cast<const u32x4*>(vq + k * 64 + c * 16);
      sk[j] = ks[k]; sv[j] = vs[k];
      bz[j] = bias ? bias[k] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float d = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[4];
        q8_unpack4(kr[j][i], f);
#pragma unroll
        for (int t = 0; t < 4; ++t) d = fmaf(qv[4 * i + t], f[t], d);
      }
      d += dpp<0xB1>(d);                             // the four lanes of a key: quad permutes [1,0,3,2] and [2,3,0,1]
      d += dpp<0x4E>(d);
      const bool see = (bits >> (j * 16 + slot)) & 1ull && !(bz[j] == -INFINITY);
      const float z = fmaf(d, sk[j] * p.scale, bz[j]);
      sc[j] = see ? z : -INFINITY;
      sv[j] = see ? sv[j] : 0.f;                     // what a masked key holds never reaches the sums
    }
    const float mn = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), m);
    const float a = rescale(m, mn);
    m = mn;
    l *= a;
#pragma unroll
    for (int d = 0; d < 16; ++d) acc[d] *= a;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float w = sc[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((sc[j] - mn) * LOG2E);
      l += w;
      const float x = w * sv[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[4];
        q8_unpack4(vr[j][i], f);
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[4 * i + t] = fmaf(x, f[t], acc[4 * i + t]);
      }
    }
  }
  // the 16 key slots of the wave, then the waves
  float M = m;
  M = fmaxf(M, dpp<0x128>(M)); M = fmaxf(M, dpp<0x124>(M));
  M = rows_reduce(M, Max());
  const float a = rescale(m, M);
  float L = l * a;
  L += dpp<0x128>(L); L += dpp<0x124>(L);      // row_ror 8 and 4 keep lane & 3
  L = rows_reduce(L, Add());
#pragma unroll
  for (int d = 0; d < 16; ++d) {
    float x = acc[d] * a;
    x += dpp<0x128>(x); x += dpp<0x124>(x);
    x = rows_reduce(x, Add());
    if (slot == 0) s_o[wave][c * 16 + d] = x;
  }
  if (lane == 0) { s_m[wave] = M; s_l[wave] = L; }
  __syncthreads();
  M = s_m[0];
  for (int w = 1; w < W1; ++w) M = fmaxf(M, s_m[w]);
  L = 0.f;
  float O = 0.f;
  for (int w = 0; w < W1; ++w) { const float x = rescale(s_m[w], M); L += s_l[w] * x; O += s_o[w][lane] * x; }
  float r = O / L;
  if (L == 0.f && p.np == 1) r = attn_q8_mean(vq, vs, n, s_red);       // the same for every thread of the block
  if (wave != 0) return;
  if (p.np == 1) {
    p.o[(long)e * p.o_bs + h * 64 + lane] = f2bf(r);
  } else {
    float* w = p.ws + ((long)blockIdx.x * p.np + piece) * 66;
    w[lane] = O;
    if (lane == 0) { w[64] = M; w[65] = L; }
  }
}

// joins the pieces of one (query, head): 4 waves take the pieces in turn
__global__ __launch_bounds__(256) void attn_q8_join_kernel(const AttnQ8 p) {
  __shared__ float s_m[4], s_l[4], s_o[4][64], s_red[256];
  const int h = blockIdx.x % p.H, b = blockIdx.x / p.H, e = b / p.G;
  const int d = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n = attn_q8_keys(p, e), np = (n + PIECE - 1) / PIECE;
  const float* w = p.ws + (long)blockIdx.x * p.np * 66;
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int i0 = wave; i0 < p.np; i0 += 32) {         // eight pieces of the wave in flight, before the length is known: those behind it have no part
    float m[8], l[8], o[8], mn = M;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float* v = w + min(i0 + j * 4, p.np - 1) * 66;
      m[j] = v[64]; l[j] = v[65]; o[j] = v[d];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (i0 + j * 4 >= np) { m[j] = -INFINITY; l[j] = 0.f; o[j] = 0.f; }
      mn = fmaxf(mn, m[j]);
    }
    const float a = rescale(M, mn);
    L *= a; O *= a; M = mn;
#pragma unroll
    for (int j = 0; j < 8; ++j) { const float x = rescale(m[j], mn); L += l[j] * x; O += o[j] * x; }
  }
  s_o[wave][d] = O;
  if (d == 0) { s_m[wave] = M; s_l[wave] = L; }
  __syncthreads();
  M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  L = O = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float x = rescale(s_m[i], M); L += s_l[i] * x; O += s_o[i][d] * x; }
  float r = O / L;
  if (L == 0.f) {                                    // the same for every thread of the block
    const long base = (long)e * p.e_rows + (long)h * p.h_rows;
    r = attn_q8_mean(p.vq + base * 64, p.vs + base, n, s_red);
  }
  if (wave == 0) p.o[(long)b * p.o_bs + h * 64 + d] = f2bf(r);
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <typename T, int NCH, int LPR, bool NORM> int rows_q8_launch(const RowsQ8& p, hipStream_t s) {
  hipLaunchKernelGGL((rows_q8_kernel<T, NCH, LPR, NORM>), dim3((unsigned)((p.rows + 256 / LPR - 1) / (256 / LPR))), dim3(256), 0, s, p);      // rows < 2^24
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}
template <typename T, bool NORM> int rows_q8_any(const RowsQ8& p, hipStream_t s) {
  if (p.cols <= 128) return rows_q8_launch<T, 1, 16, NORM>(p, s);
  if (p.cols <= 256) return rows_q8_launch<T, 1, 32, NORM>(p, s);
  if (p.cols <= 512) return rows_q8_launch<T, 1, 64, NORM>(p, s);
  if (p.cols <= 1024) return rows_q8_launch<T, 2, 64, NORM>(p, s);
  if (p.cols <= 2048) return rows_q8_launch<T, 1, 256, NORM>(p, s);
  if (p.cols <= 4096) return rows_q8_launch<T, 2, 256, NORM>(p, s);
  return rows_q8_launch<T, 4, 256, NORM>(p, s);
}

int kv_check(const char* who, const v2s_kv_q8* c, const void* k, const void* v, int64_t bs, int64_t rs, int32_t T) {
  V2S_CHECK(c && c->k && c->ks && c->v && c->vs && k && v, V2S_ERR_ARG, "%s: NULL pointer", who);
  V2S_CHECK(c->entries > 0 && c->heads > 0 && c->maxlen > 0 && T > 0, V2S_ERR_SHAPE, "%s: entries, heads, maxlen and T must be positive", who);
  V2S_CHECK(c->h_rows >= c->maxlen && c->e_rows >= c->maxlen, V2S_ERR_SHAPE, "%s: row strides must be at least maxlen (%d)", who, c->maxlen);
  V2S_CHECK(aligned(c->k, 16) && aligned(c->v, 16) && aligned(k, 16) && aligned(v, 16) && aligned(c->ks, 4) && aligned(c->vs, 4) && bs % 8 == 0 && rs % 8 == 0,
            V2S_ERR_ALIGN, "%s: pointers must be 16-byte aligned and strides multiples of 8 elements", who);
  const int64_t units = (int64_t)c->entries * ((c->heads + 7) & ~7) * (((int64_t)T + 7) & ~7);
  V2S_CHECK(units < 1 << 29, V2S_ERR_SHAPE, "%s: entries x heads x T too large for one launch", who);      // 2^32 threads
  return V2S_OK;
}

KvQ8 kv_args(const v2s_kv_q8* c, const void* k, const void* v, int64_t bs, int64_t rs, int32_t T, int32_t pos0, const int32_t* pos, const int32_t* pos_dev,
             const int32_t* count) {
  KvQ8 p;
  p.kq = (i8*)c->k; p.vq = (i8*)c->v; p.ks = c->ks; p.vs = c->vs; p.e_rows = c->e_rows; p.h_rows = c->h_rows;
  p.E = c->entries; p.H = c->heads; p.maxlen = c->maxlen; p.T = T;
  p.k = (bf16_t*)k; p.v = (bf16_t*)v; p.bs = bs; p.rs = rs;
  p.pos = pos; p.pos_dev = pos_dev; p.count = count; p.pos0 = pos0;
  return p;
}
unsigned kv_blocks(const KvQ8& p, bool tokens) {
  const int64_t units = tokens ? (int64_t)p.E * p.H * ((p.T + 7) & ~7) : (int64_t)p.E * p.T * ((p.H + 7) & ~7);
  return (unsigned)((units + 31) / 32);
}

}  // namespace

extern "C" int v2s_quant_rows_q8(const void* x, int32_t x_dtype, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int32_t rows, int32_t cols, void* stream) {
  V2S_CHECK(x && q && scale, V2S_ERR_ARG, "v2s_quant_rows_q8: NULL pointer");
  V2S_CHECK(x_dtype == V2S_BF16 || x_dtype == V2S_F32, V2S_ERR_DTYPE, "v2s_quant_rows_q8: x must be bf16 or fp32");
  V2S_CHECK(rows > 0 && rows < 1 << 24 && cols > 0 && cols % 8 == 0 && cols <= 8192, V2S_ERR_SHAPE,
            "v2s_quant_rows_q8: unsupported shape rows=%d cols=%d (rows below 2^24, cols a multiple of 8, <= 8192)", rows, cols);
  V2S_CHECK(ldx >= cols && ldq >= cols, V2S_ERR_SHAPE, "v2s_quant_rows_q8: a row stride is shorter than the row");
  V2S_CHECK(aligned(x, 16) && aligned(q, 8) && aligned(scale, 4) && ldx % 8 == 0 && ldq % 8 == 0, V2S_ERR_ALIGN,
            "v2s_quant_rows_q8: x must be 16-byte and q 8-byte aligned, strides multiples of 8");
  RowsQ8 p = {};
  p.x = x; p.ldx = ldx; p.q = (i8*)q; p.ldq = ldq; p.scale = scale; p.rows = rows; p.cols = cols;
  return x_dtype == V2S_F32 ? rows_q8_any<float, false>(p, (hipStream_t)stream) : rows_q8_any<bf16_t, false>(p, (hipStream_t)stream);
}

extern "C" int v2s_rmsnorm_q8(const void* x, int64_t ldx, const void* delta, int64_t ldd, const float* w, void* h, int64_t ldh, int8_t* q, int64_t ldq,
                              float* scale, int32_t rows, int32_t cols, float eps, void* stream) {
  V2S_CHECK(x && w && q && scale, V2S_ERR_ARG, "v2s_rmsnorm_q8: NULL pointer");
  V2S_CHECK(!h || delta, V2S_ERR_ARG, "v2s_rmsnorm_q8: h is the sum x + delta, it needs delta");
  V2S_CHECK(eps >= 0.f, V2S_ERR_ARG, "v2s_rmsnorm_q8: eps must not be negative");
  V2S_CHECK(rows > 0 && rows < 1 << 24 && cols > 0 && cols % 8 == 0 && cols <= 8192, V2S_ERR_SHAPE,
            "v2s_rmsnorm_q8: unsupported shape rows=%d cols=%d (rows below 2^24, cols a multiple of 8, <= 8192)", rows, cols);
  V2S_CHECK(ldx >= cols && ldq >= cols && (!delta || ldd >= cols) && (!h || ldh >= cols), V2S_ERR_SHAPE, "v2s_rmsnorm_q8: a row stride is shorter than the row");
  V2S_CHECK(aligned(x, 16) && aligned(delta, 16) && aligned(h, 16) && aligned(w, 16) && aligned(q, 8) && aligned(scale, 4) && ldx % 8 == 0 && ldq % 8 == 0 &&
                (!delta || ldd % 8 == 0) && (!h || ldh % 8 == 0),
            V2S_ERR_ALIGN, "v2s_rmsnorm_q8: x, delta, w and h must be 16-byte and q 8-byte aligned, strides multiples of 8");
  RowsQ8 p = {};
  p.x = x; p.ldx = ldx; p.delta = (const bf16_t*)delta; p.ldd = ldd; p.w = w; p.h = (bf16_t*)h; p.ldh = ldh; p.q = (i8*)q; p.ldq = ldq; p.scale = scale;
  p.rows = rows; p.cols = cols; p.eps = eps;
  return rows_q8_any<bf16_t, true>(p, (hipStream_t)stream);
}

extern "C" int v2s_dequant_q8(const int8_t* q, int64_t ldq, const float* scale, void* y, int64_t ldy, int32_t rows, int32_t cols, void* stream) {
  V2S_CHECK(q && scale && y, V2S_ERR_ARG, "v2s_dequant_q8: NULL pointer");
  V2S_CHECK(rows > 0 && cols > 0 && cols % 8 == 0, V2S_ERR_SHAPE, "v2s_dequant_q8: unsupported shape rows=%d cols=%d (cols a multiple of 8)", rows, cols);
  V2S_CHECK(ldq >= cols && ldy >= cols, V2S_ERR_SHAPE, "v2s_dequant_q8: a row stride is shorter than the row");
  V2S_CHECK(aligned(q, 8) && aligned(y, 16) && aligned(scale, 4) && ldq % 8 == 0 && ldy % 8 == 0, V2S_ERR_ALIGN,
            "v2s_dequant_q8: q must be 8-byte and y 16-byte aligned, strides multiples of 8");
  const int64_t blocks = ((int64_t)rows * (cols / 8) + 255) / 256;
  V2S_CHECK(blocks < 1 << 24, V2S_ERR_SHAPE, "v2s_dequant_q8: too many elements for one launch");
  hipLaunchKernelGGL(dequant_q8_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, (const i8*)q, (long)ldq, scale, (bf16_t*)y, (long)ldy, rows, cols / 8);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}

extern "C" int v2s_kv_append_q8(const v2s_kv_q8* cache, const void* k, const void* v, int64_t src_bs, int64_t src_rs, int32_t T, int32_t pos0,
                                const int32_t* pos, const int32_t* pos_dev, const int32_t* count, void* stream) {
  if (int e = kv_check("v2s_kv_append_q8", cache, k, v, src_bs, src_rs, T)) return e;
  const KvQ8 p = kv_args(cache, k, v, src_bs, src_rs, T, pos0, pos, pos_dev, count);
  if (T >= 8) hipLaunchKernelGGL(kv_append_q8_kernel<true>, dim3(kv_blocks(p, true)), dim3(256), 0, (hipStream_t)stream, p);
  else hipLaunchKernelGGL(kv_append_q8_kernel<false>, dim3(kv_blocks(p, false)), dim3(256), 0, (hipStream_t)stream, p);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}

extern "C" int v2s_kv_read_q8(const v2s_kv_q8* cache, void* k, void* v, int64_t dst_bs, int64_t dst_rs, int32_t T, int32_t pos0, const int32_t* pos,
                              const int32_t* pos_dev, const int32_t* count, void* stream) {
  if (int e = kv_check("v2s_kv_read_q8", cache, k, v, dst_bs, dst_rs, T)) return e;
  const KvQ8 p = kv_args(cache, k, v, dst_bs, dst_rs, T, pos0, pos, pos_dev, count);
  if (T >= 8) hipLaunchKernelGGL(kv_read_q8_kernel<true>, dim3(kv_blocks(p, true)), dim3(256), 0, (hipStream_t)stream, p);
  else hipLaunchKernelGGL(kv_read_q8_kernel<false>, dim3(kv_blocks(p, false)), dim3(256), 0, (hipStream_t)stream, p);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}

extern "C" int64_t v2s_decode_attn_q8_workspace_floats(int32_t B, int32_t H, int32_t Nk) {
  if (B <= 0 || H <= 0 || Nk <= PIECE) return 0;
  return (int64_t)B * H * ((Nk + PIECE - 1) / PIECE) * 66;
}

extern "C" int v2s_decode_attn_q8(const v2s_decode_attn_q8_args* a, void* stream) {
  V2S_CHECK(a && a->q && a->cache.k && a->cache.ks && a->cache.v && a->cache.vs && a->o, V2S_ERR_ARG, "v2s_decode_attn_q8: NULL pointer");
  const v2s_kv_q8& c = a->cache;
  const int G = a->group > 1 ? a->group : 1;
  V2S_CHECK(a->B > 0 && c.heads > 0 && c.entries > 0 && a->Nk > 0, V2S_ERR_SHAPE, "v2s_decode_attn_q8: B, heads, entries and Nk must be positive");
  V2S_CHECK(a->B == (int64_t)c.entries * G, V2S_ERR_SHAPE, "v2s_decode_attn_q8: %d query rows for %d cache entries of %d queries each", a->B, c.entries, G);
  V2S_CHECK(a->Nk <= c.maxlen && c.h_rows >= c.maxlen && c.e_rows >= c.maxlen, V2S_ERR_SHAPE, "v2s_decode_attn_q8: Nk %d, maxlen %d and the row strides do not fit", a->Nk, c.maxlen);
  V2S_CHECK(!(a->klen && a->pos_dev), V2S_ERR_ARG, "v2s_decode_attn_q8: klen and pos_dev exclude each other");
  V2S_CHECK(!a->bias_row || (a->pos_dev ? a->bias_maxlen >= a->Nk && a->bias_ld >= 2 * (int64_t)a->bias_maxlen - 1 : a->bias_ld >= a->Nk), V2S_ERR_SHAPE,
            "v2s_decode_attn_q8: the bias rows are too short for Nk keys");
  V2S_CHECK(!a->key_mask || a->mask_ld >= a->Nk, V2S_ERR_SHAPE, "v2s_decode_attn_q8: mask_ld is smaller than Nk");
  const int64_t width = (int64_t)c.heads * 64;
  V2S_CHECK(a->q_bs >= width && a->o_bs >= width, V2S_ERR_SHAPE, "v2s_decode_attn_q8: a row stride is shorter than heads * 64");
  V2S_CHECK(aligned(a->q, 16) && aligned(c.k, 16) && aligned(c.v, 16) && aligned(c.ks, 4) && aligned(c.vs, 4) && aligned(a->o, 2) && a->q_bs % 8 == 0, V2S_ERR_ALIGN,
            "v2s_decode_attn_q8: pointers must be 16-byte aligned and q_bs a multiple of 8");
  AttnQ8 p;
  p.B = a->B; p.H = c.heads; p.Nk = a->Nk; p.G = G; p.np = (a->Nk + PIECE - 1) / PIECE;
  p.q = (const bf16_t*)a->q; p.q_bs = a->q_bs; p.kq = (const i8*)c.k; p.vq = (const i8*)c.v; p.ks = c.ks; p.vs = c.vs; p.e_rows = c.e_rows; p.h_rows = c.h_rows;
  p.o = (bf16_t*)a->o; p.o_bs = a->o_bs; p.bias = a->bias_row; p.bias_ld = a->bias_ld; p.pos_dev = a->pos_dev; p.bias_maxlen = a->bias_maxlen;
  p.klen = a->klen; p.mask = a->key_mask; p.mask_ld = a->mask_ld; p.scale = a->scale; p.ws = (float*)a->workspace;
  const int64_t need = v2s_decode_attn_q8_workspace_floats(a->B, c.heads, a->Nk) * 4;
  V2S_CHECK(need == 0 || (a->workspace && a->workspace_bytes >= need && aligned(a->workspace, 4)), V2S_ERR_ARG,
            "v2s_decode_attn_q8: %lld bytes of workspace needed for %d keys, got %lld", (long long)need, a->Nk, (long long)(a->workspace ? a->workspace_bytes : 0));
  p.gchunks = (G + 15) / 16;
  V2S_CHECK((int64_t)a->B * c.heads < 1 << 24 && p.np <= 65535, V2S_ERR_SHAPE, "v2s_decode_attn_q8: too many rows or keys for one launch");
  const dim3 grid((unsigned)(c.entries * c.heads * p.gchunks), (unsigned)p.np);
  hipStream_t s = (hipStream_t)stream;
  if (G == 1) hipLaunchKernelGGL(attn_q8_one_kernel, grid, dim3(W1 * 64), 0, s, p);
  else hipLaunchKernelGGL(attn_q8_kernel, grid, dim3(WG * 64), 0, s, p);
  V2S_LAUNCH_CHECK();
  if (p.np > 1) {
    hipLaunchKernelGGL(attn_q8_join_kernel, dim3((unsigned)(a->B * c.heads)), dim3(256), 0, s, p);
    V2S_LAUNCH_CHECK();
  }
  return V2S_OK;
}
