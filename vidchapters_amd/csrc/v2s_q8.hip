// 8-bit decoding for gfx950: rows of activations to int8 codes with one fp32 scale per row (with the residual addition and the RMSNorm in
// front of it), the int8 key / value cache, and the single-query attention that reads it.
//   code q and scale s of a row y:  s = max(amax|y|, 127 * 2^-126) / 127,  q = round_to_even(y / s),  so that |y - s q| <= s / 2 (1 + 2^-23)
// The floor of s keeps 1 / s finite: rows below it (1.5e-36) keep the smallest normal scale and fewer codes.  A row that holds a NaN or an
// infinity gets s = NaN and zero codes: every value that is read back is NaN, none of them is a plausible number.
//   RMSNorm: model/modeling_t5.py:263-277 (T5LayerNorm.forward); the cache it replaces: model/modeling_t5.py:555-556
#include <math.h>
#include "v2s_common.h"

namespace {

typedef signed char i8;
constexpr float Q8_TINY = 127.0f * 1.17549435e-38f;

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) { const uint32_t w = (uint32_t)__shfl_xor((int)v, o, 64); v = v > w ? v : w; }
  return v;
}
// scale of a row whose largest magnitude has these bits (the maximum is taken on the bits: infinities and NaN are the largest), and 1 / scale
__device__ __forceinline__ void q8_scale(uint32_t amax, float& scale, float& inv) {
  const float a = fmaxf(__uint_as_float(amax), Q8_TINY);
  const bool ok = amax < 0x7f800000u;
  scale = ok ? a * (1.0f / 127.0f) : __uint_as_float(0x7fc00000u);
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

// one wave per row, NCH chunks of 512 columns held in registers: every byte is read once and written once
template <typename T, int NCH, bool NORM>
__global__ __launch_bounds__(256) void rows_q8_kernel(const RowsQ8 p) {
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.x * (blockDim.x >> 6) + (threadIdx.x >> 6);
  if (row >= p.rows) return;
  const int nch = p.cols >> 3;
  const T* x = (const T*)p.x + (long)row * p.ldx;
  float v[NCH][8];
  float ss = 0.f;
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = lane + i * 64;
    if (c < nch) {
      ld8(x + c * 8, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    }
  }
  if (NORM) {
    if (p.delta) {
#pragma unroll
      for (int i = 0; i < NCH; ++i) {
        const int c = lane + i * 64;
        if (c < nch) {
          float d[8];
          ld8(p.delta + (long)row * p.ldd + c * 8, d);
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] += v[i][j];
          const uint4 s = pack8(d);           // the residual stream is bf16: the norm sees the value that the next layer will read
          unpack8(s, v[i]);
          if (p.h) *reinterpret_cast<uint4*>(p.h + (long)row * p.ldh + c * 8) = s;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
    const float rstd = rsqrtf(wave_sum(ss) / p.cols + p.eps);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = lane + i * 64;
      if (c < nch) {
        float w[8];
        ld8(p.w + c * 8, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = w[j] * (v[i][j] * rstd);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) { const uint32_t b = abs_bits(v[i][j]); amax = amax > b ? amax : b; }
  amax = wave_umax(amax);
  float scale, inv;
  q8_scale(amax, scale, inv);
  const bool ok = amax < 0x7f800000u;
  if (lane == 0) p.scale[row] = scale;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = lane + i * 64;
    if (c < nch) {
      uint2 o;
      o.x = q8_pack4(v[i], inv, ok); o.y = q8_pack4(v[i] + 4, inv, ok);
      *reinterpret_cast<uint2*>(p.q + (long)row * p.ldq + c * 8) = o;
    }
  }
}

// y[row][c] = scale[row] * q[row][c], 8 columns per lane
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
  *reinterpret_cast<uint4*>(y + (long)row * ldy + c * 8) = pack8(f);
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

// eight lanes per (entry, head, token); TOKENS: eight tokens of one head per wave (512 contiguous bytes of codes), else eight heads of one token
template <bool TOKENS>
__device__ __forceinline__ bool kv_unit(const KvQ8& p, int& e, int& h, int& t, int& at) {
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
  if (e >= p.E || h >= p.H || t >= p.T) return false;
  if (p.count && t >= p.count[e]) return false;
  const long a = (long)(p.pos ? p.pos[e] : p.pos0) + (p.pos_dev ? *p.pos_dev : 0) + t;
  at = (int)a;
  return a >= 0 && a < p.maxlen;     // a token behind the cache's end has no row
}

template <bool TOKENS>
__global__ __launch_bounds__(256) void kv_append_q8_kernel(const KvQ8 p) {
  int e = 0, h = 0, t = 0, at = 0;
  if (!kv_unit<TOKENS>(p, e, h, t, at)) return;      // whole groups of eight lanes
  const int c = threadIdx.x & 7;
  const long src = (long)e * p.bs + (long)t * p.rs + h * 64 + c * 8;
  const uint4 kr = *reinterpret_cast<const uint4*>(p.k + src), vr = *reinterpret_cast<const uint4*>(p.v + src);
  const long row = (long)e * p.e_rows + (long)h * p.h_rows + at;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float f[8];
    unpack8(w ? vr : kr, f);
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { const uint32_t b = abs_bits(f[j]); amax = amax > b ? amax : b; }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) { const uint32_t b = (uint32_t)__shfl_xor((int)amax, o, 64); amax = amax > b ? amax : b; }
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
  int e = 0, h = 0, t = 0, at = 0;
  if (!kv_unit<TOKENS>(p, e, h, t, at)) return;
  const int c = threadIdx.x & 7;
  const long dst = (long)e * p.bs + (long)t * p.rs + h * 64 + c * 8;
  const long row = (long)e * p.e_rows + (long)h * p.h_rows + at;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const uint2 u = *reinterpret_cast<const uint2*>((w ? p.vq : p.kq) + row * 64 + c * 8);
    const float s = (w ? p.vs : p.ks)[row];
    float f[8];
    q8_unpack4(u.x, f); q8_unpack4(u.y, f + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= s;
    *reinterpret_cast<uint4*>((w ? p.v : p.k) + dst) = pack8(f);
  }
}

// ---- single-query attention over the cache --------------------------------------------------------------------------------------------------
//   z_j = scale * ks_j <q, kq_j> + bias_j,   o = sum_j exp(z_j - m) vs_j vq_j / sum_j exp(z_j - m)
// A masked key is not part of the sums at all (whatever its codes and scale hold); a query that sees no key -- all masked, or a bias of
// -infinity everywhere -- gets the mean of its keys' values, as softmax over equal scores gives (modeling_t5.py:996,559), and a query without
// keys gets zeros.
constexpr int PIECE = 512;            // keys per block; fixed, so that a sequence's result does not depend on its batch
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

template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

// mean of the values of n keys of one (entry, head) by a block of 256 threads; lds: 256 floats.  The rare row without a visible key.
__device__ float attn_q8_mean(const i8* vq, const float* vs, int n, float* lds) {
  const int d = threadIdx.x & 63, part = threadIdx.x >> 6;
  float s = 0.f;
  for (int k = part; k < n; k += 4) s += vs[k] * (float)vq[(long)k * 64 + d];
  __syncthreads();
  lds[threadIdx.x] = s;
  __syncthreads();
  s = lds[d] + lds[64 + d] + lds[128 + d] + lds[192 + d];
  __syncthreads();
  return n > 0 ? s / (float)n : 0.f;
}

// block = 4 waves = up to PIECE keys of one (entry, head) against G of its queries.  lane = (key slot lane >> 2, 16 dimensions lane & 3): one
// wave load is 16 whole keys (1 KiB)
template <int G>
__global__ __launch_bounds__(256) void attn_q8_kernel(const AttnQ8 p) {
  __shared__ float s_m[G][4], s_l[G][4], s_o[G][4][64], s_red[256];
  __shared__ unsigned long long s_bits[PIECE / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slot = lane >> 2, c = lane & 3;
  const int gc = blockIdx.x % p.gchunks, eh = blockIdx.x / p.gchunks;
  const int h = eh % p.H, e = eh / p.H;
  const int piece = blockIdx.y, k0 = piece * PIECE;
  const int n = attn_q8_keys(p, e);
  if (k0 >= n && piece > 0) return;
  const int end = min(n - k0, PIECE);
  const int g0 = gc * G, ng = min(G, p.G - g0);
  const long base = (long)e * p.e_rows + (long)h * p.h_rows;
  const i8 *kq = p.kq + base * 64, *vq = p.vq + base * 64;
  const float *ks = p.ks + base, *vs = p.vs + base;
  const float* bias = nullptr;
  if (p.bias) bias = p.bias + (long)h * p.bias_ld + (p.pos_dev ? p.bias_maxlen - 1 - *p.pos_dev : 0);
  // visible keys of the piece, one bit each
  for (int r = 0; r < PIECE / 256; ++r) {
    const int k = r * 256 + tid;
    bool see = k < end;
    if (see && p.mask) see = p.mask[(long)e * p.mask_ld + k0 + k] != 0;
    const unsigned long long b = __ballot(see);
    if (lane == 0) s_bits[r * 4 + wave] = b;
  }
  float qv[G][16];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const long qr = (long)(e * p.G + g0 + (g < ng ? g : 0)) * p.q_bs + h * 64 + c * 16;
    ld8(p.q + qr, qv[g]); ld8(p.q + qr + 8, qv[g] + 8);
  }
  __syncthreads();
  float m[G], l[G], acc[G][16];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY; l[g] = 0.f;
#pragma unroll
    for (int d = 0; d < 16; ++d) acc[g][d] = 0.f;
  }
  for (int ch = wave; ch < PIECE / 64; ch += 4) {
    const unsigned long long bits = s_bits[ch];
    if (bits == 0) continue;
    uint4 kr[4], vr[4];
    float sk[4], sv[4], bz[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int k = ch * 64 + j * 16 + slot;
      k = k0 + (k < end ? k : end - 1);
      kr[j] = *reinterpret_cast<const uint4*>(kq + (long)k * 64 + c * 16);
      vr[j] = *reinterpret_cast<const uint4*>(vq + (long)k * 64 + c * 16);
      sk[j] = ks[k]; sv[j] = vs[k];
      bz[j] = bias ? bias[k] : 0.f;
    }
    float sc[G][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[16];
      q8_unpack4(kr[j].x, f); q8_unpack4(kr[j].y, f + 4); q8_unpack4(kr[j].z, f + 8); q8_unpack4(kr[j].w, f + 12);
      const bool see = (bits >> (j * 16 + slot)) & 1ull;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float d = 0.f;
#pragma unroll
        for (int t = 0; t < 16; ++t) d = fmaf(qv[g][t], f[t], d);
        d = dpp_add<0xB1>(d);                       // the four lanes of a key: quad permutes [1,0,3,2] and [2,3,0,1]
        d = dpp_add<0x4E>(d);
        sc[g][j] = see ? d * sk[j] * p.scale + bz[j] : -INFINITY;
      }
      if (!see) sv[j] = 0.f;                        // what a masked key holds never reaches the sums
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float mn = fmaxf(fmaxf(fmaxf(sc[g][0], sc[g][1]), fmaxf(sc[g][2], sc[g][3])), m[g]);
      const float a = rescale(m[g], mn);
      m[g] = mn;
      l[g] *= a;
#pragma unroll
      for (int d = 0; d < 16; ++d) acc[g][d] *= a;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = sc[g][j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((sc[g][j] - mn) * LOG2E);
        l[g] += w;
        sc[g][j] = w * sv[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[16];
      q8_unpack4(vr[j].x, f); q8_unpack4(vr[j].y, f + 4); q8_unpack4(vr[j].z, f + 8); q8_unpack4(vr[j].w, f + 12);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int d = 0; d < 16; ++d) acc[g][d] = fmaf(sc[g][j], f[d], acc[g][d]);
    }
  }
  // the 16 key slots of the wave, then the waves
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float M = m[g];
#pragma unroll
    for (int o = 4; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    const float a = rescale(m[g], M);
    float L = l[g] * a;
    L = dpp_add<0x128>(L); L = dpp_add<0x124>(L);   // row_ror 8 and 4 keep lane & 3
    L += __shfl_xor(L, 16, 64); L += __shfl_xor(L, 32, 64);
#pragma unroll
    for (int d = 0; d < 16; ++d) {
      float s = acc[g][d] * a;
      s = dpp_add<0x128>(s); s = dpp_add<0x124>(s);
      s += __shfl_xor(s, 16, 64); s += __shfl_xor(s, 32, 64);
      if (slot == 0) s_o[g][wave][c * 16 + d] = s;
    }
    if (lane == 0) { s_m[g][wave] = M; s_l[g][wave] = L; }
  }
  __syncthreads();
  bool none = false;                                 // a query of this block without a visible key (single-piece form only)
#pragma unroll
  for (int g = 0; g < G; ++g) none |= s_l[g][0] + s_l[g][1] + s_l[g][2] + s_l[g][3] == 0.f;
  float mean = 0.f;
  if (none && p.np == 1) mean = attn_q8_mean(vq, vs, n, s_red);
  for (int t = tid; t < ng * 64; t += 256) {
    const int g = t >> 6, d = t & 63;
    float M = s_m[g][0];
    for (int w = 1; w < 4; ++w) M = fmaxf(M, s_m[g][w]);
    float L = 0.f, O = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float a = rescale(s_m[g][w], M);
      L += s_l[g][w] * a; O += s_o[g][w][d] * a;
    }
    const long b = (long)e * p.G + g0 + g;
    if (p.np == 1) {
      p.o[b * p.o_bs + h * 64 + d] = f2bf(L == 0.f ? mean : O / L);
    } else {
      float* w = p.ws + ((b * p.H + h) * p.np + piece) * 66;
      w[d] = O;
      if (d == 0) { w[64] = M; w[65] = L; }
    }
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
  for (int i = wave; i < np; i += 4) {
    const float mi = w[i * 66 + 64], li = w[i * 66 + 65], oi = w[i * 66 + d];
    const float mn = fmaxf(M, mi), a = rescale(M, mn), c = rescale(mi, mn);
    L = L * a + li * c; O = O * a + oi * c;
    M = mn;
  }
  s_o[wave][d] = O;
  if (d == 0) { s_m[wave] = M; s_l[wave] = L; }
  __syncthreads();
  M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  L = 0.f; O = 0.f;
  for (int i = 0; i < 4; ++i) { const float a = rescale(s_m[i], M); L += s_l[i] * a; O += s_o[i][d] * a; }
  float r = O / L;
  if (L == 0.f) {                                    // the same for every thread of the block
    const long base = (long)e * p.e_rows + (long)h * p.h_rows;
    r = attn_q8_mean(p.vq + base * 64, p.vs + base, n, s_red);
  }
  if (wave == 0) p.o[(long)b * p.o_bs + h * 64 + d] = f2bf(r);
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

template <typename T, bool NORM> int rows_q8_launch(const RowsQ8& p, hipStream_t s) {
  const dim3 grid((unsigned)((p.rows + 3) / 4)), block(256);
  if (p.cols <= 512) hipLaunchKernelGGL((rows_q8_kernel<T, 1, NORM>), grid, block, 0, s, p);
  else if (p.cols <= 1024) hipLaunchKernelGGL((rows_q8_kernel<T, 2, NORM>), grid, block, 0, s, p);
  else if (p.cols <= 2048) hipLaunchKernelGGL((rows_q8_kernel<T, 4, NORM>), grid, block, 0, s, p);
  else if (p.cols <= 4096) hipLaunchKernelGGL((rows_q8_kernel<T, 8, NORM>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((rows_q8_kernel<T, 16, NORM>), grid, block, 0, s, p);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}

int kv_check(const char* who, const v2s_kv_q8* c, const void* k, const void* v, int64_t bs, int64_t rs, int32_t T) {
  V2S_CHECK(c && c->k && c->ks && c->v && c->vs && k && v, V2S_ERR_ARG, "%s: NULL pointer", who);
  V2S_CHECK(c->entries > 0 && c->heads > 0 && c->maxlen > 0 && T > 0, V2S_ERR_SHAPE, "%s: entries, heads, maxlen and T must be positive", who);
  V2S_CHECK(c->h_rows >= c->maxlen && c->e_rows >= c->maxlen, V2S_ERR_SHAPE, "%s: row strides must be at least maxlen (%d)", who, c->maxlen);
  V2S_CHECK(aligned(c->k, 16) && aligned(c->v, 16) && aligned(k, 16) && aligned(v, 16) && aligned(c->ks, 4) && aligned(c->vs, 4) && bs % 8 == 0 && rs % 8 == 0,
            V2S_ERR_ALIGN, "%s: pointers must be 16-byte aligned and strides multiples of 8 elements", who);
  const int64_t units = (int64_t)c->entries * ((c->heads + 7) & ~7) * (((int64_t)T + 7) & ~7);
  V2S_CHECK(units < (int64_t)0xffffff00u, V2S_ERR_SHAPE, "%s: entries x heads x T too large for one launch", who);
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
  V2S_CHECK(rows > 0 && cols > 0 && cols % 8 == 0 && cols <= 8192, V2S_ERR_SHAPE, "v2s_quant_rows_q8: unsupported shape rows=%d cols=%d (cols a multiple of 8, <= 8192)", rows, cols);
  V2S_CHECK(ldx >= cols && ldq >= cols, V2S_ERR_SHAPE, "v2s_quant_rows_q8: a row stride is shorter than the row");
  V2S_CHECK(aligned(x, 16) && aligned(q, 8) && aligned(scale, 4) && ldx % 8 == 0 && ldq % 8 == 0, V2S_ERR_ALIGN,
            "v2s_quant_rows_q8: x must be 16-byte and q 8-byte aligned, strides multiples of 8");
  RowsQ8 p = {};
  p.x = x; p.ldx = ldx; p.q = (i8*)q; p.ldq = ldq; p.scale = scale; p.rows = rows; p.cols = cols;
  return x_dtype == V2S_F32 ? rows_q8_launch<float, false>(p, (hipStream_t)stream) : rows_q8_launch<bf16_t, false>(p, (hipStream_t)stream);
}

extern "C" int v2s_rmsnorm_q8(const void* x, int64_t ldx, const void* delta, int64_t ldd, const float* w, void* h, int64_t ldh, int8_t* q, int64_t ldq,
                              float* scale, int32_t rows, int32_t cols, float eps, void* stream) {
  V2S_CHECK(x && w && q && scale, V2S_ERR_ARG, "v2s_rmsnorm_q8: NULL pointer");
  V2S_CHECK(!h || delta, V2S_ERR_ARG, "v2s_rmsnorm_q8: h is the sum x + delta, it needs delta");
  V2S_CHECK(eps >= 0.f, V2S_ERR_ARG, "v2s_rmsnorm_q8: eps must not be negative");
  V2S_CHECK(rows > 0 && cols > 0 && cols % 8 == 0 && cols <= 8192, V2S_ERR_SHAPE, "v2s_rmsnorm_q8: unsupported shape rows=%d cols=%d (cols a multiple of 8, <= 8192)", rows, cols);
  V2S_CHECK(ldx >= cols && ldq >= cols && (!delta || ldd >= cols) && (!h || ldh >= cols), V2S_ERR_SHAPE, "v2s_rmsnorm_q8: a row stride is shorter than the row");
  V2S_CHECK(aligned(x, 16) && aligned(delta, 16) && aligned(h, 16) && aligned(w, 16) && aligned(q, 8) && aligned(scale, 4) && ldx % 8 == 0 && ldq % 8 == 0 &&
                (!delta || ldd % 8 == 0) && (!h || ldh % 8 == 0),
            V2S_ERR_ALIGN, "v2s_rmsnorm_q8: x, delta, w and h must be 16-byte and q 8-byte aligned, strides multiples of 8");
  RowsQ8 p = {};
  p.x = x; p.ldx = ldx; p.delta = (const bf16_t*)delta; p.ldd = ldd; p.w = w; p.h = (bf16_t*)h; p.ldh = ldh; p.q = (i8*)q; p.ldq = ldq; p.scale = scale;
  p.rows = rows; p.cols = cols; p.eps = eps;
  return rows_q8_launch<bf16_t, true>(p, (hipStream_t)stream);
}

extern "C" int v2s_dequant_q8(const int8_t* q, int64_t ldq, const float* scale, void* y, int64_t ldy, int32_t rows, int32_t cols, void* stream) {
  V2S_CHECK(q && scale && y, V2S_ERR_ARG, "v2s_dequant_q8: NULL pointer");
  V2S_CHECK(rows > 0 && cols > 0 && cols % 8 == 0, V2S_ERR_SHAPE, "v2s_dequant_q8: unsupported shape rows=%d cols=%d (cols a multiple of 8)", rows, cols);
  V2S_CHECK(ldq >= cols && ldy >= cols, V2S_ERR_SHAPE, "v2s_dequant_q8: a row stride is shorter than the row");
  V2S_CHECK(aligned(q, 8) && aligned(y, 16) && aligned(scale, 4) && ldq % 8 == 0 && ldy % 8 == 0, V2S_ERR_ALIGN,
            "v2s_dequant_q8: q must be 8-byte and y 16-byte aligned, strides multiples of 8");
  const int64_t blocks = ((int64_t)rows * (cols / 8) + 255) / 256;
  V2S_CHECK(blocks <= 0x7fffffff, V2S_ERR_SHAPE, "v2s_dequant_q8: too many elements for one launch");
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
  const int per = G >= 4 ? 4 : (G >= 2 ? 2 : 1);
  p.gchunks = (G + per - 1) / per;
  V2S_CHECK((int64_t)c.entries * c.heads * p.gchunks <= 0x7fffffff && p.np <= 65535, V2S_ERR_SHAPE, "v2s_decode_attn_q8: too many rows or keys for one launch");
  const dim3 grid((unsigned)(c.entries * c.heads * p.gchunks), (unsigned)p.np);
  hipStream_t s = (hipStream_t)stream;
  if (per == 4) hipLaunchKernelGGL(attn_q8_kernel<4>, grid, dim3(256), 0, s, p);
  else if (per == 2) hipLaunchKernelGGL(attn_q8_kernel<2>, grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL(attn_q8_kernel<1>, grid, dim3(256), 0, s, p);
  V2S_LAUNCH_CHECK();
  if (p.np > 1) {
    hipLaunchKernelGGL(attn_q8_join_kernel, dim3((unsigned)(a->B * c.heads)), dim3(256), 0, s, p);
    V2S_LAUNCH_CHECK();
  }
  return V2S_OK;
}
