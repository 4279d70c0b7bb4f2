// One sampling step from given random numbers (gfx950): temperature, top-k, top-p and min-p over rows of logits, one block per row.
// Replaces transformers==4.28.0 sample()'s warpers and multinomial draw (call site model/vid2seq.py:150-162) where the caller owns the random
// numbers.
//   w_i = exp((z_i - max z) / T);  order: larger logit first, equal logits by index;  top-k: the first k;  top-p: preceding mass < p * mass;
//   min-p: w_i >= min_p;  draw: the first token in index order whose running kept mass exceeds u * kept mass
// No sort: the boundary of top-k / top-p is found by a histogram over the distance to the maximum (counts, or masses), which names the one bin
// that holds it, and by ranking the few tokens of that bin exactly.  Masses are 64-bit integers (2^46 = weight one): their sums are exact, so the
// result depends neither on the order of the atomics nor on how the row is cut.  A row of 32768 logits stays in the registers of its block and is
// read once.
#include <math.h>
#include "v2s_common.h"

namespace {

typedef unsigned long long u64;
constexpr int NT = 1024, STEP = NT * 4;     // tokens per pass of the block: four consecutive ones per thread
constexpr int NBIN = 2048, CAP = 1024;
constexpr float BIN_RANGE = 33.0f;          // exp(-33) < 2^-47: what lies further from the maximum has no mass
constexpr double ONE = 70368744177664.0;    // 2^46: 131072 tokens of weight one sum to 2^63

struct SampleP {
  const void* logits; long ld; int V;
  double inv_temp; float bin_scale;
  int top_k; double top_p, min_p;
  const float* u; long u_ld; int u_steps;
  long* next_tok; float* logp; int* unfinished; int eos_id, pad_id;
  long* seq_out; long seq_ld; const int* pos_dev; int min_length;
};

__device__ __forceinline__ float logit_of(float v) { return v; }
__device__ __forceinline__ float logit_of(bf16_t v) { return bf2f(v); }
// ascending in the order of the tokens: larger logits first, then lower indexes (z is never -0 or NaN here)
__device__ __forceinline__ u64 order_key(float z, int idx) {
  const uint32_t b = __float_as_uint(z);
  const uint32_t asc = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return ((u64)(~asc) << 32) | (uint32_t)idx;
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += (u64)__shfl_xor((long long)v, o, 64);
  return v;
}
__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) {      // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const u64 w = (u64)__shfl_up((long long)v, o, 64); if (lane >= o) v += w; }
  return v;
}
__device__ u64 block_sum64(u64 v, u64* red, int tid) {
  v = wave_sum64(v);
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = v;
  __syncthreads();
  u64 s = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += red[i];
  return s;
}

// NJ passes of the block hold the row in registers; NJ = 0: the row is read again for every pass (V > 32768)
template <typename T, int NJ>
__global__ __launch_bounds__(NT) void sample_kernel(const SampleP p) {
  __shared__ u64 s_mass[NBIN];
  __shared__ uint32_t s_cnt[NBIN];
  __shared__ u64 s_key[CAP], s_w[CAP];
  __shared__ u64 s_red[NT / 64], s_thr, s_base;
  __shared__ float s_max[NT / 64];
  __shared__ int s_n, s_bin, s_nan, s_pick;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x, V = p.V;
  const T* z0 = (const T*)p.logits + (long)row * p.ld;
  const int step = p.pos_dev ? *p.pos_dev : 0;
  const int ban = (p.eos_id >= 0 && (p.pos_dev ? step + 1 : 0) < p.min_length) ? p.eos_id : -1;
  const int nj = NJ ? NJ : (V + STEP - 1) / STEP;
  float zr[NJ ? NJ : 1][4];
  int nan_at = V;
  float zmax = -INFINITY;

  auto load = [&](int j, float (&z)[4]) {
    const int i0 = j * STEP + tid * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = i0 + i < V && i0 + i != ban ? logit_of(z0[i0 + i]) + 0.0f : -INFINITY;
  };
  auto each = [&](auto f) {                 // f(j, index, logit) for the tokens of this thread, in index order
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) { const int idx = j * STEP + tid * 4 + i; if (idx < V) f(j, idx, zr[j][i]); }
    } else {
      for (int j = 0; j < nj; ++j) {
        float z[4];
        load(j, z);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const int idx = j * STEP + tid * 4 + i; if (idx < V) f(j, idx, z[i]); }
      }
    }
  };

  if constexpr (NJ > 0) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) load(j, zr[j]);
  }
  each([&](int, int idx, float z) {
    if (z != z) nan_at = min(nan_at, idx);
    zmax = fmaxf(zmax, z);
  });
  zmax = wave_max(zmax);
  if (tid == 0) { s_nan = V; s_pick = -1; s_n = 0; s_bin = NBIN; }
  if (lane == 0) s_max[wave] = zmax;
  for (int b = tid; b < NBIN; b += NT) { s_cnt[b] = 0; s_mass[b] = 0; }
  __syncthreads();
  if (nan_at < V) atomicMin(&s_nan, nan_at);
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) zmax = fmaxf(zmax, s_max[i]);
  __syncthreads();

  auto finish = [&](int tok, float lp) {    // one thread
    long t = tok;
    if (p.unfinished) {
      const int un = p.unfinished[row];
      if (!un) { t = p.pad_id; lp = 0.f; }
      p.unfinished[row] = un && t != p.eos_id;
    }
    p.next_tok[row] = t;
    if (p.logp) p.logp[row] = lp;
    if (p.seq_out && step + 1 >= 0 && step + 1 < p.seq_ld) p.seq_out[(long)row * p.seq_ld + step + 1] = t;
  };
  if (s_nan < V) {                          // the same for the whole block
    if (tid == 0) finish(s_nan, __uint_as_float(0x7fc00000u));
    return;
  }

  auto bin_of = [&](float z) { return z == zmax ? 0 : (int)fminf((zmax - z) * p.bin_scale, (float)(NBIN - 1)); };
  auto weight = [&](float z) -> double { return z == zmax ? 1.0 : exp(((double)z - (double)zmax) * p.inv_temp); };
  auto mass = [&](float z) -> u64 {         // round to nearest: 2^46 w < 2^52, so the sum below holds it in its low bits
    return (u64)__double_as_longlong(weight(z) * ONE + 4503599627370496.0) & 0xfffffffffffffull;
  };

  // bin of the boundary: the first one at which the running sum (of counts or masses) reaches the goal; s_base = the sum before it
  auto find_bin = [&](auto value, auto reached) {
    const u64 a = value(2 * tid), b = value(2 * tid + 1);
    const u64 inc = wave_scan64(a + b, lane);
    __syncthreads();
    if (lane == 63) s_red[wave] = inc;
    if (tid == 0) { s_bin = NBIN - 1; s_n = 0; }
    __syncthreads();
    u64 pre = inc - (a + b);
    for (int i = 0; i < wave; ++i) pre += s_red[i];
    if (!reached(pre) && reached(pre + a)) { s_bin = 2 * tid; s_base = pre; }
    else if (!reached(pre + a) && reached(pre + a + b)) { s_bin = 2 * tid + 1; s_base = pre + a; }
    __syncthreads();
  };
  // the last kept token of that bin, as an order key: the first one at which the running sum of `value` over the bin's tokens in order reaches
  // the goal.  `in` = tokens that take part at all
  auto resolve = [&](auto in, auto value, auto reached) -> u64 {
    const int bin = s_bin;
    const u64 base = s_base;
    each([&](int, int idx, float z) {
      if (bin_of(z) == bin && in(z, idx)) {
        const int at = atomicAdd(&s_n, 1);
        if (at < CAP) { s_key[at] = order_key(z, idx); s_w[at] = value(z); }
      }
    });
    __syncthreads();
    const int n = s_n;
    if (n <= CAP) {
      if (tid < n) {
        const u64 key = s_key[tid], w = s_w[tid];
        u64 pre = base;
        for (int i = 0; i < n; ++i) pre += s_key[i] < key ? s_w[i] : 0;
        if (!reached(pre) && reached(pre + w)) s_thr = key;
      }
      __syncthreads();
      return s_thr;
    }
    // too many tokens within one bin (a plateau of equal logits): bisection on the order key
    u64 lo = 0, hi = ~0ull;                 // sum(keys <= hi) reaches the goal
    while (lo < hi) {
      const u64 mid = lo + ((hi - lo) >> 1);
      u64 s = 0;
      each([&](int, int idx, float z) {
        if (bin_of(z) == bin && in(z, idx) && order_key(z, idx) <= mid) s += value(z);
      });
      s = block_sum64(s, s_red, tid);
      if (reached(base + s)) hi = mid; else lo = mid + 1;
    }
    return lo;
  };

  u64 thr = ~0ull;                          // order key of the last token that top-k and top-p keep
  if (p.top_k > 0 && p.top_k < V) {
    each([&](int, int, float z) { const int b = bin_of(z); if (b < NBIN - 1) atomicAdd(&s_cnt[b], 1u); });
    __syncthreads();
    const u64 k = (u64)p.top_k;
    find_bin([&](int b) { return (u64)s_cnt[b]; }, [&](u64 s) { return s >= k; });
    if (s_bin < NBIN - 1)                   // otherwise every token with any mass is among the first k
      thr = resolve([](float, int) { return true; }, [](float) { return (u64)1; }, [&](u64 s) { return s >= k; });
    __syncthreads();
  }
  if (p.top_p < 1.0) {
    const u64 kt = thr;
    u64 total = 0;
    each([&](int, int idx, float z) {
      const int b = bin_of(z);
      if (b < NBIN - 1 && order_key(z, idx) <= kt) { const u64 m = mass(z); total += m; atomicAdd(&s_mass[b], m); }
    });
    total = block_sum64(total, s_red, tid);
    const double goal = p.top_p * (double)total;
    const auto reached = [&](u64 s) { return (double)s >= goal; };
    find_bin([&](int b) { return s_mass[b]; }, reached);
    thr = resolve([&](float z, int idx) { return order_key(z, idx) <= kt; }, mass, reached);
    __syncthreads();
  }

  // kept mass of each segment of 256 consecutive tokens (one wave of one pass); segments in index order are (pass, wave)
  u64* seg = s_mass;                        // [nj][16] <= 512
  auto kept = [&](float z, int idx) -> u64 {
    if (bin_of(z) >= NBIN - 1 || order_key(z, idx) > thr) return 0;
    const double w = weight(z);
    return w >= p.min_p ? (u64)__double_as_longlong(w * ONE + 4503599627370496.0) & 0xfffffffffffffull : 0;
  };
  {
    u64 own = 0;
    int at = 0;
    auto flush = [&](int j) {
      const u64 s = wave_sum64(own);
      if (lane == 0) seg[j * (NT / 64) + wave] = s;
      own = 0;
    };
    if constexpr (NJ > 0) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { const int idx = j * STEP + tid * 4 + i; if (idx < V) own += kept(zr[j][i], idx); }
        flush(j);
      }
    } else {
      for (at = 0; at < nj; ++at) {
        float z[4];
        load(at, z);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const int idx = at * STEP + tid * 4 + i; if (idx < V) own += kept(z[i], idx); }
        flush(at);
      }
    }
  }
  __syncthreads();
  // the segment in which the running mass passes u * total (one wave: up to 512 segments, eight per lane), else the last one with any mass
  const int nseg = nj * (NT / 64);
  const float uf = p.u[(p.pos_dev ? (long)max(0, min(step, p.u_steps - 1)) * p.u_ld : 0) + row];
  const double u = (double)fmaxf(uf, 0.f);
  if (wave == 0) {
    u64 own = 0;
    for (int i = 0; i < 8; ++i) { const int sgi = lane * 8 + i; if (sgi < nseg) own += seg[sgi]; }
    const u64 inc = wave_scan64(own, lane);
    const u64 total = (u64)__shfl((long long)inc, 63, 64);
    const double goal = u * (double)total;
    u64 run = inc - own;
    int found = -1, last = -1;
    u64 fpre = 0, lpre = 0;
    for (int i = 0; i < 8; ++i) {
      const int sgi = lane * 8 + i;
      const u64 m = sgi < nseg ? seg[sgi] : 0;
      if (m > 0) { last = sgi; lpre = run; }
      if (found < 0 && m > 0 && (double)(run + m) > goal) { found = sgi; fpre = run; }
      run += m;
    }
    const u64 any = __ballot(found >= 0), have = __ballot(last >= 0);
    const int src = any ? __builtin_ctzll(any) : 63 - __builtin_clzll(have);
    if (lane == src) { s_bin = any ? found : last; s_base = any ? fpre : lpre; s_thr = total; }
  }
  __syncthreads();
  const int sg = s_bin, sj = sg / (NT / 64);
  if (wave == sg % (NT / 64)) {
    const double goal = u * (double)s_thr;
    float z[4];
    load(sj, z);
    u64 m[4], own = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) { const int idx = sj * STEP + tid * 4 + i; m[i] = idx < V ? kept(z[i], idx) : 0; own += m[i]; }
    u64 run = s_base + wave_scan64(own, lane) - own;
    int found = -1, last = -1;
    float fz = 0.f, lz = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (m[i] > 0) { last = sj * STEP + tid * 4 + i; lz = z[i]; }
      if (found < 0 && m[i] > 0 && (double)(run + m[i]) > goal) { found = sj * STEP + tid * 4 + i; fz = z[i]; }
      run += m[i];
    }
    const u64 any = __ballot(found >= 0), have = __ballot(last >= 0);
    const int src = any ? __builtin_ctzll(any) : 63 - __builtin_clzll(have);
    if (lane == src) {
      const float zp = any ? fz : lz;
      const double d = zp == zmax ? 0.0 : ((double)zp - (double)zmax) * p.inv_temp;
      finish(any ? found : last, (float)(d - log((double)s_thr / ONE)));
    }
  }
}

template <typename T> int sample_launch(const SampleP& p, int rows, hipStream_t s) {
  const int nj = (p.V + STEP - 1) / STEP;
  const dim3 grid(rows), block(NT);
  if (nj <= 1) hipLaunchKernelGGL((sample_kernel<T, 1>), grid, block, 0, s, p);
  else if (nj <= 2) hipLaunchKernelGGL((sample_kernel<T, 2>), grid, block, 0, s, p);
  else if (nj <= 4) hipLaunchKernelGGL((sample_kernel<T, 4>), grid, block, 0, s, p);
  else if (nj <= 8) hipLaunchKernelGGL((sample_kernel<T, 8>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((sample_kernel<T, 0>), grid, block, 0, s, p);
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}

}  // namespace

extern "C" int v2s_sample_step(const void* logits, int32_t logits_dtype, int64_t ld, int32_t rows, int32_t V, double temperature, int32_t top_k, double top_p,
                               double min_p, const float* u, int64_t u_ld, int32_t u_steps, int64_t* next_tok, float* logp, int32_t* unfinished, int32_t eos_id,
                               int32_t pad_id, int64_t* seq_out, int64_t seq_ld, const int32_t* pos_dev, int32_t min_length, void* stream) {
  V2S_CHECK(logits && u && next_tok, V2S_ERR_ARG, "v2s_sample_step: NULL pointer");
  V2S_CHECK(logits_dtype == V2S_F32 || logits_dtype == V2S_BF16, V2S_ERR_DTYPE, "v2s_sample_step: logits must be fp32 or bf16");
  V2S_CHECK(rows > 0 && V > 0 && V <= 131072 && ld >= V, V2S_ERR_SHAPE, "v2s_sample_step: unsupported shape rows=%d V=%d ld=%lld (V <= 131072, ld >= V)", rows, V, (long long)ld);
  V2S_CHECK(temperature >= 1e-6 && temperature <= 1e6, V2S_ERR_ARG, "v2s_sample_step: temperature must be in [1e-6, 1e6]");
  V2S_CHECK(top_k >= 0 && top_p > 0.0 && top_p <= 1.0 && min_p >= 0.0 && min_p <= 1.0, V2S_ERR_ARG, "v2s_sample_step: top_k >= 0, top_p in (0, 1], min_p in [0, 1]");
  V2S_CHECK(!seq_out || pos_dev, V2S_ERR_ARG, "v2s_sample_step: seq_out needs pos_dev");
  V2S_CHECK(!pos_dev || (u_ld >= rows && u_steps > 0), V2S_ERR_SHAPE, "v2s_sample_step: with pos_dev, u is a table of u_steps > 0 rows of u_ld >= rows numbers");
  SampleP p;
  p.logits = logits; p.ld = ld; p.V = V; p.inv_temp = 1.0 / temperature; p.bin_scale = (float)((NBIN - 1) / (BIN_RANGE * temperature));
  p.top_k = top_k; p.top_p = top_p; p.min_p = min_p; p.u = u; p.u_ld = u_ld; p.u_steps = u_steps; p.next_tok = (long*)next_tok; p.logp = logp; p.unfinished = unfinished;
  p.eos_id = eos_id; p.pad_id = pad_id; p.seq_out = (long*)seq_out; p.seq_ld = seq_ld; p.pos_dev = pos_dev; p.min_length = min_length;
  return logits_dtype == V2S_F32 ? sample_launch<float>(p, rows, (hipStream_t)stream) : sample_launch<bf16_t>(p, rows, (hipStream_t)stream);
}
