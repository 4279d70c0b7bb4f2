// One sampling step from given random numbers (gfx950): temperature, top-k, top-p and min-p over rows of logits, one block per row.
// Replaces transformers==4.28.0 sample()'s warpers and multinomial draw (call site model/vid2seq.py:150-162) where the caller owns the random
// numbers.
//   w_i = exp((z_i - max z) / T);  order: larger logit first, equal logits by index;  top-k: the first k;  top-p: preceding mass < p * mass;
//   min-p: w_i >= min_p;  draw: the first token in index order whose running kept mass exceeds u * kept mass
// No sort: the boundary of top-k / top-p is found by a histogram over the distance to the maximum (counts, or masses), which names the one bin
// that holds it, and by ranking the few tokens of that bin exactly.  Masses are 64-bit integers (2^46 = weight one): their sums are exact, so the
// result depends neither on the order of the atomics nor on how the row is cut.
// A row of up to 32768 logits is read from memory once and stays in LDS as fp32 (larger ones are read again for every pass, mostly from L2).  The
// passes over it are bound by VALU issue, not by memory: one instruction per logit costs a block 0.2 us at V = 32228.  Hence: the weights' exponential
// is a table and five terms of its own, small top-k never touches most logits, and the last pass compares all tokens but weighs only those it keeps.
// 64 rows of 32228 logits, top-k 50 and top-p 0.95: 11.5 us; 256 rows, top-p 0.92 and min-p: 27.5 us, a third of it the exact masses.
#include <math.h>
#include "v2s_common.h"

namespace {

typedef unsigned long long u64;
constexpr int NT = 1024, STEP = NT * 4;     // tokens per pass of the block: four consecutive ones per thread
constexpr int NBIN = 2048, CAP = 512;
constexpr int ROW_MAX = 8;                  // passes whose logits fit LDS: 32768 fp32 = 128 KiB, next to 24 KiB of tables
constexpr int SMALL_K = 128, SMALL_N = NT / 4; // top-k by candidate list: every step costs each candidate a walk over the others, four threads share it
constexpr float BIN_RANGE = 33.0f;          // exp(-33) < 2^-47: what lies further from the maximum has no mass
constexpr double ONE = 70368744177664.0;    // 2^46: 131072 tokens of weight one sum to 2^63

struct SampleP {
  const void* logits; long ld; int V, cpt, log_cpt;
  double inv_temp, exp2_scale; float bin_scale;   // 1 / T, log2(e) / T, bins per unit of logit
  int top_k; double top_p, min_p;
  const float* u; long u_ld; int u_steps;
  long* next_tok; float* logp; int* unfinished; int eos_id, pad_id;
  long* seq_out; long seq_ld; const int* pos_dev; int min_length;
};

// ascending in the order of the tokens: larger logits first, then lower indexes (z is never -0 or NaN here)
__device__ __forceinline__ u64 order_key(float z, int idx) {
  const uint32_t b = __float_as_uint(z);
  const uint32_t asc = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  return ((u64)(~asc) << 32) | (uint32_t)idx;
}
__device__ __forceinline__ float key_logit(u64 key) {
  const uint32_t asc = ~(uint32_t)(key >> 32);
  return __uint_as_float((asc >> 31) ? asc ^ 0x80000000u : ~asc);
}
// 2^46 * 2^t for t <= 0 by a table of 2^(i / 64), which the compiler sums from the series of exp(i / 64 ln 2), and the first terms of the same series: t = n / 64
// + r, |r| <= 1 / 128 (remainder below 2^-54).  Sixteen instructions in 64 bits; the series alone took 25, the library's exp over 40.
constexpr double LN2 = 0.69314718055994530942;
struct Powers {
  double v[64];
  constexpr Powers() : v() {
    for (int i = 0; i < 64; ++i) {
      v[i] = 1.0;
      for (int k = 19; k > 0; --k) v[i] = v[i] * (i / 64.0 * LN2) / k + 1.0;
    }
  }
};
__device__ constexpr Powers POWERS;
__device__ __forceinline__ double exp2_mass(double t, const double* tab) {
  constexpr double MAGIC = 105553116266496.0;      // 1.5 * 2^46: adding it leaves multiples of 1 / 64
  constexpr double C1 = LN2, C2 = C1 * LN2 / 2, C3 = C2 * LN2 / 3, C4 = C3 * LN2 / 4, C5 = C4 * LN2 / 5;
  const double t2 = t + MAGIC;
  const int n = __double2loint(t2);
  const double r = t - (t2 - MAGIC);
  const double s = fma(fma(fma(fma(fma(C5, r, C4), r, C3), r, C2), r, C1), r, 1.0);
  return tab[n & 63] * s * __hiloint2double(((n >> 6) + 46 + 1023) << 20, 0);
}
// round to nearest: 2^46 w < 2^52, so the sum holds it in its low bits
__device__ __forceinline__ u64 mass_of(double w46) { return (u64)__double_as_longlong(w46 + 4503599627370496.0) & 0xfffffffffffffull; }
// scan and sum of a wave by row shifts and row broadcasts of the vector unit (a shuffle through LDS costs five times the latency a step)
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t lane_step(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS> __device__ __forceinline__ u64 lane_step(u64 v) {
  return (u64)lane_step<CTRL, ROWS>((uint32_t)v) | ((u64)lane_step<CTRL, ROWS>((uint32_t)(v >> 32)) << 32);
}
template <typename U> __device__ __forceinline__ U wave_scan(U v) {       // inclusive
  v += lane_step<0x111, 0xf>(v); v += lane_step<0x112, 0xf>(v); v += lane_step<0x114, 0xf>(v); v += lane_step<0x118, 0xf>(v);      // row_shr 1, 2, 4, 8
  v += lane_step<0x142, 0xa>(v);                                          // the last lane of row 0 to row 1, of row 2 to row 3
  return v + lane_step<0x143, 0xc>(v);                                    // lane 31 to the rows 2 and 3
}
__device__ __forceinline__ u64 last_lane(u64 v) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63) | ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32);
}
__device__ __forceinline__ u64 wave_sum64(u64 v) { return last_lane(wave_scan(v)); }
// sum of the first n of 16 numbers, by every wave for itself: a row of lanes reads and adds them (a loop over all of them costs a block 1000 cycles)
__device__ __forceinline__ u64 first_sum(const u64* red, int n, int lane) {
  u64 v = (lane & 15) < n ? red[lane & 15] : 0;
  v += lane_step<0x128, 0xf>(v); v += lane_step<0x124, 0xf>(v); v += lane_step<0x122, 0xf>(v);      // row_ror 8, 4, 2, 1
  return v + lane_step<0x121, 0xf>(v);
}
__device__ u64 block_sum64(u64 v, u64* red, int tid) {
  v = wave_sum64(v);
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = v;
  __syncthreads();
  return first_sum(red, NT / 64, tid & 63);
}
// u64 sums of a loop of independent LDS reads, eight in flight
template <class F> __device__ __forceinline__ void list_loop(int n8, F f) {
#pragma unroll 1
  for (int i = 0; i < n8; i += 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f(i + j);
  }
}
// four consecutive logits in one load, whatever the row's alignment (one element at a time: 20000 instead of 8000 cycles for a row of 30113)
__device__ __forceinline__ void load4(const float* z, int i0, int V, float (&o)[4]) {
  typedef __attribute__((ext_vector_type(4), aligned(4))) float F4;
  if (i0 + 4 <= V) {
    const F4 v = *reinterpret_cast<const F4*>(z + i0);
    o[0] = v[0]; o[1] = v[1]; o[2] = v[2]; o[3] = v[3];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = i0 + i < V ? z[i0 + i] : -INFINITY;
  }
}
__device__ __forceinline__ void load4(const bf16_t* z, int i0, int V, float (&o)[4]) {
  typedef __attribute__((ext_vector_type(2), aligned(2))) uint32_t U2;
  if (i0 + 4 <= V) {
    const U2 v = *reinterpret_cast<const U2*>(z + i0);
    o[0] = __uint_as_float(v[0] << 16); o[1] = __uint_as_float(v[0] & 0xffff0000u); o[2] = __uint_as_float(v[1] << 16); o[3] = __uint_as_float(v[1] & 0xffff0000u);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = i0 + i < V ? bf2f(z[i0 + i]) : -INFINITY;
  }
}

// ROW: the row is held in LDS (zs): a thread owns 4 CPT consecutive tokens, CPT = 1, 2, 4 or 8 groups of four, group c of thread t at place c ^ t of its
// own (eight threads then read eight different banks).  Else every pass reads the row again, four consecutive tokens per thread and step.
template <typename T, bool ROW>
__global__ __launch_bounds__(NT) void sample_kernel(const SampleP p) {
  extern __shared__ __attribute__((aligned(16))) float zs[];
  __shared__ u64 s_mass[NBIN];
  __shared__ u64 s_key[CAP + 32], s_w[CAP + 32];
  __shared__ double s_tab[64];
  __shared__ u64 s_red[NT / 64], s_scan[NT / 64], s_thr, s_base;
  __shared__ float s_max[NT / 64];
  __shared__ int s_n, s_bin, s_nan;
  uint32_t* const s_cnt = reinterpret_cast<uint32_t*>(s_mass);      // the counts of top-k, before the masses of top-p
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x, V = p.V, cpt = p.cpt;
  const int nj = ROW ? cpt : (V + STEP - 1) / STEP;
  const T* z0 = (const T*)p.logits + (long)row * p.ld;
  const int step = p.pos_dev ? *p.pos_dev : 0;
  const int ban = (p.eos_id >= 0 && (p.pos_dev ? step + 1 : 0) < p.min_length) ? p.eos_id : -1;
  int edge = 0;                             // 1: the maximum is +infinity, its tokens share everything; -1: every token is -infinity, all are equal

  auto fetch = [&](int g, float (&z)[4]) {  // group g of four tokens as the caller's rules leave them; -0 becomes +0, behind the row -infinity
    load4(z0, g * 4, V, z);
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = g * 4 + i == ban ? -INFINITY : z[i] + 0.0f;
  };
  auto settle = [&](float z, int idx) { return edge > 0 ? (z == INFINITY ? 0.f : -INFINITY) : (edge < 0 && idx < V ? 0.f : z); };
  auto group = [&](int j) { return ROW ? tid * cpt + j : j * NT + tid; };
  auto own = [&](int j) { return tid * cpt + ((j ^ tid) & (cpt - 1)); };      // place(group(j))
  auto place = [&](int g) { return (g & ~(cpt - 1)) | ((g ^ (g >> p.log_cpt)) & (cpt - 1)); };
  auto get = [&](int j, float (&z)[4]) {
    if constexpr (ROW) {
      const float4 v = *reinterpret_cast<const float4*>(zs + own(j) * 4);
      z[0] = v.x; z[1] = v.y; z[2] = v.z; z[3] = v.w;
    } else {
      fetch(group(j), z);
      if (edge) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = settle(z[i], group(j) * 4 + i);
      }
    }
  };
  auto each = [&](auto f) {                 // f(index, logit) for the tokens of this thread, in index order
#pragma unroll 1
    for (int j = 0; j < nj; ++j) {
      float z[4];
      get(j, z);
      const int idx = group(j) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) f(idx + i, z[i]);
    }
  };

  int nan_at = V;
  float tmax = -INFINITY;                   // maximum of the tokens this thread has read
  if constexpr (ROW) {
    float z[ROW_MAX][4];
#pragma unroll
    for (int j = 0; j < ROW_MAX; ++j) if (j < cpt) fetch(j * NT + tid, z[j]);       // every load in flight before the first is used
    if (tid < 64) s_tab[tid] = POWERS.v[tid];
#pragma unroll
    for (int j = 0; j < ROW_MAX; ++j)
      if (j < cpt) {
        const int g = j * NT + tid;
#pragma unroll
        for (int i = 3; i >= 0; --i) {
          tmax = fmaxf(tmax, z[j][i]);
          if (z[j][i] != z[j][i]) nan_at = min(nan_at, g * 4 + i);
        }
        *reinterpret_cast<float4*>(zs + place(g) * 4) = make_float4(z[j][0], z[j][1], z[j][2], z[j][3]);
      }
  } else {
    if (tid < 64) s_tab[tid] = POWERS.v[tid];
    each([&](int idx, float z) {
      if (z != z) nan_at = min(nan_at, idx);
      tmax = fmaxf(tmax, z);
    });
  }
  float zmax = wave_max(tmax);
  if (tid == 0) { s_nan = V; s_n = 0; }
  if (lane == 0) s_max[wave] = zmax;
  s_mass[tid] = 0; s_mass[tid + NT] = 0;
  __syncthreads();
  if (nan_at < V) atomicMin(&s_nan, nan_at);
  zmax = s_max[lane & 15];
  zmax = fmaxf(zmax, __uint_as_float(lane_step<0x128, 0xf>(__float_as_uint(zmax)))); zmax = fmaxf(zmax, __uint_as_float(lane_step<0x124, 0xf>(__float_as_uint(zmax))));
  zmax = fmaxf(zmax, __uint_as_float(lane_step<0x122, 0xf>(__float_as_uint(zmax)))); zmax = fmaxf(zmax, __uint_as_float(lane_step<0x121, 0xf>(__float_as_uint(zmax))));
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
  if (!(fabsf(zmax) < INFINITY)) {
    edge = zmax > 0.f ? 1 : -1;
    tmax = settle(tmax, 0);                 // (a thread behind the row counts as one more token; the list below is gathered from the tokens)
    if constexpr (ROW) {
      for (int j = 0; j < nj; ++j) {
        float z[4];
        get(j, z);
        const int g = group(j);
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = settle(z[i], g * 4 + i);
        *reinterpret_cast<float4*>(zs + place(g) * 4) = make_float4(z[0], z[1], z[2], z[3]);
      }
    }
    zmax = 0.f;
  }
  const float uf = p.u[(p.pos_dev ? (long)max(0, min(step, p.u_steps - 1)) * p.u_ld : 0) + row];
  const double u = (double)fmaxf(uf, 0.f), dmax = (double)zmax, min_w = p.min_p * ONE;

  auto far_of = [&](float z) { return (zmax - z) * p.bin_scale; };                        // in bins; the last bin holds what has no mass
  auto bin_of = [&](float z) { return (int)fminf(far_of(z), (float)(NBIN - 1)); };
  auto weight = [&](float z) -> double { return exp2_mass(((double)z - dmax) * p.exp2_scale, s_tab); };      // 2^46 w
  auto log_prob = [&](float z, u64 total) { return (float)(((double)z - dmax) * p.inv_temp - log((double)total / ONE)); };

  // bin of the boundary: the first one at which the running sum (of counts or masses) reaches the goal, which `aim` may take from the whole sum; s_base = the
  // sum before it
  auto find_bin = [&](auto value, auto aim, auto reached) {
    const auto a = value(2 * tid), b = value(2 * tid + 1);
    const auto inc = wave_scan(a + b);
    if (lane == 63) s_scan[wave] = inc;
    if (tid == 0) { s_bin = NBIN - 1; s_n = 0; }
    __syncthreads();
    const u64 pre = inc - (a + b) + first_sum(s_scan, wave, lane);
    aim(first_sum(s_scan, NT / 64, lane));
    if (!reached(pre) && reached(pre + a)) { s_bin = 2 * tid; s_base = pre; }
    else if (!reached(pre + a) && reached(pre + a + b)) { s_bin = 2 * tid + 1; s_base = pre + a; }
    __syncthreads();
  };
  auto clear = [&]() { s_mass[tid] = 0; s_mass[tid + NT] = 0; __syncthreads(); };
  const bool cut_k = p.top_k > 0 && p.top_k < V;

  // Small top-k: the k-th largest of the 1024 threads' maxima is a lower bound of the k-th largest logit, so the tokens at or above (the bin of) it
  // contain the first k, and there are few more of them.  Everything else is decided among these candidates.
  if (cut_k && p.top_k <= SMALL_K) {
    const int b0 = bin_of(tmax);
    if (b0 < NBIN - 1) atomicAdd(&s_cnt[b0], 1u);
    __syncthreads();
    const u64 k = (u64)p.top_k;
    find_bin([&](int b) { return s_cnt[b]; }, [](u64) {}, [&](u64 s) { return s >= k; });
    const int bin = s_bin;
    if (bin < NBIN - 1) {
      const float limit = (float)(bin + 1);
#pragma unroll 2
      for (int j = 0; j < nj; ++j) {
        float z[4];
        get(j, z);
        if (far_of(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]))) < limit) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (far_of(z[i]) < limit) {
              const int at = atomicAdd(&s_n, 1);
              if (at < SMALL_N) s_key[at] = order_key(z[i], group(j) * 4 + i);
            }
        }
      }
      __syncthreads();
      const int n = s_n, pad = (n + 31) & ~31;
      if (n >= p.top_k && n <= SMALL_N) {   // the same for the whole block
        if (tid >= n && tid < pad) s_key[tid] = ~0ull;
        __syncthreads();
        // four threads per candidate, each with a quarter of the list
        const int c = tid >> 2, q = tid & 3;
        auto quarter = [&](auto f) { list_loop(pad >> 2, [&](int i) { f(i * 4 + q); }); };
        auto quad_sum = [](auto v) { v += lane_step<0xB1, 0xf>(v); return v + lane_step<0x4E, 0xf>(v); };      // quad permutes [1,0,3,2], [2,3,0,1]
        u64 key = ~0ull, w = 0;
        double wd = 0.0;
        float z = 0.f;
        bool in = false;
        if (c < n) {
          key = s_key[c];
          z = key_logit(key);
          uint32_t rank = 0;
          quarter([&](int i) { rank += s_key[i] < key ? 1u : 0u; });
          in = (int)quad_sum(rank) < p.top_k;
          if (in) { wd = weight(z); w = mass_of(wd); }
        }
        if (q == 0 && c < pad) s_w[c] = w;
        __syncthreads();
        u64 total = 0, pre = 0;
        if (c < n) quarter([&](int i) { const u64 x = s_w[i]; total += x; pre += s_key[i] < key ? x : 0; });
        total = quad_sum(total); pre = quad_sum(pre);
        __syncthreads();
        const bool keep = in && w > 0 && wd >= min_w && (p.top_p >= 1.0 || (double)pre < p.top_p * (double)total);
        if (q == 0 && c < n) s_w[c] = keep ? w : 0;
        __syncthreads();
        if (keep) {                         // the same for the four
          u64 run = 0;
          total = 0;
          quarter([&](int i) { const u64 x = s_w[i]; total += x; run += (uint32_t)s_key[i] <= (uint32_t)key ? x : 0; });
          total = quad_sum(total); run = quad_sum(run);
          const double goal = u * (double)total;
          if (q == 0 && (((double)run > goal && !((double)(run - w) > goal)) || (!((double)total > goal) && run == total)))
            finish((int)(uint32_t)key, log_prob(z, total));
        }
        return;
      }
    }
    __syncthreads();
    clear();
  }

  // The last kept token of the boundary's bin, as an order key: the first one at which the running sum of `value` over the bin's tokens in order reaches
  // the goal; `in` = tokens that take part at all.  On the way the thread's tokens that take part are told apart (ROW, a bit each): those in the bins
  // before the boundary's, and those in it.  After a cut `pass` has the thread's tokens that it left, and the next passes visit only these.
  uint32_t sure = 0, maybe = 0, pass = 0;
  bool told = false, few = false;           // pass describes the cut; it left so few tokens that visiting them one by one is faster than all in order
  auto logit = [&](int b) { return zs[own(b >> 2) * 4 + (b & 3)]; };
  auto visit = [&](uint32_t m, auto f) {    // f(bit, index, logit)
    for (; m; m &= m - 1) { const int b = __builtin_ctz(m); f(b, tid * cpt * 4 + b, logit(b)); }
  };
  auto resolve = [&](auto in, auto value, auto reached) -> u64 {
    const u64 base = s_base;
    const float lo = (float)s_bin, hi = (float)(s_bin + 1);
    sure = maybe = 0;
    auto put = [&](int idx, float z) {
      const int at = atomicAdd(&s_n, 1);
      if (at < CAP) s_key[at] = order_key(z, idx);
    };
    if (ROW && few) {
      visit(pass, [&](int b, int idx, float z) {
        const float far = far_of(z);
        if (far < lo) sure |= 1u << b;
        else if (far < hi) { maybe |= 1u << b; put(idx, z); }
      });
    } else {
#pragma unroll 1
      for (int j = 0; j < nj; ++j) {
        float z[4];
        get(j, z);
        uint32_t before = 0, here = 0;      // without branches for the many, the few of the boundary's bin one by one
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float far = far_of(z[i]);
          before |= far < lo ? 1u << i : 0u;
          here |= far >= lo && far < hi ? 1u << i : 0u;
        }
        for (uint32_t m = here; m; m &= m - 1) {
          const int i = __builtin_ctz(m);
          const float zi = i == 0 ? z[0] : i == 1 ? z[1] : i == 2 ? z[2] : z[3];
          if (in(zi, group(j) * 4 + i)) put(group(j) * 4 + i, zi); else here &= ~(1u << i);
        }
        if constexpr (ROW) { sure |= before << (j * 4); maybe |= here << (j * 4); }
      }
    }
    __syncthreads();
    const int n = s_n, n8 = (n + 7) & ~7;
    if (n <= CAP) {
      u64 key = ~0ull, w = 0;
      if (tid < n) { key = s_key[tid]; w = value(key_logit(key)); }
      else if (tid < n8) s_key[tid] = key;
      if (tid < n8) s_w[tid] = w;
      __syncthreads();
      if (tid < n) {
        u64 pre = base;
        list_loop(n8, [&](int i) { pre += s_key[i] < key ? s_w[i] : 0; });
        if (!reached(pre) && reached(pre + w)) s_thr = key;
      }
      __syncthreads();
      return s_thr;
    }
    // more than CAP tokens within one bin (equal logits, a row whose logits lie within a few bins, or over 100000 tokens of any ordinary row): bisection on the order
    // key, 64 passes over the row at most.  64 rows, top-p 0.9: 32228 logits spread by 0.001 600 us (by 2.5: 24), 131072 unit-normal ones 1.34 ms (spread by 2.5: 0.12)
    u64 first = 0, last = ~0ull;            // sum(keys <= last) reaches the goal
    while (first < last) {
      const u64 mid = first + ((last - first) >> 1);
      u64 s = 0;
      each([&](int idx, float z) {
        const float far = far_of(z);
        if (far >= lo && far < hi && in(z, idx) && order_key(z, idx) <= mid) s += value(z);
      });
      s = block_sum64(s, s_red, tid);
      if (reached(base + s)) last = mid; else first = mid + 1;
    }
    return first;
  };

  // the last token that top-k and top-p keep, and whether a token is not behind it
  float thr_z = -INFINITY;
  int thr_i = V;
  auto upto = [&](float z, int idx) { return z > thr_z || (z == thr_z && idx <= thr_i); };
  auto set_thr = [&](u64 key) {
    thr_z = key_logit(key); thr_i = (int)(uint32_t)key;
    if constexpr (ROW) {
      pass = sure;
      visit(maybe, [&](int b, int idx, float z) { pass |= upto(z, idx) ? 1u << b : 0u; });
      told = true;
    }
  };
  if (cut_k) {
    each([&](int, float z) { const int b = bin_of(z); if (b < NBIN - 1) atomicAdd(&s_cnt[b], 1u); });
    __syncthreads();
    const u64 k = (u64)p.top_k;
    find_bin([&](int b) { return s_cnt[b]; }, [](u64) {}, [&](u64 s) { return s >= k; });
    if (s_bin < NBIN - 1) {                 // otherwise every token with any mass is among the first k
      set_thr(resolve([](float, int) { return true; }, [](float) { return (u64)1; }, [&](u64 s) { return s >= k; }));
      few = told && p.top_k < V / 4;
    }
    __syncthreads();
    clear();
  }
  if (p.top_p < 1.0) {
    auto add = [&](float z) {
      const float far = far_of(z);
      if (far < (float)(NBIN - 1)) atomicAdd(&s_mass[(int)far], mass_of(weight(z)));
    };
    if (ROW && few) visit(pass, [&](int, int, float z) { add(z); });
    else if (cut_k) each([&](int idx, float z) { if (upto(z, idx)) add(z); });
    else each([&](int, float z) { add(z); });
    __syncthreads();
    double goal = 0.0;
    const auto reached = [&](u64 s) { return (double)s >= goal; };
    find_bin([&](int b) { return s_mass[b]; }, [&](u64 total) { goal = p.top_p * (double)total; }, reached);
    if (cut_k) set_thr(resolve(upto, [&](float z) { return mass_of(weight(z)); }, reached));
    else set_thr(resolve([](float, int) { return true; }, [&](float z) { return mass_of(weight(z)); }, reached));
    __syncthreads();
  }

  // a token that carries mass at all and is not behind the threshold
  auto kept = [&](float z, int idx) { return far_of(z) < (float)(NBIN - 1) && upto(z, idx); };
  auto mass_kept = [&](float z) -> u64 { const double w = weight(z); return w >= min_w ? mass_of(w) : 0; };
  // of the masses m[] of eight consecutive tokens or segments of this lane with `pre` before them: the first one at which the running mass passes the
  // goal, else (u = 1) the last one with any mass; one lane of the wave gets it
  auto pick8 = [&](const u64 (&m)[8], u64 pre, double goal, int& at, u64& before) -> bool {
    int found = -1, last = -1;
    u64 run = pre, fpre = 0, lpre = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (m[i] > 0) { last = i; lpre = run; }
      if (found < 0 && m[i] > 0 && (double)(run + m[i]) > goal) { found = i; fpre = run; }
      run += m[i];
    }
    const u64 any = __ballot(found >= 0), have = __ballot(last >= 0);
    at = any ? found : last;
    before = any ? fpre : lpre;
    return lane == (any ? __builtin_ctzll(any) : 63 - __builtin_clzll(have));
  };
  if constexpr (ROW) {
    // mass of each thread's consecutive tokens: only the kept ones are weighed, two at a time (a weight is one long chain)
    if (!told) {
#pragma unroll 1
      for (int j = 0; j < nj; ++j) {
        float z[4];
        get(j, z);
#pragma unroll
        for (int i = 0; i < 4; ++i) pass |= far_of(z[i]) < (float)(NBIN - 1) ? 1u << (j * 4 + i) : 0u;
      }
    }
    u64 own = 0;
    for (uint32_t m = pass; m;) {
      const int b0 = __builtin_ctz(m);
      m &= m - 1;
      const int b1 = m ? __builtin_ctz(m) : b0;
      const u64 x0 = mass_kept(logit(b0)), x1 = mass_kept(logit(b1));
      own += x0 + (m ? x1 : 0);
      m &= m - 1;
    }
    const u64 inc = wave_scan(own);
    __syncthreads();
    if (lane == 63) s_red[wave] = inc;
    __syncthreads();
    const u64 pre = inc - own + first_sum(s_red, wave, lane), total = first_sum(s_red, NT / 64, lane);
    const double goal = u * (double)total;
    const bool here = own > 0 && ((double)(pre + own) > goal ? !((double)pre > goal) : pre + own == total && !((double)total > goal));
    const u64 owner = __ballot(here);       // one thread of the block: its wave looks at that thread's tokens, a lane each
    if (owner) {
      const int src = __builtin_ctzll(owner), t = wave * 64 + src;
      const uint32_t m = (uint32_t)__builtin_amdgcn_readlane((int)pass, src);
      const u64 before = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)pre, src) | ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(pre >> 32), src) << 32);
      float z = 0.f;
      u64 x = 0;
      if (lane < 32 && (m >> lane & 1)) {
        z = zs[place(t * cpt + (lane >> 2)) * 4 + (lane & 3)];
        x = mass_kept(z);
      }
      const u64 run = before + wave_scan(x), past = __ballot(x > 0 && (double)run > goal), any = __ballot(x > 0);
      if (lane == (past ? __builtin_ctzll(past) : 63 - __builtin_clzll(any))) finish(t * cpt * 4 + lane, log_prob(z, total));
    }
  } else {
    // mass of each segment of 256 consecutive tokens (one wave of one step), segments in index order: [nj][16] <= 512; then within the drawn one
    __syncthreads();
    u64* const seg = s_mass;
    auto masses = [&](int j, float (&z)[4], u64 (&m)[8]) {
      get(j, z);
#pragma unroll
      for (int i = 0; i < 8; ++i) m[i] = i < 4 && kept(z[i & 3], group(j) * 4 + i) ? mass_kept(z[i & 3]) : 0;
    };
#pragma unroll 1
    for (int j = 0; j < nj; ++j) {
      float z[4];
      u64 m[8];
      masses(j, z, m);
      const u64 own = wave_sum64(m[0] + m[1] + m[2] + m[3]);
      if (lane == 0) seg[j * (NT / 64) + wave] = own;
    }
    __syncthreads();
    int at;
    u64 before;
    if (wave == 0) {
      u64 m[8], own = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) { m[i] = lane * 8 + i < nj * (NT / 64) ? seg[lane * 8 + i] : 0; own += m[i]; }
      const u64 inc = wave_scan(own), total = last_lane(inc);
      if (pick8(m, inc - own, u * (double)total, at, before)) { s_bin = lane * 8 + at; s_base = before; s_thr = total; }
    }
    __syncthreads();
    const int sj = s_bin / (NT / 64);
    if (wave == s_bin % (NT / 64)) {
      const u64 total = s_thr;
      float z[4];
      u64 m[8];
      masses(sj, z, m);
      const u64 own = m[0] + m[1] + m[2] + m[3];
      if (pick8(m, s_base + wave_scan(own) - own, u * (double)total, at, before))
        finish(group(sj) * 4 + at, log_prob(at == 0 ? z[0] : (at == 1 ? z[1] : (at == 2 ? z[2] : z[3])), total));
    }
  }
}

template <typename T> int sample_launch(SampleP& p, int rows, hipStream_t s) {
  const int nj = (p.V + STEP - 1) / STEP;
  p.log_cpt = nj <= 1 ? 0 : (nj <= 2 ? 1 : (nj <= 4 ? 2 : 3)); p.cpt = 1 << p.log_cpt;
  if (nj <= ROW_MAX) {
    static bool attr = false;
    if (!attr) { (void)hipFuncSetAttribute((const void*)sample_kernel<T, true>, hipFuncAttributeMaxDynamicSharedMemorySize, ROW_MAX * STEP * 4); attr = true; }
    hipLaunchKernelGGL((sample_kernel<T, true>), dim3(rows), dim3(NT), (size_t)p.cpt * STEP * 4, s, p);
  } else {
    hipLaunchKernelGGL((sample_kernel<T, false>), dim3(rows), dim3(NT), 0, s, p);
  }
  V2S_LAUNCH_CHECK();
  return V2S_OK;
}

}  // namespace

extern "C" int v2s_sample_step(const void* logits, int32_t logits_dtype, int64_t ld, int32_t rows, int32_t V, double temperature, int32_t top_k, double top_p,
                               double min_p, const float* u, int64_t u_ld, int32_t u_steps, int64_t* next_tok, float* logp, int32_t* unfinished, int32_t eos_id,
                               int32_t pad_id, int64_t* seq_out, int64_t seq_ld, const int32_t* pos_dev, int32_t min_length, void* stream) {
  V2S_CHECK(logits && u && next_tok, V2S_ERR_ARG, "v2s_sample_step: NULL pointer");
  V2S_CHECK(logits_dtype == V2S_F32 || logits_dtype == V2S_BF16, V2S_ERR_DTYPE, "v2s_sample_step: logits must be fp32 or bf16");
  V2S_CHECK(rows > 0 && rows < 1 << 22 && V > 0 && V <= 131072 && ld >= V, V2S_ERR_SHAPE, "v2s_sample_step: unsupported shape rows=%d V=%d ld=%lld (rows below 2^22, V <= 131072, ld >= V)", rows, V, (long long)ld);
  V2S_CHECK(temperature >= 1e-6 && temperature <= 1e6, V2S_ERR_ARG, "v2s_sample_step: temperature must be in [1e-6, 1e6]");
  V2S_CHECK(top_k >= 0 && top_p > 0.0 && top_p <= 1.0 && min_p >= 0.0 && min_p <= 1.0, V2S_ERR_ARG, "v2s_sample_step: top_k >= 0, top_p in (0, 1], min_p in [0, 1]");
  V2S_CHECK(!seq_out || pos_dev, V2S_ERR_ARG, "v2s_sample_step: seq_out needs pos_dev");
  V2S_CHECK(!pos_dev || (u_ld >= rows && u_steps > 0), V2S_ERR_SHAPE, "v2s_sample_step: with pos_dev, u is a table of u_steps > 0 rows of u_ld >= rows numbers");
  SampleP p;
  p.logits = logits; p.ld = ld; p.V = V; p.inv_temp = 1.0 / temperature; p.exp2_scale = 1.44269504088896340736 / temperature; p.bin_scale = (float)((NBIN - 1) / (BIN_RANGE * temperature));
  p.top_k = top_k; p.top_p = top_p; p.min_p = min_p; p.u = u; p.u_ld = u_ld; p.u_steps = u_steps; p.next_tok = (long*)next_tok; p.logp = logp; p.unfinished = unfinished;
  p.eos_id = eos_id; p.pad_id = pad_id; p.seq_out = (long*)seq_out; p.seq_ld = seq_ld; p.pos_dev = pos_dev; p.min_length = min_length;
  return logits_dtype == V2S_F32 ? sample_launch<float>(p, rows, (hipStream_t)stream) : sample_launch<bf16_t>(p, rows, (hipStream_t)stream);
}
