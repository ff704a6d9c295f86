// Sampling items from score rows: temperature, top-k, top-p, min-p, draws without replacement from given uniforms.  C ABI and the
// definition: include/recpack_hip.h, rphip_sample.
//
// Candidates are ranked by (score descending, index ascending); everything below works on that order.  The kept set is a prefix of it,
// a draw inverts the cumulative mass along it.  Whole numbers come out, so sums next to a border decide: masses are float64 (short
// lists) or 64-bit fixed point (whole rows, where the order of the adds must not matter), never float32.
#include "rp_ops.h"

#include <algorithm>

namespace {

constexpr int RPS_SHORT = 1024;      // longest prefix the list form ranks completely
constexpr int SL_CAP = 4096;         // candidates collected in LDS
constexpr int SL_THREADS = 1024;
constexpr int SB_BINS = 4096;        // mass bins of the whole-row form: 64 per e-fold, the last one takes what lies below e^-64
constexpr float SB_PER_E = 64.0f;

struct sample_args {
  int64_t rows, ld, ld_ids, ld_u;
  int width, draws;
  const void* scores;
  const int32_t* lengths;
  const int32_t* ids;
  const float* u;
  float temperature, top_p, min_p;
  int32_t top_k;
  const float* temperature_dev;
  const float* top_p_dev;
  const float* min_p_dev;
  const int32_t* top_k_dev;
  int32_t* idx;
  float* prob;
  int32_t* nnz;
  int64_t row0;
};

// a row's settings; scalars where no array is given.  Values out of range (arrays are not checked on the host) are moved into it.
struct row_set {
  float temperature, top_p, min_p;
  int k, len;
};
__device__ __forceinline__ row_set rs_load(const sample_args& a, int64_t r) {
  row_set s;
  s.temperature = a.temperature_dev ? a.temperature_dev[r] : a.temperature;
  s.top_p = a.top_p_dev ? a.top_p_dev[r] : a.top_p;
  s.min_p = a.min_p_dev ? a.min_p_dev[r] : a.min_p;
  if (!(s.temperature > 0.0f)) s.temperature = 0.0f;
  if (!(s.top_p < 1.0f)) s.top_p = 1.0f;
  if (s.top_p < 0.0f) s.top_p = 0.0f;
  if (!(s.min_p > 0.0f)) s.min_p = 0.0f;
  if (s.min_p > 1.0f) s.min_p = 1.0f;
  s.len = a.lengths ? min(max(a.lengths[r], 0), a.width) : a.width;
  const int bound = a.top_k > 0 ? a.top_k : a.width;
  const int k = a.top_k_dev ? a.top_k_dev[r] : a.top_k;
  s.k = k > 0 ? min(k, bound) : bound;
  return s;
}

// scores as 32-bit keys in the order of the scores (-0 = +0); 0: no candidate (NaN, -inf)
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if ((b & 0x7fffffffu) > 0x7f800000u || b == 0xff800000u) return 0u;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// log of a mass relative to the best score; equal scores give 0 (+inf among them)
__device__ __forceinline__ double z_of(float x, float best, double inv_t_num) { return x == best ? 0.0 : ((double)x - (double)best) / inv_t_num; }

__device__ __forceinline__ double shfl_up_f64(double v, int d) { return __hiloint2double(__shfl_up(__double2hiint(v), d), __shfl_up(__double2loint(v), d)); }
__device__ __forceinline__ double shfl_f64(double v, int src) { return __hiloint2double(__shfl(__double2hiint(v), src), __shfl(__double2loint(v), src)); }
__device__ __forceinline__ unsigned long long shfl_xor_u64(unsigned long long v, int m) {
  const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, m), hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), m);
  return ((unsigned long long)hi << 32) | lo;
}
__device__ __forceinline__ double wave_scan_f64(double v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double t = shfl_up_f64(v, d);
    if (lane >= d) v += t;
  }
  return v;
}

// bitonic sort of 64 * PER entries, descending; entry lane * PER + i: steps shorter than PER stay in the lane's registers
template <int PER>
__device__ __forceinline__ void wave_sort(unsigned long long (&e)[PER], int lane) {
#pragma unroll 1
  for (int size = 2; size <= 64 * PER; size <<= 1) {
#pragma unroll 1
    for (int step = size >> 1; step >= PER; step >>= 1) {
      const int ls = step / PER;
      const bool low = (lane & ls) == 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const unsigned long long o = shfl_xor_u64(e[i], ls);
        const bool desc = ((lane * PER + i) & size) == 0;
        e[i] = (low == desc) == (e[i] > o) ? e[i] : o;
      }
    }
#pragma unroll
    for (int step = PER >> 1; step > 0; step >>= 1) {
      if (step >= size) continue;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (i & step) continue;
        const bool desc = ((lane * PER + i) & size) == 0;
        const unsigned long long x = e[i], y = e[i + step];
        const bool swap = desc ? x < y : x > y;
        e[i] = swap ? y : x;
        e[i + step] = swap ? x : y;
      }
    }
  }
}

// One wave finishes a row from its leading candidates, ranked: entry lane * PER + i = key << 32 | ~index (0: none), all of the first
// s.k ranks present.  Masses are float64 relative to the best candidate; when everything that carries mass has been drawn the rest is
// taken relative to the best one left (a low temperature underflows: the definition does not).
template <int PER>
__device__ void finish_row(const sample_args& a, int64_t r, const row_set& s, const unsigned long long (&e)[PER], int lane) {
  int have = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) have += e[i] != 0 && lane * PER + i < s.k ? 1 : 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) have += __shfl_xor(have, d);
  const float best = score_of((uint32_t)__shfl((int)(uint32_t)(e[0] >> 32), 0));
  const double t = (double)s.temperature;
  double m[PER];
  int kept = have;
  if (s.temperature > 0.0f) {
    double own = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      m[i] = lane * PER + i < have ? exp(z_of(score_of((uint32_t)(e[i] >> 32)), best, t)) : 0.0;
      own += m[i];
    }
    const double incl = wave_scan_f64(own, lane);
    const double total = shfl_f64(incl, 63);
    double c = incl - own;
    const double border = (double)s.top_p * total;
    int n = 0;  // leading ranks kept: those with less than top_p of the mass before them and at least min_p of the best one's mass
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int rank = lane * PER + i;
      if (rank < have && (s.top_p >= 1.0f || rank == 0 || c < border) && m[i] >= (double)s.min_p) ++n;
      c += m[i];
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    kept = n;
  }
  const int n_out = min(a.draws, kept);
  uint32_t gone = 0;  // bit i: rank lane * PER + i has been drawn
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (lane * PER + i >= kept) gone |= 1u << i;
  float from = best;  // what the masses are relative to
  for (int d = 0; d < n_out; ++d) {
    int rank;
    double p = 1.0;
    if (s.temperature > 0.0f) {
      double own = 0.0, incl, total;
      for (;;) {
        own = 0.0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (!((gone >> i) & 1)) own += m[i];
        incl = wave_scan_f64(own, lane);
        total = shfl_f64(incl, 63);
        if (total >= 1e-200) break;
        // the best rank left becomes the reference (it gets mass 1)
        float top = -INFINITY;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i)
          if (!((gone >> i) & 1)) top = score_of((uint32_t)(e[i] >> 32));
        const unsigned long long who = __ballot(gone != (PER == 32 ? 0xffffffffu : (1u << PER) - 1u));
        from = __uint_as_float((uint32_t)__shfl((int)__float_as_uint(top), (int)__ffsll((long long)who) - 1));
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (!((gone >> i) & 1)) m[i] = exp(z_of(score_of((uint32_t)(e[i] >> 32)), from, t));
      }
      float uu = a.u[r * a.ld_u + d];
      uu = uu > 0.0f ? fminf(uu, 0x1.fffffep-1f) : 0.0f;
      const double want = (double)uu * total;
      // the lane whose ranks pass the border; the last one with mass left if rounding lets none pass
      unsigned long long cand = __ballot(incl > want && own > 0.0);
      if (!cand) cand = 1ull << (63 - __clzll((long long)__ballot(own > 0.0)));
      const int who = (int)__ffsll((long long)cand) - 1;
      double c = incl - own, got = 0.0;
      int at = 0;
      bool passed = false;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if ((gone >> i) & 1) continue;
        c += m[i];
        if (!passed && m[i] > 0.0) at = i, got = m[i], passed = c > want;
      }
      rank = __shfl(lane * PER + at, who);
      p = shfl_f64(got, who) / total;
    } else {
      rank = d;
    }
    if (rank / PER == lane) {
      const int i = rank % PER;
      gone |= 1u << i;
      unsigned long long v = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) v = j == i ? e[j] : v;
      const int32_t at = (int32_t)~(uint32_t)v;
      a.idx[r * a.draws + d] = a.ids ? a.ids[r * a.ld_ids + at] : at;
      a.prob[r * a.draws + d] = (float)p;
    }
  }
  for (int d = n_out + lane; d < a.draws; d += 64) {
    a.idx[r * a.draws + d] = -1;
    a.prob[r * a.draws + d] = 0.0f;
  }
  if (lane == 0 && a.nnz) a.nnz[r] = n_out;
}

// ---- rows that one wave holds ------------------------------------------------------------------------------------------------------
// One wave per row: up to 64 * PER scores in registers, sorted there.
template <class T, int PER>
__global__ __launch_bounds__(256) void k_sample_wave(sample_args a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = a.row0 + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= a.rows) return;
  const row_set s = rs_load(a, r);
  const T* p = (const T*)a.scores + r * a.ld;
  unsigned long long e[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {  // (any order will do: neighbouring lanes read neighbours)
    const int j = i * 64 + lane;
    const uint32_t k = j < s.len ? key_of(rp_to_f32(p[j])) : 0u;
    e[i] = k ? ((unsigned long long)k << 32) | (uint32_t)~j : 0ull;
  }
  wave_sort<PER>(e, lane);
  finish_row<PER>(a, r, s, e, lane);
}

// ---- block helpers -------------------------------------------------------------------------------------------------------------------
template <int THREADS>
__device__ __forceinline__ uint32_t block_max_u32(uint32_t v, uint32_t* red) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) v = max(v, red[w]);
  return v;
}
template <int THREADS>
__device__ __forceinline__ unsigned long long block_sum_u64(unsigned long long v, unsigned long long* red) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += shfl_xor_u64(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) v += red[w];
  return v;
}

// bitonic sort of n (a power of two <= SL_CAP) entries in LDS, descending
__device__ void block_sort(unsigned long long* e, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      __syncthreads();
      for (int q = threadIdx.x; q < n / 2; q += SL_THREADS) {
        const int i = (q / step) * 2 * step + q % step, j = i + step;
        const unsigned long long x = e[i], y = e[j];
        const bool desc = (i & size) == 0;
        if (desc ? x < y : x > y) e[i] = y, e[j] = x;
      }
    }
  __syncthreads();
}

// The exact form of "the n-th of the row in rank order" for any row (thousands of equal scores, adversarial orders): radix descent over
// the keys by count, then ties by index.  Returns the key of rank n - 1 (n >= 1, at most the number of candidates) and, in *equal, how
// many candidates with exactly that key belong to the first n.
struct sel_shared {
  uint32_t hist[256];
  uint32_t digit, before;
};
template <class T>
__device__ uint32_t select_key(const T* p, int len, int n, sel_shared& sh, int* equal) {
  uint32_t prefix = 0, left = (uint32_t)n;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += SL_THREADS) sh.hist[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < len; j += SL_THREADS) {
      const uint32_t k = key_of(rp_to_f32(p[j]));
      if (k && (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))) atomicAdd(&sh.hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t c = 0;
      int d = 255;
      for (; d > 0; --d) {
        if (c + sh.hist[d] >= left) break;
        c += sh.hist[d];
      }
      sh.digit = d;
      sh.before = c;
    }
    __syncthreads();
    prefix |= sh.digit << shift;
    left -= sh.before;
  }
  *equal = (int)left;
  return prefix;
}

// ---- whole rows, a short prefix ------------------------------------------------------------------------------------------------------
// k <= 1024: one workgroup per row finds a score that at least k candidates reach, collects those candidates, ranks them.
// The threshold: every thread takes the best of two groups of the row's scores; if k of those 2048 group maxima reach a value, k
// candidates do.  For rows in no particular order few more than k candidates reach the k-th largest group maximum (1.1 k at k = 200,
// 1.4 k at 1000).  Rows that break this - thousands of equal scores - take the radix descent.
template <class T>
__global__ __launch_bounds__(SL_THREADS) void k_sample_topk(sample_args a) {
  __shared__ unsigned long long list[SL_CAP];
  __shared__ uint32_t red[SL_THREADS / 64];
  __shared__ uint32_t n_list, cnt;
  __shared__ sel_shared sel;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = a.row0 + blockIdx.x;
  const row_set s = rs_load(a, r);
  const T* p = (const T*)a.scores + r * a.ld;
  uint32_t g0 = 0, g1 = 0;
  {
    int j = threadIdx.x;
    for (; j + SL_THREADS < s.len; j += 2 * SL_THREADS) {
      g0 = max(g0, key_of(rp_to_f32(p[j])));
      g1 = max(g1, key_of(rp_to_f32(p[j + SL_THREADS])));
    }
    if (j < s.len) g0 = max(g0, key_of(rp_to_f32(p[j])));
  }
  // the largest prefix of key bits that at least k group maxima reach; 1 (every candidate) if fewer than k groups have one
  uint32_t floor_key = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = floor_key | (1u << bit);
    __syncthreads();
    if (threadIdx.x == 0) cnt = 0;
    __syncthreads();
    const uint32_t c = (uint32_t)__popcll(__ballot(g0 >= t)) + (uint32_t)__popcll(__ballot(g1 >= t));
    if (lane == 0 && c) atomicAdd(&cnt, c);
    __syncthreads();
    const uint32_t n = cnt;
    if (n >= (uint32_t)s.k) {
      floor_key = t;
      if (n <= (uint32_t)s.k + (uint32_t)s.k / 4) break;
    }
  }
  if (floor_key == 0) floor_key = 1;
  __syncthreads();
  if (threadIdx.x == 0) n_list = 0;
  __syncthreads();
  for (int j0 = wave * 64; j0 < s.len; j0 += SL_THREADS) {
    const int j = j0 + lane;
    const uint32_t k = j < s.len ? key_of(rp_to_f32(p[j])) : 0u;
    const unsigned long long hit = __ballot(k >= floor_key);
    if (hit == 0) continue;
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(&n_list, (uint32_t)__popcll(hit));
    at = (uint32_t)__shfl((int)at, 0) + (uint32_t)__popcll(hit & ((1ull << lane) - 1ull));
    if (k >= floor_key && at < SL_CAP) list[at] = ((unsigned long long)k << 32) | (uint32_t)~j;
  }
  __syncthreads();
  int n = (int)n_list;
  if (n > SL_CAP) {  // (so the row has more than k candidates)
    int equal = 0;
    const uint32_t kk = select_key<T>(p, s.len, s.k, sel, &equal);
    __syncthreads();
    if (threadIdx.x == 0) n_list = 0, cnt = 0;
    __syncthreads();
    for (int j0 = 0; j0 < s.len; j0 += SL_THREADS) {  // in index order: the first `equal` ties are taken
      const int j = j0 + threadIdx.x;
      const uint32_t k = j < s.len ? key_of(rp_to_f32(p[j])) : 0u;
      const unsigned long long tie = __ballot(k == kk);
      __syncthreads();
      if (lane == 0) red[wave] = (uint32_t)__popcll(tie);
      __syncthreads();
      uint32_t before = cnt, all = 0;
      for (int w = 0; w < SL_THREADS / 64; ++w) {
        before += w < wave ? red[w] : 0u;
        all += red[w];
      }
      const bool take = k > kk || (k == kk && before + (uint32_t)__popcll(tie & ((1ull << lane) - 1ull)) < (uint32_t)equal);
      if (take) list[atomicAdd(&n_list, 1u)] = ((unsigned long long)k << 32) | (uint32_t)~j;  // (s.k <= 1024 entries in all)
      __syncthreads();
      if (threadIdx.x == 0) cnt += all;
    }
    __syncthreads();
    n = (int)n_list;
  }
  if (n > RPS_SHORT) {
    int n2 = 2 * RPS_SHORT;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += SL_THREADS) list[i] = 0;
    block_sort(list, n2);
    n = RPS_SHORT;  // (s.k of them count)
  }
  if (wave != 0) return;
  if (n <= 256) {
    unsigned long long e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = lane * 4 + i < n ? list[lane * 4 + i] : 0ull;
    wave_sort<4>(e, lane);
    finish_row<4>(a, r, s, e, lane);
  } else {
    unsigned long long e[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) e[i] = lane * 16 + i < n ? list[lane * 16 + i] : 0ull;
    wave_sort<16>(e, lane);
    finish_row<16>(a, r, s, e, lane);
  }
}

// ---- whole rows, any prefix, one draw ------------------------------------------------------------------------------------------------
// 2^(z log2 e) for z <= 0 in fixed point: Taylor to the 11th power on [-1/2, 1/2] (remainder < 2^-47 relative), 0 below 2^-shift.
__device__ __forceinline__ double exp_le0(double z) {
  const double t = fmax(z * 1.4426950408889634074, -1000.0);
  const double n = rint(t), f = (t - n) * 0.69314718055994530942;
  double q = 1.0 / 39916800.0;
  q = fma(q, f, 1.0 / 3628800.0);
  q = fma(q, f, 1.0 / 362880.0);
  q = fma(q, f, 1.0 / 40320.0);
  q = fma(q, f, 1.0 / 5040.0);
  q = fma(q, f, 1.0 / 720.0);
  q = fma(q, f, 1.0 / 120.0);
  q = fma(q, f, 1.0 / 24.0);
  q = fma(q, f, 1.0 / 6.0);
  q = fma(q, f, 0.5);
  q = fma(q, f, 1.0);
  q = fma(q, f, 1.0);
  return ldexp(q, (int)n);
}

struct row_mass {
  float best;
  double t;      // temperature
  double scale;  // 2^shift
  bool greedy;
  __device__ __forceinline__ double z(float x) const { return x == best ? 0.0 : greedy ? -1000.0 : ((double)x - (double)best) / t; }
  __device__ __forceinline__ int bin(double z) const { return (int)fmin(-z * (double)SB_PER_E, (double)(SB_BINS - 1)); }
  __device__ __forceinline__ unsigned long long mass(double z) const { return z <= -690.0 ? 0ull : (unsigned long long)rint(exp_le0(z) * scale); }
};

struct seek_shared {
  unsigned long long list[SL_CAP];
  unsigned long long red64[SL_THREADS / 64];
  unsigned long long before64, mass64;
  uint32_t red32[SL_THREADS / 64];
  uint32_t n_list, before32, bin, digit, found;
  unsigned long long hist_m[256];
  uint32_t hist_c[256];
};

// First candidate in rank order with (by_count: rank + 1 >= target; otherwise: cumulative mass up to and with it >= target).  hist_m /
// hist_c: the row's masses and counts per bin.  Returns its index (-1: none) and, in *incl / *own, the cumulative mass with it and its own.
template <class T>
__device__ int seek(const T* p, int len, const row_mass& rm, const unsigned long long* hist_m, const uint32_t* hist_c, bool by_count, unsigned long long target,
                    seek_shared& sh, unsigned long long* incl, unsigned long long* own) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the bin: thread t owns the bins [4 t, 4 t + 4)
  constexpr int PB = SB_BINS / SL_THREADS;
  unsigned long long c[PB], m[PB], sc = 0, sm = 0;
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    m[i] = hist_m[threadIdx.x * PB + i];
    c[i] = hist_c ? hist_c[threadIdx.x * PB + i] : 0u;
    sc += c[i];
    sm += m[i];
  }
  unsigned long long ic = sc, im = sm;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t a0 = __shfl_up((uint32_t)ic, d), a1 = __shfl_up((uint32_t)(ic >> 32), d), b0 = __shfl_up((uint32_t)im, d), b1 = __shfl_up((uint32_t)(im >> 32), d);
    if (lane >= d) {
      ic += ((unsigned long long)a1 << 32) | a0;
      im += ((unsigned long long)b1 << 32) | b0;
    }
  }
  __syncthreads();
  if (lane == 63) sh.red64[wave] = by_count ? ic : im;
  if (threadIdx.x == 0) sh.bin = SB_BINS, sh.n_list = 0, sh.found = 0xffffffffu;
  __syncthreads();
  unsigned long long run = (by_count ? ic - sc : im - sm);
  for (int w = 0; w < wave; ++w) run += sh.red64[w];
  // masses before the bin are wanted for both kinds of target
  unsigned long long run_m = im - sm;
  __syncthreads();
  if (lane == 63) sh.red64[wave] = im;
  __syncthreads();
  for (int w = 0; w < wave; ++w) run_m += sh.red64[w];
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const unsigned long long step = by_count ? c[i] : m[i];
    if (run < target && run + step >= target) {
      sh.bin = threadIdx.x * PB + i;
      sh.before32 = (uint32_t)(by_count ? run : 0);
      sh.before64 = run_m;
    }
    run += step;
    run_m += m[i];
  }
  __syncthreads();
  const int b = (int)sh.bin;
  if (b >= SB_BINS) return -1;
  unsigned long long mass_before = sh.before64;
  unsigned long long count_before = sh.before32;
  // collect the bin
  for (int j0 = wave * 64; j0 < len; j0 += SL_THREADS) {
    const int j = j0 + lane;
    const float x = j < len ? rp_to_f32(p[j]) : 0.0f;
    const uint32_t k = j < len ? key_of(x) : 0u;
    const bool in = k != 0 && rm.bin(rm.z(score_of(k))) == b;
    const unsigned long long hit = __ballot(in);
    if (hit == 0) continue;
    uint32_t at = 0;
    if (lane == 0) at = atomicAdd(&sh.n_list, (uint32_t)__popcll(hit));
    at = (uint32_t)__shfl((int)at, 0) + (uint32_t)__popcll(hit & ((1ull << lane) - 1ull));
    if (in && at < SL_CAP) sh.list[at] = ((unsigned long long)k << 32) | (uint32_t)~j;
  }
  __syncthreads();
  const int n = (int)sh.n_list;
  if (n <= SL_CAP) {
    int n2 = 64;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += SL_THREADS) sh.list[i] = 0;
    block_sort(sh.list, n2);
    // cumulative sums along the sorted list: 1024 entries at a time
    for (int i0 = 0; i0 < n; i0 += SL_THREADS) {
      const int i = i0 + threadIdx.x;
      const unsigned long long mine = i < n ? rm.mass(rm.z(score_of((uint32_t)(sh.list[i] >> 32)))) : 0ull;
      unsigned long long s = mine;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t b0 = __shfl_up((uint32_t)s, d), b1 = __shfl_up((uint32_t)(s >> 32), d);
        if (lane >= d) s += ((unsigned long long)b1 << 32) | b0;
      }
      __syncthreads();
      if (lane == 63) sh.red64[wave] = s;
      __syncthreads();
      unsigned long long off = mass_before, all = 0;
      for (int w = 0; w < SL_THREADS / 64; ++w) {
        off += w < wave ? sh.red64[w] : 0ull;
        all += sh.red64[w];
      }
      const unsigned long long cum = off + s;
      const bool hit = i < n && (by_count ? count_before + i + 1 == target : cum >= target && cum - mine < target);
      if (hit) {
        sh.found = (uint32_t)i;
        sh.before64 = cum;
        sh.mass64 = mine;
      }
      __syncthreads();
      if (sh.found != 0xffffffffu) break;
      mass_before += all;
    }
    const uint32_t f = sh.found;
    const unsigned long long got = f == 0xffffffffu ? 0ull : sh.list[f];
    *incl = sh.before64;
    *own = sh.mass64;
    __syncthreads();
    return f == 0xffffffffu ? -1 : (int)~(uint32_t)got;
  }
  // a bin of thousands: radix descent over the keys inside it, then the ties by index
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += SL_THREADS) sh.hist_m[i] = 0, sh.hist_c[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < len; j += SL_THREADS) {
      const uint32_t k = key_of(rp_to_f32(p[j]));
      if (k == 0 || (shift != 24 && (k >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
      const double z = rm.z(score_of(k));
      if (rm.bin(z) != b) continue;
      atomicAdd(&sh.hist_c[(k >> shift) & 255], 1u);
      const unsigned long long mm = rm.mass(z);
      if (mm) atomicAdd(&sh.hist_m[(k >> shift) & 255], mm);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long cc = count_before, mm = mass_before;
      int d = 255;
      for (; d > 0; --d) {
        if (by_count ? cc + sh.hist_c[d] >= target : mm + sh.hist_m[d] >= target) break;
        cc += sh.hist_c[d];
        mm += sh.hist_m[d];
      }
      sh.digit = d;
      sh.before32 = (uint32_t)cc;
      sh.before64 = mm;
    }
    __syncthreads();
    prefix |= sh.digit << shift;
    count_before = sh.before32;
    mass_before = sh.before64;
  }
  const unsigned long long each = rm.mass(rm.z(score_of(prefix)));
  // the ordinal among the equal scores
  const unsigned long long nth = by_count ? target - count_before : each ? (target - mass_before + each - 1) / each : 1ull;
  *incl = mass_before + nth * each;
  *own = each;
  __syncthreads();
  if (threadIdx.x == 0) sh.found = 0xffffffffu, sh.n_list = 0;
  __syncthreads();
  for (int j0 = 0; j0 < len; j0 += SL_THREADS) {
    const int j = j0 + threadIdx.x;
    const uint32_t k = j < len ? key_of(rp_to_f32(p[j])) : 0u;
    const unsigned long long tie = __ballot(k == prefix);
    __syncthreads();
    if (lane == 0) sh.red32[wave] = (uint32_t)__popcll(tie);
    __syncthreads();
    uint32_t before = sh.n_list, all = 0;
    for (int w = 0; w < SL_THREADS / 64; ++w) {
      before += w < wave ? sh.red32[w] : 0u;
      all += sh.red32[w];
    }
    if (k == prefix && (unsigned long long)before + (unsigned long long)__popcll(tie & ((1ull << lane) - 1ull)) + 1ull == nth) sh.found = (uint32_t)j;
    __syncthreads();
    if (threadIdx.x == 0) sh.n_list += all;
    if (sh.found != 0xffffffffu) break;
  }
  __syncthreads();
  return (int)sh.found;
}

// One workgroup per row: best score, masses and counts per bin, then three seeks - the k-th candidate (only if k cuts), the end of the
// top-p prefix, the draw.
template <class T>
__global__ __launch_bounds__(SL_THREADS) void k_sample_row(sample_args a, int shift) {
  __shared__ unsigned long long hist_m[SB_BINS];
  __shared__ uint32_t hist_c[SB_BINS];
  __shared__ seek_shared sh;
  const int64_t r = a.row0 + blockIdx.x;
  const row_set s = rs_load(a, r);
  const T* p = (const T*)a.scores + r * a.ld;
  for (int i = threadIdx.x; i < SB_BINS; i += SL_THREADS) hist_m[i] = 0, hist_c[i] = 0;
  uint32_t best = 0;
  for (int j = threadIdx.x; j < s.len; j += SL_THREADS) best = max(best, key_of(rp_to_f32(p[j])));
  best = block_max_u32<SL_THREADS>(best, sh.red32);
  if (best == 0) {  // nothing to draw from
    if (threadIdx.x == 0) {
      a.idx[r] = -1;
      a.prob[r] = 0.0f;
      if (a.nnz) a.nnz[r] = 0;
    }
    return;
  }
  row_mass rm;
  rm.best = score_of(best);
  rm.greedy = s.temperature == 0.0f;
  rm.t = rm.greedy ? 1.0 : (double)s.temperature;
  rm.scale = ldexp(1.0, shift);
  unsigned long long above = 0, count = 0;  // mass of the candidates with at least min_p of the best one's mass
  for (int j = threadIdx.x; j < s.len; j += SL_THREADS) {
    const uint32_t k = key_of(rp_to_f32(p[j]));
    if (k == 0) continue;
    const double z = rm.z(score_of(k));
    const unsigned long long m = rm.mass(z);
    const int b = rm.bin(z);
    if (m) atomicAdd(&hist_m[b], m);
    atomicAdd(&hist_c[b], 1u);
    ++count;
    if (s.min_p <= 0.0f || exp_le0(z) >= (double)s.min_p) above += m;
  }
  above = block_sum_u64<SL_THREADS>(above, sh.red64);
  count = block_sum_u64<SL_THREADS>(count, sh.red64);
  unsigned long long incl = 0, own = 0;
  unsigned long long total = 0;
  for (int i = threadIdx.x; i < SB_BINS; i += SL_THREADS) total += hist_m[i];
  total = block_sum_u64<SL_THREADS>(total, sh.red64);
  if ((unsigned long long)s.k < count) {
    seek<T>(p, s.len, rm, hist_m, hist_c, true, (unsigned long long)s.k, sh, &incl, &own);
    total = incl;
  }
  unsigned long long kept = total;
  if (s.top_p < 1.0f && !rm.greedy) {
    const unsigned long long border = max((unsigned long long)ceil((double)s.top_p * (double)total), 1ull);
    if (border < kept) {
      seek<T>(p, s.len, rm, hist_m, hist_c, false, border, sh, &incl, &own);
      kept = incl;
    }
  }
  if (!rm.greedy) kept = min(kept, max(above, (unsigned long long)rm.scale));
  float u = a.u[r * a.ld_u];
  u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
  const unsigned long long want = rm.greedy ? 1ull : min((unsigned long long)floor((double)u * (double)kept) + 1ull, kept);
  const int at = seek<T>(p, s.len, rm, hist_m, hist_c, false, want, sh, &incl, &own);
  if (threadIdx.x == 0) {
    a.idx[r] = at < 0 ? -1 : a.ids ? a.ids[r * a.ld_ids + at] : at;
    a.prob[r] = at < 0 ? 0.0f : rm.greedy ? 1.0f : (float)((double)own / (double)kept);
    if (a.nnz) a.nnz[r] = at < 0 ? 0 : 1;
  }
}

bool bad_fraction(float v) { return !(v >= 0.0f && v <= 1.0f); }

}  // namespace

extern "C" int rphip_sample_workspace(rphip_ctx* ctx, int64_t rows, int64_t width, int32_t draws, int32_t top_k, int64_t* bytes_out) {
  if (!ctx || !bytes_out) RP_FAIL(RPHIP_EINVAL, "sample_workspace: NULL argument");
  (void)rows, (void)width, (void)draws, (void)top_k;
  *bytes_out = 0;
  return RPHIP_OK;
}

extern "C" int rphip_sample(rphip_ctx* ctx, void* stream, int64_t rows, int64_t width, const void* scores_dev, int32_t type, int64_t ld, const int32_t* lengths_dev,
                            const int32_t* ids_dev, int64_t ld_ids, int32_t draws, const float* u_dev, int64_t ld_u, const rphip_sample_params* params, int32_t* idx_dev,
                            float* prob_dev, int32_t* nnz_dev, void* workspace_dev, int64_t workspace_bytes) {
  rp_op_scope scope;
  if (!params) RP_FAIL(RPHIP_EINVAL, "sample: params is NULL");
  if (type != RPHIP_F32 && type != RPHIP_F16 && type != RPHIP_BF16) RP_FAIL(RPHIP_EINVAL, "sample: element type %d: RPHIP_F32, RPHIP_F16 or RPHIP_BF16 expected", type);
  if (rows < 0 || width < 0 || width > ((int64_t)1 << 30)) RP_FAIL(RPHIP_EINVAL, "sample: %lld rows of %lld scores", (long long)rows, (long long)width);
  if (draws < 1) RP_FAIL(RPHIP_EINVAL, "sample: draws = %d", draws);
  if (ld < width || (ids_dev && ld_ids < width) || ld_u < draws) RP_FAIL(RPHIP_EINVAL, "sample: a leading dimension is smaller than its rows");
  if (!(params->temperature >= 0.0f) || params->temperature > 3.4e38f) RP_FAIL(RPHIP_EINVAL, "sample: temperature %g: a finite number >= 0 expected", params->temperature);
  if (bad_fraction(params->top_p) || bad_fraction(params->min_p)) RP_FAIL(RPHIP_EINVAL, "sample: top_p %g, min_p %g: 0 .. 1 expected", params->top_p, params->min_p);
  if (params->top_k < 0) RP_FAIL(RPHIP_EINVAL, "sample: top_k = %d", params->top_k);
  if (params->top_k_dev && params->top_k == 0) RP_FAIL(RPHIP_EINVAL, "sample: top_k per row needs top_k as their bound");
  const int64_t k = params->top_k > 0 ? std::min<int64_t>(params->top_k, width) : width;
  if (draws > 1 && k > RPS_SHORT)
    RP_FAIL(RPHIP_ELIMIT, "sample: %d draws without replacement need top_k (or the width) <= %d, got %lld", draws, RPS_SHORT, (long long)k);
  if (rows == 0) return RPHIP_OK;
  if (!idx_dev || !prob_dev || !u_dev || (width > 0 && !scores_dev)) RP_FAIL(RPHIP_EINVAL, "sample: NULL argument");
  if ((uintptr_t)scores_dev % rp_type_bytes(type)) RP_FAIL(RPHIP_EINVAL, "sample: scores are not aligned to their elements");
  RP_TRY(scope.enter(ctx));
  (void)workspace_dev, (void)workspace_bytes;
  sample_args a = {rows, ld, ld_ids, ld_u, (int)width, draws, scores_dev, lengths_dev, ids_dev, u_dev, params->temperature, params->top_p, params->min_p, params->top_k,
                   params->temperature_dev, params->top_p_dev, params->min_p_dev, params->top_k_dev, idx_dev, prob_dev, nnz_dev, 0};
  int bits = 0;
  while (((int64_t)1 << bits) < width) ++bits;
  const int shift = 61 - bits;  // the row's masses add up to at most width * 2^shift
  return rp_by_type(type, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    const hipStream_t st = (hipStream_t)stream;
    constexpr int64_t STRIP = 1 << 20;  // rows of a launch
    for (a.row0 = 0; a.row0 < rows; a.row0 += STRIP) {
      const unsigned n = (unsigned)std::min<int64_t>(STRIP, rows - a.row0);
      if (width <= 256) k_sample_wave<T, 4><<<(n + 3) / 4, 256, 0, st>>>(a);
      else if (width <= RPS_SHORT) k_sample_wave<T, 16><<<(n + 3) / 4, 256, 0, st>>>(a);
      else if (k <= RPS_SHORT) k_sample_topk<T><<<n, SL_THREADS, 0, st>>>(a);
      else k_sample_row<T><<<n, SL_THREADS, 0, st>>>(a, shift);
      RP_LAUNCHED();
    }
    return RPHIP_OK;
  });
}
