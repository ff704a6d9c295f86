// Sampling items from score rows: temperature, top-k, top-p, min-p, draws without replacement from given uniforms.  C ABI and the
// definition: include/recpack_hip.h, rphip_sample.
//
// Candidates are ranked by (score descending, index ascending); everything below works on that order.  The kept set is a prefix of it,
// a draw inverts the cumulative mass along it.  Whole numbers come out, so sums next to a border decide: masses are float64 (short
// lists) or whole numbers of 64 bits (whole rows, where the order of the adds must not matter), never float32.
#include "rp_ops.h"

#include <algorithm>
#include <type_traits>

#include <float.h>

namespace {

constexpr int RPS_SHORT = 1024;      // longest prefix the list form ranks completely
constexpr int SL_CAP = 4096;         // candidates collected in LDS
constexpr int SL_THREADS = 1024;
constexpr int SB_BINS = 4096;        // mass bins of the whole-row form: 128 per factor of two, the last one takes what lies below 2^-32
constexpr int SB_PER = 128;
constexpr int SB_CAP = 2048;         // entries of a list collected ahead
constexpr int RC_FOUND = 512;        // ... of a workgroup's own part of them, in LDS
constexpr int SR_THREADS = 256;      // threads of a workgroup that takes a slice of a row

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

// ---- exchanges inside a wave: in the vector unit where it can (data-parallel moves, lane swaps), no LDS round trips -----------------
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {  // lanes without a source get 0
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp_f64(double v) {
  return __hiloint2double((int)dpp<CTRL, ROWS>((uint32_t)__double2hiint(v)), (int)dpp<CTRL, ROWS>((uint32_t)__double2loint(v)));
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ unsigned long long dpp_u64(unsigned long long v) {
  return ((unsigned long long)dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32) | dpp<CTRL, ROWS>((uint32_t)v);
}
__device__ __forceinline__ double wave_scan_f64(double v) {  // inclusive
  v += dpp_f64<0x111>(v);       // row_shr:1, 2, 4, 8
  v += dpp_f64<0x112>(v);
  v += dpp_f64<0x114>(v);
  v += dpp_f64<0x118>(v);
  v += dpp_f64<0x142, 0xa>(v);  // row_bcast:15, 31
  v += dpp_f64<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ unsigned long long wave_scan_u64(unsigned long long v) {
  v += dpp_u64<0x111>(v);
  v += dpp_u64<0x112>(v);
  v += dpp_u64<0x114>(v);
  v += dpp_u64<0x118>(v);
  v += dpp_u64<0x142, 0xa>(v);
  v += dpp_u64<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t lane_u32(uint32_t v, int src) { return (uint32_t)__builtin_amdgcn_readlane((int)v, src); }  // src: the same in every lane
__device__ __forceinline__ double lane_f64(double v, int src) {
  return __hiloint2double((int)lane_u32((uint32_t)__double2hiint(v), src), (int)lane_u32((uint32_t)__double2loint(v), src));
}
__device__ __forceinline__ unsigned long long lane_u64(unsigned long long v, int src) {
  return ((unsigned long long)lane_u32((uint32_t)(v >> 32), src) << 32) | lane_u32((uint32_t)v, src);
}
__device__ __forceinline__ double wave_scan(double v) { return wave_scan_f64(v); }
__device__ __forceinline__ unsigned long long wave_scan(unsigned long long v) { return wave_scan_u64(v); }
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
template <int M>
__device__ __forceinline__ uint32_t xor_lane(uint32_t v, int lane) {
  if constexpr (M == 1) return dpp<0xb1>(v);                 // quad_perm [1,0,3,2]
  else if constexpr (M == 2) return dpp<0x4e>(v);            // quad_perm [2,3,0,1]
  else if constexpr (M == 4) return dpp<0x1b>(dpp<0x141>(v));  // half mirror (xor 7), then quad_perm [3,2,1,0] (xor 3)
  else if constexpr (M == 8) return dpp<0x128>(v);           // row_ror:8
  else if constexpr (M == 16) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return lane & 16 ? r.x : r.y;
  } else {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return lane & 32 ? r.x : r.y;
  }
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v, int lane) {
  v = max(v, xor_lane<1>(v, lane));
  v = max(v, xor_lane<2>(v, lane));
  v = max(v, xor_lane<4>(v, lane));
  v = max(v, xor_lane<8>(v, lane));
  v = max(v, xor_lane<16>(v, lane));
  return lane_u32(max(v, xor_lane<32>(v, lane)), 0);
}

// bitonic sort of 64 * PER entries, descending; entry lane * PER + i: steps shorter than PER stay in the lane's registers
template <int PER, int LS>
__device__ __forceinline__ void sort_step(unsigned long long (&e)[PER], int lane, int size) {
  const bool first = ((lane & LS) == 0) == (((lane * PER) & size) == 0);  // this lane keeps the larger one (size > PER here)
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const unsigned long long o = ((unsigned long long)xor_lane<LS>((uint32_t)(e[i] >> 32), lane) << 32) | xor_lane<LS>((uint32_t)e[i], lane);
    e[i] = first == (e[i] > o) ? e[i] : o;
  }
}
template <int PER>
__device__ __forceinline__ void wave_sort(unsigned long long (&e)[PER], int lane) {
#pragma unroll 1
  for (int size = 2; size <= 64 * PER; size <<= 1) {
#pragma unroll 1
    for (int ls = size / (2 * PER); ls > 0; ls >>= 1) {
      switch (ls) {
        case 1: sort_step<PER, 1>(e, lane, size); break;
        case 2: sort_step<PER, 2>(e, lane, size); break;
        case 4: sort_step<PER, 4>(e, lane, size); break;
        case 8: sort_step<PER, 8>(e, lane, size); break;
        case 16: sort_step<PER, 16>(e, lane, size); break;
        default: sort_step<PER, 32>(e, lane, size); break;
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

// a row's scores by 16 bytes: f(first index, scores, how many) for the pieces tid, tid + n, ... of [begin, end); four loads in flight
template <class T>
constexpr int PIECE = 16 / (int)sizeof(T);
template <class T, class F>
__device__ __forceinline__ void scan_row(const T* p, int begin, int end, int tid, int n, F&& f) {
  constexpr int E = PIECE<T>;
  const int64_t step = (int64_t)n * E;
  int64_t j = begin + (int64_t)tid * E;
  for (; j + 3 * step + E <= end; j += 4 * step) {
    rp_vec<T, E> v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = rp_load_vec<T, E>(p + j + q * step);
#pragma unroll
    for (int q = 0; q < 4; ++q) f((int)(j + q * step), v[q], E);
  }
  for (; j < end; j += step) {
    rp_vec<T, E> v;
    const int m = (int)min((int64_t)E, end - j);
    if (m == E) v = rp_load_vec<T, E>(p + j);
    else {
#pragma unroll
      for (int i = 0; i < E; ++i) v.v[i] = i < m ? p[j + i] : rp_from_f32<T>(-INFINITY);
    }
    f((int)j, v, m);
  }
}

// 2^y for -1000 <= y <= 0: Taylor series of exp to the 11th power on [-ln2 / 2, ln2 / 2] (remainder < 2^-47 relative).  The coefficients are
// kept in scalar registers: as vector constants, ahead of a loop, they take 22 of the 64 registers that eight waves per SIMD leave.
__device__ __forceinline__ double in_scalar(double c) {
  asm("" : "+s"(c));
  return c;
}
__device__ __forceinline__ double exp2_le0(double y) {
  const double n = rint(y), f = (y - n) * in_scalar(0.69314718055994530942);
  double q = fma(f, in_scalar(1.0 / 39916800.0), in_scalar(1.0 / 3628800.0));
  q = fma(q, f, in_scalar(1.0 / 362880.0));
  q = fma(q, f, in_scalar(1.0 / 40320.0));
  q = fma(q, f, in_scalar(1.0 / 5040.0));
  q = fma(q, f, in_scalar(1.0 / 720.0));
  q = fma(q, f, in_scalar(1.0 / 120.0));
  q = fma(q, f, in_scalar(1.0 / 24.0));
  q = fma(q, f, in_scalar(1.0 / 6.0));
  q = fma(q, f, 0.5);
  q = fma(q, f, 1.0);
  q = fma(q, f, 1.0);
  return ldexp(q, (int)n);
}

// One wave finishes a row from its leading candidates: sorted[] (in LDS) holds 64 * PER of them ranked, key << 32 | ~index, key 0 where there
// is none, all of the first s.k ranks among them.  Lane l has the ranks l PER .. l PER + PER - 1: their masses in float64 relative to the best
// candidate, and the masses up to and with each of them; NaN instead where there is nothing to draw.  A draw asks all lanes for the first
// one that the uniform falls into and takes that mass off those behind it: a chain of a dozen dependent instructions, whatever PER is.  What is left is summed
// again when it has come down to 2^-6 of the last full sum (so that it keeps a relative precision of 2^-46), and when it has next to no mass
// (a low temperature: the masses underflow, the definition does not) taken relative to the best one left.
template <int PER>
__device__ __forceinline__ void finish_row(const sample_args& a, int64_t r, const row_set& s, const unsigned long long* sorted, int lane) {
  const bool greedy = s.temperature == 0.0f;
  const double c = greedy ? 0.0 : 1.4426950408889634074 / (double)s.temperature;
  auto score_at = [&](int rank) __attribute__((always_inline)) { return score_of((uint32_t)(sorted[rank] >> 32)); };
  float from = score_at(0);  // what the masses are relative to
  auto mass_of = [&](float v) __attribute__((always_inline)) { return v == from ? 1.0 : exp2_le0(fmax(((double)v - (double)from) * c, -1000.0)); };
  double m[PER], upto[PER], total = 0.0;
  uint32_t out = 0;  // bit i: this lane's i-th rank is not kept, or drawn
  auto add_up = [&]() __attribute__((always_inline)) {
    double own = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      own += (out >> i) & 1 ? 0.0 : m[i];
      upto[i] = own;
    }
    const double all = wave_scan_f64(own);
    total = lane_f64(all, 63);
#pragma unroll
    for (int i = 0; i < PER; ++i) upto[i] += all - own;
  };
  int have = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int rank = lane * PER + i;
    const uint32_t key = (uint32_t)(sorted[rank] >> 32);
    const bool candidate = key != 0 && rank < s.k;
    have += (int)__popcll(__ballot(candidate));
    m[i] = candidate && !greedy ? mass_of(score_of(key)) : 0.0;
  }
  int kept = have;
  if (!greedy) {
    add_up();
    // leading ranks kept: those with less than top_p of the mass before them and at least min_p of the best one's mass
    const double border = (double)s.top_p * total;
    kept = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int rank = lane * PER + i;
      kept += (int)__popcll(__ballot(rank < have && (s.top_p >= 1.0f || rank == 0 || upto[i] - m[i] < border) && m[i] >= (double)s.min_p));
    }
  }
  const int own_kept = min(max(kept - lane * PER, 0), PER);
  out = ~((1u << own_kept) - 1u);
  auto hide = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) upto[i] = (out >> i) & 1 ? (double)NAN : upto[i];
  };
  double floor_of = 0.0;
  if (!greedy) {
    if (kept < have) add_up();
    floor_of = total * 0.015625;
    hide();
  }
  const int n_out = min(a.draws, kept);
  for (int d0 = 0; d0 < a.draws; d0 += 64) {  // lane l keeps draw d0 + l
    const int nd = min(64, n_out - d0);
    float u = d0 + lane < n_out ? a.u[r * a.ld_u + d0 + lane] : 0.0f;
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    int pick = d0 + lane;
    double part = 1.0, whole = 1.0;
    for (int d = 0; !greedy && d < nd; ++d) {
      if (total < floor_of) {
        add_up();
        if (total < 1e-200) {  // (kept candidates are left)
          const uint32_t in = ~out & ((1u << PER) - 1u);
          const int who = (int)__ffsll((long long)__ballot(in != 0)) - 1;
          from = score_at(who * PER + (int)lane_u32((uint32_t)__ffs((int)in) - 1u, who));
#pragma unroll
          for (int i = 0; i < PER; ++i) m[i] = (in >> i) & 1 ? mass_of(score_at(lane * PER + i)) : 0.0;
          add_up();
        }
        floor_of = total * 0.015625;
        hide();
      }
      const double want = (double)__uint_as_float(lane_u32(__float_as_uint(u), d)) * total;
      int at = -1;
      double own = 0.0;
#pragma unroll
      for (int i = PER - 1; i >= 0; --i) {
        const bool here = upto[i] > want;
        at = here ? i : at;
        own = here ? m[i] : own;
      }
      unsigned long long pass = __ballot(at >= 0);
      if (pass == 0) {  // (u < 1: only if rounding lets none pass) the last one
        const uint32_t in = ~out & ((1u << PER) - 1u);
        at = 31 - (int)__clz((int)in);
        pass = __ballot(in != 0);
        pass = 1ull << (63 - (int)__clzll((long long)pass));
#pragma unroll
        for (int i = 0; i < PER; ++i) own = i == at ? m[i] : own;
      }
      const int who = (int)__ffsll((long long)pass) - 1;
      const double got = lane_f64(own, who);
      const int drawn = who * PER + (int)lane_u32((uint32_t)at, who), mine = drawn - lane * PER;
      if (lane == d) pick = drawn, part = got, whole = total;
      out |= (uint32_t)mine < (uint32_t)PER ? 1u << mine : 0u;
#pragma unroll
      for (int i = 0; i < PER; ++i) upto[i] -= i > mine ? got : i == mine ? (double)NAN : 0.0;
      total -= got;
    }
    if (d0 + lane < a.draws) {
      const bool drawn = d0 + lane < n_out;
      int32_t item = -1;
      if (drawn) {
        const int32_t at = (int32_t) ~(uint32_t)sorted[pick];
        item = a.ids ? a.ids[r * a.ld_ids + at] : at;
      }
      a.idx[r * a.draws + d0 + lane] = item;
      a.prob[r * a.draws + d0 + lane] = drawn ? (float)(part / whole) : 0.0f;
    }
  }
  if (lane == 0 && a.nnz) a.nnz[r] = n_out;
}

// sort in registers, ranks to this wave's LDS
template <int PER>
__device__ __forceinline__ void rank_row(unsigned long long (&e)[PER], unsigned long long* sorted, int lane) {
  wave_sort<PER>(e, lane);
#pragma unroll
  for (int i = 0; i < PER; ++i) sorted[lane * PER + i] = e[i];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (one wave: its LDS accesses stay in order)
  __builtin_amdgcn_wave_barrier();
}

// ---- rows that one wave holds ------------------------------------------------------------------------------------------------------
// wave_sort for 32-bit entries: a step is one exchange and one instruction (the median with the largest or the smallest number)
__device__ __forceinline__ uint32_t larger_if(uint32_t x, uint32_t y, uint32_t all_ones) { return max(min(x, y), min(max(x, y), all_ones)); }
template <int PER>
__device__ __forceinline__ void wave_sort_u32(uint32_t (&e)[PER], int lane) {
#pragma unroll
  for (int size = 2; size <= 64 * PER; size <<= 1) {
    const uint32_t down = ((lane * PER) & size) == 0 ? ~0u : 0u;  // (size >= PER: of the whole lane)
#pragma unroll
    for (int ls = size / (2 * PER); ls > 0; ls >>= 1) {
      const uint32_t keep = (lane & ls) == 0 ? down : ~down;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t o = ls == 1    ? xor_lane<1>(e[i], lane)
                           : ls == 2  ? xor_lane<2>(e[i], lane)
                           : ls == 4  ? xor_lane<4>(e[i], lane)
                           : ls == 8  ? xor_lane<8>(e[i], lane)
                           : ls == 16 ? xor_lane<16>(e[i], lane)
                                      : xor_lane<32>(e[i], lane);
        e[i] = larger_if(e[i], o, keep);
      }
    }
#pragma unroll
    for (int step = PER >> 1; step > 0; step >>= 1) {
      if (step >= size) continue;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (i & step) continue;
        const uint32_t keep = size >= PER ? down : (i & size) == 0 ? ~0u : 0u, x = e[i], y = e[i + step];
        e[i] = larger_if(x, y, keep);
        e[i + step] = larger_if(x, y, ~keep);
      }
    }
  }
}

// Ranks a row's keys (lane l has the positions l, 64 + l, ..) into this wave's LDS: by their leading bits first, with the position in place of
// the others - a third of the work of sorting 64-bit entries.  Scores that differ in the last 8 to 10 bits of 32 only may then stand the
// wrong way round: two rounds of exchanges between neighbours put that right where it is rare, the full sort where it is not (16-bit
// scores never need it).
template <int PER>
__device__ __forceinline__ void rank_keys(const uint32_t (&key)[PER], unsigned long long* sorted, int lane) {
  constexpr uint32_t AT = 64 * PER - 1;
  uint32_t* keys = (uint32_t*)sorted;
  uint32_t p[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t at = i * 64 + lane;
    keys[at] = key[i];
    p[i] = (key[i] & ~AT) | (AT - at);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (one wave: its LDS accesses stay in order)
  __builtin_amdgcn_wave_barrier();
  wave_sort_u32<PER>(p, lane);
  unsigned long long e[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t at = AT - (p[i] & AT);
    e[i] = ((unsigned long long)keys[at] << 32) | (uint32_t)~at;
  }
  auto next = [&]() __attribute__((always_inline)) {
    const unsigned long long v = __shfl(e[0], min(lane + 1, 63));
    return lane < 63 ? v : 0ull;
  };
  auto wrong = [&]() __attribute__((always_inline)) {
    bool w = e[PER - 1] < next();
#pragma unroll
    for (int i = 0; i + 1 < PER; ++i) w = w || e[i] < e[i + 1];
    return __ballot(w) != 0;
  };
  if (wrong()) {
#pragma unroll 1
    for (int round = 0; round < (PER > 1 ? 2 : 0); ++round) {
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        unsigned long long last = 0, first = 0;
        if (odd) {
          const unsigned long long behind = next(), ahead = __shfl(e[PER - 1], max(lane - 1, 0));
          last = max(e[PER - 1], behind);
          first = lane > 0 ? min(ahead, e[0]) : e[0];
        }
#pragma unroll
        for (int i = odd; i + 1 < PER; i += 2) {
          const unsigned long long x = e[i], y = e[i + 1];
          e[i] = max(x, y), e[i + 1] = min(x, y);
        }
        if (odd) e[0] = first, e[PER - 1] = last;
      }
    }
    if (wrong()) wave_sort<PER>(e, lane);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int i = 0; i < PER; ++i) sorted[lane * PER + i] = e[i];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// One wave per row: up to 64 * PER scores in registers, sorted there.  Bound by the vector unit, which is busy in 92 % of the cycles: 8192 rows of 200, ten
// draws, 24 us, of which the draws are 6; the bytes would take 3.  8192 rows of 1000 (PER = 16), twenty draws: 107 us.
template <class T, int PER>
__global__ __launch_bounds__(256) void k_sample_wave(sample_args a) {
  __shared__ unsigned long long sorted[4][64 * PER];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = a.row0 + (int64_t)blockIdx.x * 4 + wave;
  if (r >= a.rows) return;
  const row_set s = rs_load(a, r);
  const T* p = (const T*)a.scores + r * a.ld;
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = i * 64 + lane < s.len ? key_of(rp_to_f32(p[i * 64 + lane])) : 0u;
  rank_keys<PER>(key, sorted[wave], lane);
  finish_row<PER>(a, r, s, sorted[wave], lane);
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
  v = wave_scan_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) v += red[w];
  return v;
}

// bitonic sort of n (a power of two, 64 .. SL_CAP) entries in LDS, descending: steps of 64 and more through LDS, the shorter ones in the
// registers of a wave that takes 64 entries at a time (15 barriers for 1024 entries instead of 55)
template <int LS>
__device__ __forceinline__ void sort_lanes(unsigned long long& e, int lane, bool desc) {
  const unsigned long long o = ((unsigned long long)xor_lane<LS>((uint32_t)(e >> 32), lane) << 32) | xor_lane<LS>((uint32_t)e, lane);
  e = (((lane & LS) == 0) == desc) == (e > o) ? e : o;
}
// ... of 64 entries, one to a lane, in the given direction
__device__ __forceinline__ void merge_lanes(unsigned long long& v, int lane, bool desc) {
  sort_lanes<32>(v, lane, desc);
  sort_lanes<16>(v, lane, desc);
  sort_lanes<8>(v, lane, desc);
  sort_lanes<4>(v, lane, desc);
  sort_lanes<2>(v, lane, desc);
  sort_lanes<1>(v, lane, desc);
}
__device__ __forceinline__ void sort_run(unsigned long long& v, int lane, bool desc) {
  sort_lanes<1>(v, lane, (lane & 2) == 0);
  sort_lanes<2>(v, lane, (lane & 4) == 0);
  sort_lanes<1>(v, lane, (lane & 4) == 0);
  sort_lanes<4>(v, lane, (lane & 8) == 0);
  sort_lanes<2>(v, lane, (lane & 8) == 0);
  sort_lanes<1>(v, lane, (lane & 8) == 0);
  sort_lanes<8>(v, lane, (lane & 16) == 0);
  sort_lanes<4>(v, lane, (lane & 16) == 0);
  sort_lanes<2>(v, lane, (lane & 16) == 0);
  sort_lanes<1>(v, lane, (lane & 16) == 0);
  sort_lanes<16>(v, lane, (lane & 32) == 0);
  sort_lanes<8>(v, lane, (lane & 32) == 0);
  sort_lanes<4>(v, lane, (lane & 32) == 0);
  sort_lanes<2>(v, lane, (lane & 32) == 0);
  sort_lanes<1>(v, lane, (lane & 32) == 0);
  merge_lanes(v, lane, desc);
}
__device__ __forceinline__ void block_sort(unsigned long long* e, int n) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  for (int i = wave * 64 + lane; i < n; i += SL_THREADS) {
    unsigned long long v = e[i];
    sort_run(v, lane, (i & 64) == 0);
    e[i] = v;
  }
  for (int size = 128; size <= n; size <<= 1) {
    for (int step = size >> 1; step >= 64; step >>= 1) {
      __syncthreads();
      for (int q = threadIdx.x; q < n / 2; q += SL_THREADS) {
        const int i = (q & ~(step - 1)) * 2 + (q & (step - 1)), j = i + step;
        const unsigned long long x = e[i], y = e[j];
        const bool desc = (i & size) == 0;
        if (desc ? x < y : x > y) e[i] = y, e[j] = x;
      }
    }
    __syncthreads();
    for (int i = wave * 64 + lane; i < n; i += SL_THREADS) {
      unsigned long long v = e[i];
      merge_lanes(v, lane, (i & size) == 0);
      e[i] = v;
    }
  }
  __syncthreads();
}

// ---- a workgroup to a row: runs of 64 candidates, one to a wave -------------------------------------------------------------------------
// how many entries of a run of LEN (a power of two, ranked) are larger; three runs side by side, so that three reads are under way
template <int LEN, int N>
__device__ __forceinline__ int count_above(const unsigned long long* const (&run)[N], unsigned long long v) {
  int c[N];
#pragma unroll
  for (int q = 0; q < N; ++q) c[q] = 0;
#pragma unroll
  for (int step = LEN / 2; step > 0; step >>= 1) {
#pragma unroll
    for (int q = 0; q < N; ++q) c[q] += run[q][c[q] + step - 1] > v ? step : 0;
  }
  int sum = 0;
#pragma unroll
  for (int q = 0; q < N; ++q) sum += c[q] + (run[q][c[q]] > v ? 1 : 0);
  return sum;
}

// Ranks 256 entries, one to a thread of four waves (t: 0 .. 255; all different): every wave sorts 64 in its registers, then the runs are joined:
// an entry's place is its own plus, in each other run, the number of larger ones.  The ranked ones stand in to[]; list[] is overwritten.
// Returns this thread's place.  Waves without entries (`on` false) call it for its barriers.
__device__ __forceinline__ int rank_256(unsigned long long& v, unsigned long long* list, unsigned long long* to, int t, bool on) {
  const int lane = t & 63, wave = t >> 6;
  int rank = 0;
  if (on) {
    sort_run(v, lane, true);
    list[t] = v;
  }
  __syncthreads();
  if (on) {
    const unsigned long long* const run[3] = {list + ((wave + 1) & 3) * 64, list + ((wave + 2) & 3) * 64, list + ((wave + 3) & 3) * 64};
    rank = lane + count_above<64>(run, v);
    to[rank] = v;
  }
  __syncthreads();
  return rank;
}

// Ranks n <= 64 * runs entries of list[] (key << 32 | ~index; runs is 4, 8 or 16), 256 at a time and these joined in the same way.  Every thread
// of the workgroup calls it; list[] holds 128 * runs entries, the ranked ones start at the pointer that is returned (behind the last:
// entries with key 0).
__device__ __forceinline__ const unsigned long long* rank_runs(unsigned long long* list, int n, int runs) {
  const int wave = threadIdx.x >> 6, mine = wave >> 2;
  unsigned long long* other = list + 64 * runs;
  unsigned long long v = 0;
  if (wave < runs) v = (int)threadIdx.x < n ? list[threadIdx.x] : (unsigned long long)threadIdx.x;  // (all different, so that places are, too)
  int rank = rank_256(v, list + mine * 256, other + mine * 256, threadIdx.x & 255, wave < runs);
  if (runs == 4) return other;
  if (wave < runs) {
    if (runs == 8) {
      const unsigned long long* const run[1] = {other + (mine ^ 1) * 256};
      rank += count_above<256>(run, v);
    } else {
      const unsigned long long* const run[3] = {other + ((mine + 1) & 3) * 256, other + ((mine + 2) & 3) * 256, other + ((mine + 3) & 3) * 256};
      rank += count_above<256>(run, v);
    }
    list[rank] = v;
  }
  __syncthreads();
  return list;
}

// The row's draws from its ranked candidates (rank_runs), as finish_row defines them: wave i has the masses of the ranks 64 i .. 64 i + 63 and
// their cumulative sums inside the run, in LDS behind that; wave 0 draws, its lane i holding run i's sum: one look finds the run, a
// second one the candidate in it, and only that run is summed again.
struct group_shared {
  double m[RPS_SHORT], cum[RPS_SHORT], sum[16];
  int count[2][16];
};
__device__ __forceinline__ void finish_group(const sample_args& a, int64_t r, const row_set& s, const unsigned long long* sorted, int runs, group_shared& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rank = threadIdx.x;
  const bool greedy = s.temperature == 0.0f;
  const double c = greedy ? 0.0 : 1.4426950408889634074 / (double)s.temperature;
  float from = score_of((uint32_t)(sorted[0] >> 32));  // what the masses are relative to
  auto mass_of = [&](float v) __attribute__((always_inline)) { return v == from ? 1.0 : exp2_le0(fmax(((double)v - (double)from) * c, -1000.0)); };
  double mine = 0.0, incl = 0.0;
  bool candidate = false;
  if (wave < runs) {
    const uint32_t key = (uint32_t)(sorted[rank] >> 32);
    candidate = key != 0 && rank < s.k;
    if (!greedy) {
      mine = candidate ? mass_of(score_of(key)) : 0.0;
      incl = wave_scan_f64(mine);
      if (lane == 63) sh.sum[wave] = incl;
    }
    const int n = (int)__popcll(__ballot(candidate));
    if (lane == 0) sh.count[0][wave] = n;
  }
  __syncthreads();
  int have = 0;
  for (int w = 0; w < runs; ++w) have += sh.count[0][w];
  int kept = have;
  if (!greedy) {
    double before = 0.0, total = 0.0;
    for (int w = 0; w < runs; ++w) {
      before += w < wave ? sh.sum[w] : 0.0;
      total += sh.sum[w];
    }
    // leading ranks kept: those with less than top_p of the mass before them and at least min_p of the best one's mass
    const double border = (double)s.top_p * total;
    if (wave < runs) {
      const int n = (int)__popcll(__ballot(candidate && (s.top_p >= 1.0f || rank == 0 || before + (incl - mine) < border) && mine >= (double)s.min_p));
      if (lane == 0) sh.count[1][wave] = n;
    }
    __syncthreads();
    kept = 0;
    for (int w = 0; w < runs; ++w) kept += sh.count[1][w];
    if (wave < runs) {
      if (kept < have) {
        if (rank >= kept) mine = 0.0;
        incl = wave_scan_f64(mine);
      }
      sh.m[rank] = mine;
      sh.cum[rank] = incl;
      if (lane == 63) sh.sum[wave] = incl;
    }
    __syncthreads();
  }
  if (wave != 0) return;
  // lane i: of run i (runs <= 16: in one row of lanes), and of the runs in front of it
  double sum = !greedy && lane < runs ? sh.sum[lane] : 0.0, floor_of = sum * 0.015625, ahead = 0.0, total = 0.0, total_floor = 0.0;
  auto add_up = [&]() __attribute__((always_inline)) {
    double upto = sum;
    upto += dpp_f64<0x111>(upto);
    upto += dpp_f64<0x112>(upto);
    upto += dpp_f64<0x114>(upto);
    upto += dpp_f64<0x118>(upto);
    ahead = upto - sum;
    total = lane_f64(upto, 15);
    total_floor = total * 0.015625;
  };
  if (!greedy) add_up();
  const int n_out = min(a.draws, kept);
  uint32_t gone = 0;  // bit i: rank 64 i + lane has been drawn
  for (int d0 = 0; d0 < a.draws; d0 += 64) {  // lane l keeps draw d0 + l
    const int nd = min(64, n_out - d0);
    float u = d0 + lane < n_out ? a.u[r * a.ld_u + d0 + lane] : 0.0f;
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    int pick = d0 + lane;
    double part = 1.0, whole = 1.0;
    for (int d = 0; !greedy && d < nd; ++d) {
      if (total < total_floor) {  // (precision: as for a run's sum below)
        add_up();
        if (total < 1e-200) {  // (kept candidates are left: relative to the best of them from here on)
          int first = -1;
          for (int i = runs - 1; i >= 0; --i) {
            const unsigned long long left = __ballot(i * 64 + lane < kept && !((gone >> i) & 1));
            first = left ? i * 64 + (int)__ffsll((long long)left) - 1 : first;
          }
          from = score_of((uint32_t)(sorted[first] >> 32));
          for (int i = 0; i < runs; ++i) {
            const int at = i * 64 + lane;
            const double mass = at < kept && !((gone >> i) & 1) ? mass_of(score_of((uint32_t)(sorted[at] >> 32))) : 0.0;
            const double in = wave_scan_f64(mass);
            sh.m[at] = mass;
            sh.cum[at] = in;
            const double all = lane_f64(in, 63);
            if (lane == i) sum = all, floor_of = all * 0.015625;
          }
          add_up();
        }
      }
      const double want = (double)__uint_as_float(lane_u32(__float_as_uint(u), d)) * total;
      // the run, then the first lane in it; the last ones with mass if rounding lets none pass (u < 1)
      const unsigned long long some = __ballot(sum > 0.0), runs_pass = __ballot(ahead + sum > want) & some;
      const int i = runs_pass ? (int)__ffsll((long long)runs_pass) - 1 : 63 - (int)__clzll((long long)some);
      double m = sh.m[i * 64 + lane], cum = sh.cum[i * 64 + lane];
      const unsigned long long with = __ballot(m > 0.0), pass = __ballot(lane_f64(ahead, i) + cum > want) & with;
      const int who = pass ? (int)__ffsll((long long)pass) - 1 : 63 - (int)__clzll((long long)with);
      const double got = lane_f64(m, who);
      if (lane == d) pick = i * 64 + who, part = got, whole = total;
      if (lane == who) m = 0.0, gone |= 1u << i, sh.m[i * 64 + who] = 0.0;
      // (what is left keeps a relative precision of 2^-46 as long as it is no less than 2^-6 of the last full sum)
      double left = lane_f64(cum, 63) - got;
      if (left >= lane_f64(floor_of, i)) {
        cum -= lane >= who ? got : 0.0;
      } else {
        cum = wave_scan_f64(m);
        left = lane_f64(cum, 63);
        if (lane == i) floor_of = left * 0.015625;
      }
      sh.cum[i * 64 + lane] = cum;
      if (lane == i) sum = left;
      ahead -= lane > i ? got : 0.0;
      total -= got;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (one wave: its LDS accesses stay in order)
      __builtin_amdgcn_wave_barrier();
    }
    if (d0 + lane < a.draws) {
      const bool drawn = d0 + lane < n_out;
      int32_t item = -1;
      if (drawn) {
        const int32_t at = (int32_t) ~(uint32_t)sorted[pick];
        item = a.ids ? a.ids[r * a.ld_ids + at] : at;
      }
      a.idx[r * a.draws + d0 + lane] = item;
      a.prob[r * a.draws + d0 + lane] = drawn ? (float)(part / whole) : 0.0f;
    }
  }
  if (lane == 0 && a.nnz) a.nnz[r] = n_out;
}

// The exact form of "the n-th of the row in rank order" for any row (thousands of equal scores, adversarial orders): radix descent over
// the keys by count, then ties by index.  Returns the key of rank n - 1 (n >= 1, at most the number of candidates) and, in *equal, how
// many candidates with exactly that key belong to the first n.
struct sel_shared {
  uint32_t hist[256];
  uint32_t digit, before;
};
template <class T>
__device__ __forceinline__ uint32_t select_key(const T* p, int len, int n, sel_shared& sh, int* equal) {
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
// 1.4 k at 1000).  Rows that break this - thousands of equal scores - take the radix descent.  A thread keeps the best score of each of its
// HELD pieces of 16 bytes and reads again only those that reach the threshold (HELD = 0: any width, the whole row is read twice: 512 x 20000
// in f32 28 us against 32).  512 x 50000 in bf16, 20 draws from the best 200: 30 us, 51 MB that would take 11; all workgroups are
// resident and read, select, rank and draw at the same time; reading and selecting are 20, the draws 5.
constexpr int TK_HELD = 8;
template <class T, int HELD>
__global__ __launch_bounds__(SL_THREADS, 8) void k_sample_topk(sample_args a) {
  constexpr int E = PIECE<T>;
  __shared__ union {
    unsigned long long list[SL_CAP];
    struct {
      unsigned long long ranked[2 * RPS_SHORT];
      group_shared group;
    };
  } sh;
  __shared__ uint32_t red[2][SL_THREADS / 64], hist[256], pick[2];
  __shared__ uint32_t n_list, cnt;
  __shared__ sel_shared sel;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t r = a.row0 + blockIdx.x;
  const row_set s = rs_load(a, r);
  const T* p = (const T*)a.scores + r * a.ld;
  if (threadIdx.x == 0) n_list = 0;
  float f0 = -INFINITY, f1 = -INFINITY, tops[HELD > 0 ? HELD : 1];
  auto maxima = [&](const rp_vec<T, E>& v) __attribute__((always_inline)) -> float {  // (as numbers: the maximum leaves NaN out)
    float x = -INFINITY, y = -INFINITY;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      x = fmaxf(x, rp_to_f32(v.v[i]));
      y = fmaxf(y, rp_to_f32(v.v[i + E / 2]));
    }
    f0 = fmaxf(f0, x);
    f1 = fmaxf(f1, y);
    return fmaxf(x, y);
  };
  if constexpr (HELD > 0) {
#pragma unroll
    for (int q0 = 0; q0 < HELD; q0 += 4) {  // (four loads in flight: sixteen waves of two workgroups do the rest)
      rp_vec<T, E> v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = ((q0 + q) * SL_THREADS + (int)threadIdx.x) * E;
        if (j + E <= s.len) v[q] = rp_load_vec<T, E>(p + j);
        else {
#pragma unroll
          for (int i = 0; i < E; ++i) v[q].v[i] = j + i < s.len ? p[j + i] : rp_from_f32<T>(-INFINITY);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) tops[q0 + q] = maxima(v[q]);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    scan_row<T>(p, 0, s.len, threadIdx.x, SL_THREADS, [&](int, const rp_vec<T, E>& v, int) __attribute__((always_inline)) { maxima(v); });
  }
  const uint32_t g0 = key_of(f0), g1 = key_of(f1);
  // a value that at least k group maxima reach, and hardly more: a histogram of 256 steps between the least and the largest of them, then
  // of the step where the k-th lies, until few enough reach its lower end.  All 2048 reach lo, `above` of them reach hi.
  uint32_t lo, hi;
  {
    uint32_t v_hi = max(g0, g1), v_lo = ~min(g0, g1);
    v_hi = wave_max_u32(v_hi, lane), v_lo = wave_max_u32(v_lo, lane);
    if (lane == 0) red[0][wave] = v_hi, red[1][wave] = v_lo;
    if (threadIdx.x < 256) hist[threadIdx.x] = 0;
    __syncthreads();
    hi = 0, lo = 0;
#pragma unroll
    for (int w = 0; w < SL_THREADS / 64; ++w) hi = max(hi, red[0][w]), lo = max(lo, red[1][w]);
    lo = ~lo;
  }
  const uint32_t k = (uint32_t)s.k, enough = k + k / 4;
  uint32_t above = 0, steps = 256;  // group maxima beyond the range [lo, lo + (steps << shift))
  for (int shift = max(24 - (int)__clz(hi - lo + 1), 0); hi > lo;) {
    const uint32_t b0 = (g0 - lo) >> shift, b1 = (g1 - lo) >> shift;
    if (g0 >= lo && b0 < steps) atomicAdd(&hist[b0], 1u);
    if (g1 >= lo && b1 < steps) atomicAdd(&hist[b1], 1u);
    __syncthreads();
    if (wave == 0) {  // lane l: the bins 255 - 4 l downwards
      uint32_t h[4], own = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = hist[255 - 4 * lane - i], own += h[i], hist[255 - 4 * lane - i] = 0;
      uint32_t incl = own;
      incl += dpp<0x111>(incl);
      incl += dpp<0x112>(incl);
      incl += dpp<0x114>(incl);
      incl += dpp<0x118>(incl);
      incl += dpp<0x142, 0xa>(incl);
      incl += dpp<0x143, 0xc>(incl);
      uint32_t run = above + incl - own;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (run < k && run + h[i] >= k) pick[0] = 255 - 4 * lane - i, pick[1] = run;
        run += h[i];
      }
    }
    __syncthreads();
    const uint32_t bin = pick[0];
    above = pick[1];
    lo += bin << shift;
    if (shift == 0) break;
    const uint32_t reach = (uint32_t)__popcll(__ballot(g0 >= lo)) + (uint32_t)__popcll(__ballot(g1 >= lo));
    if (lane == 0) red[0][wave] = reach;
    __syncthreads();
    uint32_t n = 0;
#pragma unroll
    for (int w = 0; w < SL_THREADS / 64; ++w) n += red[0][w];
    if (n <= enough) break;
    steps = shift >= 8 ? 256u : 1u << shift;
    shift = max(shift - 8, 0);
  }
  const float least = lo > 0x00800000u ? score_of(lo) : -FLT_MAX;  // (every candidate: neither -inf nor NaN passes)
  auto take = [&](int j, const rp_vec<T, E>& v, int m) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float x = rp_to_f32(v.v[i]);
      if (i < m && x >= least) {
        const uint32_t at = atomicAdd(&n_list, 1u);
        if (at < SL_CAP) sh.list[at] = ((unsigned long long)key_of(x) << 32) | (uint32_t) ~(j + i);
      }
    }
  };
  if constexpr (HELD > 0) {  // the few pieces that hold one are read again
    uint32_t hits = 0;
#pragma unroll
    for (int q = 0; q < HELD; ++q) hits |= tops[q] >= least ? 1u << q : 0u;
    while (hits) {
      const int j = (((int)__ffs((int)hits) - 1) * SL_THREADS + (int)threadIdx.x) * E;
      hits &= hits - 1;
      rp_vec<T, E> v;
      const int m = min(E, s.len - j);
      if (m == E) v = rp_load_vec<T, E>(p + j);
      else {
#pragma unroll
        for (int i = 0; i < E; ++i) v.v[i] = i < m ? p[j + i] : (T)0.0f;
      }
      take(j, v, m);
    }
  } else {
    scan_row<T>(p, 0, s.len, threadIdx.x, SL_THREADS, [&](int j, const rp_vec<T, E>& v, int m) __attribute__((always_inline)) {
      float top = rp_to_f32(v.v[0]);
#pragma unroll
      for (int i = 1; i < E; ++i) top = fmaxf(top, rp_to_f32(v.v[i]));
      if (top >= least) take(j, v, m);
    });
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
      const uint32_t key = j < s.len ? key_of(rp_to_f32(p[j])) : 0u;
      const unsigned long long tie = __ballot(key == kk);
      __syncthreads();
      if (lane == 0) red[0][wave] = (uint32_t)__popcll(tie);
      __syncthreads();
      uint32_t before = cnt, all = 0;
      for (int w = 0; w < SL_THREADS / 64; ++w) {
        before += w < wave ? red[0][w] : 0u;
        all += red[0][w];
      }
      const bool in = key > kk || (key == kk && before + (uint32_t)__popcll(tie & ((1ull << lane) - 1ull)) < (uint32_t)equal);
      if (in) sh.list[atomicAdd(&n_list, 1u)] = ((unsigned long long)key << 32) | (uint32_t)~j;  // (s.k <= 1024 entries in all)
      __syncthreads();
      if (threadIdx.x == 0) cnt += all;
    }
    __syncthreads();
    n = (int)n_list;
  }
  if (n > RPS_SHORT) {  // (ties, or an order the groups did not expect) the best of them, s.k count
    int n2 = 2 * RPS_SHORT;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += SL_THREADS) sh.list[i] = 0;
    block_sort(sh.list, n2);
    n = RPS_SHORT;
  }
  const int runs = n <= 256 ? 4 : n <= 512 ? 8 : 16;
  finish_group(a, r, s, rank_runs(sh.list, n, runs), runs, sh.group);
}

// ---- whole rows, any prefix, one draw ------------------------------------------------------------------------------------------------
// Masses of a row's candidates relative to its best score, by t = 128 log2(mass) (0 for the best score, +inf among them; -16000 where nothing
// is left).  Its nearest whole number is the bin; 2^(t / 128) is a power of two from a table of 128, times a polynomial of degree 4
// on +-ln2 / 256 (remainder < 2^-49 relative).  Some 20 instructions; a series of degree 11 and the conversion to 64 bits took 40 (this pass over 512
// rows of 100000: 99 us, 84 so).
// A bin's are added up as whole numbers, so that no order matters, in a unit of its octave (the power of two at or above the bin): 2^-(shift +
// octave).  In one unit for all of them the tail of a very wide row would round away (2^25 masses of 2^-37); so each is kept to 2^-(shift + 1) of
// itself, 2^-45 at 100000 scores and 2^-32 at 2^30, down to 2^-32 of the best one's, and to 2^-(shift + 33) of that below (the last bin): the
// sums are right to 2^-31 at any width.  A bin's sum fits 64 bits (width * 2^(shift + 1) <= 2^62); the sums along the bins are float64, always
// added in the same order.
constexpr int SB_OCTAVES = SB_BINS / SB_PER;
__device__ __forceinline__ int octave_of(int bin) { return (bin + SB_PER - 1) / SB_PER; }
struct row_mass {
  float best;
  double c;      // 128 log2(e) / temperature
  int shift;
  double scale;  // 2^shift
  bool greedy;
  const double* powers;  // 2^(j / 128), in LDS
  __device__ __forceinline__ double t_of(float x) const { return x == best ? 0.0 : greedy ? -16000.0 : fmax(((double)x - (double)best) * c, -16000.0); }
  __device__ __forceinline__ int bin(double t) const { return min(-(int)rint(t), SB_BINS - 1); }
  __device__ __forceinline__ double in_octave(double t) const {  // the mass times 2^octave: 1 .. 2, less in the last bin
    constexpr double L = 0.69314718055994530942 / SB_PER;
    const double n = rint(t), f = t - n;
    const int i = (int)n;
    double q = fma(f, in_scalar(L * L * L * L / 24.0), in_scalar(L * L * L / 6.0));
    q = fma(q, f, in_scalar(L * L / 2.0));
    q = fma(q, f, in_scalar(L));
    q = fma(q, f, 1.0);
    return ldexp(powers[i & (SB_PER - 1)], min((i >> 7) + SB_OCTAVES, 0)) * q;
  }
  __device__ __forceinline__ double value(double t) const { return ldexp(in_octave(t), -octave_of(bin(t))); }
  // (shift <= 50: the add of 2^52 rounds)
  __device__ __forceinline__ unsigned long long whole(double in_octave) const { return (unsigned long long)__double_as_longlong(fma(in_octave, scale, 0x1p52)) ^ 0x4330000000000000ull; }
  __device__ __forceinline__ unsigned long long mass(double t) const { return whole(in_octave(t)); }
  __device__ __forceinline__ double sum(unsigned long long masses, int bin) const { return ldexp((double)masses, -shift - octave_of(bin)); }
  __device__ __forceinline__ double kept(double t) const { return sum(mass(t), bin(t)); }  // the mass as it is added up
};
// The bins around min_p: every candidate in front of them has more than min_p of the best one's mass, those behind them have less; `above` adds up
// those inside that have as much, in units of 2^-(shift + unit).  (A logarithm in float32 is off by less than a hundredth of a bin.)  No min_p: none.
struct near_bins {
  int first, last, unit;
  __device__ __forceinline__ bool holds(int b) const { return b >= first && b <= last; }
};
__device__ __forceinline__ near_bins near_of(const row_mass& rm, float min_p) {
  if (!(min_p > 0.0f)) return {SB_BINS, -1, 0};
  const int b = rm.bin(fmax((double)(SB_PER * __builtin_amdgcn_logf(min_p)), -16000.0)), first = max(b - 1, 0);
  return {first, min(b + 1, SB_BINS - 1), min(octave_of(first) + 1, SB_OCTAVES)};
}
// (every thread of the workgroup; a barrier has to follow; without `powers` for t and bins only)
__device__ __forceinline__ row_mass rm_make(uint32_t best, const row_set& s, int shift, double* powers) {
  if (powers && threadIdx.x < SB_PER) powers[threadIdx.x] = 2.0 * exp2_le0((double)threadIdx.x / SB_PER - 1.0);
  row_mass rm;
  rm.best = score_of(best);
  rm.greedy = s.temperature == 0.0f;
  rm.c = rm.greedy ? 1.0 : 1.4426950408889634074 * SB_PER / (double)s.temperature;
  rm.shift = shift;
  rm.scale = ldexp(1.0, shift);
  rm.powers = powers;
  return rm;
}

// a row's part of the workspace
struct row_ws {
  unsigned long long hist_m[SB_BINS];  // masses per bin
  unsigned long long above, count;     // mass of the candidates of the bins around min_p that reach it (near_bins); candidates
  double total, most, before[2];       // all mass; that of the candidates that reach min_p; the masses in front of the lists' bins
  unsigned long long list[2][SB_CAP];  // candidates of bin b1 (where top-p ends) and of the bins b2 (where the draw can fall)
  uint32_t hist_c[SB_BINS];            // candidates per bin
  uint32_t n_list[2];
  int32_t b1, b2_lo, b2_hi;            // b1 < 0: top-p does not cut; b2_hi < b2_lo: nothing was collected
  uint32_t best[64];                   // per slice
};

struct seek_shared {
  unsigned long long list[SL_CAP];
  double red64[SL_THREADS / 64];
  double before64;
  uint32_t red32[SL_THREADS / 64];
  uint32_t n_list, before32, bin, digit, found;
  unsigned long long hist_m[256];
  uint32_t hist_c[256];
};

// Cumulative masses or counts over the bins, four to a thread (in rounds, if the workgroup has fewer than 1024): bin_at(i) starts at before[i] and
// ends where the next one starts, at end(before, i).  The adds come in the same order whatever the number of threads.
template <int THREADS>
struct bin_sums {
  static constexpr int ROUNDS = SB_BINS / 4 / THREADS, N = ROUNDS * 4;
  static __device__ __forceinline__ int bin_at(int i) { return ((i >> 2) * THREADS + (int)threadIdx.x) * 4 + (i & 3); }
  template <class V> using sums = V[ROUNDS * 5];  // (a round: four bins, and the end of the last one)
  template <class V>
  static __device__ __forceinline__ const V& start(const sums<V>& before, int i) { return before[(i >> 2) * 5 + (i & 3)]; }
  template <class V>
  static __device__ __forceinline__ const V& end(const sums<V>& before, int i) { return before[(i >> 2) * 5 + (i & 3) + 1]; }
  // value(bin) -> V; returns the total.  red: SB_BINS / 256 entries
  template <class V, class F>
  static __device__ __forceinline__ V scan(F&& value, sums<V>& before, V* red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    V incl[ROUNDS];
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
      V run = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        before[q * 5 + i] = run;
        run += value(bin_at(q * 4 + i));
      }
      incl[q] = wave_scan(run);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q)
      if (lane == 63) red[q * (THREADS / 64) + wave] = incl[q];
    __syncthreads();
    V at[ROUNDS] = {}, total = 0;
#pragma unroll
    for (int w = 0; w < SB_BINS / 256; ++w) {
#pragma unroll
      for (int q = 0; q < ROUNDS; ++q) at[q] = w == q * (THREADS / 64) + wave ? total : at[q];
      total += red[w];
    }
#pragma unroll
    for (int q = 0; q < ROUNDS; ++q) {
      const V first = at[q] + below(incl[q], lane), last = at[q] + incl[q];
#pragma unroll
      for (int i = 0; i < 4; ++i) before[q * 5 + i] = min(first + before[q * 5 + i], last);  // (rounding: no bin ends before it starts)
      before[q * 5 + 4] = last;
    }
    return total;
  }
  static __device__ __forceinline__ double below(double v, int lane) {
    const double t = __shfl_up(v, 1);
    return lane > 0 ? t : 0.0;
  }
  static __device__ __forceinline__ unsigned long long below(unsigned long long v, int lane) {
    const unsigned long long t = __shfl_up(v, 1);
    return lane > 0 ? t : 0ull;
  }
};

// what a cumulative mass has to reach: top_p of the total; more than u of what is kept (u < 1)
__device__ __forceinline__ double border_of(float top_p, double total) { return fmax((double)top_p * total, DBL_MIN); }
__device__ __forceinline__ double want_of(float u, double kept) {
  u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
  return fmin(nextafter((double)u * kept, (double)INFINITY), kept);
}

// First candidate in rank order with (by_count: rank + 1 >= target; otherwise: cumulative mass up to and with it >= target).
// bm / bc: the masses and counts (by_count only) in front of this thread's bins.  ahead / n_ahead: the candidates of the bins lo .. hi, if they
// were collected (n_ahead >= 0).  Returns its index (-1: none) and, in *incl, the cumulative mass with it.
using seek_sums = bin_sums<SL_THREADS>;
template <class T>
__device__ __forceinline__ int seek(const T* p, int len, const row_mass& rm, const seek_sums::sums<double>& bm, const seek_sums::sums<unsigned long long>& bc, bool by_count,
                                    double target, int count, seek_shared& sh, const unsigned long long* ahead, int n_ahead, int lo, int hi, double* incl) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) sh.bin = SB_BINS, sh.n_list = 0, sh.found = 0xffffffffu;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < seek_sums::N; ++i)
    if (by_count ? bc[i] < (unsigned long long)count && bc[i + 1] >= (unsigned long long)count : bm[i] < target && bm[i + 1] >= target)
      atomicMin(&sh.bin, (uint32_t)seek_sums::bin_at(i));  // (rounding can let two neighbours end at the same mass)
  __syncthreads();
  const bool have = n_ahead >= 0 && (int)sh.bin >= lo && (int)sh.bin <= hi;  // (never by count)
#pragma unroll
  for (int i = 0; i < seek_sums::N; ++i)
    if (seek_sums::bin_at(i) == (have ? lo : (int)sh.bin)) sh.before64 = bm[i], sh.before32 = (uint32_t)bc[i];
  __syncthreads();
  const int b = (int)sh.bin;
  if (b >= SB_BINS) return -1;
  double mass_before = sh.before64;
  int count_before = (int)sh.before32;
  int n = n_ahead;
  if (have && n > 256) {
    for (int i = threadIdx.x; i < n; i += SL_THREADS) sh.list[i] = ahead[i];
  } else if (!have) {  // collect the bin
    scan_row<T>(p, 0, len, threadIdx.x, SL_THREADS, [&](int j, const rp_vec<T, PIECE<T>>& v, int) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < PIECE<T>; ++i) {
        const uint32_t k = key_of(rp_to_f32(v.v[i]));
        if (k != 0 && rm.bin(rm.t_of(score_of(k))) == b) {
          const uint32_t at = atomicAdd(&sh.n_list, 1u);
          if (at < SL_CAP) sh.list[at] = ((unsigned long long)k << 32) | (uint32_t) ~(j + i);
        }
      }
    });
    __syncthreads();
    n = (int)sh.n_list;
  }
  if (n <= 256) {  // one wave ranks them and adds up
    if (wave == 0) {
      unsigned long long e[4];
      const unsigned long long* from = have ? ahead : sh.list;
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = i * 64 + lane < n ? from[i * 64 + lane] : 0ull;
      rank_row<4>(e, sh.list, lane);
      double run = mass_before;
      bool looking = true;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rank = i * 64 + lane;
        const double cum = run + wave_scan(rank < n ? rm.kept(rm.t_of(score_of((uint32_t)(sh.list[rank] >> 32)))) : 0.0);
        const unsigned long long pass = __ballot(rank < n && (by_count ? count_before + rank + 1 == count : cum >= target || rank == n - 1));  // (rounding: the last one)
        if (looking && pass) {
          const int who = (int)__ffsll((long long)pass) - 1;
          looking = false;
          if (lane == who) sh.found = (uint32_t)rank, sh.before64 = cum;
        }
        run = lane_f64(cum, 63);
      }
    }
    __syncthreads();
    const uint32_t f = sh.found;
    const unsigned long long got = f == 0xffffffffu ? 0ull : sh.list[f];
    *incl = sh.before64;
    __syncthreads();
    return f == 0xffffffffu ? -1 : (int)~(uint32_t)got;
  }
  if (n <= SL_CAP) {
    int n2 = 64;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += SL_THREADS) sh.list[i] = 0;
    block_sort(sh.list, n2);
    // cumulative sums along the sorted list: 1024 entries at a time
    for (int i0 = 0; i0 < n; i0 += SL_THREADS) {
      const int i = i0 + threadIdx.x;
      const double s = wave_scan(i < n ? rm.kept(rm.t_of(score_of((uint32_t)(sh.list[i] >> 32)))) : 0.0);
      __syncthreads();
      if (lane == 63) sh.red64[wave] = s;
      __syncthreads();
      double off = mass_before, all = 0.0;
      for (int w = 0; w < SL_THREADS / 64; ++w) {
        off += w < wave ? sh.red64[w] : 0.0;
        all += sh.red64[w];
      }
      const double cum = off + s;
      if (i < n && (by_count ? count_before + i + 1 == count : cum >= target || i == n - 1)) atomicMin(&sh.found, (uint32_t)i);
      __syncthreads();
      if (sh.found == (uint32_t)i) sh.before64 = cum;
      if (sh.found != 0xffffffffu) break;
      mass_before += all;
    }
    __syncthreads();
    const uint32_t f = sh.found;
    const unsigned long long got = f == 0xffffffffu ? 0ull : sh.list[f];
    *incl = sh.before64;
    __syncthreads();
    return f == 0xffffffffu ? -1 : (int)~(uint32_t)got;
  }
  // a bin of thousands: radix descent over the keys inside it, then the ties by index
  uint32_t prefix = 0, ties = 1;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += SL_THREADS) sh.hist_m[i] = 0, sh.hist_c[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < len; j += SL_THREADS) {
      const uint32_t k = key_of(rp_to_f32(p[j]));
      if (k == 0 || (shift != 24 && (k >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
      const double z = rm.t_of(score_of(k));
      if (rm.bin(z) != b) continue;
      atomicAdd(&sh.hist_c[(k >> shift) & 255], 1u);
      const unsigned long long mm = rm.mass(z);
      if (mm) atomicAdd(&sh.hist_m[(k >> shift) & 255], mm);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int cc = count_before, digit = 0, cc_at = cc;
      double mm = mass_before, mm_at = mm;
      for (int d = 255; d >= 0; --d) {  // (rounding may let none reach a target at the bin's end: the last one with candidates)
        if (sh.hist_c[d] == 0) continue;
        digit = d, cc_at = cc, mm_at = mm;
        cc += (int)sh.hist_c[d];
        mm += rm.sum(sh.hist_m[d], b);
        if (by_count ? cc >= count : mm >= target) break;
      }
      sh.digit = digit;
      sh.before32 = (uint32_t)cc_at;
      sh.before64 = mm_at;
    }
    __syncthreads();
    prefix |= sh.digit << shift;
    count_before = (int)sh.before32;
    mass_before = sh.before64;
    ties = sh.hist_c[sh.digit];
  }
  const double each = rm.kept(rm.t_of(score_of(prefix)));
  // the ordinal among the equal scores
  const double nth_of = each > 0.0 ? fmin(fmax(ceil((target - mass_before) / each), 1.0), (double)ties) : 1.0;
  const unsigned long long nth = by_count ? (unsigned long long)(count - count_before) : (unsigned long long)nth_of;
  *incl = mass_before + (double)nth * each;
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

// The whole-row form: for few wide rows in four or five launches, three of them with a row's slices spread over workgroups,
//   best     the slices' best scores; clears the row's workspace
//   hist     masses and counts per bin (fixed point: the order of the atomics does not matter)
//   bins     the bin where top-p ends and the bins where the draw can fall (known up to one bin's mass); very few rows: inside collect
//   collect  the candidates of these bins
//   draw     one workgroup: the exact end of the kept prefix, then the draw
// otherwise the same in one launch (k_row_one).  Read three times, from memory once where it fits the caches.  (The last slice of hist in the
// place of bins needs a fence in every workgroup that writes its XCD's cache back: 16 us instead of 7 for one row.)  One row of 100000: 25
// us, four launches one after the other.
__device__ __forceinline__ void slice_of(int len, int slices, int s, int& begin, int& end) {
  const int64_t pieces = ((int64_t)len + 7) / 8;
  begin = (int)(pieces * s / slices * 8);
  end = (int)min(pieces * (s + 1) / slices * 8, (int64_t)len);
}

template <class T>
__global__ __launch_bounds__(SR_THREADS) void k_row_best(sample_args a, row_ws* __restrict__ wss) {
  __shared__ uint32_t red[SR_THREADS / 64];
  const int slices = gridDim.y, sl = blockIdx.y;
  const int64_t r = a.row0 + blockIdx.x;
  row_ws& ws = wss[blockIdx.x];
  for (int i = sl * SR_THREADS + threadIdx.x; i < SB_BINS; i += slices * SR_THREADS) ws.hist_m[i] = 0, ws.hist_c[i] = 0;
  if (sl == 0 && threadIdx.x == 0) ws.above = 0, ws.count = 0, ws.n_list[0] = 0, ws.n_list[1] = 0;
  const row_set s = rs_load(a, r);
  int begin, end;
  slice_of(s.len, slices, sl, begin, end);
  uint32_t best = 0;
  scan_row<T>((const T*)a.scores + r * a.ld, begin, end, threadIdx.x, SR_THREADS, [&](int, const rp_vec<T, PIECE<T>>& v, int) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) best = max(best, key_of(rp_to_f32(v.v[i])));
  });
  best = block_max_u32<SR_THREADS>(best, red);
  if (threadIdx.x == 0) ws.best[sl] = best;
}

// (one load a lane: a loop over the slices is a chain of as many scalar loads, 10 us of a launch)
__device__ __forceinline__ uint32_t best_of(const row_ws& ws, int slices) {
  const int lane = threadIdx.x & 63;
  return wave_max_u32(lane < slices ? ws.best[lane] : 0u, lane);
}

template <class T, bool COUNT>
__global__ __launch_bounds__(SR_THREADS) void k_row_hist(sample_args a, row_ws* __restrict__ wss, int shift) {
  __shared__ double powers[SB_PER];
  __shared__ unsigned long long hist_m[SB_BINS];
  __shared__ uint32_t hist_c[COUNT ? SB_BINS : 1];
  __shared__ unsigned long long red[SR_THREADS / 64];
  const int slices = gridDim.y, sl = blockIdx.y;
  const int64_t r = a.row0 + blockIdx.x;
  row_ws& ws = wss[blockIdx.x];
  const row_set s = rs_load(a, r);
  const uint32_t best = best_of(ws, slices);
  if (best == 0) return;
  const row_mass rm = rm_make(best, s, shift, powers);
  for (int i = threadIdx.x; i < SB_BINS; i += SR_THREADS) {
    hist_m[i] = 0;
    if (COUNT) hist_c[i] = 0;
  }
  __syncthreads();
  int begin, end;
  slice_of(s.len, slices, sl, begin, end);
  unsigned long long above = 0, count = 0;
  const double least = (double)s.min_p;
  const near_bins near = near_of(rm, s.min_p);
  scan_row<T>((const T*)a.scores + r * a.ld, begin, end, threadIdx.x, SR_THREADS, [&](int, const rp_vec<T, PIECE<T>>& v, int) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) {
      const uint32_t k = key_of(rp_to_f32(v.v[i]));
      if (k == 0) continue;
      const double t = rm.t_of(score_of(k)), e = rm.in_octave(t);
      const unsigned long long m = rm.whole(e);
      const int b = rm.bin(t);
      if (m) atomicAdd(&hist_m[b], m);
      if (COUNT) {
        atomicAdd(&hist_c[b], 1u);
        ++count;
      }
      if (near.holds(b) && ldexp(e, -octave_of(b)) >= least) above += m << (near.unit - octave_of(b));
    }
  });
  above = block_sum_u64<SR_THREADS>(above, red);
  if (COUNT) count = block_sum_u64<SR_THREADS>(count, red);
  __syncthreads();
  for (int i = threadIdx.x; i < SB_BINS; i += SR_THREADS) {
    if (hist_m[i]) atomicAdd(&ws.hist_m[i], hist_m[i]);
    if (COUNT && hist_c[i]) atomicAdd(&ws.hist_c[i], hist_c[i]);
  }
  if (threadIdx.x == 0) {
    if (above) atomicAdd(&ws.above, above);
    if (COUNT && count) atomicAdd(&ws.count, count);
  }
}

// where top-p ends, and between which masses the draw falls: every thread of the workgroup
struct row_bins {
  int b1, lo, hi;
  double total, most;
};
template <int THREADS, bool COUNT>
__device__ __forceinline__ row_bins find_bins(const row_ws& ws, const row_mass& rm, const row_set& s, float u, const near_bins& near,
                                              typename bin_sums<THREADS>::template sums<double>& before) {
  using B = bin_sums<THREADS>;
  __shared__ double red[SB_BINS / 256], range[2], ahead;
  __shared__ int bins[3];
  if (threadIdx.x == 0) bins[0] = -1, bins[1] = SB_BINS, bins[2] = -1;
  const double total = B::template scan<double>([&](int b) __attribute__((always_inline)) { return rm.sum(ws.hist_m[b], b); }, before, red);
#pragma unroll
  for (int i = 0; i < B::N; ++i)
    if (B::bin_at(i) == near.first) ahead = B::start(before, i);
  __syncthreads();
  const double most = near.last < 0 ? total : ahead + ldexp((double)ws.above, -rm.shift - near.unit);
  const bool known = s.temperature != 0.0f && !(COUNT && (unsigned long long)s.k < ws.count);  // (otherwise the total itself is not known yet)
  if (known) {
    const double border = border_of(s.top_p, total);
    const bool cuts = s.top_p < 1.0f && border < total;
    if (threadIdx.x == 0) range[0] = range[1] = total;
    __syncthreads();
    if (cuts) {
#pragma unroll
      for (int i = 0; i < B::N; ++i)
        if (B::start(before, i) < border && B::end(before, i) >= border) atomicMax(&bins[0], B::bin_at(i));  // (rounding can let two neighbours end at the same mass)
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < B::N; ++i)
      if (B::bin_at(i) == bins[0]) range[0] = border, range[1] = B::end(before, i);
    __syncthreads();
    const double w0 = want_of(u, fmin(range[0], most)), w1 = want_of(u, fmin(range[1], most));
#pragma unroll
    for (int i = 0; i < B::N; ++i) {
      if (B::start(before, i) < w0 && B::end(before, i) >= w0) atomicMin(&bins[1], B::bin_at(i));
      if (B::start(before, i) < w1 && B::end(before, i) >= w1) atomicMax(&bins[2], B::bin_at(i));
    }
  }
  __syncthreads();
  return {bins[0], bins[1], bins[2], total, most};
}
template <int THREADS>
__device__ __forceinline__ void keep_bins(row_ws& ws, const row_bins& b, const typename bin_sums<THREADS>::template sums<double>& before) {
  using B = bin_sums<THREADS>;
  if (threadIdx.x == 0) ws.b1 = b.b1, ws.b2_lo = b.lo, ws.b2_hi = b.hi, ws.total = b.total, ws.most = b.most;
#pragma unroll
  for (int i = 0; i < B::N; ++i) {
    if (B::bin_at(i) == b.b1) ws.before[0] = B::start(before, i);
    if (B::bin_at(i) == b.lo) ws.before[1] = B::start(before, i);
  }
}
template <bool COUNT>
__global__ __launch_bounds__(SL_THREADS) void k_row_bins(sample_args a, row_ws* __restrict__ wss, int slices, int shift) {
  const int64_t r = a.row0 + blockIdx.x;
  row_ws& ws = wss[blockIdx.x];
  const row_set s = rs_load(a, r);
  const uint32_t best = best_of(ws, slices);
  if (best == 0) return;
  bin_sums<SL_THREADS>::sums<double> before;
  const row_mass rm = rm_make(best, s, shift, nullptr);
  const row_bins b = find_bins<SL_THREADS, COUNT>(ws, rm, s, a.u[r * a.ld_u], near_of(rm, s.min_p), before);
  keep_bins<SL_THREADS>(ws, b, before);
}

// between which scores the bins b1 and lo .. hi lie, half a bin more on either side, and a float's step: all others are passed over by
// comparisons
struct row_ranges {
  float low1, high1, low2, high2;
  __device__ __forceinline__ bool holds(float x) const { return (x >= low1 && x <= high1) || (x >= low2 && x <= high2); }
};
__device__ __forceinline__ row_ranges ranges_of(const row_mass& rm, const row_bins& b) {
  auto above = [&](int bin) __attribute__((always_inline)) { return nextafterf((float)((double)rm.best + (1.0 - bin) / rm.c), INFINITY); };
  auto below = [&](int bin) __attribute__((always_inline)) { return bin == SB_BINS - 1 ? -INFINITY : nextafterf((float)((double)rm.best - (1.0 + bin) / rm.c), -INFINITY); };
  return {b.b1 < 0 ? INFINITY : below(b.b1), b.b1 < 0 ? -INFINITY : above(b.b1), b.hi < b.lo ? INFINITY : below(b.hi), b.hi < b.lo ? -INFINITY : above(b.lo)};
}

// (FIND: every workgroup finds the bins itself, where one launch less is more)
template <class T, bool COUNT, bool FIND>
__global__ __launch_bounds__(SR_THREADS) void k_row_collect(sample_args a, row_ws* __restrict__ wss, int slices, int shift) {
  __shared__ unsigned long long found[2][RC_FOUND];
  __shared__ uint32_t n_found[2], at_found[2];
  const int sl = blockIdx.y;
  const int64_t r = a.row0 + blockIdx.x;
  row_ws& ws = wss[blockIdx.x];
  const row_set s = rs_load(a, r);
  const uint32_t best = best_of(ws, slices);
  if (best == 0) return;
  const row_mass rm = rm_make(best, s, shift, nullptr);
  if (threadIdx.x < 2) n_found[threadIdx.x] = 0;
  __syncthreads();
  row_bins bins;
  if constexpr (FIND) {
    bin_sums<SR_THREADS>::sums<double> before;
    bins = find_bins<SR_THREADS, COUNT>(ws, rm, s, a.u[r * a.ld_u], near_of(rm, s.min_p), before);
    if (sl == 0) keep_bins<SR_THREADS>(ws, bins, before);
  } else {
    bins = {ws.b1, ws.b2_lo, ws.b2_hi, 0, 0};
  }
  const int b1 = bins.b1, lo = bins.lo, hi = bins.hi;
  if (b1 < 0 && hi < lo) return;
  const row_ranges ranges = ranges_of(rm, bins);
  int begin, end;
  slice_of(s.len, gridDim.y, sl, begin, end);
  scan_row<T>((const T*)a.scores + r * a.ld, begin, end, threadIdx.x, SR_THREADS, [&](int j, const rp_vec<T, PIECE<T>>& v, int) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) {
      const float x = rp_to_f32(v.v[i]);
      if (!ranges.holds(x)) continue;
      const uint32_t k = key_of(x);
      if (k == 0) continue;
      const int b = rm.bin(rm.t_of(score_of(k)));
      const unsigned long long entry = ((unsigned long long)k << 32) | (uint32_t) ~(j + i);
      auto put = [&](int which) __attribute__((always_inline)) {
        uint32_t at = atomicAdd(&n_found[which], 1u);
        if (at < RC_FOUND) found[which][at] = entry;
        else if ((at = atomicAdd(&ws.n_list[which], 1u)) < SB_CAP) ws.list[which][at] = entry;
      };
      if (b == b1) put(0);
      if (b >= lo && b <= hi) put(1);
    }
  });
  // (one reservation per workgroup: thousands of atomics on one address would be the launch)
  __syncthreads();
  if (threadIdx.x < 2) at_found[threadIdx.x] = atomicAdd(&ws.n_list[threadIdx.x], min(n_found[threadIdx.x], (uint32_t)RC_FOUND));
  __syncthreads();
#pragma unroll
  for (int which = 0; which < 2; ++which)
    for (uint32_t i = threadIdx.x; i < min(n_found[which], (uint32_t)RC_FOUND); i += SR_THREADS)
      if (at_found[which] + i < SB_CAP) ws.list[which][at_found[which] + i] = found[which][i];
}

// A list of at most 256 candidates, ranked by four waves: sorted[] and the cumulative masses with those in front of the list, and each one's own.
struct ranked_list {
  unsigned long long runs[256], sorted[256];
  double cum[256], own[256], sum[4];
};
// the first rank whose cumulative mass reaches the target (n if none); a whole wave
__device__ __forceinline__ int rank_reaching(const ranked_list& l, int n, double target, int lane) {
  int at = n;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    const unsigned long long pass = __ballot(i * 64 + lane < n && l.cum[i * 64 + lane] >= target);
    if (pass) at = i * 64 + (int)__ffsll((long long)pass) - 1;
  }
  return at;
}

union draw_shared {
  seek_shared seek;
  ranked_list two[2];
};
__device__ __forceinline__ void nothing_drawn(const sample_args& a, int64_t r) {
  if (threadIdx.x == 0) {
    a.idx[r] = -1;
    a.prob[r] = 0.0f;
    if (a.nnz) a.nnz[r] = 0;
  }
}
// the draw from what was collected; a workgroup of SL_THREADS
template <class T, bool COUNT>
__device__ __forceinline__ void draw_row(const sample_args& a, int64_t r, const row_set& s, const T* p, const row_mass& rm, const row_ws& ws, draw_shared& sh) {
  __shared__ double red_m[SB_BINS / 256];
  __shared__ unsigned long long red_c[SB_BINS / 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b1 = ws.b1, b2_lo = ws.b2_lo, b2_hi = ws.b2_hi;
  const int n1 = b1 >= 0 && ws.n_list[0] <= SB_CAP ? (int)ws.n_list[0] : -1;
  const int n2 = b2_hi >= b2_lo && ws.n_list[1] <= SB_CAP ? (int)ws.n_list[1] : -1;
  const int which = wave >> 2, t = threadIdx.x & 255;  // (waves 0 - 3: the first list, 4 - 7: the second one)
  unsigned long long e = t;
  if (which < 2 && t < (which == 0 ? n1 : n2)) e = ws.list[which][t];
  __syncthreads();
  const double most = ws.most;
  const bool cut_by_count = COUNT && (unsigned long long)s.k < ws.count;
  // the common case - both lists are there and short: four waves each, side by side
  if (!cut_by_count && !rm.greedy && (b1 < 0 || (n1 >= 1 && n1 <= 256)) && n2 >= 1 && n2 <= 256) {
    const bool on = which == 1 || (which == 0 && b1 >= 0);
    ranked_list& mine = sh.two[which & 1];
    const int rank = rank_256(e, mine.runs, mine.sorted, t, on);
    double cum = 0.0;
    const double before = ws.before[which & 1];
    // (this thread's entry, where it belongs)
    if (on) mine.own[rank] = rank < (which == 0 ? n1 : n2) ? rm.kept(rm.t_of(score_of((uint32_t)(e >> 32)))) : 0.0;
    __syncthreads();
    if (on) {
      cum = wave_scan(mine.own[t]);
      if (lane == 63) mine.sum[wave & 3] = cum;
    }
    __syncthreads();
    if (on) {
      cum += before;
#pragma unroll
      for (int w = 0; w < 3; ++w) cum += w < (wave & 3) ? mine.sum[w] : 0.0;
      mine.cum[t] = cum;
    }
    __syncthreads();
    if (wave != 0) return;
    double kept = ws.total;
    if (b1 >= 0) kept = sh.two[0].cum[min(rank_reaching(sh.two[0], n1, border_of(s.top_p, kept), lane), n1 - 1)];
    kept = fmin(kept, most);
    const int at_rank = min(rank_reaching(sh.two[1], n2, want_of(a.u[r * a.ld_u], kept), lane), n2 - 1);
    if (lane == 0) {
      const unsigned long long entry = sh.two[1].sorted[at_rank];
      const int at = (int)~(uint32_t)entry;
      a.idx[r] = a.ids ? a.ids[r * a.ld_ids + at] : at;
      a.prob[r] = (float)(rm.value(rm.t_of(score_of((uint32_t)(entry >> 32)))) / kept);
      if (a.nnz) a.nnz[r] = 1;
    }
    return;
  }
  double incl = 0.0;
  seek_sums::sums<double> bm;
  seek_sums::sums<unsigned long long> bc = {};
  double total = seek_sums::scan<double>([&](int b) __attribute__((always_inline)) { return rm.sum(ws.hist_m[b], b); }, bm, red_m);
  if (cut_by_count) {
    seek_sums::scan<unsigned long long>([&](int b) __attribute__((always_inline)) { return (unsigned long long)ws.hist_c[b]; }, bc, red_c);
    seek<T>(p, s.len, rm, bm, bc, true, 0.0, s.k, sh.seek, nullptr, -1, 0, -1, &incl);
    total = incl;
  }
  double kept = total;
  if (s.top_p < 1.0f && !rm.greedy) {
    const double border = border_of(s.top_p, total);
    if (border < kept) {
      seek<T>(p, s.len, rm, bm, bc, false, border, 0, sh.seek, ws.list[0], n1, b1, b1, &incl);
      kept = incl;
    }
  }
  if (!rm.greedy) kept = fmin(kept, most);
  const double want = rm.greedy ? DBL_MIN : want_of(a.u[r * a.ld_u], kept);
  const int at = seek<T>(p, s.len, rm, bm, bc, false, want, 0, sh.seek, ws.list[1], n2, b2_lo, b2_hi, &incl);
  if (threadIdx.x == 0) {
    a.idx[r] = at < 0 ? -1 : a.ids ? a.ids[r * a.ld_ids + at] : at;
    a.prob[r] = at < 0 ? 0.0f : rm.greedy ? 1.0f : (float)(rm.value(rm.t_of(rp_to_f32(p[at]))) / kept);
    if (a.nnz) a.nnz[r] = at < 0 ? 0 : 1;
  }
}

template <class T, bool COUNT>
__global__ __launch_bounds__(SL_THREADS) void k_row_draw(sample_args a, const row_ws* __restrict__ wss, int slices, int shift) {
  __shared__ double powers[SB_PER];
  __shared__ draw_shared sh;
  const int64_t r = a.row0 + blockIdx.x;
  const row_ws& ws = wss[blockIdx.x];
  const row_set s = rs_load(a, r);
  const uint32_t best = best_of(ws, slices);
  if (best == 0) return nothing_drawn(a, r);
  const row_mass rm = rm_make(best, s, shift, powers);
  draw_row<T, COUNT>(a, r, s, (const T*)a.scores + r * a.ld, rm, ws, sh);
}

// ... all of it in one launch, a workgroup to a row, its workspace in LDS (151 KB with the draw's: one to a CU).  Bound by the vector unit (some 25 instructions
// in 64 bits a score and the LDS atomics) and by what one workgroup has under way: 512 rows of 100000 in f32 165 us, where reading them takes 43.
struct one_shared {
  row_ws ws;
  draw_shared draw;
};
template <class T, bool COUNT>
__global__ __launch_bounds__(SL_THREADS) void k_row_one(sample_args a, int shift) {
  extern __shared__ __attribute__((aligned(16))) char one_lds[];
  __shared__ double powers[SB_PER];
  __shared__ uint32_t red[SL_THREADS / 64];
  __shared__ unsigned long long red64[SL_THREADS / 64];
  row_ws& ws = ((one_shared*)one_lds)->ws;
  const int64_t r = a.row0 + blockIdx.x;
  const row_set s = rs_load(a, r);
  const T* p = (const T*)a.scores + r * a.ld;
  const float u = a.u[r * a.ld_u];
  uint32_t best = 0;
  scan_row<T>(p, 0, s.len, threadIdx.x, SL_THREADS, [&](int, const rp_vec<T, PIECE<T>>& v, int) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) best = max(best, key_of(rp_to_f32(v.v[i])));
  });
  for (int i = threadIdx.x; i < SB_BINS; i += SL_THREADS) {
    ws.hist_m[i] = 0;
    if (COUNT) ws.hist_c[i] = 0;
  }
  if (threadIdx.x < 2) ws.n_list[threadIdx.x] = 0;
  best = block_max_u32<SL_THREADS>(best, red);
  if (best == 0) return nothing_drawn(a, r);
  const row_mass rm = rm_make(best, s, shift, powers);
  __syncthreads();
  unsigned long long above = 0, count = 0;
  const double least = (double)s.min_p;
  const near_bins near = near_of(rm, s.min_p);
  scan_row<T>(p, 0, s.len, threadIdx.x, SL_THREADS, [&](int, const rp_vec<T, PIECE<T>>& v, int) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PIECE<T>; ++i) {
      const uint32_t k = key_of(rp_to_f32(v.v[i]));
      if (k == 0) continue;
      const double t = rm.t_of(score_of(k)), e = rm.in_octave(t);
      const unsigned long long m = rm.whole(e);
      const int b = rm.bin(t);
      if (m) atomicAdd(&ws.hist_m[b], m);
      if (COUNT) {
        atomicAdd(&ws.hist_c[b], 1u);
        ++count;
      }
      if (near.holds(b) && ldexp(e, -octave_of(b)) >= least) above += m << (near.unit - octave_of(b));
    }
  });
  above = block_sum_u64<SL_THREADS>(above, red64);
  if (COUNT) count = block_sum_u64<SL_THREADS>(count, red64);
  if (threadIdx.x == 0) ws.above = above, ws.count = count;
  __syncthreads();
  bin_sums<SL_THREADS>::sums<double> before;
  const row_bins bins = find_bins<SL_THREADS, COUNT>(ws, rm, s, u, near, before);
  keep_bins<SL_THREADS>(ws, bins, before);
  if (bins.b1 >= 0 || bins.hi >= bins.lo) {
    const row_ranges ranges = ranges_of(rm, bins);
    scan_row<T>(p, 0, s.len, threadIdx.x, SL_THREADS, [&](int j, const rp_vec<T, PIECE<T>>& v, int) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < PIECE<T>; ++i) {
        const float x = rp_to_f32(v.v[i]);
        if (!ranges.holds(x)) continue;
        const uint32_t k = key_of(x);
        if (k == 0) continue;
        const int b = rm.bin(rm.t_of(score_of(k)));
        const unsigned long long entry = ((unsigned long long)k << 32) | (uint32_t) ~(j + i);
        auto put = [&](int which) __attribute__((always_inline)) {
          const uint32_t at = atomicAdd(&ws.n_list[which], 1u);
          if (at < SB_CAP) ws.list[which][at] = entry;
        };
        if (b == bins.b1) put(0);
        if (b >= bins.lo && b <= bins.hi) put(1);
      }
    });
  }
  __syncthreads();
  draw_row<T, COUNT>(a, r, s, p, rm, ws, ((one_shared*)one_lds)->draw);
}

// which form a call takes, and its workspace
enum sample_form { FORM_WAVE, FORM_LISTS, FORM_ROWS };
sample_form form_of(int64_t width, int64_t k) { return width <= RPS_SHORT ? FORM_WAVE : k <= RPS_SHORT ? FORM_LISTS : FORM_ROWS; }
// One workgroup to a row and launch, or slices of few wide rows over the card: 1 x 12000 20 us against 26, 256 x 12000 22 against 61, 64 x 50000 42
// against 62, 512 x 100000 165 against 198; but 1 x 50000 37 against 25 and 16 x 100000 67 against 43 (f32).
bool one_launch(int64_t rows, int64_t width) { return width <= 20000 || rows >= 64; }
int64_t workspace_of(int64_t rows, int64_t width, int64_t k) {
  switch (form_of(width, k)) {
    case FORM_ROWS: return one_launch(rows, width) ? 0 : rows * (int64_t)sizeof(row_ws);
    default: return 0;
  }
}
int64_t reach_of(int64_t width, int32_t top_k) { return top_k > 0 ? std::min<int64_t>(top_k, width) : width; }

bool bad_fraction(float v) { return !(v >= 0.0f && v <= 1.0f); }

}  // namespace

extern "C" int rphip_sample_workspace(rphip_ctx* ctx, int64_t rows, int64_t width, int32_t draws, int32_t top_k, int64_t* bytes_out) {
  if (!ctx || !bytes_out) RP_FAIL(RPHIP_EINVAL, "sample_workspace: NULL argument");
  if (rows < 0 || width < 0 || draws < 1 || top_k < 0) RP_FAIL(RPHIP_EINVAL, "sample_workspace: %lld rows of %lld, draws = %d, top_k = %d", (long long)rows, (long long)width, draws, top_k);
  *bytes_out = workspace_of(rows, width, reach_of(width, top_k));
  return RPHIP_OK;
}

extern "C" int rphip_sample(rphip_ctx* ctx, void* stream, int64_t rows, int64_t width, const void* scores_dev, int32_t type, int64_t ld, const int32_t* lengths_dev,
                            const int32_t* ids_dev, int64_t ld_ids, int32_t draws, const float* u_dev, int64_t ld_u, const rphip_sample_params* params, int32_t* idx_dev,
                            float* prob_dev, int32_t* nnz_dev, void* workspace_dev, int64_t workspace_bytes) {
  rp_op_scope scope;
  if (!params) RP_FAIL(RPHIP_EINVAL, "sample: params is NULL");
  if (type != RPHIP_F32 && type != RPHIP_F16 && type != RPHIP_BF16) RP_FAIL(RPHIP_EINVAL, "sample: element type %d: RPHIP_F32, RPHIP_F16 or RPHIP_BF16 expected", type);
  if (rows < 0 || width < 0 || width > ((int64_t)1 << 30)) RP_FAIL(RPHIP_EINVAL, "sample: %lld rows of %lld scores", (long long)rows, (long long)width);
  if (draws < 1 || draws > 1 << 30) RP_FAIL(RPHIP_EINVAL, "sample: draws = %d", draws);
  if (ld < width || (ids_dev && ld_ids < width) || ld_u < draws) RP_FAIL(RPHIP_EINVAL, "sample: a leading dimension is smaller than its rows");
  if (!(params->temperature >= 0.0f) || params->temperature > 3.4e38f) RP_FAIL(RPHIP_EINVAL, "sample: temperature %g: a finite number >= 0 expected", params->temperature);
  if (bad_fraction(params->top_p) || bad_fraction(params->min_p)) RP_FAIL(RPHIP_EINVAL, "sample: top_p %g, min_p %g: 0 .. 1 expected", params->top_p, params->min_p);
  if (params->top_k < 0) RP_FAIL(RPHIP_EINVAL, "sample: top_k = %d", params->top_k);
  if (params->top_k_dev && params->top_k == 0) RP_FAIL(RPHIP_EINVAL, "sample: top_k per row needs top_k as their bound");
  const int64_t k = reach_of(width, params->top_k);
  if (draws > 1 && k > RPS_SHORT)
    RP_FAIL(RPHIP_ELIMIT, "sample: %d draws without replacement need top_k (or the width) <= %d, got %lld", draws, RPS_SHORT, (long long)k);
  if (rows == 0) return RPHIP_OK;
  if (!idx_dev || !prob_dev || !u_dev || (width > 0 && !scores_dev)) RP_FAIL(RPHIP_EINVAL, "sample: NULL argument");
  if ((uintptr_t)scores_dev % rp_type_bytes(type)) RP_FAIL(RPHIP_EINVAL, "sample: scores are not aligned to their elements");
  RP_TRY(scope.enter(ctx));
  const int64_t need = workspace_of(rows, width, k);
  if (workspace_bytes < need || (need > 0 && !workspace_dev) || ((uintptr_t)workspace_dev & 255))
    RP_FAIL(RPHIP_EINVAL, "sample: a workspace of %lld bytes, aligned to 256, is needed (rphip_sample_workspace)", (long long)need);
  sample_args a = {rows, ld, ld_ids, ld_u, (int)width, draws, scores_dev, lengths_dev, ids_dev, u_dev, params->temperature, params->top_p, params->min_p, params->top_k,
                   params->temperature_dev, params->top_p_dev, params->min_p_dev, params->top_k_dev, idx_dev, prob_dev, nnz_dev, 0};
  int bits = 0;
  while (((int64_t)1 << bits) < width) ++bits;
  const int shift = 61 - bits;  // (row_mass: 31 .. 50)
  return rp_by_type(type, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    const hipStream_t st = (hipStream_t)stream;
    switch (form_of(width, k)) {
      case FORM_WAVE:
        for (a.row0 = 0; a.row0 < rows; a.row0 += 1 << 20) {
          const unsigned n = (unsigned)std::min<int64_t>(1 << 20, rows - a.row0);
          if (width <= 64) k_sample_wave<T, 1><<<(n + 3) / 4, 256, 0, st>>>(a);
          else if (width <= 256) k_sample_wave<T, 4><<<(n + 3) / 4, 256, 0, st>>>(a);
          else if (width <= 512) k_sample_wave<T, 8><<<(n + 3) / 4, 256, 0, st>>>(a);
          else k_sample_wave<T, 16><<<(n + 3) / 4, 256, 0, st>>>(a);
          RP_LAUNCHED();
        }
        return RPHIP_OK;
      case FORM_LISTS:
        for (a.row0 = 0; a.row0 < rows; a.row0 += 1 << 20) {
          const unsigned n = (unsigned)std::min<int64_t>(1 << 20, rows - a.row0);
          constexpr int64_t piece = SL_THREADS * PIECE<T>;
          if (width <= TK_HELD * piece) k_sample_topk<T, TK_HELD><<<n, SL_THREADS, 0, st>>>(a);
          else k_sample_topk<T, 0><<<n, SL_THREADS, 0, st>>>(a);
          RP_LAUNCHED();
        }
        return RPHIP_OK;
      default: {
        auto go = [&](auto by_count) -> int {
          constexpr bool COUNT = decltype(by_count)::value;
          if (one_launch(rows, width)) {
            RP_HIP(hipFuncSetAttribute((const void*)k_row_one<T, COUNT>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(one_shared)));
            for (a.row0 = 0; a.row0 < rows; a.row0 += 1 << 20) {
              k_row_one<T, COUNT><<<(unsigned)std::min<int64_t>(1 << 20, rows - a.row0), SL_THREADS, sizeof(one_shared), st>>>(a, shift);
              RP_LAUNCHED();
            }
            return RPHIP_OK;
          }
          // slices of a row: about eight workgroups per CU in all, of no fewer than 1024 scores
          const unsigned n = (unsigned)rows;
          const int slices = (int)std::max<int64_t>(1, std::min<int64_t>({8 * (int64_t)ctx->n_cu / rows, width / 1024, 64}));
          row_ws* ws = (row_ws*)workspace_dev;
          k_row_best<T><<<dim3(n, slices), SR_THREADS, 0, st>>>(a, ws);
          RP_LAUNCHED();
          k_row_hist<T, COUNT><<<dim3(n, slices), SR_THREADS, 0, st>>>(a, ws, shift);
          RP_LAUNCHED();
          // very few rows: a launch (3 - 4 us) costs more than finding the bins in every slice (one row of 100000: 25.2 us against 26.5; 8 rows the same,
          // 16 rows 44 against 42)
          if (n <= 8) {
            k_row_collect<T, COUNT, true><<<dim3(n, slices), SR_THREADS, 0, st>>>(a, ws, slices, shift);
          } else {
            k_row_bins<COUNT><<<n, SL_THREADS, 0, st>>>(a, ws, slices, shift);
            RP_LAUNCHED();
            k_row_collect<T, COUNT, false><<<dim3(n, slices), SR_THREADS, 0, st>>>(a, ws, slices, shift);
          }
          RP_LAUNCHED();
          k_row_draw<T, COUNT><<<n, SL_THREADS, 0, st>>>(a, ws, slices, shift);
          RP_LAUNCHED();
          return RPHIP_OK;
        };
        return params->top_k > 0 ? go(std::true_type{}) : go(std::false_type{});
      }
    }
  });
}
