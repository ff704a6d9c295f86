// C[M,N] = A[M,K] W[N,K]^T with W in MXFP4 (one scale per 32 along K) and A in f32 / f16 / bf16, or MXFP4 as well.  f32 accumulate.
// C ABI: include/recpack_hip.h, rphip_mxfp4_gemm_nt.
//
// 16- and 32-bit A: every element of W is a bf16 number exactly (two significant bits times a power of two), and every element of A a
// sum of one (bf16) or three (f32: 8 + 8 + 8 bits) of them, so the product runs on v_mfma_f32_16x16x32_bf16 with exact operands; the
// planes of A are cut once into a workspace, W is converted in registers.  f16 A runs on v_mfma_f32_16x16x32_f16 as it is: a row of W
// relative to the power of two of its largest block is a row of f16 numbers exactly as long as its blocks' scales lie within 2^36 of each other
// (subnormals included), and its sums are scaled back as they are stored.  Rows of W that span more are found beforehand and their
// columns of C are computed again with f16 as two bf16 planes (8 + 3 bits).
// MXFP4 A: v_mfma_scale_f32_16x16x128_f8f6f4, which takes codes and scales as they are.
#include "rp_ops.h"

#include <algorithm>
#include <type_traits>

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int KC = 128;  // K of a chunk: four MX blocks

// ---- the operands' workspace forms ---------------------------------------------------------------------------------------------------
// A fragment is what the 64 lanes of a wave hand to one matrix instruction: lane (row = l & 15, g = l >> 4) holds 16 bytes.  Chunk c of a
// row is its MX blocks 4 c .. 4 c + 3; lane group g takes block 4 c + g.  Inside a chunk K runs in the order (step s, g, 8 elements) for the
// bf16 instruction and (g, 32 elements) for the 4-bit one - the same for both operands, which is all a product asks - so a lane's 16
// code bytes are one MX block with one scale in either kernel.

// by truncation: the high part never overflows, each remainder is exact down to 2^-133, bf16's least number (of an f32 element below 2^-110 the
// bits under that are left out)
template <int P>
__device__ __forceinline__ void cut_planes(float x, uint16_t (&h)[P]) {
  const uint32_t b = __float_as_uint(x);
  if ((b & 0x7f800000u) == 0x7f800000u) {  // Inf, NaN (kept a NaN)
    h[0] = (uint16_t)(b >> 16) | ((b & 0x7fffffu) ? 0x40 : 0);
#pragma unroll
    for (int p = 1; p < P; ++p) h[p] = 0;
    return;
  }
  float r = x;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t t = __float_as_uint(r) & 0xffff0000u;
    h[p] = (uint16_t)(t >> 16);
    r -= __uint_as_float(t);
  }
}

// A -> planes [16-row block][chunk][plane][step 4][lane 64][8 bf16], zero beyond K and M: fragments are contiguous KB.  One wave per
// (block, chunk, step), the four steps of a chunk in one workgroup: together they read whole lines.
template <class T, int P>
__device__ __forceinline__ void cut_fragment(const T* __restrict__ a, int64_t lda, int M, int K, int nc, int64_t frag, int s, int lane, uint16_t* __restrict__ out) {
  const int64_t mb = frag / nc, m = mb * 16 + (lane & 15);
  const int c = (int)(frag - mb * nc), k = c * KC + (lane >> 4) * 32 + s * 8;
  const T* p = a + m * lda + k;
  float v[8];
  if (m < M && k + 8 <= K) {
    const rp_vec<T, 8> t = rp_load_vec<T, 8>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = rp_to_f32(t.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = m < M && k + i < K ? rp_to_f32(p[i]) : 0.0f;
  }
  uint16_t h[8][P];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (std::is_same<T, _Float16>::value) h[i][0] = __builtin_bit_cast(uint16_t, (_Float16)v[i]);  // (as it is: P = 1)
    else cut_planes<P>(v[i], h[i]);
  }
  uint4* o = (uint4*)(out + (frag * P * 4 + s) * 512) + lane;
#pragma unroll
  for (int pl = 0; pl < P; ++pl) {
    uint4 w;
    w.x = h[0][pl] | (uint32_t)h[1][pl] << 16;
    w.y = h[2][pl] | (uint32_t)h[3][pl] << 16;
    w.z = h[4][pl] | (uint32_t)h[5][pl] << 16;
    w.w = h[6][pl] | (uint32_t)h[7][pl] << 16;
    o[pl * 4 * 64] = w;
  }
}

// Scales -> [16-row block][four chunks][lane 64] words: byte cc = the scale of the lane's block of chunk 4 q + cc.  Blocks beyond the
// row get 0 (2^-127): whatever their codes hold, the product underflows to nothing.  Rows beyond the matrix repeat the last one.
__device__ __forceinline__ void pack_scales(const uint8_t* __restrict__ s, int64_t lds, int rows, int nb, int nq, int64_t unit, uint32_t* __restrict__ out) {
  const int lane = (int)(unit & 63);
  const int64_t f = unit >> 6, rb = f / nq;
  const int q = (int)(f - rb * nq);
  const int64_t r = min(rb * 16 + (lane & 15), (int64_t)rows - 1);
  const int b = q * 16 + (lane >> 4);
  uint32_t w = 0;
#pragma unroll
  for (int cc = 0; cc < 4; ++cc)
    if (b + cc * 4 < nb) w |= (uint32_t)s[r * lds + b + cc * 4] << (8 * cc);
  out[unit] = w;
}

// The same for W beside f16 A, a workgroup to 16 rows: scales relative to the row's largest one, which becomes 2^HALF_TOP (6 * 2^13 is an f16
// number); top[] keeps the largest, wide[block] has a bit for each row with an element that f16 does not hold then.
constexpr int HALF_TOP = 13, HALF_SPAN = 36;  // (.5 * 2^(13 - 36) = 2^-24, the least f16 number)
__device__ __forceinline__ void pack_scales_half(const uint8_t* __restrict__ s, int64_t lds, const uint8_t* __restrict__ codes, int64_t ldc, int rows, int nb, int nq, int64_t rb,
                                                 uint32_t* __restrict__ out, uint8_t* __restrict__ top, uint16_t* __restrict__ wide) {
  __shared__ uint32_t best[16], lost;
  const int t = threadIdx.x, row = t >> 4;
  if (t < 16) best[t] = 0;
  if (t == 0) lost = 0;
  __syncthreads();
  const int64_t r = min(rb * 16 + row, (int64_t)rows - 1);
  uint32_t m = 0;
  for (int b = t & 15; b < nb; b += 16) {
    const uint32_t v = s[r * lds + b];
    m = max(m, v == 255u ? 0u : v);
  }
  atomicMax(&best[row], m);
  __syncthreads();
  for (int u = t; u < nq * 64; u += 256) {
    const int lane = u & 63, b = (u >> 6) * 16 + (lane >> 4);
    const int64_t rr = min(rb * 16 + (lane & 15), (int64_t)rows - 1);
    const int e = (int)best[lane & 15];
    uint32_t w = 0;
#pragma unroll
    for (int cc = 0; cc < 4; ++cc) {
      if (b + cc * 4 >= nb) break;
      const int v = s[rr * lds + b + cc * 4], span = e - v;
      if (v != 255 && span > HALF_SPAN) {
        const uint4 q = *(const uint4*)(codes + rr * ldc + (int64_t)(b + cc * 4) * 16);
        if (((q.x | q.y | q.z | q.w) & 0x77777777u) != 0) atomicOr(&lost, 1u << (lane & 15));  // (blocks of zeros lose nothing; codes behind the last column are 0)
      }
      w |= (uint32_t)(v == 255 ? 255 : max(127 + HALF_TOP - span, 0)) << (8 * cc);
    }
    out[rb * nq * 64 + u] = w;
  }
  __syncthreads();
  if (t < 16) top[rb * 16 + t] = (uint8_t)best[t];
  if (t == 0) wide[rb] = (uint16_t)lost;
}

// One launch for all of them (2^23 workgroups at a time, from wg0): workgroups [0, wg_w) pack W's scales, the others cut A (P > 0) or pack A's scales.  2048 x 20000 of A in f16 and
// the scales of 20000 x 20000 of W: 52 us of 1.37 ms (once a call: 4 bytes an element of A and 2 a scale, read and written).
struct half_args {  // (f16 A only)
  const uint8_t* codes;
  int64_t ldc;
  uint8_t* top;
  uint16_t* wide;
};
template <class T, int P>
__global__ __launch_bounds__(256) void k_mxg_prepare(const uint8_t* __restrict__ ws, int64_t ldws, int N, int nb, int nq, int64_t w_units, uint32_t* __restrict__ w_out,
                                                     int64_t wg0, int64_t wg_w, const T* __restrict__ a, int64_t lda, int M, int K, int nc, int64_t a_units,
                                                     void* __restrict__ a_out, half_args half) {
  int64_t wg = wg0 + blockIdx.x;
  if (wg < wg_w) {
    if constexpr (std::is_same<T, _Float16>::value) {
      pack_scales_half(ws, ldws, half.codes, half.ldc, N, nb, nq, wg, w_out, half.top, half.wide);
      return;
    }
    const int64_t unit = wg * 256 + threadIdx.x;
    if (unit < w_units) pack_scales(ws, ldws, N, nb, nq, unit, w_out);
    return;
  }
  wg -= wg_w;
  if constexpr (P > 0) {
    if (wg < a_units) cut_fragment<T, P>(a, lda, M, K, nc, wg, threadIdx.x >> 6, threadIdx.x & 63, (uint16_t*)a_out);
  } else {
    const int64_t unit = wg * 256 + threadIdx.x;
    if (unit < a_units) pack_scales(a, lda, M, nb, nq, unit, (uint32_t*)a_out);
  }
}

// eight codes (a dword) to eight bf16
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t w, float s) {
  rp_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
  rp_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
  bf16x8 r = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  return r;
}

__device__ __forceinline__ f16x8 codes_f16(uint32_t w, float s) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 1);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, 3);
  return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

struct gemm_args {
  int M, N, nb, nc, nq;      // nb: blocks of a row of W (and of an MXFP4 A); nc: chunks; nq: groups of four chunks
  const uint8_t* planes;     // 16-bit form of A
  const uint8_t* a_codes; int64_t lda; const uint32_t* a_scales;  // MXFP4 A (scales in the workspace form)
  const uint8_t* w; int64_t ldw; const uint32_t* w_scales;
  const uint8_t* w_top;      // f16 A: the largest scale of each row of W (padded to 16 rows)
  void* c; int64_t ldc;
  float* part;               // split K: partial sums [split][M][N]
  int split;
  int gx, gy, blocked;       // tiles, and whether the grid runs in blocks of 4 x 8
  int first, parts, n_tail;  // the last, incomplete round: its first block (tile), the parts of K its tiles are cut into (0: not this), its tiles
};

// Workgroups go to the 8 XCDs round-robin and an XCD runs 32 of them at a time; those 32 become a block of 4 tile rows x 8 tile columns,
// so that an XCD's L2 serves 12 operand panels for 32 tiles.  Grids of fewer than 256 such tiles, or of less than four rows, go row by
// row: blocks would leave XCDs idle.
struct tile_at {
  int tm, tn, z, parts, nth;  // which part of K, of how many; the tile's number in the last round
};
__device__ __forceinline__ bool tile_of_block(const gemm_args& g, unsigned block, unsigned pp, int& tm, int& tn) {
  const unsigned nbc = ((unsigned)g.gx + 7) / 8, row = block / nbc, col = block - row * nbc;
  tm = (int)(row * 4 + pp / 8);
  tn = (int)(col * 8 + pp % 8);
  return tm < g.gy && tn < g.gx;
}
__device__ __forceinline__ bool tile_of(const gemm_args& g, tile_at& at) {
  const unsigned L = blockIdx.x, cut = g.parts ? (unsigned)g.parts : 1u;
  at.parts = g.parts ? g.parts : g.split;
  if (!g.blocked) {
    const unsigned tile = g.first + L / cut;
    at.z = g.parts ? (int)(L % cut) : (int)blockIdx.y;
    at.nth = (int)(L / cut);
    at.tm = (int)(tile / g.gx);
    at.tn = (int)(tile % g.gx);
    return true;
  }
  const unsigned x = L & 7u, s8 = L >> 3, unit = (s8 >> 5) * 8u + x, pp = s8 & 31u;
  at.z = g.parts ? (int)(unit % cut) : (int)blockIdx.y;
  at.nth = (int)(unit / cut * 32 + pp);
  return tile_of_block(g, g.first + unit / cut, pp, at.tm, at.tn) && (g.parts == 0 || at.nth < g.n_tail);
}

__device__ __forceinline__ void dma16(const uint8_t* from, uint8_t* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

template <int N>
__device__ __forceinline__ void wait_loads_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");  // (my reads of the stage about to be refilled have landed)
  __builtin_amdgcn_s_barrier();  // bare: the fence of __syncthreads() would wait for every load in flight
  asm volatile("" ::: "memory");
}

// D = W fragment x A fragment: a lane holds four neighbouring columns n of one row m.
template <class OT, int BM, int BN, int TM, int TN, bool HALF = false>
__device__ __forceinline__ void store_tile(const gemm_args& g, const tile_at& at, f32x4 (&acc)[TM][TN], int wm, int wn, int lane) {
  const int m0 = at.tm * BM + wm * 16, n0 = at.tn * BN + wn * 16, z = at.z;
  if constexpr (HALF) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + j * 16 + (lane >> 4) * 4;
      const uint32_t top = n < g.N ? *(const uint32_t*)(g.w_top + n) : 0u;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = ldexpf(acc[i][j][e], (int)((top >> (8 * e)) & 255u) - 127 - HALF_TOP);
    }
  }
  if (g.parts) {  // (whole tiles: k_mxg_join_tail leaves out what lies beyond C)
    float* o = g.part + ((int64_t)z * g.n_tail + at.nth) * (BM * BN) + (wm * 16 + (lane & 15)) * BN + wn * 16 + (lane >> 4) * 4;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) *(f32x4*)(o + i * 16 * BN + j * 16) = acc[i][j];
    return;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + i * 16 + (lane & 15);
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + j * 16 + (lane >> 4) * 4;
      if (g.split > 1) {
        float* o = g.part + ((int64_t)z * g.M + m) * g.N + n;
        if (n + 4 <= g.N) {
          rp_vec<float, 4> t = {{acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]}};
          rp_store_vec<float, 4>(o, t);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < g.N) o[e] = acc[i][j][e];
        }
      } else {
        OT* o = (OT*)g.c + (int64_t)m * g.ldc + n;
        if (n + 4 <= g.N) {
          rp_vec<OT, 4> t;
#pragma unroll
          for (int e = 0; e < 4; ++e) t.v[e] = rp_from_f32<OT>(acc[i][j][e]);
          rp_store_vec<OT, 4>(o, t);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < g.N) o[e] = rp_from_f32<OT>(acc[i][j][e]);
        }
      }
    }
  }
}

// Everything a loop reads comes through LDS: a load into registers beside LDS-DMA requests makes the compiler wait for all of them.
// Fragments' rows and blocks past the matrices repeat the last ones: their sums are not stored, or meet zeros of A (bf16) or scales of
// 2^-127 (4-bit).

// 16-bit form.  Tile BM x BN, WM x WN waves.  A in a ring of three stages, each the half of a plane of a chunk (two of its four steps),
// requested two stages ahead; W's codes and scales in two slots, a chunk ahead, converted in registers once per plane and wave (4 conversions
// per 8 codes against TM matrix instructions that use them).  Bound by the matrix pipe as far as it is fed: 2048 x 20000 x 20000 f16 1.37 ms
// (1.2 PF, with preparing), bf16 1.4, f32 3.7 (three planes: 1.3 PF); a bf16 library product of that size takes 1.07 to 1.26 ms.
template <class OT, int P, bool HALF, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void k_mxg_bf16(gemm_args g) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, RING = 3;
  constexpr int STAGE = BM * 128, D = BM / 8 / WAVES;                // A: bytes of a stage, KB a wave requests of it
  constexpr int WCODES = BN * 64, DW = BN / 16 / WAVES;              // W: bytes of a slot, KB a wave requests of it
  constexpr int WSCALES = BN * 16, SLANES = BN / WAVES;              // scales: bytes of a slot, lanes of a wave's request
  constexpr int WOFF = RING * STAGE, SOFF = WOFF + 2 * WCODES, X = DW + 1;
  static_assert(D * WAVES * 8 == BM && DW * WAVES * 16 == BN && SLANES <= 64, "every wave requests the same number of pieces");
  extern __shared__ __attribute__((aligned(1024))) uint8_t ring[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  tile_at at;
  if (!tile_of(g, at)) return;
  const int tm = at.tm, tn = at.tn;
  const int m0 = tm * BM, wm = (wave / WN) * TM, wn = (wave % WN) * TN;  // (wm, wn in fragments of the tile)
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  const int c0 = (int)((int64_t)g.nc * at.z / at.parts), c1 = (int)((int64_t)g.nc * (at.z + 1) / at.parts);
  const int t0 = c0 * P * 2, t1 = c1 * P * 2;
  const int mblocks = (g.M + 15) / 16, nblocks = (g.N + 15) / 16;
  const uint8_t* asrc[D];
#pragma unroll
  for (int d = 0; d < D; ++d) {
    const int f = wave * D + d, mb = min(m0 / 16 + (f >> 1), mblocks - 1);
    asrc[d] = g.planes + ((int64_t)mb * g.nc * P) * 4096 + (f & 1) * 1024 + lane * 16;
  }
  auto request_a = [&](int t, int stage) __attribute__((always_inline)) {
    const int tt = min(t, t1 - 1);  // (past the end: the last one again, the counted waits stay uniform)
    uint8_t* to = ring + stage * STAGE + wave * D * 1024;
#pragma unroll
    for (int d = 0; d < D; ++d) dma16(asrc[d] + (int64_t)tt * 2048, to + d * 1024);
  };
  const uint8_t* wsrc[DW];
#pragma unroll
  for (int d = 0; d < DW; ++d) wsrc[d] = g.w + (int64_t)min(tn * BN + (wave * DW + d) * 16 + (lane & 15), g.N - 1) * g.ldw;
  const uint8_t* ssrc = (const uint8_t*)g.w_scales + (int64_t)min(tn * (BN / 16) + (wave * SLANES + lane) / 16, nblocks - 1) * g.nq * 256 + (lane & 15) * 16;
  auto request_w = [&](int c) __attribute__((always_inline)) {
    const int cc = min(c, c1 - 1), b = min(cc * 4 + (lane >> 4), g.nb - 1);
#pragma unroll
    for (int d = 0; d < DW; ++d) dma16(wsrc[d] + (int64_t)b * 16, ring + WOFF + (c & 1) * WCODES + (wave * DW + d) * 1024);
    if (SLANES == 64 || lane < SLANES) dma16(ssrc + (int64_t)(cc >> 2) * 256, ring + SOFF + (c & 1) * WSCALES + wave * SLANES * 16);
  };
  if (t0 < t1) {
    request_w(c0);
    request_a(t0, 0);
    request_a(t0 + 1, 1);
    int t = t0, stage = 0;
    i32x4 wq[TN];
    uint32_t sc[TN];
    for (int c = c0; c < c1; ++c) {
#pragma unroll(P < 3 ? P : 1)
      for (int pl = 0; pl < P; ++pl)
#pragma unroll
      for (int h = 0; h < 2; ++h, ++t) {
        const int s4 = pl * 2 + h;
        // newer than this stage: the next one, and the W requests if the step before made some
        if (s4 == 1) wait_loads_and_meet<D + X>();
        else wait_loads_and_meet<D>();
        if (s4 == 0) request_w(c + 1);
        request_a(t + 2, stage == 0 ? 2 : stage - 1);
        if (s4 == 0) {
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            wq[j] = *(const i32x4*)(ring + WOFF + (c & 1) * WCODES + (wn + j) * 1024 + lane * 16);
            sc[j] = ((*(const uint32_t*)(ring + SOFF + (c & 1) * WSCALES + (wn + j) * 256 + lane * 4) >> (8 * (c & 3))) & 255u) << 23;
          }
        }
        const uint8_t* st = ring + stage * STAGE + lane * 16;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          using frag = typename std::conditional<HALF, f16x8, bf16x8>::type;
          frag wf[TN];
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            if constexpr (HALF) wf[j] = codes_f16((uint32_t)wq[j][h * 2 + s], __uint_as_float(sc[j]));
            else wf[j] = codes_bf16((uint32_t)wq[j][h * 2 + s], __uint_as_float(sc[j]));
          }
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const frag af = *(const frag*)(st + ((wm + i) * 2 + s) * 1024);
#pragma unroll
            for (int j = 0; j < TN; ++j) {
              if constexpr (HALF) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[j], af, acc[i][j], 0, 0, 0);
              else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[j], af, acc[i][j], 0, 0, 0);
            }
          }
        }
        stage = stage == 2 ? 0 : stage + 1;
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the trailing requests write LDS)
  }
  store_tile<OT, BM, BN, TM, TN, HALF>(g, at, acc, wm, wn, lane);
}

// 4-bit form: codes of both operands in two slots, a stage (two chunks of both) ahead; scales in two slots of four chunks.  A piece is
// eight rows of 128 bytes: 64 bytes a row and chunk fetched every cache line twice (1.16 -> 0.98 ms at 4096 x 20000 x 20000).  Bound by
// how little its two halves overlap: two normal matrices, quantised, 4096 x 20000 x 20000 take 917 us with the scales' packing; without the
// requests, so matrix instructions and the reads of LDS alone, 726; requests and reads without matrix instructions 668; every stage from one
// panel that stays in the L2 827.  The matrix pipe is busy in half of the cycles: a stage's requests are waited for completely, one stage after they were made.
// (128 x 256 tiles three stages deep, half again the bytes: 17 % slower.)
template <class OT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void k_mxg_fp4(gemm_args g) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int STAGE = (BM + BN) * 128, D = (BM + BN) / 8 / WAVES;
  constexpr int SCALES = (BM + BN) * 16, SLANES = (BM + BN) / WAVES, SOFF = 2 * STAGE;
  static_assert(D * WAVES * 8 == BM + BN && SLANES <= 64, "every wave requests the same number of pieces");
  extern __shared__ __attribute__((aligned(1024))) uint8_t ring[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  tile_at at;
  if (!tile_of(g, at)) return;
  const int tm = at.tm, tn = at.tn;
  const int wm = (wave / WN) * TM, wn = (wave % WN) * TN;  // (in fragments of the tile)
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  const int q0 = (int)((int64_t)g.nq * at.z / at.parts), q1 = (int)((int64_t)g.nq * (at.z + 1) / at.parts);
  const int s0 = q0 * 2, s1 = min(q1 * 2, (g.nc + 1) / 2);  // stages: two chunks
  const int mblocks = (g.M + 15) / 16, nblocks = (g.N + 15) / 16;
  // a piece: 8 rows x 128 bytes; row r's block j of the stage lies at j ^ (r & 7)
  const int pr = lane >> 3, pj = (lane & 7) ^ pr;
  const uint8_t* src[D];
#pragma unroll
  for (int d = 0; d < D; ++d) {
    const int f = wave * D + d;
    src[d] = f < BM / 8 ? g.a_codes + (int64_t)min(tm * BM + f * 8 + pr, g.M - 1) * g.lda : g.w + (int64_t)min(tn * BN + (f - BM / 8) * 8 + pr, g.N - 1) * g.ldw;
  }
  auto request = [&](int s) __attribute__((always_inline)) {
    const int b = min(min(s, s1 - 1) * 8 + pj, g.nb - 1);
    uint8_t* to = ring + (s & 1) * STAGE + wave * D * 1024;
#pragma unroll
    for (int d = 0; d < D; ++d) dma16(src[d] + (int64_t)b * 16, to + d * 1024);
  };
  const int sf = (wave * SLANES + lane) / 16;  // the fragment whose scales this lane requests
  const uint8_t* ssrc = (sf < BM / 16 ? (const uint8_t*)g.a_scales + (int64_t)min(tm * (BM / 16) + sf, mblocks - 1) * g.nq * 256
                                      : (const uint8_t*)g.w_scales + (int64_t)min(tn * (BN / 16) + sf - BM / 16, nblocks - 1) * g.nq * 256) + (lane & 15) * 16;
  auto request_scales = [&](int q) __attribute__((always_inline)) {
    if (SLANES == 64 || lane < SLANES) dma16(ssrc + (int64_t)min(q, q1 - 1) * 256, ring + SOFF + (q & 1) * SCALES + wave * SLANES * 16);
  };
  if (s0 < s1) {
    request_scales(q0);
    request(s0);
    int sc[TM + TN];
    const int fr = lane & 15, fg = lane >> 4;
    const uint8_t* rd = ring + fr * 128;
    for (int q = q0; q < q1; ++q) {
      auto stage = [&](auto tag, int s) __attribute__((always_inline)) {
        constexpr int H = decltype(tag)::value;
        wait_loads_and_meet<0>();
        if (H == 0) request_scales(q + 1);
        request(s + 1);
        if (H == 0) {
          const uint8_t* ss = ring + SOFF + (q & 1) * SCALES + lane * 4;
#pragma unroll
          for (int i = 0; i < TM; ++i) sc[i] = *(const int*)(ss + (wm + i) * 256);
#pragma unroll
          for (int j = 0; j < TN; ++j) sc[TM + j] = *(const int*)(ss + (BM / 16 + wn + j) * 256);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint8_t* st = rd + H * STAGE + (((p * 4 + fg) ^ (fr & 7)) * 16);
          i32x8 wf[TN];
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const i32x4 v = *(const i32x4*)(st + (BM / 16 + wn + j) * 2048);
            wf[j] = i32x8{v.x, v.y, v.z, v.w, 0, 0, 0, 0};
          }
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const i32x4 v = *(const i32x4*)(st + (wm + i) * 2048);
            const i32x8 af = {v.x, v.y, v.z, v.w, 0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < TN; ++j) {
              if (p == 0) acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], af, acc[i][j], 4, 4, H * 2, sc[TM + j], H * 2, sc[i]);
              else acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[j], af, acc[i][j], 4, 4, H * 2 + 1, sc[TM + j], H * 2 + 1, sc[i]);
            }
          }
        }
      };
      stage(std::integral_constant<int, 0>{}, q * 2);
      if (q * 2 + 1 < s1) stage(std::integral_constant<int, 1>{}, q * 2 + 1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the trailing requests write LDS)
  }
  store_tile<OT, BM, BN, TM, TN>(g, at, acc, wm, wn, lane);
}

// ---- few rows of A -------------------------------------------------------------------------------------------------------------------
// M <= 4: every element of W is wanted M times, so its bytes are the time, and the vector unit keeps up: half a conversion and M
// multiply-adds in float32 per element (no planes, no workspace).  A wave takes GV_ROWS rows of W at once, a lane every 64th MX block of
// them: 1 KB contiguous per row and step.  The four waves of a workgroup share A's 2048 elements of a step in LDS as float32, in
// the order [16 bytes of a block][block]: a lane reads its block without bank conflicts (from memory, 64 - 128 bytes apart, these reads
// took longer than W: 80 us instead of 48 at 1 x 20000 x 20000 in f32).  Bound by W's bytes: 45 us, 4.7 TB/s.
constexpr int GV_ROWS = 4;
template <class T, class OT, int M>
__global__ __launch_bounds__(256) void k_mxg_rows(const T* __restrict__ a, int64_t lda, int m_real, int N, int K, int nb, const uint8_t* __restrict__ w, int64_t ldw,
                                                  const uint8_t* __restrict__ ws, int64_t ldws, OT* __restrict__ c, int64_t ldc) {
  __shared__ f32x4 sa[M][8 * 64];
  const int lane = threadIdx.x & 63;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * GV_ROWS;
  const uint8_t* wr[GV_ROWS];
  const uint8_t* sr[GV_ROWS];
#pragma unroll
  for (int r = 0; r < GV_ROWS; ++r) {
    const int64_t n = min(n0 + r, (int64_t)N - 1);
    wr[r] = w + n * ldw;
    sr[r] = ws + n * ldws;
  }
  float acc[GV_ROWS][M];
#pragma unroll
  for (int r = 0; r < GV_ROWS; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) acc[r][m] = 0.0f;
  uint4 q[GV_ROWS], qn[GV_ROWS];
  uint32_t s[GV_ROWS], sn[GV_ROWS];
  auto fetch = [&](int b) __attribute__((always_inline)) {
    const int bb = min(b, nb - 1);  // (a block beyond the row: A is zero there, the scale 2^-127: no infinity meets a zero)
#pragma unroll
    for (int r = 0; r < GV_ROWS; ++r) {
      qn[r] = *(const uint4*)(wr[r] + (int64_t)bb * 16);
      sn[r] = b < nb ? sr[r][bb] : 0u;
    }
  };
  rp_vec<T, 8> an[M];  // this thread's eight elements of the next step
  auto fetch_a = [&](int b0) __attribute__((always_inline)) {
    const int64_t k = (int64_t)b0 * RP_MX + threadIdx.x * 8;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const T* p = a + (int64_t)min(m, m_real - 1) * lda + k;
      if (k + 8 <= K) an[m] = rp_load_vec<T, 8>(p);
      else {
#pragma unroll
        for (int i = 0; i < 8; ++i) an[m].v[i] = k + i < K ? p[i] : (T)0.0f;
      }
    }
  };
  fetch(lane);
  fetch_a(0);
  for (int b0 = 0; b0 < nb; b0 += 64) {
    __syncthreads();
    const int at = (threadIdx.x & 3) * 2 * 64 + (threadIdx.x >> 2);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      sa[m][at] = f32x4{rp_to_f32(an[m].v[0]), rp_to_f32(an[m].v[1]), rp_to_f32(an[m].v[2]), rp_to_f32(an[m].v[3])};
      sa[m][at + 64] = f32x4{rp_to_f32(an[m].v[4]), rp_to_f32(an[m].v[5]), rp_to_f32(an[m].v[6]), rp_to_f32(an[m].v[7])};
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < GV_ROWS; ++r) q[r] = qn[r], s[r] = sn[r];
    fetch(b0 + 64 + lane);
    fetch_a(b0 + 64);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 v[M][2];
#pragma unroll
      for (int m = 0; m < M; ++m) v[m][0] = sa[m][g * 128 + lane], v[m][1] = sa[m][g * 128 + 64 + lane];
#pragma unroll
      for (int r = 0; r < GV_ROWS; ++r) {
        float x[8];
        rp_mx_unpack8(g == 0 ? q[r].x : g == 1 ? q[r].y : g == 2 ? q[r].z : q[r].w, rp_mx_scale(s[r]), x);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[r][m] = fmaf(v[m][i >> 2][i & 3], x[i], acc[r][m]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < GV_ROWS; ++r)
#pragma unroll
    for (int m = 0; m < M; ++m) {
      float t = acc[r][m];
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) t += __shfl_xor(t, d);
      if (lane == 0 && n0 + r < N && m < m_real) c[(int64_t)m * ldc + n0 + r] = rp_from_f32<OT>(t);
    }
}

// ---- small products ------------------------------------------------------------------------------------------------------------------
// One launch, no workspace: a workgroup takes 16 x 64 of C (4-bit A: 32 x 32), its eight waves every eighth chunk of K each, operands from memory into registers
// as a lane hands them to the matrix instruction (A cut or its scales taken there), a chunk ahead; the waves' sums are joined in LDS
// in wave order.  A is read once per tile column and W once per tile row, so this is for products whose time is launches and latency:
// 97 x 1999 x 2003 in f32 12 us, three launches of the tiles' form 20.
constexpr int SD_WAVES = 8;
constexpr int sd_tm(int planes) { return planes ? 1 : 2; }  // (cutting A is most of the work: 16 rows of A to 64 of W)
constexpr int sd_tn(int planes) { return planes ? 4 : 2; }

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void swap16(uint32_t& x, uint32_t& y) {
  const u32x2 r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
  x = r.x, y = r.y;
}
__device__ __forceinline__ void swap32(uint32_t& x, uint32_t& y) {
  const u32x2 r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = r.x, y = r.y;
}
// eight elements to planes; one with an infinity or a NaN among them (in any lane) the careful way
template <int P>
__device__ __forceinline__ void cut8(const float (&v)[8], bf16x8 (&out)[P]) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) << 1);
  i32x4 q[P];
  if (__any(top >= 0xff000000u)) {
    uint16_t h[8][P];
#pragma unroll
    for (int e = 0; e < 8; ++e) cut_planes<P>(v[e], h[e]);
#pragma unroll
    for (int pl = 0; pl < P; ++pl)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[pl][e] = (int)(h[2 * e][pl] | (uint32_t)h[2 * e + 1][pl] << 16);
  } else {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = v[e];
#pragma unroll
    for (int pl = 0; pl < P; ++pl) {
#pragma unroll
      for (int e = 0; e < 4; ++e) q[pl][e] = (int)__builtin_amdgcn_perm(__float_as_uint(r[2 * e + 1]), __float_as_uint(r[2 * e]), 0x07060302u);  // (the high halves)
      if (pl + 1 < P) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] -= __uint_as_float(__float_as_uint(r[e]) & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int pl = 0; pl < P; ++pl) out[pl] = __builtin_bit_cast(bf16x8, q[pl]);
}
template <class T, class OT, int P>
__global__ __launch_bounds__(64 * SD_WAVES) void k_mxg_direct(const T* __restrict__ a, int64_t lda, const uint8_t* __restrict__ as, int64_t ldas, int M, int N, int K, int nb,
                                                              const uint8_t* __restrict__ w, int64_t ldw, const uint8_t* __restrict__ ws, int64_t ldws, OT* __restrict__ c,
                                                              int64_t ldc, const uint16_t* __restrict__ wide) {
  constexpr int TM = sd_tm(P), TN = sd_tn(P);
  __shared__ f32x4 part[SD_WAVES][TM * TN][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), fr = lane & 15, fg = lane >> 4;
  const int n0 = (int)blockIdx.x * TN * 16, nc = (nb + 3) / 4;
  if (wide) {  // (f16 A, after the product: only columns that f16 does not hold; the others of their tiles stay as they are)
    bool any = false;
#pragma unroll
    for (int j = 0; j < TN; ++j) any = any || (n0 + j * 16 < N && wide[n0 / 16 + j] != 0);
    if (!any) return;
  }
  for (int m0 = (int)blockIdx.y * TM * 16; m0 < M; m0 += (int)gridDim.y * TM * 16) {
    const T* ap[TM];
    const uint8_t* asp[TM];
    const uint8_t* wp[TN];
    const uint8_t* wsp[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {  // (rows past the matrices: the last one again; not stored)
      const int64_t m = min(m0 + i * 16 + fr, M - 1);
      ap[i] = a + m * lda;
      if (P == 0) asp[i] = as + m * ldas;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t n = min(n0 + j * 16 + fr, N - 1);
      wp[j] = w + n * ldw;
      wsp[j] = ws + n * ldws;
    }
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
    rp_vec<T, 8> av[2][TM][P > 0 ? 4 : 1];
    uint4 aq[2][TM], wq[2][TN];
    uint32_t sa[2][TM], sw[2][TN];
    auto fetch = [&](auto tag, int ch) __attribute__((always_inline)) {
      constexpr int S = decltype(tag)::value;
      const int b = ch * 4 + fg, bb = min(b, nb - 1);  // (a block past the row: scale 2^-127 meets zeros of A, or its like)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        wq[S][j] = *(const uint4*)(wp[j] + (int64_t)bb * 16);
        sw[S][j] = b < nb ? wsp[j][bb] : 0u;
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if constexpr (P == 0) {
          aq[S][i] = *(const uint4*)(ap[i] + (int64_t)bb * 16);
          sa[S][i] = b < nb ? asp[i][bb] : 0u;
        } else {
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int64_t k = (int64_t)ch * KC + s * 32 + fg * 8;
            if (k + 8 <= K) av[S][i][s] = rp_load_vec<T, 8>(ap[i] + k);
            else {
#pragma unroll
              for (int e = 0; e < 8; ++e) av[S][i][s].v[e] = k + e < K ? ap[i][k + e] : (T)0.0f;
            }
          }
        }
      }
    };
    auto add = [&](auto tag) __attribute__((always_inline)) {
      constexpr int S = decltype(tag)::value;
      if constexpr (P == 0) {
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const i32x8 wf = {(int)wq[S][j].x, (int)wq[S][j].y, (int)wq[S][j].z, (int)wq[S][j].w, 0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const i32x8 af = {(int)aq[S][i].x, (int)aq[S][i].y, (int)aq[S][i].z, (int)aq[S][i].w, 0, 0, 0, 0};
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, af, acc[i][j], 4, 4, 0, (int)sw[S][j], 0, (int)sa[S][i]);
          }
        }
      } else {
        // step s takes the elements 32 s + 8 g .. of the chunk (A's loads then share lines): of W, dword g of block s, which lane group s holds
        uint32_t wd[TN][4], sc[TN][4];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          wd[j][0] = wq[S][j].x, wd[j][1] = wq[S][j].y, wd[j][2] = wq[S][j].z, wd[j][3] = wq[S][j].w;
          swap16(wd[j][0], wd[j][1]);
          swap16(wd[j][2], wd[j][3]);
          swap32(wd[j][0], wd[j][2]);
          swap32(wd[j][1], wd[j][3]);
          sc[j][0] = sc[j][1] = sw[S][j] << 23;
          swap16(sc[j][0], sc[j][1]);
          sc[j][2] = sc[j][0], sc[j][3] = sc[j][1];
          swap32(sc[j][0], sc[j][2]);
          swap32(sc[j][1], sc[j][3]);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          bf16x8 wf[TN];
#pragma unroll
          for (int j = 0; j < TN; ++j) wf[j] = codes_bf16(wd[j][s], __uint_as_float(sc[j][s]));
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = rp_to_f32(av[S][i][s].v[e]);
            bf16x8 af[P];
            cut8<P>(v, af);
#pragma unroll
            for (int pl = 0; pl < P; ++pl)
#pragma unroll
              for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[j], af[pl], acc[i][j], 0, 0, 0);
          }
        }
      }
    };
    using set0 = std::integral_constant<int, 0>;
    using set1 = std::integral_constant<int, 1>;
    int ch = wave;
    if (ch < nc) {
      fetch(set0{}, ch);
      for (; ch < nc; ch += 2 * SD_WAVES) {
        fetch(set1{}, min(ch + SD_WAVES, nc - 1));
        add(set0{});
        if (ch + SD_WAVES >= nc) break;
        fetch(set0{}, min(ch + 2 * SD_WAVES, nc - 1));
        add(set1{});
      }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) part[wave][i * TN + j][lane] = acc[i][j];
    __syncthreads();
    // a lane holds four neighbouring columns n of one row m
    const int m = m0 + wave / TN * 16 + fr, n = n0 + wave % TN * 16 + fg * 4;
    if (wave < TM * TN && m < M) {
      f32x4 t = part[0][wave][lane];
#pragma unroll
      for (int q = 1; q < SD_WAVES; ++q) t += part[q][wave][lane];
      OT* o = c + (int64_t)m * ldc + n;
      const uint32_t mine = wide ? (n < N ? (uint32_t)wide[n >> 4] >> (n & 15) : 0u) & 15u : 15u;
      if (n + 4 <= N && mine == 15u) {
        rp_vec<OT, 4> v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v.v[e] = rp_from_f32<OT>(t[e]);
        rp_store_vec<OT, 4>(o, v);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < N && ((mine >> e) & 1)) o[e] = rp_from_f32<OT>(t[e]);
      }
    }
    __syncthreads();
  }
}

// split K: the parts in order, one rounding
template <class OT>
__global__ __launch_bounds__(256) void k_mxg_join(const float* __restrict__ part, int split, int M, int N, OT* __restrict__ c, int64_t ldc) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)M * N) return;
  float s = 0.0f;
  for (int z = 0; z < split; ++z) s += part[(int64_t)z * M * N + i];
  c[i / N * ldc + i % N] = rp_from_f32<OT>(s);
}

// the last round's tiles: the parts in order, one rounding
template <class OT, int BM, int BN>
__global__ __launch_bounds__(256) void k_mxg_join_tail(gemm_args g) {
  int tm, tn;
  const int nth = blockIdx.x;
  if (g.blocked) {
    if (!tile_of_block(g, (unsigned)(g.first + nth / 32), (unsigned)nth & 31u, tm, tn)) return;
  } else {
    tm = (g.first + nth) / g.gx, tn = (g.first + nth) % g.gx;
  }
  const int i = (int)blockIdx.y * 256 + threadIdx.x, m = tm * BM + i / (BN / 4), n = tn * BN + i % (BN / 4) * 4;
  if (m >= g.M || n >= g.N) return;
  f32x4 t = f32x4{0, 0, 0, 0};
  for (int z = 0; z < g.parts; ++z) t += *(const f32x4*)(g.part + ((int64_t)z * g.n_tail + nth) * (BM * BN) + (int64_t)i * 4);
  OT* o = (OT*)g.c + (int64_t)m * g.ldc + n;
  if (n + 4 <= g.N) {
    rp_vec<OT, 4> v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v.v[e] = rp_from_f32<OT>(t[e]);
    rp_store_vec<OT, 4>(o, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < g.N) o[e] = rp_from_f32<OT>(t[e]);
  }
}

struct plan {
  int planes = 0, split = 1, nc = 0, nq = 0;
  bool rows = false;    // few rows of A: k_mxg_rows
  bool direct = false;  // small: k_mxg_direct
  bool half = false;    // f16 A as it is
  int first = 0, parts = 0, n_tail = 0;  // the last round of tiles (gemm_args)
  int bm = 16, bn = 64;
  int64_t plane_bytes = 0, a_scale_bytes = 0, w_scale_bytes = 0, top_bytes = 0, wide_bytes = 0, part_bytes = 0;
  int64_t total() const { return plane_bytes + a_scale_bytes + w_scale_bytes + top_bytes + wide_bytes + part_bytes; }
};

struct tile_grid {
  int gx, gy;
  bool blocked;
  int64_t blocks, tiles;
};
tile_grid grid_of(int64_t M, int64_t N, int bm, int bn) {
  tile_grid t;
  t.gx = (int)rp_cdiv(N, bn), t.gy = (int)rp_cdiv(M, bm);
  t.tiles = (int64_t)t.gx * t.gy;
  t.blocked = t.gy >= 4 && t.tiles >= 256;
  t.blocks = rp_cdiv(t.gx, 8) * rp_cdiv(t.gy, 4);
  return t;
}

// Tiles of one workgroup to a CU: an incomplete round of them behind complete ones is cut along K, as often as it leaves CUs idle
// (bf16 1500 x 12000 x 12000 538 -> 445 us; f16 2048 x 20000 x 20000, two and a half rounds: 1.71 -> 1.51 ms).  hundredths: the rounds' time.
struct last_round {
  int first, parts, n_tail;
  int64_t hundredths;
};
last_round last_round_of(int n_cu, const tile_grid& t, int nc) {
  const int64_t units = t.blocked ? t.blocks : t.tiles, round = t.blocked ? std::max(n_cu / 32, 1) : n_cu, rest = units % round;
  const int64_t parts = rest && units > round ? std::max<int64_t>(1, std::min<int64_t>({round / rest, nc / 16, 8})) : 1;
  return {(int)(units - rest), (int)parts, (int)(t.blocked ? rest * 32 : rest), units / round * 100 + (rest ? 100 / parts : 0)};
}

// Which tile, and into how many parts K is split: by rounds of workgroups over the CUs.  Measured on W of 20000 x 20000 unless said.
plan make_plan(int n_cu, int64_t M, int64_t N, int64_t K, int32_t a_type) {
  plan p;
  p.planes = a_type == RPHIP_BF16 || a_type == RPHIP_F16 ? 1 : a_type == RPHIP_F32 ? 3 : 0;
  p.half = a_type == RPHIP_F16;
  p.nc = (int)rp_cdiv(K, KC);
  p.nq = (int)rp_cdiv(p.nc, 4);
  // the vector unit's form: f32 99 us against 118 at M = 4, 16 bits 73 against 91 (bf16) and 108 (f16) at M = 2 (but 108 against 90 and 106 against 107
  // at 3)
  p.rows = p.planes != 0 && M <= (p.planes == 3 ? 4 : 2) && K > 0;
  if (p.rows) return p;
  // small products, by tiles and by what a tile's latency comes to: f32 97 x 1999 x 2003 13.7 us against 20.2, bf16 256 x 2000 x 2000 16.5
  // against 17.6; but bf16 64 x 2000 x 8000 26 against 21, 128 x 4000 x 4000 32 against 22, 1000 x 1000 x 1000 29 against 18.  4-bit (with
  // A's quantising): 1000 x 1000 x 1000 24 against 28, 16 x 16000 x 8000 25 against 28; but 300 x 8000 x 1000 41 against 27.
  const int64_t small = rp_cdiv(M, 16 * sd_tm(p.planes)) * rp_cdiv(N, 16 * sd_tn(p.planes)), latency = small * (p.nc + 8);
  p.direct = K > 0 && (p.planes ? small <= 2 * n_cu && p.nc <= 32 && latency <= 48 * n_cu : p.nc <= 128 && latency <= 140 * n_cu);
  if (p.direct) return p;
  auto tiles = [&](int bm, int bn) { return std::max<int64_t>(rp_cdiv(M, bm) * rp_cdiv(N, bn), 1); };
  auto rounds = [&](int bm, int bn, int per_cu) { return rp_cdiv(tiles(bm, bn), per_cu * n_cu); };
  auto hundredths = [&](int bm, int bn) { return last_round_of(n_cu, grid_of(M, N, bm, bn), p.nc).hundredths; };
  if (p.planes) {
    const int64_t steps = (int64_t)p.nc * p.planes * 2;
    int per_cu = 1;  // workgroups a CU should see when K is split: small tiles wait for memory together
    if (M <= 16) {
      p.bm = 16, p.bn = 64, per_cu = 5;
    } else if (M > 128 && tiles(128, 256) >= n_cu) {
      // a 128 x 256 tile takes 0.57 of a 256 x 256 one (527 and 302 us a round); three planes do not fit the larger one's registers
      p.bn = 256;
      p.bm = p.planes == 3 || hundredths(128, 256) * 57 < hundredths(256, 256) * 100 ? 128 : 256;
    } else if (M > 64 && tiles(128, 128) * steps >= 40000) {
      p.bm = 128, p.bn = 128, per_cu = 5;  // (bf16, M = 128: 160 us in eight parts, 202 with 64 x 64 tiles; 1000 x 3000 x 3000, 64 x 64: 37)
    } else {
      p.bm = 64, p.bn = 64, per_cu = 4;
    }
    const int64_t n = tiles(p.bm, p.bn);
    // (a part of fewer than 24 steps costs more to join than it saves: 500 x 2000 x 2000 in f16 24 us whole, 28 in four parts)
    p.split = (int)std::max<int64_t>(1, std::min<int64_t>({(per_cu * (int64_t)n_cu + n / 2) / n, steps / 24, 16}));
  } else {
    // a round of 64 x 64 tiles (four a CU), 128 x 128 (two), 256 x 256 (one) takes 34, 45, 58 us at K = 8000
    const int64_t t64 = rounds(64, 64, 4) * 58, t128 = rounds(128, 128, 2) * 76, t256 = hundredths(256, 256);
    p.bm = M <= 32 ? 32 : t64 <= t128 && t64 <= t256 ? 64 : t128 <= t256 ? 128 : 256;
    p.bn = p.bm;
    const int64_t n = tiles(p.bm, p.bn);
    p.split = (int)std::max<int64_t>(1, std::min<int64_t>({(n_cu + n / 2) / n, p.nq / 8, 16}));
  }
  auto room = [](int64_t b) { return (b + 255) & ~(int64_t)255; };
  p.plane_bytes = room(rp_cdiv(M, 16) * p.nc * p.planes * 4096);
  p.a_scale_bytes = p.planes ? 0 : room(rp_cdiv(M, 16) * p.nq * 256);
  p.w_scale_bytes = room(rp_cdiv(N, 16) * p.nq * 256);
  p.top_bytes = p.half ? room(rp_cdiv(N, 16) * 16) : 0;
  p.wide_bytes = p.half ? room(rp_cdiv(N, 16) * 2) : 0;
  p.part_bytes = p.split > 1 ? M * N * 4 * p.split : 0;
  if (p.split == 1 && p.bn == 256) {
    const last_round l = last_round_of(n_cu, grid_of(M, N, p.bm, p.bn), p.nc);
    if (l.parts > 1) {
      p.first = l.first, p.parts = l.parts, p.n_tail = l.n_tail;
      p.part_bytes = (int64_t)p.parts * p.n_tail * p.bm * p.bn * 4;
    }
  }
  return p;
}

template <class OT, int BM, int BN, class Kernel>
int launch_tiles(Kernel kernel, gemm_args g, int threads, int lds, hipStream_t st) {
  const tile_grid t = grid_of(g.M, g.N, BM, BN);
  g.gx = t.gx, g.gy = t.gy, g.blocked = t.blocked;
  auto workgroups = [&](int64_t units) { return t.blocked ? rp_cdiv(units, 8) * 8 * 32 : units; };
  const gemm_args tail = g;
  const int64_t units = t.blocked ? t.blocks : t.tiles, whole = g.parts ? g.first : units;
  if (workgroups(units) * threads >= ((int64_t)1 << 32)) RP_FAIL(RPHIP_ELIMIT, "mxfp4_gemm_nt: %d x %d is more than a launch takes", g.M, g.N);
  if (lds > 64 * 1024) RP_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  g.first = g.parts = 0;
  kernel<<<dim3((unsigned)workgroups(whole), (unsigned)g.split), threads, lds, st>>>(g);
  RP_LAUNCHED();
  if constexpr (BN == 256) {
    if (tail.parts) {
      kernel<<<(unsigned)workgroups((units - whole) * tail.parts), threads, lds, st>>>(tail);
      RP_LAUNCHED();
      k_mxg_join_tail<OT, BM, BN><<<dim3((unsigned)tail.n_tail, BM * BN / 4 / 256), 256, 0, st>>>(tail);
      RP_LAUNCHED();
    }
  }
  return RPHIP_OK;
}
template <class OT, int BM, int BN, int WM, int WN>
int launch_fp4(const gemm_args& g, hipStream_t st) {
  return launch_tiles<OT, BM, BN>(k_mxg_fp4<OT, BM, BN, WM, WN>, g, WM * WN * 64, 2 * (BM + BN) * 128 + 2 * (BM + BN) * 16, st);
}
template <class OT, int BM, int BN, int WM, int WN>
int launch_bf16(const gemm_args& g, int planes, bool half, hipStream_t st) {
  constexpr int threads = WM * WN * 64, lds = 3 * BM * 128 + 2 * BN * 64 + 2 * BN * 16;
  if (half) return launch_tiles<OT, BM, BN>(k_mxg_bf16<OT, 1, true, BM, BN, WM, WN>, g, threads, lds, st);
  if (planes == 1) return launch_tiles<OT, BM, BN>(k_mxg_bf16<OT, 1, false, BM, BN, WM, WN>, g, threads, lds, st);
  if constexpr (BM * BN < 256 * 256) return launch_tiles<OT, BM, BN>(k_mxg_bf16<OT, 3, false, BM, BN, WM, WN>, g, threads, lds, st);
  RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt: no such tile");
}

int check_sizes(const char* who, int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0 || N > INT32_MAX || K > INT32_MAX) RP_FAIL(RPHIP_EINVAL, "%s: %lld x %lld x %lld", who, (long long)M, (long long)N, (long long)K);
  if (N > ((int64_t)1 << 28)) RP_FAIL(RPHIP_ELIMIT, "%s: at most 2^28 rows of W in a call, got %lld", who, (long long)N);
  if (M > 65535 * 16) RP_FAIL(RPHIP_ELIMIT, "%s: at most %d rows of A in a call, got %lld", who, 65535 * 16, (long long)M);
  return RPHIP_OK;
}

}  // namespace

extern "C" int rphip_mxfp4_gemm_nt_workspace(rphip_ctx* ctx, int64_t M, int64_t N, int64_t K, int32_t a_type, int64_t* bytes_out) {
  if (!ctx || !bytes_out) RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt_workspace: NULL argument");
  RP_TRY(check_sizes("mxfp4_gemm_nt_workspace", M, N, K));
  if (a_type < RPHIP_F32 || a_type > RPHIP_MXFP4) RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt_workspace: element type %d", a_type);
  const plan p = make_plan(ctx->n_cu, M, N, K, a_type);
  *bytes_out = p.total();
  return RPHIP_OK;
}

extern "C" int rphip_mxfp4_gemm_nt(rphip_ctx* ctx, void* stream, int64_t M, int64_t N, int64_t K, const void* A_dev, int32_t a_type, int64_t lda,
                                   const uint8_t* a_scales_dev, int64_t ld_a_scales, const uint8_t* w_codes_dev, int64_t ld_w, const uint8_t* w_scales_dev,
                                   int64_t ld_w_scales, void* C_dev, int32_t c_type, int64_t ldc, void* workspace_dev, int64_t workspace_bytes) {
  rp_op_scope scope;
  RP_TRY(check_sizes("mxfp4_gemm_nt", M, N, K));
  if (a_type < RPHIP_F32 || a_type > RPHIP_MXFP4) RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt: element type %d of A", a_type);
  if (c_type < RPHIP_F32 || c_type > RPHIP_BF16) RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt: element type %d of C", c_type);
  RP_TRY(rp_mx_check("mxfp4_gemm_nt (W)", N, K, w_codes_dev, ld_w, w_scales_dev, ld_w_scales));
  if (a_type == RPHIP_MXFP4) RP_TRY(rp_mx_check("mxfp4_gemm_nt (A)", M, K, (const uint8_t*)A_dev, lda, a_scales_dev, ld_a_scales));
  if (M == 0 || N == 0) return RPHIP_OK;
  if (!C_dev || (K > 0 && !A_dev)) RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt: NULL argument");
  if (a_type != RPHIP_MXFP4 && (lda < K || (uintptr_t)A_dev % rp_type_bytes(a_type))) RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt: lda < K, or A is not aligned to its elements");
  if (ldc < N || (uintptr_t)C_dev % rp_type_bytes(c_type)) RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt: ldc < N, or C is not aligned to its elements");
  RP_TRY(scope.enter(ctx));
  const plan p = make_plan(ctx->n_cu, M, N, K, a_type);
  if (workspace_bytes < p.total() || (p.total() > 0 && !workspace_dev) || ((uintptr_t)workspace_dev & 255))
    RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt: a workspace of %lld bytes, aligned to 256, is needed (rphip_mxfp4_gemm_nt_workspace)", (long long)p.total());
  const hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)workspace_dev;
  gemm_args g = {};
  g.M = (int)M, g.N = (int)N, g.nb = (int)rp_cdiv(K, RP_MX), g.nc = p.nc, g.nq = p.nq;
  g.planes = (const uint8_t*)ws;
  g.a_codes = (const uint8_t*)A_dev, g.lda = lda, g.a_scales = (const uint32_t*)(ws + p.plane_bytes);
  g.w = w_codes_dev, g.ldw = ld_w, g.w_scales = (const uint32_t*)(ws + p.plane_bytes + p.a_scale_bytes);
  uint8_t* top = (uint8_t*)ws + p.plane_bytes + p.a_scale_bytes + p.w_scale_bytes;
  uint16_t* wide = (uint16_t*)(top + p.top_bytes);
  g.w_top = top;
  g.c = C_dev, g.ldc = ldc, g.part = (float*)((char*)wide + p.wide_bytes), g.split = p.split;
  g.first = p.first, g.parts = p.parts, g.n_tail = p.n_tail;
  if (p.rows)
    return rp_by_type(a_type, [&](auto at) -> int {
      return rp_by_type(c_type, [&](auto ct) -> int {
        using T = typename decltype(at)::T;
        using OT = typename decltype(ct)::T;
        auto go = [&](auto kernel) -> int {
          for (int64_t n0 = 0; n0 < N; n0 += (int64_t)1 << 27) {  // (a launch takes less than 2^32 threads)
            const int n = (int)std::min<int64_t>(N - n0, (int64_t)1 << 27);
            kernel<<<(unsigned)rp_cdiv(n, 4 * GV_ROWS), 256, 0, st>>>((const T*)A_dev, lda, (int)M, n, (int)K, g.nb, w_codes_dev + n0 * ld_w, ld_w,
                                                                      w_scales_dev + n0 * ld_w_scales, ld_w_scales, (OT*)C_dev + n0, ldc);
            RP_LAUNCHED();
          }
          return RPHIP_OK;
        };
        return M == 1 ? go(k_mxg_rows<T, OT, 1>) : M == 2 ? go(k_mxg_rows<T, OT, 2>) : go(k_mxg_rows<T, OT, 4>);
      });
    });
  // the direct form: the whole product, or (wide) what f16 did not hold
  auto direct = [&](auto kernel, auto type, auto out, int planes, const uint16_t* flags) -> int {
    const unsigned gx = (unsigned)rp_cdiv(N, 16 * sd_tn(planes)), gy = (unsigned)rp_cdiv(M, 16 * sd_tm(planes));
    kernel<<<dim3(gx, flags ? std::min(gy, 16u) : gy), 64 * SD_WAVES, 0, st>>>((const decltype(type)*)A_dev, lda, a_scales_dev, ld_a_scales, (int)M, (int)N, (int)K, g.nb, w_codes_dev,
                                                                               ld_w, w_scales_dev, ld_w_scales, (decltype(out)*)C_dev, ldc, flags);
    RP_LAUNCHED();
    return RPHIP_OK;
  };
  if (p.direct)
    return rp_by_type(c_type, [&](auto ct) -> int {
      using OT = typename decltype(ct)::T;
      if (a_type == RPHIP_BF16) return direct(k_mxg_direct<__bf16, OT, 1>, __bf16{}, OT{}, 1, nullptr);
      if (a_type == RPHIP_F16) return direct(k_mxg_direct<_Float16, OT, 2>, _Float16{}, OT{}, 2, nullptr);
      if (a_type == RPHIP_F32) return direct(k_mxg_direct<float, OT, 3>, 0.0f, OT{}, 3, nullptr);
      return direct(k_mxg_direct<uint8_t, OT, 0>, uint8_t{0}, OT{}, 0, nullptr);
    });
  if (p.nc) {
    const int64_t w_units = rp_cdiv(N, 16) * p.nq * 64, wg_w = p.half ? rp_cdiv(N, 16) : rp_cdiv(w_units, 256);
    const int64_t a_units = p.planes ? rp_cdiv(M, 16) * p.nc : rp_cdiv(M, 16) * p.nq * 64, wg_a = p.planes ? a_units : rp_cdiv(a_units, 256);
    auto go = [&](auto kernel, auto type, const void* a, int64_t ld, void* o) -> int {
      using T = decltype(type);
      for (int64_t wg0 = 0; wg0 < wg_w + wg_a; wg0 += (int64_t)1 << 23) {
        kernel<<<(unsigned)std::min<int64_t>(wg_w + wg_a - wg0, (int64_t)1 << 23), 256, 0, st>>>(w_scales_dev, ld_w_scales, (int)N, g.nb, p.nq, w_units, (uint32_t*)g.w_scales, wg0,
                                                                                               wg_w, (const T*)a, ld, (int)M, (int)K, p.nc, a_units, o,
                                                                                               half_args{w_codes_dev, ld_w, top, wide});
        RP_LAUNCHED();
      }
      return RPHIP_OK;
    };
    if (a_type == RPHIP_BF16) RP_TRY(go(k_mxg_prepare<__bf16, 1>, __bf16{}, A_dev, lda, (void*)g.planes));
    else if (a_type == RPHIP_F16) RP_TRY(go(k_mxg_prepare<_Float16, 1>, _Float16{}, A_dev, lda, (void*)g.planes));
    else if (a_type == RPHIP_F32) RP_TRY(go(k_mxg_prepare<float, 3>, 0.0f, A_dev, lda, (void*)g.planes));
    else RP_TRY(go(k_mxg_prepare<uint8_t, 0>, uint8_t{0}, a_scales_dev, ld_a_scales, (void*)g.a_scales));
  }
  return rp_by_type(c_type, [&](auto tag) -> int {
    using OT = typename decltype(tag)::T;
    if (p.planes == 0) {
      if (p.bm == 32) RP_TRY((launch_fp4<OT, 32, 32, 1, 2>(g, st)));
      else if (p.bm == 64) RP_TRY((launch_fp4<OT, 64, 64, 2, 2>(g, st)));
      else if (p.bm == 128) RP_TRY((launch_fp4<OT, 128, 128, 2, 2>(g, st)));
      else RP_TRY((launch_fp4<OT, 256, 256, 2, 4>(g, st)));
    } else {
      if (p.bm == 16) RP_TRY((launch_bf16<OT, 16, 64, 1, 2>(g, p.planes, p.half, st)));
      else if (p.bm == 64) RP_TRY((launch_bf16<OT, 64, 64, 2, 2>(g, p.planes, p.half, st)));
      else if (p.bm == 128 && p.bn == 128) RP_TRY((launch_bf16<OT, 128, 128, 2, 2>(g, p.planes, p.half, st)));
      else if (p.bm == 128) RP_TRY((launch_bf16<OT, 128, 256, 2, 4>(g, p.planes, p.half, st)));
      else RP_TRY((launch_bf16<OT, 256, 256, 2, 4>(g, p.planes, p.half, st)));
    }
    if (p.split > 1) {
      k_mxg_join<OT><<<(unsigned)rp_cdiv(M * N, 256), 256, 0, st>>>(g.part, p.split, g.M, g.N, (OT*)C_dev, ldc);
      RP_LAUNCHED();
    }
    if (p.half && p.nc) return direct(k_mxg_direct<_Float16, OT, 2>, _Float16{}, OT{}, 2, wide);
    return RPHIP_OK;
  });
}
