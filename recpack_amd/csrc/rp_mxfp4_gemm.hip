// C[M,N] = A[M,K] W[N,K]^T with W in MXFP4 (one scale per 32 along K) and A in f32 / f16 / bf16, or MXFP4 as well.  f32 accumulate.
// C ABI: include/recpack_hip.h, rphip_mxfp4_gemm_nt.
//
// 16- and 32-bit A: every element of W is a bf16 number exactly (two significant bits times a power of two), and every element of A a
// sum of one (bf16), two (f16: 8 + 3 bits) or three (f32: 8 + 8 + 8 bits) of them, so the product runs on v_mfma_f32_16x16x32_bf16
// with exact operands; the planes of A are cut once into a workspace, W is converted in registers.
// MXFP4 A: v_mfma_scale_f32_16x16x128_f8f6f4, which takes codes and scales as they are.
#include "rp_ops.h"

#include <algorithm>

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int KC = 128;  // K of a chunk: four MX blocks

// ---- A as planes of bf16: [row][chunk][plane][128], zero beyond K --------------------------------------------------------------------
// by truncation: the high part never overflows, each remainder is exact
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

template <class T, int P>
__global__ __launch_bounds__(256) void k_mxg_planes(const T* __restrict__ a, int64_t lda, int M, int K, int nc, uint16_t* __restrict__ out) {
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x;  // eight elements
  const int upr = nc * (KC / 8);
  const int64_t m = unit / upr;
  if (m >= M) return;
  const int q = (int)(unit - m * upr), k = q * 8;
  const T* p = a + m * lda + k;
  float v[8];
  if (k + 8 <= K) {
    const rp_vec<T, 8> t = rp_load_vec<T, 8>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = rp_to_f32(t.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? rp_to_f32(p[i]) : 0.0f;
  }
  uint16_t h[8][P];
#pragma unroll
  for (int i = 0; i < 8; ++i) cut_planes<P>(v[i], h[i]);
  uint16_t* o = out + (m * nc + q / (KC / 8)) * (P * KC) + (q % (KC / 8)) * 8;
#pragma unroll
  for (int pl = 0; pl < P; ++pl) {
    uint4 w;
    w.x = h[0][pl] | (uint32_t)h[1][pl] << 16;
    w.y = h[2][pl] | (uint32_t)h[3][pl] << 16;
    w.z = h[4][pl] | (uint32_t)h[5][pl] << 16;
    w.w = h[6][pl] | (uint32_t)h[7][pl] << 16;
    *(uint4*)(o + pl * KC) = w;
  }
}

// eight codes (a dword) to eight bf16
__device__ __forceinline__ bf16x8 codes_bf16(uint32_t w, float s) {
  rp_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1);
  rp_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3);
  bf16x8 r = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
  return r;
}

struct gemm_args {
  int M, N, nb, nc;          // nb: blocks of a row of W (and of an MXFP4 A), nc: chunks
  const uint16_t* planes;    // 16-bit form of A
  const uint8_t* a_codes; int64_t lda; const uint8_t* a_scales; int64_t ldas;  // MXFP4 A
  const uint8_t* w; int64_t ldw; const uint8_t* ws; int64_t ldws;
  void* c; int64_t ldc;
  float* part;               // split K: partial sums [split][M][N]
  int split;
};

// Tile BM x BN, WM x WN waves.  The lane (l & 15, l >> 4) = (row, g) of a fragment holds block 4 c + g of its row; K runs in the order
// (step s, g, 8 elements) inside a chunk - the same for both operands, which is all a product asks - so a lane's 16 code bytes are
// one MX block with one scale.
template <class OT, int P, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void k_mxg_bf16(gemm_args g) {
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16, THREADS = WM * WN * 64;
  __shared__ uint4 tile[BM * 16];  // one plane of a chunk: row r's 16-byte piece j at j ^ (r & 15)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fg = lane >> 4;
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
  const int wm = (wave / WN) * TM * 16, wn = (wave % WN) * TN * 16;
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  const int c_begin = (int)((int64_t)g.nc * blockIdx.z / g.split), c_end = (int)((int64_t)g.nc * (blockIdx.z + 1) / g.split);
  for (int c = c_begin; c < c_end; ++c) {
    uint4 wq[TN];
    float wsc[TN];
    const int b = c * 4 + fg;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = min(n0 + wn + j * 16 + fr, g.N - 1);
      wq[j] = make_uint4(0, 0, 0, 0);
      uint32_t byte = 127;
      if (b < g.nb) {
        wq[j] = *(const uint4*)(g.w + (int64_t)n * g.ldw + (int64_t)b * 16);
        byte = g.ws[(int64_t)n * g.ldws + b];
      }
      wsc[j] = rp_mx_scale(byte);
    }
    for (int p = 0; p < P; ++p) {
      __syncthreads();
      for (int q = threadIdx.x; q < BM * 16; q += THREADS) {
        const int r = q >> 4, j = q & 15, m = min(m0 + r, g.M - 1);
        tile[r * 16 + (j ^ (r & 15))] = *(const uint4*)(g.planes + (((int64_t)m * g.nc + c) * P + p) * KC + j * 8);
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        bf16x8 wf[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) wf[j] = codes_bf16(s == 0 ? wq[j].x : s == 1 ? wq[j].y : s == 2 ? wq[j].z : wq[j].w, wsc[j]);
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          const int r = wm + i * 16 + fr;
          const bf16x8 af = __builtin_bit_cast(bf16x8, tile[r * 16 + ((fg * 4 + s) ^ (r & 15))]);
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, wf[j], acc[i][j], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + wm + i * 16 + fg * 4 + e, n = n0 + wn + j * 16 + fr;
        if (m >= g.M || n >= g.N) continue;
        if (g.split > 1) g.part[((int64_t)blockIdx.z * g.M + m) * g.N + n] = acc[i][j][e];
        else ((OT*)g.c)[(int64_t)m * g.ldc + n] = rp_from_f32<OT>(acc[i][j][e]);
      }
}

template <class OT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64) void k_mxg_fp4(gemm_args g) {
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int fr = lane & 15, fg = lane >> 4;
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
  const int wm = (wave / WN) * TM * 16, wn = (wave % WN) * TN * 16;
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0, 0, 0, 0};
  const int c_begin = (int)((int64_t)g.nc * blockIdx.z / g.split), c_end = (int)((int64_t)g.nc * (blockIdx.z + 1) / g.split);
  for (int c = c_begin; c < c_end; ++c) {
    const int b = c * 4 + fg;
    uint4 aq[TM], wq[TN];
    int as[TM], wsc[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = min(m0 + wm + i * 16 + fr, g.M - 1);
      aq[i] = make_uint4(0, 0, 0, 0);
      as[i] = 127;
      if (b < g.nb) aq[i] = *(const uint4*)(g.a_codes + (int64_t)m * g.lda + (int64_t)b * 16), as[i] = g.a_scales[(int64_t)m * g.ldas + b];
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = min(n0 + wn + j * 16 + fr, g.N - 1);
      wq[j] = make_uint4(0, 0, 0, 0);
      wsc[j] = 127;
      if (b < g.nb) wq[j] = *(const uint4*)(g.w + (int64_t)n * g.ldw + (int64_t)b * 16), wsc[j] = g.ws[(int64_t)n * g.ldws + b];
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const i32x8 af = {(int)aq[i].x, (int)aq[i].y, (int)aq[i].z, (int)aq[i].w, 0, 0, 0, 0};
        const i32x8 wf = {(int)wq[j].x, (int)wq[j].y, (int)wq[j].z, (int)wq[j].w, 0, 0, 0, 0};
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(af, wf, acc[i][j], 4, 4, 0, as[i], 0, wsc[j]);
      }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + wm + i * 16 + fg * 4 + e, n = n0 + wn + j * 16 + fr;
        if (m >= g.M || n >= g.N) continue;
        if (g.split > 1) g.part[((int64_t)blockIdx.z * g.M + m) * g.N + n] = acc[i][j][e];
        else ((OT*)g.c)[(int64_t)m * g.ldc + n] = rp_from_f32<OT>(acc[i][j][e]);
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

struct plan {
  int planes = 0, split = 1;
  int bm = 16, bn = 64;
  int64_t plane_bytes = 0, part_bytes = 0;
  int nc = 0;
};

plan make_plan(int n_cu, int64_t M, int64_t N, int64_t K, int32_t a_type) {
  plan p;
  p.planes = a_type == RPHIP_BF16 ? 1 : a_type == RPHIP_F16 ? 2 : a_type == RPHIP_F32 ? 3 : 0;
  p.nc = (int)rp_cdiv(K, KC);
  p.bm = M <= 16 ? 16 : M <= 256 ? 64 : 128;
  p.bn = p.bm == 128 ? 128 : 64;
  const int64_t tiles = rp_cdiv(M, p.bm) * rp_cdiv(N, p.bn);
  p.split = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(2 * n_cu / std::max<int64_t>(tiles, 1), p.nc / 4), 32));
  p.plane_bytes = (M * p.nc * p.planes * KC * 2 + 255) & ~(int64_t)255;
  p.part_bytes = p.split > 1 ? M * N * 4 * p.split : 0;
  return p;
}

template <class OT, int BM, int BN, int WM, int WN>
void launch_tiles(const gemm_args& g, int planes, hipStream_t st) {
  const dim3 grid((unsigned)rp_cdiv(g.N, BN), (unsigned)rp_cdiv(g.M, BM), (unsigned)g.split);
  const int threads = WM * WN * 64;
  if (planes == 0) k_mxg_fp4<OT, BM, BN, WM, WN><<<grid, threads, 0, st>>>(g);
  else if (planes == 1) k_mxg_bf16<OT, 1, BM, BN, WM, WN><<<grid, threads, 0, st>>>(g);
  else if (planes == 2) k_mxg_bf16<OT, 2, BM, BN, WM, WN><<<grid, threads, 0, st>>>(g);
  else k_mxg_bf16<OT, 3, BM, BN, WM, WN><<<grid, threads, 0, st>>>(g);
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
  *bytes_out = p.plane_bytes + p.part_bytes;
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
  if (workspace_bytes < p.plane_bytes + p.part_bytes || (p.plane_bytes + p.part_bytes > 0 && !workspace_dev) || ((uintptr_t)workspace_dev & 255))
    RP_FAIL(RPHIP_EINVAL, "mxfp4_gemm_nt: a workspace of %lld bytes, aligned to 256, is needed (rphip_mxfp4_gemm_nt_workspace)", (long long)(p.plane_bytes + p.part_bytes));
  const hipStream_t st = (hipStream_t)stream;
  gemm_args g = {};
  g.M = (int)M, g.N = (int)N, g.nb = (int)rp_cdiv(K, RP_MX), g.nc = p.nc;
  g.planes = (const uint16_t*)workspace_dev;
  g.a_codes = (const uint8_t*)A_dev, g.lda = lda, g.a_scales = a_scales_dev, g.ldas = ld_a_scales;
  g.w = w_codes_dev, g.ldw = ld_w, g.ws = w_scales_dev, g.ldws = ld_w_scales;
  g.c = C_dev, g.ldc = ldc, g.part = (float*)((char*)workspace_dev + p.plane_bytes), g.split = p.split;
  if (p.planes && p.nc) {
    const int64_t strip = std::max<int64_t>(1, ((int64_t)1 << 31) / ((int64_t)p.nc * (KC / 8)));  // rows of a launch of below 2^32 threads
    for (int64_t m0 = 0; m0 < M; m0 += strip) {
      const int m = (int)std::min(strip, M - m0);
      const unsigned grid = (unsigned)rp_cdiv((int64_t)m * p.nc * (KC / 8), 256);
      uint16_t* o = (uint16_t*)workspace_dev + m0 * p.nc * p.planes * KC;
      if (a_type == RPHIP_BF16) k_mxg_planes<__bf16, 1><<<grid, 256, 0, st>>>((const __bf16*)A_dev + m0 * lda, lda, m, (int)K, p.nc, o);
      else if (a_type == RPHIP_F16) k_mxg_planes<_Float16, 2><<<grid, 256, 0, st>>>((const _Float16*)A_dev + m0 * lda, lda, m, (int)K, p.nc, o);
      else k_mxg_planes<float, 3><<<grid, 256, 0, st>>>((const float*)A_dev + m0 * lda, lda, m, (int)K, p.nc, o);
      RP_LAUNCHED();
    }
  }
  return rp_by_type(c_type, [&](auto tag) -> int {
    using OT = typename decltype(tag)::T;
    if (p.bm == 16) launch_tiles<OT, 16, 64, 1, 4>(g, p.planes, st);
    else if (p.bm == 64) launch_tiles<OT, 64, 64, 2, 2>(g, p.planes, st);
    else launch_tiles<OT, 128, 128, 2, 2>(g, p.planes, st);
    RP_LAUNCHED();
    if (p.split > 1) {
      k_mxg_join<OT><<<(unsigned)rp_cdiv(M * N, 256), 256, 0, st>>>(g.part, p.split, g.M, g.N, (OT*)C_dev, ldc);
      RP_LAUNCHED();
    }
    return RPHIP_OK;
  });
}
