// MXFP4 matrices (microscaled 4-bit floating point): quantisation of rows or columns, reading back, and the scores of histories
// against a quantised item-item matrix.  C ABI: include/recpack_hip.h, section "4-bit matrices".
#include "rp_ops.h"

#include <algorithm>
#include <type_traits>

int rp_mx_check(const char* who, int64_t rows, int64_t cols, const uint8_t* codes, int64_t ld_codes, const uint8_t* scales, int64_t ld_scales) {
  const int64_t nb = rp_cdiv(cols, RP_MX);
  if (rows < 0 || cols < 0 || rows > INT32_MAX || cols > INT32_MAX) RP_FAIL(RPHIP_EINVAL, "%s: %lld x %lld is no matrix size", who, (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return RPHIP_OK;
  if (!codes || !scales) RP_FAIL(RPHIP_EINVAL, "%s: NULL codes or scales", who);
  if (((uintptr_t)codes & 15) || (ld_codes & 15)) RP_FAIL(RPHIP_EINVAL, "%s: codes and their leading dimension must be multiples of 16 bytes", who);
  if (ld_codes < nb * 16 || ld_scales < nb)
    RP_FAIL(RPHIP_EINVAL, "%s: leading dimensions %lld / %lld bytes are too small for %lld columns (%lld blocks)", who, (long long)ld_codes, (long long)ld_scales,
            (long long)cols, (long long)nb);
  return RPHIP_OK;
}

// ---- quantise --------------------------------------------------------------------------------------------------------------------
// Four lanes per block of 32, eight elements each: the block's largest magnitude is two exchanges inside the quad.  Bound by HBM
// (4 or 2 bytes read, 0.53 written per element): 4096 x 20000 in f32 70 us, 5.3 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_mx_quantize(const T* __restrict__ x, int64_t ldx, int rows, int cols, int nb, uint8_t* __restrict__ codes,
                                                     int64_t ldc, uint8_t* __restrict__ scales, int64_t lds) {
  const int upr = nb * 4;  // units (eight elements) of a row
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r64 = unit / upr;
  if (r64 >= rows) return;  // (upr is a multiple of 4: a quad leaves together)
  const int q = (int)(unit - r64 * upr);
  const T* p = x + r64 * ldx + (int64_t)q * 8;
  float v[8];
  if (q * 8 + 8 <= cols) {
    const rp_vec<T, 8> t = rp_load_vec<T, 8>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = rp_to_f32(t.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = q * 8 + i < cols ? rp_to_f32(p[i]) : 0.0f;
  }
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);  // as integers: NaN above Inf above every number
  a = max(a, (uint32_t)__shfl_xor((int)a, 1));
  a = max(a, (uint32_t)__shfl_xor((int)a, 2));
  const uint32_t byte = rp_mx_scale_byte(a);
  const uint32_t w = byte == 255u ? 0u : rp_mx_pack8(v, rp_mx_scale(byte));
  *(uint32_t*)(codes + r64 * ldc + (int64_t)q * 4) = w;
  if ((q & 3) == 0) scales[r64 * lds + (q >> 2)] = (uint8_t)byte;
}

// The transpose: out row = column of x, blocks down the rows.  A wave takes 32 rows x 64 columns (a lane: one column, its block in
// registers; loads of a row are contiguous over the lanes); eight waves take 256 rows, so that a line of 128 code bytes is written
// whole, through LDS (16-byte pieces scattered over the lines otherwise).  Bound by HBM: 20000 x 20000 in f32 395 us, 4.6 TB/s.
constexpr int MXT_WAVES = 8, MXT_COLS = 64, MXT_LD = MXT_WAVES * 4 + 1;  // (LDS words of a column, odd: conflict-free either way)
template <class T>
__global__ __launch_bounds__(MXT_WAVES * 64) void k_mx_quantize_t(const T* __restrict__ x, int64_t ldx, int rows, int cols, int nb, uint8_t* __restrict__ codes,
                                                                  int64_t ldc, uint8_t* __restrict__ scales, int64_t lds) {
  __shared__ uint32_t tile[MXT_COLS * MXT_LD];
  __shared__ uint8_t sbyte[MXT_COLS * MXT_WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b0 = blockIdx.y * MXT_WAVES;          // first block (of 32 rows)
  const int c0 = blockIdx.x * MXT_COLS, c = c0 + lane;
  const int r0 = (b0 + wave) * RP_MX;
  if (r0 < rows) {
    float v[32];
    const T* p = x + (int64_t)r0 * ldx + c;
    if (r0 + 32 <= rows && c < cols) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = rp_to_f32(p[i * ldx]);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = (r0 + i < rows && c < cols) ? rp_to_f32(p[i * ldx]) : 0.0f;
    }
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);
    const uint32_t byte = rp_mx_scale_byte(a);
    const float s = rp_mx_scale(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) tile[lane * MXT_LD + wave * 4 + i] = byte == 255u ? 0u : rp_mx_pack8(v + 8 * i, s);
    sbyte[lane * MXT_WAVES + wave] = (uint8_t)byte;
  }
  __syncthreads();
  // thread: one block (16 bytes) of one column, eight neighbouring lanes write one line
  const int col = threadIdx.x >> 3, b = threadIdx.x & 7;
  if (c0 + col < cols && b0 + b < nb) {
    uint4 w;
    w.x = tile[col * MXT_LD + b * 4];
    w.y = tile[col * MXT_LD + b * 4 + 1];
    w.z = tile[col * MXT_LD + b * 4 + 2];
    w.w = tile[col * MXT_LD + b * 4 + 3];
    *(uint4*)(codes + (int64_t)(c0 + col) * ldc + (int64_t)(b0 + b) * 16) = w;
    scales[(int64_t)(c0 + col) * lds + b0 + b] = sbyte[col * MXT_WAVES + b];
  }
}

static int mx_type_ok(const char* who, int32_t type) {
  if (type != RPHIP_F32 && type != RPHIP_F16 && type != RPHIP_BF16) RP_FAIL(RPHIP_EINVAL, "%s: element type %d: RPHIP_F32, RPHIP_F16 or RPHIP_BF16 expected", who, type);
  return RPHIP_OK;
}

extern "C" int rphip_mxfp4_quantize(rphip_ctx* ctx, void* stream, int64_t rows, int64_t cols, const void* x_dev, int32_t x_type, int64_t ldx, int32_t transpose,
                                    uint8_t* codes_dev, int64_t ld_codes, uint8_t* scales_dev, int64_t ld_scales) {
  rp_op_scope scope;
  RP_TRY(mx_type_ok("mxfp4_quantize", x_type));
  RP_TRY(rp_mx_check("mxfp4_quantize", transpose ? cols : rows, transpose ? rows : cols, codes_dev, ld_codes, scales_dev, ld_scales));
  if (rows == 0 || cols == 0) return RPHIP_OK;
  if (!x_dev) RP_FAIL(RPHIP_EINVAL, "mxfp4_quantize: x is NULL");
  if ((uintptr_t)x_dev % rp_type_bytes(x_type)) RP_FAIL(RPHIP_EINVAL, "mxfp4_quantize: x is not aligned to its elements");
  if (ldx < cols) RP_FAIL(RPHIP_EINVAL, "mxfp4_quantize: ldx %lld < cols %lld", (long long)ldx, (long long)cols);
  if (transpose && cols > ((int64_t)1 << 28)) RP_FAIL(RPHIP_ELIMIT, "mxfp4_quantize: the transpose takes at most 2^28 columns");
  RP_TRY(scope.enter(ctx));
  const int nb = (int)rp_cdiv(transpose ? rows : cols, RP_MX);
  return rp_by_type(x_type, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    if (transpose) {
      const int64_t gy = rp_cdiv(nb, MXT_WAVES), gx = rp_cdiv(cols, MXT_COLS);
      // (grid.y is 16 bits wide: 65 535 * 256 rows; larger inputs go in strips of rows)
      for (int64_t y0 = 0; y0 < gy; y0 += 65535) {
        const int64_t r0 = y0 * MXT_WAVES * RP_MX, b0 = y0 * MXT_WAVES;
        k_mx_quantize_t<T><<<dim3((unsigned)gx, (unsigned)std::min<int64_t>(gy - y0, 65535)), MXT_WAVES * 64, 0, (hipStream_t)stream>>>(
            (const T*)x_dev + r0 * ldx, ldx, (int)(rows - r0), (int)cols, (int)(nb - b0), codes_dev + b0 * 16, ld_codes, scales_dev + b0, ld_scales);
        RP_LAUNCHED();
      }
    } else {
      // strips of rows keep a launch below 2^32 threads
      const int64_t strip = std::max<int64_t>(1, ((int64_t)1 << 31) / ((int64_t)nb * 4));
      for (int64_t r0 = 0; r0 < rows; r0 += strip) {
        const int64_t n = std::min(strip, rows - r0);
        k_mx_quantize<T><<<(unsigned)rp_cdiv(n * nb * 4, 256), 256, 0, (hipStream_t)stream>>>((const T*)x_dev + r0 * ldx, ldx, (int)n, (int)cols, nb,
                                                                                            codes_dev + r0 * ld_codes, ld_codes, scales_dev + r0 * ld_scales, ld_scales);
        RP_LAUNCHED();
      }
    }
    return RPHIP_OK;
  });
}

// ---- reading back ------------------------------------------------------------------------------------------------------------------
// Eight elements to a lane: one dword of codes, one 32-byte (16-byte) store.  Bound by HBM: 20000 x 20000 to f32 350 us, 5.2 TB/s.
template <class T>
__global__ __launch_bounds__(256) void k_mx_dequantize(const uint8_t* __restrict__ codes, int64_t ldc, const uint8_t* __restrict__ scales, int64_t lds, int rows,
                                                       int cols, int upr, T* __restrict__ out, int64_t ldo) {
  const int64_t unit = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = unit / upr;
  if (r >= rows) return;
  const int q = (int)(unit - r * upr);
  const uint32_t w = *(const uint32_t*)(codes + r * ldc + (int64_t)q * 4);
  float v[8];
  rp_mx_unpack8(w, rp_mx_scale(scales[r * lds + (q >> 2)]), v);
  T* p = out + r * ldo + (int64_t)q * 8;
  if (q * 8 + 8 <= cols) {
    rp_vec<T, 8> t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t.v[i] = rp_from_f32<T>(v[i]);
    rp_store_vec<T, 8>(p, t);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (q * 8 + i < cols) p[i] = rp_from_f32<T>(v[i]);
  }
}

extern "C" int rphip_mxfp4_dequantize(rphip_ctx* ctx, void* stream, int64_t rows, int64_t cols, const uint8_t* codes_dev, int64_t ld_codes, const uint8_t* scales_dev,
                                      int64_t ld_scales, void* out_dev, int32_t out_type, int64_t ld_out) {
  rp_op_scope scope;
  RP_TRY(mx_type_ok("mxfp4_dequantize", out_type));
  RP_TRY(rp_mx_check("mxfp4_dequantize", rows, cols, codes_dev, ld_codes, scales_dev, ld_scales));
  if (rows == 0 || cols == 0) return RPHIP_OK;
  if (!out_dev) RP_FAIL(RPHIP_EINVAL, "mxfp4_dequantize: out is NULL");
  if ((uintptr_t)out_dev % rp_type_bytes(out_type)) RP_FAIL(RPHIP_EINVAL, "mxfp4_dequantize: out is not aligned to its elements");
  if (ld_out < cols) RP_FAIL(RPHIP_EINVAL, "mxfp4_dequantize: ld_out %lld < cols %lld", (long long)ld_out, (long long)cols);
  RP_TRY(scope.enter(ctx));
  const int upr = (int)rp_cdiv(cols, 8);
  return rp_by_type(out_type, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    const int64_t strip = std::max<int64_t>(1, ((int64_t)1 << 31) / upr);
    for (int64_t r0 = 0; r0 < rows; r0 += strip) {
      const int64_t n = std::min(strip, rows - r0);
      k_mx_dequantize<T><<<(unsigned)rp_cdiv(n * upr, 256), 256, 0, (hipStream_t)stream>>>(codes_dev + r0 * ld_codes, ld_codes, scales_dev + r0 * ld_scales, ld_scales,
                                                                                         (int)n, (int)cols, upr, (T*)out_dev + r0 * ld_out, ld_out);
      RP_LAUNCHED();
    }
    return RPHIP_OK;
  });
}

// ---- scores of histories -----------------------------------------------------------------------------------------------------------
// out[u, :] = sum over the entries e of user u of w_e * W[idx_e, :], in f32.  The rows of a history are contiguous and their blocks run along
// the output.  A workgroup of four waves takes (user, 2048 columns).  The order of the adds does not depend on the number of users: a user's
// scores are the same bits alone and in any batch.
constexpr int MXS_COLS = 64 * RP_MX, MXS_WAVES = 4;

// Which user and column tile.  Workgroups go to the 8 XCDs round-robin: while eight tiles are left each XCD takes one of them for all
// users, so that its L2 meets every history's pieces (1 KB) of the popular rows; the remaining tiles go through the XCDs together.
__device__ __forceinline__ void mxs_task(unsigned users, int tiles, unsigned& user, int& tile) {
  const unsigned L = blockIdx.x, full = (unsigned)tiles / 8 * 8;
  if (L < full * users) {
    const unsigned s = L >> 3;
    tile = (int)(s / users * 8 + (L & 7));
    user = s % users;
  } else {
    const unsigned s = L - full * users;
    tile = (int)(full + s / users);
    user = s % users;
  }
}

// what both forms share: the entries of a chunk of 64, those that count moved to the front, in order; the history's own columns
struct mxs_chunk {
  int idx, m;
  float wgt;
};
template <bool WEIGHTED>
__device__ __forceinline__ mxs_chunk mxs_load(const int32_t* __restrict__ indices, const float* __restrict__ weights, int64_t e0, int64_t e1, int lane) {
  mxs_chunk k = {-1, (int)min((int64_t)64, max(e1 - e0, (int64_t)0)), 0.0f};  // (m: entries)
  if (lane < k.m) {
    k.idx = indices[e0 + lane];
    if (WEIGHTED) k.wgt = weights[e0 + lane];
  }
  return k;
}
template <bool WEIGHTED>
__device__ __forceinline__ mxs_chunk mxs_entries(mxs_chunk k, int rows, bool mark, int c0, uint32_t* drop, int lane) {  // (m: entries that count)
  const int n = k.m;
  if ((unsigned)k.idx >= (unsigned)rows) k.idx = -1;
  if (mark && k.idx >= c0 && k.idx < c0 + MXS_COLS) atomicOr(&drop[(k.idx - c0) >> 5], 1u << (k.idx & 31));
  const unsigned long long good = __ballot(k.idx >= 0);
  k.m = (int)__popcll(good);
  if (k.m < n) {
    const int dst = k.idx >= 0 ? (int)__popcll(good & ((1ull << lane) - 1ull)) : 63;
    k.idx = __builtin_amdgcn_ds_permute(dst * 4, k.idx);
    if (WEIGHTED) k.wgt = __int_as_float(__builtin_amdgcn_ds_permute(dst * 4, __float_as_int(k.wgt)));
  }
  return k;
}

// Binary histories on the matrix pipe.  v_mfma_scale_f32_16x16x128 sums over K = 4 groups of 32, each with its own scale: the groups are four
// history rows, the 16 columns of its right operand 16 MX blocks of them as they lie in memory (lane (block, row): 16 bytes and a
// scale), its left operand a one per output row that picks one element of the 32.  Two such selections turn four rows' blocks into
// 16 x 32 sums without a conversion: 64 elements a cycle and SIMD against 5 - 7 converted and added in the vector unit.  The selection
// is laid out so that a lane ends with 8 neighbouring columns of its block.  A wave takes 512 of the 2048 columns and all entries, in their order, up to
// 64 under way together (one wave for all columns, eight entries under way: 64 histories of 100 against 20000 x 20000 29 us, 16 so).  Bound by the rows'
// bytes: 1024 histories of 50 against 50000 x 50000 230 us, where each row read once and the scores written take 177 at the rate of a copy (238 us with the tiles in any order, 257 with
// the sums in the vector unit).
typedef int mxs_i32x8 __attribute__((ext_vector_type(8)));
typedef int mxs_i32x4 __attribute__((ext_vector_type(4)));
template <class T>
__global__ __launch_bounds__(64 * MXS_WAVES) void k_mx_scores_sum(const int32_t* __restrict__ indptr, const int32_t* __restrict__ indices, int64_t nnz, int rows, int cols, int nb,
                                                              const uint8_t* __restrict__ codes, int64_t ldc, const uint8_t* __restrict__ scales, int64_t lds, int exclude,
                                                              const uint8_t* __restrict__ keep, T* __restrict__ out, int64_t ldo, int64_t user0, unsigned users, int tiles) {
  constexpr int STEPS = 8;  // groups of four entries: half a chunk
  __shared__ uint32_t drop[64];  // bit c of word l: column 32 l + c of the tile gets -inf
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fg = lane >> 4;
  unsigned user;
  int tile;
  mxs_task(users, tiles, user, tile);
  const int64_t u = user0 + user;
  const int b = tile * 64 + wave * 16 + fr;  // this lane's block
  if (wave == 0) drop[lane] = 0;
  __syncthreads();
  // left operand: output row q (this lane's fr) of half h picks element (q >> 2) * 8 + h * 4 + (q & 3) of every group's 32; code of 1.0: 2
  mxs_i32x8 pick[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int j = (fr >> 2) * 8 + h * 4 + (fr & 3);
#pragma unroll
    for (int w = 0; w < 8; ++w) pick[h][w] = w == j / 8 ? 2 << (j % 8 * 4) : 0;
  }
  rp_f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  const int64_t at = min(b, nb - 1);  // (past the row: the last one; not stored)
  const int64_t e1 = min((int64_t)indptr[u + 1], nnz);
  int64_t e0 = max((int64_t)indptr[u], (int64_t)0);
  mxs_chunk next = mxs_load<false>(indices, nullptr, e0, e1, lane);
  for (; e0 < e1; e0 += 64) {
    const mxs_chunk ch = mxs_entries<false>(next, rows, exclude && wave == 0, tile * MXS_COLS, drop, lane);
    next = mxs_load<false>(indices, nullptr, e0 + 64, e1, lane);
    mxs_i32x4 w[2][STEPS];
    int sc[2][STEPS];
    auto fetch = [&](auto tag, int k0) __attribute__((always_inline)) {  // entries k .. k + 3, one a lane group; past the end: zeros
      constexpr int S = decltype(tag)::value;
#pragma unroll
      for (int t = 0; t < STEPS; ++t) {
        const int k = k0 + t * 4;
        const int64_t row = __shfl(ch.idx, (k + fg) & 63);
        w[S][t] = mxs_i32x4{0, 0, 0, 0};
        sc[S][t] = 0;
        if (k + fg < ch.m) {
          w[S][t] = *(const mxs_i32x4*)(codes + row * ldc + at * 16);
          sc[S][t] = scales[row * lds + at];
        }
      }
    };
    auto add = [&](auto tag, int k0) __attribute__((always_inline)) {
      constexpr int S = decltype(tag)::value;
#pragma unroll
      for (int t = 0; t < STEPS; ++t) {
        if (k0 + t * 4 >= ch.m) break;
        const mxs_i32x8 v = {w[S][t].x, w[S][t].y, w[S][t].z, w[S][t].w, 0, 0, 0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(pick[h], v, acc[h], 4, 4, 0, 127, 0, sc[S][t]);
      }
    };
    using set0 = std::integral_constant<int, 0>;
    using set1 = std::integral_constant<int, 1>;
    if (ch.m > 0) {  // (both sets once; written without the loop they take more registers than four waves a SIMD leave)
      fetch(set0{}, 0);
      for (int k = 0; k < ch.m; k += 8 * STEPS) {
        fetch(set1{}, k + 4 * STEPS);
        add(set0{}, k);
        if (k + 8 * STEPS < ch.m) fetch(set0{}, k + 8 * STEPS);
        add(set1{}, k + 4 * STEPS);
      }
    }
  }
  __syncthreads();
  // lane (fr, fg): columns 8 fg .. 8 fg + 7 of its block
  if (b >= nb) return;
  const int c = b * RP_MX + fg * 8, left = min(8, cols - c);
  uint32_t gone = drop[wave * 16 + fr] >> (fg * 8);
  if (keep)
    for (int i = 0; i < left; ++i) gone |= keep[c + i] ? 0u : 1u << i;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (gone >> i) & 1 ? -INFINITY : acc[i >> 2][i & 3];
  T* p = out + u * ldo + c;
  if (left == 8) {
    rp_vec<T, 8> t;
#pragma unroll
    for (int i = 0; i < 8; ++i) t.v[i] = rp_from_f32<T>(v[i]);
    rp_store_vec<T, 8>(p, t);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = rp_from_f32<T>(v[i]);
  }
}

// Weighted histories in the vector unit: a lane owns one block of 32 columns of every row and keeps its 32 sums in registers, half a
// conversion and one multiply-add per element; four rows in flight while four are added.  (The matrix pipe would take five planes per weight.)
// The waves take groups of four entries in turn and add their sums up in wave order, however many users there are: waves that share the
// columns out instead convert as much and address four times as many rows (251 histories of 100 against 20000 x 20000: 72 us); one wave alone is
// a little faster where there are many users (1024 histories of 50 against 50000 x 50000: 257 us, 274 so), and sums in another order.
// Bound by the gathered pieces: 251 histories of 100 against 20000 x 20000 in bf16 48 us, 266 MB at 5.5 TB/s (117 MB of rows are different ones, but
// an XCD meets a row again when its L2 has long seen others).
template <class T>
__global__ __launch_bounds__(64 * MXS_WAVES) void k_mx_scores_weighted(const int32_t* __restrict__ indptr, const int32_t* __restrict__ indices, const float* __restrict__ weights,
                                                          int64_t nnz, int rows, int cols, int nb, const uint8_t* __restrict__ codes, int64_t ldc,
                                                          const uint8_t* __restrict__ scales, int64_t lds, int exclude, const uint8_t* __restrict__ keep,
                                                          T* __restrict__ out, int64_t ldo, int64_t user0, unsigned users, int tiles) {
  __shared__ uint32_t drop[64];  // bit c of word l: column 32 l + c of the tile gets -inf
  __shared__ float sums[MXS_WAVES * 32 * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  unsigned user;
  int tile;
  mxs_task(users, tiles, user, tile);
  const int64_t u = user0 + user;
  const int c0 = tile * MXS_COLS;
  const int b = min(tile * 64 + lane, nb - 1);  // this lane's block of columns (lanes beyond the row repeat the last one)
  if (wave == 0) drop[lane] = 0;
  __syncthreads();
  float acc[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.0f;
  const uint8_t* cbase = codes + (int64_t)b * 16;
  const uint8_t* sbase = scales + b;
  const int64_t e1 = min((int64_t)indptr[u + 1], nnz);
  int64_t e0 = max((int64_t)indptr[u], (int64_t)0);
  mxs_chunk next = mxs_load<true>(indices, weights, e0, e1, lane);
  for (; e0 < e1; e0 += 64) {
    const mxs_chunk ch = mxs_entries<true>(next, rows, exclude && wave == 0, c0, drop, lane);
    next = mxs_load<true>(indices, weights, e0 + 64, e1, lane);
    const int idx = ch.idx, m = ch.m;
    const float wgt = ch.wgt;
    uint4 w[2][4];
    uint32_t sc[2][4];
    auto fetch = [&](auto tag, int k) __attribute__((always_inline)) {  // rows k .. k + 3 (past the end: the last one again)
      constexpr int S = decltype(tag)::value;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = __builtin_amdgcn_readlane(idx, min(k + i, m - 1));
        w[S][i] = *(const uint4*)(cbase + row * ldc);
        sc[S][i] = sbase[row * lds];
      }
    };
    auto add = [&](auto tag, int k) __attribute__((always_inline)) {
      constexpr int S = decltype(tag)::value;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (k + i >= m) break;
        const float s = rp_mx_scale(sc[S][i]);
        const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wgt), k + i));
        const uint32_t q[4] = {w[S][i].x, w[S][i].y, w[S][i].z, w[S][i].w};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float v[8];
          rp_mx_unpack8(q[g], s, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[g * 8 + j] = fmaf(f, v[j], acc[g * 8 + j]);
        }
      }
    };
    constexpr int STEP = 4 * MXS_WAVES;
    int k = wave * 4;
    if (k < m) {
      fetch(std::integral_constant<int, 0>{}, k);
      for (; k < m; k += 2 * STEP) {
        fetch(std::integral_constant<int, 1>{}, k + STEP);
        add(std::integral_constant<int, 0>{}, k);
        fetch(std::integral_constant<int, 0>{}, k + 2 * STEP);
        add(std::integral_constant<int, 1>{}, k + STEP);
      }
    }
  }
  const bool mine = tile * 64 + lane < nb;
  const int c = b * RP_MX;
  const int left = min(RP_MX, cols - c);
  T* p = out + u * ldo + c;
  // a lane of wave w ends with the columns [w * PC, (w + 1) * PC) of its block
  constexpr int PC = 32 / MXS_WAVES;
#pragma unroll
  for (int i = 0; i < 32; ++i) sums[(wave * 32 + i) * 64 + lane] = acc[i];
  __syncthreads();
  if (!mine) return;
  const uint32_t gone = drop[lane];
  float v[PC];
#pragma unroll
  for (int i = 0; i < PC; ++i) {
    const int col = wave * PC + i;
    v[i] = 0.0f;
#pragma unroll
    for (int o = 0; o < MXS_WAVES; ++o) v[i] += sums[(o * 32 + col) * 64 + lane];
    if (((gone >> col) & 1) || (keep && col < left && !keep[c + col])) v[i] = -INFINITY;
  }
  if (left == RP_MX) {
    rp_vec<T, PC> t;
#pragma unroll
    for (int i = 0; i < PC; ++i) t.v[i] = rp_from_f32<T>(v[i]);
    rp_store_vec<T, PC>(p + wave * PC, t);
  } else {
#pragma unroll
    for (int i = 0; i < PC; ++i)
      if (wave * PC + i < left) p[wave * PC + i] = rp_from_f32<T>(v[i]);
  }
}

extern "C" int rphip_mxfp4_scores(rphip_ctx* ctx, void* stream, int64_t n_users, int64_t nnz, const int32_t* indptr_dev, const int32_t* indices_dev,
                                  const float* weights_dev, int64_t rows, int64_t cols, const uint8_t* codes_dev, int64_t ld_codes, const uint8_t* scales_dev,
                                  int64_t ld_scales, int32_t exclude_history, const uint8_t* item_keep_dev, void* out_dev, int32_t out_type, int64_t ld_out) {
  rp_op_scope scope;
  RP_TRY(mx_type_ok("mxfp4_scores", out_type));
  if (n_users < 0 || nnz < 0 || n_users > INT32_MAX - 1 || nnz > INT32_MAX) RP_FAIL(RPHIP_EINVAL, "mxfp4_scores: %lld users, %lld entries", (long long)n_users, (long long)nnz);
  RP_TRY(rp_mx_check("mxfp4_scores", rows, cols, codes_dev, ld_codes, scales_dev, ld_scales));
  if (exclude_history && rows != cols) RP_FAIL(RPHIP_EINVAL, "mxfp4_scores: exclude_history needs a square matrix, got %lld x %lld", (long long)rows, (long long)cols);
  if (n_users == 0 || cols == 0) return RPHIP_OK;
  if (!indptr_dev || !out_dev || (nnz > 0 && !indices_dev)) RP_FAIL(RPHIP_EINVAL, "mxfp4_scores: NULL argument");
  if ((uintptr_t)out_dev % rp_type_bytes(out_type)) RP_FAIL(RPHIP_EINVAL, "mxfp4_scores: out is not aligned to its elements");
  if (ld_out < cols) RP_FAIL(RPHIP_EINVAL, "mxfp4_scores: ld_out %lld < cols %lld", (long long)ld_out, (long long)cols);
  RP_TRY(scope.enter(ctx));
  const int nb = (int)rp_cdiv(cols, RP_MX);
  const int64_t tiles = rp_cdiv(nb, 64);
  if (tiles > 65535) RP_FAIL(RPHIP_ELIMIT, "mxfp4_scores: at most %d columns", 65535 * MXS_COLS);
  return rp_by_type(out_type, [&](auto tag) -> int {
    using T = typename decltype(tag)::T;
    const hipStream_t st = (hipStream_t)stream;
    const int64_t strip = std::max<int64_t>(1, ((int64_t)1 << 22) / tiles);  // (users of a launch: below 2^32 threads)
    for (int64_t u0 = 0; u0 < n_users; u0 += strip) {
      const unsigned users = (unsigned)std::min(strip, n_users - u0), grid = users * (unsigned)tiles;
      if (weights_dev)
        k_mx_scores_weighted<T><<<grid, 64 * MXS_WAVES, 0, st>>>(indptr_dev, indices_dev, weights_dev, nnz, (int)rows, (int)cols, nb, codes_dev, ld_codes, scales_dev, ld_scales,
                                                                 exclude_history, item_keep_dev, (T*)out_dev, ld_out, u0, users, (int)tiles);
      else
        k_mx_scores_sum<T><<<grid, 64 * MXS_WAVES, 0, st>>>(indptr_dev, indices_dev, nnz, (int)rows, (int)cols, nb, codes_dev, ld_codes, scales_dev, ld_scales, exclude_history,
                                                            item_keep_dev, (T*)out_dev, ld_out, u0, users, (int)tiles);
      RP_LAUNCHED();
    }
    return RPHIP_OK;
  });
}
