// Shared by the dense operators on caller-owned device arrays (rp_mxfp4.hip, rp_mxfp4_gemm.hip, rp_sample.hip): element types, the
// guard of an entry point, unaligned vector loads, the MXFP4 conversions.
#pragma once

#include "rp_common.h"

// Entry guard: the context's lock and its device for the duration of the call, the caller's current device afterwards (these entry
// points are called beside torch, whose current device they must not move).
struct rp_op_scope {
  std::unique_lock<std::recursive_mutex> lock;
  int prev = -1, device = -1;
  int enter(rphip_ctx* ctx) {
    if (!ctx) RP_FAIL(RPHIP_EINVAL, "ctx is NULL");
    lock = std::unique_lock<std::recursive_mutex>(ctx->api_mu);
    RP_HIP(hipGetDevice(&prev));
    device = ctx->device;
    if (prev != device) RP_HIP(hipSetDevice(device));
    return RPHIP_OK;
  }
  ~rp_op_scope() {
    if (prev >= 0 && prev != device) hipSetDevice(prev);
  }
};

#define RP_LAUNCHED() RP_HIP(hipGetLastError())

// dispatch on an element type of the header: fn is a generic lambda taking a value of the type's tag
struct rp_f32 { using T = float; static constexpr int bytes = 4; };
struct rp_f16 { using T = _Float16; static constexpr int bytes = 2; };
struct rp_bf16 { using T = __bf16; static constexpr int bytes = 2; };
template <class F>
static inline int rp_by_type(int32_t type, F&& fn) {
  switch (type) {
    case RPHIP_F32: return fn(rp_f32{});
    case RPHIP_F16: return fn(rp_f16{});
    case RPHIP_BF16: return fn(rp_bf16{});
  }
  RP_FAIL(RPHIP_EINVAL, "element type %d: RPHIP_F32, RPHIP_F16 or RPHIP_BF16 expected", type);
}
static inline int rp_type_bytes(int32_t type) { return type == RPHIP_F32 ? 4 : 2; }

template <class T> __device__ __forceinline__ float rp_to_f32(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T rp_from_f32(float v) { return (T)v; }  // round to nearest even (one rounding)

// N elements at any element-aligned address (gfx950 serves unaligned vector accesses: one instruction)
template <class T, int N>
struct rp_vec { T v[N]; };
template <class T, int N>
__device__ __forceinline__ rp_vec<T, N> rp_load_vec(const T* p) {
  rp_vec<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <class T, int N>
__device__ __forceinline__ void rp_store_vec(T* p, const rp_vec<T, N>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}

// ---- MXFP4 (OCP microscaling formats 1.0: E2M1 elements, one E8M0 scale per 32) ---------------------------------------------------
constexpr int RP_MX = 32;  // elements of a block
typedef float rp_f32x2 __attribute__((ext_vector_type(2)));
typedef float rp_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 rp_bf16x2 __attribute__((ext_vector_type(2)));

// scale byte of a block from the largest magnitude's bits: floor(log2 max) - 2, at least 2^-127; a block with Inf or NaN: 255
__device__ __forceinline__ uint32_t rp_mx_scale_byte(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// the scale operand of the conversion instructions: the byte in a float's exponent field (they read nothing else of it - byte 0
// means 2^-127, byte 255 NaN; checked for all 256 code pairs)
__device__ __forceinline__ float rp_mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// eight elements (even index in the low nibble) <- eight floats; v_cvt_scalef32_pk_fp4_f32 rounds to nearest even and saturates at 6
__device__ __forceinline__ uint32_t rp_mx_pack8(const float* v, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
  return w;
}
__device__ __forceinline__ void rp_mx_unpack8(uint32_t w, float scale, float* v) {
  rp_f32x2 t;
  t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0); v[0] = t.x; v[1] = t.y;
  t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1); v[2] = t.x; v[3] = t.y;
  t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2); v[4] = t.x; v[5] = t.y;
  t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3); v[6] = t.x; v[7] = t.y;
}

// checks of an MXFP4 operand: codes rows of 16-byte blocks (base and leading dimension multiples of 16), one scale byte per block
int rp_mx_check(const char* who, int64_t rows, int64_t cols, const uint8_t* codes, int64_t ld_codes, const uint8_t* scales, int64_t ld_scales);
