// Device helpers of the quantised outputs, shared by the norms' epilogues and the MX cache: moves
// and maxima inside a wave, and fp8 E4M3 / fp4 E2M1 encoding by gfx950's conversion instructions.
#ifndef VELOGRAD_MX_DEVICE_H
#define VELOGRAD_MX_DEVICE_H

#include "common.h"
#include "fp8_e4m3.h"
#include "mx_formats.h"

namespace vg {

template <int CTRL>
__device__ inline uint32_t dpp_move_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}

__device__ inline uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Largest value over aligned groups of L lanes (L = 4 or 8), on every lane of the group.
template <int L>
__device__ inline uint32_t lane_group_max(uint32_t v) {
  static_assert(L == 4 || L == 8, "MX blocks span 4 or 8 lanes");
  v = umax(v, dpp_move_u32<0xB1>(v));     // quad_perm [1,0,3,2]
  v = umax(v, dpp_move_u32<0x4E>(v));     // quad_perm [2,3,0,1]
  if constexpr (L == 8) v = umax(v, dpp_move_u32<0x141>(v));  // row_half_mirror
  return v;
}

// ------------------------------------------------------------------------------------------
// fp8 E4M3 codes on the device.  gfx950's v_cvt_pk_fp8_f32 converts two fp32 values to OCP
// e4m3fn with round to nearest even (one instruction per pair instead of the integer steps of
// vg_fp8::e4m3_encode, which the CPU tests pin against the oracle).  It is not saturating, and
// needs not be here: the inputs are y * (1 / scale) with |y| <= amax, so |y * inv| <=
// 448 * (1 + 2^-22), which rounds to 448 (values up to the 464 midpoint do); the exception,
// inv = 1 for a row whose scale is below the smallest normal float, has |y| < 2^-117.  NaN
// converts to a NaN code.  Build with -DVG_FP8_SOFT_ENCODE=1 to use the integer encoder.
// ------------------------------------------------------------------------------------------
#ifndef VG_FP8_SOFT_ENCODE
#define VG_FP8_SOFT_ENCODE 0
#endif

__device__ inline uint32_t e4m3x4(float a, float b, float c, float d) {
#if VG_FP8_SOFT_ENCODE
  return vg_fp8::e4m3_encode(a) | (vg_fp8::e4m3_encode(b) << 8) | (vg_fp8::e4m3_encode(c) << 16) |
         (vg_fp8::e4m3_encode(d) << 24);
#else
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
#endif
}

__device__ inline uint32_t e4m3x1(float a) {
#if VG_FP8_SOFT_ENCODE
  return vg_fp8::e4m3_encode(a);
#else
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, a, 0, false) & 0xffu;
#endif
}

// fp4 E2M1 nibbles on the device: gfx950's v_cvt_scalef32_pk_fp4_f32 converts two fp32 values
// divided by a scale to E2M1, round to nearest even, saturating, the first value in the low
// nibble of the selected byte (checked against the oracle's nearest-value encoder on every
// midpoint and a dense sweep at scales 0.5..4).  The block factor 2^-s is applied by an exact
// multiplication first and the instruction's scale is 1.  Build with -DVG_FP4_SOFT_ENCODE=1 to
// use vg_mx::e2m1_encode (the comparison chain the CPU tests pin) instead.
#ifndef VG_FP4_SOFT_ENCODE
#define VG_FP4_SOFT_ENCODE 0
#endif

template <int SEL>
__device__ inline uint32_t e2m1x2(uint32_t old, float a, float b) {
#if VG_FP4_SOFT_ENCODE
  return old | ((vg_mx::e2m1_encode(a) | (vg_mx::e2m1_encode(b) << 4)) << (8 * SEL));
#else
  return (uint32_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, 1.0f, SEL);
#endif
}

// ------------------------------------------------------------------------------------------
// The MX cache's shape, as its entry points take it.
// ------------------------------------------------------------------------------------------
inline int32_t check_mx_cache(const char* what, int64_t kv_heads, int64_t head_dim, int64_t pages,
                              int64_t page_size, int32_t mx_format) {
  if (mx_format != VELOGRAD_MX_E4M3 && mx_format != VELOGRAD_MX_E2M1)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: unsupported mx_format %d", what, (int)mx_format);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: head_dim=%lld must be 64, 128 or 256", what,
                (long long)head_dim);
  if (page_size < 16 || page_size > 32768 || (page_size & (page_size - 1)) != 0)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT,
                "%s: page_size=%lld must be a power of two from 16 to 32768", what,
                (long long)page_size);
  if (kv_heads < 1 || kv_heads > 65535 || pages < 0 || pages > INT32_MAX)
    return fail(VELOGRAD_ERR_INVALID_ARGUMENT, "%s: invalid cache shape pages=%lld kv_heads=%lld", what,
                (long long)pages, (long long)kv_heads);
  return 0;
}

}  // namespace vg

#endif  // VELOGRAD_MX_DEVICE_H
