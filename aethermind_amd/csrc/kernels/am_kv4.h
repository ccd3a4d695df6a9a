// The 4-bit KV cache format (AM_KV_MXFP4) on the device, and host checks shared by its
// entry points.
#pragma once

#include "am_kernel_common.h"

namespace am {

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

// The scale operand of the conversions: the E8M0 byte as an fp32 exponent.  The
// conversions read it as E8M0: 0 is 2^-127 and 255 gives NaN.  Bytes from kScaleNan on
// (253 and 254 lie beyond bf16 and are never written) count as NaN.
constexpr uint32_t kScaleNan = 253;
__device__ __forceinline__ float e8m0_scale(uint32_t e) { return __uint_as_float(e << 23); }
__device__ __forceinline__ float e8m0_scale_or_nan(uint32_t e) { return e8m0_scale(e >= kScaleNan ? 255u : e); }

// 8 codes (one 32-bit word of a row) as bf16 values, exact: v_cvt_scalef32_pk_bf16_fp4,
// one instruction per two values at the rate of a byte permute.
__device__ __forceinline__ void fp4_to_bf16(uint32_t w, float scale, uint32_t (&out)[4]) {
  out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
  out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
  out[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
  out[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
}

// position start + s, saturated far outside any cache instead of wrapping
__device__ __forceinline__ int64_t seq_position(int64_t start, int64_t s) {
  constexpr int64_t kFar = int64_t{1} << 62;
  return min(max(start, -kFar), kFar) + s;
}

// Live rows of sequence b of a padded batch of `seq` rows each.
__device__ __forceinline__ int32_t live_rows(const int32_t* lens, int64_t b, int32_t seq) {
  return lens != nullptr ? min(max(lens[b], 0), seq) : seq;
}

// ---- host ----
inline bool Aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// The stream belongs to the current device (whose CU count and kernels a call uses).
am_status_code CheckStreamDevice(hipStream_t s);
// Layout rules of AM_KV_MXFP4: head_dim, capacity, stride and alignment of the four caches.
am_status_code CheckKv4Cache(const void* kc, const void* ks, const void* vc, const void* vs, int64_t batch,
                             int64_t head_dim, int64_t capacity, int64_t cbs, const am_gfx950_kv_pages* pages);

}  // namespace am
