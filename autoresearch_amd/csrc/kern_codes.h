// kern_codes.h -- the 8-bit codes of FG_I8 and FG_E4M3 pages as numbers.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/fgpt.h"

namespace fgpt {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// Four codes in order as fp32. Both kinds are exact in bf16 too: integers up to
// 127, and three bits behind a leading one.
template <int KT>
__device__ __forceinline__ void code_values(uint32_t w, float* x) {
  static_assert(KT == FG_I8 || KT == FG_E4M3, "an 8-bit type");
  if constexpr (KT == FG_E4M3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = (float)(int8_t)(w >> (8 * k));
  }
}

// Codes 2 i and 2 i + 1 of four as a pair of bf16.
template <int KT>
__device__ __forceinline__ uint32_t codes_bf16x2(uint32_t w, int i) {
  static_assert(KT == FG_I8 || KT == FG_E4M3, "an 8-bit type");
  if constexpr (KT == FG_E4M3) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t v = i ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, true)
                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, false);
    return __builtin_bit_cast(uint32_t, v);
  } else {
    // (a byte select of the conversion; the compiler moves its shifts out of loops)
    float a, b;
    if (i) {
      asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(a) : "v"(w));
      asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(b) : "v"(w));
    } else {
      asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(a) : "v"(w));
      asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(b) : "v"(w));
    }
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
  }
}

// Eight codes as an MFMA operand.
template <int KT>
__device__ __forceinline__ bf16x8_t codes_bf16(uint32_t a, uint32_t b) {
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(bf16x8_t, u32x4_t{codes_bf16x2<KT>(a, 0), codes_bf16x2<KT>(a, 1),
                                              codes_bf16x2<KT>(b, 0), codes_bf16x2<KT>(b, 1)});
}

}  // namespace fgpt
