// Microscaled rows (mx.hip, mx_score.hip): blocks of 32 consecutive values that share one
// power of two.
//
//   data  [rows, P * BITS / 8]  elements: E2M1 (BITS = 4, two per byte, the even one in the
//                               low nibble) or E4M3 (BITS = 8); P = dim rounded up to 32,
//                               the values behind dim are zero
//   scale [rows, P / 32]        E8M0: byte s stands for 2^(s - 127), 255 for NaN
#pragma once
#include "common.h"

namespace fps {

constexpr int MX_BLOCK = 32;

typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
typedef short mx_i16x2 __attribute__((ext_vector_type(2)));

// 2^(s - 127) for s in [0, 254]; 2^-127 is the subnormal 0x00400000
__device__ __forceinline__ float mx_scale_value(uint32_t s) {
  return __uint_as_float(s ? s << 23 : 0x00400000u);
}

// The scale byte of a block whose largest magnitude has the float bits `amax`: the exponent
// field (floor(log2) + 127; 0 for zeros and subnormals) less the element's largest exponent
// (2 for E2M1, 8 for E4M3), not below 0.  An infinity or a NaN in the block -- their bits
// compare above every finite magnitude's -- gives 255: the whole block reads back NaN.
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  constexpr int emax = BITS == 4 ? 2 : 8;
  const int e = (int)(amax >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - emax, 0);
}

// Waits for all loads, where the compiler sees it: a register that a branch may or may not have loaded is
// else waited for at each later use, with all that was sent since.
__device__ __forceinline__ void settle_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }  // vmcnt(0)

}  // namespace fps
