// Microscaled tables: quantise rows as they are written, read rows back (gfx950).
//
//   write  s = exponent(max |x| over a block of 32) - emax,  q = RNE(x / 2^(s - 127)), saturated
//   read   y = q * 2^(s - 127)
//
// Both are bound by memory: a write reads 4 or 2 B per value and writes 17/32 B (fp4) or
// 33/32 B (fp8) of it, a read the other way round.  Four lanes own one block, eight values a
// lane, so the maximum takes two cross-lane steps inside a quad and every load and store is
// 4 to 16 B wide.  The rounding itself is one conversion instruction per two values
// (v_cvt_scalef32_pk_*): round to nearest even; the 4-bit form saturates, the 8-bit form
// turns anything past 464 into NaN, so its operands are clamped to 448 first.
//
// A row index outside the table is a padding slot: skipped by a write, a zero row in a read.
// The same index twice in one write: the later row wins whole.  A claim pass keeps the last
// position per slot (an integer maximum, so its order does not matter), the writing pass
// compares and empties the slots it used, so the claims are clean for the next call.
#include <hip/hip_fp16.h>

#include "mx.h"

using namespace fps;

namespace {

constexpr int VPL = 8;            // values per lane
constexpr int LPB = MX_BLOCK / VPL;  // lanes per block

enum { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };

__device__ __forceinline__ int64_t row_of(const void* idx, int idx64, int64_t r) {
  if (idx == nullptr) return r;
  return idx64 ? ((const int64_t*)idx)[r] : (int64_t)((const int32_t*)idx)[r];
}

template <int T>
__device__ __forceinline__ float load1(const void* x, int64_t i) {
  if (T == T_F32) return ((const float*)x)[i];
  const uint16_t b = ((const uint16_t*)x)[i];
  return T == T_BF16 ? bf16_to_f32(b) : __half2float(__ushort_as_half(b));
}

// eight values of a row from column d on; columns >= D are zero
template <int T, bool VEC>
__device__ __forceinline__ void load8(const void* x, int64_t row, int D, int d, float v[VPL]) {
  if (VEC) {
    if (T == T_F32) {
      const float* p = (const float*)x + row * D + d;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // D is a multiple of 4: a group of four is in or out whole
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (d + 4 * h < D) f = *(const float4*)(p + 4 * h);
        v[4 * h] = f.x; v[4 * h + 1] = f.y; v[4 * h + 2] = f.z; v[4 * h + 3] = f.w;
      }
    } else {  // D is a multiple of 8
      uint4 u = make_uint4(0, 0, 0, 0);
      if (d < D) u = *(const uint4*)((const uint16_t*)x + row * D + d);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint16_t lo = (uint16_t)w[j], hi = (uint16_t)(w[j] >> 16);
        v[2 * j] = T == T_BF16 ? bf16_to_f32(lo) : __half2float(__ushort_as_half(lo));
        v[2 * j + 1] = T == T_BF16 ? bf16_to_f32(hi) : __half2float(__ushort_as_half(hi));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < VPL; ++j) v[j] = d + j < D ? load1<T>(x, row * D + d + j) : 0.f;
  }
}

__global__ void __launch_bounds__(256) mx_claim_kernel(const void* __restrict__ idx, int idx64, int64_t n,
                                                       int64_t rows, int32_t* __restrict__ owner) {
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < n; r += (int64_t)gridDim.x * 256) {
    const int64_t slot = row_of(idx, idx64, r);
    if (slot >= 0 && slot < rows) atomicMax(owner + slot, (int32_t)r);
  }
}

// `lpr` lanes per row (LPB per block), `rpp` rows per pass of the workgroup; rows wider than
// the workgroup are walked in steps of its size
template <int T, int BITS, bool VEC, bool CLAIM>
__global__ void __launch_bounds__(256) mx_set_rows_kernel(const void* __restrict__ x, const void* __restrict__ idx,
                                                          int idx64, int64_t n, int D, int64_t rows,
                                                          uint8_t* __restrict__ data, uint8_t* __restrict__ scale,
                                                          int lpr, int rpp, int32_t* __restrict__ owner) {
  const int lane_row = threadIdx.x / lpr, g0 = threadIdx.x - lane_row * lpr;
  const int nblk = lpr / LPB;
  const int64_t row_bytes = (int64_t)nblk * MX_BLOCK * BITS / 8;
  const int step = rpp == 1 ? blockDim.x : lpr;
  for (int64_t r0 = (int64_t)blockIdx.x * rpp; r0 < n; r0 += (int64_t)gridDim.x * rpp) {
    const int64_t r = r0 + lane_row;
    int64_t slot = -1;
    if (lane_row < rpp && r < n) {
      slot = row_of(idx, idx64, r);
      if (slot >= rows) slot = -1;
    }
    if (CLAIM) {  // every lane of the row reads the claim before one of them empties it
      bool won = false;
      if (slot >= 0) won = __hip_atomic_load(owner + slot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)r;
      __syncthreads();
      if (won && g0 == 0) __hip_atomic_store(owner + slot, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (!won) slot = -1;
    }
    if (slot < 0) continue;  // (the loop's barrier is the first thing of every pass)
    for (int g = g0; g < lpr; g += step) {
      float v[VPL];
      load8<T, VEC>(x, r, D, g * VPL, v);
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < VPL; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
      m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
      m = max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
      const uint32_t s = mx_scale_byte<BITS>(m);
      const float f = mx_scale_value(s & 255u);
      const int64_t at = slot * row_bytes + (int64_t)g * (VPL * BITS / 8);
      if (BITS == 4) {
        uint32_t q = 0;
        if (s != 255u) {
          q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], f, 0);
          q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], f, 1);
          q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], f, 2);
          q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], f, 3);
        }
        *(uint32_t*)(data + at) = q;
      } else {
        mx_i16x2 lo = {0, 0}, hi = {0, 0};
        if (s != 255u) {
          const float top = 448.f * f;
#pragma unroll
          for (int j = 0; j < VPL; ++j) v[j] = fminf(fmaxf(v[j], -top), top);
          lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, v[0], v[1], f, false);
          lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, v[2], v[3], f, true);
          hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, v[4], v[5], f, false);
          hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, v[6], v[7], f, true);
        }
        *(uint2*)(data + at) = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
      }
      if ((g & (LPB - 1)) == 0) scale[slot * nblk + g / LPB] = (uint8_t)s;
    }
  }
}

template <int T>
__device__ __forceinline__ uint16_t to16(float f) {
  return T == T_BF16 ? f32_to_bf16(f) : __half_as_ushort(__float2half_rn(f));
}

template <int T, int BITS, bool VEC>
__global__ void __launch_bounds__(256) mx_gather_rows_kernel(const uint8_t* __restrict__ data,
                                                             const uint8_t* __restrict__ scale, int64_t rows, int D,
                                                             const void* __restrict__ idx, int idx64, int64_t n,
                                                             void* __restrict__ out, int lpr, int rpp) {
  const int lane_row = threadIdx.x / lpr, g0 = threadIdx.x - lane_row * lpr;
  const int nblk = lpr / LPB;
  const int64_t row_bytes = (int64_t)nblk * MX_BLOCK * BITS / 8;
  const int step = rpp == 1 ? blockDim.x : lpr;
  if (lane_row >= rpp) return;
  for (int64_t r = (int64_t)blockIdx.x * rpp + lane_row; r < n; r += (int64_t)gridDim.x * rpp) {
    int64_t slot = row_of(idx, idx64, r);
    if (slot >= rows) slot = -1;
    for (int g = g0; g < lpr; g += step) {
      float v[VPL] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      const int d = g * VPL;
      if (d >= D) break;
      if (slot >= 0) {
        const uint32_t s = scale[slot * nblk + g / LPB];
        const float f = s == 255u ? __uint_as_float(0x7fc00000u) : mx_scale_value(s);
        const int64_t at = slot * row_bytes + (int64_t)g * (VPL * BITS / 8);
        mx_f32x2 p[4];
        if (BITS == 4) {
          const uint32_t q = *(const uint32_t*)(data + at);
          p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 0);
          p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 1);
          p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 2);
          p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 3);
        } else {
          const uint2 q = *(const uint2*)(data + at);
          p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q.x, 1.f, false);
          p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q.x, 1.f, true);
          p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q.y, 1.f, false);
          p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q.y, 1.f, true);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // an exact product unless it leaves fp32's range
          v[2 * j] = p[j][0] * f;
          v[2 * j + 1] = p[j][1] * f;
        }
      }
      if (VEC) {
        if (T == T_F32) {
          float* o = (float*)out + r * D + d;
          *(float4*)o = make_float4(v[0], v[1], v[2], v[3]);
          if (d + 4 < D) *(float4*)(o + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = (uint32_t)to16<T>(v[2 * j]) | ((uint32_t)to16<T>(v[2 * j + 1]) << 16);
          *(uint4*)((uint16_t*)out + r * D + d) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          if (d + j < D) {
            if (T == T_F32) ((float*)out)[r * D + d + j] = v[j];
            else ((uint16_t*)out)[r * D + d + j] = to16<T>(v[j]);
          }
      }
    }
  }
}

struct RowShape {
  int lpr, rpp, threads, grid;
};

// as many whole rows per workgroup as 256 threads hold, in a workgroup of whole waves
RowShape row_shape(int64_t n, int D) {
  RowShape s;
  s.lpr = (D + MX_BLOCK - 1) / MX_BLOCK * LPB;
  s.rpp = s.lpr >= 256 ? 1 : 256 / s.lpr;
  const int used = s.rpp == 1 && s.lpr > 256 ? 256 : s.rpp * s.lpr;
  s.threads = (used + 63) / 64 * 64;
  s.grid = grid_for(n, s.rpp, 256 * 64);
  return s;
}

// 16-byte accesses need every row to start on 16 bytes
bool wide(const void* p, int D, int type) { return ((uintptr_t)p & 15) == 0 && D % (type == T_F32 ? 4 : 8) == 0; }

template <int T, int BITS>
void set_rows(bool vec, bool claim, const RowShape& s, hipStream_t st, const void* x, const void* idx, int idx64,
              int64_t n, int D, int64_t rows, uint8_t* data, uint8_t* scale, int32_t* owner) {
#define FPS_MX_SET(V, C)                                                                                         \
  hipLaunchKernelGGL((mx_set_rows_kernel<T, BITS, V, C>), dim3(s.grid), dim3(s.threads), 0, st, x, idx, idx64, n, \
                     D, rows, data, scale, s.lpr, s.rpp, owner)
  if (vec) { if (claim) FPS_MX_SET(true, true); else FPS_MX_SET(true, false); }
  else { if (claim) FPS_MX_SET(false, true); else FPS_MX_SET(false, false); }
#undef FPS_MX_SET
}

template <int T, int BITS>
void gather_rows(bool vec, const RowShape& s, hipStream_t st, const uint8_t* data, const uint8_t* scale, int64_t rows,
                 int D, const void* idx, int idx64, int64_t n, void* out) {
  if (vec)
    hipLaunchKernelGGL((mx_gather_rows_kernel<T, BITS, true>), dim3(s.grid), dim3(s.threads), 0, st, data, scale, rows,
                       D, idx, idx64, n, out, s.lpr, s.rpp);
  else
    hipLaunchKernelGGL((mx_gather_rows_kernel<T, BITS, false>), dim3(s.grid), dim3(s.threads), 0, st, data, scale,
                       rows, D, idx, idx64, n, out, s.lpr, s.rpp);
}

}  // namespace

// x [n, D] (type 0 fp32, 1 bf16, 2 fp16) into rows idx[r] (nullptr: row r) of the table;
// owner [rows], all -1 between calls: needed when idx may repeat (n > 1)
FPS_API int fps_mx_set_rows(const void* x, int type, const void* idx, int idx64, int64_t n, int D, int64_t rows,
                            void* data, void* scale, int bits, int32_t* owner, void* stream) {
  if (n <= 0 || rows <= 0) return 0;
  if (D <= 0 || (bits != 4 && bits != 8) || type < 0 || type > 2 || n > INT32_MAX) return (int)hipErrorInvalidValue;
  const bool claim = idx != nullptr && n > 1;
  if (claim && owner == nullptr) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  if (claim) {
    hipLaunchKernelGGL(mx_claim_kernel, dim3(grid_for(n, 256)), dim3(256), 0, st, idx, idx64, n, rows, owner);
    FPS_CHECK_LAUNCH();
  }
  const RowShape s = row_shape(n, D);
  const bool vec = wide(x, D, type);
#define FPS_MX_SET_T(T)                                                                                               \
  if (bits == 4) set_rows<T, 4>(vec, claim, s, st, x, idx, idx64, n, D, rows, (uint8_t*)data, (uint8_t*)scale, owner); \
  else set_rows<T, 8>(vec, claim, s, st, x, idx, idx64, n, D, rows, (uint8_t*)data, (uint8_t*)scale, owner)
  if (type == T_F32) { FPS_MX_SET_T(T_F32); }
  else if (type == T_BF16) { FPS_MX_SET_T(T_BF16); }
  else { FPS_MX_SET_T(T_F16); }
#undef FPS_MX_SET_T
  FPS_CHECK_LAUNCH();
  return 0;
}

// out [n, D] = the values of rows idx[r] (nullptr: row r) of the table
FPS_API int fps_mx_gather_rows(const void* data, const void* scale, int64_t rows, int D, int bits, const void* idx,
                               int idx64, int64_t n, void* out, int type, void* stream) {
  if (n <= 0) return 0;
  if (D <= 0 || (bits != 4 && bits != 8) || type < 0 || type > 2) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  const RowShape s = row_shape(n, D);
  const bool vec = wide(out, D, type);
#define FPS_MX_GET_T(T)                                                                                              \
  if (bits == 4) gather_rows<T, 4>(vec, s, st, (const uint8_t*)data, (const uint8_t*)scale, rows, D, idx, idx64, n, out); \
  else gather_rows<T, 8>(vec, s, st, (const uint8_t*)data, (const uint8_t*)scale, rows, D, idx, idx64, n, out)
  if (type == T_F32) { FPS_MX_GET_T(T_F32); }
  else if (type == T_BF16) { FPS_MX_GET_T(T_BF16); }
  else { FPS_MX_GET_T(T_F16); }
#undef FPS_MX_GET_T
  FPS_CHECK_LAUNCH();
  return 0;
}
