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
// The same index twice in one write: the later row wins whole.  owner[slot] takes the position of some
// row that names the slot, then a row that finds an earlier one there raises it (only repeated
// indices do), then the writing pass writes the rows that own their slots.  Only named slots are
// read, and each was stored by this call: the entries need no clearing.  (One pass of integer
// maxima over cleared entries in place of the first two: 37 us for 1M rows, against 20.)
//
// The lanes' shares of all rows lie one after another over the waves, whatever the width of a row
// (whole rows per wave left half of the lanes of 300-wide rows idle: 36 us for a read that takes
// 28 so).  Nothing but registers is shared; a wave takes UNROLL units of 64 together, their
// loads all in flight before the first store.
#include <hip/hip_fp16.h>

#include "mx.h"

using namespace fps;

namespace {

constexpr int VPL = 8;            // values per lane of a write
constexpr int LPB = MX_BLOCK / VPL;  // lanes per block

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

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
        f32x4 f = {0.f, 0.f, 0.f, 0.f};
        if (d + 4 * h < D) f = *(const f32x4*)(p + 4 * h);
        v[4 * h] = f[0]; v[4 * h + 1] = f[1]; v[4 * h + 2] = f[2]; v[4 * h + 3] = f[3];
      }
    } else {  // D is a multiple of 8
      u32x4 w = {0, 0, 0, 0};
      if (d < D) w = *(const u32x4*)((const uint16_t*)x + row * D + d);
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

constexpr int UNROLL = 4;  // units a wave takes together

__global__ void __launch_bounds__(256) mx_claim_kernel(const void* __restrict__ idx, int idx64, int64_t n,
                                                       int64_t rows, int32_t* __restrict__ owner) {
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < n; r += (int64_t)gridDim.x * 256) {
    const int64_t slot = row_of(idx, idx64, r);
    if (slot >= 0 && slot < rows) owner[slot] = (int32_t)r;  // some row of those that name the slot
  }
}

__global__ void __launch_bounds__(256) mx_raise_kernel(const void* __restrict__ idx, int idx64, int64_t n,
                                                       int64_t rows, int32_t* owner) {
  for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < n; r += (int64_t)gridDim.x * 256) {
    const int64_t slot = row_of(idx, idx64, r);
    // (a stale value is an earlier row's: the maximum settles it)
    if (slot >= 0 && slot < rows && owner[slot] < (int32_t)r) atomicMax(owner + slot, (int32_t)r);
  }
}

// Both in one launch for few rows: one workgroup, the barrier between the stores and the reads.
// (4096 rows: 5.5 us, against 4.8 us in two launches and what the second costs the host.)
constexpr int FEW_ROWS = 4096;
__global__ void __launch_bounds__(1024) mx_claim_few_kernel(const void* __restrict__ idx, int idx64, int n, int64_t rows,
                                                            int32_t* owner) {
  int64_t slot[FEW_ROWS / 1024];
#pragma unroll
  for (int k = 0; k < FEW_ROWS / 1024; ++k) {
    const int r = threadIdx.x + k * 1024;
    slot[k] = r < n ? row_of(idx, idx64, r) : -1;
    if (slot[k] >= rows) slot[k] = -1;
  }
#pragma unroll
  for (int k = 0; k < FEW_ROWS / 1024; ++k)
    if (slot[k] >= 0)
      __hip_atomic_store(owner + slot[k], (int32_t)(threadIdx.x + k * 1024), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < FEW_ROWS / 1024; ++k) {
    const int32_t r = threadIdx.x + k * 1024;
    if (slot[k] >= 0 && __hip_atomic_load(owner + slot[k], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) < r)
      atomicMax(owner + slot[k], r);
  }
}

// `lpr` lanes per row; lane l of unit u has share 64 u + l of the n * lpr.
struct RowShape {
  int lpr, grid;
  float inv;                       // 1 / lpr
  int unit_rows, unit_rem;         // 64 shares further: so many rows and shares
  int64_t units, step_rows;        // a step of the whole grid
  int step_rem;
};
struct Place {
  int64_t row;
  int g;        // the lane's share within the row
  bool on;
};
// the first share of a unit; moved along without divisions
struct Walk {
  int64_t row;
  int rem;
  __device__ __forceinline__ void move(int64_t rows, int more, int lpr) {
    row += rows;
    rem += more;
    if (rem >= lpr) { rem -= lpr; ++row; }
  }
  __device__ __forceinline__ Place place(const RowShape& s, int64_t n) const {
    const int t = rem + (threadIdx.x & 63);
    int q = (int)((float)t * s.inv);  // t / lpr, one off at most
    int g = t - q * s.lpr;
    if (g < 0) { g += s.lpr; --q; }
    if (g >= s.lpr) { g -= s.lpr; ++q; }
    return Place{row + q, g, row + q < n};
  }
};
__device__ __forceinline__ int64_t first_unit() {
  return ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * UNROLL;
}
__device__ __forceinline__ Walk walk_from(const RowShape& s, int64_t unit) {
  const int64_t share = unit * 64, row = share / s.lpr;
  return Walk{row, (int)(share - row * s.lpr)};
}

// The indices of UNROLL places as they lie in memory (places past the end: the last index), and the slots they
// name.  Apart, so that the loads leave together: widened at once, each 32-bit index would be waited for.
struct RawIndex { int32_t lo, hi; };
__device__ __forceinline__ void load_indices(const void* idx, int idx64, int64_t n, const Place (&w)[UNROLL],
                                             RawIndex (&raw)[UNROLL]) {
  if (idx == nullptr) return;
  if (idx64) {
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) raw[k] = ((const RawIndex*)idx)[min(w[k].row, n - 1)];
  } else {
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) raw[k].lo = ((const int32_t*)idx)[min(w[k].row, n - 1)];
  }
}
// -1 where there is none
__device__ __forceinline__ int64_t slot_of(const void* idx, int idx64, const Place& w, const RawIndex& raw, int64_t rows) {
  int64_t slot = w.row;
  if (idx != nullptr) slot = idx64 ? (int64_t)((uint64_t)(uint32_t)raw.hi << 32 | (uint32_t)raw.lo) : (int64_t)raw.lo;
  return w.on && slot < rows ? slot : -1;
}

template <int BITS>
__device__ __forceinline__ void quantise(float v[VPL], uint32_t& s, uint2& q) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < VPL; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
  s = mx_scale_byte<BITS>(m);
  const float f = mx_scale_value(s & 255u);
  q = make_uint2(0, 0);
  if (BITS == 4) {
    q.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q.x, v[0], v[1], f, 0);
    q.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q.x, v[2], v[3], f, 1);
    q.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q.x, v[4], v[5], f, 2);
    q.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q.x, v[6], v[7], f, 3);
  } else {
    const float top = 448.f * f;
    mx_i16x2 lo = {0, 0}, hi = {0, 0};
#pragma unroll
    for (int j = 0; j < VPL; ++j) v[j] = fminf(fmaxf(v[j], -top), top);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, v[0], v[1], f, false);
    lo = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(lo, v[2], v[3], f, true);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, v[4], v[5], f, false);
    hi = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(hi, v[6], v[7], f, true);
    q = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
  }
  if (s == 255u) q = make_uint2(0, 0);
}

template <int T, int BITS, bool VEC, bool CLAIM>
__global__ void __launch_bounds__(256) mx_set_rows_kernel(const void* __restrict__ x, const void* __restrict__ idx,
                                                          int idx64, int64_t n, int D, int64_t rows,
                                                          uint8_t* __restrict__ data, uint8_t* __restrict__ scale,
                                                          RowShape shape, const int32_t* __restrict__ owner) {
  const int nblk = shape.lpr / LPB;
  const int64_t row_bytes = (int64_t)nblk * MX_BLOCK * BITS / 8;
  Walk walk = walk_from(shape, first_unit());
  for (int64_t u0 = first_unit(); u0 < shape.units; u0 += (int64_t)gridDim.x * 4 * UNROLL) {
    Place w[UNROLL];
    RawIndex raw[UNROLL];
    int64_t slot[UNROLL];
    float v[UNROLL][VPL];
    Walk unit = walk;
    walk.move(shape.step_rows, shape.step_rem, shape.lpr);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      w[k] = unit.place(shape, n);
      unit.move(shape.unit_rows, shape.unit_rem, shape.lpr);
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      if (w[k].on) load8<T, VEC>(x, w[k].row, D, w[k].g * VPL, v[k]);
    load_indices(idx, idx64, n, w, raw);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) slot[k] = slot_of(idx, idx64, w[k], raw[k], rows);
    if (CLAIM) {
      settle_loads();
      int32_t own[UNROLL];
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) own[k] = owner[max(slot[k], (int64_t)0)];
#pragma unroll
      for (int k = 0; k < UNROLL; ++k)
        if (own[k] != (int32_t)w[k].row) slot[k] = -1;
    }
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      if (slot[k] < 0) continue;
      uint32_t s;
      uint2 q;
      quantise<BITS>(v[k], s, q);
      const int64_t at = slot[k] * row_bytes + (int64_t)w[k].g * (VPL * BITS / 8);
      if (BITS == 4) *(uint32_t*)(data + at) = q.x;
      else *(uint2*)(data + at) = q;
      if ((w[k].g & (LPB - 1)) == 0) scale[slot[k] * nblk + w[k].g / LPB] = (uint8_t)s;
    }
  }
}

template <int T>
__device__ __forceinline__ uint16_t to16(float f) {
  return T == T_BF16 ? f32_to_bf16(f) : __half_as_ushort(__float2half_rn(f));
}

// Read back V values a lane: 16 bytes of output, so that a wave's store is one run of whole lines (8 fp32
// values a lane, two stores 32 bytes apart: 74 us for 1M x 64 in order against 56), past the
// caches, which keep the table instead (42 us; rows in random order 70 -> 64 us).
template <int BITS, int V>
__device__ __forceinline__ void values(uint2 q, uint32_t s, float v[V]) {
  const float f = s == 255u ? __uint_as_float(0x7fc00000u) : mx_scale_value(s);
  mx_f32x2 p[4];
  if (BITS == 4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q.x, 1.f, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q.x, 1.f, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q.x, 1.f, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q.x, 1.f, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q.x, 1.f, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q.x, 1.f, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q.y, 1.f, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q.y, 1.f, true);
  }
#pragma unroll
  for (int j = 0; j < V / 2; ++j) {  // an exact product unless it leaves fp32's range
    v[2 * j] = p[j][0] * f;
    v[2 * j + 1] = p[j][1] * f;
  }
}

template <int T, int V, bool VEC>
__device__ __forceinline__ void store_values(void* out, int64_t r, int D, int d, const float v[V]) {
  if (VEC) {  // D is a multiple of V
    if constexpr (T == T_F32) {
      __builtin_nontemporal_store((f32x4){v[0], v[1], v[2], v[3]}, (f32x4*)((float*)out + r * D + d));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (uint32_t)to16<T>(v[2 * j]) | ((uint32_t)to16<T>(v[2 * j + 1]) << 16);
      __builtin_nontemporal_store((u32x4){w[0], w[1], w[2], w[3]}, (u32x4*)((uint16_t*)out + r * D + d));
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (d + j < D) {
        if (T == T_F32) ((float*)out)[r * D + d + j] = v[j];
        else ((uint16_t*)out)[r * D + d + j] = to16<T>(v[j]);
      }
  }
}

// V values of a packed row from byte `at` on
template <int BITS, int V>
__device__ __forceinline__ uint2 load_packed(const uint8_t* p) {
  if (BITS * V == 16) return make_uint2(*(const uint16_t*)p, 0);
  if (BITS * V == 32) return make_uint2(*(const uint32_t*)p, 0);
  return *(const uint2*)p;
}

template <int T, int BITS, bool VEC>
__global__ void __launch_bounds__(256) mx_gather_rows_kernel(const uint8_t* __restrict__ data,
                                                             const uint8_t* __restrict__ scale, int64_t rows, int D,
                                                             const void* __restrict__ idx, int idx64, int64_t n,
                                                             void* __restrict__ out, RowShape shape) {
  constexpr int V = T == T_F32 ? 4 : 8, PER = MX_BLOCK / V;
  const int nblk = shape.lpr / PER;
  const int64_t row_bytes = (int64_t)nblk * MX_BLOCK * BITS / 8;
  Walk walk = walk_from(shape, first_unit());
  for (int64_t u0 = first_unit(); u0 < shape.units; u0 += (int64_t)gridDim.x * 4 * UNROLL) {
    Place w[UNROLL];
    RawIndex raw[UNROLL];
    int64_t slot[UNROLL];
    uint2 q[UNROLL];
    uint32_t s[UNROLL];
    Walk unit = walk;
    walk.move(shape.step_rows, shape.step_rem, shape.lpr);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      w[k] = unit.place(shape, n);
      unit.move(shape.unit_rows, shape.unit_rem, shape.lpr);
      w[k].on = w[k].on && w[k].g * V < D;
    }
    load_indices(idx, idx64, n, w, raw);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) slot[k] = slot_of(idx, idx64, w[k], raw[k], rows);
    settle_loads();
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      q[k] = make_uint2(0, 0);
      s[k] = 127;
      if (slot[k] >= 0) {
        q[k] = load_packed<BITS, V>(data + slot[k] * row_bytes + (int64_t)w[k].g * (V * BITS / 8));
        s[k] = scale[slot[k] * nblk + w[k].g / PER];
      }
    }
    settle_loads();  // here, and not again between the stores, each of which would be waited for
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      float v[V];
      values<BITS, V>(q[k], s[k], v);
      if (w[k].on) store_values<T, V, VEC>(out, w[k].row, D, w[k].g * V, v);
    }
  }
}

RowShape row_shape(int64_t n, int D, int lanes_per_block) {
  RowShape s;
  s.lpr = (D + MX_BLOCK - 1) / MX_BLOCK * lanes_per_block;
  s.inv = 1.f / (float)s.lpr;
  s.unit_rows = 64 / s.lpr;
  s.unit_rem = 64 % s.lpr;
  s.units = (n * s.lpr + 63) / 64;
  s.grid = grid_for(s.units, 4 * UNROLL, 256 * 32);
  const int64_t step = (int64_t)s.grid * 4 * UNROLL * 64;
  s.step_rows = step / s.lpr;
  s.step_rem = (int)(step % s.lpr);
  return s;
}

// 16-byte accesses need every row to start on 16 bytes
bool wide(const void* p, int D, int type) { return ((uintptr_t)p & 15) == 0 && D % (type == T_F32 ? 4 : 8) == 0; }

template <int T, int BITS>
void set_rows(bool vec, bool claim, const RowShape& s, hipStream_t st, const void* x, const void* idx, int idx64,
              int64_t n, int D, int64_t rows, uint8_t* data, uint8_t* scale, int32_t* owner) {
#define FPS_MX_SET(V, C)                                                                                         \
  hipLaunchKernelGGL((mx_set_rows_kernel<T, BITS, V, C>), dim3(s.grid), dim3(256), 0, st, x, idx, idx64, n, \
                     D, rows, data, scale, s, owner)
  if (vec) { if (claim) FPS_MX_SET(true, true); else FPS_MX_SET(true, false); }
  else { if (claim) FPS_MX_SET(false, true); else FPS_MX_SET(false, false); }
#undef FPS_MX_SET
}

template <int T, int BITS>
void gather_rows(bool vec, const RowShape& s, hipStream_t st, const uint8_t* data, const uint8_t* scale, int64_t rows,
                 int D, const void* idx, int idx64, int64_t n, void* out) {
  if (vec)
    hipLaunchKernelGGL((mx_gather_rows_kernel<T, BITS, true>), dim3(s.grid), dim3(256), 0, st, data, scale, rows,
                       D, idx, idx64, n, out, s);
  else
    hipLaunchKernelGGL((mx_gather_rows_kernel<T, BITS, false>), dim3(s.grid), dim3(256), 0, st, data, scale,
                       rows, D, idx, idx64, n, out, s);
}

}  // namespace

// x [n, D] (type 0 fp32, 1 bf16, 2 fp16) into rows idx[r] (nullptr: row r) of the table;
// owner [rows]: workspace, needed for more than one indexed row
FPS_API int fps_mx_set_rows(const void* x, int type, const void* idx, int idx64, int64_t n, int D, int64_t rows,
                            void* data, void* scale, int bits, int32_t* owner, void* stream) {
  if (n <= 0 || rows <= 0) return 0;
  if (D <= 0 || D > INT32_MAX - MX_BLOCK || (bits != 4 && bits != 8) || type < 0 || type > 2) return (int)hipErrorInvalidValue;
  const bool claim = idx != nullptr && n > 1;
  if (claim && (owner == nullptr || n > INT32_MAX)) return (int)hipErrorInvalidValue;  // (claims are 32-bit)
  hipStream_t st = (hipStream_t)stream;
  if (claim && n <= FEW_ROWS) {
    hipLaunchKernelGGL(mx_claim_few_kernel, dim3(1), dim3(1024), 0, st, idx, idx64, (int)n, rows, owner);
    FPS_CHECK_LAUNCH();
  } else if (claim) {
    hipLaunchKernelGGL(mx_claim_kernel, dim3(grid_for(n, 256)), dim3(256), 0, st, idx, idx64, n, rows, owner);
    FPS_CHECK_LAUNCH();
    hipLaunchKernelGGL(mx_raise_kernel, dim3(grid_for(n, 256)), dim3(256), 0, st, idx, idx64, n, rows, owner);
    FPS_CHECK_LAUNCH();
  }
  const RowShape s = row_shape(n, D, LPB);
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
  if (D <= 0 || D > INT32_MAX - MX_BLOCK || (bits != 4 && bits != 8) || type < 0 || type > 2) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  const RowShape s = row_shape(n, D, type == T_F32 ? MX_BLOCK / 4 : MX_BLOCK / 8);
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
