// Inner products of queries with every row of a microscaled table (gfx950).
//
//   S[b, i] = sum_d Q[b, d] X[i, d]      X: E2M1 or E4M3 blocks of 32 with a power of two each
//
// Two forms.  bf16 queries: X's elements become bf16 in registers, their block's power of two
// included (exact), and v_mfma_f32_32x32x16_bf16 sums in fp32.  Queries in E2M1 blocks
// against an E2M1 table: v_mfma_scale_f32_32x32x64_f8f6f4 on the packed elements.  (An
// 8-bit table takes the bf16 form too: the 8-bit matrix instructions keep only about 2^-13
// of the sum of magnitudes on this card, the 4-bit and the bf16 ones 2^-24.)
//
// Layout.  The queries are the A operand (rows of the result), the table the B operand
// (columns), so a lane holds one table row's scores for 16 queries.  A wave owns IT * 32
// consecutive table rows, lane l the rows IT * (l % 32) .. + IT - 1: its IT scores of a query are
// neighbours and leave in one store, 32 lanes cover IT * 32 consecutive scores.
// The sum over d may be taken in any order as long as both operands agree: in a chunk of
// 2 * S blocks (S <= 4) the lower half of the wave takes blocks 0 .. S-1, the upper half S .. 2S-1,
// so a lane reads 16 * S (fp4) contiguous bytes of its row and its S scales are neighbours.
// The table goes from memory to registers, one chunk ahead of its use; nothing of it is
// shared between waves.  The queries go through LDS, rows 16 bytes off a power of two
// (the eight lanes of a 16-byte access phase then fall into distinct banks).
#include <hip/hip_fp16.h>

#include "mx.h"

using namespace fps;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

enum { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };

constexpr int WAVES = 4;      // waves per workgroup
constexpr int IT = 2;         // table rows per lane

// acc register r of a lane: query row (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5) of the 32
__device__ __forceinline__ int acc_row(int lane, int r) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }

// one block (32 elements) of a table row
template <int XB> struct Block;
template <> struct Block<4> { uint4 v; };
template <> struct Block<8> { uint4 v, w; };

__device__ __forceinline__ uint32_t dword(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// elements 8 s .. 8 s + 7 of a block as bf16, times f
__device__ __forceinline__ bf16x8 to_bf16(const Block<4>& b, int s, float f) {
  const uint32_t q = dword(b.v, s);
  const bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 0);
  const bf16x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 1);
  const bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 2);
  const bf16x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 3);
  return bf16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}
__device__ __forceinline__ bf16x8 to_bf16(const Block<8>& b, int s, float f) {
  const uint4& v = s < 2 ? b.v : b.w;
  const uint32_t lo = dword(v, (s & 1) * 2), hi = dword(v, (s & 1) * 2 + 1);
  const bf16x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, f, false);
  const bf16x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, f, true);
  const bf16x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, f, false);
  const bf16x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, f, true);
  return bf16x8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// a lane's blocks of one chunk, for its IT rows, with their scale bytes
template <int XB>
struct Chunk {
  Block<XB> b[IT][4];
  uint32_t s[IT];  // byte j: block j's scale
};

struct Args {
  const void* q;         // bf16 [B, D] or E2M1 [B, nblk * 16]
  const uint8_t* qs;     // E2M1 queries: scales [B, nblk]
  const uint8_t* x;      // table rows
  const uint8_t* xs;     // table scales [N, nblk]
  void* out;
  int64_t ld, N;
  int B, D, nblk;
  int out_type, pair;    // pair: every even column starts a 2-score store
  int q_vec;             // bf16 queries: rows start on 16 bytes
  int s_word;            // nblk % 4 == 0: four scales in one load
  int qtiles, itiles;
};

// blocks half h of the wave takes from the chunk at block c0: [first, first + S)
__device__ __forceinline__ int chunk_s(int nblk, int c0) { return min(4, (nblk - c0 + 1) >> 1); }

template <int XB>
__device__ __forceinline__ void load_chunk(const Args& a, int64_t row0, int c0, int h, Chunk<XB>& ch) {
  const int S = chunk_s(a.nblk, c0), first = c0 + h * S;
#pragma unroll
  for (int t = 0; t < IT; ++t) {
    const int64_t row = min(row0 + t, a.N - 1);  // rows past the end: loaded again, not stored
    const uint8_t* p = a.x + (row * a.nblk + first) * (MX_BLOCK * XB / 8);
    const uint8_t* sp = a.xs + row * a.nblk + first;
    uint32_t s = 0x7f7f7f7fu;  // a block that is not there: zeros times one
    if (S == 4 && a.s_word) s = *(const uint32_t*)sp;  // nblk % 4 == 0: first + 4 <= nblk
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Block<XB>& b = ch.b[t][j];
      b.v = make_uint4(0, 0, 0, 0);
      if constexpr (XB == 8) b.w = make_uint4(0, 0, 0, 0);
      if (j < S && first + j < a.nblk) {
        b.v = *(const uint4*)(p + j * (MX_BLOCK * XB / 8));
        if constexpr (XB == 8) b.w = *(const uint4*)(p + j * 32 + 16);
        if (!(S == 4 && a.s_word)) s = (s & ~(255u << (8 * j))) | ((uint32_t)sp[j] << (8 * j));
      }
    }
    ch.s[t] = s;
  }
}

// Stage queries [q0, q0 + 32 QT) x blocks [c0, c0 + nb) into LDS rows of `stride` bytes.
// A bf16 block is 64 bytes, an E2M1 block 16 (its scale goes to qsl, one byte per block).
template <bool Q4, int QT>
__device__ __forceinline__ void stage_queries(const Args& a, int q0, int c0, int nb, uint8_t* ql, uint8_t* qsl,
                                              int stride, int sstride) {
  constexpr int CB = Q4 ? 1 : 4;  // 16-byte pieces per block
  const int pieces = nb * CB;
  for (int e = threadIdx.x; e < 32 * QT * pieces; e += WAVES * 64) {
    const int r = e / pieces, c = e - r * pieces;
    const int q = q0 + r, blk = c0 + c / CB;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (q < a.B && blk < a.nblk) {
      if (Q4) {
        v = *(const uint4*)((const uint8_t*)a.q + ((int64_t)q * a.nblk + blk) * 16);
      } else {
        const int d = blk * 32 + (c % CB) * 8;
        const uint16_t* p = (const uint16_t*)a.q + (int64_t)q * a.D + d;
        if (a.q_vec && d + 8 <= a.D) {
          v = *(const uint4*)p;
        } else {
          uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (d + j < a.D) w[j >> 1] |= (uint32_t)p[j] << (16 * (j & 1));
          v = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    *(uint4*)(ql + r * stride + c * 16) = v;
    if (Q4) qsl[r * sstride + c] = (q < a.B && blk < a.nblk) ? a.qs[(int64_t)q * a.nblk + blk] : 127;
  }
}

template <int T>
__device__ __forceinline__ uint16_t to16(float f) {
  return T == T_BF16 ? f32_to_bf16(f) : __half_as_ushort(__float2half_rn(f));
}

template <int T>
__device__ __forceinline__ void store_pair(const Args& a, int64_t at, int64_t row, float v0, float v1) {
  if (row >= a.N) return;
  const bool two = row + 1 < a.N;
  if (T == T_F32) {
    float* o = (float*)a.out + at;
    if (two && a.pair) *(float2*)o = make_float2(v0, v1);
    else { o[0] = v0; if (two) o[1] = v1; }
  } else {
    uint16_t* o = (uint16_t*)a.out + at;
    const uint16_t x = to16<T>(v0), y = to16<T>(v1);
    if (two && a.pair) *(uint32_t*)o = (uint32_t)x | ((uint32_t)y << 16);
    else { o[0] = x; if (two) o[1] = y; }
  }
}

// KC: blocks of the queries held in LDS at a time.
template <int XB, bool Q4, int QT, int KC, int T>
__global__ void __launch_bounds__(256) mx_score_kernel(Args a) {
  constexpr int QBYTES = Q4 ? 16 : 64;
  constexpr int STRIDE = KC * QBYTES + 16, SSTRIDE = KC + 4;
  __shared__ __attribute__((aligned(16))) uint8_t ql[32 * QT * STRIDE];
  __shared__ __attribute__((aligned(16))) uint8_t qsl[Q4 ? 32 * QT * SSTRIDE : 16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
  const bool once = a.nblk <= KC;  // the queries fit: staged once for all tiles of this workgroup
  const int total = a.qtiles * a.itiles;
  int staged = -1;
  for (int w = blockIdx.x; w < total; w += gridDim.x) {
    const int tile = xcd_remap(w, total);  // query tiles of one table panel are neighbours on one XCD
    const int q0 = (tile % a.qtiles) * 32 * QT;
    const int64_t row0 = (int64_t)(tile / a.qtiles) * (WAVES * 32 * IT) + wave * (32 * IT) + (lane & 31) * IT;
    f32x16 acc[IT][QT];
#pragma unroll
    for (int t = 0; t < IT; ++t)
#pragma unroll
      for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][q][r] = 0.f;
    Chunk<XB> cur, nxt;
    load_chunk<XB>(a, row0, 0, h, cur);
    for (int k0 = 0; k0 < a.nblk; k0 += KC) {
      const int kn = min(KC, a.nblk - k0);
      if (!once || staged != q0) {
        __syncthreads();
        stage_queries<Q4, QT>(a, q0, k0, (kn + 7) / 8 * 8, ql, qsl, STRIDE, SSTRIDE);
        __syncthreads();
        staged = q0;
      }
      for (int c0 = k0; c0 < k0 + kn; c0 += 8) {
        if (c0 + 8 < a.nblk) load_chunk<XB>(a, row0, c0 + 8, h, nxt);
        const int S = chunk_s(a.nblk, c0), first = c0 - k0 + h * S;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (j < S) {
            if constexpr (Q4) {
              i32x8 qa[QT];
              int qsc[QT];
#pragma unroll
              for (int q = 0; q < QT; ++q) {
                const uint4 v = *(const uint4*)(ql + (q * 32 + (lane & 31)) * STRIDE + (first + j) * 16);
                qa[q] = i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
                qsc[q] = qsl[(q * 32 + (lane & 31)) * SSTRIDE + first + j];
              }
#pragma unroll
              for (int t = 0; t < IT; ++t) {
                const uint4 v = cur.b[t][j].v;
                const i32x8 xb = {(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
#pragma unroll
                for (int q = 0; q < QT; ++q)
                  acc[t][q] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(qa[q], xb, acc[t][q], 4, 4, 0, qsc[q], 0,
                                                                              (int)(cur.s[t] >> (8 * j)));
              }
            } else {
              float f[IT];
#pragma unroll
              for (int t = 0; t < IT; ++t) {
                const uint32_t s = (cur.s[t] >> (8 * j)) & 255u;
                f[t] = s == 255u ? __uint_as_float(0x7fc00000u) : mx_scale_value(s);
              }
#pragma unroll
              for (int s = 0; s < 4; ++s) {
                bf16x8 xb[IT];
#pragma unroll
                for (int t = 0; t < IT; ++t) xb[t] = to_bf16(cur.b[t][j], s, f[t]);
#pragma unroll
                for (int q = 0; q < QT; ++q) {
                  const uint4 v = *(const uint4*)(ql + (q * 32 + (lane & 31)) * STRIDE + (first + j) * 64 + s * 16);
                  const bf16x8 qa = __builtin_bit_cast(bf16x8, v);
#pragma unroll
                  for (int t = 0; t < IT; ++t)
                    acc[t][q] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qa, xb[t], acc[t][q], 0, 0, 0);
                }
              }
            }
          }
        }
        cur = nxt;
      }
    }
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int b = q0 + q * 32 + acc_row(lane, r);
        if (b < a.B) store_pair<T>(a, (int64_t)b * a.ld + row0, row0, acc[0][q][r], acc[1][q][r]);
      }
  }
}

template <int XB, bool Q4, int QT, int KC>
void launch(Args& a, hipStream_t st) {
  a.qtiles = (a.B + 32 * QT - 1) / (32 * QT);
  a.itiles = (int)((a.N + WAVES * 32 * IT - 1) / (WAVES * 32 * IT));
  const int64_t total = (int64_t)a.qtiles * a.itiles;
  const int grid = (int)(total < 2048 ? total : 2048);
  if (a.out_type == T_F32) hipLaunchKernelGGL((mx_score_kernel<XB, Q4, QT, KC, T_F32>), dim3(grid), dim3(256), 0, st, a);
  else if (a.out_type == T_BF16) hipLaunchKernelGGL((mx_score_kernel<XB, Q4, QT, KC, T_BF16>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((mx_score_kernel<XB, Q4, QT, KC, T_F16>), dim3(grid), dim3(256), 0, st, a);
}

}  // namespace

// out [B, N] (row stride ld, type 0 fp32 / 1 bf16 / 2 fp16) = q . x^T.  qs == nullptr: q is bf16
// [B, D]; else q holds E2M1 blocks and qs their scales (then xbits must be 4).
FPS_API int fps_mx_score(const void* q, const void* qs, const void* x, const void* xs, int xbits, int B, int64_t N,
                         int D, void* out, int out_type, int64_t ld, void* stream) {
  if (B <= 0 || N <= 0) return 0;
  if (D <= 0 || (xbits != 4 && xbits != 8) || (qs && xbits != 4) || ld < N || out_type < 0 || out_type > 2)
    return (int)hipErrorInvalidValue;
  Args a;
  a.q = q; a.qs = (const uint8_t*)qs; a.x = (const uint8_t*)x; a.xs = (const uint8_t*)xs;
  a.out = out; a.ld = ld; a.N = N; a.B = B; a.D = D;
  a.nblk = (D + MX_BLOCK - 1) / MX_BLOCK;
  a.out_type = out_type;
  a.pair = ld % 2 == 0 && ((uintptr_t)out & (out_type == T_F32 ? 7 : 3)) == 0;
  a.q_vec = D % 8 == 0 && ((uintptr_t)q & 15) == 0;
  a.s_word = a.nblk % 4 == 0 && ((uintptr_t)xs & 3) == 0;
  if (N > (int64_t)INT32_MAX * 32 || (int64_t)((B + 31) / 32) * ((N + 255) / 256) > INT32_MAX)
    return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  const bool few = B <= 32;
  if (qs) {
    if (few) launch<4, true, 1, 32>(a, st); else launch<4, true, 4, 16>(a, st);
  } else if (xbits == 4) {
    if (few) launch<4, false, 1, 16>(a, st); else launch<4, false, 4, 8>(a, st);
  } else {
    if (few) launch<8, false, 1, 16>(a, st); else launch<8, false, 4, 8>(a, st);
  }
  FPS_CHECK_LAUNCH();
  return 0;
}
