// Inner products of queries with every row of a microscaled table (gfx950).
//
//   S[b, i] = sum_d Q[b, d] X[i, d]      X: E2M1 or E4M3 blocks of 32 with a power of two each
//
// Two forms.  bf16 queries: X's elements become bf16 in registers, their block's power of two
// included (exact down to bf16's smallest subnormal, 2^-133, which only E4M3 blocks of scale bytes below 3
// pass), and v_mfma_f32_32x32x16_bf16 sums in fp32.  Queries in E2M1 blocks
// against an E2M1 table: v_mfma_scale_f32_32x32x64_f8f6f4 on the packed elements.  (An
// 8-bit table takes the bf16 form too: the 8-bit matrix instructions keep only about 2^-13
// of the sum of magnitudes on this card, the 4-bit and the bf16 ones 2^-24.)
//
// Layout.  The queries are the A operand (rows of the result), the table the B operand
// (columns), so a lane holds table rows' scores for 16 queries.  A wave owns IT * 32
// consecutive table rows, lane l the rows IT * (l % 32) .. + IT - 1: its IT scores of a query are
// neighbours and leave in one store, 32 lanes cover IT * 32 consecutive scores.
// The sum over d may be taken in any order as long as both operands agree: in a chunk of
// 2 * S blocks (S <= CS) the lower half of the wave takes blocks 0 .. S-1, the upper half S .. 2S-1,
// so a lane reads 16 * S (fp4) or 32 * S (fp8) contiguous bytes of its row and its S scales are
// neighbours.  The table goes from memory to registers, one chunk ahead of its use; nothing of
// it is shared between waves.  The queries go through LDS, rows 16 bytes off a power of two
// (the eight lanes of a 16-byte access phase then fall into distinct banks).
//
// Short rows (the queries' 32 QT rows fit in LDS whole): a workgroup stages its queries once and
// walks the table; bound by memory, the scores' writes above all.  Long rows: one tile per
// workgroup, the queries' next chunk on its way into the other half of LDS during the present
// one's products.
#include <hip/hip_fp16.h>

#include "mx.h"

using namespace fps;

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int WAVES = 4;      // waves per workgroup
constexpr int THREADS = WAVES * 64;

// (acc register r of a lane: query row (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5) of the 32)

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

// A lane's blocks of one chunk, for its IT rows, with their scale bytes as they were loaded, CS in a load
// (byte by byte and put together, each would be waited for before the next block's load is sent:
// 37 x 100003 x 300 in fp8 21.5 us against 17).  `late`: how many of them lie before the chunk's first.
template <int CS> struct Scales { typedef uint32_t Word; typedef uint32_t Any __attribute__((aligned(1))); };
template <> struct Scales<2> { typedef uint16_t Word; typedef uint16_t Any __attribute__((aligned(1))); };
template <> struct Scales<1> { typedef uint8_t Word; typedef uint8_t Any; };
template <int XB, int IT, int CS>
struct Chunk {
  Block<XB> b[IT][CS];
  typename Scales<CS>::Word s[IT];  // (widened at use: a load widened at once would be waited for)
  int late;
  // byte j: block j's scale, 0 for a block that is not there (zeros times 2^-127)
  __device__ __forceinline__ uint32_t scales(int t) const { return late >= CS ? 0u : (uint32_t)s[t] >> (8 * late); }
};

struct Args {
  const void* q;         // bf16 [B, D] or E2M1 [B, nblk * 16]
  const uint8_t* qs;     // E2M1 queries: scales [B, nblk]
  const uint8_t* x;      // table rows
  const uint8_t* xs;     // table scales [N, nblk]
  void* out;
  int64_t ld, N;
  int B, D, nblk;
  int vec;               // every lane's IT scores start on their own size
  int s_word;            // nblk % 4 == 0: scales in loads of four
  int qtiles, itiles;
};

// blocks half h of the wave takes from the chunk at block c0: [c0 + h S, c0 + h S + S)
template <int CS>
__device__ __forceinline__ int chunk_s(int nblk, int c0) { return min(CS, (nblk - c0 + 1) >> 1); }

template <int XB, int IT, int CS>
__device__ __forceinline__ void load_chunk(const Args& a, int64_t row0, int c0, int h, Chunk<XB, IT, CS>& ch) {
  static_assert(CS == 1 || CS == 2 || CS == 4, "scale bytes in one load");
  const int S = chunk_s<CS>(a.nblk, c0), first = c0 + h * S;
  const int from = min(first, a.nblk - CS);  // (nblk >= CS in every launch)
  ch.late = first - from;
#pragma unroll
  for (int t = 0; t < IT; ++t) {
    const int64_t row = min(row0 + t, a.N - 1);  // rows past the end: loaded again, not stored
    const uint8_t* p = a.x + (row * a.nblk + first) * (MX_BLOCK * XB / 8);
    const uint8_t* sp = a.xs + row * a.nblk + from;
    ch.s[t] = *(const typename Scales<CS>::Any*)sp;
#pragma unroll
    for (int j = 0; j < CS; ++j) {
      Block<XB>& b = ch.b[t][j];
      b.v = make_uint4(0, 0, 0, 0);
      if constexpr (XB == 8) b.w = make_uint4(0, 0, 0, 0);
      if (j < S && first + j < a.nblk) {
        b.v = *(const uint4*)(p + j * (MX_BLOCK * XB / 8));
        if constexpr (XB == 8) b.w = *(const uint4*)(p + j * 32 + 16);
      }
    }
  }
}

// 16 bytes of a query: piece c of block blk (bf16: 4 pieces a block, E2M1: 1).  A row of bf16 values may
// start and end anywhere: the piece over its end is loaded as the row's last 8 values, and settle()
// moves them to their places and zeros behind them (apart, so that loads do not wait for each other).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
template <bool Q4, bool NARROW>
__device__ __forceinline__ uint4 load_piece(const Args& a, int q, int blk, int c) {
  if (Q4) {
    if (q >= a.B || blk >= a.nblk) return make_uint4(0, 0, 0, 0);
    return *(const uint4*)((const uint8_t*)a.q + ((int64_t)q * a.nblk + blk) * 16);
  }
  const int d = blk * 32 + c * 8;
  if (q >= a.B || d >= a.D) return make_uint4(0, 0, 0, 0);
  const uint16_t* p = (const uint16_t*)a.q + (int64_t)q * a.D;
  if (NARROW && a.D < 8) {
    uint64_t w[2] = {0, 0};
#pragma unroll 1
    for (int j = a.D - 1; j >= 0; --j) {
      w[1] = w[1] << 16 | w[0] >> 48;
      w[0] = w[0] << 16 | p[j];
    }
    return make_uint4((uint32_t)w[0], (uint32_t)(w[0] >> 32), (uint32_t)w[1], (uint32_t)(w[1] >> 32));
  }
  const u32x4_any v = *(const u32x4_any*)(p + min(d, a.D - 8));
  return make_uint4(v[0], v[1], v[2], v[3]);
}
template <bool Q4>
__device__ __forceinline__ uint4 settle(const Args& a, int blk, int c, uint4 v) {
  if (Q4 || (a.D & 7) == 0 || a.D < 8) return v;
  const int n = max(blk * 32 + c * 8 - (a.D - 8), 0);  // values too early (8 and more: the piece is zeros)
  if (n & 4) v = make_uint4(v.z, v.w, 0, 0);
  if (n & 2) v = make_uint4(v.y, v.z, v.w, 0);
  if (n & 1) v = make_uint4(v.x >> 16 | v.y << 16, v.y >> 16 | v.z << 16, v.z >> 16 | v.w << 16, v.w >> 16);
  return v;
}
__device__ __forceinline__ uint8_t load_qscale(const Args& a, int q, int blk) {
  return q < a.B && blk < a.nblk ? a.qs[(int64_t)q * a.nblk + blk] : (uint8_t)127;
}

typedef __bf16 bf16_2 __attribute__((ext_vector_type(2)));
typedef float f32_2 __attribute__((ext_vector_type(2)));
template <int T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {  // round to nearest even
  if (T == T_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32_2){lo, hi}, bf16_2));
  return (uint32_t)__half_as_ushort(__float2half_rn(lo)) | (uint32_t)__half_as_ushort(__float2half_rn(hi)) << 16;
}

// IT neighbouring scores to o; `left` of them exist
template <int T, int IT>
__device__ __forceinline__ void store_scores(char* at, bool whole, int left, const float v[IT]) {
  if (T == T_F32) {
    float* o = (float*)at;
    if (whole) {
      if constexpr (IT == 4) *(float4*)o = make_float4(v[0], v[1], v[2], v[3]);
      else *(float2*)o = make_float2(v[0], v[1]);
    } else {
#pragma unroll
      for (int t = 0; t < IT; ++t)
        if (t < left) o[t] = v[t];
    }
  } else {
    uint16_t* o = (uint16_t*)at;
    uint32_t w[IT / 2];
#pragma unroll
    for (int t = 0; t < IT / 2; ++t) w[t] = pack16<T>(v[2 * t], v[2 * t + 1]);
    if (whole) {
      if constexpr (IT == 4) *(uint2*)o = make_uint2(w[0], w[1]);
      else *(uint32_t*)o = w[0];
    } else {
#pragma unroll
      for (int t = 0; t < IT; ++t)
        if (t < left) o[t] = (uint16_t)(w[t / 2] >> (16 * (t & 1)));
    }
  }
}

// acc += one chunk: this lane's S blocks of cur by the queries' blocks first .. first + S - 1 in LDS
template <int XB, bool Q4, int QT, int IT, int CS, int STRIDE, int SSTRIDE>
__device__ __forceinline__ void multiply(const uint8_t* qrow, const uint8_t* qsrow, int first, int S,
                                         const Chunk<XB, IT, CS>& cur, f32x16 (&acc)[IT][QT]) {
  uint32_t sc[IT];
#pragma unroll
  for (int t = 0; t < IT; ++t) sc[t] = cur.scales(t);
#pragma unroll
  for (int j = 0; j < CS; ++j) {
    if (j < S) {
      if constexpr (Q4) {
        i32x8 qa[QT];
        int qsc[QT];
#pragma unroll
        for (int q = 0; q < QT; ++q) {
          const uint4 v = *(const uint4*)(qrow + q * 32 * STRIDE + (first + j) * 16);
          qa[q] = i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
          qsc[q] = qsrow[q * 32 * SSTRIDE + first + j];
        }
#pragma unroll
        for (int t = 0; t < IT; ++t) {
          const uint4 v = cur.b[t][j].v;
          const i32x8 xb = {(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
#pragma unroll
          for (int q = 0; q < QT; ++q)
            acc[t][q] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(qa[q], xb, acc[t][q], 4, 4, 0, qsc[q], 0,
                                                                        (int)(sc[t] >> (8 * j)));
        }
      } else {
        float f[IT];
#pragma unroll
        for (int t = 0; t < IT; ++t) {
          const uint32_t s = (sc[t] >> (8 * j)) & 255u;
          f[t] = s == 255u ? __uint_as_float(0x7fc00000u) : mx_scale_value(s);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          bf16x8 xb[IT];
#pragma unroll
          for (int t = 0; t < IT; ++t) xb[t] = to_bf16(cur.b[t][j], s, f[t]);
#pragma unroll
          for (int q = 0; q < QT; ++q) {
            const bf16x8 qa = __builtin_bit_cast(bf16x8, *(const uint4*)(qrow + q * 32 * STRIDE + (first + j) * 64 + s * 16));
#pragma unroll
            for (int t = 0; t < IT; ++t) acc[t][q] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qa, xb[t], acc[t][q], 0, 0, 0);
          }
        }
      }
    }
  }
}

// 16-byte pieces 0 .. pieces - 1 of 32 QT queries from block blk0 on to LDS, U in flight a thread
template <bool Q4, bool NARROW, int QT, int STRIDE, int SSTRIDE, int U>
__device__ __forceinline__ void stage_queries(const Args& a, int q0, int blk0, int pieces, uint8_t* ql, uint8_t* qsl) {
  constexpr int CB = Q4 ? 1 : 4;
  for (int e0 = threadIdx.x; e0 < 32 * QT * pieces; e0 += U * THREADS) {
    uint4 v[U];
    uint8_t s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * THREADS, r = e / pieces, c = e - r * pieces;
      if (e < 32 * QT * pieces) {
        v[u] = load_piece<Q4, NARROW>(a, q0 + r, blk0 + c / CB, c % CB);
        if (Q4) s[u] = load_qscale(a, q0 + r, blk0 + c);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * THREADS, r = e / pieces, c = e - r * pieces;
      if (e < 32 * QT * pieces) {
        *(uint4*)(ql + r * STRIDE + c * 16) = settle<Q4>(a, blk0 + c / CB, c % CB, v[u]);
        if (Q4) qsl[r * SSTRIDE + c] = s[u];
      }
    }
  }
}

// LB: blocks of a query held in LDS
template <int XB, bool Q4, int QT, int IT, int CS, int LB, int T>
__global__ void __launch_bounds__(THREADS, 2) mx_score_kernel(Args a) {
  constexpr int QBYTES = Q4 ? 16 : 64, CB = QBYTES / 16;
  constexpr int STRIDE = LB * QBYTES + 16, SSTRIDE = LB + 4;
  constexpr int KC = 2 * CS;  // blocks per chunk
  constexpr int QREGS = 32 * QT * KC * CB / THREADS > 0 ? 32 * QT * KC * CB / THREADS : 1;
  static_assert(CS == 1 || LB >= 2 * KC, "two chunks of queries");
  __shared__ __attribute__((aligned(16))) uint8_t ql[32 * QT * STRIDE];
  __shared__ __attribute__((aligned(16))) uint8_t qsl[Q4 ? 32 * QT * SSTRIDE : 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const bool once = CS == 1 || a.nblk <= LB;
  // once: one query tile, every stride-th table tile (the workgroups of one table tile are on one XCD);
  // else one tile
  int qt, it, step;
  if (once) {
    const int u = blockIdx.x >> 3;
    qt = u % a.qtiles;
    it = (u / a.qtiles) * 8 + (blockIdx.x & 7);
    step = gridDim.x / a.qtiles;
  } else {
    const int tile = xcd_remap(blockIdx.x, a.qtiles * a.itiles);
    qt = tile % a.qtiles;
    it = tile / a.qtiles;
    step = a.itiles;
  }
  if (it >= a.itiles) return;
  const int q0 = qt * 32 * QT;
  const auto row_of_tile = [&](int i) { return (int64_t)i * (WAVES * 32 * IT) + wave * (32 * IT) + (lane & 31) * IT; };
  Chunk<XB, IT, CS> cur, nxt;
  load_chunk<XB, IT, CS>(a, row_of_tile(it), 0, h, cur);  // on its way while the queries are staged
  {  // all of the queries, or their first chunk
    const int nb = once ? (a.nblk + KC - 1) / KC * KC : KC;
    constexpr int U = 32 * QT * LB * CB / THREADS;
    stage_queries<Q4, CS == 1, QT, STRIDE, SSTRIDE, U < 1 ? 1 : U < 6 ? U : 6>(a, q0, 0, min(nb, LB) * CB, ql, qsl);
    __syncthreads();
  }
  const uint8_t* qrow = ql + (lane & 31) * STRIDE;
  const uint8_t* qsrow = qsl + (lane & 31) * SSTRIDE;
  settle_loads();  // (else cur's first use in the loop waits, every time, for nxt as well)
  int half = 0;  // not once: the half of LDS that holds the present chunk's queries
  for (; it < a.itiles; it += step) {
    const int64_t row0 = row_of_tile(it);
    f32x16 acc[IT][QT];
#pragma unroll
    for (int t = 0; t < IT; ++t)
#pragma unroll
      for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][q][r] = 0.f;
    for (int c0 = 0; c0 < a.nblk; c0 += KC) {
      const bool more = c0 + KC < a.nblk;
      if (more || it + step < a.itiles)
        load_chunk<XB, IT, CS>(a, more ? row0 : row_of_tile(it + step), more ? c0 + KC : 0, h, nxt);
      uint4 qn[QREGS];
      uint8_t qsn[QREGS];
      if (CS > 1 && !once && more) {
#pragma unroll
        for (int i = 0; i < QREGS; ++i) {
          const int e = threadIdx.x + i * THREADS, r = e / (KC * CB), c = e % (KC * CB);
          qn[i] = load_piece<Q4, false>(a, q0 + r, c0 + KC + c / CB, c % CB);
          if (Q4) qsn[i] = load_qscale(a, q0 + r, c0 + KC + c);
        }
      }
      const int S = chunk_s<CS>(a.nblk, c0), first = (once ? c0 : half * KC) + h * S;
      multiply<XB, Q4, QT, IT, CS, STRIDE, SSTRIDE>(qrow, qsrow, first, S, cur, acc);
      if (CS > 1 && !once && more) {
#pragma unroll
        for (int i = 0; i < QREGS; ++i) {
          const int e = threadIdx.x + i * THREADS, r = e / (KC * CB), c = e % (KC * CB);
          *(uint4*)(ql + r * STRIDE + (half ^ 1) * (KC * QBYTES) + c * 16) = settle<Q4>(a, c0 + KC + c / CB, c % CB, qn[i]);
          if (Q4) qsl[r * SSTRIDE + (half ^ 1) * KC + c] = qsn[i];
        }
        half ^= 1;
        __syncthreads();
      }
      cur = nxt;
    }
    // (one pointer, moved from row to row: kept per row, the addresses would fill the registers)
    constexpr int ES = T == T_F32 ? 4 : 2;
    const int left = (int)min(a.N - row0, (int64_t)IT), rows = a.B - q0 - 4 * h;
    const bool whole = a.vec && left == IT;
    char* o = (char*)a.out + ((int64_t)(q0 + 4 * h) * a.ld + row0) * ES;
    const int64_t down = a.ld * ES;
    if (left > 0) {
#pragma unroll
      for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float v[IT];
#pragma unroll
          for (int t = 0; t < IT; ++t) v[t] = acc[t][q][r];
          if (q * 32 + (r & 3) + 8 * (r >> 2) < rows) store_scores<T, IT>(o, whole, left, v);
          o += (r & 3) == 3 ? 5 * down : down;
        }
    }
  }
}

// Few tiles and long rows: the four waves of a workgroup take the same 64 table rows and every fourth
// chunk each, and their sums are joined in LDS.  (The rule, with both sides measured, is where it is
// launched.)
template <int XB, bool Q4, int T>
__global__ void __launch_bounds__(THREADS, 2) mx_score_split_kernel(Args a) {
  constexpr int QT = 1, IT = 2, CS = 2, KC = 2 * CS, LB = WAVES * KC;
  constexpr int QBYTES = Q4 ? 16 : 64, CB = QBYTES / 16;
  constexpr int STRIDE = LB * QBYTES + 16, SSTRIDE = LB + 4;
  constexpr int QL = 32 * QT * STRIDE, RED = WAVES * 32 * QT * 64 * 4;
  __shared__ __attribute__((aligned(16))) uint8_t ql[QL > RED ? QL : RED];
  __shared__ __attribute__((aligned(16))) uint8_t qsl[Q4 ? 32 * QT * SSTRIDE : 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int tile = xcd_remap(blockIdx.x, a.qtiles * a.itiles);
  const int q0 = tile % a.qtiles * 32 * QT;
  const int64_t row0 = (int64_t)(tile / a.qtiles) * (32 * IT) + (lane & 31) * IT;
  const uint8_t* qrow = ql + (lane & 31) * STRIDE;
  const uint8_t* qsrow = qsl + (lane & 31) * SSTRIDE;
  f32x16 acc[IT][QT];
#pragma unroll
  for (int t = 0; t < IT; ++t)
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][q][r] = 0.f;
  Chunk<XB, IT, CS> cur, nxt;
  const int c1 = wave * KC;
  if (c1 < a.nblk) load_chunk<XB, IT, CS>(a, row0, c1, h, cur);
  settle_loads();  // (else cur's first use in the loop waits, every time, for nxt as well)
  for (int s0 = 0; s0 < a.nblk; s0 += LB) {
    const int c0 = s0 + c1;
    if (c0 + LB < a.nblk) load_chunk<XB, IT, CS>(a, row0, c0 + LB, h, nxt);
    __syncthreads();
    stage_queries<Q4, false, QT, STRIDE, SSTRIDE, 4>(a, q0, s0, LB * CB, ql, qsl);
    __syncthreads();
    if (c0 < a.nblk) {
      const int S = chunk_s<CS>(a.nblk, c0);
      multiply<XB, Q4, QT, IT, CS, STRIDE, SSTRIDE>(qrow, qsrow, c1 + h * S, S, cur, acc);
    }
    cur = nxt;
  }
  __syncthreads();
  float* red = (float*)ql;
#pragma unroll
  for (int t = 0; t < IT; ++t)
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int r = 0; r < 16; ++r) red[((wave * IT + t) * QT + q) * 1024 + r * 64 + lane] = acc[t][q][r];
  __syncthreads();
  // wave w joins registers 4 w .. 4 w + 3: queries 8 w + (0 .. 3) + 4 h of each 32
  constexpr int ES = T == T_F32 ? 4 : 2;
  const int left = (int)min(a.N - row0, (int64_t)IT);
  const bool whole = a.vec && left == IT;
  if (left <= 0) return;
#pragma unroll
  for (int q = 0; q < QT; ++q)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = q0 + q * 32 + 8 * wave + i + 4 * h;
      float v[IT];
#pragma unroll
      for (int t = 0; t < IT; ++t) {
        const float* p = red + (t * QT + q) * 1024 + (4 * wave + i) * 64 + lane;
        v[t] = (p[0] + p[IT * QT * 1024]) + (p[2 * IT * QT * 1024] + p[3 * IT * QT * 1024]);
      }
      if (b < a.B) store_scores<T, IT>((char*)a.out + ((int64_t)b * a.ld + row0) * ES, whole, left, v);
    }
}

template <int XB, bool Q4>
void launch_split(Args& a, int type, hipStream_t st) {
  a.vec = (a.B == 1 || a.ld % 2 == 0) && ((uintptr_t)a.out & (type == T_F32 ? 7 : 3)) == 0;
  a.qtiles = (a.B + 31) / 32;
  a.itiles = (int)((a.N + 63) / 64);
  const dim3 grid((unsigned)(a.qtiles * a.itiles));
  if (type == T_F32) hipLaunchKernelGGL((mx_score_split_kernel<XB, Q4, T_F32>), grid, dim3(THREADS), 0, st, a);
  else if (type == T_BF16) hipLaunchKernelGGL((mx_score_split_kernel<XB, Q4, T_BF16>), grid, dim3(THREADS), 0, st, a);
  else hipLaunchKernelGGL((mx_score_split_kernel<XB, Q4, T_F16>), grid, dim3(THREADS), 0, st, a);
}

template <int XB, bool Q4, int QT, int IT, int CS, int LB, int T>
void launch_as(Args& a, hipStream_t st) {
  const int es = T == T_F32 ? 4 : 2;
  a.vec = (a.B == 1 || a.ld % IT == 0) && ((uintptr_t)a.out & (IT * es - 1)) == 0;
  a.qtiles = (a.B + 32 * QT - 1) / (32 * QT);
  a.itiles = (int)((a.N + WAVES * 32 * IT - 1) / (WAVES * 32 * IT));
  int64_t grid = (int64_t)a.qtiles * a.itiles;
  if (CS == 1 || a.nblk <= LB) {
    // about four workgroups a CU, a multiple of 8 per query tile
    const int64_t per = max((int64_t)1, min(((int64_t)a.itiles + 7) / 8, (int64_t)1024 / (8 * a.qtiles)));
    grid = per * 8 * a.qtiles;
  }
  hipLaunchKernelGGL((mx_score_kernel<XB, Q4, QT, IT, CS, LB, T>), dim3((unsigned)grid), dim3(THREADS), 0, st, a);
}

template <int XB, bool Q4, int QT, int IT, int CS, int LB>
void launch(Args& a, int type, hipStream_t st) {
  if (type == T_F32) launch_as<XB, Q4, QT, IT, CS, LB, T_F32>(a, st);
  else if (type == T_BF16) launch_as<XB, Q4, QT, IT, CS, LB, T_BF16>(a, st);
  else launch_as<XB, Q4, QT, IT, CS, LB, T_F16>(a, st);
}

// By the width of the rows and the number of queries (us; fp4 table, bf16 queries where not said).
// One or two blocks a row: a block a lane; so many rows a lane that a store of many queries' scores is 256
// bytes long (2 against 4 rows: 300 x 200000 x 64 fp32 scores 40.3 / 44.1, 256 x 1M x 64 bf16 ones 120.6 /
// 115.6), two for few queries (more waves in flight: one query x 1M x 64 11.6 against 13.7).  Longer
// rows: chunks of 2 blocks a lane, of 4 for fp4 where that fills chunks (2 against 4: 256 x 100003 x
// 300 36.9 / 41.2, 1 x 1M x 128 17.7 / 19.6, but 64 x 65536 x 4096 62.6 / 60.1, 8 x 65536 x 4096 42.0 /
// 37.2; fp4 queries, 37 x 300000 x 512 31.4 / 26.1; fp8 table with 4 blocks, 37 x 100003 x 300 23.2 / 16.5).
// QT = 2 query tiles a wave is what the registers hold beside them (QT = 4, spilling: 512 x 65536 x 4096 417
// against 351 when it was tried; 287 since, 484 for an fp8 table).
template <int XB, bool Q4>
void launch_rows(Args& a, bool few, int type, hipStream_t st) {
  if (a.nblk <= 2) {
    if (few) launch<XB, Q4, 1, 2, 1, 2>(a, type, st);
    else if (type == T_F32) launch_as<XB, Q4, 2, 2, 1, 2, T_F32>(a, st);
    else if (type == T_BF16) launch_as<XB, Q4, 2, 4, 1, 2, T_BF16>(a, st);
    else launch_as<XB, Q4, 2, 4, 1, 2, T_F16>(a, st);
  } else if (few) {
    if (XB == 8 || a.nblk <= 4) launch<XB, Q4, 1, 2, 2, 32>(a, type, st);
    else if constexpr (XB == 4) launch<XB, Q4, 1, 2, 4, 32>(a, type, st);
  } else {
    if (XB == 8 || a.nblk <= (Q4 ? 12 : 32)) launch<XB, Q4, 2, 2, 2, 16>(a, type, st);
    else if constexpr (XB == 4) launch<XB, Q4, 2, 2, 4, 16>(a, type, st);
  }
}

// Both sides in 4 bits, many queries, long rows: bound by the matrix instructions, so both operands
// go through LDS (a table row is used by two waves, a query by four) and the loads are whole cache
// lines.  A workgroup of 8 waves owns 256 queries x 256 table rows, a wave 128 x 64.  A chunk is 256
// values of every row, 8 pieces of 16 bytes: the next chunk moves from memory to the other LDS
// buffer, past the registers, during the present one's products.  Piece p of row r lies in slot
// p ^ (r' & 7) of its 128 bytes (r' = r for queries; r / 2 for table rows, of which a lane takes
// two neighbours), so the lanes of an access phase, 8 rows of one piece, fall into distinct banks.
// Blocks past the row's end are loaded as some block that is there and given the scale 2^-127 on
// both sides: their products vanish below fp32's range.
typedef __attribute__((address_space(3))) uint8_t LdsByte;
// 16 bytes a lane from base + off to LDS, lane after lane from byte `to` on.  In assembly because the
// compiler waits for every such load of its own before the next read of LDS, whichever buffer that
// is of; here wait_loads() does, before the barrier that hands the buffer over.  (m0 holds the
// destination; a load to LDS may read it one wait state after it is written, and the compiler puts
// none inside a block.  Nothing is returned in registers.)
__device__ __forceinline__ void load_to_lds(const uint8_t* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

constexpr int WT = 256;   // queries and table rows per workgroup
constexpr int WTHREADS = 512;
constexpr int WCHUNK = 8; // blocks per chunk

struct WideLds {
  uint8_t data[2][2][WT * 128];     // buffer, operand (0: queries)
  uint32_t scale[2][2][2][WT];      // buffer, operand, half of the chunk
};

template <int T>
__global__ void __launch_bounds__(WTHREADS, 2) mx_score_wide_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) WideLds lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l = lane & 31;
  const int tile = xcd_remap(blockIdx.x, a.qtiles * a.itiles);
  const int q0 = tile % a.qtiles * WT;
  const int64_t i0 = (int64_t)(tile / a.qtiles) * WT;
  const int wq = (wave & 1) * 128, wi = (wave >> 1) * 64;
  // This wave brings in 8 x 8 rows, 4 x 8 of each operand: a lane moves 16 bytes straight to LDS, eight
  // lanes one row's 128; slot i of a row gets the piece that the rule above puts there.
  const uint32_t row_bytes = (uint32_t)a.nblk * 16;
  const uint8_t* qbase = (const uint8_t*)a.q + (int64_t)q0 * row_bytes;
  const uint8_t* xbase = a.x + i0 * row_bytes;
  const int qlast = min(a.B - q0, WT) - 1, xlast = (int)min(a.N - i0, (int64_t)WT) - 1;  // rows past the end: the last again
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(LdsByte*)lds.data[0][0] + wave * 4096);
  const int srow = tid & (WT - 1), sop = tid >> 8;
  const uint8_t* ssrc = sop ? a.xs + (i0 + min(srow, xlast)) * a.nblk : a.qs + (int64_t)(q0 + min(srow, qlast)) * a.nblk;
  uint32_t sin0 = 0, sin1 = 0;
  const auto load = [&](int c0, int buf) {
    const int there = c0 + WCHUNK <= a.nblk ? 7 : 3;  // nblk % 4 == 0: the last chunk may hold half
    const uint32_t at = c0 * 16;
    const uint32_t to = lds0 + buf * (2 * WT * 128);
    const int i = lane & 7;
    int r = lane >> 3;  // row & 7 == r, (row >> 1) & 7 == (r >> 1) + 4 (k & 1)
    asm("" : "+v"(r));  // the offsets are computed here: kept over the loop they would not fit the registers
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = (wave * 4 + k) * 8 + r;
      load_to_lds(qbase, min(row, qlast) * row_bytes + at + ((i ^ r) & there) * 16, to + k * 1024);
      load_to_lds(xbase, min(row, xlast) * row_bytes + at + ((i ^ ((r >> 1) + 4 * (k & 1))) & there) * 16,
                  to + WT * 128 + k * 1024);
    }
    sin0 = *(const uint32_t*)(ssrc + c0);
    sin1 = c0 + 4 < a.nblk ? *(const uint32_t*)(ssrc + c0 + 4) : 0u;
  };
  const auto put_scales = [&](int buf) {
    lds.scale[buf][sop][0][srow] = sin0;
    lds.scale[buf][sop][1][srow] = sin1;
  };
  f32x16 acc[2][4];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][q][r] = 0.f;
  load(0, 0);
  put_scales(0);
  wait_loads();
  __syncthreads();
  int buf = 0;
  for (int c0 = 0; c0 < a.nblk; c0 += WCHUNK) {
    const bool more = c0 + WCHUNK < a.nblk;
    const uint8_t* qd = lds.data[buf][0] + (wq + l) * 128;
    const uint8_t* xd = lds.data[buf][1] + (wi + 2 * l) * 128;
    if (more) load(c0 + WCHUNK, buf ^ 1);
    uint32_t qsc[4], xsc[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) qsc[q] = lds.scale[buf][0][h][wq + 32 * q + l];
#pragma unroll
    for (int t = 0; t < 2; ++t) xsc[t] = lds.scale[buf][1][h][wi + 2 * l + t];
    // step j's operands are read during step j - 1's products
    uint4 qa[2][4], xb[2][2];
    const auto read = [&](int j) {
      const int at = ((h * 4 + j) ^ (l & 7)) * 16;
#pragma unroll
      for (int q = 0; q < 4; ++q) qa[j & 1][q] = *(const uint4*)(qd + q * 32 * 128 + at);
#pragma unroll
      for (int t = 0; t < 2; ++t) xb[j & 1][t] = *(const uint4*)(xd + t * 128 + at);
    };
    read(0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < 3) read(j + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint4 u = qa[j & 1][q], v = xb[j & 1][t];
          acc[t][q] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
              i32x8{(int)u.x, (int)u.y, (int)u.z, (int)u.w, 0, 0, 0, 0}, i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0},
              acc[t][q], 4, 4, 0, (int)(qsc[q] >> (8 * j)), 0, (int)(xsc[t] >> (8 * j)));
        }
      __builtin_amdgcn_sched_barrier(0);  // (also: the products are not moved behind the wait)
    }
    put_scales(buf ^ 1);  // (after the last chunk: not read)
    wait_loads();
    __syncthreads();
    buf ^= 1;
  }
  // Eight queries at a time, for which one branch decides: those past the last are jumped over, and where all
  // is there the stores follow each other.  (512 x 20000 x 1024: 17.7 us against 20.3 with conditions for each
  // store; the other kernel's short calls lose by the two copies of the code: 100 x 20000 x 300 8.0 / 6.9.)
  constexpr int ES = T == T_F32 ? 4 : 2;
  const int64_t row0 = i0 + wi + 2 * l;
  const int left = (int)min(a.N - row0, (int64_t)2);
  const bool whole = a.vec && left == 2, full = a.vec && i0 + wi + 64 <= a.N;
  char* o = (char*)a.out + ((int64_t)(q0 + wq + 4 * h) * a.ld + row0) * ES;
  const int64_t down = a.ld * ES;
#pragma unroll
  for (int g = 0; g < 16; ++g) {
    const int first = q0 + wq + 8 * g;
    if (first >= a.B) return;
    float v[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) v[i][t] = acc[t][g >> 2][4 * (g & 3) + i];
    if (full && first + 8 <= a.B) {
#pragma unroll
      for (int i = 0; i < 4; ++i) store_scores<T, 2>(o + i * down, true, 2, v[i]);
    } else if (left > 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (first + 4 * h + i < a.B) store_scores<T, 2>(o + i * down, whole, left, v[i]);
    }
    o += 8 * down;
  }
}

void launch_wide(Args& a, int type, hipStream_t st) {
  a.vec = (a.B == 1 || a.ld % 2 == 0) && ((uintptr_t)a.out & (type == T_F32 ? 7 : 3)) == 0;
  a.qtiles = (a.B + WT - 1) / WT;
  a.itiles = (int)((a.N + WT - 1) / WT);
  const dim3 grid((unsigned)(a.qtiles * a.itiles));
  if (type == T_F32) hipLaunchKernelGGL((mx_score_wide_kernel<T_F32>), grid, dim3(WTHREADS), 0, st, a);
  else if (type == T_BF16) hipLaunchKernelGGL((mx_score_wide_kernel<T_BF16>), grid, dim3(WTHREADS), 0, st, a);
  else hipLaunchKernelGGL((mx_score_wide_kernel<T_F16>), grid, dim3(WTHREADS), 0, st, a);
}

// A launch's threads must fit 32 bits: so many queries a launch (the smallest tile is 32 queries by 256
// rows), 256 at least (with the rows that fit in memory, fewer tiles than that).
int64_t queries_per_launch(int64_t N) {
  const int64_t tiles = (int64_t)UINT32_MAX / WTHREADS, per = tiles / ((N + 255) / 256) * 32 / 256 * 256;
  return min((int64_t)1 << 20, max((int64_t)256, per));
}

int score(const void* q, const void* qs, const void* x, const void* xs, int xbits, int B, int64_t N, int D, void* out,
          int out_type, int64_t ld, hipStream_t st) {
  Args a;
  a.q = q; a.qs = (const uint8_t*)qs; a.x = (const uint8_t*)x; a.xs = (const uint8_t*)xs;
  a.out = out; a.ld = ld; a.N = N; a.B = B; a.D = D;
  a.nblk = (D + MX_BLOCK - 1) / MX_BLOCK;
  a.s_word = a.nblk % 4 == 0 && ((uintptr_t)xs & 3) == 0;
  const bool few = B <= 32;
  // Few queries, long rows and too few rows to give every CU its 256: the waves split the row instead.  (us, whole
  // rows against split: 1000 x 4096 fp4 30.7 / 16.1, fp8 48.3 / 20.2, 30000 x 4096 fp4 34.4 / 20.6,
  // 20000 x 1024 fp4 11.3 / 7.9; 8 queries x 65536 x 4096 fp4 37.0 / 43.1, fp8 72.5 / 63.9, 20 x 65536 x 2048 fp8
  // 31.7 / 34.3, 130000 x 2048 fp4 28.4 / 37.9.)
  if (few && a.nblk >= 16 && N <= 160 * 256) {
    if (qs) launch_split<4, true>(a, out_type, st);
    else if (xbits == 4) launch_split<4, false>(a, out_type, st);
    else launch_split<8, false>(a, out_type, st);
  } else if (qs && !few && a.nblk > 16 && a.nblk < (1 << 20) && a.s_word && ((uintptr_t)qs & 3) == 0) {
    // Both sides in 4 bits and rows long enough to amortise it: the tiled form (us, against the other: 512 x
    // 20000 x 1024 17.4 / 28.0, 64 x 65536 x 4096 39 / 45; few rows leave it few workgroups: 33 x 7 x
    // 4096 29.5 / 22.8).  Its scales are read in words, and its offsets within a tile's 256 rows are 32-bit
    // ones.
    launch_wide(a, out_type, st);
  } else if (qs) {
    launch_rows<4, true>(a, few, out_type, st);
  } else if (xbits == 4) {
    launch_rows<4, false>(a, few, out_type, st);
  } else {
    launch_rows<8, false>(a, few, out_type, st);
  }
  FPS_CHECK_LAUNCH();
  return 0;
}

}  // namespace

// out [B, N] (row stride ld, type 0 fp32 / 1 bf16 / 2 fp16) = q . x^T.  qs == nullptr: q is bf16
// [B, D]; else q holds E2M1 blocks and qs their scales (then xbits must be 4).
FPS_API int fps_mx_score(const void* q, const void* qs, const void* x, const void* xs, int xbits, int B, int64_t N,
                         int D, void* out, int out_type, int64_t ld, void* stream) {
  if (B <= 0 || N <= 0) return 0;
  if (D <= 0 || D > INT32_MAX - MX_BLOCK || (xbits != 4 && xbits != 8) || (qs && xbits != 4) || ld < N || out_type < 0 ||
      out_type > 2)
    return (int)hipErrorInvalidValue;
  if (N > (int64_t)INT32_MAX * 32) return (int)hipErrorInvalidValue;
  const int64_t per = queries_per_launch(N);
  const int64_t nblk = (D + MX_BLOCK - 1) / MX_BLOCK, q_bytes = qs ? nblk * 16 : (int64_t)D * 2;
  for (int64_t b = 0; b < B; b += per) {
    const int rc = score((const char*)q + b * q_bytes, qs ? (const char*)qs + b * nblk : nullptr, x, xs, xbits,
                         (int)min(per, B - b), N, D, (char*)out + b * ld * (out_type == T_F32 ? 4 : 2), out_type, ld,
                         (hipStream_t)stream);
    if (rc) return rc;
  }
  return 0;
}
