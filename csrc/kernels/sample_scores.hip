// One index per row of scores, drawn from the softmax cut by top-k, top-p and min-p, from a
// given uniform number (gfx950).
//
//   w_i  = exp((s_i - max s) / T)                  -inf and NaN are masked (w = 0)
//   top-k  the k best (equal scores: lowest index first)
//   top-p  of those, best first, the ones before which less than p of their mass lies
//   min-p  of those, the ones with w_i >= min_p    (the best one has w = 1)
//   answer the first index i with sum_{j <= i, j kept} w_j > u * sum_{j kept} w_j
//
// Bound by one read of the scores, so a long row (> 16384) is read once in full where it can
// be: the stats pass takes the largest score of every segment of 256 (and its mass, where
// nothing is cut), and the finishing workgroup of a row then reads only segments whose
// largest score can matter: about k of them for a short top-k, one without a cut.  Other
// cuts need counts or masses of all scores above a threshold: passes over the row, spread
// over the chip (a histogram, then the segments' masses above the threshold's bin and a list of
// the scores inside it); a long top-k and then top-p take them twice.  Shorter rows take one
// launch.  (Rows of 16384: 16 us either way without a cut; 32768: 26 us in one launch, 15 so.)
//
// Nothing is sorted.  Thresholds are found over bins of (max s - s) / T, and the scores of the
// bin that holds the threshold are ranked against each other (up to 256 of them) or split
// by the bits of the scores.  Weights are computed in 64 bits: an answer depends on
// which side of u * total a sum of up to N weights falls.  Where masses meet in atomics (the
// histograms, which find thresholds, and the scores listed from a threshold's bin) they are
// whole multiples of a unit taken from the row's own total or the bin's weights, so their order
// does not matter; the other sums, the draw's above all, are 64-bit ones in a fixed order.
#include <hip/hip_fp16.h>

#include "common.h"

using namespace fps;

namespace {

constexpr int SEG = 256;        // scores per segment: one wave, four a lane
constexpr int BINS = 2048;
constexpr int THREADS = 512;    // of a finishing workgroup
constexpr int WAVES = THREADS / 64;
constexpr int PER = BINS / THREADS;   // bins per thread of a search
constexpr int LIST = 1024;      // scores listed in LDS
constexpr int LIST_SHIFT = 51;  // unit 2^-51: all their masses together stay below 2^62
constexpr int RANK = 256;       // listed scores ranked against each other; more are split by bits
constexpr int SHORT_K = 512;    // top-k up to this lists its candidates
constexpr int CACHED_SEGS = 64;      // segments of a row that takes one launch
constexpr int PASS_SEGS = 64;   // segments per workgroup of the passes over long rows

// a listed score: its key above the complement of its index (the larger word is the better score,
// equal scores by the lower index), and its weight
struct Entry {
  uint64_t at;
  uint64_t w;
  __device__ uint32_t key() const { return (uint32_t)(at >> 32); }
  __device__ int32_t idx() const { return (int32_t)~(uint32_t)at; }
};
__device__ __forceinline__ Entry make_entry(uint32_t key, int32_t idx, uint64_t w) {
  return Entry{(uint64_t)key << 32 | (uint32_t)~idx, w};
}

// What the passes over a long row share.  A round finds one threshold: by count (top-k), or by mass
// (top-p) among the scores above `floor_key` and the first `ties` equal to it (what top-k left); or none
// (NO_CUT), for the segments' masses alone.
enum { IDLE = 0, BY_TOP_K = 1, BY_TOP_P = 2, NO_CUT = 3 };
struct RowState {
  int mode;
  float M, cb;         // largest score; bins per unit of score
  int shift;           // masses are multiples of 2^-shift
  uint32_t floor_key, ties;
  double target;       // count, or mass, that the threshold's bin reaches; < 0: p * all mass, which
  double part;         // then stands here
  uint64_t above;      // what the bins before `bin` hold of it
  uint64_t all;        // bin == BINS: what all bins hold
  int bin;             // the threshold's; BINS: all scores above floor_key stay
  uint32_t listed;     // scores in it
};

struct Args {
  const void* s;
  int64_t ld, N, nseg;
  int B;
  const float* u;
  // per row, or nullptr and the same for all rows
  const float* temperature; double temperature0;
  const int32_t* top_k; int64_t top_k0;
  const float* top_p; double top_p0;
  const float* min_p; double min_p0;
  int32_t* out;
  float* prob;
  // workspace (long rows)
  double* segmass;   // [B, nseg]
  uint64_t* hmass;   // [B, BINS]     } rows that may take passes
  Entry* list;       // [B, listcap]  }
  RowState* state;   // [B]           }
  float* segmax;     // [B, nseg]
  int32_t* segtie;   // [B, nseg]
  uint64_t* listed;  // [B, nseg], of rows whose segments do not fit in LDS
  int listcap;
};

struct Row {
  double c;      // log2(e) / T
  double p, minp;
  int64_t k;     // 0: off
  bool cut_p, cut_min;
  __device__ bool direct() const { return k == 0 && !cut_p; }
  __device__ bool by_mass() const { return k == 0 && cut_p; }
  // a top-k for which the k largest scores are listed outright
  __device__ bool short_k() const { return k > 0 && k <= SHORT_K; }
};

__device__ __forceinline__ Row row_settings(const Args& a, int b) {
  Row r;
  const double T = a.temperature ? (double)a.temperature[b] : a.temperature0;
  r.k = a.top_k ? (int64_t)a.top_k[b] : a.top_k0;
  r.p = a.top_p ? (double)a.top_p[b] : a.top_p0;
  r.minp = a.min_p ? (double)a.min_p[b] : a.min_p0;
  r.c = fmin(1.4426950408889634 / T, 1e300);  // finite: 0 * c is 0 at the best score
  if (!(T > 0)) {  // greedy: the best alone
    r.c = 1.4426950408889634;
    r.k = 1;
  }
  if (r.k <= 0 || r.k >= a.N) r.k = 0;
  r.cut_p = r.p < 1;
  r.cut_min = r.minp > 0;
  r.minp = fmin(r.minp, 1.0);
  return r;
}

// order-preserving float -> uint32; masked scores are -inf, the smallest key in use
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float score_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
constexpr uint32_t KEY_NONE = 0x007fffffu;  // key_of(-inf)

// p f + c with the coefficient in scalar registers (the compiler's form copies each coefficient
// into vector registers first: 5 us of a pass over 16.7M scores that takes 27 so)
__device__ __forceinline__ double horner(double p, double f, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(p), "v"(f), "s"(c));
  return r;
}

// 2^((s - M) c) = p 2^n: interpolation of 2^f at the Chebyshev nodes of [-1/2, 1/2], degree 8 (relative
// error 1.1e-12: two answers differ where u * total falls that near to a step), and the power of two.
// (Built from the bits of t + 1.5 * 2^52, with a comparison for what is too small, a pass over 16.7M scores
// took 28.5 us against 26.)
struct Power {
  double p;  // in [0.7, 1.42]; 1 at the best score
  int n;     // -2000 at least, where weights and masses vanish
};
__device__ __forceinline__ Power power(float s, float M, double c) {
  const double t0 = ((double)s - (double)M) * c;  // exactly 0 at the best score
  const double t = fmax(t0, -2000.0);  // (a NaN too: a masked score at an endless temperature)
  const double n = __builtin_rint(t);
  const double f = t - n;
  double p = 0x1.63d1363a7ecb6p-20;
  p = horner(p, f, 0x1.00dc4a534054dp-16);
  p = horner(p, f, 0x1.4308ac85a6c21p-13);
  p = horner(p, f, 0x1.5d8745a72827ap-10);
  p = horner(p, f, 0x1.3b2ab7181b778p-7);
  p = horner(p, f, 0x1.c6b08dd6fd236p-5);
  p = horner(p, f, 0x1.ebfbdff823cedp-3);
  p = horner(p, f, 0x1.62e42fef84cf0p-1);
  p = horner(p, f, 0x1.0000000000000p+0);
  return Power{p, (int)n};
}
__device__ __forceinline__ double weight(float s, float M, double c) {
  if (M == INFINITY) return s == M ? 1.0 : 0.0;  // (one branch for a whole row)
  const Power w = power(s, M, c);
  return __builtin_ldexp(w.p, w.n);
}

// A weight as a whole multiple of 2^-shift: the significand with its leading one in bit 62, moved down.
// `place` (0 .. 255, a score's place in its segment; without it the rest below the unit is cut off) spreads
// the rounding: place / 256 of a unit is added first, so that of equal scores all over a segment so many
// are rounded up that their sum is right to one unit, and others' errors have no common sign.
// weight * 2^shift may reach 2^60.
__device__ __forceinline__ uint64_t mass(float s, float M, double c, int shift, uint32_t place = 0) {
  if (M == INFINITY) return s == M ? 1ull << shift : 0ull;
  const Power w = power(s, M, c);
  const uint64_t bits = (uint64_t)__double_as_longlong(w.p);
  uint64_t m = (bits << 10 & 0x3fffffffffffffffull) | 1ull << 62;
  const int down = 63 - shift - w.n - (int)(bits >> 52 & 1);  // (p in [1, 2) or [1/2, 1))
  m += ((uint64_t)place << 56) >> (-down & 63);  // (down in 1 .. 63; past that nothing is left)
  return down > 63 ? 0 : m >> (down & 63);
}
// The unit for a row whose weights sum up to `total` at most (and 1 at least): all masses together stay
// below 2^62, and what rounding takes from N scores is about 2^-69 N of a total that is known to a factor
// of two.  (By the length of the row, as if every weight were 1, a best score over a flat tail loses the
// tail: each of a million scores cut at 2^-42.)
__device__ __forceinline__ int shift_for(double total) {
  return min(60, 61 - (int)((__double_as_longlong(total) >> 52) - 1023));
}

// (the median of three with a NaN is the smallest of the others, and a NaN is made by s = M alone, with an
// infinite M or cb, or by all scores alike, with cb = 0)
__device__ __forceinline__ int bin_of(float s, float M, float cb) {
  return (int)__builtin_amdgcn_fmed3f((M - s) * cb, 0.f, (float)(BINS - 1));
}

// loads of four scores: a row may start at any score
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2), aligned(2)));

// NaN is masked; -0 and +0 are one score
__device__ __forceinline__ float clean(float f) { return fmaxf(f + 0.f, -INFINITY); }

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// This lane's four scores of a segment as they lie in memory; places past the row are masked.  They are
// unpacked where they are used, and a wave takes one branch for a group of segments: converted at once,
// or with a branch for each, a load would be waited for before the next is sent (softmax over 16M fp32
// scores: stats pass 24 us against 21).
template <int T> struct Raw { u32x2 w; };
template <> struct Raw<T_F32> { f32x4 f; };

template <int T, int G>
__device__ __forceinline__ void load_segs(const Args& a, int b, int lane, const int64_t (&seg)[G], Raw<T> (&r)[G]) {
  bool whole = true;
#pragma unroll
  for (int g = 0; g < G; ++g) whole = whole && (seg[g] + 1) * SEG <= a.N;
  const int64_t row = (int64_t)b * a.ld + lane * 4;
  if (whole) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if constexpr (T == T_F32) r[g].f = *(const f32x4*)((const float*)a.s + row + seg[g] * SEG);
      else r[g].w = *(const u32x2*)((const uint16_t*)a.s + row + seg[g] * SEG);
    }
  } else {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int64_t i = seg[g] * SEG + lane * 4;
      if constexpr (T == T_F32) {
        const float* p = (const float*)a.s + row + seg[g] * SEG;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[g].f[j] = i + j < a.N ? p[j] : -INFINITY;
      } else {
        const uint16_t* p = (const uint16_t*)a.s + row + seg[g] * SEG;
        const uint32_t none = T == T_BF16 ? 0xff80u : 0xfc00u;  // -inf
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = i + j < a.N ? p[j] : none;
        r[g].w = u32x2{h[0] | h[1] << 16, h[2] | h[3] << 16};
      }
    }
  }
}
// G segments of a row, `step` apart (those behind the row's last: the last again)
template <int T, int G>
__device__ __forceinline__ void load_segs(const Args& a, int b, int lane, int64_t first, int step, Raw<T> (&r)[G]) {
  int64_t seg[G];
#pragma unroll
  for (int g = 0; g < G; ++g) seg[g] = min(first + g * step, a.nseg - 1);
  load_segs<T, G>(a, b, lane, seg, r);
}
template <int T>
__device__ __forceinline__ void unpack(const Raw<T>& r, float v[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (T == T_F32) {
      v[j] = r.f[j];
    } else {
      const uint16_t h = (uint16_t)(r.w[j >> 1] >> (16 * (j & 1)));
      v[j] = T == T_BF16 ? bf16_to_f32(h) : __half2float(__ushort_as_half(h));
    }
    v[j] = clean(v[j]);
  }
}
template <int T>
__device__ __forceinline__ void load_seg(const Args& a, int b, int64_t seg, int lane, float v[4]) {
  const int64_t at[1] = {seg};
  Raw<T> raw[1];
  load_segs<T, 1>(a, b, lane, at, raw);
  unpack<T>(raw[0], v);
}
template <int T>
__device__ __forceinline__ float load_score(const Args& a, int b, int64_t i) {
  const int64_t at = (int64_t)b * a.ld + i;
  if (T == T_F32) return clean(((const float*)a.s)[at]);
  const uint16_t h = ((const uint16_t*)a.s)[at];
  return clean(T == T_BF16 ? bf16_to_f32(h) : __half2float(__ushort_as_half(h)));
}
__device__ __forceinline__ float max4(const float v[4]) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); }

// ---- wave and workgroup sums ---------------------------------------------------------------
// A step of a 64-lane scan: the value `from` lanes below inside rows of 16 (CTRL 0x111 .. 0x118), or
// the last of the row(s) before (0x142, 0x143); 0 where there is none.  Register moves
// between lanes: a step costs a few cycles where a shuffle through LDS costs ~100.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lanes_below(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, ROWS == 0xf);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t lanes_below(uint64_t v) {
  return (uint64_t)lanes_below<CTRL, ROWS>((uint32_t)v) | ((uint64_t)lanes_below<CTRL, ROWS>((uint32_t)(v >> 32)) << 32);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double lanes_below(double v) {
  return __longlong_as_double((int64_t)lanes_below<CTRL, ROWS>((uint64_t)__double_as_longlong(v)));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float lanes_below(float v) {
  return __uint_as_float(lanes_below<CTRL, ROWS>(__float_as_uint(v)));
}
// inclusive sum over the lanes of the wave (all 64 active)
template <typename V>
__device__ __forceinline__ V wave_scan(V v) {
  v += lanes_below<0x111, 0xf>(v);
  v += lanes_below<0x112, 0xf>(v);
  v += lanes_below<0x114, 0xf>(v);
  v += lanes_below<0x118, 0xf>(v);
  v += lanes_below<0x142, 0xa>(v);
  v += lanes_below<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int l) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int l) {
  return (uint64_t)lane_value((uint32_t)v, l) | ((uint64_t)lane_value((uint32_t)(v >> 32), l) << 32);
}
__device__ __forceinline__ float lane_value(float v, int l) { return __uint_as_float(lane_value(__float_as_uint(v), l)); }
__device__ __forceinline__ double lane_value(double v, int l) {
  return __longlong_as_double((int64_t)lane_value((uint64_t)__double_as_longlong(v), l));
}
// The total, which only the last lane has to come by: the steps between rows go to all rows, the moves
// need no cleared register before them, and 32-bit ones are operands of the sums.  The order is the scan's.
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
  v += lanes_below<0x111, 0xf>(v);
  v += lanes_below<0x112, 0xf>(v);
  v += lanes_below<0x114, 0xf>(v);
  v += lanes_below<0x118, 0xf>(v);
  v += lanes_below<0x142, 0xf>(v);
  v += lanes_below<0x143, 0xf>(v);
  return lane_value(v, 63);
}
// (over keys: where no lane is below, 0 takes part, the smallest of them)
__device__ __forceinline__ float wave_max(float f) {
  uint32_t v = key_of(f);
  v = max(v, lanes_below<0x111, 0xf>(v));
  v = max(v, lanes_below<0x112, 0xf>(v));
  v = max(v, lanes_below<0x114, 0xf>(v));
  v = max(v, lanes_below<0x118, 0xf>(v));
  v = max(v, lanes_below<0x142, 0xf>(v));
  v = max(v, lanes_below<0x143, 0xf>(v));
  return score_of(lane_value(v, 63));
}

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t min_below(uint32_t v) {
  return min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
  v = min_below<0x111, 0xf>(v);
  v = min_below<0x112, 0xf>(v);
  v = min_below<0x114, 0xf>(v);
  v = min_below<0x118, 0xf>(v);
  v = min_below<0x142, 0xa>(v);
  v = min_below<0x143, 0xc>(v);
  return lane_value(v, 63);
}

// inclusive sum over the workgroup in thread order, and the total; tmp: one V per wave
template <typename V>
__device__ __forceinline__ V block_scan(V v, V* tmp, V& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if (lane == 63) tmp[wave] = v;
  __syncthreads();
  V t = lane < nw ? tmp[lane] : V(0);
  t = wave_scan(t);
  total = lane_value(t, nw - 1);
  return wave ? lane_value(t, wave - 1) + v : v;
}

__device__ __forceinline__ float block_max(float v, float* tmp) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  const int nw = blockDim.x >> 6, lane = threadIdx.x & 63;
  return wave_max(lane < nw ? tmp[lane] : -INFINITY);
}

// ---- long rows, pass 1: the largest score of every segment, its mass where masses decide ----
constexpr int STAT_SEGS = 4;  // per wave
template <int T>
__global__ void __launch_bounds__(256) stats_kernel(Args a) {
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const Row r = row_settings(a, b);
  const int64_t seg0 = ((int64_t)blockIdx.x * 4 + wave_id()) * STAT_SEGS;
  if (seg0 >= a.nseg) return;
  const bool exact = r.direct() && !r.cut_min;
  // rows that cut by mass: fp32 sums, for the unit of their masses and to place the histogram's bins
  const bool rough = r.by_mass();
  // A sum may be too large (it costs the masses bits), never too small (they would pass 64 bits): a temperature at
  // which scores that differ by more than fp32's range may still have weight gives every score 1.
  const bool flat = r.c < 0x1p-100;
  const float cf = fminf((float)r.c, 0x1p100f);
  Raw<T> raw[STAT_SEGS];
  load_segs<T, STAT_SEGS>(a, b, lane, seg0, 1, raw);
  float ms = -INFINITY;
  double ws = 0;
#pragma unroll
  for (int j = 0; j < STAT_SEGS; ++j) {
    float v[4];
    unpack<T>(raw[j], v);
    const float m = wave_max(max4(v));
    if (lane == j) ms = m;
    if (exact) {
      double w = 0;
      if (m > -INFINITY) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w += weight(v[i], m, r.c);
        w = wave_sum(w);
      }
      if (lane == j) ws = w;
    } else if (rough) {
      float w = 0;  // (nothing reads that of a segment without scores)
      if (m < INFINITY && !flat) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w += __builtin_amdgcn_exp2f((v[i] - m) * cf);
      } else {
        const float least = m < INFINITY ? -__FLT_MAX__ : m;
#pragma unroll
        for (int i = 0; i < 4; ++i) w += v[i] >= least ? 1.f : 0.f;
      }
      w = wave_sum(w);
      if (lane == j) ws = w;
    }
  }
  if (lane < STAT_SEGS && seg0 + lane < a.nseg) {
    const int64_t at = (int64_t)b * a.nseg + seg0 + lane;
    a.segmax[at] = ms;
    if (exact || rough) a.segmass[at] = ws;
  }
}

// ---- histograms ----------------------------------------------------------------------------

// add one score to a histogram in LDS; a wave whose lanes all hit one bin adds once
template <bool COUNT, bool MASS>
__device__ __forceinline__ void hist_add(uint32_t* hc, unsigned long long* hm, bool on, int bin, uint64_t w) {
  const uint64_t live = __ballot(on);
  if (live == 0) return;
  const int first = __builtin_amdgcn_readlane(bin, __ffsll((unsigned long long)live) - 1);
  if (__ballot(on && bin == first) == live) {
    uint64_t sum = 0;
    if (MASS) sum = wave_sum(on ? w : (uint64_t)0);
    if ((threadIdx.x & 63) == 0) {
      if (COUNT) atomicAdd(hc + first, (uint32_t)__popcll(live));
      if (MASS) atomicAdd(hm + first, (unsigned long long)sum);
    }
  } else if (on) {
    if (COUNT) atomicAdd(hc + bin, 1u);
    if (MASS) atomicAdd(hm + bin, (unsigned long long)w);
  }
}

constexpr int WANTED = 8 * THREADS;  // segments looked at together
constexpr int KEPT = 8 * THREADS;    // segments' maxima that a long row's workgroup keeps in LDS

template <bool COUNTS>
struct Hist {
  unsigned long long hm[BINS];
  uint32_t hc[COUNTS ? BINS : 1];
  uint64_t scan_m[WAVES];
  uint32_t scan_c[WAVES];
  int wave_hit[WAVES], wave_any[WAVES];
  // what a search found, written by one thread
  int bin;
  uint32_t before_c;
  unsigned long long before_m;
  double target;
};

struct Shared : Hist<true> {
  Entry list[LIST];
  uint32_t rank[RANK];
  unsigned long long before[RANK];
  uint16_t segs[WANTED];
  int nsegs, seg_base, n;
  float tmp[WAVES];
  double scan_d[WAVES];
  uint32_t kmin, ties;
  unsigned long long kept_m;
};

__device__ __forceinline__ void clear_hist(Shared& sh) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS) { sh.hc[i] = 0; sh.hm[i] = 0; }
  __syncthreads();
}

// the first value of the wave's lanes that have one (-1: none), and the last
__device__ __forceinline__ int first_of(int v) {
  const uint64_t m = __ballot(v >= 0);
  return m ? __builtin_amdgcn_readlane(v, __ffsll((unsigned long long)m) - 1) : -1;
}
__device__ __forceinline__ int last_of(int v) {
  const uint64_t m = __ballot(v >= 0);
  return m ? __builtin_amdgcn_readlane(v, 63 - __clzll(m)) : -1;
}

enum Search { BY_COUNT, BY_COUNT_WITH_MASS, BY_MASS };

// The bin of the histogram in sh (bin 0 best) in which the count first reaches `need`, or the mass,
// added to `above`, first reaches the target: sh.bin, and what lies before it: sh.before_c,
// sh.before_m.  part >= 0: the target is that part of all mass (sh.target).  Where rounding lets no
// bin reach it: the last bin that holds anything.
template <Search S, typename H>
__device__ __forceinline__ void find_bin(H& sh, uint32_t need, uint64_t above = 0, double target = 0, double part = -1) {
  const int i = threadIdx.x, lane = i & 63, wave = wave_id();
  uint32_t c[PER], ct = 0, cc = 0, call;
  uint64_t m[PER], mt = 0, mm = 0, mall;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    c[j] = S == BY_MASS ? 0 : sh.hc[PER * i + j];
    m[j] = S == BY_COUNT ? 0 : sh.hm[PER * i + j];
    ct += c[j];
    mt += m[j];
  }
  if (S != BY_MASS) cc = block_scan(ct, sh.scan_c, call) - ct;
  if (S != BY_COUNT) mm = block_scan(mt, sh.scan_m, mall) - mt;
  if (S == BY_MASS && part >= 0) target = part * (double)mall;
  int hit = -1, any = -1;
  uint32_t c_hit = 0, c_any = 0;
  uint64_t m_hit = 0, m_any = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (S == BY_MASS ? m[j] != 0 : c[j] != 0) {
      any = PER * i + j;
      c_any = cc;
      m_any = mm;
      if (hit < 0 && (S == BY_MASS ? (double)(above + mm + m[j]) >= target : cc + c[j] >= need)) {
        hit = any;
        c_hit = cc;
        m_hit = mm;
      }
    }
    cc += c[j];
    mm += m[j];
  }
  const int wh = first_of(hit), wa = last_of(any);
  if (lane == 0) { sh.wave_hit[wave] = wh; sh.wave_any[wave] = wa; }
  __syncthreads();
  int bin = -1, last = -1;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (bin < 0) bin = sh.wave_hit[w];
    last = max(last, sh.wave_any[w]);
  }
  const bool found = bin >= 0;
  if (!found) bin = last;
  if (bin == (found ? hit : any)) {
    sh.bin = bin;
    sh.before_c = found ? c_hit : c_any;
    sh.before_m = found ? m_hit : m_any;
    sh.target = target;
  }
  __syncthreads();
}

// ---- the finishing workgroup of a row ------------------------------------------------------

// Where it has the row: its one segment per wave in registers (ROW_REGS), or in memory, the
// segments' maxima in LDS (ROW_CACHED) or from the stats pass (ROW_LONG).
enum { ROW_REGS = 0, ROW_CACHED = 1, ROW_LONG = 2 };

template <int T, int R>
struct Source {
  const Args& a;
  const int b, lane, wave;
  const float* in_lds;   // the maxima, or
  const float* in_memory;
  float v[4];
  __device__ Source(const Args& a_, int b_, const float* lds, const float* memory)
      : a(a_), b(b_), lane(threadIdx.x & 63), wave(wave_id()), in_lds(lds), in_memory(memory) {}
  __device__ __forceinline__ bool kept() const { return R != ROW_LONG || a.nseg <= KEPT; }
  __device__ __forceinline__ float segmax(int64_t s) const { return kept() ? in_lds[s] : in_memory[s]; }
  // inside each_batch's f: the segment at a place
  __device__ __forceinline__ int32_t segment(const Shared& sh, int place) const { return sh.seg_base + sh.segs[place]; }
  // f(segment, scores) for the segments whose largest score (not -inf) is wanted.
  template <typename P, typename F>
  __device__ __forceinline__ void each(Shared& sh, P want, F f) {
    each_batch<4>(sh, want, [&](const int64_t* seg, const float (*x)[4], int count, int) {
#pragma unroll
      for (int j = 0; j < (R == ROW_REGS ? 1 : 4); ++j)
        if (j < count) f(seg[j], x[j]);
    });
  }
  // f(segments, scores, how many, place of the first): up to G of them.  The segments' maxima are looked
  // at first, many together; the waves share out the wanted ones and load G at a time.
  template <int G, typename P, typename F>
  __device__ __forceinline__ void each_batch(Shared& sh, P want, F f) {
    if constexpr (R == ROW_REGS) {
      const int64_t seg[1] = {wave};
      if (wave < a.nseg) f(seg, &v, 1, 0);
    } else {
      for (int64_t base = 0; base < a.nseg; base += WANTED) {
        __syncthreads();
        if (threadIdx.x == 0) { sh.nsegs = 0; sh.seg_base = (int)base; }
        float m[WANTED / THREADS];
#pragma unroll
        for (int j = 0; j < WANTED / THREADS; ++j) {
          const int64_t at = base + j * THREADS + threadIdx.x;
          m[j] = at < a.nseg ? segmax(at) : -INFINITY;
        }
        __syncthreads();
        uint64_t mask[WANTED / THREADS];
        int total = 0, at = 0;
#pragma unroll
        for (int j = 0; j < WANTED / THREADS; ++j) {
          mask[j] = __ballot(m[j] > -INFINITY && want(m[j]));
          total += __popcll(mask[j]);
        }
        if (total) {
          if (lane == 0) at = atomicAdd(&sh.nsegs, total);
          at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
          for (int j = 0; j < WANTED / THREADS; ++j) {
            if (mask[j] >> lane & 1) sh.segs[at + __popcll(mask[j] & ((1ull << lane) - 1))] = (uint16_t)(j * THREADS + threadIdx.x);
            at += __popcll(mask[j]);
          }
        }
        __syncthreads();
        const int n = sh.nsegs;
        for (int q = wave * G; q < n; q += G * WAVES) {
          Raw<T> x[G];
          int64_t seg[G];
#pragma unroll
          for (int j = 0; j < G; ++j) seg[j] = base + __builtin_amdgcn_readfirstlane((int)sh.segs[min(q + j, n - 1)]);
          load_segs<T, G>(a, b, lane, seg, x);
          float y[G][4];
#pragma unroll
          for (int j = 0; j < G; ++j) unpack<T>(x[j], y[j]);
          f(seg, y, min(n - q, G), q);
        }
      }
    }
  }
};

// The walk of every listed score (n <= RANK) over the list is shared out: a group of G waves has a
// lane per score, each of the WAVES / G groups takes a part of the list.
struct Share {
  int i, j0, j1;  // this lane's score; its part of the list
};
__device__ __forceinline__ Share share_list(int n) {
  const int wave = wave_id();
  const int G = n <= 64 ? 1 : n <= 128 ? 2 : 4;
  const int parts = WAVES / G, part = wave / G, per = (n + parts - 1) / parts;
  return Share{(wave % G) * 64 + (int)(threadIdx.x & 63), min(n, part * per), min(n, (part + 1) * per)};
}

// Thread i < n: is score i among the best k (k = 0: all), given above_c better ones outside the list, and
// what mass of the list is better than it; sh.kept_m: the mass that top-k keeps.
struct Slot {
  bool kept;
  uint64_t before;
};

__device__ __forceinline__ Slot rank_list(Shared& sh, int n, int64_t k, uint32_t above_c) {
  const int i = threadIdx.x;
  if (i < RANK) { sh.rank[i] = 0; sh.before[i] = 0; }
  const Share w = share_list(n);
  uint64_t mine = 0;
  if (w.i < n) mine = sh.list[w.i].at;
  uint32_t rank = 0;
  uint64_t before = 0;
#pragma unroll 4
  for (int j = w.j0; j < w.j1; ++j) {
    const Entry o = sh.list[j];
    const bool better = o.at > mine;
    rank += better;
    before += better ? o.w : (uint64_t)0;
  }
  __syncthreads();
  if (w.i < n) {
    atomicAdd(&sh.rank[w.i], rank);
    atomicAdd(&sh.before[w.i], (unsigned long long)before);
  }
  __syncthreads();
  Slot s{false, 0};
  uint64_t weight = 0, all;
  if (i < n) {
    s.before = sh.before[i];
    s.kept = k == 0 || (int64_t)above_c + sh.rank[i] < k;
    if (s.kept) weight = sh.list[i].w;
  }
  block_scan(weight, sh.scan_m, all);
  if (i == 0) sh.kept_m = all;
  __syncthreads();
  return s;
}

__device__ __forceinline__ void cut_by_mass(Slot& s, uint64_t above_m, double target) {
  const uint64_t before = above_m + s.before;
  s.kept = s.kept && (before == 0 || (double)before < target);  // the best one always stays
}

// the kept entries of the list as a threshold: smallest key, and how many of it
__device__ __forceinline__ void list_threshold(Shared& sh, const Slot& s) {
  if (threadIdx.x == 0) { sh.kmin = 0xffffffffu; sh.ties = 0; }
  __syncthreads();
  const uint32_t key = s.kept ? sh.list[threadIdx.x].key() : 0xffffffffu;
  const uint32_t least = wave_min(key);
  if ((threadIdx.x & 63) == 0) atomicMin(&sh.kmin, least);
  __syncthreads();
  if (s.kept && key == sh.kmin) atomicAdd(&sh.ties, 1u);
  __syncthreads();
}

// Places in a list for the scores of a segment that the lanes want (on[4]): one atomic on its count per
// segment.  Returns how many the wave took.
__device__ __forceinline__ int take_places(const bool on[4], int* count, int place[4]) {
  const int lane = threadIdx.x & 63;
  int total = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t mask = __ballot(on[j]);
    place[j] = total + __popcll(mask & ((1ull << lane) - 1));
    total += __popcll(mask);
  }
  if (total == 0) return 0;
  int at = 0;
  if (lane == 0) at = atomicAdd(count, total);
  at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
  for (int j = 0; j < 4; ++j) place[j] += at;
  return total;
}

// Put the scores for which pick(score) holds into sh.list; sh.n counts them all.
template <int T, int R, typename P, typename F>
__device__ __forceinline__ void collect(Source<T, R>& src, Shared& sh, float M, const Row& r, int shift, P want, F pick) {
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  if constexpr (R == ROW_REGS) {
    src.each(sh, want, [&](int64_t seg, const float* v) {
      bool on[4];
      int place[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) on[j] = v[j] > -INFINITY && pick(v[j]);
      if (take_places(on, &sh.n, place) == 0) return;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (on[j] && place[j] < LIST) sh.list[place[j]].at = make_entry(key_of(v[j]), (int32_t)(seg * SEG + src.lane * 4 + j), 0).at;
    });
  } else {
    // 16 segments together: a bit per score, then the lanes take out their bits, one each in a turn, and load those
    // scores again.  (Few of the scores are picked, and instructions that run once cost their fetch:
    // with every place worked out in line this took 4.6 us of a row's 21, so 1.7.)
    src.template each_batch<16>(sh, want, [&](const int64_t* seg, const float (*v)[4], int count, int q) {
      uint32_t bits[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) bits[j >> 3] += bits[j >> 3] + (uint32_t)(v[j][i] > -INFINITY && pick(v[j][i]));
      const int gone = 16 - count;  // (the last segment stands in for those behind it)
      bits[1] &= gone >= 8 ? 0u : ~0u << 4 * gone;
      bits[0] &= gone > 8 ? ~0u << 4 * (gone - 8) : ~0u;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        uint32_t left = h ? bits[1] : bits[0];
#pragma unroll 1
        for (uint64_t mask; (mask = __ballot(left != 0)) != 0;) {
          int at = 0;
          if (src.lane == 0) at = atomicAdd(&sh.n, (int)__popcll(mask));
          at = __builtin_amdgcn_readfirstlane(at);
          if (at > LIST) {  // the list is not used: count the rest
            const uint32_t rest = wave_sum((uint32_t)__popc(left)) - (uint32_t)__popcll(mask);
            if (src.lane == 0 && rest) atomicAdd(&sh.n, (int)rest);
            break;
          }
          if (left) {
            const int k = __clz(left);
            left &= ~(0x80000000u >> k);
            const int32_t i = src.segment(sh, q + 8 * h + (k >> 2)) * SEG + src.lane * 4 + (k & 3);
            const int place = at + __popcll(mask & ((1ull << src.lane) - 1));
            if (place < LIST) sh.list[place].at = make_entry(key_of(load_score<T>(src.a, src.b, i)), i, 0).at;
          }
        }
      }
    });
  }
  __syncthreads();
  if (sh.n <= LIST)
    for (int i = threadIdx.x; i < sh.n; i += THREADS) sh.list[i].w = mass(score_of(sh.list[i].key()), M, r.c, shift);
  __syncthreads();
}

// Split a set of scores by their bits until one score value is left: the threshold key sh.kmin, how
// many scores equal to it stay (sh.ties) and the mass above it (sh.before_m).  By count: `need` of
// the set stay; by mass: those before which above_m + mass < target.  Only keys >= floor_key take
// part.  each(g) calls g(on, key, w) for the set, all lanes of a wave together.
template <Search S, typename E>
__device__ __forceinline__ void split(Shared& sh, E each, uint32_t need, uint64_t above_m, double target,
                                      uint32_t floor_key) {
  uint32_t prefix = 0, mask = 0;
  for (int level = 0; level < 3; ++level) {
    const int sft = level == 0 ? 21 : level == 1 ? 10 : 0;
    const uint32_t width = level == 2 ? 1023u : 2047u;
    clear_hist(sh);
    each([&](bool on, uint32_t key, uint64_t w) {
      hist_add<true, true>(sh.hc, sh.hm, on && (key & mask) == prefix && key >= floor_key,
                           (int)(width - ((key >> sft) & width)), w);
    });
    __syncthreads();
    find_bin<S>(sh, need, above_m, target);
    prefix |= (width - (uint32_t)sh.bin) << sft;
    mask |= width << sft;
    if (S != BY_MASS) need -= min(need, sh.before_c);
    above_m += sh.before_m;
  }
  const uint32_t cnt = sh.hc[sh.bin];
  uint32_t ties = need;
  if (S == BY_MASS) {  // tie number j stays while above + j w < target, w = all / cnt
    const double all = (double)sh.hm[sh.bin], room = target - (double)above_m;
    ties = room > all ? cnt : all > 0 ? (uint32_t)fmax(0.0, ceil(room * ((double)cnt / all))) : 0;
    if (above_m == 0 && ties == 0) ties = 1;
  }
  __syncthreads();
  if (threadIdx.x == 0) { sh.kmin = prefix; sh.ties = min(ties, cnt); sh.before_m = above_m; }
  __syncthreads();
}

// the first n of `list` for split()
template <typename G>
__device__ __forceinline__ void each_listed(const Entry* list, int n, G g) {
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + threadIdx.x;
    Entry e{0, 0};
    if (i < n) e = list[i];
    g(i < n, e.key(), e.w);
  }
}

// Draw from the kept entries of the list (n <= RANK), in index order: their weights put in that order and summed.
__device__ __forceinline__ void draw_from_list(const Args& a, int b, Shared& sh, int n, Slot s, const Row& r, float M) {
  const int i = threadIdx.x, lane = i & 63, wave = wave_id();
  uint32_t at = 0;
  double mine = 0;
  if (i < n) {
    at = (uint32_t)sh.list[i].idx();
    mine = s.kept ? weight(score_of(sh.list[i].key()), M, r.c) : 0.0;
    if (r.cut_min && mine < r.minp) mine = 0;
  }
  if (i < RANK) sh.rank[i] = 0;
  __syncthreads();
  const Share w = share_list(n);
  uint32_t idx = 0, place = 0;
  if (w.i < n) idx = (uint32_t)sh.list[w.i].idx();
#pragma unroll 4
  for (int j = w.j0; j < w.j1; ++j) place += (uint32_t)sh.list[j].idx() < idx;
  if (w.i < n) atomicAdd(&sh.rank[w.i], place);
  __syncthreads();
  double* weights = (double*)sh.before;
  uint32_t* indices = sh.hc;
  static_assert(BINS >= RANK, "the histogram is done with");
  if (i < n) {
    weights[sh.rank[i]] = mine;
    indices[sh.rank[i]] = at;
  }
  __syncthreads();
  const double x = i < n ? weights[i] : 0.0;
  double total;
  const double cum = block_scan(x, sh.scan_d, total);
  const double target = (double)a.u[b] * total;
  // the lowest index past the target; else the highest with weight
  const int hit = first_of(x > 0 && cum > target ? i : -1), last = last_of(x > 0 ? i : -1);
  if (lane == 0) { sh.wave_hit[wave] = hit; sh.wave_any[wave] = last; }
  __syncthreads();
  int pick = -1, end = -1;
#pragma unroll
  for (int v = 0; v < WAVES; ++v) {
    if (pick < 0) pick = sh.wave_hit[v];
    end = max(end, sh.wave_any[v]);
  }
  if (i == (pick >= 0 ? pick : end)) {
    a.out[b] = (int32_t)indices[i];
    if (a.prob) a.prob[b] = (float)(x / total);
  }
}

__device__ __forceinline__ void no_answer(const Args& a, int b) {
  if (threadIdx.x == 0) {
    a.out[b] = -1;
    if (a.prob) a.prob[b] = 0.f;
  }
}

// ---- a draw over a row's segments, given what stays: keys above t and the first `ties` equal to t

struct Found {
  int64_t seg;     // -1: no segment has mass
  double before;   // mass of the segments before it
  uint32_t ties;   // ties in the segments before it
  double total, target;
};

// The segment in which u * total falls: every lane sums a run of segments, the lane whose run holds
// the target has its wave walk it.  get(seg, mass, ties): a segment's mass of keys above t and its
// count of ties (false: nothing of it stays); wt: a tie's weight.
template <typename G>
__device__ __forceinline__ Found find_segment(const Args& a, int b, Shared& sh, uint32_t ties, double wt, G get, Found* found) {
  double* tmp_v = sh.scan_d;
  const int lane = threadIdx.x & 63, wave = wave_id();
  const int64_t run = (a.nseg + THREADS - 1) / THREADS;
  const int64_t s0 = min(run * threadIdx.x, a.nseg), s1 = min(s0 + run, a.nseg);
  uint32_t tie0 = 0, tall;
  if (ties) {
    uint32_t c = 0;
#pragma unroll 4
    for (int64_t s = s0; s < s1; ++s) {
      double m;
      uint32_t x = 0;
      if (get(s, m, x)) c += x;
    }
    tie0 = block_scan(c, sh.scan_c, tall) - c;
  }
  double sum = 0;
  uint32_t tie = tie0;
#pragma unroll 8
  for (int64_t s = s0; s < s1; ++s) {
    double m = 0;
    uint32_t x = 0;
    if (!get(s, m, x)) { m = 0; x = 0; }
    if (ties) {
      m += (tie < ties ? min(ties - tie, x) : 0u) * wt;
      tie += x;
    }
    sum += m;
  }
  const double in_wave = wave_scan(sum);
  if (threadIdx.x == 0) found->seg = -1;
  __syncthreads();
  if (lane == 63) tmp_v[wave] = in_wave;
  __syncthreads();
  double total = 0;
  for (int w = 0; w < WAVES; ++w) total += tmp_v[w];
  const double target = (double)a.u[b] * total;
  int pick = -1, last = -1;
  double cum = 0, pick_before = 0, last_before = 0;
  for (int w = 0; w < WAVES; ++w) {
    const double m = tmp_v[w];
    if (m > 0) {
      last = w;
      last_before = cum;
      if (pick < 0 && cum + m > target) { pick = w; pick_before = cum; }
    }
    cum += m;
  }
  // rounding may put u * total past the last sum: then the last score of the last segment with mass
  const bool over = pick < 0;
  if (wave == (over ? last : pick)) {
    // the first of 64 values, in order after `before`, that has mass and passes the target (or the last
    // with mass): lane -1 if none has mass
    const auto choose = [&](double m, double before, bool& hit) {
      const double upto = before + wave_scan(m);
      const uint64_t has = __ballot(m > 0), hits = over ? 0 : __ballot(m > 0 && upto > target);
      hit = hits != 0;
      return hits ? __ffsll((unsigned long long)hits) - 1 : has ? 63 - __clzll(has) : -1;
    };
    bool hit;
    double before = over ? last_before : pick_before;
    const int l = choose(sum, before, hit);
    before += lane_value(in_wave, l) - lane_value(sum, l);
    tie = lane_value(tie0, l);
    const int64_t first = run * (wave * 64 + l), end = min(first + run, a.nseg);
    Found f{-1, before, 0, total, over ? INFINITY : target};
    for (int64_t s = first; s < end; s += 64) {
      double m = 0;
      uint32_t x = 0;
      if (s + lane >= end || !get(s + lane, m, x)) { m = 0; x = 0; }
      uint32_t tb = tie;
      if (ties) {
        const uint32_t scan = wave_scan(x);
        tb = tie + scan - x;
        tie += lane_value(scan, 63);
        m += (tb < ties ? min(ties - tb, x) : 0u) * wt;
      }
      const int at = choose(m, before, hit);
      const double upto = wave_scan(m);
      if (at >= 0) {
        f.seg = s + at;
        f.before = before + (lane_value(upto, at) - lane_value(m, at));
        f.ties = lane_value(tb, at);
        if (hit) break;
      }
      before += lane_value(upto, 63);
    }
    if (lane == 0) *found = f;
  }
  __syncthreads();
  return *found;
}

// One wave: the first kept score of the segment at which the mass passes the target (or its last).
__device__ __forceinline__ void pick_in_segment(const Args& a, int b, const Found& f, const float v[4], const Row& r, float M,
                                                uint32_t t, uint32_t ties) {
  const int lane = threadIdx.x & 63;
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) c += v[j] > -INFINITY && key_of(v[j]) == t;
  uint32_t tie = f.ties + wave_scan(c) - c;
  double w[4], m = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t key = key_of(v[j]);
    const bool kept = v[j] > -INFINITY && (key > t || (key == t && tie < ties));
    tie += v[j] > -INFINITY && key == t;
    w[j] = kept ? weight(v[j], M, r.c) : 0.0;
    if (r.cut_min && w[j] < r.minp) w[j] = 0;
    m += w[j];
  }
  double cum = f.before + (wave_scan(m) - m);
  int hit = -1, end = -1;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    cum += w[j];
    if (w[j] > 0) {
      if (hit < 0 && cum > f.target) hit = j;
      end = j;
    }
  }
  const uint64_t hits = __ballot(hit >= 0), ends = __ballot(end >= 0);
  const int win = hits ? __ffsll((unsigned long long)hits) - 1 : 63 - __clzll(ends);
  if (lane == win) {
    const int j = hits ? hit : end;
    a.out[b] = (int32_t)(f.seg * SEG + lane * 4 + j);
    if (a.prob) a.prob[b] = (float)((j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3]) / f.total);
  }
}

template <int T, int R>
__device__ __forceinline__ void draw_from_row(const Args& a, int b, Source<T, R>& src, Shared& sh, const Row& r, float M,
                                              uint32_t t, uint32_t ties, double* segmass, int32_t* segtie, bool have_mass) {
  __shared__ Found found;
  const float bound = score_of(max(t, KEY_NONE));
  double wt = 0;
  if (ties) {
    wt = weight(bound, M, r.c);
    if (r.cut_min && wt < r.minp) { wt = 0; ties = 0; }
  }
  if (!have_mass)
    src.each(sh, [&](float m) { return m >= bound; }, [&](int64_t seg, const float* v) {
      double m = 0;
      uint32_t c = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t key = key_of(v[j]);
        if (v[j] > -INFINITY && key > t) {
          const double w = weight(v[j], M, r.c);
          m += !r.cut_min || w >= r.minp ? w : 0.0;
        }
        c += v[j] > -INFINITY && key == t;
      }
      m = wave_sum(m);
      c = wave_sum(c);
      if (src.lane == 0) { segmass[seg] = m; segtie[seg] = (int32_t)c; }
    });
  __syncthreads();
  const Found f = find_segment(
      a, b, sh, ties, wt,
      [&](int64_t s, double& m, uint32_t& c) {
        const float x = src.segmax(s);
        if (!(x >= bound) || x == -INFINITY) return false;
        m = segmass[s];
        if (have_mass) m *= weight(x, M, r.c);
        else c = (uint32_t)segtie[s];
        return true;
      },
      &found);
  if (f.seg < 0) {
    no_answer(a, b);
    return;
  }
  if (src.wave == (R == ROW_REGS ? (int)f.seg : 0)) {
    float v[4];
    if constexpr (R == ROW_REGS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = src.v[j];
    } else {
      load_seg<T>(a, b, f.seg, src.lane, v);
    }
    pick_in_segment(a, b, f, v, r, M, t, ties);
  }
}

// the unit of a row's masses from its segments' largest scores, each taken for the whole segment
template <int T, int R>
__device__ __forceinline__ int shift_from_maxima(const Args& a, const Source<T, R>& src, const Row& r, float M) {
  double sum = 0;
  for (int64_t s = src.lane; s < a.nseg; s += 64) sum += weight(src.segmax(s), M, r.c);
  return shift_for(SEG * wave_sum(sum));
}

// A row from its scores alone (rows of one launch; long rows with a long top-k, or whose lists ran
// over): histogram, threshold of top-k, threshold of top-p, draw.
template <int T, int R>
__device__ __forceinline__ void finish_general(const Args& a, int b, Source<T, R>& src, Shared& sh, const Row& r, float M,
                                               int shift, double* segmass, int32_t* segtie) {
  const float cb = (float)(r.c * 32);  // 32 bins to an octave of weight
  const uint32_t place = src.lane * 4;
  const auto any = [](float) { return true; };
  clear_hist(sh);
  src.each(sh, any, [&](int64_t, const float* v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t w = r.cut_p ? mass(v[j], M, r.c, shift, place + j) : 0;
      hist_add<true, true>(sh.hc, sh.hm, v[j] > -INFINITY, bin_of(v[j], M, cb), w);
    }
  });
  __syncthreads();
  const auto reaches = [&](int bin) { return [=](float m) { return bin_of(m, M, cb) <= bin; }; };
  const auto of_bin = [&](int bin) {
    return [=, &src, &sh, &r](auto g) {
      src.each(sh, [=](float m) { return bin_of(m, M, cb) <= bin; }, [&](int64_t, const float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          g(v[j] > -INFINITY && bin_of(v[j], M, cb) == bin, key_of(v[j]),
            mass(v[j], M, r.c, shift, place + j));
      });
    };
  };
  uint32_t t = KEY_NONE, ties = 0;
  uint64_t total = 0;
  int kbin = BINS;        // bin of the top-k threshold
  uint32_t c[PER];        // this thread's bins, kept for the search by mass
  uint64_t m[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    c[j] = sh.hc[PER * threadIdx.x + j];
    m[j] = sh.hm[PER * threadIdx.x + j];
  }
  if (r.k > 0) {
    find_bin<BY_COUNT_WITH_MASS>(sh, (uint32_t)r.k);
    kbin = sh.bin;
    const uint64_t kbefore = sh.before_m;
    const uint32_t cbefore = sh.before_c;
    if (cbefore + sh.hc[kbin] <= (uint32_t)r.k) {  // the whole bin stays: above the key below its smallest
      total = kbefore + sh.hm[kbin];
      if (threadIdx.x == 0) sh.kmin = 0xffffffffu;
      uint32_t least = 0xffffffffu;
      src.each(sh, reaches(kbin), [&](int64_t, const float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          least = min(least, v[j] > -INFINITY && bin_of(v[j], M, cb) == kbin ? key_of(v[j]) : 0xffffffffu);
      });
      __syncthreads();
      least = wave_min(least);
      if (src.lane == 0) atomicMin(&sh.kmin, least);
      __syncthreads();
      t = sh.kmin - 1;
    } else {
      collect<T, R>(src, sh, M, r, shift, reaches(kbin), [&](float x) { return bin_of(x, M, cb) == kbin; });
      const int n = sh.n;
      if (n <= RANK) {
        const Slot s = rank_list(sh, n, r.k, cbefore);
        total = kbefore + sh.kept_m;
        list_threshold(sh, s);
      } else {
        const uint32_t need = (uint32_t)(r.k - cbefore);
        if (n <= LIST) split<BY_COUNT_WITH_MASS>(sh, [&](auto g) { each_listed(sh.list, n, g); }, need, kbefore, 0.0, 0);
        else split<BY_COUNT_WITH_MASS>(sh, of_bin(kbin), need, kbefore, 0.0, 0);
        total = sh.before_m + (uint64_t)(sh.ties * __builtin_ldexp(weight(score_of(sh.kmin), M, r.c), shift));
      }
      t = sh.kmin;
      ties = sh.ties;
    }
    if (r.cut_p) {  // the histogram of the scores that top-k left: bins past its threshold's are empty
      __syncthreads();
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = PER * threadIdx.x + j;
        sh.hc[i] = i <= kbin ? c[j] : 0;
        sh.hm[i] = i < kbin ? m[j] : i == kbin ? total - kbefore : 0;
      }
      __syncthreads();
    }
  }
  if (r.cut_p) {
    find_bin<BY_MASS>(sh, 0, 0, 0, fmax(r.p, 0.0));
    const double target = sh.target;
    const int bin = sh.bin;
    const uint64_t above = sh.before_m;
    const uint32_t floor_key = bin == kbin ? (ties ? t : t + 1) : 0;  // what top-k left of this bin
    const uint32_t tie_cap = bin == kbin && ties ? ties : 0xffffffffu;
    collect<T, R>(src, sh, M, r, shift, reaches(bin),
                  [&](float x) { return bin_of(x, M, cb) == bin && key_of(x) >= floor_key; });
    const int n = sh.n;
    // (scores equal to top-k's threshold beyond its ties rank behind all that stay, and the mass
    // before them has reached the total: the cut drops them)
    if (n <= RANK) {
      Slot s = rank_list(sh, n, 0, 0);
      cut_by_mass(s, above, target);
      list_threshold(sh, s);
    } else if (n <= LIST) {
      split<BY_MASS>(sh, [&](auto g) { each_listed(sh.list, n, g); }, 0, above, target, floor_key);
    } else {
      split<BY_MASS>(sh, of_bin(bin), 0, above, target, floor_key);
    }
    t = sh.kmin;
    ties = t == floor_key ? min(sh.ties, tie_cap) : sh.ties;
  }
  __syncthreads();
  draw_from_row<T, R>(a, b, src, sh, r, M, t, ties, segmass, segtie, false);
}

// One workgroup per row.  Rows of one launch and long rows that need no pass over all masses are
// answered; `passes`: long rows that cut by mass alone get their RowState.
template <int T, int R>
__global__ void __launch_bounds__(THREADS) finish_kernel(Args a, int passes) {
  __shared__ Shared sh;
  constexpr int SMALL = R == ROW_REGS ? WAVES : R == ROW_CACHED ? CACHED_SEGS : 1;
  __shared__ float small_max[R == ROW_LONG ? KEPT : SMALL];
  __shared__ double small_mass[SMALL];
  __shared__ int32_t small_tie[SMALL];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = wave_id();
  const Row r = row_settings(a, b);
  constexpr bool own = R != ROW_LONG;
  double* segmass = own ? small_mass : a.segmass + (int64_t)b * a.nseg;
  int32_t* segtie = own ? small_tie : a.segtie + (int64_t)b * a.nseg;
  Source<T, R> src(a, b, small_max, own ? nullptr : a.segmax + (int64_t)b * a.nseg);
  float m = -INFINITY;
  if constexpr (R == ROW_REGS) {
    if (wave < a.nseg) {
      load_seg<T>(a, b, wave, lane, src.v);
      m = wave_max(max4(src.v));
      if (lane == 0) small_max[wave] = m;
    }
  } else if constexpr (R == ROW_CACHED) {
    for (int64_t seg0 = wave; seg0 < a.nseg; seg0 += 4 * WAVES) {
      Raw<T> raw[4];
      load_segs<T, 4>(a, b, lane, seg0, WAVES, raw);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (seg0 + j * WAVES < a.nseg) {
          float x[4];
          unpack<T>(raw[j], x);
          const float y = wave_max(max4(x));
          if (lane == 0) small_max[seg0 + j * WAVES] = y;
          m = fmaxf(m, y);
        }
    }
  } else {
    const bool keep = src.kept();
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < a.nseg; i += THREADS) {
      const float x = src.in_memory[i];
      if (keep) small_max[i] = x;
      m = fmaxf(m, x);
    }
  }
  const float M = block_max(m, sh.tmp);
  if (M == -INFINITY) {  // nothing is left of the row
    no_answer(a, b);
    if (threadIdx.x == 0 && passes) a.state[b].mode = IDLE;
    return;
  }
  if (R == ROW_LONG && passes) {
    RowState st{IDLE, M, 0.f, 0, KEY_NONE, 0, -1.0, 0.0, 0, 0, 0, 0};
    if (r.by_mass()) {
      double sum = 0, total;
      for (int64_t i = threadIdx.x; i < a.nseg; i += THREADS)
        if (src.segmax(i) > -INFINITY) sum += segmass[i] * weight(src.segmax(i), M, r.c);
      block_scan(sum, sh.scan_d, total);
      st.shift = shift_for(2 * total);
      // N scores below (1 - p) total / N hold less than (1 - p) total: the threshold is not among
      // them, and the bins but the last span the octaves above that
      const double least = fmax((1 - r.p) * total / (double)a.N, 0x1p-60);
      const double octaves = fmax(-log2(least), 0.0) + 0.125;
      st.mode = BY_TOP_P;
      st.cb = (float)(r.c * (BINS - 1) / octaves);
    } else if (r.k > 0 && !r.short_k()) {
      // the bins span eight times the range of the segments' maxima, which for scores of any common
      // distribution is beyond their bulk; a threshold in the last bin, of all below, still stands
      float low = INFINITY;
      for (int64_t i = threadIdx.x; i < a.nseg; i += THREADS)
        if (src.segmax(i) > -INFINITY) low = fminf(low, src.segmax(i));
      low = -block_max(-low, sh.tmp);
      const float range = 8 * (M - low);
      st.mode = BY_TOP_K;
      st.cb = range > 0 && range < INFINITY ? (float)(BINS - 1) / range : 32.f;
      st.target = (double)r.k;
    } else if (r.direct() && r.cut_min) {
      st.mode = NO_CUT;
      st.bin = BINS;
    }
    if (threadIdx.x == 0) a.state[b] = st;
    for (int i = threadIdx.x; i < BINS; i += THREADS) a.hmass[(int64_t)b * BINS + i] = 0;
    if (st.mode != IDLE) return;
  }
  if (r.direct()) {
    draw_from_row<T, R>(a, b, src, sh, r, M, KEY_NONE, 0, segmass, segtie, R == ROW_LONG && !r.cut_min);
    return;
  }
  if (r.short_k()) {
    // A short list: the k best lie in bins up to the one in which the count of scores reaches k.  On a
    // long row the segments' maxima are counted where they are at least 2 k: that many scores, one
    // a segment, are in those bins already, and few others.  (32 rows of 32768: k = 50 17 us so, k = 100, by
    // all scores, 27.)
    const float cb = (float)(r.c * 32);
    const auto any = [](float) { return true; };
    clear_hist(sh);
    if (R == ROW_LONG && r.k <= a.nseg / 2) {
      for (int i = threadIdx.x; i < a.nseg; i += THREADS) {
        const float x = src.segmax(i);
        if (x > -INFINITY) atomicAdd(&sh.hc[bin_of(x, M, cb)], 1u);
      }
    } else {
      src.each(sh, any, [&](int64_t, const float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          hist_add<true, false>(sh.hc, sh.hm, v[j] > -INFINITY, bin_of(v[j], M, cb), 0);
      });
    }
    __syncthreads();
    find_bin<BY_COUNT>(sh, (uint32_t)r.k);
    // Candidates are the scores above one a little below the last of those bins, so that each takes one
    // comparison (fp32 rounds M - s and its product by 2^-23 or so: a few candidates more do no harm).
    // Fewer unmasked than k: everything unmasked.
    const bool all = sh.before_c + sh.hc[sh.bin] < (uint32_t)r.k || sh.bin == BINS - 1 || !(M < INFINITY);
    const double low = (double)M - (double)(sh.bin + 1) / (double)cb * (1 + 1e-6) - fabs((double)M) * 1e-6;
    const float cut = all ? -INFINITY : (float)low;
    collect<T, R>(src, sh, M, r, LIST_SHIFT, [=](float x) { return x >= cut; }, [=](float x) { return x >= cut; });
    const int n = sh.n;
    if (n <= RANK) {
      Slot s = rank_list(sh, n, r.k, 0);
      if (r.cut_p) cut_by_mass(s, 0, r.p * (double)sh.kept_m);
      draw_from_list(a, b, sh, n, s, r, M);
      return;
    }
    if (n <= LIST) {
      const auto listed = [&](auto g) { each_listed(sh.list, n, g); };
      split<BY_COUNT_WITH_MASS>(sh, listed, (uint32_t)r.k, 0, 0.0, 0);
      uint32_t t = sh.kmin, ties = sh.ties;
      if (r.cut_p) {
        const uint64_t total = sh.before_m + (uint64_t)ties * mass(score_of(t), M, r.c, LIST_SHIFT);
        split<BY_MASS>(sh, listed, 0, 0, r.p * (double)total, t);
        ties = sh.kmin == t ? min(ties, sh.ties) : sh.ties;
        t = sh.kmin;
      }
      draw_from_row<T, R>(a, b, src, sh, r, M, t, ties, segmass, segtie, false);
      return;
    }
  }
  finish_general<T, R>(a, b, src, sh, r, M, shift_from_maxima<T, R>(a, src, r, M), segmass, segtie);
}

// ---- a round of passes over long rows: counts or masses by bin, then what lies above the threshold's
// bin and in it, then the threshold

template <int T>
__global__ void __launch_bounds__(THREADS) hist_kernel(Args a) {
  __shared__ unsigned long long hm[BINS];
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = wave_id();
  const RowState st = a.state[b];
  if (st.mode == IDLE || st.mode == NO_CUT) return;
  const Row r = row_settings(a, b);
  const bool counts = st.mode == BY_TOP_K;
  const float floor_score = score_of(st.floor_key);
  for (int i = threadIdx.x; i < BINS; i += THREADS) hm[i] = 0;
  __syncthreads();
  const uint32_t place = lane * 4;
  uint64_t rest = 0;  // the last bin's: scores that can hardly hold the threshold
  const int64_t s1 = min((int64_t)(blockIdx.x + 1) * PASS_SEGS, a.nseg);
  for (int64_t seg0 = (int64_t)blockIdx.x * PASS_SEGS + wave; seg0 < s1; seg0 += 4 * WAVES) {
    Raw<T> raw[4];
    load_segs<T, 4>(a, b, lane, seg0, WAVES, raw);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (seg0 + j * WAVES >= s1) continue;
      float x[4];
      unpack<T>(raw[j], x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = x[i];
        const int bin = bin_of(v, st.M, st.cb);
        const bool in = v > floor_score;
        uint64_t w = in;
        if (!counts) w = in ? mass(v, st.M, r.c, st.shift, place + i) : (uint64_t)0;
        if (in && bin < BINS - 1) atomicAdd(&hm[bin], (unsigned long long)w);
        else rest += w;
      }
    }
  }
  rest = wave_sum(rest);
  if (lane == 0 && rest) atomicAdd(&hm[BINS - 1], (unsigned long long)rest);
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS)
    if (hm[i]) atomicAdd((unsigned long long*)a.hmass + (int64_t)b * BINS + i, hm[i]);
}

constexpr int PASS_LIST = 512;  // scores of the threshold's bin that a workgroup lists

template <int T>
__global__ void __launch_bounds__(THREADS) collect_kernel(Args a) {
  __shared__ Hist<false> sh;
  __shared__ Entry listed[PASS_LIST];
  __shared__ float above[WAVES][SEG];
  __shared__ int count;
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = wave_id();
  const RowState st = a.state[b];  // (of which this kernel writes bin, above and listed, and reads none of them)
  const double st_target = st.target;
  if (st.mode == IDLE) return;
  const Row r = row_settings(a, b);
  const float floor_score = score_of(st.floor_key);
  const int64_t s1 = min((int64_t)(blockIdx.x + 1) * PASS_SEGS, a.nseg);
  const int64_t first = (int64_t)blockIdx.x * PASS_SEGS + wave;
  Raw<T> raw[4];
  load_segs<T, 4>(a, b, lane, first, WAVES, raw);  // on their way during the search
  static_assert(PASS_SEGS % (4 * WAVES) == 0 && PASS_SEGS / WAVES <= 64, "a lane per segment of a wave");
  float largest = -INFINITY;  // lane l: of the wave's l-th segment
  if (lane < PASS_SEGS / WAVES && first + lane * WAVES < s1) largest = a.segmax[(int64_t)b * a.nseg + first + lane * WAVES];
  // min-p drops scores from the draw, not from the total of which top-p keeps a part
  const bool drop = r.cut_min && !(st.mode == BY_TOP_K && r.cut_p);
  int bin = BINS;
  if (st.mode != NO_CUT) {
    for (int i = threadIdx.x; i < BINS; i += THREADS) sh.hm[i] = a.hmass[(int64_t)b * BINS + i];
    __syncthreads();
    find_bin<BY_MASS>(sh, 0, 0, st_target, st_target < 0 ? fmax(r.p, 0.0) : -1.0);
    bin = sh.bin;
    // all that lies above top-k's ties is less than top-p's part: the threshold is those ties
    if (st.mode == BY_TOP_P && st.ties && (bin < 0 || (double)(sh.before_m + sh.hm[bin]) < sh.target)) bin = BINS;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      if (st.mode == BY_TOP_P && st_target < 0) a.state[b].part = sh.target;
      a.state[b].bin = bin;
      a.state[b].above = sh.before_m;
      a.state[b].all = bin == BINS ? sh.before_m + (sh.bin >= 0 ? sh.hm[sh.bin] : 0) : 0;
    }
  }
  // The least score that may count: the next above the floor, and none that is surely below min-p (the weights
  // themselves decide next to it).  That bound is at most M, whatever underflows in it, and rounding to fp32 moves it
  // past no score at or above it: compared with >=, it drops neither the best score nor any other that stays.  (A NaN,
  // where M is infinite, drops nothing; above a floor of +inf there is nothing, and a NaN to compare with.)
  uint32_t up_key = st.floor_key + 1;
  if (drop) {
    const double lim = (double)st.M + ((double)__builtin_amdgcn_logf((float)r.minp) * (1 + 1e-5) - 1e-5) / r.c;
    up_key = max(up_key, key_of(fmaxf((float)(lim - fabs(lim) * 1e-6), -INFINITY)));
  }
  const float up_floor = score_of(up_key);
  // segments without a score that counts (of peaked scores nearly all: 256 x 128000, min-p 0.05 87 us without this)
  bool counts = largest > -INFINITY;
  if (bin < BINS) counts = counts && largest > floor_score && bin_of(largest, st.M, st.cb) <= bin;
  else counts = counts && (largest >= up_floor || (st.ties && largest >= floor_score));
  const uint32_t wanted = (uint32_t)__ballot(counts);
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  const auto put = [&](uint32_t at, Entry e) {
    if (st.mode == BY_TOP_P) e.w = mass(score_of(e.key()), st.M, r.c, st.shift);  // (counts need none)
    if (at < (uint32_t)a.listcap) a.list[(int64_t)b * a.listcap + at] = e;
  };
  for (int g = 0; g < PASS_SEGS / WAVES; g += 4) {
    if (first + g * WAVES >= s1) break;
    if (g && (wanted >> g & 15)) load_segs<T, 4>(a, b, lane, first + g * WAVES, WAVES, raw);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t seg = first + (g + j) * WAVES;
      if (seg >= s1) continue;
      if (!(wanted >> (g + j) & 1)) {
        if (lane == 0) a.segmass[(int64_t)b * a.nseg + seg] = 0;
        if (lane == 0 && bin == BINS && st.ties) a.segtie[(int64_t)b * a.nseg + seg] = 0;
        continue;
      }
      float x[4];
      unpack<T>(raw[j], x);
      // scores above the threshold's bin are moved together, so that a wave computes 64 weights at once
      bool up[4], in[4];
      int place[4], n = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at_bin = bin_of(x[i], st.M, st.cb);
        in[i] = at_bin == bin && x[i] > floor_score;
        up[i] = at_bin < bin && x[i] >= up_floor;
        const uint64_t mask = __ballot(up[i]);
        if (up[i]) above[wave][n + __popcll(mask & ((1ull << lane) - 1))] = x[i];
        n += __popcll(mask);
      }
      double sum = 0;
      for (int i = lane; i < n; i += 64) {
        const double w = weight(above[wave][i], st.M, r.c);
        if (!drop || w >= r.minp) sum += w;
      }
      sum = wave_sum(sum);
      if (lane == 0) a.segmass[(int64_t)b * a.nseg + seg] = sum;
      if (bin == BINS && st.ties) {  // the scores equal to the floor: not listed, counted here
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) c += x[i] == floor_score;
        c = wave_sum(c);
        if (lane == 0) a.segtie[(int64_t)b * a.nseg + seg] = (int32_t)c;
      }
      if (__ballot(in[0] | in[1] | in[2] | in[3]) && take_places(in, &count, place))
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (in[i]) {
            const Entry e = make_entry(key_of(x[i]), (int32_t)(seg * SEG + lane * 4 + i), 0);
            if (place[i] < PASS_LIST) listed[place[i]] = e;
            else put(atomicAdd(&a.state[b].listed, 1u), e);  // more than this workgroup lists
          }
    }
  }
  __syncthreads();
  const int n = min(count, PASS_LIST);
  __syncthreads();
  if (threadIdx.x == 0 && n) count = (int)atomicAdd(&a.state[b].listed, (uint32_t)n);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += THREADS) put((uint32_t)(count + i), listed[i]);
}

// The unit 2^-shift for sums of listed scores' weights, by the bound that their bin sets: (M - s) cb is at least its number,
// but for the rounding of the two.  A listcap of masses of up to 2^46 stays below 2^62.
__device__ __forceinline__ int listed_shift(const RowState& st, const Row& r) {
  const double gap = st.bin ? fmin((double)st.bin / (double)st.cb, 3.4e38) : 0.0;  // (M - s may have passed fp32's range)
  return 46 + (int)fmin(fmax(gap * (1 - 1e-6) * r.c, 0.0), 900.0);
}

// The threshold inside the listed bin; then the draw, or, after top-k where top-p is to follow, the state of a
// second round.
template <int T>
__global__ void __launch_bounds__(THREADS) finish_passes_kernel(Args a) {
  __shared__ Shared sh;
  __shared__ Found found;
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const RowState st = a.state[b];
  if (st.mode == IDLE) return;
  const Row r = row_settings(a, b);
  double* segmass = a.segmass + (int64_t)b * a.nseg;
  __syncthreads();
  if (threadIdx.x == 0) a.state[b].mode = IDLE;
  if (st.bin < BINS && st.listed > (uint32_t)a.listcap) {  // more than a list of equal or near-equal scores: the row again
    __shared__ float maxima[KEPT];
    Source<T, ROW_LONG> src(a, b, maxima, a.segmax + (int64_t)b * a.nseg);
    if (src.kept())
      for (int i = threadIdx.x; i < a.nseg; i += THREADS) maxima[i] = src.in_memory[i];
    __syncthreads();
    const int shift = r.by_mass() ? st.shift : shift_from_maxima<T, ROW_LONG>(a, src, r, st.M);
    finish_general<T, ROW_LONG>(a, b, src, sh, r, st.M, shift, segmass, a.segtie + (int64_t)b * a.nseg);
    return;
  }
  const int n = st.bin < BINS ? (int)st.listed : 0;
  const Entry* list = a.list + (int64_t)b * a.listcap;
  const int lshift = listed_shift(st, r);
  const double target = st.target < 0 ? st.part : st.target;
  uint32_t t, ties;
  if (st.bin == BINS) {  // everything above the floor, and of its ties those that top-p's part still takes
    t = st.floor_key;
    ties = 0;
    if (st.mode == BY_TOP_P) {
      const double w = __builtin_ldexp(weight(score_of(t), st.M, r.c), st.shift);
      const double room = target - (double)st.all;
      ties = w == 0 || room > w * (double)st.ties ? st.ties : (uint32_t)fmax(0.0, ceil(room / w));
      if (st.all == 0 && ties == 0) ties = 1;
      ties = min(ties, st.ties);
    }
  } else {
    const bool counts = st.mode == BY_TOP_K;
    const uint32_t need = counts ? (uint32_t)(r.k - (int64_t)st.above) : 0;
    if (n <= RANK) {
      if ((int)threadIdx.x < n) sh.list[threadIdx.x] = list[threadIdx.x];
      __syncthreads();
      Slot s = rank_list(sh, n, need, 0);
      if (!counts) cut_by_mass(s, st.above, target);
      list_threshold(sh, s);
    } else if (counts) {
      split<BY_COUNT_WITH_MASS>(sh, [&](auto g) { each_listed(list, n, g); }, need, 0, 0.0, 0);
    } else {
      split<BY_MASS>(sh, [&](auto g) { each_listed(list, n, g); }, 0, st.above, target, 0);
    }
    t = sh.kmin;
    ties = sh.ties;
    if (counts && r.cut_p) {
      // what top-k leaves: the bins above, the listed scores above t, the ties
      double mine = 0, total;
      for (int64_t s = threadIdx.x; s < a.nseg; s += THREADS) mine += segmass[s];
      uint64_t in_bin = 0, all_in_bin;
      for (int i = threadIdx.x; i < n; i += THREADS) {
        const Entry e = list[i];
        if (e.key() > t) in_bin += mass(score_of(e.key()), st.M, r.c, lshift);
      }
      block_scan(mine, sh.scan_d, total);
      block_scan(in_bin, sh.scan_m, all_in_bin);
      total += __builtin_ldexp((double)all_in_bin, -lshift) + ties * weight(score_of(t), st.M, r.c);
      for (int i = threadIdx.x; i < BINS; i += THREADS) a.hmass[(int64_t)b * BINS + i] = 0;
      if (threadIdx.x == 0) {
        RowState next = st;
        const float range = st.M - score_of(t);
        next.mode = BY_TOP_P;
        next.cb = range > 0 && range < INFINITY ? (float)(BINS - 2) / range : 32.f;
        next.floor_key = t;
        next.ties = ties;
        next.shift = shift_for(2 * total);
        next.target = __builtin_ldexp(fmax(r.p, 0.0) * total, next.shift);
        next.above = 0;
        next.bin = 0;
        next.listed = 0;
        a.state[b] = next;
      }
      return;
    }
  }
  double wt = weight(score_of(t), st.M, r.c);
  if (r.cut_min && wt < r.minp) { wt = 0; ties = 0; }
  // Listed scores above t add to their segments' masses (as whole numbers: their order does not matter), ties are
  // counted per segment: in LDS where they fit, else in the workspace.
  const auto add = [&](auto plus_mass, auto plus_tie) {
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const Entry e = list[i];
      if (e.key() > t) {
        // (a weight below the unit counts as one: a kept score can be the first or the last of its row)
        const float x = score_of(e.key());
        const double w = weight(x, st.M, r.c);
        if (w > 0 && (!r.cut_min || w >= r.minp)) plus_mass(e.idx() / SEG, max(mass(x, st.M, r.c, lshift), (uint64_t)1));
      } else if (e.key() == t && ties) {
        plus_tie(e.idx() / SEG);
      }
    }
  };
  Found f;
  if (a.nseg <= KEPT) {
    __shared__ unsigned long long more[KEPT];
    uint32_t* tied = (uint32_t*)sh.hm;
    static_assert(KEPT * 4 <= BINS * 8, "a tie count per segment");
    __syncthreads();
    for (int s = threadIdx.x; s < a.nseg; s += THREADS) {
      more[s] = 0;
      tied[s] = st.bin == BINS && ties ? (uint32_t)a.segtie[(int64_t)b * a.nseg + s] : 0u;
    }
    __syncthreads();
    add([&](int s, uint64_t w) { atomicAdd(more + s, (unsigned long long)w); }, [&](int s) { atomicAdd(tied + s, 1u); });
    __syncthreads();
    f = find_segment(a, b, sh, ties, wt, [&](int64_t s, double& m, uint32_t& c) {
      m = segmass[s] + __builtin_ldexp((double)more[s], -lshift);
      c = tied[s];
      return true;
    }, &found);
  } else {
    // agent-scope accesses meet in the L2 that this one workgroup works through; the waits put the
    // zeros before the sums and the sums before the reads
    int32_t* segtie = a.segtie + (int64_t)b * a.nseg;
    uint64_t* more = a.listed + (int64_t)b * a.nseg;
    if (st.bin < BINS)
      for (int64_t s = threadIdx.x; s < a.nseg; s += THREADS) {
        __hip_atomic_store(segtie + s, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(more + s, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    add([&](int s, uint64_t w) { atomicAdd((unsigned long long*)more + s, (unsigned long long)w); },
        [&](int s) { atomicAdd(segtie + s, 1); });
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    f = find_segment(a, b, sh, ties, wt, [&](int64_t s, double& m, uint32_t& c) {
      m = segmass[s];
      if (st.bin < BINS) m += __builtin_ldexp((double)__hip_atomic_load(more + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), -lshift);
      c = (uint32_t)__hip_atomic_load(segtie + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      return true;
    }, &found);
  }
  if (f.seg < 0) {
    no_answer(a, b);
    return;
  }
  if (threadIdx.x < 64) {
    float v[4];
    load_seg<T>(a, b, f.seg, lane, v);
    pick_in_segment(a, b, f, v, r, st.M, t, ties);
  }
}

template <int T>
int run(Args& a, int rounds, hipStream_t st) {
  if (a.nseg <= WAVES) {
    hipLaunchKernelGGL((finish_kernel<T, ROW_REGS>), dim3(a.B), dim3(THREADS), 0, st, a, 0);
  } else if (a.nseg <= CACHED_SEGS) {
    hipLaunchKernelGGL((finish_kernel<T, ROW_CACHED>), dim3(a.B), dim3(THREADS), 0, st, a, 0);
  } else {
    const int per = 4 * STAT_SEGS;
    hipLaunchKernelGGL((stats_kernel<T>), dim3((unsigned)((a.nseg + per - 1) / per), a.B), dim3(256), 0, st, a);
    FPS_CHECK_LAUNCH();
    hipLaunchKernelGGL((finish_kernel<T, ROW_LONG>), dim3(a.B), dim3(THREADS), 0, st, a, rounds);
    for (int i = 0; i < rounds; ++i) {
      FPS_CHECK_LAUNCH();
      const dim3 grid((unsigned)((a.nseg + PASS_SEGS - 1) / PASS_SEGS), a.B);
      hipLaunchKernelGGL((hist_kernel<T>), grid, dim3(THREADS), 0, st, a);
      FPS_CHECK_LAUNCH();
      hipLaunchKernelGGL((collect_kernel<T>), grid, dim3(THREADS), 0, st, a);
      FPS_CHECK_LAUNCH();
      hipLaunchKernelGGL((finish_passes_kernel<T>), dim3(a.B), dim3(THREADS), 0, st, a);
    }
  }
  FPS_CHECK_LAUNCH();
  return 0;
}

constexpr int64_t kShortRow = (int64_t)CACHED_SEGS * SEG;  // rows up to this take no workspace
constexpr int LAUNCH_ROWS = 1 << 22;  // of those, so many at most a launch (its threads must fit 32 bits)

int list_cap(int64_t N) { return (int)(N / 8 < 16384 ? N / 8 : 16384); }

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

// How many rounds of passes can a row need?  (Scalars decide here, per-row settings on the device.)
int rounds_of(int64_t N, const float* temperature, double temperature0, const int32_t* top_k, int64_t top_k0,
              const float* top_p, double top_p0, const float* min_p, double min_p0) {
  const bool greedy = !temperature && !(temperature0 > 0);
  const bool can_long_k = !greedy && (top_k || (top_k0 > SHORT_K && top_k0 < N));
  const bool can_no_k = !greedy && (top_k || top_k0 <= 0 || top_k0 >= N);
  const bool can_p = top_p || top_p0 < 1, can_min = min_p || min_p0 > 0;
  return can_long_k && can_p ? 2 : can_long_k || (can_no_k && (can_p || can_min)) ? 1 : 0;
}

}  // namespace

// bytes of workspace for B rows of N scores with these settings (as below); what only the passes use is left
// out where no row can take them
FPS_API int64_t fps_sample_scores_ws_bytes(int64_t B, int64_t N, const float* temperature, double temperature0,
                                           const int32_t* top_k, int64_t top_k0, const float* top_p, double top_p0,
                                           const float* min_p, double min_p0) {
  if (B <= 0 || N <= kShortRow) return 0;
  const int64_t nseg = (N + SEG - 1) / SEG;
  int64_t bytes = B * nseg * 16 + 16;
  if (rounds_of(N, temperature, temperature0, top_k, top_k0, top_p, top_p0, min_p, min_p0))
    bytes += B * (list_cap(N) * (int64_t)sizeof(Entry)) + round16(B * sizeof(RowState)) + B * BINS * 8 +
             (nseg > KEPT ? B * nseg * 8 : 0);
  return bytes;
}

// s [B, N] (row stride ld, type 0 fp32 / 1 bf16 / 2 fp16); u [B]; temperature / top_k / top_p /
// min_p: per row, or nullptr and the scalar after it.  out [B] indices (-1: nothing left of
// the row), prob [B] or nullptr.
FPS_API int fps_sample_scores(const void* s, int type, int B, int64_t N, int64_t ld, const float* u,
                              const float* temperature, double temperature0, const int32_t* top_k, int64_t top_k0,
                              const float* top_p, double top_p0, const float* min_p, double min_p0, int32_t* out,
                              float* prob, void* ws, void* stream) {
  if (B <= 0) return 0;
  if (N <= 0 || N > INT32_MAX || ld < N || type < 0 || type > 2 || (B > 65535 && N > kShortRow))
    return (int)hipErrorInvalidValue;
  Args a;
  a.s = s; a.ld = ld; a.N = N; a.nseg = (N + SEG - 1) / SEG; a.B = B;
  a.u = u;
  a.temperature = temperature; a.temperature0 = temperature0;
  a.top_k = top_k; a.top_k0 = top_k0;
  a.top_p = top_p; a.top_p0 = top_p0;
  a.min_p = min_p; a.min_p0 = min_p0;
  a.out = out; a.prob = prob;
  a.segmass = nullptr; a.hmass = nullptr; a.list = nullptr; a.state = nullptr; a.segmax = nullptr; a.segtie = nullptr; a.listed = nullptr;
  a.listcap = 0;
  int rounds = 0;
  if (N > kShortRow) {
    if (ws == nullptr || ((uintptr_t)ws & 15)) return (int)hipErrorInvalidValue;
    rounds = rounds_of(N, temperature, temperature0, top_k, top_k0, top_p, top_p0, min_p, min_p0);
    char* p = (char*)ws;
    if (rounds) {
      a.listcap = list_cap(N);
      a.list = (Entry*)p; p += (int64_t)B * a.listcap * sizeof(Entry);
      a.state = (RowState*)p; p += round16(B * sizeof(RowState));
      a.hmass = (uint64_t*)p; p += (int64_t)B * BINS * 8;
      if (a.nseg > KEPT) { a.listed = (uint64_t*)p; p += (int64_t)B * a.nseg * 8; }
    }
    a.segmass = (double*)p; p += (int64_t)B * a.nseg * 8;
    a.segmax = (float*)p; p += (int64_t)B * a.nseg * 4;
    a.segtie = (int32_t*)p;
  }
  hipStream_t st = (hipStream_t)stream;
  const auto launch = [&] {
    return type == T_F32 ? run<T_F32>(a, rounds, st) : type == T_BF16 ? run<T_BF16>(a, rounds, st) : run<T_F16>(a, rounds, st);
  };
  if (B <= LAUNCH_ROWS) return launch();
  for (int64_t b = 0; b < B; b += LAUNCH_ROWS) {
    a.B = (int)(B - b < LAUNCH_ROWS ? B - b : LAUNCH_ROWS);
    a.s = (const char*)s + b * ld * (type == T_F32 ? 4 : 2);
    a.u = u + b;
    a.temperature = temperature ? temperature + b : nullptr;
    a.top_k = top_k ? top_k + b : nullptr;
    a.top_p = top_p ? top_p + b : nullptr;
    a.min_p = min_p ? min_p + b : nullptr;
    a.out = out + b;
    a.prob = prob ? prob + b : nullptr;
    const int rc = launch();
    if (rc) return rc;
  }
  return 0;
}
