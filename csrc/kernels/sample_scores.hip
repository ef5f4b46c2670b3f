// One index per row of scores, drawn from the softmax cut by top-k, top-p and min-p, from a
// given uniform number (gfx950).
//
//   w_i  = exp((s_i - max s) / T)                  -inf and NaN are masked (w = 0)
//   top-k  the k best (equal scores: lowest index first)
//   top-p  of those, best first, the ones before which less than p of their mass lies
//   min-p  of those, the ones with w_i >= min_p    (the best one has w = 1)
//   answer the first index i with sum_{j <= i, j kept} w_j > u * sum_{j kept} w_j
//
// Bound by one read of the scores, so a long row is read once in full (stats pass: the
// largest score of every segment of 256, and its mass where no top-k or top-p is asked
// for); the finishing workgroup of a row then reads only segments whose largest score can
// matter.  A row of up to 32768 scores takes one launch: its workgroup holds it in registers (up
// to 4096) or reads it again from the cache.
//
// Nothing is sorted.  Thresholds are found over 2048 bins of (max s - s) / T, 32 to an octave of
// weight, and the few scores of the bin that holds the threshold are ranked against each
// other; a bin with too many (ties, a very high T) is split by the bits of the scores.
// Weights are computed in 64 bits: an answer depends on which side of u * total a sum of up
// to N weights falls.  Where masses meet in atomics they are whole multiples of 2^-shift, so
// their order does not matter; the other sums are in a fixed order.
#include <hip/hip_fp16.h>

#include "common.h"

using namespace fps;

namespace {

enum { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };

constexpr int SEG = 256;        // scores per segment: one wave, four a lane
constexpr int BINS = 2048;
constexpr int THREADS = 1024;   // of the finishing workgroup
constexpr int WAVES = THREADS / 64;
constexpr int LIST = 2048;      // scores ranked against each other
constexpr int SHORT_K = 512;    // top-k up to this may take its candidates from the segments' maxima
constexpr int HIST_SEGS = 128;  // segments per workgroup of the histogram pass

struct Args {
  const void* s;
  int64_t ld, N, nseg;
  int B, type, vec;
  const float* u;
  // per row, or nullptr and the same for all rows
  const float* temperature; double temperature0;
  const int32_t* top_k; int64_t top_k0;
  const float* top_p; double top_p0;
  const float* min_p; double min_p0;
  int32_t* out;
  float* prob;
  // workspace (long rows)
  float* segmax;    // [B, nseg]
  double* segmass;  // [B, nseg]
  int32_t* segtie;  // [B, nseg]
  uint32_t* hcount; // [B, BINS]
  uint64_t* hmass;  // [B, BINS]
};

struct Row {
  double c;      // log2(e) / T
  double p, minp;
  int64_t k;     // 0: off
  bool cut_p, cut_min;
  __device__ bool direct() const { return k == 0 && !cut_p; }
  __device__ bool short_list(int64_t nseg) const { return k > 0 && k <= SHORT_K && nseg >= k; }
};

__device__ __forceinline__ Row row_settings(const Args& a, int b) {
  Row r;
  const double T = a.temperature ? (double)a.temperature[b] : a.temperature0;
  r.k = a.top_k ? (int64_t)a.top_k[b] : a.top_k0;
  r.p = a.top_p ? (double)a.top_p[b] : a.top_p0;
  r.minp = a.min_p ? (double)a.min_p[b] : a.min_p0;
  r.c = 1.4426950408889634 / T;
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

// 2^((s - M) c): interpolation of 2^f at the Chebyshev nodes of [-1/2, 1/2], degree 10
// (relative error 3e-16), times the power of two
__device__ __forceinline__ double weight(float s, float M, double c) {
  if (s == M) return 1.0;
  const double t = ((double)s - (double)M) * c;
  if (!(t > -1020.0)) return 0.0;
  const double n = __builtin_rint(t), f = t - n;
  double p = 0x1.e6063bb9d7e13p-28;
  p = __builtin_fma(p, f, 0x1.b675bcea1ca08p-24);
  p = __builtin_fma(p, f, 0x1.62bfd4792ba8bp-20);
  p = __builtin_fma(p, f, 0x1.ffcb5405de21bp-17);
  p = __builtin_fma(p, f, 0x1.430913096f0eap-13);
  p = __builtin_fma(p, f, 0x1.5d87fe9d7a7abp-10);
  p = __builtin_fma(p, f, 0x1.3b2ab6fba1de4p-7);
  p = __builtin_fma(p, f, 0x1.c6b08d703ce47p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff82c598p-3);
  p = __builtin_fma(p, f, 0x1.62e42fefa3a19p-1);
  p = __builtin_fma(p, f, 1.0);
  return __longlong_as_double(__double_as_longlong(p) + ((int64_t)(int)n << 52));
}

// w in [0, 1] as a whole multiple of 2^-shift, shift <= 51 (rounded to nearest even)
__device__ __forceinline__ uint64_t fixed(double w, int shift) {
  const double magic = 4503599627370496.0;  // 2^52
  const double d = __builtin_fma(w, (double)(1ull << shift), magic);
  return (uint64_t)__double_as_longlong(d) & 0x000fffffffffffffull;
}
// N weights must not pass 2^63
__device__ __forceinline__ int shift_for(int64_t N) { return min(51, 62 - (64 - __clzll((uint64_t)N))); }

__device__ __forceinline__ int bin_of(float s, float M, float cb) {
  if (s == M) return 0;
  return (int)fminf((M - s) * cb, (float)(BINS - 1));
}

template <int T>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  float f;
  if (T == T_F32) f = ((const float*)p)[i];
  else {
    const uint16_t b = ((const uint16_t*)p)[i];
    f = T == T_BF16 ? bf16_to_f32(b) : __half2float(__ushort_as_half(b));
  }
  return f;
}

// NaN is masked; -0 and +0 are one score
__device__ __forceinline__ float clean(float f) { return f == f ? f + 0.f : -INFINITY; }

// this lane's four scores of a segment; places past the row are masked
template <int T>
__device__ __forceinline__ void load_seg(const Args& a, int b, int64_t seg, int lane, float v[4]) {
  const int64_t i = seg * SEG + lane * 4, at = (int64_t)b * a.ld + i;
  if (a.vec && i + 4 <= a.N) {
    if (T == T_F32) {
      const float4 f = *(const float4*)((const float*)a.s + at);
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      const uint2 u = *(const uint2*)((const uint16_t*)a.s + at);
      const uint32_t w[2] = {u.x, u.y};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint16_t lo = (uint16_t)w[j], hi = (uint16_t)(w[j] >> 16);
        v[2 * j] = T == T_BF16 ? bf16_to_f32(lo) : __half2float(__ushort_as_half(lo));
        v[2 * j + 1] = T == T_BF16 ? bf16_to_f32(hi) : __half2float(__ushort_as_half(hi));
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j < a.N ? load1<T>(a.s, at + j) : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = clean(v[j]);
}

__device__ __forceinline__ float wave_max(float v) { return group_max<64>(v); }

template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ---- long rows, pass 1: the largest score of every segment, its mass for direct rows --------
constexpr int STAT_SEGS = 8;  // per wave
template <int T>
__global__ void __launch_bounds__(256) stats_kernel(Args a, int hist) {
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const Row r = row_settings(a, b);
  if (hist)  // the histogram pass adds to these
    for (int i = blockIdx.x * 256 + threadIdx.x; i < BINS; i += gridDim.x * 256) {
      a.hcount[(int64_t)b * BINS + i] = 0;
      a.hmass[(int64_t)b * BINS + i] = 0;
    }
  const int64_t seg0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * STAT_SEGS;
  const bool mass = r.direct() && !r.cut_min;
#pragma unroll 4
  for (int j = 0; j < STAT_SEGS; ++j) {
    const int64_t seg = seg0 + j;
    if (seg >= a.nseg) return;
    float v[4];
    load_seg<T>(a, b, seg, lane, v);
    const float m = wave_max(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
    double w = 0;
    if (mass && m > -INFINITY) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w += weight(v[i], m, r.c);
      w = wave_sum(w);
    }
    if (lane == 0) {
      a.segmax[(int64_t)b * a.nseg + seg] = m;
      if (mass) a.segmass[(int64_t)b * a.nseg + seg] = w;
    }
  }
}

__device__ __forceinline__ float block_max(float v, float* tmp) {
  v = wave_max(v);
  const int nw = blockDim.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
  __syncthreads();
  float m = tmp[0];
  for (int i = 1; i < nw; ++i) m = fmaxf(m, tmp[i]);
  return m;
}

// add one score to a histogram in LDS; a wave whose lanes all hit one bin adds once
__device__ __forceinline__ void hist_add(uint32_t* hc, unsigned long long* hm, bool on, int bin, uint64_t w) {
  const uint64_t live = __ballot(on);
  if (live == 0) return;
  const int first = __shfl(bin, __ffsll((unsigned long long)live) - 1, 64);
  if (__ballot(on && bin == first) == live) {
    const uint64_t sum = wave_sum(on ? w : 0ull);
    if ((threadIdx.x & 63) == 0) {
      atomicAdd(hc + first, (uint32_t)__popcll(live));
      atomicAdd(hm + first, (unsigned long long)sum);
    }
  } else if (on) {
    atomicAdd(hc + bin, 1u);
    atomicAdd(hm + bin, (unsigned long long)w);
  }
}

// ---- long rows, pass 2 (rows that cut by mass, or by a long top-k): counts and masses by bin ---
template <int T>
__global__ void __launch_bounds__(THREADS) hist_kernel(Args a) {
  __shared__ uint32_t hc[BINS];
  __shared__ unsigned long long hm[BINS];
  __shared__ float tmp[WAVES];
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Row r = row_settings(a, b);
  if (r.direct() || r.short_list(a.nseg)) return;
  for (int i = threadIdx.x; i < BINS; i += THREADS) { hc[i] = 0; hm[i] = 0; }
  float m = -INFINITY;
  for (int64_t i = threadIdx.x; i < a.nseg; i += THREADS) m = fmaxf(m, a.segmax[(int64_t)b * a.nseg + i]);
  const float M = block_max(m, tmp);
  if (M == -INFINITY) return;
  const int shift = shift_for(a.N);
  const float cb = (float)(r.c * 32);
  const int64_t s0 = (int64_t)blockIdx.x * HIST_SEGS;
  for (int64_t seg = s0 + wave; seg < s0 + HIST_SEGS && seg < a.nseg; seg += WAVES) {
    float v[4];
    load_seg<T>(a, b, seg, lane, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) hist_add(hc, hm, v[j] > -INFINITY, bin_of(v[j], M, cb), fixed(weight(v[j], M, r.c), shift));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS)
    if (hc[i]) {
      atomicAdd(a.hcount + (int64_t)b * BINS + i, hc[i]);
      atomicAdd((unsigned long long*)a.hmass + (int64_t)b * BINS + i, hm[i]);
    }
}

// ---- the finishing workgroup of a row ------------------------------------------------------

struct Entry {
  uint32_t key;
  int32_t idx;
  uint64_t w;
};

struct Shared {
  uint32_t hc[BINS];
  unsigned long long hm[BINS];
  Entry list[LIST];
  float tmp[WAVES];
  uint32_t scan_c[WAVES];
  unsigned long long scan_m[WAVES];
  double scan_d[WAVES];
  // results of searches, written by one thread
  int bin, n, best;
  uint32_t kmin, ties, before_c;
  unsigned long long before_m, total_m, kept_m;
  int64_t seg;
  double seg_before, seg_mass;
};

// Where the finishing workgroup has the row: its one segment per wave in registers
// (ROW_REGS), or in memory, the segments' maxima in LDS (ROW_CACHED) or from the stats
// pass (ROW_LONG).
enum { ROW_REGS = 0, ROW_CACHED = 1, ROW_LONG = 2 };
constexpr int CACHED_SEGS = 8 * WAVES;

template <int T, int R>
struct Source {
  const Args& a;
  const int b, lane, wave;
  const float* segmax;
  float v[4];
  __device__ Source(const Args& a_, int b_, const float* sm)
      : a(a_), b(b_), lane(threadIdx.x & 63), wave(threadIdx.x >> 6), segmax(sm) {}
  // f(segment, scores) for every segment whose largest score is >= bound, waves in turn
  template <typename F>
  __device__ __forceinline__ void each(float bound, F f) {
    if constexpr (R == ROW_REGS) {
      if (wave < a.nseg) f((int64_t)wave, v);
    } else {
      for (int64_t seg = wave; seg < a.nseg; seg += WAVES) {
        if (segmax[seg] < bound || segmax[seg] == -INFINITY) continue;
        float x[4];
        load_seg<T>(a, b, seg, lane, x);
        f(seg, x);
      }
    }
  }
};

// Inclusive sums over the workgroup of (count, mass), thread order.
__device__ __forceinline__ void block_scan(uint32_t& c, uint64_t& m, Shared& sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t c2 = __shfl_up(c, o, 64);
    const uint64_t m2 = __shfl_up((unsigned long long)m, o, 64);
    if (lane >= o) { c += c2; m += m2; }
  }
  __syncthreads();
  if (lane == 63) { sh.scan_c[wave] = c; sh.scan_m[wave] = m; }
  __syncthreads();
  for (int i = 0; i < wave; ++i) { c += sh.scan_c[i]; m += sh.scan_m[i]; }
}

__device__ __forceinline__ double block_scan_d(double d, Shared& sh, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double d2 = __shfl_up(d, o, 64);
    if (lane >= o) d += d2;
  }
  __syncthreads();
  if (lane == 63) sh.scan_d[wave] = d;
  __syncthreads();
  double before = 0;
  total = 0;
  for (int i = 0; i < WAVES; ++i) {
    if (i == wave) before = total;
    total += sh.scan_d[i];
  }
  return before + d;
}

// The bin of the histogram in sh (bin 0 best) in which the count first reaches `need` (by_mass
// false) or the mass, added to `above`, first reaches `target`; sh.bin, sh.before_c, sh.before_m.
// Where rounding lets no bin reach it: the last bin that holds anything.
__device__ __forceinline__ void find_bin(Shared& sh, bool by_mass, uint32_t need, uint64_t above, double target) {
  const int i = threadIdx.x;
  const uint32_t c0 = sh.hc[2 * i], c1 = sh.hc[2 * i + 1];
  const uint64_t m0 = sh.hm[2 * i], m1 = sh.hm[2 * i + 1];
  uint32_t c = c0 + c1;
  uint64_t m = m0 + m1;
  block_scan(c, m, sh);
  if (i == 0) { sh.bin = BINS; sh.best = -1; }
  __syncthreads();
  const uint32_t cb0 = c - c1;       // count through bin 2 i
  const uint64_t mb0 = m - m1;
  const bool h0 = c0 && (by_mass ? (double)(above + mb0) >= target : cb0 >= need);
  const bool h1 = c1 && (by_mass ? (double)(above + m) >= target : c >= need);
  if (h0) atomicMin(&sh.bin, 2 * i);
  else if (h1) atomicMin(&sh.bin, 2 * i + 1);
  if (c1) atomicMax(&sh.best, 2 * i + 1);
  else if (c0) atomicMax(&sh.best, 2 * i);
  __syncthreads();
  const int bin = sh.bin < BINS ? sh.bin : sh.best;
  if (bin == 2 * i) { sh.before_c = cb0 - c0; sh.before_m = mb0 - m0; }
  else if (bin == 2 * i + 1) { sh.before_c = cb0; sh.before_m = mb0; }
  if (i == THREADS - 1) sh.total_m = m;
  __syncthreads();
  if (i == 0) sh.bin = bin;
  __syncthreads();
}

// Among the n listed scores, which stay: rank + above_c < k (k = 0: all), then, with `cut`,
// mass before + above_m < p * total; sh.kept_m their mass after top-k alone, kept bits in the
// caller's two slots (entries threadIdx.x and threadIdx.x + THREADS).
struct Slot {
  bool in, kept;
  uint64_t before;
};

__device__ __forceinline__ void rank_list(Shared& sh, int n, int64_t k, uint32_t above_c, Slot s[2]) {
  if (threadIdx.x == 0) sh.kept_m = 0;
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = threadIdx.x + h * THREADS;
    s[h].in = i < n;
    s[h].kept = false;
    s[h].before = 0;
    if ((i & ~63) < n) {  // whole waves
      const Entry e = sh.list[i < n ? i : 0];
      uint32_t rank = 0;
      uint64_t before = 0;
      for (int j = 0; j < n; ++j) {
        const Entry o = sh.list[j];
        const bool better = o.key > e.key || (o.key == e.key && o.idx < e.idx);
        rank += better;
        before += better ? o.w : 0ull;
      }
      s[h].before = before;
      s[h].kept = i < n && (k == 0 || (int64_t)above_c + rank < k);
      const uint64_t sum = wave_sum(s[h].kept ? e.w : 0ull);
      if ((threadIdx.x & 63) == 0) atomicAdd(&sh.kept_m, (unsigned long long)sum);
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void cut_by_mass(Slot s[2], uint64_t above_m, double target) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (s[h].kept) {
      const uint64_t before = above_m + s[h].before;
      s[h].kept = before == 0 || (double)before < target;  // the best one always stays
    }
}

// Put the scores for which pick(key, bin) holds into sh.list; sh.n counts them all.
template <int T, int R, typename F>
__device__ __forceinline__ void collect(Source<T, R>& src, Shared& sh, float bound, float M, const Row& r, float cb,
                                        int shift, F pick) {
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  src.each(bound, [&](int64_t seg, const float* v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool on = v[j] > -INFINITY && pick(key_of(v[j]), bin_of(v[j], M, cb));
      if (on) {
        const int at = atomicAdd(&sh.n, 1);
        if (at < LIST)
          sh.list[at] = Entry{key_of(v[j]), (int32_t)(seg * SEG + src.lane * 4 + j), fixed(weight(v[j], M, r.c), shift)};
      }
    }
  });
  __syncthreads();
}

// Split bin `bin` by the bits of the scores until one score value is left: the threshold key
// sh.kmin and how many scores equal to it stay (sh.ties).  By count: `need` of the bin's scores
// stay; by mass: those before which above_m + mass < target.  Only keys >= floor take part.
template <int T, int R>
__device__ __forceinline__ void split_bin(Source<T, R>& src, Shared& sh, float bound, float M, const Row& r, float cb,
                                          int shift, int bin, bool by_mass, uint32_t need, uint64_t above_m,
                                          double target, uint32_t floor_key) {
  uint32_t prefix = 0, mask = 0;
  for (int level = 0; level < 3; ++level) {
    const int sft = level == 0 ? 21 : level == 1 ? 10 : 0;
    const uint32_t width = level == 2 ? 1023u : 2047u;
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += THREADS) { sh.hc[i] = 0; sh.hm[i] = 0; }
    __syncthreads();
    src.each(bound, [&](int64_t, const float* v) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t key = key_of(v[j]);
        const bool on = v[j] > -INFINITY && bin_of(v[j], M, cb) == bin && (key & mask) == prefix && key >= floor_key;
        hist_add(sh.hc, sh.hm, on, (int)(width - ((key >> sft) & width)), on ? fixed(weight(v[j], M, r.c), shift) : 0);
      }
    });
    __syncthreads();
    find_bin(sh, by_mass, need, above_m, target);
    prefix |= (width - (uint32_t)sh.bin) << sft;
    mask |= width << sft;
    need -= min(need, sh.before_c);
    above_m += sh.before_m;
    if (level == 2) {
      const uint32_t cnt = sh.hc[sh.bin];
      uint32_t ties = need;
      if (by_mass) {  // tie number j stays while above + j w < target
        const uint64_t w = cnt ? sh.hm[sh.bin] / cnt : 0;
        const double room = target - (double)above_m;
        ties = w == 0 || room > (double)w * (double)cnt ? cnt : (uint32_t)fmax(0.0, ceil(room / (double)w));
        if (above_m == 0 && ties == 0) ties = 1;
      }
      __syncthreads();
      if (threadIdx.x == 0) { sh.kmin = prefix; sh.ties = min(ties, cnt); sh.before_m = above_m; }
    }
    __syncthreads();
  }
}

// the kept entries of the list as a threshold: smallest key, and how many of it
__device__ __forceinline__ void list_threshold(Shared& sh, const Slot s[2]) {
  if (threadIdx.x == 0) { sh.kmin = 0xffffffffu; sh.ties = 0; }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (s[h].kept) atomicMin(&sh.kmin, sh.list[threadIdx.x + h * THREADS].key);
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (s[h].kept && sh.list[threadIdx.x + h * THREADS].key == sh.kmin) atomicAdd(&sh.ties, 1u);
  __syncthreads();
}

// Draw from the kept entries of the list, in index order.
__device__ __forceinline__ void draw_from_list(const Args& a, int b, Shared& sh, int n, Slot s[2], const Row& r, float M) {
  __syncthreads();
  if (threadIdx.x == 0) { sh.kept_m = 0; sh.best = INT32_MAX; sh.bin = -1; }
  __syncthreads();
  Entry mine[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = threadIdx.x + h * THREADS;
    mine[h] = sh.list[i < n ? i : 0];
    if (s[h].kept && r.cut_min) s[h].kept = weight(score_of(mine[h].key), M, r.c) >= r.minp;
    if (!s[h].kept) mine[h].w = 0;
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = threadIdx.x + h * THREADS;
    if (i < n) sh.list[i].w = mine[h].w;
    const uint64_t sum = wave_sum(mine[h].w);
    if ((threadIdx.x & 63) == 0) atomicAdd(&sh.kept_m, (unsigned long long)sum);
  }
  __syncthreads();
  const double total = (double)sh.kept_m, target = (double)a.u[b] * total;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = threadIdx.x + h * THREADS;
    if ((i & ~63) < n) {
      uint64_t cum = 0;
      for (int j = 0; j < n; ++j) {
        const Entry o = sh.list[j];
        cum += o.idx <= mine[h].idx ? o.w : 0ull;
      }
      if (i < n && mine[h].w) {
        if ((double)cum > target) atomicMin(&sh.best, mine[h].idx);
        atomicMax(&sh.bin, mine[h].idx);
      }
    }
  }
  __syncthreads();
  const int pick = sh.best != INT32_MAX ? sh.best : sh.bin;
  if (threadIdx.x == 0) a.out[b] = pick;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (threadIdx.x + h * THREADS < n && mine[h].w && mine[h].idx == pick && a.prob) a.prob[b] = (float)((double)mine[h].w / total);
}

// Draw from the scores above key t and the first `ties` equal to it, in index order.
template <int T, int R>
__device__ __forceinline__ void draw_from_row(const Args& a, int b, Source<T, R>& src, Shared& sh, const Row& r, float M,
                                              uint32_t t, uint32_t ties, double* segmass, int32_t* segtie, bool have_mass) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float bound = score_of(max(t, KEY_NONE));
  const float tie_score = bound;
  double wt = 0;
  if (ties) {
    wt = weight(tie_score, M, r.c);
    if (r.cut_min && wt < r.minp) { wt = 0; ties = 0; }
  }
  if (!have_mass)
    src.each(bound, [&](int64_t seg, const float* v) {
      double m = 0;
      int c = 0;
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
      if (lane == 0) { segmass[seg] = m; segtie[seg] = c; }
    });
  __syncthreads();
  // two walks over the segments: the total, then the segment in which u * total falls
  double total = 0, target = 0;
  for (int walk = 0; walk < 2; ++walk) {
    uint32_t tie_before = 0;
    double before = 0;
    if (threadIdx.x == 0 && walk) { sh.seg = -1; }
    bool found = false;
    int64_t last = -1;
    for (int64_t base = 0; base < a.nseg; base += THREADS) {
      const int64_t seg = base + threadIdx.x;
      double m = 0;
      uint32_t c = 0;
      if (seg < a.nseg && src.segmax[seg] >= bound && src.segmax[seg] > -INFINITY) {
        m = segmass[seg];
        if (have_mass) m *= weight(src.segmax[seg], M, r.c);
        else c = (uint32_t)segtie[seg];
      }
      uint32_t cc = c;
      if (ties) {
        uint64_t none = 0;
        block_scan(cc, none, sh);
        const uint32_t t0 = tie_before + cc - c;  // ties in earlier segments
        const uint32_t kept = t0 < ties ? min(ties - t0, c) : 0;
        m += kept * wt;
        __syncthreads();
        if (threadIdx.x == THREADS - 1) sh.before_c = cc;
        __syncthreads();
        tie_before += sh.before_c;
      }
      double part;
      const double cum = before + block_scan_d(m, sh, part);
      if (walk) {
        if (threadIdx.x == 0) { sh.best = INT32_MAX; sh.bin = -1; }
        __syncthreads();
        if (m > 0) {
          if (!found && cum > target) atomicMin(&sh.best, (int)threadIdx.x);
          atomicMax(&sh.bin, (int)threadIdx.x);
        }
        __syncthreads();
        const int hit = sh.best, any = sh.bin;
        if (!found && (hit != INT32_MAX || any >= 0)) {
          const int at = hit != INT32_MAX ? hit : any;
          // ties kept before this segment, for its scan
          if ((int)threadIdx.x == at) {
            sh.seg = seg;
            sh.seg_before = cum - m;
            sh.ties = ties ? tie_before - sh.before_c + cc - c : 0;
          }
          last = 0;
          if (hit != INT32_MAX) found = true;
        }
        __syncthreads();
        if (found) break;
      }
      before += part;
    }
    if (!walk) {
      total = before;
      target = (double)a.u[b] * total;
    } else if (!found && last == 0) {
      target = INFINITY;  // rounding put u * total past the last mass: its last score
    }
    __syncthreads();
  }
  const int64_t seg = sh.seg;
  if (wave == (R == ROW_REGS ? (int)seg : 0) && seg >= 0) {
    float v[4];
    if constexpr (R == ROW_REGS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = src.v[j];
    } else {
      load_seg<T>(a, b, seg, lane, v);
    }
    int c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) c += v[j] > -INFINITY && key_of(v[j]) == t;
    int cs = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int c2 = __shfl_up(cs, o, 64);
      if (lane >= o) cs += c2;
    }
    uint32_t tie = sh.ties + cs - c;
    double w[4], m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t key = key_of(v[j]);
      w[j] = 0;
      if (v[j] > -INFINITY) {
        if (key > t) {
          w[j] = weight(v[j], M, r.c);
          if (r.cut_min && w[j] < r.minp) w[j] = 0;
        } else if (key == t) {
          if (tie < ties) w[j] = wt;
          ++tie;
        }
      }
      m += w[j];
    }
    double ms = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double m2 = __shfl_up(ms, o, 64);
      if (lane >= o) ms += m2;
    }
    double cum = sh.seg_before + (ms - m);
    int hit = -1, end = -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      cum += w[j];
      if (w[j] > 0) {
        if (hit < 0 && cum > target) hit = j;
        end = j;
      }
    }
    const uint64_t hits = __ballot(hit >= 0), ends = __ballot(end >= 0);
    const int win = hits ? __ffsll((unsigned long long)hits) - 1 : 63 - __clzll(ends);
    if (lane == win) {
      const int j = hits ? hit : end;
      a.out[b] = (int32_t)(seg * SEG + lane * 4 + j);
      if (a.prob) a.prob[b] = (float)((j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3]) / total);
    }
  }
}

template <int T, int R>
__global__ void __launch_bounds__(THREADS) finish_kernel(Args a, int have_hist) {
  __shared__ Shared sh;
  constexpr int SMALL = R == ROW_REGS ? WAVES : R == ROW_CACHED ? CACHED_SEGS : 1;
  __shared__ float small_max[SMALL];
  __shared__ double small_mass[SMALL];
  __shared__ int32_t small_tie[SMALL];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Row r = row_settings(a, b);
  const bool own = R != ROW_LONG;
  const float* segmax = own ? small_max : a.segmax + (int64_t)b * a.nseg;
  double* segmass = own ? small_mass : a.segmass + (int64_t)b * a.nseg;
  int32_t* segtie = own ? small_tie : a.segtie + (int64_t)b * a.nseg;
  Source<T, R> src(a, b, segmax);
  float m = -INFINITY;
  if constexpr (R != ROW_LONG) {
    for (int64_t seg = wave; seg < a.nseg; seg += WAVES) {  // (ROW_REGS: one)
      load_seg<T>(a, b, seg, lane, src.v);
      const float x = wave_max(fmaxf(fmaxf(src.v[0], src.v[1]), fmaxf(src.v[2], src.v[3])));
      if (lane == 0) small_max[seg] = x;
      m = fmaxf(m, x);
    }
  } else {
    for (int64_t i = threadIdx.x; i < a.nseg; i += THREADS) m = fmaxf(m, segmax[i]);
  }
  const float M = block_max(m, sh.tmp);
  if (M == -INFINITY) {  // nothing is left of the row
    if (threadIdx.x == 0) {
      a.out[b] = -1;
      if (a.prob) a.prob[b] = 0.f;
    }
    return;
  }
  const float cb = (float)(r.c * 32);
  if (r.direct()) {
    draw_from_row<T, R>(a, b, src, sh, r, M, KEY_NONE, 0, segmass, segtie, R == ROW_LONG && !r.cut_min);
    return;
  }
  if (r.short_list(a.nseg)) {
    // The k best scores lie in bins up to the one in which the count of segment maxima
    // reaches k: that many scores, one a segment, are already in them.
    for (int i = threadIdx.x; i < BINS; i += THREADS) { sh.hc[i] = 0; sh.hm[i] = 0; }
    __syncthreads();
    for (int64_t i0 = 0; i0 < a.nseg; i0 += THREADS) {
      const int64_t i = i0 + threadIdx.x;
      const float x = i < a.nseg ? segmax[i] : -INFINITY;
      if (x > -INFINITY) atomicAdd(&sh.hc[bin_of(x, M, cb)], 1u);
    }
    __syncthreads();
    find_bin(sh, false, (uint32_t)r.k, 0, 0.0);
    // fewer unmasked segments than k: everything unmasked is a candidate
    const bool all = sh.before_c + sh.hc[sh.bin] < (uint32_t)r.k;
    const int edge = all ? BINS : sh.bin;
    collect<T, R>(src, sh, -INFINITY, M, r, cb, 51, [&](uint32_t, int bin) { return bin <= edge; });
    const int n = sh.n;
    if (n <= LIST) {
      Slot s[2];
      rank_list(sh, n, r.k, 0, s);
      if (r.cut_p) cut_by_mass(s, 0, r.p * (double)sh.kept_m);
      draw_from_list(a, b, sh, n, s, r, M);
      return;
    }
  }
  const int shift = shift_for(a.N);
  const bool ready = have_hist && !r.short_list(a.nseg);
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS) {
    sh.hc[i] = ready ? a.hcount[(int64_t)b * BINS + i] : 0;
    sh.hm[i] = ready ? a.hmass[(int64_t)b * BINS + i] : 0;
  }
  __syncthreads();
  if (!ready) {
    src.each(-INFINITY, [&](int64_t, const float* v) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        hist_add(sh.hc, sh.hm, v[j] > -INFINITY, bin_of(v[j], M, cb), fixed(weight(v[j], M, r.c), shift));
    });
    __syncthreads();
  }
  // threshold key and ties of the scores that stay
  uint32_t t = KEY_NONE, ties = 0;
  uint64_t total;
  int kbin = BINS;        // bin of the top-k threshold
  uint64_t kbefore = 0;   // mass of the bins before it
  if (r.k > 0) {
    const bool cut_p = r.cut_p;
    // (the p search below needs the histogram again: keep this thread's two bins)
    const uint32_t c0 = sh.hc[2 * threadIdx.x], c1 = sh.hc[2 * threadIdx.x + 1];
    const uint64_t m0 = sh.hm[2 * threadIdx.x], m1 = sh.hm[2 * threadIdx.x + 1];
    find_bin(sh, false, (uint32_t)min(r.k, (int64_t)UINT32_MAX), 0, 0.0);
    kbin = sh.bin;
    kbefore = sh.before_m;
    const uint32_t cbefore = sh.before_c;
    const float bound = -INFINITY;
    if (cbefore + sh.hc[kbin] <= r.k) {  // the whole bin stays
      t = KEY_NONE;
      ties = 0;
      total = kbefore + sh.hm[kbin];
      // everything in bins <= kbin: the smallest key among them is the threshold
      if (threadIdx.x == 0) sh.kmin = 0xffffffffu;
      __syncthreads();
      src.each(bound, [&](int64_t, const float* v) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (v[j] > -INFINITY && bin_of(v[j], M, cb) == kbin) atomicMin(&sh.kmin, key_of(v[j]));
      });
      __syncthreads();
      t = sh.kmin - 1;  // keys above t stay
    } else {
      collect<T, R>(src, sh, bound, M, r, cb, shift, [&](uint32_t, int bin) { return bin == kbin; });
      const int n = sh.n;
      if (n <= LIST) {
        Slot s[2];
        rank_list(sh, n, r.k, cbefore, s);
        total = kbefore + sh.kept_m;
        list_threshold(sh, s);
        t = sh.kmin;
        ties = sh.ties;
      } else {
        split_bin<T, R>(src, sh, bound, M, r, cb, shift, kbin, false, (uint32_t)(r.k - cbefore), kbefore, 0.0, 0);
        t = sh.kmin;
        ties = sh.ties;
        total = sh.before_m + (uint64_t)ties * fixed(weight(score_of(t), M, r.c), shift);
      }
    }
    if (cut_p) {
      __syncthreads();
      // the histogram of the scores that top-k left: bins past its threshold's are empty
      const int i0 = 2 * threadIdx.x, i1 = i0 + 1;
      sh.hc[i0] = i0 <= kbin ? c0 : 0;
      sh.hc[i1] = i1 <= kbin ? c1 : 0;
      sh.hm[i0] = i0 < kbin ? m0 : i0 == kbin ? total - kbefore : 0;
      sh.hm[i1] = i1 < kbin ? m1 : i1 == kbin ? total - kbefore : 0;
      __syncthreads();
    }
  }
  if (r.cut_p) {
    if (r.k == 0) {
      // the total is the last inclusive sum of the scan
      find_bin(sh, true, 0, 0, INFINITY);
      total = sh.total_m;
    }
    const double target = r.p * (double)total;
    find_bin(sh, true, 0, 0, target);
    const int bin = sh.bin;
    const uint64_t above = sh.before_m;
    const uint32_t floor_key = bin == kbin ? (ties ? t : t + 1) : 0;  // what top-k left of this bin
    const uint32_t tie_cap = bin == kbin && ties ? ties : 0xffffffffu;
    collect<T, R>(src, sh, -INFINITY, M, r, cb, shift,
                  [&](uint32_t key, int x) { return x == bin && key >= floor_key; });
    const int n = sh.n;
    if (n <= LIST) {
      // (scores equal to top-k's threshold beyond its ties are ranked behind all that stay, and
      // the mass before them has reached the total: the cut drops them)
      Slot s[2];
      rank_list(sh, n, 0, 0, s);
      cut_by_mass(s, above, target);
      list_threshold(sh, s);
    } else {
      split_bin<T, R>(src, sh, -INFINITY, M, r, cb, shift, bin, true, 0, above, target, floor_key);
    }
    __syncthreads();
    const uint32_t t2 = sh.kmin, ties2 = sh.ties;
    ties = t2 == floor_key ? min(ties2, tie_cap) : ties2;
    t = t2;
  }
  __syncthreads();
  draw_from_row<T, R>(a, b, src, sh, r, M, t, ties, segmass, segtie, false);
}

template <int T>
int run(Args& a, int hist, hipStream_t st) {
  if (a.nseg <= WAVES) {
    hipLaunchKernelGGL((finish_kernel<T, ROW_REGS>), dim3(a.B), dim3(THREADS), 0, st, a, 0);
  } else if (a.nseg <= CACHED_SEGS) {
    hipLaunchKernelGGL((finish_kernel<T, ROW_CACHED>), dim3(a.B), dim3(THREADS), 0, st, a, 0);
  } else {
    const int per = 4 * STAT_SEGS;
    hipLaunchKernelGGL((stats_kernel<T>), dim3((unsigned)((a.nseg + per - 1) / per), a.B), dim3(256), 0, st, a, hist);
    FPS_CHECK_LAUNCH();
    if (hist) {
      hipLaunchKernelGGL((hist_kernel<T>), dim3((unsigned)((a.nseg + HIST_SEGS - 1) / HIST_SEGS), a.B), dim3(THREADS), 0,
                         st, a);
      FPS_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL((finish_kernel<T, ROW_LONG>), dim3(a.B), dim3(THREADS), 0, st, a, hist);
  }
  FPS_CHECK_LAUNCH();
  return 0;
}

constexpr int64_t kShortRow = (int64_t)CACHED_SEGS * SEG;  // rows up to this take no workspace

}  // namespace

// bytes of workspace for B rows of N scores
FPS_API int64_t fps_sample_scores_ws_bytes(int64_t B, int64_t N) {
  if (B <= 0 || N <= kShortRow) return 0;
  const int64_t nseg = (N + SEG - 1) / SEG;
  return B * (BINS * 12 + nseg * 16);
}

// s [B, N] (row stride ld, type 0 fp32 / 1 bf16 / 2 fp16); u [B]; temperature / top_k / top_p /
// min_p: per row, or nullptr and the scalar after it.  out [B] indices (-1: nothing left of
// the row), prob [B] or nullptr.
FPS_API int fps_sample_scores(const void* s, int type, int B, int64_t N, int64_t ld, const float* u,
                              const float* temperature, double temperature0, const int32_t* top_k, int64_t top_k0,
                              const float* top_p, double top_p0, const float* min_p, double min_p0, int32_t* out,
                              float* prob, void* ws, void* stream) {
  if (B <= 0) return 0;
  if (N <= 0 || N > INT32_MAX || ld < N || type < 0 || type > 2 || (B > 65535 && N > kShortRow)) return (int)hipErrorInvalidValue;
  Args a;
  a.s = s; a.ld = ld; a.N = N; a.nseg = (N + SEG - 1) / SEG; a.B = B; a.type = type;
  a.vec = (B == 1 || ld % 4 == 0) && ((uintptr_t)s & (type == T_F32 ? 15 : 7)) == 0;
  a.u = u;
  a.temperature = temperature; a.temperature0 = temperature0;
  a.top_k = top_k; a.top_k0 = top_k0;
  a.top_p = top_p; a.top_p0 = top_p0;
  a.min_p = min_p; a.min_p0 = min_p0;
  a.out = out; a.prob = prob;
  a.segmax = nullptr; a.segmass = nullptr; a.segtie = nullptr; a.hcount = nullptr; a.hmass = nullptr;
  int hist = 0;
  if (N > kShortRow) {
    if (ws == nullptr) return (int)hipErrorInvalidValue;
    char* p = (char*)ws;
    a.hmass = (uint64_t*)p; p += (int64_t)B * BINS * 8;
    a.segmass = (double*)p; p += (int64_t)B * a.nseg * 8;
    a.hcount = (uint32_t*)p; p += (int64_t)B * BINS * 4;
    a.segmax = (float*)p; p += (int64_t)B * a.nseg * 4;
    a.segtie = (int32_t*)p;
    // can a row need the histogram?  (scalars decide here, per-row settings on the device)
    const bool greedy = !temperature && !(temperature0 > 0);
    const int64_t k = top_k0 <= 0 || top_k0 >= N ? 0 : top_k0;
    if (greedy) hist = 0;
    else if (top_k) hist = 1;
    else if (k) hist = k > SHORT_K || a.nseg < k;
    else hist = top_p || top_p0 < 1;
  }
  hipStream_t st = (hipStream_t)stream;
  return type == T_F32 ? run<T_F32>(a, hist, st) : type == T_BF16 ? run<T_BF16>(a, hist, st) : run<T_F16>(a, hist, st);
}
