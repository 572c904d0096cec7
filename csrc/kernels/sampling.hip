// One token per row of logits, from a given random number: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T)                     weights; x ordered by (value descending, index ascending)
//   top-k: the first k of that order;  top-p: of what is left, the shortest head whose mass reaches p of it;
//   min-p: of what is left, w_i >= min_p (w of the best is 1);
//   token = the first index, in index order, whose cumulative kept mass exceeds u * (kept mass).
//
// A choice next to a border turns on the last bits of these sums, so weights are computed in 64 bits and summed as
// integers of 2^-shift, shift = min(50, 62 - bits of V) (50 up to 4,096 tokens, 45 at 131,072, 42 at 2^20): integer sums do
// not depend on the order they are taken in, so a row's token is the same in every launch.  A weight is off by half a unit
// and, from its series, by 2e-13 of itself; rows taken from the start use exp instead.  Which way a row goes depends on the
// row and its settings alone.  No sort.  Four launches; a row is cut into chunks of 512 logits (a wave's load) and groups of
// 32 or 128:
//   peaks_kernel   every group's largest logit;
//   bins_kernel    knows the row's largest.  Without top-k and top-p: the kept mass of every chunk.  Top-p alone: masses
//                  over 2,047 bins of 1/64 in log2 of the weight, and of the tail behind them;
//   sweep_kernel   top-p alone: finds the bin of the border, sums what lies above it per chunk, lists what lies in it;
//   choose_kernel  one workgroup per row: the border's place in the list, the chunk, the token.  Top-k (up to half the
//                  groups and 512) is done here alone: the k-th best group's largest logit bounds the k-th best logit from
//                  below, so some k groups are read, and the few logits above the bound are ranked all against all.
// Rows that fit none of this (a larger k, an infinite logit, a border in the tail or with more than 8,192 logits in its
// bin, a number below 2^-40 or from 1 on) are taken from the start in choose_kernel: radix selection on the ordered bits of
// the logits.
//
// Measured: 256 rows of 131,072 bf16 logits with settings of their own 99 - 107 us (peaks 15, 4.6 TB/s; bins 39 and sweep 42:
// 45 % of the rows have work there, whose slices lie unevenly on the CUs, busy 55 - 65 % of the time, and vector instructions
// fill two thirds of a busy one's issue slots; choose 26, bound by latency); 32 of 50,257 fp32 with top-k and top-p 13 (two
// launches); 64 of 32,000 fp16 with min-p 15 (three); one of 32,000 with top-p 23 - 28 (four, 3 - 9 each).  From the start: 32
// rows of 32,000 with k = 513 67 us (k = 500: 41), 256 such rows 80, 32 of 131,072 158, all logits equal 151 - 173.  Min-p alone
// skips the weights of logits below its floor: 256 x 131,072 with a deviation of 0.7, 1.5 and 2.5 take 61, 55 and 41 us,
// without that 59, 60 and 49.  choose_kernel with its arguments in registers alone, one inlined call of the rare path, is
// 4 - 9 us shorter than with that path as a function.
#include "common.h"

namespace pd {
namespace smp {

typedef unsigned long long u64;
constexpr int kChunk = 512, kMaxChunks = 2048;   // V <= 2^20
constexpr int kBins = 2048, kList = 8192, kShort = 1024, kMaxK = 512, kWide = 8;

// bits that order as the values do; NaN as -inf, -0 as +0
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// Lanes of a wave summed by data-parallel moves (row_shr 1, 2, 4, 8, then row_bcast 15 and 31): a fifth of the latency of
// shuffles through LDS.  Lanes without a source add 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int old, int v) {
  return __builtin_amdgcn_update_dpp(old, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved64(u64 v) {
  const unsigned lo = (unsigned)moved<CTRL, ROWS>(0, (int)(unsigned)v), hi = (unsigned)moved<CTRL, ROWS>(0, (int)(v >> 32));
  return ((u64)hi << 32) | lo;
}
// inclusive prefix over the lanes
__device__ __forceinline__ u64 wave_scan64(u64 v) {
  v += moved64<0x111, 0xf>(v);
  v += moved64<0x112, 0xf>(v);
  v += moved64<0x114, 0xf>(v);
  v += moved64<0x118, 0xf>(v);
  v += moved64<0x142, 0xa>(v);
  v += moved64<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ int wave_scan32(int v) {
  v += moved<0x111, 0xf>(0, v);
  v += moved<0x112, 0xf>(0, v);
  v += moved<0x114, 0xf>(0, v);
  v += moved<0x118, 0xf>(0, v);
  v += moved<0x142, 0xa>(0, v);
  v += moved<0x143, 0xc>(0, v);
  return v;
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
  v = wave_scan64(v);
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, 63);
  return ((u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32) | lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved_max(float v) {
  const int i = __float_as_int(v);
  return fmaxf(v, __int_as_float(moved<CTRL, ROWS>(i, i)));
}
__device__ __forceinline__ float wave_peak(float v) {
  v = moved_max<0x111, 0xf>(v);
  v = moved_max<0x112, 0xf>(v);
  v = moved_max<0x114, 0xf>(v);
  v = moved_max<0x118, 0xf>(v);
  v = moved_max<0x142, 0xa>(v);
  v = moved_max<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// 8 logits from index i; -inf past the row's end and for NaN.  Rows of odd lengths start at odd addresses: the copy
// lets the compiler use one unaligned 16-byte load.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int i, int V, float (&x)[8]) {
  if (i + 8 <= V) {
    T raw[8];
    __builtin_memcpy(raw, row + i, sizeof(raw));
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = Elt<T>::ld(raw + j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = i + j < V ? Elt<T>::ld(row + i + j) : -INFINITY;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = x[j] != x[j] ? -INFINITY : x[j];
}

struct Row {
  float top;      // the row's largest logit
  double inv_t;   // 1 / temperature
  double unit;    // 2^shift
};
__device__ __forceinline__ double weight(const Row& r, float x) {
  if (x == r.top) return 1.0;   // also where both are +inf
  if (x == -INFINITY) return 0.0;
  return exp(((double)x - (double)r.top) * r.inv_t);
}
__device__ __forceinline__ u64 fixed(const Row& r, double w) { return (u64)(w * r.unit + 0.5); }

// f(chunk, x) for those of the chunks c, c + step, c + 2 step .. < c1 that want(chunk) names, by one wave.  want is asked
// by a lane per chunk; the loads of four chunks are in flight before the first is worked on (one at a time, the latency of
// each was most of the time).
template <typename T, typename Want, typename F>
__device__ __forceinline__ void walk(const T* __restrict__ row, int V, int c, int c1, int step, Want want, F f) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  constexpr int N = 4, Q = sizeof(T) / 2;   // 16-byte loads per lane and chunk
  const int lane = threadIdx.x & 63;
  for (; c < c1; c += 64 * step) {
    u64 todo = __ballot(c + lane * step < c1 && want(c + lane * step));
    while (todo) {
      u32x4 raw[N][Q];
      int at[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        at[n] = todo ? c + (__ffsll((long long)todo) - 1) * step : -1;
        todo &= todo - 1;
        if (at[n] >= 0 && (at[n] + 1) * kChunk <= V) __builtin_memcpy(raw[n], row + (long)at[n] * kChunk + lane * 8, 16 * Q);
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (at[n] < 0) break;
        float x[8];
        if ((at[n] + 1) * kChunk <= V) {
          T t[8];
          __builtin_memcpy(t, raw[n], sizeof(t));
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            x[j] = Elt<T>::ld(t + j);
            x[j] = x[j] != x[j] ? -INFINITY : x[j];
          }
        } else {
          load8(row, at[n] * kChunk + lane * 8, V, x);
        }
        f(at[n], x);
      }
    }
  }
}

struct Setting {
  const float* p;   // one value per row, or null
  float v;
};

// Everything a launch needs; settings per row (pointers) or for all rows.
template <typename T>
struct Args {
  const T* logits;
  long stride;
  int V, chunks, groups, group_lanes, shift;   // a group: group_lanes x 8 logits
  const float* uniform;
  Setting temp, top_p, min_p;
  const int* top_ks;
  int top_k;
  u64* mass;       // [B][chunks] kept mass of a chunk (of the bins above the border's)
  u64* hist;       // [B][kBins] mass per bin; the last: of all the rest (null: no row can need it, nor the list)
  u64* list;       // [B][kList] logits of the border's bin: key << 32 | index
  int* listed;     // [B] how many
  float* peaks;    // [B][groups] largest logit of a group
  int64_t* out;
};

// a row's settings: loaded together, whichever of them are tensors (the others load their number's place holder)
struct Of {
  float t, p, m, u;
  int k;   // 0: off
};
template <typename T>
__device__ __forceinline__ Of row_of(const Args<T>& a, int b) {
  const float u = a.uniform[b];
  const float t = (a.temp.p ? a.temp.p : a.uniform)[b], p = (a.top_p.p ? a.top_p.p : a.uniform)[b];
  const float m = (a.min_p.p ? a.min_p.p : a.uniform)[b];
  const int k = (a.top_ks ? a.top_ks : reinterpret_cast<const int*>(a.uniform))[b];
  Of r;
  r.u = u;
  r.t = a.temp.p ? t : a.temp.v;
  r.p = a.top_p.p ? p : a.top_p.v;
  r.m = a.min_p.p ? m : a.min_p.v;
  r.k = a.top_ks ? k : a.top_k;
  if (r.k <= 0 || r.k >= a.V) r.k = 0;
  return r;
}
enum Kind { kGreedy, kPlain, kTopP, kShortK, kFromStart };
template <typename T>
__device__ __forceinline__ Kind kind_of(const Args<T>& a, const Of& r, float top) {
  if (!(r.t > 0.f) || top == -INFINITY) return kGreedy;
  if (top == INFINITY || !(r.u >= 9.094947e-13f) || r.u >= 1.f) return kFromStart;   // 2^-40
  if (r.k) return r.k <= a.groups / 2 && r.k <= kMaxK ? kShortK : kFromStart;
  return r.p < 1.f ? kTopP : kPlain;
}
// least mass that top-p keeps of z
__device__ __forceinline__ u64 share_of(float p, u64 z) {
  const u64 n = (u64)ceil(fmax((double)p, 0.0) * (double)z);
  return n < 1 ? (u64)1 : n > z ? z : n;
}

// p * r + c with c left in its registers: the compiler's choice, the two-operand form, copies c first, a third more
// instructions over the series below
__device__ __forceinline__ double horner(double p, double r, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(p), "v"(r), "v"(c));
  return d;
}

// 2^y as an integer of 2^-shift, y = (x - top) / (T ln 2) <= 0: y = k + r, |r| <= 1/2, 2^r by its series to r^10 (2e-13
// off; tables of 2^(j / 256) in LDS took longer: their random reads share one pipe).  Adding 1.5 * 2^52 leaves k in the
// low word of the sum.
struct Weigher {
  float top;
  double scale;      // 1 / (T ln 2)
  float bin_scale;   // bins per unit of x
  int shift;
  __device__ __forceinline__ u64 operator()(float x) const {
    const double y0 = ((double)x - (double)top) * scale, y = fmax(y0, -64.0);   // below: 2^(50 - 64) rounds to 0
    const double magic = 6755399441055744.0, t = y + magic;
    const int k = (int)(unsigned)__double_as_longlong(t);
    const double r = y - (t - magic);
    double p = 7.0549116208011e-09;              // (ln 2)^n / n!, n = 10 .. 0
    p = horner(p, r, 1.01780860092397e-07);
    p = horner(p, r, 1.32154867901443e-06);
    p = horner(p, r, 1.5252733804059840e-05);
    p = horner(p, r, 1.5403530393381608e-04);
    p = horner(p, r, 1.3333558146428443e-03);
    p = horner(p, r, 9.6181291076284772e-03);
    p = horner(p, r, 5.5504108664821580e-02);
    p = horner(p, r, 2.4022650695910071e-01);
    p = horner(p, r, 6.9314718055994531e-01);
    p = fma(p, r, 1.0);
    const double w = ldexp(p, k + shift);
    return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;   // w <= 2^50: rounded to an integer
  }
  // bin of a logit, not decreasing as x falls; the last one holds all the rest.  wide_bin: twice as wide, so that the
  // last one weighs nothing (2^-64); halves, whose difference does not pass the largest number
  __device__ __forceinline__ int bin(float x) const { return (int)fminf((top - x) * bin_scale, (float)(kBins - 1)); }
  __device__ __forceinline__ int wide_bin(float x) const {
    return (int)fminf((0.5f * top - 0.5f * x) * bin_scale, (float)(kBins - 1));
  }
};
__device__ __forceinline__ Weigher weigher(float top, float t, int shift) {
  Weigher w;
  w.top = top;
  w.scale = 1.4426950408889634 / (double)t;
  w.bin_scale = (float)fmin(w.scale * 64.0, 3e38);
  w.shift = shift;
  return w;
}
// least weight that min-p keeps
__device__ __forceinline__ u64 least_weight(float min_p, int shift) {
  if (!(min_p > 0.f)) return 0;
  return (u64)ceil(ldexp((double)fminf(min_p, 1.f), shift));
}

// grid (slices, B), 256 threads
template <typename T>
__global__ __launch_bounds__(256) void peaks_kernel(Args<T> a) {
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const T* row = a.logits + (long)b * a.stride;
  const int per = (a.chunks + gridDim.x - 1) / gridDim.x, c0 = blockIdx.x * per, c1 = min(a.chunks, c0 + per);
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  walk(row, a.V, c0 + wv, c1, 4, [](int) { return true; }, [&](int c, const float (&x)[8]) {
    float m = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, x[j]);
    // the last lane of a group gets its largest (groups of 4 lanes or of a row of 16)
    m = moved_max<0x111, 0xf>(m);
    m = moved_max<0x112, 0xf>(m);
    if (a.group_lanes == 16) {
      m = moved_max<0x114, 0xf>(m);
      m = moved_max<0x118, 0xf>(m);
    }
    const int g = (c * 64 + lane) / a.group_lanes;
    if ((lane & (a.group_lanes - 1)) == a.group_lanes - 1 && g < a.groups) a.peaks[(long)b * a.groups + g] = m;
  });
  if (!a.hist) return;   // (no row takes top-p alone)
  for (int i = blockIdx.x * 256 + threadIdx.x; i < kBins; i += gridDim.x * 256) a.hist[(long)b * kBins + i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.listed[b] = 0;
}

// the row's largest logit, from its groups', for every thread
template <int WAVES>
__device__ __forceinline__ float row_peak(const float* peaks, int groups, float* red) {
  float m = -INFINITY;
  for (int g = threadIdx.x; g < groups; g += WAVES * 64) m = fmaxf(m, peaks[g]);
  m = wave_peak(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) m = fmaxf(m, red[i]);
  return m;
}
// the largest logit of a chunk, by one lane
__device__ __forceinline__ float chunk_peak(const float* peaks, int c, int groups, int group_lanes) {
  const int n = 64 / group_lanes, g0 = c * n;
  float m = -INFINITY;
  for (int i = 0; i < n; i += 4)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, peaks[min(g0 + i + j, groups - 1)]);
  return m;
}

// sum of v over the workgroup, for every thread
template <int WAVES>
__device__ __forceinline__ u64 group_sum(u64 v, u64* red) {
  v = wave_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) s += red[i];
  return s;
}

// The first of n <= WAVES * 64 * PER entries (in LDS or global memory) at which the running sum passes want(total), the sum
// before it, and want, in found[0 .. 2]; the last entry where none does.  All threads take part.
template <int WAVES, int PER, typename Want>
__device__ __forceinline__ void group_find(const u64* v, int n, u64* red, u64* found, Want want_of) {
  const int per = (n + WAVES * 64 - 1) / (WAVES * 64), i0 = threadIdx.x * per;
  u64 x[PER], s = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    x[j] = j < per && i0 + j < n ? v[i0 + j] : 0;
    s += x[j];
  }
  const int wv = threadIdx.x >> 6;
  u64 cum = wave_scan64(s);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[wv] = cum;
  __syncthreads();
  u64 total = 0;
  cum -= s;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    cum += i < wv ? red[i] : 0;
    total += red[i];
  }
  const u64 want = want_of(total);
  if (want >= total ? threadIdx.x == 0 : cum <= want && want < cum + s) {
    int at = n - 1;
    u64 before = 0;
    bool open = want < total;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (open && cum + x[j] > want) {
        at = i0 + j;
        before = cum;
        open = false;
      }
      cum += x[j];
    }
    found[0] = at;
    found[1] = before;
    found[2] = want;
  }
  __syncthreads();
}

// grid (slices, B).  Wide workgroups: every one adds its bins to the row's in global memory
template <typename T>
__global__ __launch_bounds__(kWide * 64) void bins_kernel(Args<T> a) {
  __shared__ u64 hist[kBins], red[kWide];
  __shared__ float redf[kWide];
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const Of of = row_of(a, b);
  if (!(of.t > 0.f) || of.k) return;
  const float* peaks = a.peaks + (long)b * a.groups;
  if (of.p < 1.f)
    for (int i = tid; i < kBins; i += kWide * 64) hist[i] = 0;
  const float top = row_peak<kWide>(peaks, a.groups, redf);   // (its barrier also publishes hist)
  const Kind kind = kind_of(a, of, top);
  if (kind != kPlain && kind != kTopP) return;
  const Weigher weigh = weigher(top, of.t, a.shift);
  const u64 least = least_weight(of.m, a.shift);
  const T* row = a.logits + (long)b * a.stride;
  const int per = (a.chunks + gridDim.x - 1) / gridDim.x, c0 = blockIdx.x * per, c1 = min(a.chunks, c0 + per);
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  u64 tail = 0;
  // min-p: a logit below this weighs less than `least` (log2 of the weight off by 2^-10, the sums by their roundings)
  const float gap = (__log2f(fminf(fmaxf(of.m, 1e-37f), 1.f)) - 1e-3f) / (float)weigh.scale;
  const float low = top + gap - 1e-6f * (fabsf(top) + fabsf(gap));
  auto weighs = [&](int c) {   // (a chunk that does not: its mass is 0)
    const u64 most = weigh(chunk_peak(peaks, c, a.groups, a.group_lanes));
    const bool yes = most > 0 && (kind != kPlain || most >= least);
    if (!yes && kind == kPlain) a.mass[(long)b * a.chunks + c] = 0;
    return yes;
  };
  walk(row, a.V, c0 + wv, c1, kWide, weighs, [&](int c, const float (&x)[8]) {
    if (kind == kPlain) {
      u64 s = 0;
      if (of.m > 0.f) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (__any(x[j] >= low)) {   // (few chunks' logits are near the best: most weights need not be computed)
            const u64 w = weigh(x[j]);
            s += w >= least ? w : 0;
          }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) s += weigh(x[j]);
      }
      s = wave_sum64(s);
      if (lane == 0) a.mass[(long)b * a.chunks + c] = s;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = weigh.bin(x[j]);
        const u64 w = weigh(x[j]);
        if (n < kBins - 1) atomicAdd(&hist[n], w);
        else tail += w;
      }
    }
  });
  if (kind == kPlain) return;
  tail = group_sum<kWide>(tail, red);
  if (tid == 0) hist[kBins - 1] = tail;
  __syncthreads();
  for (int i = tid; i < kBins; i += kWide * 64)
    if (hist[i]) atomicAdd(&a.hist[(long)b * kBins + i], hist[i]);   // integers: any order gives the same sums
}

// The bin of the border of what top-p alone keeps of a row, and the mass it keeps of that bin; false: in the tail.
template <int WAVES>
__device__ __forceinline__ bool border_bin(const u64* hist, float p, u64* red, u64* found, int& bin, u64& left) {
  group_find<WAVES, kBins / 64 / WAVES>(hist, kBins, red, found, [&](u64 z) { return share_of(p, z) - 1; });
  bin = (int)found[0];
  left = found[2] + 1 - found[1];
  return bin < kBins - 1;
}

// grid (slices, B); rows of top-p alone
template <typename T>
__global__ __launch_bounds__(kWide * 64) void sweep_kernel(Args<T> a) {
  constexpr int kPart = 4096;
  __shared__ u64 red[kWide], found[3], list[kPart];
  __shared__ float redf[kWide];
  __shared__ int listed, place;
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const Of of = row_of(a, b);
  if (!(of.t > 0.f) || of.k || !(of.p < 1.f)) return;
  if (tid == 0) listed = 0;
  const float* peaks = a.peaks + (long)b * a.groups;
  const float top = row_peak<kWide>(peaks, a.groups, redf);
  if (kind_of(a, of, top) != kTopP) return;
  int bin;
  u64 left;
  if (!border_bin<kWide>(a.hist + (long)b * kBins, of.p, red, found, bin, left)) return;
  const Weigher weigh = weigher(top, of.t, a.shift);
  const u64 least = least_weight(of.m, a.shift);
  const T* row = a.logits + (long)b * a.stride;
  const int per = (a.chunks + gridDim.x - 1) / gridDim.x, c0 = blockIdx.x * per, c1 = min(a.chunks, c0 + per);
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto reaches = [&](int c) {
    const bool yes = weigh.bin(chunk_peak(peaks, c, a.groups, a.group_lanes)) <= bin;
    if (!yes) a.mass[(long)b * a.chunks + c] = 0;
    return yes;
  };
  walk(row, a.V, c0 + wv, c1, kWide, reaches, [&](int c, const float (&x)[8]) {
    u64 s = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = weigh.bin(x[j]);
      if (n < bin) {
        const u64 w = weigh(x[j]);
        s += w >= least ? w : 0;
      } else if (n == bin) {
        const int at = atomicAdd(&listed, 1);
        if (at < kPart) list[at] = ((u64)key_of(x[j]) << 32) | (unsigned)(c * kChunk + lane * 8 + j);
      }
    }
    s = wave_sum64(s);
    if (lane == 0) a.mass[(long)b * a.chunks + c] = s;
  });
  // this workgroup's part of the list, in one piece; too long a one makes the row's count too long as well
  __syncthreads();
  const int n = listed;
  if (n == 0) return;
  if (tid == 0) place = atomicAdd(&a.listed[b], n <= kPart ? n : kList + 1);
  __syncthreads();
  if (n > kPart) return;
  for (int i = tid; i < n; i += kWide * 64)
    if (place + i < kList) a.list[(long)b * kList + place + i] = list[i];
}

struct Shared {   // of choose_kernel
  u64 red[16], found[4], part[kMaxChunks], hist[kBins], list[kList], weight[kShort];
  int listed;
};

// ---- a row from the start, by radix selection
template <int kWaves, typename T>
__device__ __forceinline__ void choose_from_start(const Args<T>& a, const Of& of, int b, Shared& sh) {
  const int V = a.V;
  u64 *const red = sh.red, *const hist = sh.hist, *const part = sh.part, *const found = sh.found;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const T* row = a.logits + (long)b * a.stride;
  const int chunks = a.chunks;

  __syncthreads();   // (sh.red may still be read)
  // ---- the best token: largest value, lowest index
  u64 best = 0;
  for (int c = wv; c < chunks; c += kWaves) {
    float x[8];
    const int i = c * kChunk + lane * 8;
    load8(row, i, V, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u64 e = ((u64)key_of(x[j]) << 32) | (unsigned)~(i + j);
      if (i + j < V && e > best) best = e;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const u64 t = __shfl_xor(best, o, 64);
    best = t > best ? t : best;
  }
  if (lane == 0) red[wv] = best;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) best = red[i] > best ? red[i] : best;
  Row r;
  r.top = value_of((unsigned)(best >> 32));
  const float t = of.t;
  if (!(t > 0.f) || r.top == -INFINITY) {   // greedy; a row with no allowed token gives 0
    if (tid == 0) a.out[b] = (unsigned)~(unsigned)best;
    return;
  }
  r.inv_t = 1.0 / (double)t;
  r.unit = __longlong_as_double((long long)(1023 + a.shift) << 52);

  // ---- threshold: keys above `kmin` are kept, and the first `ties` of those that equal it
  unsigned kmin = 0;
  u64 ties = ~0ull;
  auto select = [&](bool mass, u64 need) {
    unsigned prefix = 0;
    for (int sh = 24; sh >= 0; sh -= 8) {
      __syncthreads();
      for (int i = tid; i < 256; i += kWaves * 64) hist[i] = 0;
      __syncthreads();
      const unsigned himask = sh == 24 ? 0u : ~0u << (sh + 8);
      for (int c = wv; c < chunks; c += kWaves) {
        float x[8];
        const int i = c * kChunk + lane * 8;
        load8(row, i, V, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned k = key_of(x[j]);
          if (i + j < V && (k & himask) == prefix && k >= kmin)
            atomicAdd(&hist[(k >> sh) & 255], mass ? fixed(r, weight(r, x[j])) : 1ull);
        }
      }
      __syncthreads();
      if (wv == 0) {   // from the top bin down: the first whose cumulative sum reaches `need`
        u64 h[4], s = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[j] = hist[255 - (lane * 4 + j)];
          s += h[j];
        }
        const u64 incl = wave_scan64(s);
        const u64 hit = __ballot(incl >= need);
        const int first = hit ? __ffsll((long long)hit) - 1 : 63;
        if (lane == first) {
          u64 cum = incl - s;
          int j = 0;
          while (j < 3 && cum + h[j] < need) cum += h[j++];
          found[0] = 255 - (lane * 4 + j);
          found[1] = need - cum;
        }
      }
      __syncthreads();
      prefix |= (unsigned)found[0] << sh;
      need = found[1];
    }
    kmin = prefix;
    return need;
  };
  // mass of what is kept so far (ties counted, not placed): for top-p's share
  auto kept_mass = [&]() {
    u64 s = 0, same = 0;
    for (int c = wv; c < chunks; c += kWaves) {
      float x[8];
      const int i = c * kChunk + lane * 8;
      load8(row, i, V, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned k = key_of(x[j]);
        if (i + j >= V || k < kmin) continue;
        if (k == kmin) ++same;
        else s += fixed(r, weight(r, x[j]));
      }
    }
    s = group_sum<kWaves>(s, red);
    same = group_sum<kWaves>(same, red);
    if (same > ties) same = ties;
    return s + (same ? same * fixed(r, weight(r, value_of(kmin))) : 0);
  };
  const int k = of.k;
  if (k) ties = select(false, (u64)k);
  const float p = of.p;
  if (p < 1.f) {
    const u64 z = kept_mass();
    u64 need = (u64)ceil(fmax((double)p, 0.0) * (double)z);
    if (need < 1) need = 1;
    if (need > z) need = z;
    const u64 left = select(true, need), one = fixed(r, weight(r, value_of(kmin)));
    ties = one ? (left + one - 1) / one : 1;
  }
  // ---- ties in index order: the last index kept among the keys equal to kmin
  int last_tie = V;
  if (ties != ~0ull) {
    __syncthreads();
    for (int c = wv; c < chunks; c += kWaves) {
      float x[8];
      const int i = c * kChunk + lane * 8;
      load8(row, i, V, x);
      u64 same = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) same += i + j < V && key_of(x[j]) == kmin;
      same = wave_sum64(same);
      if (lane == 0) part[c] = same;
    }
    __syncthreads();
    // the chunk that holds tie number `ties` (counted from 1), then the element
    group_find<kWaves, kMaxChunks / 64 / kWaves>(part, chunks, red, found, [&](u64) { return ties - 1; });
    const int at = (int)found[0];
    const u64 before = found[1];
    __syncthreads();
    if (wv == 0) {
      if (lane == 0) found[0] = V;
      {
        float x[8];
        const int i = at * kChunk + lane * 8;
        load8(row, i, V, x);
        u64 same = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) same += i + j < V && key_of(x[j]) == kmin;
        u64 n = before + wave_scan64(same) - same;
        if (n < ties && n + same >= ties) {
          int at_j = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (i + j < V && key_of(x[j]) == kmin && ++n == ties) at_j = i + j;
          found[0] = at_j;
        }
      }
    }
    __syncthreads();
    last_tie = (int)found[0];
    __syncthreads();
  }
  // ---- kept mass per chunk, then the chunk, lane and element where the cumulative mass passes u * total
  // The number 0 draws the first kept token of any weight above 0, one from 1 on the last, also where that is below the
  // integers' unit: they are counted.  One between 0 and 2^-40 is compared in integers of 2^(1 - shift) of u * total; a weight
  // above u * total, which passes it alone, counts as the next number.
  const float mp = of.m, uf = of.u;
  const bool last_kept = uf >= 1.f, counted = last_kept || !(uf > 0.f), small = !counted && uf < 9.094947e-13f;
  const u64 at_target = 1ull << (a.shift - 1);
  double finer = 0.0;
  auto kept = [&](float x, int i) -> u64 {
    const unsigned ky = key_of(x);
    if (i >= V || ky < kmin || (ky == kmin && i > last_tie)) return 0;
    const double w = weight(r, x);
    if (!(w >= (double)mp || x == r.top || !(mp == mp))) return 0;
    if (finer > 0.0) return (u64)fmin(w * finer + 0.5, (double)(at_target + 1));
    return counted ? (u64)(w > 0.0) : fixed(r, w);
  };
  auto masses = [&]() {
    u64 mine = 0;
    for (int c = wv; c < chunks; c += kWaves) {
      float x[8];
      const int i = c * kChunk + lane * 8;
      load8(row, i, V, x);
      u64 s = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += kept(x[j], i + j);
      s = wave_sum64(s);
      if (lane == 0) part[c] = s;
      mine += lane == 0 ? s : 0;
    }
    return group_sum<kWaves>(mine, red);
  };
  u64 total = masses(), want = counted ? 0 : (u64)fmin((double)uf * (double)total, 9.0e18);
  if (small) {
    finer = (double)at_target * r.unit / ((double)uf * (double)total);
    total = masses();
    want = at_target;
  }
  if (last_kept || want >= total) want = total - 1;
  group_find<kWaves, kMaxChunks / 64 / kWaves>(part, chunks, red, found, [&](u64) { return want; });
  if (wv == 0) {
    const int at = (int)found[0];
    const u64 before = found[1];
    float x[8];
    const int i = at * kChunk + lane * 8;
    load8(row, i, V, x);
    u64 w[8], s = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = kept(x[j], i + j);
      s += w[j];
    }
    u64 cum = before + wave_scan64(s) - s;
    if (cum <= want && want < cum + s) {
      int token = i;
      bool open = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cum += w[j];
        if (open && cum > want) {
          token = i + j;
          open = false;
        }
      }
      a.out[b] = token;
    }
  }
}

// Where the border lies among n <= kList listed logits (key << 32 | index, in any order; LDS): the entry at which those
// before it in the order (larger key, then smaller index) hold less than `left` of the mass, and with it `left` or more.
// The entries before it go to `keep(entry, weight)`.  The list is used up.
template <int kWaves, typename Keep>
__device__ __forceinline__ u64 resolve(Shared& sh, int n, u64 left, const Weigher& weigh, Keep keep) {
  constexpr u64 kFlip = 0xffffffffull;   // index reversed: the order is then that of falling numbers
  constexpr int kThreads = kWaves * 64;
  const int tid = threadIdx.x;
  while (n > 256) {   // narrow down by the highest ten bits that differ
    u64 lo = ~0ull, hi = 0, e[kList / kThreads];
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) {
      const int at = tid + i * kThreads;
      e[i] = at < n ? sh.list[at] ^ kFlip : 0;
      if (at < n) {
        lo = e[i] < lo ? e[i] : lo;
        hi = e[i] > hi ? e[i] : hi;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const u64 l = __shfl_xor(lo, o, 64), h = __shfl_xor(hi, o, 64);
      lo = l < lo ? l : lo;
      hi = h > hi ? h : hi;
    }
    __syncthreads();
    if ((tid & 63) == 0) {
      sh.red[tid >> 6] = lo;
      sh.hist[1024 + (tid >> 6)] = hi;
    }
    for (int i = tid; i < 1024; i += kThreads) sh.hist[i] = 0;
    if (tid == 0) sh.listed = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      lo = sh.red[i] < lo ? sh.red[i] : lo;
      hi = sh.hist[1024 + i] > hi ? sh.hist[1024 + i] : hi;
    }
    const int bits = 64 - __clzll((long long)(lo ^ hi)), cut = bits > 10 ? bits - 10 : 0;
    u64 w[kList / kThreads];
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) {
      w[i] = 0;
      if (tid + i * kThreads < n) {
        w[i] = weigh(value_of((unsigned)(e[i] >> 32)));
        atomicAdd(&sh.hist[1023 - (int)((e[i] >> cut) & 1023)], w[i]);
      }
    }
    __syncthreads();
    group_find<kWaves, 1024 / 64 / kWaves>(sh.hist, 1024, sh.red, sh.found, [&](u64) { return left - 1; });
    const int digit = 1023 - (int)sh.found[0];
    left -= sh.found[1];
#pragma unroll
    for (int i = 0; i < kList / kThreads; ++i) {
      if (tid + i * kThreads >= n) continue;
      const int d = (int)((e[i] >> cut) & 1023);
      if (d > digit) keep(e[i] ^ kFlip, w[i]);
      if (d == digit) sh.list[atomicAdd(&sh.listed, 1)] = e[i] ^ kFlip;
    }
    __syncthreads();
    n = sh.listed;
    __syncthreads();
  }
  if (tid < n) sh.weight[tid] = weigh(value_of((unsigned)(sh.list[tid] >> 32)));
  __syncthreads();
  if (tid < n) {
    const u64 mine = sh.list[tid], w = sh.weight[tid];
    u64 before = 0;
    for (int i = 0; i < n; ++i) before += (sh.list[i] ^ kFlip) > (mine ^ kFlip) ? sh.weight[i] : 0;
    if (before < left) {
      if (before + w >= left) sh.found[3] = mine;
      else keep(mine, w);
    }
  }
  __syncthreads();
  return sh.found[3];
}

// v[0 .. kShort) becomes its inclusive prefix sums (the caller's barrier before it, its own after it)
template <int WAVES>
__device__ __forceinline__ void group_scan(u64* v, u64* red) {
  constexpr int PER = kShort / (WAVES * 64);
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  u64 x[PER], sum = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) sum += x[j] = v[threadIdx.x * PER + j];
  u64 run = wave_scan64(sum);
  if (lane == 63) red[wv] = run;
  __syncthreads();
  run -= sum;
  for (int i = 0; i < wv; ++i) run += red[i];
#pragma unroll
  for (int j = 0; j < PER; ++j) v[threadIdx.x * PER + j] = run += x[j];
  __syncthreads();
}

// a row whose sums or peaks the other kernels have prepared; false: it has to be taken from the start
template <int kWaves, typename T>
__device__ __forceinline__ bool choose_by_mass(const Args<T>& a, const Of& of, int b, Shared& sh, float top, Kind kind) {
  constexpr int kThreads = kWaves * 64;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, V = a.V, chunks = a.chunks;
  const T* row = a.logits + (long)b * a.stride;
  const float* peaks = a.peaks + (long)b * a.groups;
  const Weigher weigh = weigher(top, of.t, a.shift);
  const u64 least = least_weight(of.m, a.shift);
  auto target = [&](u64 total) {
    const u64 want = (u64)fmin((double)of.u * (double)total, 9.0e18);
    return want >= total ? total - 1 : want;
  };
  if (kind == kShortK) {
    // the bound: the first bin at which k groups have their largest logit (or all that weighs anything)
    for (int i = tid; i < kBins; i += kThreads) sh.hist[i] = 0;
    __syncthreads();
    for (int g = tid; g < a.groups; g += kThreads) atomicAdd(&sh.hist[weigh.wide_bin(peaks[g])], 1ull);
    __syncthreads();
    group_find<kWaves, kBins / 64 / kWaves>(sh.hist, kBins, sh.red, sh.found, [&](u64) { return (u64)of.k - 1; });
    const int bound = min((int)sh.found[0], kBins - 2);
    // the groups at or above it, then their logits at or above it; group_lanes lanes take a group
    int* groups = reinterpret_cast<int*>(sh.hist);
    __syncthreads();
    for (int g = tid; g < a.groups; g += kThreads)
      if (weigh.wide_bin(peaks[g]) <= bound) {
        const int at = atomicAdd(&sh.listed, 1);
        if (at < 2 * kBins) groups[at] = g;
      }
    __syncthreads();
    const int n_groups = sh.listed;
    __syncthreads();
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    const bool ok = n_groups <= 2 * kBins;
    for (int at = tid / a.group_lanes; ok && at < n_groups; at += kThreads / a.group_lanes) {
      float x[8];
      const int i = (groups[at] * a.group_lanes + (tid & (a.group_lanes - 1))) * 8;
      load8(row, i, V, x);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j < V && weigh.wide_bin(x[j]) <= bound) {
          const int to = atomicAdd(&sh.listed, 1);
          if (to < kShort) sh.list[to] = ((u64)key_of(x[j]) << 32) | (unsigned)(i + j);
        }
    }
    __syncthreads();
    const int n = sh.listed;
    if (!ok || n > kShort) {
      __syncthreads();
      return false;
    }
    // Ranks by counting, all against all, `parts` threads to an entry where there are fewer entries than threads; masses by
    // prefix sums of the weights in that order: by logit for what top-k and top-p keep, then by index for the token
    constexpr u64 kFlip = 0xffffffffull;   // (the lower index first, as the larger logit)
    u64 *const upto = sh.part, *const weight = sh.weight;
    int *const rank = reinterpret_cast<int*>(sh.hist), *const place = rank + kShort;
    int step = 64;
    while (step < n && step < kThreads) step *= 2;
    const int part = tid / step, parts = kThreads / step, first = tid & (step - 1);
    const int per = (n + parts - 1) / parts, i0 = part * per, i1 = min(n, i0 + per);
    __syncthreads();
    for (int at = tid; at < kShort; at += kThreads) {
      if (at < n) {
        sh.list[at] ^= kFlip;
        weight[at] = weigh(value_of((unsigned)(sh.list[at] >> 32)));
      }
      upto[at] = 0, rank[at] = 0, place[at] = 0;
    }
    __syncthreads();
    for (int at = first; at < n; at += step) {
      const u64 mine = sh.list[at];
      int ahead = 0, left = 0;
#pragma unroll 8
      for (int i = i0; i < i1; ++i) {
        const u64 other = sh.list[i];
        ahead += other > mine;
        left += (unsigned)other > (unsigned)mine;
      }
      if (parts == 1) rank[at] = ahead, place[at] = left;
      else atomicAdd(&rank[at], ahead), atomicAdd(&place[at], left);
    }
    __syncthreads();
    for (int at = tid; at < n; at += kThreads) upto[rank[at]] = weight[at];
    __syncthreads();
    group_scan<kWaves>(upto, sh.red);
    const u64 share = of.p < 1.f ? share_of(of.p, upto[min(of.k, n) - 1]) : ~0ull;
    for (int at = tid; at < n; at += kThreads) {
      const bool kept = rank[at] < of.k && upto[rank[at]] - weight[at] < share && weight[at] >= least;
      if (!kept) weight[at] = 0;
    }
    __syncthreads();
    for (int at = tid; at < n; at += kThreads) upto[place[at]] = weight[at];
    __syncthreads();
    group_scan<kWaves>(upto, sh.red);
    const u64 want = target(upto[n - 1]);
    for (int at = tid; at < n; at += kThreads) {
      const u64 end = upto[place[at]];
      if (weight[at] && end - weight[at] <= want && want < end) a.out[b] = (int64_t)(unsigned)~(unsigned)sh.list[at];
    }
    return true;
  }
  // a logit is kept when its key is above kmin, or equals it at an index up to last, and its weight is `least` or more
  unsigned kmin = 0;
  int last = V;
  for (int c = tid; c < chunks; c += kThreads) sh.part[c] = a.mass[(long)b * chunks + c];
  if (kind == kTopP) {
    int bin = 0;
    u64 left = 0;
    const int n = a.listed[b];
    if (!border_bin<kWaves>(a.hist + (long)b * kBins, of.p, sh.red, sh.found, bin, left) || n > kList) {
      return false;
    }
    for (int i = tid; i < n; i += kThreads) sh.list[i] = a.list[(long)b * kList + i];
    __syncthreads();
    auto keep = [&](u64 e, u64 w) {
      if (w >= least) atomicAdd(&sh.part[(unsigned)e / kChunk], w);
    };
    const u64 edge = resolve<kWaves>(sh, n, left, weigh, keep);
    kmin = (unsigned)(edge >> 32);
    last = (int)(unsigned)edge;
    if (tid == 0) keep(edge, weigh(value_of(kmin)));
  }
  __syncthreads();
  group_find<kWaves, kMaxChunks / 64 / kWaves>(sh.part, chunks, sh.red, sh.found, target);
  const u64 want = sh.found[2];
  if (wv == 0) {
    float x[8];
    const int i = (int)sh.found[0] * kChunk + lane * 8;
    load8(row, i, V, x);
    u64 w[8], s = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned k = key_of(x[j]);
      w[j] = k < kmin || (k == kmin && i + j > last) ? 0 : weigh(x[j]);
      w[j] = w[j] >= least ? w[j] : 0;
      s += w[j];
    }
    u64 cum = sh.found[1] + wave_scan64(s) - s;
    if (cum <= want && want < cum + s) {
      int token = i;
      bool open = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        cum += w[j];
        if (open && cum > want) {
          token = i + j;
          open = false;
        }
      }
      a.out[b] = token;
    }
  }
  return true;
}

// grid B, one row each
template <typename T, int kWaves>
__global__ __launch_bounds__(kWaves * 64) void choose_kernel(Args<T> a) {
  constexpr int kThreads = kWaves * 64;
  __shared__ Shared sh;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, V = a.V;
  const T* row = a.logits + (long)b * a.stride;
  const float* peaks = a.peaks + (long)b * a.groups;
  const Of of = row_of(a, b);
  if (tid == 0) sh.listed = 0;
  const float top = row_peak<kWaves>(peaks, a.groups, reinterpret_cast<float*>(sh.red));
  const Kind kind = kind_of(a, of, top);
  if (kind == kGreedy) {   // the lowest index of the largest logit; 0 where no token is allowed
    int g = a.groups;
    for (int i = tid; i < a.groups; i += kThreads)
      if (peaks[i] == top) {
        g = i;
        break;
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) g = min(g, __shfl_xor(g, o, 64));
    if (lane == 0) sh.part[wv] = g;
    __syncthreads();
    if (wv == 0) {
      g = lane < kWaves ? (int)sh.part[lane] : a.groups;
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) g = min(g, __shfl_xor(g, o, 64));
      float x[8];
      const int i = g * a.group_lanes * 8 + (lane & (a.group_lanes - 1)) * 8;
      load8(row, i, V, x);
      int first = 8;
#pragma unroll
      for (int j = 7; j >= 0; --j) first = x[j] == top ? j : first;
      const u64 hit = __ballot(first < 8 && lane < a.group_lanes);
      if (lane == (hit ? __ffsll((long long)hit) - 1 : 0)) a.out[b] = hit && top > -INFINITY ? i + first : 0;
    }
    return;
  }
  // (one call of choose_from_start, which is inlined then: as a function it had the arguments in scratch memory)
  if (kind == kFromStart || !choose_by_mass<kWaves>(a, of, b, sh, top, kind)) choose_from_start<kWaves>(a, of, b, sh);
}

}  // namespace smp
}  // namespace pd

using namespace pd;

// logits per group: small ones allow a larger top-k (half the groups), large ones keep the list of their peaks short
static int sample_group(int V) { return V <= 65536 ? 32 : 128; }

// What some row may need, of a call's settings: tensors (rows), or numbers
struct Needs {
  bool warm, always_k, p;   // a temperature; top-k in every row; top-p alone
};
static Needs sample_needs(int V, bool temp_rows, float temp, bool k_rows, int top_k, bool p_rows, float top_p) {
  Needs n;
  n.warm = temp_rows || temp > 0.f;
  n.always_k = !k_rows && top_k > 0 && top_k < V;
  n.p = n.warm && !n.always_k && (p_rows || top_p < 1.f);
  return n;
}

// bytes of scratch for B rows of V logits: 82 KB a row with top-p alone, else a hundredth to a tenth of the logits
extern "C" long pd_sample_workspace(int B, int V, int temp_rows, float temp, int k_rows, int top_k, int p_rows, float top_p) {
  const long chunks = (V + smp::kChunk - 1) / smp::kChunk, per = sample_group(V), groups = (V + per - 1) / per;
  const bool p = sample_needs(V, temp_rows, temp, k_rows, top_k, p_rows, top_p).p;
  return (long)B * (8 * (chunks + (p ? smp::kBins + smp::kList : 0)) + 4 * (groups + 1));
}

extern "C" int pd_sample(int dt, const void* logits, long stride, int B, int V, const float* uniform, const float* temps,
                         float temp, const int* top_ks, int top_k, const float* top_ps, float top_p, const float* min_ps,
                         float min_p, int64_t* out, void* workspace, void* stream) {
  if (B <= 0) return 0;
  if (V < 1 || V > smp::kChunk * smp::kMaxChunks || B > 65535 || !workspace) return -1;
  int bits = 0;
  while ((1L << bits) < V) ++bits;
  const int shift = 62 - bits < 50 ? 62 - bits : 50;   // V weights of at most 2^shift stay under 2^62
  const int chunks = (V + smp::kChunk - 1) / smp::kChunk, per = sample_group(V), groups = (V + per - 1) / per;
  // workgroups per row: a chunk a wave, but about two thousand narrow (four waves) or a thousand wide ones in all
  auto slices_of = [&](int waves, int all) {
    const int most = (chunks + waves - 1) / waves, enough = (all + B - 1) / B;
    return most < enough ? most : enough;
  };
  const dim3 narrow(slices_of(4, 2048), B), wide(slices_of(smp::kWide, 1024), B);
  hipStream_t st = (hipStream_t)stream;
  // kernels that no row can need are not launched: the settings that are numbers say so
  const Needs needs = sample_needs(V, temps, temp, top_ks, top_k, top_ps, top_p);
  smp::u64* const mass = (smp::u64*)workspace;
  smp::u64* const hist = needs.p ? mass + (long)B * chunks : nullptr;
  smp::u64* const list = needs.p ? hist + (long)B * smp::kBins : nullptr;
  int* const listed = (int*)(needs.p ? list + (long)B * smp::kList : mass + (long)B * chunks);
  float* const peaks = (float*)(listed + B);
  PD_DISPATCH_FLOAT(dt, T, {
    const smp::Args<T> a{(const T*)logits, stride, V, chunks, groups, per / 8, shift, uniform, {temps, temp}, {top_ps, top_p},
                         {min_ps, min_p}, top_ks, top_k, mass, hist, list, listed, peaks, out};
    smp::peaks_kernel<T><<<narrow, 256, 0, st>>>(a);
    if (needs.warm && !needs.always_k) smp::bins_kernel<T><<<wide, smp::kWide * 64, 0, st>>>(a);
    if (needs.p) smp::sweep_kernel<T><<<wide, smp::kWide * 64, 0, st>>>(a);
    if (V <= 65536) smp::choose_kernel<T, 8><<<B, 512, 0, st>>>(a);
    else smp::choose_kernel<T, 16><<<B, 1024, 0, st>>>(a);
  });
  return (int)hipGetLastError();
}
