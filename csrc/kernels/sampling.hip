// One token per row of logits, from a given random number: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T)                     weights; x ordered by (value descending, index ascending)
//   top-k: the first k of that order;  top-p: of what is left, the shortest head whose mass reaches p of it;
//   min-p: of what is left, w_i >= min_p (w of the best is 1);
//   token = the first index, in index order, whose cumulative kept mass exceeds u * (kept mass).
//
// A choice next to a border turns on the last bits of these sums, so weights are computed in 64 bits and summed as
// integers of 2^-shift (shift = 62 - bits of V): integer sums do not depend on the order they are taken in, so a row's
// token is the same in every launch.  No sort.  Four launches; a row is cut into chunks of 512 logits (a wave's load)
// and groups of 128:
//   peaks_kernel   every group's largest logit;
//   bins_kernel    knows the row's largest.  Without top-k and top-p: the kept mass of every chunk.  Top-p alone: masses
//                  over 2,047 bins of 1/64 in log2 of the weight, and of the tail behind them;
//   sweep_kernel   top-p alone: finds the bin of the border, sums what lies above it per chunk, lists what lies in it;
//   choose_kernel  one workgroup per row: the border's place in the list, the chunk, the token.  Top-k (up to half the
//                  groups and 512) is done here alone: the k-th best group's largest logit bounds the k-th best logit from
//                  below, so some k groups are read, and the few logits above the bound are ranked all against all.
// Rows that fit none of this (a larger k, an infinite logit, a border in the tail or with more than 8,192 logits in its
// bin, a number below 2^-40) are taken from the start in choose_kernel: radix selection on the ordered bits of the logits.
#include "common.h"

namespace pd {
namespace smp {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWaves = kThreads / 64, kChunk = 512, kMaxChunks = 2048;   // V <= 2^20
constexpr int kGroup = 128, kBins = 2048, kList = 8192, kShort = 1024, kMaxK = 512, kTable = 256;

// bits that order as the values do; NaN as -inf, -0 as +0
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// inclusive prefix over the lanes
__device__ __forceinline__ u64 wave_scan64(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 t = __shfl_up(v, o, 64);
    if (lane >= o) v += t;
  }
  return v;
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

struct Setting {
  const float* p;   // one value per row, or null
  float v;
  __device__ __forceinline__ float of(int b) const { return p ? p[b] : v; }
};

// Everything a launch needs; settings per row (pointers) or for all rows.
template <typename T>
struct Args {
  const T* logits;
  long stride;
  int V, chunks, groups, shift;
  const float* uniform;
  Setting temp, top_p, min_p;
  const int* top_ks;
  int top_k;
  u64* mass;       // [B][chunks] kept mass of a chunk (of the bins above the border's)
  u64* hist;       // [B][kBins] mass per bin; the last: of all the rest
  u64* list;       // [B][kList] logits of the border's bin: key << 32 | index
  int* listed;     // [B] how many
  float* peaks;    // [B][groups] largest logit of a group
  int64_t* out;
  __device__ __forceinline__ int k_of(int b) const {   // 0: off
    const int k = top_ks ? top_ks[b] : top_k;
    return k > 0 && k < V ? k : 0;
  }
};
enum Kind { kGreedy, kPlain, kTopP, kShortK, kFromStart };
template <typename T>
__device__ __forceinline__ Kind kind_of(const Args<T>& a, int b, float top) {
  if (!(a.temp.of(b) > 0.f) || top == -INFINITY) return kGreedy;
  if (top == INFINITY || !(a.uniform[b] >= 9.094947e-13f)) return kFromStart;   // 2^-40
  const int k = a.k_of(b);
  if (k) return k <= a.groups / 2 && k <= kMaxK ? kShortK : kFromStart;
  return a.top_p.of(b) < 1.f ? kTopP : kPlain;
}
// least mass that top-p keeps of z
__device__ __forceinline__ u64 share_of(float p, u64 z) {
  const u64 n = (u64)ceil(fmax((double)p, 0.0) * (double)z);
  return n < 1 ? (u64)1 : n > z ? z : n;
}

// 2^y as an integer of 2^-shift, y = (x - top) / (T ln 2) <= 0: y = k / 256 + r, 2^(k / 256) from a table of 2^(j / 256),
// 2^r by its series to r^4 (|r| <= 2^-9: 4e-17 off).  Adding 1.5 * 2^44 leaves k in the low word of the sum.
struct Weigher {
  float top;
  double scale;         // 1 / (T ln 2)
  float bin_scale;      // bins per unit of x
  int shift;
  const double* table;  // 2^(j / 256) in LDS
  __device__ __forceinline__ u64 operator()(float x) const {
    const double y = ((double)x - (double)top) * scale;
    if (!(y > -(double)(shift + 2))) return 0;   // also -inf
    const double magic = 26388279066624.0, t = y + magic;
    const int k = (int)(unsigned)__double_as_longlong(t);
    const double r = y - (t - magic);
    const double p = fma(fma(fma(fma(0.009618129107628477, r, 0.055504108664821580), r, 0.24022650695910072), r,
                             0.69314718055994531), r, 1.0);
    const double w = ldexp(p * table[k & (kTable - 1)], (k >> 8) + shift);
    return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;   // w <= 2^50: rounded to an integer
  }
  // bin of a logit, not decreasing as x falls; the last one holds all the rest.  wide_bin: twice as wide, so that the
  // last one weighs nothing (2^-64)
  __device__ __forceinline__ int bin(float x) const { return (int)fminf((top - x) * bin_scale, (float)(kBins - 1)); }
  __device__ __forceinline__ int wide_bin(float x) const {
    return (int)fminf((top - x) * bin_scale * 0.5f, (float)(kBins - 1));
  }
};
__device__ __forceinline__ void fill_table(double* table) {
  for (int j = threadIdx.x; j < kTable; j += blockDim.x) table[j] = exp2((double)j / kTable);
}
__device__ __forceinline__ Weigher weigher(float top, float t, int shift, const double* table) {
  Weigher w;
  w.top = top;
  w.scale = 1.4426950408889634 / (double)t;
  w.bin_scale = (float)fmin(w.scale * 64.0, 3e38);
  w.shift = shift;
  w.table = table;
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
  for (int c = c0 + (threadIdx.x >> 6); c < c1; c += 4) {
    float x[8];
    load8(row, c * kChunk + lane * 8, a.V, x);
    float m = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, x[j]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const int g = c * (kChunk / kGroup) + (lane >> 4);
    if ((lane & 15) == 0 && g < a.groups) a.peaks[(long)b * a.groups + g] = m;
  }
  for (int i = blockIdx.x * 256 + threadIdx.x; i < kBins; i += gridDim.x * 256) a.hist[(long)b * kBins + i] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.listed[b] = 0;
}

// the row's largest logit, from its groups', for every thread
__device__ __forceinline__ float row_peak(const float* peaks, int groups, float* red) {
  float m = -INFINITY;
  for (int g = threadIdx.x; g < groups; g += blockDim.x) m = fmaxf(m, peaks[g]);
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = red[0];
  for (int i = 1; i < (int)blockDim.x / 64; ++i) m = fmaxf(m, red[i]);
  return m;
}
__device__ __forceinline__ float chunk_peak(const float* peaks, int c, int groups) {
  float m = -INFINITY;
#pragma unroll
  for (int g = 0; g < kChunk / kGroup; ++g) m = fmaxf(m, peaks[min(c * (kChunk / kGroup) + g, groups - 1)]);
  return m;
}

// sum of v over the workgroup, for every thread; WAVES of it
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

// The first of n <= WAVES * 64 * 8 entries (in LDS, or global memory) at which the running sum passes `want`, and the sum
// before it, in found[0], found[1]; the last entry where none does.  All threads take part.
template <int WAVES>
__device__ __forceinline__ void group_find(const u64* v, int n, u64 want, u64* red, u64* found) {
  const int per = (n + WAVES * 64 - 1) / (WAVES * 64), i0 = threadIdx.x * per;
  u64 x[8], s = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = j < per && i0 + j < n ? v[i0 + j] : 0;
    s += x[j];
  }
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  u64 cum = wave_scan64(s, lane);
  __syncthreads();
  if (lane == 63) red[wv] = cum;
  if (threadIdx.x == 0) {
    found[0] = n - 1;
    found[1] = 0;
  }
  __syncthreads();
  cum -= s;
  for (int i = 0; i < wv; ++i) cum += red[i];
  if (cum <= want && want < cum + s) {
    int at = -1;
    u64 before = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (at < 0 && cum + x[j] > want) {
        at = i0 + j;
        before = cum;
      }
      cum += x[j];
    }
    found[0] = at;
    found[1] = before;
  }
  __syncthreads();
}

// grid (slices, B), 256 threads
template <typename T>
__global__ __launch_bounds__(256) void bins_kernel(Args<T> a) {
  __shared__ u64 hist[kBins], red[4];
  __shared__ double table[kTable];
  __shared__ float redf[4];
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  if (!(a.temp.of(b) > 0.f) || a.k_of(b)) return;
  const float* peaks = a.peaks + (long)b * a.groups;
  fill_table(table);
  for (int i = tid; i < kBins; i += 256) hist[i] = 0;
  const float top = row_peak(peaks, a.groups, redf);   // (its barrier also publishes hist and table)
  const Kind kind = kind_of(a, b, top);
  if (kind != kPlain && kind != kTopP) return;
  const Weigher weigh = weigher(top, a.temp.of(b), a.shift, table);
  const u64 least = least_weight(a.min_p.of(b), a.shift);
  const T* row = a.logits + (long)b * a.stride;
  const int per = (a.chunks + gridDim.x - 1) / gridDim.x, c0 = blockIdx.x * per, c1 = min(a.chunks, c0 + per);
  u64 tail = 0;
  for (int c = c0 + (tid >> 6); c < c1; c += 4) {
    const u64 most = weigh(chunk_peak(peaks, c, a.groups));
    float x[8];
    if (kind == kPlain) {
      u64 s = 0;
      if (most > 0 && most >= least) {
        load8(row, c * kChunk + lane * 8, a.V, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const u64 w = weigh(x[j]);
          s += w >= least ? w : 0;
        }
        s = wave_sum64(s);
      }
      if (lane == 0) a.mass[(long)b * a.chunks + c] = s;
    } else if (most > 0) {
      load8(row, c * kChunk + lane * 8, a.V, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = weigh.bin(x[j]);
        const u64 w = weigh(x[j]);
        if (n < kBins - 1) atomicAdd(&hist[n], w);
        else tail += w;
      }
    }
  }
  if (kind == kPlain) return;
  tail = group_sum<4>(tail, red);
  if (tid == 0) hist[kBins - 1] = tail;
  __syncthreads();
  for (int i = tid; i < kBins; i += 256)
    if (hist[i]) atomicAdd(&a.hist[(long)b * kBins + i], hist[i]);   // integers: any order gives the same sums
}

// What top-p alone keeps of a row: its share of the mass, the border's bin and the mass before it; false: the tail.
template <int WAVES>
__device__ __forceinline__ bool border_bin(const u64* hist, float p, u64* red, u64* found, int& bin, u64& left) {
  u64 z = 0;
  for (int i = threadIdx.x; i < kBins; i += WAVES * 64) z += hist[i];
  const u64 need = share_of(p, group_sum<WAVES>(z, red));
  group_find<WAVES>(hist, kBins, need - 1, red, found);
  bin = (int)found[0];
  left = need - found[1];
  __syncthreads();
  return bin < kBins - 1;
}

// grid (slices, B), 256 threads; rows of top-p alone
template <typename T>
__global__ __launch_bounds__(256) void sweep_kernel(Args<T> a) {
  __shared__ u64 red[4], found[2];
  __shared__ double table[kTable];
  __shared__ float redf[4];
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  if (!(a.temp.of(b) > 0.f) || a.k_of(b) || !(a.top_p.of(b) < 1.f)) return;
  const float* peaks = a.peaks + (long)b * a.groups;
  fill_table(table);
  const float top = row_peak(peaks, a.groups, redf);
  if (kind_of(a, b, top) != kTopP) return;
  int bin;
  u64 left;
  if (!border_bin<4>(a.hist + (long)b * kBins, a.top_p.of(b), red, found, bin, left)) return;
  const Weigher weigh = weigher(top, a.temp.of(b), a.shift, table);
  const u64 least = least_weight(a.min_p.of(b), a.shift);
  const T* row = a.logits + (long)b * a.stride;
  const int per = (a.chunks + gridDim.x - 1) / gridDim.x, c0 = blockIdx.x * per, c1 = min(a.chunks, c0 + per);
  for (int c = c0 + (tid >> 6); c < c1; c += 4) {
    u64 s = 0;
    if (weigh.bin(chunk_peak(peaks, c, a.groups)) <= bin) {
      float x[8];
      const int i = c * kChunk + lane * 8;
      load8(row, i, a.V, x);
      int mine = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int n = weigh.bin(x[j]);
        if (n < bin) {
          const u64 w = weigh(x[j]);
          s += w >= least ? w : 0;
        }
        mine += n == bin;
      }
      s = wave_sum64(s);
      if (__any(mine)) {   // room in the list for the whole wave at once
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int t = __shfl_up(upto, o, 64);
          if (lane >= o) upto += t;
        }
        int at = 0;
        if (lane == 63) at = atomicAdd(&a.listed[b], upto);
        at = __shfl(at, 63, 64) + upto - mine;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (weigh.bin(x[j]) == bin) {
            if (at < kList) a.list[(long)b * kList + at] = ((u64)key_of(x[j]) << 32) | (unsigned)(i + j);
            ++at;
          }
      }
    }
    if (lane == 0) a.mass[(long)b * a.chunks + c] = s;
  }
}

struct Shared {   // of choose_kernel
  u64 red[kWaves], found[4], part[kMaxChunks], hist[kBins], list[kList], weight[kShort];
  double table[kTable];
  int listed;
};

// ---- a row from the start, by radix selection
template <typename T>
__device__ void choose_from_start(const Args<T>& a, int b, Shared& sh) {
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
  const float t = a.temp.of(b);
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
      if (tid < 256) hist[tid] = 0;
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
        const u64 incl = wave_scan64(s, lane);
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
  const int k = a.k_of(b);
  if (k) ties = select(false, (u64)k);
  const float p = a.top_p.of(b);
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
    group_find<kWaves>(part, chunks, ties - 1, red, found);
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
        u64 n = before + wave_scan64(same, lane) - same;
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
  // A number below 2^-40 draws the first kept token of any weight above 0, also one that is below the integers' unit.
  const float mp = a.min_p.of(b), uf = a.uniform[b];
  const bool first_kept = !(uf >= 9.094947e-13f);
  auto kept = [&](float x, int i) -> u64 {
    const unsigned ky = key_of(x);
    if (i >= V || ky < kmin || (ky == kmin && i > last_tie)) return 0;
    const double w = weight(r, x);
    if (!(w >= (double)mp || x == r.top || !(mp == mp))) return 0;
    return first_kept ? (u64)(w > 0.0) : fixed(r, w);
  };
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
  const u64 total = group_sum<kWaves>(mine, red);
  u64 want = first_kept ? 0 : (u64)fmin((double)uf * (double)total, 9.0e18);
  if (want >= total) want = total - 1;
  group_find<kWaves>(part, chunks, want, red, found);
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
    u64 cum = before + wave_scan64(s, lane) - s;
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
template <typename Keep>
__device__ __forceinline__ u64 resolve(Shared& sh, int n, u64 left, const Weigher& weigh, Keep keep) {
  constexpr u64 kFlip = 0xffffffffull;   // index reversed: the order is then that of falling numbers
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
    if (tid < 1024) sh.hist[tid] = 0;
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
    group_find<kWaves>(sh.hist, 1024, left - 1, sh.red, sh.found);
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
      if (before + w >= left) sh.found[2] = mine;
      else keep(mine, w);
    }
  }
  __syncthreads();
  return sh.found[2];
}

// grid B, one row each
template <typename T>
__global__ __launch_bounds__(kThreads) void choose_kernel(Args<T> a) {
  __shared__ Shared sh;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, V = a.V, chunks = a.chunks;
  const T* row = a.logits + (long)b * a.stride;
  const float* peaks = a.peaks + (long)b * a.groups;
  fill_table(sh.table);
  if (tid == 0) sh.listed = 0;
  const float top = row_peak(peaks, a.groups, reinterpret_cast<float*>(sh.red));
  const Kind kind = kind_of(a, b, top);
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
      const int i = g * kGroup + (lane & 15) * 8;
      load8(row, i, V, x);
      int first = 8;
#pragma unroll
      for (int j = 7; j >= 0; --j) first = x[j] == top ? j : first;
      const u64 hit = __ballot(first < 8 && lane < 16);
      if (lane == (hit ? __ffsll((long long)hit) - 1 : 0)) a.out[b] = hit && top > -INFINITY ? i + first : 0;
    }
    return;
  }
  if (kind == kFromStart) {
    choose_from_start(a, b, sh);
    return;
  }
  const float uf = a.uniform[b];
  const Weigher weigh = weigher(top, a.temp.of(b), a.shift, sh.table);
  const u64 least = least_weight(a.min_p.of(b), a.shift);
  auto target = [&](u64 total) {
    const u64 want = (u64)fmin((double)uf * (double)total, 9.0e18);
    return want >= total ? total - 1 : want;
  };
  if (kind == kShortK) {
    // the bound: the first bin at which k groups have their largest logit (or all that weighs anything)
    const int k = a.k_of(b);
    for (int i = tid; i < kBins; i += kThreads) sh.hist[i] = 0;
    __syncthreads();
    for (int g = tid; g < a.groups; g += kThreads) atomicAdd(&sh.hist[weigh.wide_bin(peaks[g])], 1ull);
    __syncthreads();
    group_find<kWaves>(sh.hist, kBins, (u64)k - 1, sh.red, sh.found);
    const int bound = min((int)sh.found[0], kBins - 2);
    // the groups at or above it, then their logits at or above it; 16 lanes take a group
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
    for (int at = tid >> 4; ok && at < n_groups; at += kThreads / 16) {
      float x[8];
      const int i = groups[at] * kGroup + (tid & 15) * 8;
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
      choose_from_start(a, b, sh);
      return;
    }
    u64 mine = 0, w = 0, before = 0;
    int rank = 0;
    if (tid < n) {
      mine = sh.list[tid] ^ 0xffffffffull;
      w = weigh(value_of((unsigned)(mine >> 32)));
      sh.weight[tid] = w;
    }
    __syncthreads();
    if (tid < n)
      for (int i = 0; i < n; ++i) {
        const bool ahead = (sh.list[i] ^ 0xffffffffull) > mine;
        rank += ahead;
        before += ahead ? sh.weight[i] : 0;
      }
    bool kept = tid < n && rank < k;
    const u64 z = group_sum<kWaves>(kept ? w : 0, sh.red);
    const float p = a.top_p.of(b);
    kept = kept && !(p < 1.f && before >= share_of(p, z)) && w >= least;
    const u64 want = target(group_sum<kWaves>(kept ? w : 0, sh.red));
    if (tid < n) sh.weight[tid] = kept ? w : 0;
    __syncthreads();
    if (kept) {
      u64 c = 0;
      for (int i = 0; i < n; ++i) c += (unsigned)sh.list[i] < ~(unsigned)mine ? sh.weight[i] : 0;
      if (c <= want && want < c + w) a.out[b] = (int64_t)(unsigned)~(unsigned)mine;
    }
    return;
  }
  // a logit is kept when its key is above kmin, or equals it at an index up to last, and its weight is `least` or more
  unsigned kmin = 0;
  int last = V;
  for (int c = tid; c < chunks; c += kThreads) sh.part[c] = a.mass[(long)b * chunks + c];
  if (kind == kTopP) {
    int bin = 0;
    u64 left = 0;
    const int n = a.listed[b];
    if (!border_bin<kWaves>(a.hist + (long)b * kBins, a.top_p.of(b), sh.red, sh.found, bin, left) || n > kList) {
      choose_from_start(a, b, sh);
      return;
    }
    for (int i = tid; i < n; i += kThreads) sh.list[i] = a.list[(long)b * kList + i];
    __syncthreads();
    auto keep = [&](u64 e, u64 w) {
      if (w >= least) atomicAdd(&sh.part[(unsigned)e / kChunk], w);
    };
    const u64 edge = resolve(sh, n, left, weigh, keep);
    kmin = (unsigned)(edge >> 32);
    last = (int)(unsigned)edge;
    if (tid == 0) keep(edge, weigh(value_of(kmin)));
  }
  __syncthreads();
  u64 total = 0;
  for (int c = tid; c < chunks; c += kThreads) total += sh.part[c];
  total = group_sum<kWaves>(total, sh.red);
  const u64 want = target(total);
  group_find<kWaves>(sh.part, chunks, want, sh.red, sh.found);
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
    u64 cum = sh.found[1] + wave_scan64(s, lane) - s;
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

}  // namespace smp
}  // namespace pd

using namespace pd;

// bytes of scratch for B rows of V logits
extern "C" long pd_sample_workspace(int B, int V) {
  const long chunks = (V + smp::kChunk - 1) / smp::kChunk, groups = (V + smp::kGroup - 1) / smp::kGroup;
  return (long)B * (8 * (chunks + smp::kBins + smp::kList) + 4 * (groups + 1));
}

extern "C" int pd_sample(int dt, const void* logits, long stride, int B, int V, const float* uniform, const float* temps,
                         float temp, const int* top_ks, int top_k, const float* top_ps, float top_p, const float* min_ps,
                         float min_p, int64_t* out, void* workspace, void* stream) {
  if (B <= 0) return 0;
  if (V < 1 || V > smp::kChunk * smp::kMaxChunks || B > 65535 || !workspace) return -1;
  int bits = 0;
  while ((1L << bits) < V) ++bits;
  const int shift = 62 - bits < 50 ? 62 - bits : 50;   // V weights of at most 2^shift stay under 2^62
  const int chunks = (V + smp::kChunk - 1) / smp::kChunk, groups = (V + smp::kGroup - 1) / smp::kGroup;
  // workgroups of four waves per row: a chunk a wave at most, about eight workgroups a CU in all
  int slices = (chunks + 3) / 4;
  const int enough = (2048 + B - 1) / B;
  if (slices > enough) slices = enough;
  hipStream_t st = (hipStream_t)stream;
  smp::u64* const mass = (smp::u64*)workspace;
  smp::u64* const hist = mass + (long)B * chunks;
  smp::u64* const list = hist + (long)B * smp::kBins;
  int* const listed = (int*)(list + (long)B * smp::kList);
  float* const peaks = (float*)(listed + B);
  // kernels that no row can need are not launched: the settings that are numbers say so
  const bool maybe_warm = temps || temp > 0.f;
  const bool maybe_short = top_ks || (top_k > 0 && top_k < V), always_k = !top_ks && maybe_short;
  const bool maybe_p = maybe_warm && !always_k && (top_ps || top_p < 1.f);
  PD_DISPATCH_FLOAT(dt, T, {
    const smp::Args<T> a{(const T*)logits, stride, V, chunks, groups, shift, uniform, {temps, temp}, {top_ps, top_p},
                         {min_ps, min_p}, top_ks, top_k, mass, hist, list, listed, peaks, out};
    smp::peaks_kernel<T><<<dim3(slices, B), 256, 0, st>>>(a);
    if (maybe_warm && !always_k) smp::bins_kernel<T><<<dim3(slices, B), 256, 0, st>>>(a);
    if (maybe_p) smp::sweep_kernel<T><<<dim3(slices, B), 256, 0, st>>>(a);
    smp::choose_kernel<T><<<B, smp::kThreads, 0, st>>>(a);
  });
  return (int)hipGetLastError();
}
