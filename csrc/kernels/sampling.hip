// One token per row of logits, from a given random number: temperature, top-k, top-p and min-p.
//
//   w_i = exp((x_i - max x) / T)                     weights; x ordered by (value descending, index ascending)
//   top-k: the first k of that order;  top-p: of what is left, the shortest head whose mass reaches p of it;
//   min-p: of what is left, w_i >= min_p (w of the best is 1);
//   token = the first index, in index order, whose cumulative kept mass exceeds u * (kept mass).
//
// A choice next to a border turns on the last bits of these sums, so weights are computed in 64 bits and summed as
// integers of 2^-shift (shift = 62 - bits of V): integer sums do not depend on the order they are taken in, so a row's
// token is the same in every launch.  No sort: the threshold of top-k / top-p is found by radix selection on the
// ordered bits of the logits (counts for top-k, masses for top-p), ties at the threshold by their index.
#include "common.h"

namespace pd {
namespace smp {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWaves = kThreads / 64, kChunk = 512, kMaxChunks = 2048;   // V <= 2^20

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

// sum of v over the workgroup, for every thread
__device__ __forceinline__ u64 group_sum(u64 v, u64* red) {
  v = wave_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 s = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) s += red[i];
  return s;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const T* __restrict__ logits, long stride, int V,
                                                         const float* __restrict__ uniform, Setting temp,
                                                         const int* __restrict__ top_ks, int top_k, Setting top_p,
                                                         Setting min_p, int shift, int64_t* __restrict__ out) {
  __shared__ u64 red[kWaves], hist[256], part[kMaxChunks], found[3];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const T* row = logits + (long)b * stride;
  const int chunks = (V + kChunk - 1) / kChunk;

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
  const float t = temp.of(b);
  if (!(t > 0.f) || r.top == -INFINITY) {   // greedy; a row with no allowed token gives 0
    if (tid == 0) out[b] = (unsigned)~(unsigned)best;
    return;
  }
  r.inv_t = 1.0 / (double)t;
  r.unit = __longlong_as_double((long long)(1023 + shift) << 52);

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
    s = group_sum(s, red);
    same = group_sum(same, red);
    if (same > ties) same = ties;
    return s + (same ? same * fixed(r, weight(r, value_of(kmin))) : 0);
  };
  int k = top_ks ? top_ks[b] : top_k;
  if (k > 0 && k < V) ties = select(false, (u64)k);
  const float p = top_p.of(b);
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
    if (wv == 0) {
      // the chunk that holds tie number `ties` (counted from 1), then the element
      u64 before = 0;
      int at = -1;
      for (int c0 = 0; c0 < chunks && at < 0; c0 += 64) {
        const u64 v = c0 + lane < chunks ? part[c0 + lane] : 0;
        const u64 incl = wave_scan64(v, lane);
        const u64 hit = __ballot(before + incl >= ties);
        if (hit) {
          const int l = __ffsll((long long)hit) - 1;
          before += __shfl(incl - v, l, 64);
          at = c0 + l;
        } else {
          before += __shfl(incl, 63, 64);
        }
      }
      if (lane == 0) found[0] = V;
      if (at >= 0) {
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
  const float mp = min_p.of(b), uf = uniform[b];
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
  const u64 total = group_sum(mine, red);
  if (wv == 0) {
    u64 want = first_kept ? 0 : (u64)fmin((double)uf * (double)total, 9.0e18);
    if (want >= total) want = total - 1;
    u64 before = 0;
    int at = -1;
    for (int c0 = 0; c0 < chunks && at < 0; c0 += 64) {
      const u64 v = c0 + lane < chunks ? part[c0 + lane] : 0;
      const u64 incl = wave_scan64(v, lane);
      const u64 hit = __ballot(before + incl > want);
      if (hit) {
        const int l = __ffsll((long long)hit) - 1;
        before += __shfl(incl - v, l, 64);
        at = c0 + l;
      } else {
        before += __shfl(incl, 63, 64);
      }
    }
    if (at < 0) at = chunks - 1;   // not reached: total > want
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
      out[b] = token;
    }
  }
}

}  // namespace smp
}  // namespace pd

using namespace pd;

extern "C" int pd_sample(int dt, const void* logits, long stride, int B, int V, const float* uniform, const float* temps,
                         float temp, const int* top_ks, int top_k, const float* top_ps, float top_p, const float* min_ps,
                         float min_p, int64_t* out, void* stream) {
  if (B <= 0) return 0;
  if (V < 1 || V > smp::kChunk * smp::kMaxChunks) return -1;
  int bits = 0;
  while ((1L << bits) < V) ++bits;
  const int shift = 62 - bits < 50 ? 62 - bits : 50;   // V weights of at most 2^shift stay under 2^62
  const smp::Setting t{temps, temp}, p{top_ps, top_p}, m{min_ps, min_p};
  PD_DISPATCH_FLOAT(dt, T, (smp::sample_kernel<T><<<B, smp::kThreads, 0, (hipStream_t)stream>>>(
                               (const T*)logits, stride, V, uniform, t, top_ks, top_k, p, m, shift, out)));
  return (int)hipGetLastError();
}
