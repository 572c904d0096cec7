// Attention of a chunk of new tokens over a paged KV cache (chunked prefill, drafted tokens, mixed steps).
//
// Packed queries q[cu[b] .. cu[b+1]) are the last n_b of the len_b tokens that sequence b holds in the cache (their
// own K / V rows are there already); query i of them, at position p = len_b - n_b + i, sees the keys 0 .. p:
//   o = sum_j exp(s_j - max s) v_j / sum_j exp(s_j - max s),   s_j = scale * q . k_j
// Token t of sequence b lives at page(b, t) * s_blk + (t % block) * s_tok + kv_head * s_head, in 64 bits.
//
//  * A workgroup (4 waves, or two groups of 4) owns 128 rows of one (sequence, kv head): rows are (token, query head of
//    the group), so a K / V tile read once serves the whole group; where a sequence has no more it owns 16 (few_rows).  Its
//    sequence is found from cu by a prefix sum over the lanes: the host never reads lengths, and the launch is the same
//    for every batch of a shape (it can be captured).
//  * S^T = K . Q^T on 32x32x16 MFMA: a lane owns one row's scores, the softmax needs one exchange between lane
//    halves, and the bf16 / fp16 P is the next product's operand as it stands.  P is rounded to 16 bits because the
//    matrix unit takes 16-bit operands.  Each P is off by half a step, and the sums of these are about as large as the
//    output's own rounding: in bf16 the error against 64 bits is 0.0017 with the output's rounding alone and 0.0020 - 0.0023
//    with both.  Scores, maxima, sums and O stay in 32 bits.
//  * 64-key tiles lie in LDS in two stages, page numbers are looked up one tile further ahead.  Where one page holds the
//    rows of a wave's load the tiles go there straight from memory, else through registers.  Keys past the rows' reach and
//    pages outside the pool give zeros, so stale pages (NaN among them) never reach a product.
//  * A hidden key has P = 0, but 0 * inf is NaN: in tiles that some row does not see in full, values that are not
//    finite enter the product as 0 and are added at the end to the rows that see them.
//  * Few tiles over a long cache: the key range is split over workgroups, and the pieces (m, l, O) are joined by a
//    second kernel.  How often is decided per tile, from its own length.
//
// Measured (bf16, D = 128, 32 heads on 8, pages of 64): 2,048 tokens over 30,720 take 975 - 1,050 us by the card, 1.01 - 1.09
// PFLOP/s, bound by the exponentials and maxima beside the products (two waves per SIMD: the matrix unit is busy 55 % of the
// time); 64 single tokens over 4,000 - 8,000 take 310 us, 5.1 TB/s, the rate of a large copy.
#include "common.h"

#include <type_traits>

namespace pd {
namespace ca {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) char lds_char;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kDefer = 8.f;   // the running maximum moves only when a row outgrows it by 2^8
// Weights are exp2(s - m + lift): float16 ends at 2^16, so 2^(8 + 7) fits, and its smallest step, 2^-24, is 2^-31 of the weight
// at m (without the lift 30,000 keys of 2^-25 each counted as nothing).  bfloat16 has the range of 32 bits.
template <bool F16>
constexpr float kLift = F16 ? 7.f : 0.f;
constexpr int kBM = 128, kBN = 64;

__device__ const u16x8 kZeros[16] = {};   // a row of D = 128
// p, or a row of zeros.  (Both are named global: chosen as plain pointers they gave flat loads, which count as LDS
// operations too and made every LDS wait one for memory.)
typedef __attribute__((address_space(1))) const u16x8 global_u16x8;
__device__ __forceinline__ global_u16x8* row_or_zeros(bool ok, const unsigned short* p) {
  return ok ? (global_u16x8*)p : (global_u16x8*)kZeros;
}

struct Args {
  const unsigned short *q, *k, *v;
  unsigned short* out;
  long sq_tok, sq_head, so_tok, so_head;   // in elements
  int s_blk, s_tok, s_head;
  const int *cu, *lens, *table;
  int B, T, Hq, Hk, G;
  int max_blocks, num_blocks, block, block_shift;
  unsigned block_mul;                               // key / block = key * block_mul >> block_shift, for keys < 2^31
  int splits, min_keys;                             // pieces of a tile's keys at most, keys of one at least
  float scale_log2;
  float *part_o, *part_ml;                          // [splits][T][Hq][D], [splits][T][Hq][2]
  int* pieces;                                      // [T] into how many a token's keys were split
};

struct Seq {
  int b, q0, n, len, tile;   // first query row, new tokens, keys, tile within the sequence (-1: none)
};
constexpr int kFewRows = 16, kFewKeys = 32;   // few rows: the rows of a tile, the keys of one wave's step

__device__ __forceinline__ void bounds_of(const Args& a, int b, int& q0, int& n) {
  q0 = min(max(a.cu[b], 0), a.T);
  n = max(min(a.cu[b + 1], a.T) - q0, 0);
}
__device__ __forceinline__ int len_of(const Args& a, int b) {
  return (int)min((long)max(a.lens[b], 0), (long)a.max_blocks * a.block);
}

__device__ __forceinline__ int xcd_remap(int bid, int n) {
  const int q = n / 8, r = n % 8, xcd = bid % 8;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + bid / 8;
}

// 64 sequences from b0, one a lane: where its queries begin, how many, its keys, and the row tiles up to and with it: all of
// 16 rows (FEW), or of 128, and beside them one of 16 for each sequence that has no more
struct Lanes {
  int q0, n, len, upto, few_upto;
};
template <bool FEW>
__device__ __forceinline__ Lanes sequences(const Args& a, int b0, int lane) {
  Lanes s;
  const int b = min(b0 + lane, a.B - 1), tile_tokens = (FEW ? kFewRows : kBM) / a.G;
  bounds_of(a, b, s.q0, s.n);
  s.len = len_of(a, b);
  if (b0 + lane >= a.B) s.n = 0;
  const bool few = !FEW && s.n > 0 && s.n <= kFewRows / a.G;
  s.upto = few ? 0 : (s.n + tile_tokens - 1) / tile_tokens;
  s.few_upto = few ? 1 : 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(s.upto, o, 64);
    if (lane >= o) s.upto += t;
    if constexpr (!FEW) {
      const int f = __shfl_up(s.few_upto, o, 64);
      if (lane >= o) s.few_upto += f;
    }
  }
  return s;
}

// This workgroup's part of the batch: a row tile, a kv head and a piece of the keys; every wave works it out for itself.
// The grid is an upper bound of the parts there are; neighbours are the kv heads of one tile, and a sequence's tiles go
// from the one that sees the most keys to the one that sees the fewest.
//  Few rows: each XCD takes an eighth of the parts, side by side, so that the heads' rows of one key, which share lines
//  and pages, are read by one XCD.
//  Many: workgroup i has part i, and an XCD every eighth: with eight heads or a multiple each has its own heads'
//  keys in its L2, and the tiles' lengths are spread evenly.  Two workgroups share a CU, and the second of each is
//  dispatched after the first of all: the second 32 of an XCD go from light to heavy, so that a heavy one has a light
//  one beside it (2,048 tokens, 32 heads, nothing cached: 74 us without, all that a CU did was one weight).
//  The tiles of many rows come first, those of few after them.
template <bool FEW>
__device__ __forceinline__ Seq find_part(const Args& a, int lane, int& hk, int& sp, bool& few) {
  Lanes s = sequences<FEW>(a, 0, lane);
  int total = __builtin_amdgcn_readlane(s.upto, 63), few_total = __builtin_amdgcn_readlane(s.few_upto, 63);
  for (int b0 = 64; b0 < a.B; b0 += 64) {
    const Lanes t = sequences<FEW>(a, b0, lane);
    total += __builtin_amdgcn_readlane(t.upto, 63);
    few_total += __builtin_amdgcn_readlane(t.few_upto, 63);
  }
  int parts = total * a.Hk * a.splits;
  int id = blockIdx.x;
  few = FEW;
  if (!FEW && id >= parts) {
    id -= parts;
    few = true;
    parts = few_total * a.Hk * a.splits;
  }
  if (id >= parts) return Seq{0, 0, 0, 0, -1};
  if (few) {
    id = xcd_remap(id, parts);
  } else {
    const int per = parts / 8;   // (full rows of eight)
    const int j = id / 8, last = min(per, 64) - 1;
    if (j >= 32 && j <= last) id = (32 + last - j) * 8 + id % 8;
  }
  hk = id % a.Hk, sp = id / a.Hk % a.splits;
  const int tile = id / (a.Hk * a.splits);
  int base = 0, b0 = 0;
  for (;;) {
    const int upto = !FEW && few ? s.few_upto : s.upto;
    const unsigned long long hit = __ballot(base + upto > tile);   // some lane, tile < total
    if (hit) {
      const int l = __builtin_amdgcn_readfirstlane(__ffsll((long long)hit) - 1);
      Seq r;
      r.b = b0 + l;
      r.q0 = __builtin_amdgcn_readlane(s.q0, l);
      r.n = __builtin_amdgcn_readlane(s.n, l);
      r.len = __builtin_amdgcn_readlane(s.len, l);
      // the tile that sees the most keys first
      r.tile = __builtin_amdgcn_readlane(upto, l) - 1 - (tile - base);
      return r;
    }
    base += __builtin_amdgcn_readlane(upto, 63);
    b0 += 64;
    if (b0 >= a.B) return Seq{0, 0, 0, 0, -1};
    s = sequences<FEW>(a, b0, lane);
  }
}

// keys per piece of a tile that sees `keys` keys: whole grains, at least min_keys, at most `splits` pieces
__device__ __forceinline__ int piece_of(const Args& a, int keys, int grain) {
  const int pieces = max(1, min(a.splits, (keys + a.min_keys - 1) / a.min_keys));
  const int per = (keys + pieces - 1) / pieces;
  return max((per + grain - 1) / grain * grain, grain);
}

template <int D>
__device__ __forceinline__ int swz(int row, int ch) {
  return ch ^ ((((row & 3) << 2) | ((row >> 2) & 3)) & (D / 8 - 1));
}
__device__ __forceinline__ s16x4 lds_tr(const char* base, int off) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)((lds_char*)base + off));
}
template <bool F16>
__device__ __forceinline__ unsigned short cvt16(float f) {
  if constexpr (F16) return f2h(f);
  else return f2bf(f);
}
template <bool F16>
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ bf16x8 pack8(const f32x16& acc, int s) {
  if constexpr (F16) {
    f16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (_Float16)acc[8 * s + j];
    return __builtin_bit_cast(bf16x8, r);
  } else {
    bf16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (__bf16)acc[8 * s + j];
    return r;
  }
}
// Barrier for LDS hand-offs: this wave's LDS operations are done, its global loads may stay in flight (__syncthreads
// would wait for them too)
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ int block_of(const Args& a, int key) {
  return (int)(((unsigned long long)(unsigned)key * a.block_mul) >> a.block_shift);
}

// Few rows (decoding, drafted tokens): 16 rows of one (sequence, kv head) per workgroup, bound by the reads of K and V.
// Each of the W waves takes every W-th 32-key tile of the piece on its own, with no barrier in the loop:
//  * S^T = K . Q^T on 16x16x32 MFMA; a lane loads its K operands (16 bytes of a key's row) straight into registers, V goes
//    through a wave's own LDS image for the transposed reads;
//  * two register sets in turn: 32 loads of 16 bytes a lane are in flight (D = 128), page numbers one tile further ahead;
//  * the waves' (m, l, O) are joined through LDS at the end.
// A step that mixes single tokens with pieces of prompts has both kinds of tiles in one launch: 45 sequences over 1,250 -
// 2,500 keys, 33 of them single tokens, take 44 us, with 128-row tiles for all of them 48 (D = 64, 16 heads on 4).  Where
// few rows are all there is, a kernel of their own with less LDS and smaller pieces: 64 single tokens over 4,000 - 8,000
// keys take 311 us in it, 338 in the other; 8 x 4 drafted tokens over 350 - 700, 32 heads, 19 us (13.5 at a copy's rate).

template <bool F16>
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <int D, bool F16, int W>
__device__ __forceinline__ void few_rows(const Args& a, const Seq& s, int hk, int sp, char* lds) {
  constexpr int KC = D / 32, DT = D / 16;
  constexpr unsigned short kExp = F16 ? 0x7c00 : 0x7f80;
  // lds: W * kFewKeys * D * 2 bytes, the waves' V images, then their O
  __shared__ float ml[W][kFewRows][2];
  __shared__ int odd_values;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, h = lane >> 4;
  const int tile_tokens = kFewRows / a.G;
  const int tok0 = s.tile * tile_tokens, ntok = min(tile_tokens, s.n - tok0);
  const int pos0 = s.len - s.n + tok0, keys = max(pos0 + ntok, 0);
  const int piece = piece_of(a, keys, W * kFewKeys), k0 = sp * piece, k1 = min(keys, k0 + piece);
  const bool whole = piece >= keys;
  if (a.splits > 1 && sp == 0 && hk == 0 && tid < ntok) a.pieces[s.q0 + tok0 + tid] = whole ? 1 : (keys + piece - 1) / piece;
  if (sp > 0 && k0 >= keys) return;
  if (tid == 0) odd_values = 0;
  lds_barrier();

  const int rt = c16 / a.G, rh = hk * a.G + c16 % a.G, pos = pos0 + rt;
  const bool live = rt < ntok;
  bf16x8 qf[KC];
  {
    const unsigned short* qp = a.q + (long)(s.q0 + tok0 + (live ? rt : 0)) * a.sq_tok + (long)(live ? rh : 0) * a.sq_head + 8 * h;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      qf[c] = *reinterpret_cast<const bf16x8*>(qp + 32 * c);
      if (!live) qf[c] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }
  const int* tab = a.table + (long)s.b * a.max_blocks;
  const unsigned head_off = hk * a.s_head + 8 * h;
  const int ntiles = k1 > k0 ? (k1 - k0 + kFewKeys - 1) / kFewKeys : 0;
  auto pages = [&](int t, int (&pg)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) pg[u] = tab[block_of(a, min(k0 + kFewKeys * t + 16 * u + c16, k1 - 1))];
  };
  auto load = [&](int t, const int (&pg)[2], u16x8 (&kk)[2][KC], u16x8 (&vv)[2][KC]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = k0 + kFewKeys * t + 16 * u + c16, blk = block_of(a, key);
      const bool ok = key < k1 && (unsigned)pg[u] < (unsigned)a.num_blocks;
      const long off = (long)pg[u] * a.s_blk + (unsigned)((key - blk * a.block) * a.s_tok + head_off);
      global_u16x8 *pk = row_or_zeros(ok, a.k + off), *pv = row_or_zeros(ok, a.v + off);
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        kk[u][c] = pk[4 * c];
        vv[u][c] = pv[4 * c];
      }
    }
  };
  f32x4 o[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const float sl2 = a.scale_log2;
  char* const vl = lds + w * (kFewKeys * D * 2);
  const int qq = c16 >> 2, pp = c16 & 3;
  // (16 rows further down the swizzle is the same, and a chunk is an XOR)
  int o_w = c16 * (D * 2) + 16 * swz<D>(c16, h);
  int o_r = (4 * h + qq) * (D * 2) + 16 * swz<D>(4 * h + qq, pp >> 1) + 8 * (pp & 1);
  auto compute = [&](int t, const u16x8 (&kk)[2][KC], u16x8 (&vv)[2][KC]) {
    const int n0 = k0 + kFewKeys * t;
    asm volatile("" : "+v"(o_w), "+v"(o_r));   // the XORs stay in the loop: hoisted they spilled
    if (n0 + kFewKeys - 1 > pos0) {   // some row does not see all of it: values that are not finite are put in at the end
      constexpr unsigned kE = kExp | (unsigned)kExp << 16, kLow = F16 ? 0x04000400u : 0x00800080u;
      unsigned hit = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          const auto x = __builtin_bit_cast(u32x4, vv[u][c]);
#pragma unroll
          for (int j = 0; j < 4; ++j) hit |= (x[j] & kE) + kLow;
        }
      if (__builtin_expect(hit & 0x80008000u, 0)) {
        odd_values = 1;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int j = 0; j < 8; ++j) vv[u][c][j] = (vv[u][c][j] & kExp) == kExp ? (unsigned short)0 : vv[u][c][j];
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < KC; ++c)
        *reinterpret_cast<u16x8*>(vl + (o_w ^ (c << 6)) + 16 * u * (D * 2)) = vv[u][c];
    f32x4 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c) sc[u] = mfma16<F16>(__builtin_bit_cast(bf16x8, kk[u][c]), qf[c], sc[u]);
    }
    const int lim = min(k1, pos + 1) - n0 - 4 * h;   // key n0 + 16 u + 4 h + e is hidden iff 16 u + e >= lim
    float mt = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[u][e] = 16 * u + e >= lim ? -INFINITY : sc[u][e] * sl2;
        mt = fmaxf(mt, sc[u][e]);
      }
    mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    const float mn = fmaxf(m, mt), top = mn == -INFINITY ? 0.f : mn, base = top - kLift<F16>;
    const float alpha = __builtin_amdgcn_exp2f(m - top);
    m = mn;
    bf16x8 pf;
    float ps = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f(sc[u][e] - base);
        ps += p;
        pf[4 * u + e] = __builtin_bit_cast(__bf16, cvt16<F16>(p));
      }
    l = l * alpha + ps;
    float ar[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ar[e] = __shfl(alpha, 4 * h + e, 64);   // O's row 4 h + e has its state in that lane
#pragma unroll
    for (int t2 = 0; t2 < DT; ++t2) {
      const s16x4 lo = lds_tr(vl, o_r ^ (t2 << 5)), hi = lds_tr(vl + 16 * (D * 2), o_r ^ (t2 << 5));
      const s16x8 v8 = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t2][e] *= ar[e];
      o[t2] = mfma16<F16>(pf, __builtin_bit_cast(bf16x8, v8), o[t2]);
    }
  };
  // Two tiles a turn without an exit between them; past the last tile keys are hidden and loads read zeros
  u16x8 ka[2][KC], va[2][KC], kb[2][KC], vb[2][KC];
  if (w < ntiles) {
    int pa[2], pb[2];
    pages(w, pa);
    pages(w + W, pb);
    load(w, pa, ka, va);
    for (int t = w; t < ntiles; t += 2 * W) {
      pages(t + 2 * W, pa);
      load(t + W, pb, kb, vb);
      __builtin_amdgcn_sched_barrier(0);   // the loads stay ahead of the work
      compute(t, ka, va);
      pages(t + 3 * W, pb);
      load(t + 2 * W, pa, ka, va);
      __builtin_amdgcn_sched_barrier(0);
      compute(t + W, kb, vb);
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __syncthreads();   // every wave is done with its V image
  float* const ow = reinterpret_cast<float*>(lds);   // [W][16][D]
  if (h == 0) {
    ml[w][c16][0] = m;
    ml[w][c16][1] = l;
  }
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) ow[(w * kFewRows + 4 * h + e) * D + 16 * t + c16] = o[t][e];
  __syncthreads();
  const int rows = ntok * a.G;
  for (int i = tid; i < rows * (D / 4); i += 64 * W) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < W; ++x) M = fmaxf(M, ml[x][row][0]);
    const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int x = 0; x < W; ++x) {
      const float wt = __builtin_amdgcn_exp2f(ml[x][row][0] - base);
      L += ml[x][row][1] * wt;
      acc += *reinterpret_cast<const f32x4*>(ow + (x * kFewRows + row) * D + d) * wt;
    }
    const int tok = row / a.G, hq = hk * a.G + row % a.G;
    if (__builtin_expect(odd_values, 0)) {   // the values that were taken out, where this row sees them
      for (int j = k0 + max(pos0 - k0, 0) / kFewKeys * kFewKeys; j < k1 && j <= pos0 + tok; ++j) {
        const int blk = block_of(a, j), page = tab[blk];
        if ((unsigned)page >= (unsigned)a.num_blocks) continue;
        const unsigned short* vr = a.v + (long)page * a.s_blk + (unsigned)((j - blk * a.block) * a.s_tok + hk * a.s_head) + d;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if ((vr[e] & kExp) == kExp) acc[e] += F16 ? h2f(vr[e]) : bf2f(vr[e]);
      }
    }
    const long trow = s.q0 + tok0 + tok;
    if (whole) {
      const float inv = L != 0.f ? 1.f / L : 0.f;
      typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
      u16x4 r;
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = cvt16<F16>(acc[e] * inv);
      *reinterpret_cast<u16x4*>(a.out + trow * a.so_tok + (long)hq * a.so_head + d) = r;
    } else {
      const long pi = ((long)sp * a.T + trow) * a.Hq + hq;
      *reinterpret_cast<f32x4*>(a.part_o + pi * D + d) = acc;
      if (d == 0) {
        a.part_ml[pi * 2] = M;
        a.part_ml[pi * 2 + 1] = L;
      }
    }
  }
}

template <int D, bool F16, int W>
__global__ __launch_bounds__(64 * W, W == 8 ? 1 : 2) void few_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) char lds[W * kFewKeys * D * 2];
  int hk, sp;
  bool few;
  const Seq s = find_part<true>(a, threadIdx.x & 63, hk, sp, few);
  if (s.tile >= 0) few_rows<D, F16, W>(a, s, hk, sp, lds);
}

// A K or V tile on its way from the pages to LDS: a thread brings chunk tid % NCH of rows tid / NCH + ROWS * i.
// UNI: the block size is a multiple of the RW rows that one wave's load covers, so a wave's rows of a load lie in one page.
// Lane i works out load i's page, byte offset and extent, and the load is a buffer load from a scalar base whose extent
// ends with the valid rows (past it, and for page numbers outside the pool, it reads zeros): K and V share all of that.
// It goes to LDS without passing registers, whose order of chunks the lanes' addresses have to follow then.
// Otherwise every thread looks up its own rows' pages, points the missing ones at a block of zeros, and stores what it
// loaded.
template <int D, bool UNI>
struct Stage {
  static constexpr int NCH = D / 8, NLOAD = kBN * NCH / 256, ROWS = 256 / NCH, RW = 64 / NCH;
  const Args& a;
  const int* tab;
  int k1, first_row, o_st, voff;
  int page[UNI ? 1 : NLOAD], rest[UNI ? 1 : NLOAD], rows;   // of the tile to come
  unsigned lo[NLOAD], hi[NLOAD];                            // UNI: of the present one (scalar)
  int bytes[NLOAD];
  u16x8 st[UNI ? 1 : NLOAD];
  __device__ __forceinline__ Stage(const Args& a_, const Seq& s, int hk, int tid, int k1_) : a(a_) {
    tab = a.table + (long)s.b * a.max_blocks;
    k1 = k1_;
    // (the swizzle has the row's lowest 4 bits, which ROWS leaves alone)
    const int lrow = tid / NCH, lch = tid % NCH, sch = swz<D>(lrow, lch);
    if constexpr (UNI) {
      o_st = __builtin_amdgcn_readfirstlane(tid >> 6) * 1024;
      first_row = (tid >> 6) * RW + ROWS * (tid & (NLOAD - 1));
      voff = (lrow % RW) * a.s_tok * 2 + (hk * a.s_head + sch * 8) * 2;
    } else {
      o_st = lrow * (D * 2) + sch * 16;
      first_row = lrow;
      voff = hk * a.s_head + lch * 8;
    }
  }
  // look up the pages of the tile at n0
  __device__ __forceinline__ void pages(int n0) {
#pragma unroll
    for (int i = 0; i < (UNI ? 1 : NLOAD); ++i) {
      const int key = n0 + first_row + ROWS * i, blk = block_of(a, min(key, k1 - 1));
      page[i] = tab[blk];
      rest[i] = (key - blk * a.block) * a.s_tok;
      if constexpr (UNI) rows = min(max(k1 - key, 0), RW);
      else rest[i] = key < k1 ? rest[i] : -1;
    }
  }
  // where they lie, once they have arrived: K and V alike
  __device__ __forceinline__ void locate(int hk) {
    if constexpr (UNI) {
      const unsigned long long off = ((unsigned long long)(unsigned)page[0] * (unsigned)a.s_blk + (unsigned)rest[0]) * 2;
      const bool ok = (unsigned)page[0] < (unsigned)a.num_blocks && rows > 0;
      // (rows of other heads may lie between: the extent reaches to the end of the last row's head)
      const int b = ok ? ((rows - 1) * a.s_tok + hk * a.s_head + D) * 2 : 0;
#pragma unroll
      for (int i = 0; i < NLOAD; ++i) {
        lo[i] = __builtin_amdgcn_readlane((int)(unsigned)off, i);
        hi[i] = __builtin_amdgcn_readlane((int)(unsigned)(off >> 32), i);
        bytes[i] = __builtin_amdgcn_readlane(b, i);
      }
    }
  }
  __device__ __forceinline__ void load(const unsigned short* cache, char* dst) {
#pragma unroll
    for (int i = 0; i < NLOAD; ++i) load(i, cache, dst);
  }
  __device__ __forceinline__ void load(int i, const unsigned short* cache, char* dst) {
    {
      if constexpr (UNI) {
        const unsigned long long at = (unsigned long long)cache + (lo[i] | (unsigned long long)hi[i] << 32);
        const i32x4 rs = {(int)at, (int)(at >> 32) & 0xffff, bytes[i], 0x00020000};
        const unsigned m0 = (unsigned)(size_t)(lds_char*)dst + o_st + i * ROWS * (D * 2);
        // (five wait states between a lane read and a buffer's use of its result; the compiler counts none inside here.
        // Its own waits for LDS reads would wait for every such load: nothing here tells it that they don't meet)
        asm volatile(
            "s_mov_b32 m0, %0\n\t"
            "s_nop 4\n\t"
            "buffer_load_dwordx4 %1, %2, 0 offen lds"
            :
            : "s"(m0), "v"(voff), "s"(rs)
            : "memory", "m0");
      } else {
        const bool ok = rest[i] >= 0 && (unsigned)page[i] < (unsigned)a.num_blocks;
        const unsigned short* p = cache + (long)page[i] * a.s_blk + (unsigned)(rest[i] + voff);
        st[i] = *row_or_zeros(ok, p);
      }
    }
  }
  __device__ __forceinline__ void store(char* dst) const {
    if constexpr (!UNI) {
#pragma unroll
      for (int i = 0; i < NLOAD; ++i) *reinterpret_cast<u16x8*>(dst + o_st + i * ROWS * (D * 2)) = st[i];
    }
  }
  __device__ __forceinline__ void take(const Stage& s) {
#pragma unroll
    for (int i = 0; i < NLOAD; ++i) lo[i] = s.lo[i], hi[i] = s.hi[i], bytes[i] = s.bytes[i];
  }
  __device__ __forceinline__ void arrived() const {
    if constexpr (UNI) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
};

// KG groups of four waves: each takes every KG-th 64-key tile of the same 128 rows, and the groups' (m, l, O) are joined
// through LDS.  KG = 2 has one workgroup on a CU where KG = 1 has two.
template <int D, bool F16, bool UNI, int KG>
__global__ __launch_bounds__(256 * KG, KG == 2 ? 1 : 2) void chunk_kernel(Args a) {
  constexpr unsigned short kExp = F16 ? 0x7c00 : 0x7f80;         // exponent bits: all set in infinities and NaN
  constexpr int KS = D / 16, DT = D / 32, TILE = kBN * D * 2;
  using St = Stage<D, UNI>;
  constexpr int NLOAD = St::NLOAD;
  __shared__ __attribute__((aligned(16))) char lds[KG * 4 * TILE];
  __shared__ int odd_values;   // finite_only took something out
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tid = threadIdx.x & 255, wv = wave & 3, group = wave >> 2;
  char* const smem = lds + group * 4 * TILE;
  const int r = lane & 31, h = lane >> 5;
  const int tile_tokens = kBM / a.G;

  int hk, sp;
  bool few;
  const Seq s = find_part<false>(a, lane, hk, sp, few);
  if (s.tile < 0) return;
  if (few) {
    few_rows<D, F16, 4 * KG>(a, s, hk, sp, lds);
    return;
  }
  const int tok0 = s.tile * tile_tokens;                        // first token of the tile within the sequence
  const int ntok = min(tile_tokens, s.n - tok0);
  const int pos0 = s.len - s.n + tok0;                          // its position (negative: it sees nothing)
  const int keys = max(pos0 + ntok, 0);                         // keys the tile's last token sees
  const int piece = piece_of(a, keys, kBN);
  const int k0 = sp * piece, k1 = min(keys, k0 + piece);
  const bool whole = piece >= keys;
  if (a.splits > 1 && sp == 0 && hk == 0)
    for (int i = threadIdx.x; i < ntok; i += 256 * KG) a.pieces[s.q0 + tok0 + i] = whole ? 1 : (keys + piece - 1) / piece;
  if (sp > 0 && k0 >= keys) return;

  const int row = wv * 32 + r;                                  // this lane's row: token row / G, head row % G
  const int rt = row / a.G, rh = hk * a.G + row % a.G;
  const bool live = rt < ntok;
  const int pos = pos0 + rt;

  bf16x8 qf[KS];
  {
    const unsigned short* qp = a.q + (long)(s.q0 + tok0 + (live ? rt : 0)) * a.sq_tok + (long)(live ? rh : 0) * a.sq_head + 8 * h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qf[ks] = *reinterpret_cast<const bf16x8*>(qp + ks * 16);
      if (!live) qf[ks] = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
    }
  }

  St stage(a, s, hk, tid, k1);
  // The thread's share of a V tile at n0 that some row does not see in full: values that are not finite become 0 (rare).
  // UNI: it lies in LDS at dst, else still in registers
  auto finite_only = [&](int n0, char* dst) {
    if (n0 + kBN - 1 <= pos0) return;
    constexpr unsigned kE = kExp | (unsigned)kExp << 16, kLow = F16 ? 0x04000400u : 0x00800080u;
    unsigned hit = 0;   // exponent + its lowest bit carries into bit 15 iff all exponent bits are set
    auto share = [&](int i) -> u16x8& {
      if constexpr (UNI) return *reinterpret_cast<u16x8*>(dst + tid * 16 + i * (St::ROWS * D * 2));
      else return stage.st[i];
    };
#pragma unroll
    for (int i = 0; i < NLOAD; ++i) {
      const auto w = __builtin_bit_cast(u32x4, share(i));
#pragma unroll
      for (int j = 0; j < 4; ++j) hit |= (w[j] & kE) + kLow;
    }
    if (__builtin_expect(hit & 0x80008000u, 0)) {
      odd_values = 1;
#pragma unroll
      for (int i = 0; i < NLOAD; ++i) {
        u16x8 v = share(i);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (v[j] & kExp) == kExp ? (unsigned short)0 : v[j];
        share(i) = v;
      }
    }
  };

  f32x16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
  float m = -INFINITY, l = 0.f;
  const float sl2 = a.scale_log2;
  const int wave_rt0 = wv * 32 / a.G, wave_rt1 = min((wv * 32 + 31) / a.G, ntok - 1);
  const int wave_last = wave_rt0 < ntok ? pos0 + wave_rt1 : -1;   // the last key that some row of the wave sees

  const int ntiles = k1 > k0 ? (k1 - k0 + kBN - 1) / kBN : 0;
  constexpr int kStep = KG * kBN;       // from one tile of a group to its next
  const int kg = k0 + group * kBN;      // the group's first
  if (threadIdx.x == 0) odd_values = 0;
  lds_barrier();
  // The tiles run one ahead: S of the next tile is multiplied while the present one is exponentiated, so K is staged two
  // tiles ahead and V one (K and V have two stages each: a stage is written in the round after its last read).
  if (ntiles > 0) {
    stage.pages(kg);
    if constexpr (UNI) {   // K and V of the first tile and K of the second, all on their way together
      St next(stage);
      next.pages(kg + kStep);
      stage.locate(hk);
      stage.load(a.k, smem);
      stage.load(a.v, smem + 2 * TILE);
      next.locate(hk);
      next.load(a.k, smem + TILE);
      stage.take(next);
      stage.pages(kg + 2 * kStep);
      stage.arrived();
      finite_only(kg, smem + 2 * TILE);
    } else {
      stage.load(a.k, smem);
      St first(stage);
      stage.load(a.v, smem);
      stage.pages(kg + kStep);
      first.store(smem);
      finite_only(kg, smem);
      stage.store(smem + 2 * TILE);
      stage.load(a.k, smem);
      stage.store(smem + TILE);
    }
  }
  lds_barrier();

  // Lane bases of the LDS reads, in the stage being read; every read is one of them with a compile-time XOR and offset:
  //  K row kb * 32 + r, 16-byte chunk 2 ks + h;  V^T: rows 16 s + 8 (j >> 2) + 4 hh + qq, chunk 4 dt + cbits
  const int g = lane >> 4, qq = (lane & 15) >> 2, pp = lane & 3, hh = g >> 1, cbits = ((g & 1) << 1) | (pp >> 1);
  int o_k = r * (D * 2) + swz<D>(r, h) * 16;
  int o_va = 2 * TILE + (4 * hh + qq) * (D * 2) + swz<D>(4 * hh + qq, cbits) * 16 + 8 * (pp & 1);
  int o_vb = 2 * TILE + (4 * hh + qq + 8) * (D * 2) + swz<D>(4 * hh + qq + 8, cbits) * 16 + 8 * (pp & 1);
  int buf = 0;   // the present tile's stage: 0 or TILE

  auto scores = [&](f32x16 (&sc)[2], int at) {   // of the K stage at byte `at`
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      sc[kb] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        sc[kb] = mfma<F16>(*reinterpret_cast<const bf16x8*>(smem + kb * 32 * (D * 2) + (at ^ (ks << 5))), qf[ks], sc[kb]);
    }
  };
  auto hide = [&](f32x16 (&sc)[2], int n0) {
    const int lim = min(k1, pos + 1) - n0 - 4 * h;   // key n0 + 4 h + c is hidden iff c >= lim
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[kb][i] = kb * 32 + (i & 3) + 8 * (i >> 2) >= lim ? -INFINITY : sc[kb][i];
  };
  // the running maximum takes in the largest of a lane's scores; l and O follow
  auto raise = [&](float mt) {
    {
      const unsigned mu = __builtin_bit_cast(unsigned, mt);
      const auto sw = __builtin_amdgcn_permlane32_swap(mu, mu, false, false);
      mt = fmaxf(__builtin_bit_cast(float, (unsigned)sw[0]), __builtin_bit_cast(float, (unsigned)sw[1]));
    }
    const float mc = fmaxf(m, mt * sl2);
    if (__builtin_expect(__any(mc > m + kDefer), 0)) {
      asm volatile("" ::: "memory");   // a branch, not selects: it is rare
      const float alpha = __builtin_amdgcn_exp2f(m - (mc == -INFINITY ? 0.f : mc));
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
      m = mc;
    }
  };
  auto largest = [&](const f32x16 (&sc)[2]) {
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx[i & 3] = fmaxf(mx[i & 3], sc[kb][i]);
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
  };
  auto v_frag = [&](int i, int dt) {   // 16 keys from 16 i, 32 columns from 32 dt
    const char* vr = smem + 16 * i * (D * 2);
    const s16x4 lo = lds_tr(vr, o_va ^ (dt << 6)), hi = lds_tr(vr, o_vb ^ (dt << 6));
    const s16x8 vv = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8, vv);
  };
  // The staging of a turn: V of the next tile, K of the one after it, and the pages of a later one are looked up.
  // Through registers V is loaded at the turn's start and stored at its middle, K loaded then and stored at its end; straight
  // to LDS both are loaded at the start and there at the end.
  auto stage_begin = [&](int n0) {
    stage.load(a.v, smem + 2 * TILE + (buf ^ TILE));
    if constexpr (UNI) {
      stage.locate(hk);
      stage.load(a.k, smem + buf);
      stage.pages(n0 + 3 * kStep);
    } else {
      stage.pages(n0 + 2 * kStep);
    }
  };
  auto stage_middle = [&](int n0, bool edge) {
    if constexpr (!UNI) {
      char* const dst = smem + 2 * TILE + (buf ^ TILE);
      if (edge) finite_only(n0 + kStep, dst);
      stage.store(dst);
      stage.locate(hk);
      stage.load(a.k, smem);
    }
  };
  auto stage_end = [&](int n0, bool edge) {
    stage.store(smem + buf);
    stage.arrived();
    if (UNI && edge) finite_only(n0 + kStep, smem + 2 * TILE + (buf ^ TILE));
    lds_barrier();
  };
  // the same in 2 * KS steps
  auto stage_step = [&](int i, int n0) {
    constexpr int N = KS, EVERY = N / NLOAD;   // V over the first KS steps, then K
    if (i < N && i % EVERY == 0) stage.load(i / EVERY, a.v, smem + 2 * TILE + (buf ^ TILE));
    if (i == N) stage.locate(hk);
    if (i >= N && i % EVERY == 0) stage.load((i - N) / EVERY, a.k, smem + buf);
    if (i == 2 * N - 1) stage.pages(n0 + 3 * kStep);
  };
  // One tile, whose scores are in cur, the next one's in nxt at the end.  EDGE: some row may not see all keys of the next
  // tile (two loops, one body each: with both in one loop O was copied between registers at their joint).
  // The order of the inner body is written down step by step: an LDS read for a later product, a product, and a share of
  // the exponentials or maxima, which take the time of the product.  Left to itself the compiler issues the 16 products
  // first and the 32 exponentials after them.
  auto tile_step = [&](auto EDGE_, int n0, f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
    constexpr bool EDGE = decltype(EDGE_)::value;
    asm volatile("" : "+v"(o_k), "+v"(o_va), "+v"(o_vb));   // the XORs stay in the loop: hoisted they spilled
    if constexpr (!UNI) stage_begin(n0);
    const int next = o_k + (buf ? -TILE : TILE);
    const float base = (m == -INFINITY ? 0.f : m) - kLift<F16>;
    float ls[4] = {0.f, 0.f, 0.f, 0.f};
    auto weight = [&](int i) {    // of the lane's score i
      float p = __builtin_amdgcn_exp2f(fmaf(cur[i >> 4][i & 15], sl2, -base));
      if constexpr (!EDGE) asm volatile("" : "+v"(p));   // (holds it to its step: scheduling barriers bind no arithmetic)
      cur[i >> 4][i & 15] = p;
      ls[i & 3] += p;
    };
    if constexpr (EDGE) {
      scores(nxt, next);
      if constexpr (UNI) stage_begin(n0);
#pragma unroll
      for (int i = 0; i < 32; ++i) weight(i);
    } else {
      constexpr int AHEAD = 3, N = 2 * KS;
      auto k_frag = [&](int i) {
        return *reinterpret_cast<const bf16x8*>(smem + (i / KS) * 32 * (D * 2) + (next ^ ((i % KS) << 5)));
      };
      bf16x8 f[AHEAD + 1];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) f[i] = k_frag(i);
      nxt[0] = f32x16{}, nxt[1] = f32x16{};
      // a wave in its exponentials goes first, the SIMD's other one has products between them (2,048 tokens over 30,720:
      // 975 us, without 1,029)
      __builtin_amdgcn_s_setprio(1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + AHEAD < N) f[(i + AHEAD) % (AHEAD + 1)] = k_frag(i + AHEAD);
        nxt[i / KS] = mfma<F16>(f[i % (AHEAD + 1)], qf[i % KS], nxt[i / KS]);
        if constexpr (UNI) stage_step(i, n0);
#pragma unroll
        for (int j = 32 * i / N; j < 32 * (i + 1) / N; ++j) weight(j);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (!EDGE) __builtin_amdgcn_s_setprio(0);
    l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    stage_middle(n0, EDGE);
    if constexpr (EDGE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 pb = pack8<F16>(cur[i >> 1], i & 1);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[dt] = mfma<F16>(v_frag(i, dt), pb, o[dt]);
      }
      hide(nxt, n0 + kStep);
      raise(largest(nxt));
    } else {
      constexpr int AHEAD = 2, N = 4 * DT;
      bf16x8 f[AHEAD + 1], pb[2];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) f[i] = v_frag(i / DT, i % DT);
      pb[0] = pack8<F16>(cur[0], 0);
      float mx[2] = {-INFINITY, -INFINITY};
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (i + AHEAD < N) f[(i + AHEAD) % (AHEAD + 1)] = v_frag((i + AHEAD) / DT, (i + AHEAD) % DT);
        o[i % DT] = mfma<F16>(f[i % (AHEAD + 1)], pb[i / DT & 1], o[i % DT]);
        if (i % DT == 0 && i / DT < 3) pb[i / DT + 1 & 1] = pack8<F16>(cur[(i / DT + 1) >> 1], (i / DT + 1) & 1);
#pragma unroll
        for (int j = 32 * i / N; j < 32 * (i + 1) / N; j += 2)
          mx[j >> 1 & 1] = fmaxf(fmaxf(mx[j >> 1 & 1], nxt[j >> 4][j & 15]), nxt[j >> 4][(j & 15) + 1]);
        asm volatile("" : "+v"(mx[0]), "+v"(mx[1]));
        __builtin_amdgcn_sched_barrier(0);
      }
      raise(fmaxf(mx[0], mx[1]));
    }
    stage_end(n0, EDGE);
  };
  auto stage_only = [&](int n0) {   // a wave with nothing to see helps to stage
    stage_begin(n0);
    stage_middle(n0, true);
    stage_end(n0, true);
  };
  auto turn = [&]() {
    const int d = buf ? -TILE : TILE;
    buf ^= TILE;
    o_k += d, o_va += d, o_vb += d;
  };
  // tiles that every row sees in full, and whose next one too; the same for every wave, as are all tiles' count: the
  // barriers are shared
  const int rounds = (ntiles + KG - 1) / KG, seen = (min(pos0 + 1, k1) - k0) / kBN;
  const int inner = max(0, min(rounds, seen / KG - 1));
  int n0 = kg, t = 0;
  if (wave_last < 0) {
    if (rounds > 0) lds_barrier();
    for (; t < rounds; ++t, n0 += kStep, turn()) stage_only(n0);
  } else if (rounds > 0) {
    f32x16 s0[2], s1[2];
    scores(s0, o_k);
    hide(s0, n0);
    raise(largest(s0));
    lds_barrier();   // the first K stage is read: it may be written
    for (; t + 2 <= inner; t += 2) {   // two a turn: the scores change places
      tile_step(std::false_type{}, n0, s0, s1);
      n0 += kStep, turn();
      tile_step(std::false_type{}, n0, s1, s0);
      n0 += kStep, turn();
    }
    for (; t < rounds; ++t, n0 += kStep, turn()) {
      if (n0 > wave_last || n0 >= k1) {
        stage_only(n0);
      } else {
        tile_step(std::true_type{}, n0, s0, s1);
        s0[0] = s1[0], s0[1] = s1[1];
      }
    }
  }

  if constexpr (KG == 2) {
    // group 1 hands its rows to the same lanes of group 0: m, l, then O register by register
    float* const x = reinterpret_cast<float*>(lds);
    if (group == 1) {
      x[tid] = m;
      x[256 + tid] = l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[(2 + dt * 16 + i) * 256 + tid] = o[dt][i];
    }
    lds_barrier();
    if (group == 1) return;
    const float m1 = x[tid], both = fmaxf(m, m1), base = both == -INFINITY ? 0.f : both;
    const float w0 = __builtin_amdgcn_exp2f(m - base), w1 = __builtin_amdgcn_exp2f(m1 - base);
    m = both;
    l = l * w0 + x[256 + tid] * w1;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] = o[dt][i] * w0 + x[(2 + dt * 16 + i) * 256 + tid] * w1;
  }

  if (__builtin_expect(odd_values, 0)) {
    // what finite_only took out comes back, for the rows that see it
    // (tiles whose last key lies past pos0; a tile begins at k0 + a multiple of kBN)
    for (int j = k0 + max(pos0 - k0, 0) / kBN * kBN; j < k1; ++j) {
      const int blk = block_of(a, j), page = stage.tab[blk];
      if ((unsigned)page >= (unsigned)a.num_blocks || !live || j > pos) continue;
      const unsigned short* vr = a.v + (long)page * a.s_blk + (unsigned)((j - blk * a.block) * a.s_tok + hk * a.s_head) + 4 * h;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned short w = vr[32 * dt + 8 * c + e];
            if ((w & kExp) == kExp) o[dt][4 * c + e] += F16 ? h2f(w) : bf2f(w);
          }
    }
  }

  // lane (row, half h) holds O[row][32 dt + 8 c + 4 h + e] in o[dt][4 c + e]
  l += __shfl_xor(l, 32, 64);
  if (whole) {
    const float inv = l != 0.f ? 1.f / l : 0.f;   // l is 0 only where a row saw no key; a NaN sum stays NaN
    if (live) {
      unsigned short* op = a.out + (long)(s.q0 + tok0 + rt) * a.so_tok + (long)rh * a.so_head + 4 * h;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
          u16x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = cvt16<F16>(o[dt][4 * c + e] * inv);
          *reinterpret_cast<u16x4*>(op + 32 * dt + 8 * c) = w;
        }
    }
  } else if (live) {
    const long pi = ((long)sp * a.T + s.q0 + tok0 + rt) * a.Hq + rh;
    float* po = a.part_o + pi * D + 4 * h;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        f32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = o[dt][4 * c + e];
        *reinterpret_cast<f32x4*>(po + 32 * dt + 8 * c) = w;
      }
    if (h == 0) {
      a.part_ml[pi * 2] = m;
      a.part_ml[pi * 2 + 1] = l;
    }
  }
}

// joins the pieces of every row that was split: grid (tokens, groups of heads), D / 4 lanes per query head
template <int D, bool F16>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  constexpr int LANES = D / 4, HEADS = 256 / LANES;
  const int tok = blockIdx.x, hq = blockIdx.y * HEADS + threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4;
  const int pieces = min(a.pieces[tok], a.splits);
  // (a row of no sequence has no count)
  if (tok < a.cu[0] || tok >= a.cu[a.B] || pieces <= 1 || hq >= a.Hq) return;
  float M = -INFINITY, L = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < pieces; p0 += 4) {   // four pieces' loads together; past the last one m is -inf
    float m[4], l[4];
    f32x4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long pi = ((long)min(p0 + i, pieces - 1) * a.T + tok) * a.Hq + hq;
      m[i] = a.part_ml[pi * 2];
      l[i] = a.part_ml[pi * 2 + 1];
      o[i] = *reinterpret_cast<const f32x4*>(a.part_o + pi * D + d);
    }
    float top = M;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p0 + i >= pieces) m[i] = -INFINITY;
      top = fmaxf(top, m[i]);
    }
    const float base = top == -INFINITY ? 0.f : top, w = __builtin_amdgcn_exp2f(M - base);
    L *= w;
    acc *= w;
    M = top;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p0 + i < pieces) {
        const float wi = __builtin_amdgcn_exp2f(m[i] - base);
        L += l[i] * wi;
        acc += o[i] * wi;
      }
  }
  const float inv = L != 0.f ? 1.f / L : 0.f;
  typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
  u16x4 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = cvt16<F16>(acc[e] * inv);
  *reinterpret_cast<u16x4*>(a.out + (long)tok * a.so_tok + (long)hq * a.so_head + d) = w;
}

}  // namespace ca
}  // namespace pd

using namespace pd;

// An upper bound of the batch's tiles of 16 or 128 rows: every sequence may end in a part of one
extern "C" long pd_chunk_attn_tiles(int T, int B, int G, int rows) {
  const int tt = rows / G, some = B < T ? B : T;
  return (T + (long)some * (tt - 1)) / tt;
}

// rows: of a tile, 16, or 128 and 16 for the sequences that have no more (one tile either way)
extern "C" int pd_chunk_attn(int f16, const void* q, long sq_tok, long sq_head, const void* k, const void* v, long s_blk,
                             long s_tok, long s_head, const int* table, int max_blocks, int num_blocks, int block,
                             const int* cu, const int* lens, void* out, long so_tok, long so_head, int B, int T, int Hq,
                             int Hk, int D, int rows, int groups, int splits, int min_keys, float scale,
                             float* part_o, float* part_ml, int* pieces, void* stream) {
  if (T <= 0 || B <= 0) return 0;
  if (Hk <= 0 || Hq % Hk || Hq / Hk > ca::kBM || block <= 0 || max_blocks <= 0 || num_blocks <= 0 || splits < 1 ||
      (rows != 16 && rows != 128) || Hq / Hk > rows || groups < 1 || groups > 2)
    return -1;
  if (splits > 1 && (!part_o || !part_ml || !pieces)) return -1;
  // a page's span in 32 bits (its number times s_blk is taken in 64)
  const long span = (long)(block - 1) * s_tok + (long)(Hk - 1) * s_head + D;
  if (s_blk < 0 || s_tok < 0 || s_head < 0 || s_blk > 0x7fffffffL || s_tok > 0x7fffffffL || s_head > 0x7fffffffL ||
      span > 0x7fffffffL)
    return -3;
  ca::Args a;
  a.q = (const unsigned short*)q;
  a.k = (const unsigned short*)k;
  a.v = (const unsigned short*)v;
  a.out = (unsigned short*)out;
  a.sq_tok = sq_tok, a.sq_head = sq_head, a.so_tok = so_tok, a.so_head = so_head;
  a.s_blk = (int)s_blk, a.s_tok = (int)s_tok, a.s_head = (int)s_head;
  a.cu = cu, a.lens = lens, a.table = table;
  a.B = B, a.T = T, a.Hq = Hq, a.Hk = Hk, a.G = Hq / Hk;
  a.max_blocks = max_blocks, a.num_blocks = num_blocks, a.block = block;
  // key / block as a product: m = ceil(2^(31 + L) / block), L = ceil(log2 block); the excess key * (m block - 2^(31 + L)) /
  // (block 2^(31 + L)) stays below 2^-L <= 1 / block for keys < 2^31
  int L = 0;
  while ((1L << L) < block) ++L;
  a.block_shift = block == 1 ? 0 : 31 + L;
  a.block_mul = block == 1 ? 1u : (unsigned)(((1UL << (31 + L)) + block - 1) / block);
  a.splits = splits, a.min_keys = min_keys < 1 ? 1 : min_keys;
  a.scale_log2 = scale * ca::kLog2e;
  a.part_o = part_o, a.part_ml = part_ml, a.pieces = pieces;
  const long wgs = pd_chunk_attn_tiles(T, B, a.G, rows) * Hk * splits;
  if (wgs > 0x7fffffffL) return -1;
  hipStream_t st = (hipStream_t)stream;
  // (a wave's load covers 512 / D rows: see Stage)
  const bool uni = block % (512 / D) == 0 && s_tok >= D && span + 8 * s_tok < 1L << 30;
#define PD_MANY(DV, F, U)                                                                   \
  do {                                                                                      \
    if (groups == 2) ca::chunk_kernel<DV, F, U, 2><<<(unsigned)wgs, 512, 0, st>>>(a);       \
    else ca::chunk_kernel<DV, F, U, 1><<<(unsigned)wgs, 256, 0, st>>>(a);                   \
  } while (0)
#define PD_FEW(DV, F)                                                                       \
  do {                                                                                      \
    if (groups == 2) ca::few_kernel<DV, F, 8><<<(unsigned)wgs, 512, 0, st>>>(a);            \
    else ca::few_kernel<DV, F, 4><<<(unsigned)wgs, 256, 0, st>>>(a);                        \
  } while (0)
#define PD_CHUNK(DV)                                                                        \
  do {                                                                                      \
    if (rows == 16 && f16) PD_FEW(DV, true);                                                \
    else if (rows == 16) PD_FEW(DV, false);                                                 \
    else if (f16 && uni) PD_MANY(DV, true, true);                                           \
    else if (f16) PD_MANY(DV, true, false);                                                 \
    else if (uni) PD_MANY(DV, false, true);                                                 \
    else PD_MANY(DV, false, false);                                                         \
    if (splits > 1) {                                                                       \
      const dim3 jg(T, (Hq * DV / 4 + 255) / 256);                                          \
      if (f16) ca::join_kernel<DV, true><<<jg, 256, 0, st>>>(a);                            \
      else ca::join_kernel<DV, false><<<jg, 256, 0, st>>>(a);                               \
    }                                                                                       \
  } while (0)
  if (D == 64) PD_CHUNK(64);
  else if (D == 128) PD_CHUNK(128);
  else return -2;
#undef PD_CHUNK
#undef PD_FEW
#undef PD_MANY
  return (int)hipGetLastError();
}
