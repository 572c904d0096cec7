// Copies of KV-cache pages, all layers in one launch.
//
// Page src[i] of every pool (K and V of every layer) is copied to page dst[i] of the same pool.  No source is a
// destination and no destination comes twice (the host checks both), so the copies are independent and nothing has
// to be ordered.  Bound by HBM: every page is read and written once.
//  * The pools' addresses and the page numbers travel as kernel arguments: a launch takes 128 pools and 360 pairs
//    (1,024 + 2,880 bytes of the 4 KB of arguments), so no table is uploaded and a captured graph owns its plan.
//  * One workgroup moves 16 KB (4 x 16 bytes a thread, all loads in flight before the first store): a single page of
//    64 tokens x 32 heads x 128 in 64 pools is 2,048 workgroups.
// Measured (64 pools, pages of 64 tokens x 32 heads x 128 in bf16, pages that no cache holds): one page 15.6 us, 4.3 TB/s (11.2
// when the same page is copied again and again, from the last-level cache); four 54.5, 4.9; sixteen 186, 5.8.
#include "common.h"

namespace pd {
namespace pages {

constexpr int kPools = 128, kPairs = 360;
struct Args {
  char* pool[kPools];
  int src[kPairs];
  int dst[kPairs];
  long page_bytes;     // bytes of one page
  long page_stride;    // bytes from one page to the next
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// V: the unit moved, 16 bytes where addresses and sizes allow, else 4 or 1
template <typename V>
__global__ __launch_bounds__(256) void copy_kernel(Args a) {
  char* const p = a.pool[blockIdx.z];
  const V* s = reinterpret_cast<const V*>(p + (long)a.src[blockIdx.y] * a.page_stride);
  V* d = reinterpret_cast<V*>(p + (long)a.dst[blockIdx.y] * a.page_stride);
  const long n = a.page_bytes / (long)sizeof(V);
  const long i0 = (long)blockIdx.x * 1024 + threadIdx.x;
  if ((long)blockIdx.x * 1024 + 1024 <= n) {
    const V r0 = s[i0], r1 = s[i0 + 256], r2 = s[i0 + 512], r3 = s[i0 + 768];
    d[i0] = r0;
    d[i0 + 256] = r1;
    d[i0 + 512] = r2;
    d[i0 + 768] = r3;
  } else {
    for (long i = i0; i < n; i += 256) d[i] = s[i];
  }
}

}  // namespace pages
}  // namespace pd

using namespace pd;

// pool: n_pools device addresses; src / dst: n page numbers, checked by the caller
extern "C" int pd_kv_copy(const uint64_t* pool, int n_pools, const int* src, const int* dst, int n, long page_bytes,
                          long page_stride, void* stream) {
  if (n_pools <= 0 || n <= 0 || page_bytes <= 0) return 0;
  pages::Args a;
  a.page_bytes = page_bytes;
  a.page_stride = page_stride;
  for (int p0 = 0; p0 < n_pools; p0 += pages::kPools) {
    const int np = n_pools - p0 < pages::kPools ? n_pools - p0 : pages::kPools;
    uint64_t low = (uint64_t)page_bytes | (uint64_t)page_stride;
    for (int i = 0; i < np; ++i) {
      a.pool[i] = reinterpret_cast<char*>(pool[p0 + i]);
      low |= pool[p0 + i];
    }
    const int unit = (low & 15) == 0 ? 16 : (low & 3) == 0 ? 4 : 1;
    const long gx = (page_bytes / unit + 1023) / 1024;
    if (gx > 0x7fffffffL) return -1;
    for (int c0 = 0; c0 < n; c0 += pages::kPairs) {
      const int nc = n - c0 < pages::kPairs ? n - c0 : pages::kPairs;
      for (int i = 0; i < nc; ++i) {
        a.src[i] = src[c0 + i];
        a.dst[i] = dst[c0 + i];
      }
      const dim3 grid((unsigned)gx, nc, np);
      hipStream_t st = (hipStream_t)stream;
      if (unit == 16) pages::copy_kernel<pages::u32x4><<<grid, 256, 0, st>>>(a);
      else if (unit == 4) pages::copy_kernel<unsigned><<<grid, 256, 0, st>>>(a);
      else pages::copy_kernel<unsigned char><<<grid, 256, 0, st>>>(a);
      const int rc = (int)hipGetLastError();
      if (rc) return rc;
    }
  }
  return 0;
}
