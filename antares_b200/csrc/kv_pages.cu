// Copies of cache pages inside their buffers (a fork's copy on write, compaction), all layers and all buffers in one launch.
// Bound by memory: 24 pages of 16 rows, 2 x 32 layers of an fp16 cache of 32 heads, 403 MB read and written in 64.1 us, 6.3 TB/s
// (96 % of a whole-buffer copy's rate).  Four 16-byte loads a thread are on their way before the first store.
#include <vector>

#include "common.cuh"

namespace ab200 {

constexpr int KP_THREADS = 256, KP_BUFFERS = 8, KP_PAIRS = 400;
constexpr int KP_UNIT = 4 * KP_THREADS;  // vectors a CTA moves: four loads in flight a thread

struct PageBuffer {
  char *base;
  long layer_stride, page_stride;  // bytes
  long vectors;                    // of `width` bytes in a page
  int layers, width, units;        // units of KP_UNIT vectors in a page
};
// by value: the pairs are the host's, a captured launch keeps them
struct PageCopies {
  PageBuffer buf[KP_BUFFERS];
  int32_t src[KP_PAIRS], dst[KP_PAIRS];
};

template <typename V>
__device__ __forceinline__ void move_unit(char *to, const char *from, long v0, long vectors) {
  V x[4];
  const V *f = reinterpret_cast<const V *>(from);
  V *t = reinterpret_cast<V *>(to);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (v0 + i * KP_THREADS < vectors) x[i] = f[v0 + i * KP_THREADS];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (v0 + i * KP_THREADS < vectors) t[v0 + i * KP_THREADS] = x[i];
}

// Grid: x = unit of a page, y = pair, z = layer of a buffer.  Sources are no destinations (checked on the host), so the
// copies do not depend on one another.
__global__ void __launch_bounds__(KP_THREADS) kv_copy_pages_kernel(const __grid_constant__ PageCopies p) {
  int b = 0, layer = blockIdx.z;
  while (layer >= p.buf[b].layers) layer -= p.buf[b++].layers;
  const PageBuffer &f = p.buf[b];
  pdl_launch_dependents();
  pdl_wait();
  if ((int)blockIdx.x >= f.units) return;
  char *base = f.base + layer * f.layer_stride;
  const char *from = base + p.src[blockIdx.y] * f.page_stride;
  char *to = base + p.dst[blockIdx.y] * f.page_stride;
  const long v0 = (long)blockIdx.x * KP_UNIT + threadIdx.x;
  if (f.width == 16) move_unit<uint4>(to, from, v0, f.vectors);
  else if (f.width == 4) move_unit<uint32_t>(to, from, v0, f.vectors);
  else move_unit<uint8_t>(to, from, v0, f.vectors);
}

}  // namespace ab200

using namespace ab200;

extern "C" int ab200_kv_copy_pages(int buffers, void *const *base_host, const int *layers_host, const long *layer_stride_host, const long *page_stride_host,
                                   const long *page_bytes_host, int pages, const int32_t *src_host, const int32_t *dst_host, int n, void *stream) {
  clear_error();
  AB200_REQUIRE(buffers > 0 && buffers <= KP_BUFFERS, "kv_copy_pages: %d buffers, 1 to %d are built", buffers, KP_BUFFERS);
  AB200_REQUIRE(base_host && layers_host && layer_stride_host && page_stride_host && page_bytes_host && pages > 0 && n >= 0 && (n == 0 || (src_host && dst_host)),
                "kv_copy_pages: bad argument");
  // what a page is in this call: untouched, a source, a destination
  std::vector<unsigned char> is;
  try {
    is.assign(pages, 0);
  } catch (...) {
    return fail(AB200_EINVAL, "kv_copy_pages: no memory for %d pages' marks", pages);
  }
  for (int i = 0; i < n; ++i) {
    AB200_REQUIRE(src_host[i] >= 0 && src_host[i] < pages && dst_host[i] >= 0 && dst_host[i] < pages, "kv_copy_pages: pair %d, %d -> %d, lies outside the %d pages", i,
                  src_host[i], dst_host[i], pages);
    AB200_REQUIRE(!(is[dst_host[i]] & 2), "kv_copy_pages: page %d is a destination twice", dst_host[i]);
    is[src_host[i]] |= 1;
    is[dst_host[i]] |= 2;
  }
  for (int i = 0; i < n; ++i) AB200_REQUIRE(is[dst_host[i]] != 3, "kv_copy_pages: page %d is a source and a destination", dst_host[i]);
  PageCopies p = {};
  int z = 0, x = 1;
  for (int b = 0; b < buffers; ++b) {
    const long bytes = page_bytes_host[b], ps = page_stride_host[b], ls = layer_stride_host[b];
    AB200_REQUIRE(base_host[b] && layers_host[b] > 0 && bytes > 0 && ps >= bytes && ls >= 0, "kv_copy_pages: buffer %d: bad layout", b);
    const long all = (long)(uintptr_t)base_host[b] | bytes | ps | ls;
    PageBuffer &f = p.buf[b];
    f.width = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
    f.base = (char *)base_host[b], f.layer_stride = ls, f.page_stride = ps, f.layers = layers_host[b];
    f.vectors = bytes / f.width;
    const long units = (f.vectors + KP_UNIT - 1) / KP_UNIT;
    AB200_REQUIRE(units < 1l << 31, "kv_copy_pages: buffer %d: pages of %ld bytes are beyond the built limit", b, bytes);
    f.units = (int)units;
    z += f.layers;
    AB200_REQUIRE(f.layers <= 65535 && z <= 65535, "kv_copy_pages: more than 65535 layers");
    if (f.units > x) x = f.units;
  }
  for (int i0 = 0; i0 < n; i0 += KP_PAIRS) {
    const int m = n - i0 < KP_PAIRS ? n - i0 : KP_PAIRS;
    for (int i = 0; i < m; ++i) p.src[i] = src_host[i0 + i], p.dst[i] = dst_host[i0 + i];
    AB200_CUDA(launch_pdl(kv_copy_pages_kernel, dim3(x, m, z), dim3(KP_THREADS), 0, (cudaStream_t)stream, p));
  }
  return AB200_OK;
}
