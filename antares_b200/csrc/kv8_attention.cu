// Attention over the 8-bit paged KV cache (layout: kv8.cuh): row r of sequence s, at position pos0[s] + r, over the cache's
// positions 0 .. pos0[s] + r; query head h reads kv head h / (Hq / Hkv).  A row with no position to attend to gives zeros.
#include <math_constants.h>

#include "kv8.cuh"

namespace ab200 {


constexpr int KD_THREADS = 128, KD_WARPS = KD_THREADS / 32;

template <typename T>
struct AttendParams {
  Kv8Cache c;
  Kv8Rows r;
  const T *q;
  long q_stride;
  T *out;
  int Hq;
  float scale;
  int *status;
};

// A CTA per row and query head; a warp takes every fourth key, a lane four dims; running maximum and sum.
template <typename T>
__global__ void __launch_bounds__(KD_THREADS) kv8_attention_kernel(AttendParams<T> p) {
  __shared__ int seq_s;
  __shared__ float m_s[KD_WARPS], l_s[KD_WARPS], o_s[KD_WARPS][KV8_D];
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Kv8Rows &r = p.r;
  pdl_launch_dependents();
  pdl_wait();
  if (tid == 0) seq_s = r.cu ? -1 : row / r.n;
  __syncthreads();
  if (r.cu) {
    for (int s = tid; s < r.S; s += KD_THREADS)
      if (row >= r.begin(s) && row < r.end(s)) seq_s = s;
    __syncthreads();
  }
  const int s = seq_s;
  if (s < 0) return;
  const int hk = h / (p.Hq / p.c.H);
  const int limit = (int)max(0l, min((long)r.pos0[s] + row - r.begin(s) + 1, (long)r.max_pages << p.c.shift));
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -CUDART_INF_F, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = (float)p.q[(size_t)row * p.q_stride + (size_t)h * KV8_D + 4 * lane + i];
  for (int pos = warp; pos < limit; pos += KD_WARPS) {
    const long page = max(kv8_page(p.c, r, s, pos, p.status), 0l);
    const size_t at = (size_t)page * p.c.H + hk;
    const int in = pos & ((1 << p.c.shift) - 1);
    const size_t elt = ((at << p.c.shift) + in) * KV8_D + 4 * lane, blk = (at << (p.c.shift - 4)) + (in >> 4);
    const uint32_t kw = *reinterpret_cast<const uint32_t *>(p.c.k + elt), vw = *reinterpret_cast<const uint32_t *>(p.c.v + elt);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) dot = fmaf(q[i], (float)(int8_t)(kw >> (8 * i)), dot);
    dot = warp_sum(dot) * p.c.ks[blk] * p.scale;
    const float m_new = fmaxf(m, dot);
    const float f = expf(m - m_new), w = expf(dot - m_new), wv = w * p.c.vs[blk];
    l = fmaf(l, f, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(acc[i], f, wv * (float)(int8_t)(vw >> (8 * i)));
    m = m_new;
  }
  if (lane == 0) m_s[warp] = m, l_s[warp] = l;
#pragma unroll
  for (int i = 0; i < 4; ++i) o_s[warp][4 * lane + i] = acc[i];
  __syncthreads();
  float mx = -CUDART_INF_F, sum = 0.f, o = 0.f;
#pragma unroll
  for (int w = 0; w < KD_WARPS; ++w) mx = fmaxf(mx, m_s[w]);
#pragma unroll
  for (int w = 0; w < KD_WARPS; ++w) {
    const float f = m_s[w] == -CUDART_INF_F ? 0.f : expf(m_s[w] - mx);
    sum = fmaf(l_s[w], f, sum);
    o = fmaf(o_s[w][tid], f, o);
  }
  p.out[((size_t)row * p.Hq + h) * KV8_D + tid] = (T)(limit > 0 ? o / sum : 0.f);
}

template <typename T>
static int attend_launch(const Kv8Cache &c, const Kv8Rows &r, const void *q, long q_stride, void *out, int Hq, float scale, cudaStream_t stream) {
  AttendParams<T> p{c, r, (const T *)q, q_stride, (T *)out, Hq, scale, kernel_error_ptr()};
  AB200_CUDA(launch_pdl(kv8_attention_kernel<T>, dim3(r.T, Hq), dim3(KD_THREADS), 0, stream, p));
  return AB200_OK;
}

static int attention_check(const char *who, const Kv8Cache &c, int T, const void *q, long q_stride, const void *out, int Hq, int D, int dtype) {
  AB200_REQUIRE(dtype == AB200_F16 || dtype == AB200_F32, "%s: unknown dtype %d", who, dtype);
  if (D != KV8_D) return fail(AB200_EUNSUPPORTED, "%s: head size %d is not the built size %d", who, D, KV8_D);
  AB200_REQUIRE(Hq > 0 && Hq <= 65535 && Hq % c.H == 0, "%s: %d query heads are not a multiple of %d kv heads", who, Hq, c.H);
  if (T == 0) return AB200_OK;
  const long vec = dtype == AB200_F16 ? 8 : 4;
  AB200_REQUIRE(q && out && aligned16(q) && aligned16(out) && q_stride % vec == 0 && q_stride >= (long)Hq * D,
                "%s: q must be 16-byte aligned rows of at least %d values, a multiple of 16 bytes apart, and out 16-byte aligned", who, Hq * D);
  return AB200_OK;
}

}  // namespace ab200

using namespace ab200;

extern "C" size_t ab200_kv8_attention_workspace_bytes(int S, int T, int max_rows, int Hq, int Hkv) {
  (void)S, (void)T, (void)max_rows, (void)Hq, (void)Hkv;
  return 0;
}

extern "C" int ab200_kv8_attention(const void *q, long q_stride, void *out, const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale, int pages,
                                   int page_rows, int Hkv, const int32_t *page_table, long table_stride, int max_pages, const int32_t *pos0_dev, const int32_t *cu_rows_dev,
                                   int S, int T, int max_rows, int Hq, int D, float scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  int rc = kv8_check("kv8_attention", k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, cu_rows_dev, S, T, &c, &r);
  if (!rc) rc = attention_check("kv8_attention", c, T, q, q_stride, out, Hq, D, dtype);
  if (rc || S == 0 || T == 0) return rc;
  return dtype == AB200_F16 ? attend_launch<__half>(c, r, q, q_stride, out, Hq, scale, (cudaStream_t)stream)
                            : attend_launch<float>(c, r, q, q_stride, out, Hq, scale, (cudaStream_t)stream);
}

extern "C" int ab200_kv8_step(const void *q, const void *k, const void *v, long q_stride, long k_stride, long v_stride, void *out, void *k_cache, void *v_cache,
                              float *k_scale, float *v_scale, int pages, int page_rows, int Hkv, const int32_t *page_table, long table_stride, int max_pages,
                              const int32_t *pos0_dev, int S, int T, int Hq, int D, const float *inv_freq, float scale, int dtype, void *workspace, size_t workspace_bytes,
                              void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  int rc = kv8_check("kv8_step", k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, nullptr, S, T, &c, &r);
  if (!rc) rc = attention_check("kv8_step", c, T, q, q_stride, out, Hq, D, dtype);
  if (rc || S == 0 || T == 0) return rc;
  // the rotated queries wait in `out`: a row's are read before its result is stored
  rc = ab200_kv8_append(k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, nullptr, S, T, k, v, k_stride, v_stride,
                        inv_freq ? q : nullptr, q_stride, inv_freq ? out : nullptr, (long)Hq * D, Hq, inv_freq, dtype, stream);
  if (rc) return rc;
  return ab200_kv8_attention(inv_freq ? out : q, inv_freq ? (long)Hq * D : q_stride, out, k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride,
                             max_pages, pos0_dev, nullptr, S, T, T / S, Hq, D, scale, dtype, workspace, workspace_bytes, stream);
}
