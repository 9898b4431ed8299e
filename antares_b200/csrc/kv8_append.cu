// Writing rows into the 8-bit paged KV cache and reading them back (layout: kv8.cuh).  Both are streams: every element is
// read once and written once, so DRAM is what they cannot do without.
//
// Append.  s = max(the block's scale if it holds rows before the new ones, max |x| / 127), code = x / s rounded to the nearest.
// 2000 rows of 32 heads, K, V and rotated queries: 82 MB in 23.3 us (3.5 TB/s; 17.2 us, 2.9 TB/s, without rotation and queries).
// Bound by the chain of loads of a short-lived CTA (whose rows, which page, the rows) and the instructions between: 64 registers
// and four CTAs an SM against 80 and three: 23.3 / 23.7 us; codes by a quotient of two bounds, repeated exactly where those differ: 31.
// Read.  The same rows: 49 MB in 8.7 us (5.7 TB/s): bound by memory.
#include <math_constants.h>

#include "kv8_quant.cuh"

namespace ab200 {

constexpr int KA_WARPS = 8, KA_THREADS = KA_WARPS * 32, KA_HEADS = KA_WARPS / 2, KA_Q_HEADS = 8;

template <typename T>
struct AppendParams {
  Kv8Cache c;
  Kv8Rows r;
  const T *k, *v, *q;
  T *q_out;
  long k_stride, v_stride, q_stride, q_out_stride;
  int Hq;
  const float *inv_freq;
  int zero_rest;
  int slots_per_seq;  // cu == nullptr
  int kv_groups;
  int beside;                // the kernel behind this one starts before it ends: what came before it has ended by then
  int *status;
};

// Whose the rows row0 .. row0 + N - 1 are (-1: nobody's) and at which positions, to shared memory.  A thread asks for all it may
// need of a sequence at once: one wait for memory, not three.
template <int N, int THREADS>
__device__ __forceinline__ void kv8_rows_of(const Kv8Rows &r, int row0, int (&row_seq)[N], long (&row_pos)[N]) {
  const int tid = threadIdx.x;
  if (tid < N) {
    const int row = row0 + tid;
    row_seq[tid] = -1;
    if (!r.cu && row < r.T) row_seq[tid] = row / r.n, row_pos[tid] = (long)r.pos0[row / r.n] + row % r.n;
  }
  __syncthreads();
  if (r.cu) {
    for (int s = tid; s < r.S; s += THREADS) {
      const int begin = r.begin(s), end = r.end(s);
      const long pos0 = r.pos0[s];
      for (int i = max(begin - row0, 0), e = min(end - row0, N); i < e; ++i) row_seq[i] = s, row_pos[i] = pos0 + row0 + i - begin;
    }
    __syncthreads();
  }
}

// Grid: x = slot, y = group of KA_HEADS kv heads, then groups of KA_Q_HEADS query heads.
// kv: a slot is a block of 16 positions that new rows of one sequence lie in.  Sequence s owns the slots from
// cu[s] / 16 + 2 s on: n rows touch at most (n + 14) / 16 + 1 blocks, and that many slots lie before the next sequence's.
// A warp takes a block of one head of K or of V: half a warp per row, 8 rows each, in registers: one pass for the largest
// value, then the codes.  Older rows of the block are only read and written when its scale grows.
// q: a slot is 16 consecutive rows.
// Rows are asked for before the sines are made.
template <typename T>
__global__ void __launch_bounds__(KA_THREADS, sizeof(T) == 2 ? 4 : 1) kv8_append_kernel(const __grid_constant__ AppendParams<T> p) {
  typedef typename KaAngle<T>::type A;
  __shared__ __align__(16) A sn[KV8_BLOCK][KV8_D / 2], cs[KV8_BLOCK][KV8_D / 2];
  __shared__ int seq_s, begin_s, end_s, row_seq[KV8_BLOCK];
  __shared__ long pos_s, row_pos[KV8_BLOCK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane & 15, hw = lane >> 4;
  const Kv8Rows &r = p.r;
  if (!p.beside) pdl_launch_dependents();
  pdl_wait();
  if (p.beside) pdl_launch_dependents();

  if ((int)blockIdx.y >= p.kv_groups) {  // ---- rotate query rows
    const int row0 = blockIdx.x * KV8_BLOCK;
    if (row0 >= r.T) return;
    kv8_rows_of<KV8_BLOCK, KA_THREADS>(r, row0, row_seq, row_pos);
    const int h0 = ((int)blockIdx.y - p.kv_groups) * KA_Q_HEADS;
    constexpr int EACH = KV8_BLOCK * KA_Q_HEADS / (KA_THREADS / 16);  // rows of heads that a half-warp has
    KaRaw<T> raw[EACH];
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const int i = (tid >> 4) + n * (KA_THREADS / 16), row = i / KA_Q_HEADS, h = h0 + i % KA_Q_HEADS;
      if (row0 + row < r.T && row_seq[row] >= 0 && h < p.Hq) ka_ask(p.q + (size_t)(row0 + row) * p.q_stride + (size_t)h * KV8_D, sub, raw[n]);
    }
    for (int i = tid; i < KV8_BLOCK * KV8_D / 2; i += KA_THREADS) {
      const int row = i >> 6;
      if (row_seq[row] >= 0) ka_sincos((float)(int)row_pos[row] * p.inv_freq[i & 63], &sn[row][i & 63], &cs[row][i & 63]);
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < EACH; ++n) {
      const int i = (tid >> 4) + n * (KA_THREADS / 16), row = i / KA_Q_HEADS, h = h0 + i % KA_Q_HEADS;
      if (row0 + row >= r.T || h >= p.Hq) continue;
      T *out = p.q_out + (size_t)(row0 + row) * p.q_out_stride + (size_t)h * KV8_D;
      if (row_seq[row] >= 0) {
        float f[8];
        ka_widen(raw[n], f);
        ka_turn(f, sn[row], cs[row], sub);
        ka_store(out, sub, f);
      } else if (p.zero_rest) {
        const float none[8] = {};
        ka_store(out, sub, none);
      }
    }
    return;
  }

  // ---- a block of K and V
  int s, slot, row0, n;
  long pos0;
  if (r.cu) {
    if (tid == 0) seq_s = -1;
    __syncthreads();
    for (int i = tid; i < r.S; i += KA_THREADS) {
      const int begin = r.begin(i), end = r.end(i), next = i + 1 < r.S ? r.begin(i + 1) : 0;
      const long pos = r.pos0[i];
      if ((int)blockIdx.x >= (begin >> 4) + 2 * i && (i + 1 == r.S || (int)blockIdx.x < (next >> 4) + 2 * (i + 1))) seq_s = i, begin_s = begin, end_s = end, pos_s = pos;
    }
    __syncthreads();
    s = seq_s;
    if (s < 0) return;
    row0 = begin_s, n = end_s - begin_s, pos0 = pos_s;
    slot = (int)blockIdx.x - (row0 >> 4) - 2 * s;
  } else {
    s = blockIdx.x / p.slots_per_seq;
    if (s >= r.S) return;
    slot = blockIdx.x % p.slots_per_seq;
    row0 = s * r.n, n = r.n, pos0 = r.pos0[s];
  }
  const long first = max(pos0, 0l), last = min(pos0 + n, (long)r.max_pages << p.c.shift) - 1;  // positions that are stored
  const long block = (first >> 4) + slot;
  if (first > last || block > (last >> 4)) return;
  const int at = (int)(block << 4);  // the block's first position
  const int lo = (int)(max(first, (long)at) - at), hi = (int)(min(last, (long)at + 15) - at);  // its rows lo .. hi are new
  const int h = blockIdx.y * KA_HEADS + (warp >> 1);
  const bool is_v = warp & 1, turn = !is_v && p.inv_freq != nullptr;
  KaRaw<T> raw[8];  // as they came: widened and rotated twice, for the largest value and for the codes, which costs less than
                    // the registers that 64 values a thread would take
  const bool whole = lo == 0 && hi == 15;
  if (h < p.c.H) {
    const long stride = is_v ? p.v_stride : p.k_stride;
    const T *src = (is_v ? p.v : p.k) + (size_t)h * KV8_D + (row0 + (at - pos0)) * stride;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = 2 * j + hw;
      if (whole || (i >= lo && i <= hi)) ka_ask(src + i * stride, sub, raw[j]);
    }
  }
  const long page = kv8_page(p.c, r, s, at, tid == 0 ? p.status : nullptr);
  if (p.inv_freq) {
    for (int i = tid + lo * (KV8_D / 2); i < (hi + 1) * (KV8_D / 2); i += KA_THREADS)
      ka_sincos((float)(at + (i >> 6)) * p.inv_freq[i & 63], &sn[i >> 6][i & 63], &cs[i >> 6][i & 63]);
  }
  __syncthreads();
  if (page < 0 || h >= p.c.H) return;
  const int in_page = at & ((1 << p.c.shift) - 1);
  const bool older = pos0 > at;  // rows before the new ones: they count for the scale
  const size_t at_head = (size_t)page * p.c.H + h;
  int8_t *dst = (is_v ? p.c.v : p.c.k) + ((at_head << p.c.shift) + in_page) * KV8_D;
  float *scale = (is_v ? p.c.vs : p.c.ks) + (at_head << (p.c.shift - 4)) + (in_page >> 4);
  const float was = older ? *scale : 0.f;
  auto row = [&](int j, float(&f)[8]) {
    ka_widen(raw[j], f);
    if (turn) ka_turn(f, sn[2 * j + hw], cs[2 * j + hw], sub);
  };
  float most = 0.f, odd = 0.f;  // the largest; not 0 if a value is not finite
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = 2 * j + hw;
    if (!whole && (i < lo || i > hi)) continue;
    float f[8];
    row(j, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e])), odd = fmaf(f[e], 0.f, odd);
  }
  const bool finite = odd == 0.f;
  if (!finite) {
    most = 0.f;
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      const int i = 2 * j + hw;
      if (i < lo || i > hi) continue;
      float f[8];
      ka_load((is_v ? p.v : p.k) + (size_t)h * KV8_D + (row0 + (at + i - pos0)) * (is_v ? p.v_stride : p.k_stride), sub, f);
      if (turn) ka_turn(f, sn[i], cs[i], sub);
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[e]) < CUDART_INF_F ? fabsf(f[e]) : 0.f);
    }
  }
  most = warp_max(most);
  float now = most * (1.f / 127.f);
  now = now < KA_LEAST_SCALE ? 0.f : now;
  now = fmaxf(was, now);
  const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
  const bool slow = !finite || now == 0.f;
  __syncwarp();  // every lane has read the scale
  if (lane == 0) *scale = now;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = 2 * j + hw;
    uint32_t *d = reinterpret_cast<uint32_t *>(dst + i * KV8_D) + sub;
    float f[8];
    if (whole || (i >= lo && i <= hi)) {
      row(j, f);
    } else if (i < lo && older && now > was) {  // the values they stood for, at the new scale
      const uint32_t a = d[0], b = d[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = (float)(int8_t)(a >> (8 * e)) * was, f[4 + e] = (float)(int8_t)(b >> (8 * e)) * was;
    } else {
      continue;
    }
    const uint2 w = kv8_codes(f, now, inv, slow);
    d[0] = w.x, d[16] = w.y;
  }
}

// k_out, v_out [T][H][128] = the values at the rows' positions; a position outside the table reads as zeros.  A CTA takes
// 8 rows, a thread 16 bytes of the result of each, K and V: 16 loads on their way at once.
constexpr int KR_ROWS = 8, KR_THREADS = 128;
template <typename T>
__global__ void __launch_bounds__(KR_THREADS) kv8_read_kernel(const __grid_constant__ Kv8Cache c, const __grid_constant__ Kv8Rows r, T *k_out, T *v_out, int zero_rest, int *status) {
  constexpr int EACH = 16 / sizeof(T);  // codes that a thread has of a row
  __shared__ int row_seq[KR_ROWS];
  __shared__ long row_pos[KR_ROWS], row_at[KR_ROWS];  // position; page * H, or -1
  __shared__ int row_in[KR_ROWS];
  const int tid = threadIdx.x, row0 = blockIdx.x * KR_ROWS;
  pdl_launch_dependents();
  pdl_wait();
  kv8_rows_of<KR_ROWS, KR_THREADS>(r, row0, row_seq, row_pos);
  if (tid < KR_ROWS) {
    const int s = row_seq[tid];
    long at = -1;
    if (s >= 0) {
      const long pos = row_pos[tid];
      if (pos >= 0 && pos < (long)r.max_pages << c.shift) {
        const long page = kv8_page(c, r, s, (int)pos, blockIdx.y == 0 ? status : nullptr);
        at = page < 0 ? -1 : page * c.H;
        row_in[tid] = (int)pos & ((1 << c.shift) - 1);
      }
    }
    row_at[tid] = at;
  }
  __syncthreads();
  const int per_row = c.H * (KV8_D / EACH), piece = blockIdx.y * KR_THREADS + tid;
  if (piece >= per_row) return;
  const int h = piece / (KV8_D / EACH), in_head = piece % (KV8_D / EACH) * EACH;
  uint2 w[KR_ROWS][2];
  float f[KR_ROWS][2];
#pragma unroll
  for (int i = 0; i < KR_ROWS; ++i) {
    const long at = row_at[i];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      w[i][which] = make_uint2(0, 0), f[i][which] = 0.f;
      if (at >= 0) {
        const int8_t *src = (which ? c.v : c.k) + (((at + h) << c.shift) + row_in[i]) * KV8_D + in_head;
        // not as read-only data: the append before may still run when this kernel starts
        if constexpr (EACH == 8) w[i][which] = __ldcg(reinterpret_cast<const uint2 *>(src));
        else w[i][which].x = __ldcg(reinterpret_cast<const uint32_t *>(src));
        f[i][which] = (which ? c.vs : c.ks)[((at + h) << (c.shift - 4)) + (row_in[i] >> 4)];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < KR_ROWS; ++i) {
    if (row0 + i >= r.T || (row_seq[i] < 0 && !zero_rest)) continue;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float x[8];
#pragma unroll
      for (int e = 0; e < EACH; ++e) x[e] = (float)(int8_t)((e < 4 ? w[i][which].x : w[i][which].y) >> (8 * (e & 3))) * f[i][which];
      T *out = (which ? v_out : k_out) + ((size_t)(row0 + i) * per_row + piece) * EACH;
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint4 *>(out) = make_uint4(h22u(__floats2half2_rn(x[0], x[1])), h22u(__floats2half2_rn(x[2], x[3])), h22u(__floats2half2_rn(x[4], x[5])),
                                                     h22u(__floats2half2_rn(x[6], x[7])));
      else
        *reinterpret_cast<float4 *>(out) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
}

template <typename T>
static int append_launch(const Kv8Cache &c, const Kv8Rows &r, const void *k, const void *v, long k_stride, long v_stride, const void *q, long q_stride, void *q_out,
                         long q_out_stride, int Hq, const float *inv_freq, int zero_rest, int beside, cudaStream_t stream) {
  AppendParams<T> p{c, r, (const T *)k, (const T *)v, (const T *)q, (T *)q_out, k_stride, v_stride, q_stride, q_out_stride, Hq, inv_freq, zero_rest, (r.n + 14) / 16 + 1,
                    (c.H + KA_HEADS - 1) / KA_HEADS, beside, kernel_error_ptr()};
  const long slots = r.cu ? (long)r.T / 16 + 2l * r.S : (long)r.S * p.slots_per_seq;
  const int q_groups = q ? (Hq + KA_Q_HEADS - 1) / KA_Q_HEADS : 0;
  const long x = q && (r.T + 15) / 16 > slots ? (r.T + 15) / 16 : slots;
  AB200_CUDA(launch_pdl(kv8_append_kernel<T>, dim3((unsigned)x, p.kv_groups + q_groups), dim3(KA_THREADS), 0, stream, p));
  return AB200_OK;
}

int kv8_append_beside(const Kv8Cache &c, const Kv8Rows &r, const void *k, const void *v, long k_stride, long v_stride, const float *inv_freq, int dtype, cudaStream_t stream) {
  if (dtype == AB200_F16) return append_launch<__half>(c, r, k, v, k_stride, v_stride, nullptr, 0, nullptr, 0, 0, inv_freq, 0, 1, stream);
  return append_launch<float>(c, r, k, v, k_stride, v_stride, nullptr, 0, nullptr, 0, 0, inv_freq, 0, 1, stream);
}

template <typename T>
static int read_launch(const Kv8Cache &c, const Kv8Rows &r, void *k_out, void *v_out, int zero_rest, cudaStream_t stream) {
  const int chunks = (r.T + KR_ROWS - 1) / KR_ROWS, pieces = c.H * (KV8_D * (int)sizeof(T) / 16);
  AB200_REQUIRE((pieces + KR_THREADS - 1) / KR_THREADS <= 65535, "kv8_read: %d heads are beyond the built limits", c.H);
  AB200_CUDA(launch_pdl(kv8_read_kernel<T>, dim3(chunks, (pieces + KR_THREADS - 1) / KR_THREADS), dim3(KR_THREADS), 0, stream, c, r, (T *)k_out, (T *)v_out, zero_rest,
                        kernel_error_ptr()));
  return AB200_OK;
}

}  // namespace ab200

using namespace ab200;

extern "C" int ab200_kv8_append(void *k_cache, void *v_cache, float *k_scale, float *v_scale, int pages, int page_rows, int Hkv, const int32_t *page_table,
                                long table_stride, int max_pages, const int32_t *pos0_dev, const int32_t *cu_rows_dev, int S, int T, const void *k, const void *v,
                                long k_stride, long v_stride, const void *q, long q_stride, void *q_out, long q_out_stride, int Hq, const float *inv_freq, int zero_rest,
                                int dtype, void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  const int rc = kv8_check("kv8_append", true, k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, cu_rows_dev, S, T, &c, &r);
  if (rc) return rc;
  AB200_REQUIRE(dtype == AB200_F16 || dtype == AB200_F32, "kv8_append: unknown dtype %d", dtype);
  if (S == 0 || T == 0) return AB200_OK;
  const long vec = dtype == AB200_F16 ? 8 : 4;
  AB200_REQUIRE(k && v && k_stride % vec == 0 && v_stride % vec == 0 && k_stride >= (long)Hkv * KV8_D && v_stride >= (long)Hkv * KV8_D && aligned16(k) && aligned16(v),
                "kv8_append: k and v must be 16-byte aligned rows of at least %d values, a multiple of 16 bytes apart", Hkv * KV8_D);
  AB200_REQUIRE((q == nullptr) == (q_out == nullptr), "kv8_append: q and q_out come together");
  if (q) {
    AB200_REQUIRE(inv_freq != nullptr, "kv8_append: q is only rotated (inv_freq is null)");
    AB200_REQUIRE(Hq > 0 && Hq <= 65535 && q_stride % vec == 0 && q_out_stride % vec == 0 && q_stride >= (long)Hq * KV8_D && q_out_stride >= (long)Hq * KV8_D && aligned16(q) &&
                      aligned16(q_out), "kv8_append: q and q_out must be 16-byte aligned rows of at least %d values, a multiple of 16 bytes apart", Hq * KV8_D);
  }
  if (dtype == AB200_F16) return append_launch<__half>(c, r, k, v, k_stride, v_stride, q, q_stride, q_out, q_out_stride, Hq, inv_freq, zero_rest, 0, (cudaStream_t)stream);
  return append_launch<float>(c, r, k, v, k_stride, v_stride, q, q_stride, q_out, q_out_stride, Hq, inv_freq, zero_rest, 0, (cudaStream_t)stream);
}

extern "C" int ab200_kv8_read(const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale, int pages, int page_rows, int Hkv,
                              const int32_t *page_table, long table_stride, int max_pages, const int32_t *pos0_dev, const int32_t *cu_rows_dev, int S, int T, void *k_out,
                              void *v_out, int zero_rest, int dtype, void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  const int rc = kv8_check("kv8_read", false, k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, cu_rows_dev, S, T, &c, &r);
  if (rc) return rc;
  AB200_REQUIRE(dtype == AB200_F16 || dtype == AB200_F32, "kv8_read: unknown dtype %d", dtype);
  if (S == 0 || T == 0) return AB200_OK;
  AB200_REQUIRE(k_out && v_out && aligned16(k_out) && aligned16(v_out), "kv8_read: k_out and v_out must be 16-byte aligned");
  if (dtype == AB200_F16) return read_launch<__half>(c, r, k_out, v_out, zero_rest, (cudaStream_t)stream);
  return read_launch<float>(c, r, k_out, v_out, zero_rest, (cudaStream_t)stream);
}
