// Writing rows into the 8-bit paged KV cache and reading them back (layout: kv8.cuh).  Both are streams: every element is
// read once and written once.
#include <math_constants.h>

#include "kv8.cuh"

namespace ab200 {

constexpr int KA_THREADS = 128, KA_HEADS = 4, KA_Q_HEADS = 8;
constexpr float KA_LEAST_SCALE = 0x1p-100f;  // below it a block is held as zeros: quotients stay clear of subnormal arithmetic

// The code of x at scale s: the quotient x / s rounded to the nearest, ties to even, as if it had all its digits.  `inv` is
// about 1 / s, so k is off by one at most; the two sums (each one rounding, so their signs are exact) say which side of the
// middle between two codes x lies on.
__device__ __forceinline__ int kv8_code(float x, float s, float inv) {
  if (!(fabsf(x) < CUDART_INF_F)) return x > 0.f ? 127 : x < 0.f ? -127 : 0;
  float k = rintf(x * inv);
  const float up = fmaf(-(k + 0.5f), s, x), down = fmaf(-(k - 0.5f), s, x);
  const bool odd = ((int)k & 1) != 0;
  if (up > 0.f || (up == 0.f && odd)) k += 1.f;
  else if (down < 0.f || (down == 0.f && odd)) k -= 1.f;
  return (int)fminf(fmaxf(k, -127.f), 127.f);
}
__device__ __forceinline__ uint32_t kv8_code4(const float (&x)[8], int at, float s, float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= (uint32_t)(kv8_code(x[at + i], s, inv) & 255) << (8 * i);
  return s == 0.f ? 0u : w;
}

// dims 4 sub .. 4 sub + 3 and 64 + the same of a row: a rotated pair is one thread's
__device__ __forceinline__ void ka_load(const __half *p, int sub, float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p + 64 * half + 4 * sub);
    const float2 a = __half22float2(u2h2(v.x)), b = __half22float2(u2h2(v.y));
    f[4 * half] = a.x, f[4 * half + 1] = a.y, f[4 * half + 2] = b.x, f[4 * half + 3] = b.y;
  }
}
__device__ __forceinline__ void ka_load(const float *p, int sub, float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float4 v = *reinterpret_cast<const float4 *>(p + 64 * half + 4 * sub);
    f[4 * half] = v.x, f[4 * half + 1] = v.y, f[4 * half + 2] = v.z, f[4 * half + 3] = v.w;
  }
}
__device__ __forceinline__ void ka_store(__half *p, int sub, const float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
    *reinterpret_cast<uint2 *>(p + 64 * half + 4 * sub) =
        make_uint2(h22u(__floats2half2_rn(f[4 * half], f[4 * half + 1])), h22u(__floats2half2_rn(f[4 * half + 2], f[4 * half + 3])));
}
__device__ __forceinline__ void ka_store(float *p, int sub, const float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) *reinterpret_cast<float4 *>(p + 64 * half + 4 * sub) = make_float4(f[4 * half], f[4 * half + 1], f[4 * half + 2], f[4 * half + 3]);
}

// Sines: fp16 rows turn with 32-bit ones.  fp32 rows with 64-bit ones: which of two codes a value next to their middle gets
// would otherwise go by the last bits of the rotation.
template <typename T> struct KaAngle { typedef float type; };
template <> struct KaAngle<float> { typedef double type; };
__device__ __forceinline__ void ka_sincos(float a, float *s, float *c) { sincosf(a, s, c); }
__device__ __forceinline__ void ka_sincos(float a, double *s, double *c) { sincos((double)a, s, c); }

template <typename A>
__device__ __forceinline__ void ka_turn(float (&f)[8], const A *sn, const A *cs, int sub) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const A s = sn[4 * sub + i], c = cs[4 * sub + i], x = f[i], y = f[4 + i];
    f[i] = (float)(x * c - y * s);
    f[4 + i] = (float)(y * c + x * s);
  }
}

template <typename T>
struct AppendParams {
  Kv8Cache c;
  Kv8Rows r;
  const T *k, *v, *q;
  T *q_out;
  long k_stride, v_stride, q_stride, q_out_stride;
  int Hq;
  const float *inv_freq;
  int slots_per_seq;  // cu == nullptr
  int kv_groups;
  int *status;
};

// Grid: x = slot, y = group of KA_HEADS kv heads, then groups of KA_Q_HEADS query heads.
// kv: a slot is a block of 16 positions that new rows of one sequence lie in.  Sequence s owns the slots from
// cu[s] / 16 + 2 s on: n rows touch at most (n + 14) / 16 + 1 blocks, and that many slots lie before the next sequence's.
// A warp takes a block of one head of K or of V: half a warp per row, 8 rows each, in registers: one pass for the largest
// value, then the codes.  Older rows of the block are only read and written when its scale grows.
// q: a slot is 16 consecutive rows.
template <typename T>
__global__ void __launch_bounds__(KA_THREADS) kv8_append_kernel(AppendParams<T> p) {
  typedef typename KaAngle<T>::type A;
  __shared__ A sn[KV8_BLOCK][KV8_D / 2], cs[KV8_BLOCK][KV8_D / 2];
  __shared__ int seq_s, row_seq[KV8_BLOCK];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane & 15, hw = lane >> 4;
  const Kv8Rows &r = p.r;
  pdl_launch_dependents();
  pdl_wait();

  if ((int)blockIdx.y >= p.kv_groups) {  // ---- rotate query rows
    const int row0 = blockIdx.x * KV8_BLOCK;
    if (row0 >= r.T) return;
    if (tid < KV8_BLOCK) row_seq[tid] = r.cu ? -1 : min((row0 + tid) / max(r.n, 1), r.S - 1);
    __syncthreads();
    if (r.cu) {
      for (int s = tid; s < r.S; s += KA_THREADS)
        for (int i = max(r.begin(s) - row0, 0), e = min(r.end(s) - row0, KV8_BLOCK); i < e; ++i) row_seq[i] = s;
      __syncthreads();
    }
    for (int i = tid; i < KV8_BLOCK * KV8_D / 2; i += KA_THREADS) {
      const int row = i >> 6, s = row_seq[row];
      if (row0 + row >= r.T || s < 0) continue;
      ka_sincos((float)(r.pos0[s] + row0 + row - r.begin(s)) * p.inv_freq[i & 63], &sn[row][i & 63], &cs[row][i & 63]);
    }
    __syncthreads();
    const int h0 = ((int)blockIdx.y - p.kv_groups) * KA_Q_HEADS;
    for (int i = tid >> 4; i < KV8_BLOCK * KA_Q_HEADS; i += KA_THREADS / 16) {
      const int row = i / KA_Q_HEADS, h = h0 + i % KA_Q_HEADS;
      if (row0 + row >= r.T || row_seq[row] < 0 || h >= p.Hq) continue;
      float f[8];
      ka_load(p.q + (size_t)(row0 + row) * p.q_stride + (size_t)h * KV8_D, sub, f);
      ka_turn(f, sn[row], cs[row], sub);
      ka_store(p.q_out + (size_t)(row0 + row) * p.q_out_stride + (size_t)h * KV8_D, sub, f);
    }
    return;
  }

  // ---- a block of K and V
  int s, slot;
  if (r.cu) {
    if (tid == 0) seq_s = -1;
    __syncthreads();
    for (int i = tid; i < r.S; i += KA_THREADS)
      if ((int)blockIdx.x >= (r.begin(i) >> 4) + 2 * i && (i + 1 == r.S || (int)blockIdx.x < (r.begin(i + 1) >> 4) + 2 * (i + 1))) seq_s = i;
    __syncthreads();
    s = seq_s;
    if (s < 0) return;
    slot = (int)blockIdx.x - (r.begin(s) >> 4) - 2 * s;
  } else {
    s = blockIdx.x / p.slots_per_seq;
    if (s >= r.S) return;
    slot = blockIdx.x % p.slots_per_seq;
  }
  const int row0 = r.begin(s), n = r.end(s) - row0;
  const long pos0 = r.pos0[s], first = max(pos0, 0l), last = min(pos0 + n, (long)r.max_pages << p.c.shift) - 1;  // positions that are stored
  const long block = (first >> 4) + slot;
  if (first > last || block > (last >> 4)) return;
  const int at = (int)(block << 4);  // the block's first position
  const int lo = (int)(max(first, (long)at) - at), hi = (int)(min(last, (long)at + 15) - at);  // its rows lo .. hi are new
  if (p.inv_freq) {
    for (int i = tid + lo * (KV8_D / 2); i < (hi + 1) * (KV8_D / 2); i += KA_THREADS)
      ka_sincos((float)(at + (i >> 6)) * p.inv_freq[i & 63], &sn[i >> 6][i & 63], &cs[i >> 6][i & 63]);
  }
  __syncthreads();
  const long page = kv8_page(p.c, r, s, at, tid == 0 ? p.status : nullptr);
  if (page < 0) return;
  const int in_page = at & ((1 << p.c.shift) - 1);
  const bool older = pos0 > at;  // rows before the new ones: they count for the scale
  for (int item = warp; item < 2 * KA_HEADS; item += KA_THREADS / 32) {
    const int h = blockIdx.y * KA_HEADS + (item >> 1);
    const bool is_v = item & 1;
    if (h >= p.c.H) break;
    const T *src = (is_v ? p.v + (size_t)h * KV8_D : p.k + (size_t)h * KV8_D);
    const long stride = is_v ? p.v_stride : p.k_stride;
    const size_t at_head = (size_t)page * p.c.H + h;
    int8_t *dst = (is_v ? p.c.v : p.c.k) + ((at_head << p.c.shift) + in_page) * KV8_D;
    float *scale = (is_v ? p.c.vs : p.c.ks) + (at_head << (p.c.shift - 4)) + (in_page >> 4);
    float f[8][8], most = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = 2 * j + hw;
      if (i >= lo && i <= hi) {
        ka_load(src + (size_t)(row0 + (at + i - pos0)) * stride, sub, f[j]);
        if (!is_v && p.inv_freq) ka_turn(f[j], sn[i], cs[i], sub);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[j][e]) < CUDART_INF_F ? fabsf(f[j][e]) : 0.f);
      }
    }
    most = warp_max(most);
    const float was = older ? *scale : 0.f;
    float now = most * (1.f / 127.f);
    now = now < KA_LEAST_SCALE ? 0.f : now;
    now = fmaxf(was, now);
    const float inv = now > 0.f ? __fdividef(1.f, now) : 0.f;
    __syncwarp();  // every lane has read the scale
    if (lane == 0) *scale = now;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = 2 * j + hw;
      uint32_t *d = reinterpret_cast<uint32_t *>(dst + i * KV8_D) + sub;
      if (i >= lo && i <= hi) {
        d[0] = kv8_code4(f[j], 0, now, inv);
        d[16] = kv8_code4(f[j], 4, now, inv);
      } else if (i < lo && older && now > was) {  // the values they stood for, at the new scale
        const uint32_t a = d[0], b = d[16];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[j][e] = (float)(int8_t)(a >> (8 * e)) * was, f[j][4 + e] = (float)(int8_t)(b >> (8 * e)) * was;
        d[0] = kv8_code4(f[j], 0, now, inv);
        d[16] = kv8_code4(f[j], 4, now, inv);
      }
    }
  }
}

// k_out, v_out [T][H][128] = the values at the rows' positions; a position outside the table reads as zeros.  A CTA takes
// 16 rows; a thread 16 codes at a time.
template <typename T>
__global__ void __launch_bounds__(KA_THREADS) kv8_read_kernel(Kv8Cache c, Kv8Rows r, T *k_out, T *v_out, int *status) {
  __shared__ int row_seq[KV8_BLOCK];
  __shared__ long row_at[KV8_BLOCK];  // page * H, or -1
  __shared__ int row_in[KV8_BLOCK];
  const int tid = threadIdx.x, row0 = blockIdx.x * KV8_BLOCK;
  pdl_launch_dependents();
  pdl_wait();
  if (tid < KV8_BLOCK) row_seq[tid] = r.cu || row0 + tid >= r.T ? -1 : (row0 + tid) / r.n;
  __syncthreads();
  if (r.cu) {
    for (int s = tid; s < r.S; s += KA_THREADS)
      for (int i = max(r.begin(s) - row0, 0), e = min(r.end(s) - row0, KV8_BLOCK); i < e; ++i) row_seq[i] = s;
    __syncthreads();
  }
  if (tid < KV8_BLOCK) {
    const int s = row_seq[tid];
    long at = -1;
    if (s >= 0) {
      const long pos = (long)r.pos0[s] + row0 + tid - r.begin(s);
      if (pos >= 0 && pos < (long)r.max_pages << c.shift) {
        const long page = kv8_page(c, r, s, (int)pos, blockIdx.y == 0 ? status : nullptr);
        at = page < 0 ? -1 : page * c.H;
        row_in[tid] = (int)pos & ((1 << c.shift) - 1);
      }
    }
    row_at[tid] = at;
  }
  __syncthreads();
  const int per_row = c.H * (KV8_D / 16), total = KV8_BLOCK * per_row;
  for (int i = blockIdx.y * KA_THREADS + tid; i < total; i += gridDim.y * KA_THREADS) {
    const int row = i / per_row, piece = i - row * per_row, h = piece >> 3;
    if (row_seq[row] < 0) continue;
    const long at = row_at[row];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      uint4 codes = make_uint4(0, 0, 0, 0);
      float f = 0.f;
      if (at >= 0) {
        codes = ldg_stream_v4((which ? c.v : c.k) + (((at + h) << c.shift) + row_in[row]) * KV8_D + (piece & 7) * 16);
        f = (which ? c.vs : c.ks)[((at + h) << (c.shift - 4)) + (row_in[row] >> 4)];
      }
      T *out = (which ? v_out : k_out) + ((size_t)(row0 + row) * per_row + piece) * 16;
      const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
      float x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3))) * f;
      if constexpr (sizeof(T) == 2) {
        uint32_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = h22u(__floats2half2_rn(x[2 * e], x[2 * e + 1]));
        reinterpret_cast<uint4 *>(out)[0] = make_uint4(u[0], u[1], u[2], u[3]);
        reinterpret_cast<uint4 *>(out)[1] = make_uint4(u[4], u[5], u[6], u[7]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) reinterpret_cast<float4 *>(out)[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
      }
    }
  }
}

template <typename T>
static int append_launch(const Kv8Cache &c, const Kv8Rows &r, const void *k, const void *v, long k_stride, long v_stride, const void *q, long q_stride, void *q_out,
                         long q_out_stride, int Hq, const float *inv_freq, cudaStream_t stream) {
  AppendParams<T> p{c, r, (const T *)k, (const T *)v, (const T *)q, (T *)q_out, k_stride, v_stride, q_stride, q_out_stride, Hq, inv_freq, (r.n + 14) / 16 + 1,
                    (c.H + KA_HEADS - 1) / KA_HEADS, kernel_error_ptr()};
  const long slots = r.cu ? (long)r.T / 16 + 2l * r.S : (long)r.S * p.slots_per_seq;
  const int q_groups = q ? (Hq + KA_Q_HEADS - 1) / KA_Q_HEADS : 0;
  const long x = q && (r.T + 15) / 16 > slots ? (r.T + 15) / 16 : slots;
  AB200_CUDA(launch_pdl(kv8_append_kernel<T>, dim3((unsigned)x, p.kv_groups + q_groups), dim3(KA_THREADS), 0, stream, p));
  return AB200_OK;
}

template <typename T>
static int read_launch(const Kv8Cache &c, const Kv8Rows &r, void *k_out, void *v_out, cudaStream_t stream) {
  const int chunks = (r.T + KV8_BLOCK - 1) / KV8_BLOCK, pieces = KV8_BLOCK * c.H * (KV8_D / 16);
  int y = (pieces + KA_THREADS * 4 - 1) / (KA_THREADS * 4);  // four pieces of K and of V a thread
  if (y > 65535) y = 65535;
  AB200_CUDA(launch_pdl(kv8_read_kernel<T>, dim3(chunks, y), dim3(KA_THREADS), 0, stream, c, r, (T *)k_out, (T *)v_out, kernel_error_ptr()));
  return AB200_OK;
}

}  // namespace ab200

using namespace ab200;

extern "C" int ab200_kv8_append(void *k_cache, void *v_cache, float *k_scale, float *v_scale, int pages, int page_rows, int Hkv, const int32_t *page_table,
                                long table_stride, int max_pages, const int32_t *pos0_dev, const int32_t *cu_rows_dev, int S, int T, const void *k, const void *v,
                                long k_stride, long v_stride, const void *q, long q_stride, void *q_out, long q_out_stride, int Hq, const float *inv_freq, int dtype,
                                void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  const int rc = kv8_check("kv8_append", k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, cu_rows_dev, S, T, &c, &r);
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
  if (dtype == AB200_F16) return append_launch<__half>(c, r, k, v, k_stride, v_stride, q, q_stride, q_out, q_out_stride, Hq, inv_freq, (cudaStream_t)stream);
  return append_launch<float>(c, r, k, v, k_stride, v_stride, q, q_stride, q_out, q_out_stride, Hq, inv_freq, (cudaStream_t)stream);
}

extern "C" int ab200_kv8_read(const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale, int pages, int page_rows, int Hkv,
                              const int32_t *page_table, long table_stride, int max_pages, const int32_t *pos0_dev, const int32_t *cu_rows_dev, int S, int T, void *k_out,
                              void *v_out, int dtype, void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  const int rc = kv8_check("kv8_read", k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, cu_rows_dev, S, T, &c, &r);
  if (rc) return rc;
  AB200_REQUIRE(dtype == AB200_F16 || dtype == AB200_F32, "kv8_read: unknown dtype %d", dtype);
  if (S == 0 || T == 0) return AB200_OK;
  AB200_REQUIRE(k_out && v_out && aligned16(k_out) && aligned16(v_out), "kv8_read: k_out and v_out must be 16-byte aligned");
  if (dtype == AB200_F16) return read_launch<__half>(c, r, k_out, v_out, (cudaStream_t)stream);
  return read_launch<float>(c, r, k_out, v_out, (cudaStream_t)stream);
}
