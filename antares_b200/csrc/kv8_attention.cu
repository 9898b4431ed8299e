// Attention over the 8-bit paged KV cache (layout: kv8.cuh): row r of sequence s, at position pos0[s] + r, over the cache's
// positions 0 .. pos0[s] + r; query head h reads kv head h / (Hq / Hkv).  A row with no position to attend to gives zeros.
//
// Mathematics.  K codes go to the tensor cores as the bytes they are, against queries cut into three bytes (23 bits of a
// row's largest value): q . k is an exact integer.  V codes are integers that fp16 holds exactly.  So nothing of the cache
// is rounded.  A block of 16 keys has one scale for K and one for V:
//   x  = (q . k_code) * scale log2(e) ks + log2(vs)          the exponent of p vs
//   P  = 2^(x - m)                                           at most 2^8, whatever the scales
//   O += P v_code,  l += sum P / vs,  result O / l
// so the V scale costs one addition where the maximum is subtracted anyway, and no product can leave fp16's range.  The
// maximum m is only raised when a score exceeds it by more than 2^8 (then O and l are rescaled).  P goes in as a pair of
// fp16 numbers, 22 bits.
#include <math_constants.h>

#include "kv8.cuh"

namespace ab200 {

constexpr int KD_WARPS = 4, KD_THREADS = KD_WARPS * 32, KD_STAGES = 4;
constexpr int KD_STAGE_BYTES = 2 * KV8_BLOCK * KV8_D;  // a block of K, a block of V
constexpr int KD_LEAST = 8;                            // blocks a CTA takes at least, two a warp
constexpr int KD_ITEM = 8;                             // what an item costs besides its blocks, in blocks
constexpr float KD_RAISE = 8.f, KD_P_EXP = 6.f;        // P is scaled by 2^6: its second half stays out of fp16's subnormals
constexpr float KD_LEAST_SCALE = 0x1p-100f;            // a V scale below it is a block of zeros

struct DecodeParams {
  Kv8Cache c;
  Kv8Rows r;
  const void *q;
  long q_stride;
  void *out;
  int Hq, group;
  float scale;               // times log2(e)
  const float *inv_freq;     // rotate the queries, or nullptr
  int few;                   // sequences with more rows than this (rows x group) are another kernel's
  float *partial;            // [CTAs][2][rows][128], then [CTAs][2][rows][2]: maximum, sum
  int4 *split;               // [CTAs]: what is begun in CTA c and ended in a later one: CTAs, first row, kv head | rows - 1 << 16 |
                             // rows with nothing to attend to << 20, first packed row
  int *status;
};

__device__ __forceinline__ uint32_t kd_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void kd_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kd_imma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kd_ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void kd_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float kd_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two of a word's four codes (flipped to 0 .. 255) as fp16: 1024 + u is the half 0x6400 | u, and 1152 less is exact.
template <int SEL>
__device__ __forceinline__ uint32_t kd_half2(uint32_t flipped) {
  return h22u(__hsub2(u2h2(__byte_perm(flipped, 0x64646464u, SEL)), u2h2(0x64806480u)));
}

// Query rows are packed: row j of a sequence is its token j / group, head j % group of the kv head's; ROWS of them are a tile.
// The blocks that tile t of sequence s attends to (one at least: a row with no key is written by the CTA that has it).
template <int ROWS>
__device__ __forceinline__ int kd_blocks(const DecodeParams &p, long pos0, int packed, int t) {
  const int last = min((t + 1) * ROWS, packed) - 1;
  const long limit = min(pos0 + last / p.group + 1, (long)p.r.max_pages << p.c.shift);
  return max(1, (int)((max(limit, 0l) + 15) >> 4));
}
template <int ROWS>
__device__ __forceinline__ long kd_weight(const DecodeParams &p, int s) {  // work of all tiles of sequence s, one kv head
  const int packed = max(0, p.r.end(s) - p.r.begin(s)) * p.group;
  if (packed == 0 || packed > p.few) return 0;
  const long pos0 = p.r.pos0[s];
  long w = 0;
  for (int t = 0; t * ROWS < packed; ++t) w += kd_blocks<ROWS>(p, pos0, packed, t) + KD_ITEM;
  return w;
}

// ROWS: packed query rows of a tile.  With 8, rows 8-15 of the tensor cores' tile carry second parts: the second byte of
// q, the second half of P; with 16, each part is a product of its own.
template <typename T, int ROWS>
__global__ void __launch_bounds__(KD_THREADS, ROWS == 8 ? 3 : 2) kv8_decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int NR = ROWS / 8;  // query rows a thread holds: lane / 4, and 8 more
  __shared__ float scales_s[KD_WARPS][KD_STAGES][2];
  __shared__ long scan_s[KD_WARPS];
  __shared__ long found_start;
  __shared__ int found_s;
  __shared__ float m_s[KD_WARPS][ROWS], l_s[KD_WARPS][ROWS];
  __shared__ uint32_t q_s[NR][3][8][32];  // bytes of the queries, as the lanes hold them
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j4 = lane & 3;
  const Kv8Rows &r = p.r;
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's share: w0 .. w1 - 1 of all work, ordered by sequence, kv head, tile, block
  long mine = 0;
  for (int s = tid; s < r.S; s += KD_THREADS) mine += kd_weight<ROWS>(p, s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) scan_s[warp] = mine;
  __syncthreads();
  long total = 0;
#pragma unroll
  for (int w = 0; w < KD_WARPS; ++w) total += scan_s[w];
  total *= p.c.H;
  const long per = max((total + gridDim.x - 1) / gridDim.x, (long)KD_LEAST);
  const long w0 = blockIdx.x * per, w1 = min(w0 + per, total);
  if (tid == 0) p.split[blockIdx.x] = make_int4(0, 0, 0, 0);
  if (w0 >= w1) return;
  long before = 0;
  for (int base = 0; base < r.S; base += KD_THREADS) {
    const int s = base + tid;
    const long w = s < r.S ? kd_weight<ROWS>(p, s) * p.c.H : 0;
    long incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) scan_s[warp] = incl;
    __syncthreads();
    long chunk = 0;
#pragma unroll
    for (int i = 0; i < KD_WARPS; ++i) {
      if (i < warp) incl += scan_s[i];
      chunk += scan_s[i];
    }
    const long start = before + incl - w;
    if (w0 >= start && w0 < start + w) found_s = s, found_start = start;
    before += chunk;
    if (before > w0) break;
  }
  __syncthreads();
  int s = found_s;
  long start = found_start;

  const uint32_t ring = kd_smem(smem) + warp * (KD_STAGES * KD_STAGE_BYTES);
  // 16-byte piece i * 32 + lane of a block: row i * 4 + lane / 8, and its place under the XOR of row and piece that ldmatrix wants
  const uint32_t put0 = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4), put1 = put0 ^ 64;
  const uint32_t k_at = (lane & 7) * 128 + (((lane >> 3) ^ (lane & 7)) << 4);                         // pieces 0-3; pieces 4-7: ^ 64
  const uint32_t v_row = 2048 + (lane & 15) * 128, v_sw = lane & 7, v_chunk = lane >> 4;
  const int8_t *const k_lane = p.c.k + lane * 16, *const v_lane = p.c.v + lane * 16;
  const float *const sc_lane = lane ? p.c.vs : p.c.ks;

  for (long w = w0; w < w1;) {
    // ---- the item that w lies in
    const int row0 = r.begin(s), rows = max(0, r.end(s) - row0) * p.group;
    const long pos0 = r.pos0[s], cap = (long)r.max_pages << p.c.shift, per_head = kd_weight<ROWS>(p, s);
    const int hk = (int)((w - start) / per_head);
    long at = (w - start) - hk * per_head;
    int t = 0, blocks = kd_blocks<ROWS>(p, pos0, rows, 0);
    while (at >= blocks + KD_ITEM) at -= blocks + KD_ITEM, blocks = kd_blocks<ROWS>(p, pos0, rows, ++t);
    const int first = t * ROWS, last = min(first + ROWS, rows) - 1;  // packed rows of the tile
    const long take = min(blocks + KD_ITEM - at, w1 - w);
    const int b0 = (int)max(0l, at - KD_ITEM), b1 = (int)max(0l, at + take - KD_ITEM);
    const long item = w - at;
    w += take;
    const int seq = s;
    if (w < w1) {  // the next sequence that has rows here
      long weight = per_head * p.c.H;
      while (w >= start + weight) start += weight, weight = kd_weight<ROWS>(p, ++s) * p.c.H;
    }
    if (b1 == 0) continue;  // ended before the item's first block
    auto limit_of = [&](int packed) { return (int)max(0l, min(pos0 + packed / p.group + 1, cap)); };
    const int full = limit_of(first), any = limit_of(last);  // keys that every row, that some row attends to

    // ---- this warp's blocks: b0 + warp, + 4, ...
    const int live = min(b1, (any + 15) >> 4);  // blocks that hold a key
    const int count = max(0, (live - b0 - warp + KD_WARPS - 1) / KD_WARPS);
    const int32_t *row_table = r.table + (size_t)seq * r.table_stride;
    int where = 0, put = 0, asked = 0;
    auto issue = [&]() {
      if (asked < count) {
        if ((asked & 31) == 0 && asked + lane < count) {  // where the next 32 blocks lie, one a lane
          const int b = b0 + warp + (asked + lane) * KD_WARPS;
          int page = row_table[b >> (p.c.shift - 4)];
          if ((unsigned)page >= (unsigned)p.c.pages) {
            atomicExch(p.status, KV8_BAD_PAGE);
            page = 0;
          }
          where = ((page * p.c.H + hk) << (p.c.shift - 4)) + (b & ((1 << (p.c.shift - 4)) - 1));
        }
        const int blk = __shfl_sync(0xffffffffu, where, asked & 31);
        const int8_t *kp = k_lane + (size_t)blk * (KV8_BLOCK * KV8_D), *vp = v_lane + (size_t)blk * (KV8_BLOCK * KV8_D);
        const uint32_t to = ring + put * KD_STAGE_BYTES;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + n * 512 + (n & 1 ? put1 : put0)), "l"(kp + n * 512) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 2048 + n * 512 + (n & 1 ? put1 : put0)), "l"(vp + n * 512) : "memory");
        }
        if (lane < 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(kd_smem(&scales_s[warp][put][lane])), "l"(sc_lane + blk) : "memory");
        ++asked;
        put = put == KD_STAGES - 1 ? 0 : put + 1;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < KD_STAGES - 1; ++i) issue();

    // ---- queries, meanwhile.  A warp takes the pieces warp and warp + 4 (a rotated pair is one thread's): thread's row(s),
    // dims 16 c + 4 j4 .. + 3.  Each row is scaled by a power of two, its largest to 2^21 .. 2^22, rounded to an integer
    // and cut into three signed bytes (the first is 64 at most): half a step is 2^-22 of the largest, and fp16 rows are
    // exact unless they span more than 11 octaves.
    float f[NR][2][4], back[NR];
    int limit[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int packed = first + 8 * n + g;
      const bool in = packed <= last;
      limit[n] = in ? limit_of(packed) : 0x7fffffff;
      const int token = in ? packed / p.group : 0, head = hk * p.group + (in ? packed - token * p.group : 0);
      const T *q = (const T *)p.q + (size_t)(row0 + token) * p.q_stride + (size_t)head * KV8_D + 16 * warp + 4 * j4;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if constexpr (sizeof(T) == 2) {
          const uint2 v = in ? *reinterpret_cast<const uint2 *>(q + 64 * c) : make_uint2(0, 0);
          const float2 a = __half22float2(u2h2(v.x)), b = __half22float2(u2h2(v.y));
          f[n][c][0] = a.x, f[n][c][1] = a.y, f[n][c][2] = b.x, f[n][c][3] = b.y;
        } else {
          const float4 v = in ? *reinterpret_cast<const float4 *>(q + 64 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
          f[n][c][0] = v.x, f[n][c][1] = v.y, f[n][c][2] = v.z, f[n][c][3] = v.w;
        }
      }
      if (p.inv_freq) {
        const float pos = (float)(int)(pos0 + token);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float sn, cs;
          sincosf(pos * p.inv_freq[16 * warp + 4 * j4 + e], &sn, &cs);
          const float a = f[n][0][e], b = f[n][1][e];
          f[n][0][e] = a * cs - b * sn;
          f[n][1][e] = b * cs + a * sn;
        }
      }
      // a row that is not finite is made of NaN: its largest, as a bit pattern, is above that of every number
      uint32_t most = 0;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max(most, __float_as_uint(f[n][c][e]) & 0x7fffffffu);
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      if (j4 == 0) m_s[warp][8 * n + g] = __uint_as_float(most);
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < KD_WARPS; ++i) most = max(most, __float_as_uint(m_s[i][8 * n + g]));
      const int e = max(-100, min(100, 21 - (int)(most >> 23) + 127));
      const float up = __int_as_float((127 + e) << 23);
      back[n] = most >= 0x7f800000u ? CUDART_NAN_F : __int_as_float((127 - e) << 23);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t part[3] = {0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          int v = __float2int_rn(f[n][c][i] * up);
#pragma unroll
          for (int k = 2; k > 0; --k) {
            const int low = (int)(int8_t)v;
            part[k] |= (uint32_t)(low & 255) << (8 * i);
            v = (v - low) >> 8;
          }
          part[0] |= (uint32_t)(v & 255) << (8 * i);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) q_s[n][k][warp + 4 * c][lane] = part[k];
      }
    }
    __syncthreads();
    uint32_t qa[NR][3][8];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int c = 0; c < 8; ++c) qa[n][k][c] = q_s[n][k][c][lane];
    float o[16][4], m[NR], l[NR];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
#pragma unroll
    for (int n = 0; n < NR; ++n) m[n] = -CUDART_INF_F, l[n] = 0.f;

    int get = 0, key0 = (b0 + warp) * 16;
    for (int i = 0; i < count; ++i, key0 += 16 * KD_WARPS) {
      asm volatile("cp.async.wait_group %0;" ::"n"(KD_STAGES - 2) : "memory");
      __syncwarp();  // every lane's pieces have landed, and everyone is done with the stage that is filled next
      issue();
      const uint32_t st = ring + get * KD_STAGE_BYTES;
      const float ks = scales_s[warp][get][0] * p.scale, vs = scales_s[warp][get][1];
      get = get == KD_STAGES - 1 ? 0 : get + 1;
      const bool zero = !(vs >= KD_LEAST_SCALE);
      const float lvs = zero ? 0.f : __log2f(vs), inv_vs = zero ? 1.f : __fdividef(1.f, vs);
      // q . k: bytes times bytes, exact; thread's rows, keys 8 hb + 2 j4, + 1
      float x[NR][4];
#pragma unroll
      for (int hb = 0; hb < 2; ++hb) {
        int a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0}, c[4] = {0, 0, 0, 0};
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t k[4];
          kd_ldsm(k, st + hb * 1024 + (cc ? k_at ^ 64 : k_at));
#pragma unroll
          for (int d = 0; d < 4; d += 2) {
            const int ch = 4 * cc + d;
            if constexpr (ROWS == 8) {
              kd_imma(a, qa[0][0][ch], qa[0][1][ch], qa[0][0][ch + 1], qa[0][1][ch + 1], k[d], k[d + 1]);
              kd_imma(b, qa[0][2][ch], 0u, qa[0][2][ch + 1], 0u, k[d], k[d + 1]);
            } else {
              kd_imma(a, qa[0][0][ch], qa[NR - 1][0][ch], qa[0][0][ch + 1], qa[NR - 1][0][ch + 1], k[d], k[d + 1]);
              kd_imma(b, qa[0][1][ch], qa[NR - 1][1][ch], qa[0][1][ch + 1], qa[NR - 1][1][ch + 1], k[d], k[d + 1]);
              kd_imma(c, qa[0][2][ch], qa[NR - 1][2][ch], qa[0][2][ch + 1], qa[NR - 1][2][ch + 1], k[d], k[d + 1]);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if constexpr (ROWS == 8) {
            x[0][2 * hb + e] = fmaf((float)a[e], 65536.f, fmaf((float)a[2 + e], 256.f, (float)b[e]));
          } else {
#pragma unroll
            for (int n = 0; n < NR; ++n) x[n][2 * hb + e] = fmaf((float)a[2 * n + e], 65536.f, fmaf((float)b[2 * n + e], 256.f, (float)c[2 * n + e]));
          }
        }
      }
      // exponents of p vs
      bool raise = false;
      float top[NR];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float f = ks * back[n];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[n][e] = fmaf(x[n][e], f, lvs);
      }
      if (key0 + 16 > full) {  // the same for the whole warp
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key0 + 8 * (e >> 1) + 2 * j4 + (e & 1) >= limit[n]) x[n][e] = -CUDART_INF_F;
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        top[n] = fmaxf(fmaxf(x[n][0], x[n][1]), fmaxf(x[n][2], x[n][3]));
        raise = raise || top[n] > m[n] + KD_RAISE;
      }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], 1));
          top[n] = fmaxf(top[n], __shfl_xor_sync(0xffffffffu, top[n], 2));
          // a row's maximum moves by its own scores alone
          const float up = top[n] > m[n] + KD_RAISE ? top[n] : m[n], f = m[n] == up ? 1.f : m[n] == -CUDART_INF_F ? 0.f : kd_ex2(m[n] - up);
          m[n] = up;
          l[n] *= f;
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            o[d][2 * n] *= f, o[d][2 * n + 1] *= f;
            if constexpr (ROWS == 8) o[d][2] *= f, o[d][3] *= f;
          }
        }
      }
      uint32_t ph[NR][2], pl[NR][2];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float shift = m[n] == -CUDART_INF_F ? 0.f : m[n] - KD_P_EXP;
        float sum = 0.f;
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
          const float a = kd_ex2(x[n][2 * hb] - shift), b = kd_ex2(x[n][2 * hb + 1] - shift);
          sum += a + b;
          const __half2 hi = __floats2half2_rn(a, b);
          const float2 hf = __half22float2(hi);
          ph[n][hb] = h22u(hi);
          pl[n][hb] = h22u(__floats2half2_rn(a - hf.x, b - hf.y));
        }
        l[n] = fmaf(sum, inv_vs, l[n]);
      }
      if (!zero) {
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
          uint32_t v[4];
          // keys 0-7 and 8-15 of piece c, then of piece c + 1; transposed: two keys, two dims a word
          kd_ldsm_t(v, st + v_row + (((c + v_chunk) ^ v_sw) << 4));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t u0 = v[2 * h] ^ 0x80808080u, u1 = v[2 * h + 1] ^ 0x80808080u;
            const uint32_t e0 = kd_half2<0x4240>(u0), e1 = kd_half2<0x4240>(u1), d0 = kd_half2<0x4341>(u0), d1 = kd_half2<0x4341>(u1);
            float(&even)[4] = o[2 * (c + h)];
            float(&odd)[4] = o[2 * (c + h) + 1];
            if constexpr (ROWS == 8) {
              kd_mma(even, ph[0][0], pl[0][0], ph[0][1], pl[0][1], e0, e1);
              kd_mma(odd, ph[0][0], pl[0][0], ph[0][1], pl[0][1], d0, d1);
            } else {
              kd_mma(even, ph[0][0], ph[NR - 1][0], ph[0][1], ph[NR - 1][1], e0, e1);
              kd_mma(odd, ph[0][0], ph[NR - 1][0], ph[0][1], ph[NR - 1][1], d0, d1);
              kd_mma(even, pl[0][0], pl[NR - 1][0], pl[0][1], pl[NR - 1][1], e0, e1);
              kd_mma(odd, pl[0][0], pl[NR - 1][0], pl[0][1], pl[NR - 1][1], d0, d1);
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // ---- the four warps' parts to shared memory (the ring is idle), then joined
    __syncthreads();
    float *part = reinterpret_cast<float *>(smem);  // [warp][ROWS][128]
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
      if (j4 == 0) m_s[warp][8 * n + g] = m[n], l_s[warp][8 * n + g] = l[n];
#pragma unroll
      for (int c = 0; c < 8; ++c) {  // thread's dims of piece c: 16 c + 4 j4 + 0 .. 3
        float4 v;
        if constexpr (ROWS == 8)
          v = make_float4(o[2 * c][0] + o[2 * c][2], o[2 * c + 1][0] + o[2 * c + 1][2], o[2 * c][1] + o[2 * c][3], o[2 * c + 1][1] + o[2 * c + 1][3]);
        else
          v = make_float4(o[2 * c][2 * n], o[2 * c + 1][2 * n], o[2 * c][2 * n + 1], o[2 * c + 1][2 * n + 1]);
        *reinterpret_cast<float4 *>(part + ((warp * ROWS + 8 * n + g) * KV8_D + 16 * c + 4 * j4)) = v;
      }
    }
    __syncthreads();
    const bool whole = b0 == 0 && b1 == blocks;
    const int empty = (int)max(0l, min((long)ROWS, -pos0 * p.group - first));  // leading rows with nothing to attend to
    const int slot = b0 == 0 ? 1 : 0;
    float *mine_o = p.partial + ((size_t)blockIdx.x * 2 + slot) * ROWS * KV8_D;
    float *mine_ml = p.partial + (size_t)gridDim.x * 2 * ROWS * KV8_D + ((size_t)blockIdx.x * 2 + slot) * ROWS * 2;
    for (int row = 0; row <= last - first; ++row) {
      float mx = -CUDART_INF_F, sum = 0.f, acc = 0.f;
#pragma unroll
      for (int i = 0; i < KD_WARPS; ++i) mx = fmaxf(mx, m_s[i][row]);
#pragma unroll
      for (int i = 0; i < KD_WARPS; ++i) {
        const float f = m_s[i][row] == -CUDART_INF_F ? 0.f : kd_ex2(m_s[i][row] - mx);
        sum = fmaf(l_s[i][row], f, sum);
        acc = fmaf(part[(i * ROWS + row) * KV8_D + tid], f, acc);
      }
      if (whole) {
        const int packed = first + row, token = packed / p.group, head = hk * p.group + packed - token * p.group;
        ((T *)p.out)[((size_t)(row0 + token) * p.Hq + head) * KV8_D + tid] = (T)(row < empty ? 0.f : acc / sum);
      } else {
        mine_o[row * KV8_D + tid] = acc;
        if (tid == 0) mine_ml[2 * row] = mx, mine_ml[2 * row + 1] = sum;
      }
    }
    if (!whole && slot == 1 && tid == 0)  // begun here: the CTAs up to the one with the item's last block have the rest
      p.split[blockIdx.x] = make_int4((int)((item + KD_ITEM + blocks - 1) / per) - (int)blockIdx.x + 1, row0, hk | (last - first) << 16 | empty << 20, first);
    __syncthreads();
  }
}

// Joins the parts of the items that several CTAs share.  A CTA per CTA of the first kernel and four rows; two warps a row,
// each every second part.
constexpr int KJ_ROWS = 4, KJ_THREADS = KJ_ROWS * 64;
template <typename T, int ROWS>
__global__ void __launch_bounds__(KJ_THREADS) kv8_join_kernel(const __grid_constant__ DecodeParams p) {
  __shared__ float4 acc_s[KJ_ROWS][32];
  __shared__ float m_s[KJ_ROWS], l_s[KJ_ROWS];
  pdl_launch_dependents();
  pdl_wait();
  const int4 split = p.split[blockIdx.x];
  const int lane = threadIdx.x & 31, sub = (threadIdx.x >> 5) & 1, i = threadIdx.x >> 6, row = blockIdx.y * KJ_ROWS + i;
  const int n = split.x, first = split.w, more = split.z >> 16 & 15, empty = split.z >> 20, hk = split.z & 0xFFFF;
  if (n == 0) return;
  const bool in = row <= more;
  float m = -CUDART_INF_F, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (in) {
    const float *ml = p.partial + (size_t)gridDim.x * 2 * ROWS * KV8_D;
#pragma unroll 4
    for (int c = sub; c < n; c += 2) {
      const size_t at = ((size_t)(blockIdx.x + c) * 2 + (c == 0 ? 1 : 0)) * ROWS + row;
      const float mc = ml[2 * at], lc = ml[2 * at + 1];
      const float4 v = *reinterpret_cast<const float4 *>(p.partial + at * KV8_D + 4 * lane);
      const float up = fmaxf(m, mc), f = m == -CUDART_INF_F ? 0.f : kd_ex2(m - up), fc = mc == -CUDART_INF_F ? 0.f : kd_ex2(mc - up);
      l = l * f + lc * fc;
      acc.x = acc.x * f + v.x * fc, acc.y = acc.y * f + v.y * fc, acc.z = acc.z * f + v.z * fc, acc.w = acc.w * f + v.w * fc;
      m = up;
    }
    if (sub == 1) {
      acc_s[i][lane] = acc;
      if (lane == 0) m_s[i] = m, l_s[i] = l;
    }
  }
  __syncthreads();
  if (!in || sub == 1) return;
  const float mc = m_s[i], lc = l_s[i], up = fmaxf(m, mc), f = m == -CUDART_INF_F ? 0.f : kd_ex2(m - up), fc = mc == -CUDART_INF_F ? 0.f : kd_ex2(mc - up);
  const float4 v = acc_s[i][lane];
  const float sum = l * f + lc * fc;
  const int packed = first + row, token = packed / p.group, head = hk * p.group + packed - token * p.group;
  T *out = (T *)p.out + ((size_t)(split.y + token) * p.Hq + head) * KV8_D + 4 * lane;
  const float x[4] = {(acc.x * f + v.x * fc) / sum, (acc.y * f + v.y * fc) / sum, (acc.z * f + v.z * fc) / sum, (acc.w * f + v.w * fc) / sum};
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(row < empty ? 0.f : x[e]);
}

// ---- host --------------------------------------------------------------------------------------------------------
struct DecodePlan {
  int rows, ctas;
  size_t partial_bytes, bytes;
};
static DecodePlan decode_plan(int S, int T, int max_rows, int Hq, int Hkv) {
  DecodePlan d;
  const long group = Hq / Hkv;
  d.rows = (long)max_rows * group <= 8 ? 8 : 16;
  d.ctas = sm_count() * (d.rows == 8 ? 3 : 2);
  d.partial_bytes = (size_t)d.ctas * 2 * d.rows * (KV8_D + 2) * sizeof(float);
  d.bytes = d.partial_bytes + (size_t)d.ctas * sizeof(int4);
  return d;
}

template <typename T, int ROWS>
static int decode_launch(const DecodeParams &p, const DecodePlan &d, cudaStream_t stream) {
  constexpr int smem = KD_WARPS * KD_STAGES * KD_STAGE_BYTES;
  static_assert(smem >= KD_WARPS * ROWS * KV8_D * (int)sizeof(float), "the warps' parts fit into the ring");
  AB200_CUDA(cudaFuncSetAttribute(kv8_decode_kernel<T, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  AB200_CUDA(launch_pdl(kv8_decode_kernel<T, ROWS>, dim3(d.ctas), dim3(KD_THREADS), smem, stream, p));
  AB200_CUDA(launch_pdl(kv8_join_kernel<T, ROWS>, dim3(d.ctas, ROWS / KJ_ROWS), dim3(KJ_THREADS), 0, stream, p));
  return AB200_OK;
}

static int attend(const char *who, const Kv8Cache &c, const Kv8Rows &r, const void *q, long q_stride, void *out, int max_rows, int Hq, int D, float scale, int dtype,
                  const float *inv_freq, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (r.T == 0 || r.S == 0) return AB200_OK;
  const DecodePlan d = decode_plan(r.S, r.T, max_rows, Hq, c.H);
  AB200_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= d.bytes, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, d.bytes, workspace_bytes);
  DecodeParams p{c, r, q, q_stride, out, Hq, Hq / c.H, scale * 1.4426950408889634f, inv_freq, 0x7fffffff, (float *)workspace,
                 (int4 *)((char *)workspace + d.partial_bytes), kernel_error_ptr()};
  AB200_REQUIRE(p.status != nullptr, "%s: cannot resolve the status word", who);
  if (dtype == AB200_F32) return d.rows == 8 ? decode_launch<float, 8>(p, d, stream) : decode_launch<float, 16>(p, d, stream);
  return d.rows == 8 ? decode_launch<__half, 8>(p, d, stream) : decode_launch<__half, 16>(p, d, stream);
}

static int attention_check(const char *who, const Kv8Cache &c, int T, const void *q, long q_stride, const void *out, int Hq, int D, int dtype) {
  AB200_REQUIRE(dtype == AB200_F16 || dtype == AB200_F32, "%s: unknown dtype %d", who, dtype);
  if (D != KV8_D) return fail(AB200_EUNSUPPORTED, "%s: head size %d is not the built size %d", who, D, KV8_D);
  AB200_REQUIRE(Hq > 0 && Hq <= 65535 && Hq % c.H == 0, "%s: %d query heads are not a multiple of %d kv heads", who, Hq, c.H);
  if (T == 0) return AB200_OK;
  AB200_REQUIRE((long)T * Hq <= 1 << 30, "%s: %d rows of %d heads are beyond the built limits", who, T, Hq);
  const long vec = dtype == AB200_F16 ? 8 : 4;
  AB200_REQUIRE(q && out && aligned16(q) && aligned16(out) && q_stride % vec == 0 && q_stride >= (long)Hq * D,
                "%s: q must be 16-byte aligned rows of at least %d values, a multiple of 16 bytes apart, and out 16-byte aligned", who, Hq * D);
  return AB200_OK;
}

}  // namespace ab200

using namespace ab200;

extern "C" size_t ab200_kv8_attention_workspace_bytes(int S, int T, int max_rows, int Hq, int Hkv) {
  if (S <= 0 || T <= 0 || Hkv <= 0 || Hq < Hkv) return 0;
  return decode_plan(S, T, max_rows, Hq, Hkv).bytes;
}

extern "C" int ab200_kv8_attention(const void *q, long q_stride, void *out, const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale, int pages,
                                   int page_rows, int Hkv, const int32_t *page_table, long table_stride, int max_pages, const int32_t *pos0_dev, const int32_t *cu_rows_dev,
                                   int S, int T, int max_rows, int Hq, int D, float scale, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  int rc = kv8_check("kv8_attention", k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, cu_rows_dev, S, T, &c, &r);
  if (!rc) rc = attention_check("kv8_attention", c, T, q, q_stride, out, Hq, D, dtype);
  if (rc) return rc;
  return attend("kv8_attention", c, r, q, q_stride, out, max_rows, Hq, D, scale, dtype, nullptr, workspace, workspace_bytes, (cudaStream_t)stream);
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
  rc = ab200_kv8_append(k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, nullptr, S, T, k, v, k_stride, v_stride,
                        nullptr, 0, nullptr, 0, 0, inv_freq, dtype, stream);
  if (rc) return rc;
  return attend("kv8_step", c, r, q, q_stride, out, T / S, Hq, D, scale, dtype, inv_freq, workspace, workspace_bytes, (cudaStream_t)stream);
}
