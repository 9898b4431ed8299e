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
//
// Bound by memory: 257 bytes for a position and kv head.  Few rows read all of it, so the warp's own matrix instructions serve:
// their 16 rows are filled by 8 packed rows and their second parts, codes go in as they are, and what a warp keeps of a block
// stays in its registers (the 5th-generation tensor cores would want 64 rows and codes widened to 16 bits in shared memory).
// us (TB/s): 64 sequences, all of 16000 positions, 8 kv heads of 4 query heads 323 (6.5, 99 % of a copy's rate); one of 131072 and
// 32 kv heads 170 (6.3); one of 131072 and 8 kv heads 54 (5.0); 64 ragged ones of up to 8000, 8 heads of 8 107 (5.2).  Where a share is
// small, starting an item (7800 cycles) and the second launch weigh: 48 ragged ones of up to 4000 45 us (4.4), of one request of
// 384 positions 6.7 us only a tenth is the stream.  16 rows a tile: products and exponentials bound it, twice a block's instructions.
// Registers and bytes spilled, equal shares: 8 rows 168 and 64 (fp32 80), three CTAs an SM; 16 rows 255 and 32 (fp32 12), two.
#include <math_constants.h>

#include <cooperative_groups.h>

#include <algorithm>

#include "kv8.cuh"
#include "kv8_prefill.cuh"
#include "kv8_quant.cuh"

namespace ab200 {

constexpr int KD_WARPS = 4, KD_THREADS = KD_WARPS * 32, KD_STAGES = 4;
constexpr int KD_STAGE_BYTES = 2 * KV8_BLOCK * KV8_D;  // a block of K, a block of V
constexpr int KD_LEAST = 8;                            // blocks a CTA takes at least, two a warp
constexpr int KD_ITEM = 16;                            // what an item costs besides its blocks, in blocks: 7800 cycles against 470 a block
constexpr int KD_CUT = 64;                             // blocks that a CTA adds up in the tensor cores alone, fp32 rows
constexpr float KD_RAISE = 8.f, KD_P_EXP = 6.f;        // P is scaled by 2^6: its second half stays out of fp16's subnormals
constexpr float KD_LEAST_SCALE = 0x1p-100f;            // a V scale below it (a block of zeros) counts as this

enum { KD_BESIDE_NONE, KD_BESIDE_PROMPTS, KD_BESIDE_APPEND };  // nothing of the first is read here; the second's blocks are waited for
struct DecodeParams {
  Kv8Cache c;
  Kv8Rows r;
  const void *q;
  long q_stride;
  void *out;
  int Hq, group;
  float scale;               // times log2(e)
  const float *inv_freq;     // rotate the queries, or nullptr
  const void *k_new, *v_new;  // this step's rows of keys and values, written first; nullptr: the cache holds them
  long k_stride, v_stride;
  int zero_rest;             // rows that are no sequence's become zeros
  int few;                   // sequences with more rows than this (rows x group) are another kernel's
  int splits, tiles;         // FIXED: CTAs of an item; tiles of a sequence's rows
  int beside;                // KD_BESIDE_*: the kernel before in the stream runs beside this one, which only ends after it
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
__device__ __forceinline__ void kd_mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {  // of a sum: adds to nothing
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// The first product of a chain starts from KD_ZERO: an integer below 2^22 added to these bits is that integer plus 1.5 * 2^23
// as a float, so a subtraction reads the sum and nothing is converted.
constexpr int KD_ZERO = 0x4B400000;
__device__ __forceinline__ float kd_sum(int bits) { return __int_as_float(bits) - 12582912.f; }
__device__ __forceinline__ void kd_imma(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
__device__ __forceinline__ void kd_ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void kd_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float kd_lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float kd_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

__device__ __forceinline__ long kd_div(long a, long b) {  // a, b >= 0; most fit into 32 bits, where a division is a fifth of the work
  return ((a | b) >> 32) == 0 ? (long)((unsigned)a / (unsigned)b) : a / b;
}
// What the threads before this one hold together; *total grows by what all hold.
__device__ __forceinline__ long kd_scan(long v, long (&s)[KD_WARPS], long *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  __syncthreads();
  if (lane == 31) s[warp] = incl;
  __syncthreads();
  long all = 0;
#pragma unroll
  for (int i = 0; i < KD_WARPS; ++i) {
    if (i == warp) incl += all;
    all += s[i];
  }
  *total += all;
  return incl - v;
}
__device__ __forceinline__ void kd_store4(float *out, float4 v, float f) { *reinterpret_cast<float4 *>(out) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }
__device__ __forceinline__ void kd_store4(__half *out, float4 v, float f) {
  *reinterpret_cast<uint2 *>(out) = make_uint2(h22u(__floats2half2_rn(v.x * f, v.y * f)), h22u(__floats2half2_rn(v.z * f, v.w * f)));
}

// A decode step's new rows go into the cache here, block by block: a block is one CTA's, which writes it before it reads it.
// One warp, one block of one head of K or V; rows lo .. hi of it are new (as in kv8_append.cu, which takes longer pieces).
__device__ __noinline__ void kd_append(int8_t *dst, float *scale, const __half *src, long stride, int lo, int hi, bool older, int at, const float *inv_freq) {
  const int lane = threadIdx.x & 31, sub = lane & 15, hw = lane >> 4;
  float f[8][8], most = 0.f, odd = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = 2 * j + hw;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[j][e] = 0.f;
    if (i < lo || i > hi) continue;
    ka_load(src + (i - lo) * stride, sub, f[j]);
    if (inv_freq) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float sn, cs;
        sincosf((float)(at + i) * inv_freq[4 * sub + e], &sn, &cs);
        ka_rotate(f[j][e], f[j][4 + e], sn, cs);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[j][e])), odd = fmaf(f[j][e], 0.f, odd);
  }
  const bool finite = odd == 0.f;
  if (!finite) {
    most = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[j][e]) < CUDART_INF_F ? fabsf(f[j][e]) : 0.f);
  }
  most = warp_max(most);
  const float was = older ? *scale : 0.f;
  float now = most * (1.f / 127.f);
  now = now < KA_LEAST_SCALE ? 0.f : now;
  now = fmaxf(was, now);
  const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
  __syncwarp();  // every lane has read the scale
  if (lane == 0) *scale = now;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = 2 * j + hw;
    uint32_t *d = reinterpret_cast<uint32_t *>(dst + i * KV8_D) + sub;
    const bool again = i < lo && older && now > was;
    if (again) {  // the values they stood for, at the new scale
      const uint32_t a = d[0], b = d[16];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[j][e] = (float)(int8_t)(a >> (8 * e)) * was, f[j][4 + e] = (float)(int8_t)(b >> (8 * e)) * was;
    }
    if (again || (i >= lo && i <= hi)) {
      const uint2 w = kv8_codes(f[j], now, inv, !finite || now == 0.f);
      d[0] = w.x, d[16] = w.y;
    }
  }
}

// ROWS: packed query rows of a tile.  With 8, rows 8-15 of the tensor cores' tile carry second parts: the second byte of
// q, the second half of P; with 16, each part is a product of its own.
// A warp takes two blocks at a time: two independent chains of products and exponentials.
// FIXED: an item is a cluster of p.splits CTAs, which take its blocks in equal shares and join them through each other's
// shared memory: one launch, nothing to look up first.  Else every CTA takes an equal share of all work.
template <typename T, int ROWS, bool FIXED>
__global__ void __launch_bounds__(KD_THREADS, ROWS == 8 ? 3 : 2) kv8_decode_kernel(const __grid_constant__ DecodeParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int NR = ROWS / 8;  // query rows a thread holds: lane / 4, and 8 more
  __shared__ __align__(16) float scales_s[KD_WARPS][KD_STAGES][2];
  __shared__ long scan_s[KD_WARPS];
  __shared__ long found_start;
  __shared__ int found_s;
  __shared__ float m_s[KD_WARPS][ROWS], l_s[KD_WARPS][ROWS], q_max_s[KD_WARPS][ROWS];
  constexpr int BYTES = 3;                    // of a query value
  __shared__ uint32_t q_s[NR][BYTES][8][32];  // as the lanes hold them
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, j4 = lane & 3;
  const Kv8Rows &r = p.r;
  pdl_launch_dependents();
  // A kernel beside this one releases it after its own wait: whatever came before that one is complete by then.  What the prompt
  // kernel writes is not read here; the blocks that new rows lie in are waited for, each warp before its first of them.  What
  // comes after this kernel waits for it alone, so it waits for the one beside it before it ends.
  if (!p.beside) pdl_wait();

  if (p.zero_rest) {  // rows in front of the first sequence's, then those behind the last one's
    const long row16 = (long)p.Hq * KV8_D * sizeof(T) / 16, front = r.begin(0) * row16, own = (r.end(r.S - 1) - r.begin(0)) * row16;
    for (long i = (long)blockIdx.x * KD_THREADS + tid; i < r.T * row16 - own; i += (long)gridDim.x * KD_THREADS)
      reinterpret_cast<uint4 *>(p.out)[i < front ? i : i + own] = make_uint4(0, 0, 0, 0);
  }

  // ---- this CTA's share: w0 .. w1 - 1 of all work, ordered by sequence, kv head, tile, block
  long total = 0, start = 0, weight = 0, per = 1, w0 = 0, w1 = 0;
  if constexpr (!FIXED) {
    for (int base = 0; base < r.S; base += KD_THREADS) {
      weight = base + tid < r.S ? kd_weight<ROWS>(p, base + tid) * p.c.H : 0;
      const long before = total;
      start = before + kd_scan(weight, scan_s, &total);
    }
    per = max((long)kd_div(total + gridDim.x - 1, gridDim.x), (long)KD_LEAST);
    w0 = blockIdx.x * per, w1 = min(w0 + per, total);
    if (tid == 0) p.split[blockIdx.x] = make_int4(0, 0, 0, 0);
    if (w0 >= w1) {
      if (p.beside) pdl_wait();
      return;
    }
    if (r.S > KD_THREADS) total = 0;
    for (int base = 0;;) {
      if (r.S > KD_THREADS) {
        weight = base + tid < r.S ? kd_weight<ROWS>(p, base + tid) * p.c.H : 0;
        const long before = total;
        start = before + kd_scan(weight, scan_s, &total);
      }
      if (w0 >= start && w0 < start + weight) found_s = base + tid, found_start = start;
      base += KD_THREADS;
      if (total > w0 || base >= r.S) break;
    }
    __syncthreads();
  }
  int s = FIXED ? 0 : found_s;
  start = FIXED ? 0 : found_start;
  long w = w0;
  const long cap = (long)r.max_pages << p.c.shift;
  // the next item, or part of one, in the share
  struct Part {
    long pos0, item;  // where the item begins in the order of all work
    int seq, row0, rows, hk, first, last, blocks, b0, b1;  // packed rows first .. last, blocks b0 .. b1 - 1 of `blocks`
  };
  auto next = [&](Part &it) {
    while (w < w1) {
      const int row0 = r.begin(s), rows = max(0, r.end(s) - row0) * p.group;
      const long per_head = kd_weight<ROWS>(p, s);
      if (w >= start + per_head * p.c.H) {
        start += per_head * p.c.H, ++s;
        continue;
      }
      it.pos0 = r.pos0[s], it.seq = s, it.row0 = row0, it.rows = rows;
      it.hk = (int)kd_div(w - start, per_head);
      long at = (w - start) - it.hk * per_head;
      int t = 0;
      it.blocks = kd_blocks<ROWS>(p, it.pos0, rows, 0);
      while (at >= it.blocks + KD_ITEM) at -= it.blocks + KD_ITEM, it.blocks = kd_blocks<ROWS>(p, it.pos0, rows, ++t);
      it.first = t * ROWS, it.last = min(it.first + ROWS, rows) - 1;
      const long take = min(it.blocks + KD_ITEM - at, w1 - w);
      it.b0 = (int)max(0l, at - KD_ITEM), it.b1 = (int)max(0l, at + take - KD_ITEM);
      it.item = w - at;
      w += take;
      if (it.b1 > 0) return true;  // else the share ends before the item's first block
    }
    return false;
  };

  unsigned char *const ring_mine = smem + warp * (KD_STAGES * KD_STAGE_BYTES);
  const uint32_t ring = kd_smem(ring_mine);
  // 16-byte piece i * 32 + lane of a block: row i * 4 + lane / 8, and its place under the XOR of row and piece that ldmatrix wants
  const uint32_t put0 = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4), put1 = put0 ^ 64;
  const uint32_t k_at = (lane & 7) * 128 + (((lane >> 3) ^ (lane & 7)) << 4);                         // pieces 0-3; pieces 4-7: ^ 64
  const uint32_t v_row = 2048 + (lane & 15) * 128, v_sw = lane & 7, v_chunk = lane >> 4;
  const int8_t *const k_lane = p.c.k + lane * 16, *const v_lane = p.c.v + lane * 16;
  const float *const sc_lane = lane ? p.c.vs : p.c.ks;
  const uint32_t sc_put = kd_smem(&scales_s[warp][0][0]) + 4 * lane;
  static_assert(KD_STAGES == 4 && KD_STAGE_BYTES == 4096, "two pairs of blocks; a pair's scales lie 16 bytes after the other's");
  const int nothing[4] = {KD_ZERO, KD_ZERO, KD_ZERO, KD_ZERO};

  // ---- this warp's blocks of a part: the pairs b0 + 2 (warp, warp + 4, ...).  The second of an odd last pair is the first
  // again, its keys masked like all behind `end`.
  Part it = {};
  int live = 0, pairs = 0, asked = 0, where = 0, fresh = 0x7fffffff;  // fresh: the first block that is being written, if any is
  uint32_t put = 0;
  auto limit_of = [&](int packed) { return (int)max(0l, min(it.pos0 + packed / p.group + 1, cap)); };
  auto issue = [&]() {
    if (asked < pairs) {
      if ((asked & 15) == 0) {  // where the next 16 pairs' blocks lie, one a lane
        const int b = min(it.b0 + 2 * (warp + (asked + (lane >> 1)) * KD_WARPS) + (lane & 1), live - 1);
        int page = r.table[(size_t)it.seq * r.table_stride + (b >> (p.c.shift - 4))];
        if ((unsigned)page >= (unsigned)p.c.pages) {
          atomicExch(p.status, KV8_BAD_PAGE);
          page = 0;
        }
        where = ((page * p.c.H + it.hk) << (p.c.shift - 4)) + (b & ((1 << (p.c.shift - 4)) - 1));
      }
      const bool written = min(it.b0 + 2 * (warp + asked * KD_WARPS) + 1, live - 1) >= fresh;
      if (written) pdl_wait();
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int blk = __shfl_sync(0xffffffffu, where, 2 * (asked & 15) + u);
        const int8_t *kp = k_lane + (size_t)blk * (KV8_BLOCK * KV8_D), *vp = v_lane + (size_t)blk * (KV8_BLOCK * KV8_D);
        const uint32_t to0 = ring + put + put0, to1 = ring + put + put1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((i & 1 ? to1 : to0) + u * KD_STAGE_BYTES + i * 512), "l"(kp + i * 512) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((i & 1 ? to1 : to0) + u * KD_STAGE_BYTES + 2048 + i * 512), "l"(vp + i * 512) : "memory");
        }
        // a scale next to it may have brought this one's line to L1 before it was written
        if (written && lane < 2) asm volatile("st.shared.f32 [%0], %1;" ::"r"(sc_put + (put >> 9) + 8 * u), "f"(__ldcg(sc_lane + blk)) : "memory");
        else if (lane < 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc_put + (put >> 9) + 8 * u), "l"(sc_lane + blk) : "memory");
      }
      ++asked;
      put ^= 2 * KD_STAGE_BYTES;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto begin = [&]() {
    if (FIXED && sizeof(T) == 2 && p.k_new) {
      // positions that are stored, and the two blocks at most that they lie in; a warp has K or V of one of them
      const long from = max(it.pos0, 0l), to = min(it.pos0 + it.rows / p.group, cap) - 1;
      const int block = (int)(from >> 4) + (warp >> 1);
      const bool here = from <= to && (int)(from >> 4) < it.b1 && (int)(to >> 4) >= it.b0;
      if (here && block <= (int)(to >> 4) && block >= it.b0 && block < it.b1) {
        const long page = kv8_page(p.c, r, it.seq, block << 4, p.status);
        if (page >= 0) {
          const int at = block << 4, in_page = at & ((1 << p.c.shift) - 1), lo = (int)(max(from, (long)at) - at), hi = (int)(min(to, (long)at + 15) - at);
          const bool is_v = warp & 1;
          const size_t head = (size_t)page * p.c.H + it.hk;
          const long stride = is_v ? p.v_stride : p.k_stride;
          kd_append((is_v ? p.c.v : p.c.k) + ((head << p.c.shift) + in_page) * KV8_D, (is_v ? p.c.vs : p.c.ks) + (head << (p.c.shift - 4)) + (in_page >> 4),
                    (const __half *)(is_v ? p.v_new : p.k_new) + (size_t)(it.row0 + (at + lo - it.pos0)) * stride + (size_t)it.hk * KV8_D, stride, lo, hi, it.pos0 > at, at,
                    is_v ? nullptr : p.inv_freq);
        }
      }
      if (here) __syncthreads();  // who reads the block is of this CTA
    }
    if (p.beside == KD_BESIDE_APPEND) fresh = (int)(max(it.pos0, 0l) >> 4);
    live = min(it.b1, (limit_of(it.last) + 15) >> 4);  // blocks that hold a key some row attends to
    pairs = max(0, ((live - it.b0 + 1) / 2 - warp + KD_WARPS - 1) / KD_WARPS);
    asked = 0, put = 0;
    issue();
  };

  bool more = true;
  if constexpr (FIXED) {
    const int item = blockIdx.x / p.splits, z = blockIdx.x - item * p.splits, t = item % p.tiles, head = item / p.tiles;
    it.hk = head % p.c.H, it.seq = head / p.c.H;
    it.row0 = r.begin(it.seq), it.rows = (r.end(it.seq) - it.row0) * p.group, it.pos0 = r.pos0[it.seq];
    it.first = t * ROWS, it.last = min(it.first + ROWS, it.rows) - 1;
    it.blocks = kd_blocks<ROWS>(p, it.pos0, it.rows, t);
    it.b0 = (int)((long)it.blocks * z / p.splits), it.b1 = (int)((long)it.blocks * (z + 1) / p.splits);
  } else {
    more = next(it);
  }
  if (more) begin();
  while (more) {
    // ---- queries, meanwhile.  A warp takes the pieces warp and warp + 4 (a rotated pair is one thread's): thread's row(s),
    // dims 16 c + 4 j4 .. + 3.  Each row is scaled by a power of two, its largest to 2^21 .. 2^22, rounded to an
    // integer and cut into signed bytes (the first is 64 at most): half a step is 2^-22 of the largest, and fp16 rows are exact
    // unless they span more than 11 octaves.
    float f[NR][2][4], back[NR];
    int limit[NR];
    const int end = 16 * live;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const int packed = it.first + 8 * i + g;
      const bool in = packed <= it.last;
      limit[i] = in ? min(limit_of(packed), end) : end;
      const int token = in ? packed / p.group : 0, head = it.hk * p.group + (in ? packed - token * p.group : 0);
      const T *q = (const T *)p.q + (size_t)(it.row0 + token) * p.q_stride + (size_t)head * KV8_D + 16 * warp + 4 * j4;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if constexpr (sizeof(T) == 2) {
          const uint2 v = in ? *reinterpret_cast<const uint2 *>(q + 64 * c) : make_uint2(0, 0);
          const float2 a = __half22float2(u2h2(v.x)), b = __half22float2(u2h2(v.y));
          f[i][c][0] = a.x, f[i][c][1] = a.y, f[i][c][2] = b.x, f[i][c][3] = b.y;
        } else {
          const float4 v = in ? *reinterpret_cast<const float4 *>(q + 64 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
          f[i][c][0] = v.x, f[i][c][1] = v.y, f[i][c][2] = v.z, f[i][c][3] = v.w;
        }
      }
      if (p.inv_freq) {
        const float pos = (float)(int)(it.pos0 + token);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float sn, cs;
          sincosf(pos * p.inv_freq[16 * warp + 4 * j4 + e], &sn, &cs);
          ka_rotate(f[i][0][e], f[i][1][e], sn, cs);
        }
      }
      // a row that is not finite is made of NaN: its largest, as a bit pattern, is above that of every number
      uint32_t most = 0;
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max(most, __float_as_uint(f[i][c][e]) & 0x7fffffffu);
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      if (j4 == 0) q_max_s[warp][8 * i + g] = __uint_as_float(most);
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < KD_WARPS; ++i) most = max(most, __float_as_uint(q_max_s[i][8 * n + g]));
      const int e = 21 - (int)(most >> 23) + 127;  // -107 .. 148
      const float up = kv8_pow2(e >> 1), up2 = kv8_pow2(e - (e >> 1));
      back[n] = most >= 0x7f800000u ? CUDART_NAN_F : kv8_pow2(-e);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t part[BYTES] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          int v = __float2int_rn(f[n][c][i] * up * up2);
#pragma unroll
          for (int k = BYTES - 1; k > 0; --k) {
            const int low = (int)(int8_t)v;
            part[k] |= (uint32_t)(low & 255) << (8 * i);
            v = (v - low) >> 8;
          }
          part[0] |= (uint32_t)(v & 255) << (8 * i);
        }
#pragma unroll
        for (int k = 0; k < BYTES; ++k) q_s[n][k][warp + 4 * c][lane] = part[k];
      }
    }
    __syncthreads();
    // A operands: step c (dims 32 c .. + 31), product i
    constexpr int PRODUCTS = ROWS == 8 ? 2 : 3;
    uint32_t qa[4][PRODUCTS][4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < PRODUCTS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qa[c][i][e] = ROWS == 8 ? q_s[0][i == 0 ? e & 1 : 2][2 * c + (e >> 1)][lane] : q_s[NR == 2 ? e & 1 : 0][i][2 * c + (e >> 1)][lane];
    float o[16][4], m[NR], l[NR];
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
#pragma unroll
    for (int n = 0; n < NR; ++n) m[n] = -CUDART_INF_F, l[n] = 0.f;

    const int full = min(limit_of(it.first), end);  // keys that every row attends to
    uint32_t get = 0;
    int key0 = (it.b0 + 2 * warp) * 16;
    for (int i = 0; i < pairs; ++i, key0 += 32 * KD_WARPS, get ^= 2 * KD_STAGE_BYTES) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();  // every lane's pieces have landed, and everyone is done with the pair that is filled next
      issue();
      const uint32_t st = ring + get;
      const float4 scales = *reinterpret_cast<const float4 *>(reinterpret_cast<const char *>(&scales_s[warp][0][0]) + (get >> 9));
      float x[2][NR][4], inv_vs[2];  // exponents of p vs: thread's rows, keys 8 hb + 2 j4, + 1 of each block
      bool raise = false;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float ks = (u ? scales.z : scales.x) * p.scale, vs = fmaxf(u ? scales.w : scales.y, KD_LEAST_SCALE);
        const float lvs = kd_lg2(vs);
        inv_vs[u] = kd_rcp(vs) * KV8_SUM;
        // q . k: bytes times bytes, exact
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
          int d[PRODUCTS][4];
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            uint32_t k[4];
            kd_ldsm(k, st + u * KD_STAGE_BYTES + hb * 1024 + (cc ? k_at ^ 64 : k_at));
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < PRODUCTS; ++e) {
                if (cc == 0 && h == 0) kd_imma(d[e], qa[0][e], k[0], k[1], nothing);
                else kd_imma(d[e], qa[2 * cc + h][e], k[2 * h], k[2 * h + 1], d[e]);
              }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if constexpr (ROWS == 8) {
              x[u][0][2 * hb + e] = fmaf(kd_sum(d[0][e]), 65536.f, fmaf(kd_sum(d[0][2 + e]), 256.f, kd_sum(d[1][e])));
            } else {
#pragma unroll
              for (int n = 0; n < NR; ++n)
                x[u][n][2 * hb + e] = fmaf(kd_sum(d[0][2 * n + e]), 65536.f, fmaf(kd_sum(d[1][2 * n + e]), 256.f, kd_sum(d[PRODUCTS - 1][2 * n + e])));
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          const float f = ks * back[n];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][n][e] = fmaf(x[u][n][e], f, lvs);
        }
      }
      if (key0 + 32 > full) {  // the same for the whole warp
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (key0 + 16 * u + 8 * (e >> 1) + 2 * j4 + (e & 1) >= limit[n]) x[u][n][e] = -CUDART_INF_F;
      }
      float top[NR];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        top[n] = fmaxf(fmaxf(fmaxf(x[0][n][0], x[0][n][1]), fmaxf(x[0][n][2], x[0][n][3])), fmaxf(fmaxf(x[1][n][0], x[1][n][1]), fmaxf(x[1][n][2], x[1][n][3])));
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
      // A operands of P: [half][..] for 16 rows; both halves in one for 8
      uint32_t pa[2][NR][4];
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float shift = m[n] == -CUDART_INF_F ? 0.f : m[n] - KD_P_EXP;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float sum = 0.f;
#pragma unroll
          for (int hb = 0; hb < 2; ++hb) {
            const float a = kd_ex2(x[u][n][2 * hb] - shift), b = kd_ex2(x[u][n][2 * hb + 1] - shift);
            sum += a + b;
            const __half2 hi = __floats2half2_rn(a, b);
            const float2 hf = __half22float2(hi);
            const uint32_t lo = h22u(__floats2half2_rn(a - hf.x, b - hf.y));
            if constexpr (ROWS == 8) pa[u][0][2 * hb] = h22u(hi), pa[u][0][2 * hb + 1] = lo;
            else pa[u][0][2 * hb + n] = h22u(hi), pa[u][NR - 1][2 * hb + n] = lo;
          }
          l[n] = fmaf(sum, inv_vs[u], l[n]);
        }
      }
      // keys 0-7 and 8-15 of piece c, then of piece c + 1; transposed: two keys, two dims a word
      auto values = [&](int u, int c, uint32_t(&v)[4]) { kd_ldsm_t(v, st + u * KD_STAGE_BYTES + v_row + (((c + v_chunk) ^ v_sw) << 4)); };
      auto product = [&](float(&even)[4], float(&odd)[4], const uint32_t(&p_)[4], uint32_t v0, uint32_t v1, bool first) {
        const uint32_t u0 = v0 ^ 0x80808080u, u1 = v1 ^ 0x80808080u;
        const uint32_t e0 = kd_half2<0x4240>(u0), e1 = kd_half2<0x4240>(u1), d0 = kd_half2<0x4341>(u0), d1 = kd_half2<0x4341>(u1);
        if (first) kd_mma_first(even, p_[0], p_[1], p_[2], p_[3], e0, e1), kd_mma_first(odd, p_[0], p_[1], p_[2], p_[3], d0, d1);
        else kd_mma(even, p_[0], p_[1], p_[2], p_[3], e0, e1), kd_mma(odd, p_[0], p_[1], p_[2], p_[3], d0, d1);
      };
      if constexpr (sizeof(T) == 2 || FIXED) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int c = 0; c < 8; c += 2) {
            uint32_t v[4];
            values(u, c, v);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int n = 0; n < NR; ++n) product(o[2 * (c + h)], o[2 * (c + h) + 1], pa[u][n], v[2 * h], v[2 * h + 1], false);
          }
      } else {
        // fp32 rows: the tensor cores cut what they add to 24 bits, always towards zero, 3e-6 of a sum over 16000 keys.  So two blocks'
        // product is a sum of its own, the low halves of P first, and joins the others by an addition that rounds.  A cluster's CTA has
        // KD_CUT blocks at most, in which 2e-7 are cut, and keeps its shorter code.  us, one sum / sums of two blocks: 5 sequences of up to 1000
        // positions 13.2 / 13.7, 64 of 16000 332 / 331, 16 times four rows 59 / 64.
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
          uint32_t v[2][4];
          values(0, c, v[0]), values(1, c, v[1]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float even[4], odd[4];
#pragma unroll
            for (int n = NR - 1; n >= 0; --n)
#pragma unroll
              for (int u = 0; u < 2; ++u) product(even, odd, pa[u][n], v[u][2 * h], v[u][2 * h + 1], n == NR - 1 && u == 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[2 * (c + h)][e] += even[e], o[2 * (c + h) + 1][e] += odd[e];
          }
        }
      }
    }
    // ---- the next part's first blocks are on their way while the four warps' parts of this one are joined in the ring's
    // other half
    const Part done = it;
    const int empty = (int)max(0l, min((long)ROWS, -it.pos0 * p.group - it.first));  // leading rows with nothing to attend to
    more = FIXED ? false : next(it);
    __syncwarp();
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
        *reinterpret_cast<float4 *>(ring_mine + 2 * KD_STAGE_BYTES + ((8 * n + g) * KV8_D + 16 * c + 4 * j4) * 4) = v;
      }
    }
    if (more) begin();
    __syncthreads();
    const bool whole = FIXED ? p.splits == 1 : done.b0 == 0 && done.b1 == done.blocks;
    const int slot = done.b0 == 0 ? 1 : 0;
    constexpr int PER_ROW = KD_THREADS / ROWS, PIECES = KV8_D / 4 / PER_ROW;  // threads of a row, four dims at a time
    const int row = tid / PER_ROW, col = tid % PER_ROW * 4;
    if (row <= done.last - done.first) {
      float mx = -CUDART_INF_F, sum = 0.f, f[KD_WARPS];
#pragma unroll
      for (int i = 0; i < KD_WARPS; ++i) mx = fmaxf(mx, m_s[i][row]);
#pragma unroll
      for (int i = 0; i < KD_WARPS; ++i) {
        f[i] = m_s[i][row] == -CUDART_INF_F ? 0.f : kd_ex2(m_s[i][row] - mx);
        sum = fmaf(l_s[i][row], f[i], sum);
      }
      const int packed = done.first + row, token = packed / p.group, head = done.hk * p.group + packed - token * p.group;
      T *out = (T *)p.out + ((size_t)(done.row0 + token) * p.Hq + head) * KV8_D + col;
      // a part to be joined: FIXED into the ring's other half, else to memory
      float *part = FIXED ? reinterpret_cast<float *>(smem) + row * KV8_D + col : p.partial + (((size_t)blockIdx.x * 2 + slot) * ROWS + row) * KV8_D + col;
      const float over = row < empty ? 0.f : KV8_SUM / sum;
#pragma unroll
      for (int c = 0; c < PIECES; ++c) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < KD_WARPS; ++i) {
          const float4 v = *reinterpret_cast<const float4 *>(smem + i * (KD_STAGES * KD_STAGE_BYTES) + 2 * KD_STAGE_BYTES + (row * KV8_D + col + c * PER_ROW * 4) * 4);
          acc.x = fmaf(v.x, f[i], acc.x), acc.y = fmaf(v.y, f[i], acc.y), acc.z = fmaf(v.z, f[i], acc.z), acc.w = fmaf(v.w, f[i], acc.w);
        }
        if (whole) kd_store4(out + c * PER_ROW * 4, acc, over);
        else *reinterpret_cast<float4 *>(part + c * PER_ROW * 4) = acc;
      }
      if (FIXED) {
        if (col == 0) q_max_s[0][row] = mx, q_max_s[1][row] = sum;
      } else if (!whole && col == 0)
        reinterpret_cast<float2 *>(p.partial + (size_t)gridDim.x * 2 * ROWS * KV8_D)[((size_t)blockIdx.x * 2 + slot) * ROWS + row] = make_float2(mx, sum);
    }
    if constexpr (FIXED) {
      if (p.splits > 1) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int z = (int)cluster.block_rank(), mine = ROWS / p.splits;  // a CTA joins its share of the rows, a thread a dim
        for (int row = z * mine; row < (z + 1) * mine && row <= done.last - done.first; ++row) {
          float mx = -CUDART_INF_F, sum = 0.f, acc = 0.f;
          for (int i = 0; i < p.splits; ++i) mx = fmaxf(mx, *cluster.map_shared_rank(&q_max_s[0][row], i));
          for (int i = 0; i < p.splits; ++i) {
            const float m = *cluster.map_shared_rank(&q_max_s[0][row], i), f = m == -CUDART_INF_F ? 0.f : kd_ex2(m - mx);
            sum = fmaf(*cluster.map_shared_rank(&q_max_s[1][row], i), f, sum);
            acc = fmaf(*cluster.map_shared_rank(reinterpret_cast<float *>(smem) + row * KV8_D + tid, i), f, acc);
          }
          const int packed = done.first + row, token = packed / p.group, head = done.hk * p.group + packed - token * p.group;
          ((T *)p.out)[((size_t)(done.row0 + token) * p.Hq + head) * KV8_D + tid] = (T)(row < empty ? 0.f : acc * (KV8_SUM / sum));
        }
        cluster.sync();  // nobody leaves while its memory is read
      }
    } else if (!whole && slot == 1 && tid == 0)  // begun here: the CTAs up to the one with the item's last block have the rest
      p.split[blockIdx.x] = make_int4((int)kd_div(done.item + KD_ITEM + done.blocks - 1, per) - (int)blockIdx.x + 1, done.row0,
                                      done.hk | (done.last - done.first) << 16 | empty << 20, done.first);
  }
  if (p.beside) pdl_wait();
}

// Joins the parts of the items that several CTAs share.  A CTA has one row of the items begun in eight CTAs of the first
// kernel, a warp each; an item in more than eight parts is all warps' work, part by part.
constexpr int KJ_WARPS = 8, KJ_THREADS = KJ_WARPS * 32;
struct Joined {
  float m, l;
  float4 acc;
  __device__ __forceinline__ Joined() { m = -CUDART_INF_F, l = 0.f, acc = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void add(float2 ml, float4 v) {
    const float up = fmaxf(m, ml.x), f = m == -CUDART_INF_F ? 0.f : kd_ex2(m - up), fc = ml.x == -CUDART_INF_F ? 0.f : kd_ex2(ml.x - up);
    l = l * f + ml.y * fc;
    acc.x = acc.x * f + v.x * fc, acc.y = acc.y * f + v.y * fc, acc.z = acc.z * f + v.z * fc, acc.w = acc.w * f + v.w * fc;
    m = up;
  }
};
// BATCH parts are loaded at once, the first two before it is known whether there are any.  With 8 a thread has 79 registers and an
// SM three CTAs, with 4 64 and four; us, 8 / 4, the whole call among others (which start while the kernel before still runs): one
// sequence of 131072 positions 57 / 62, 48 ragged requests 58.7 / 61; tiles of 16 rows, 16 sequences of four 24.1 / 22.5.  Before, with 64
// registers and parts asked for when known: 64.8, 63.3, 23.0, and 377 for 64 sequences of 16000 positions (323 now).
template <typename T, int ROWS>
__global__ void __launch_bounds__(KJ_THREADS) kv8_join_kernel(const __grid_constant__ DecodeParams p, int ctas) {
  constexpr int BATCH = ROWS == 8 ? 8 : 4;
  __shared__ float4 acc_s[KJ_WARPS][32];
  __shared__ float2 ml_s[KJ_WARPS];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y, c0 = blockIdx.x * KJ_WARPS;
  const int4 my = lane < KJ_WARPS && c0 + lane < ctas ? p.split[c0 + lane] : make_int4(0, 0, 0, 0);
  const float2 *const ml = reinterpret_cast<const float2 *>(p.partial + (size_t)ctas * 2 * ROWS * KV8_D) + row;
  const float4 *const acc = reinterpret_cast<const float4 *>(p.partial + row * KV8_D) + lane;
  auto part = [&](int c, int i) { return ((size_t)(c + i) * 2 + (i == 0 ? 1 : 0)) * ROWS; };
  auto store = [&](int4 sp, const Joined &a) {
    const int packed = sp.w + row, token = packed / p.group, head = (sp.z & 0xFFFF) * p.group + packed - token * p.group;
    T *out = (T *)p.out + ((size_t)(sp.y + token) * p.Hq + head) * KV8_D + 4 * lane;
    const bool none = row < sp.z >> 20;
    kd_store4(out, a.acc, none ? 0.f : KV8_SUM / a.l);
  };
  // the parts of an item that two CTAs share, before it is known whether there is one
  float2 s0[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  float4 v0[2] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (c0 + warp + i < ctas) s0[i] = ml[part(c0 + warp, i)], v0[i] = acc[part(c0 + warp, i) * (KV8_D / 4)];
  for (int k = 0; k < KJ_WARPS; ++k) {
    const int4 sp = make_int4(__shfl_sync(0xffffffffu, my.x, k), __shfl_sync(0xffffffffu, my.y, k), __shfl_sync(0xffffffffu, my.z, k), __shfl_sync(0xffffffffu, my.w, k));
    if (sp.x == 0 || row > (sp.z >> 16 & 15) || (sp.x <= KJ_WARPS && k != warp)) continue;
    const int step = sp.x <= KJ_WARPS ? 1 : KJ_WARPS;
    Joined a;
    if (step == 1) a.add(s0[0], v0[0]), a.add(s0[1], v0[1]);  // two at least
    for (int i0 = step == 1 ? 2 : warp; i0 < sp.x; i0 += BATCH * step) {
      float2 s[BATCH];
      float4 v[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int i = i0 + j * step;
        s[j] = i < sp.x ? ml[part(c0 + k, i)] : make_float2(-CUDART_INF_F, 0.f);
        v[j] = i < sp.x ? acc[part(c0 + k, i) * (KV8_D / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) a.add(s[j], v[j]);
    }
    if (step > 1) {  // every warp is here
      __syncthreads();
      acc_s[warp][lane] = a.acc;
      if (lane == 0) ml_s[warp] = make_float2(a.m, a.l);
      __syncthreads();
      if (k != warp) continue;
      a = Joined();
#pragma unroll
      for (int j = 0; j < KJ_WARPS; ++j) a.add(ml_s[j], acc_s[j][lane]);
    }
    store(sp, a);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------
struct DecodePlan {
  int rows, ctas;
  int splits;  // > 0: an item to a cluster of this many CTAs; 0: equal shares and a second launch that joins them
  int tiles;
  size_t partial_bytes, bytes;
};
static DecodePlan decode_plan(int S, int T, int max_rows, int Hq, int Hkv, bool uniform, long capacity, int dtype) {
  DecodePlan d;
  const long group = Hq / Hkv;
  d.rows = (long)max_rows * group <= 8 ? 8 : 16;
  d.ctas = sm_count() * (d.rows == 8 ? 3 : 2);
  d.partial_bytes = (size_t)d.ctas * 2 * d.rows * (KV8_D + 2) * sizeof(float);
  d.bytes = d.partial_bytes + (size_t)d.ctas * sizeof(int4);
  // One launch where no CTA then has 24 blocks more to do than its equal share (what the lookups and the second launch take):
  // one sequence as long as its pages allow, of several the longest so long and half as much in the mean.
  // us, clusters / equal shares: one request of 384 positions and 32 heads 6.7 / 10.8; five of up to 1000 12.8 / 16.1;
  // 16 times four rows of up to 3000 29 / 22.
  const long tiles = ((long)(T / S) * group + d.rows - 1) / d.rows, items = S * Hkv * tiles, blocks = (capacity + 15) / 16;
  d.tiles = (int)tiles;
  d.splits = 0;
  if (uniform && items <= d.ctas) {
    int c = 1;
    while (c < 8 && items * c * 2 <= d.ctas) c *= 2;
    const long each = (blocks + c - 1) / c;
    if (each <= items * blocks / (S == 1 ? 1 : 2) / d.ctas + 24 && (dtype == AB200_F16 || each <= KD_CUT)) d.splits = c;
  }
  return d;
}

template <typename T, int ROWS>
static int decode_launch(DecodeParams p, const DecodePlan &d, cudaStream_t stream) {
  constexpr int smem = KD_WARPS * KD_STAGES * KD_STAGE_BYTES;
  static_assert(KD_STAGES / 2 * KD_STAGE_BYTES >= ROWS * KV8_D * (int)sizeof(float), "a warp's part fits into half its ring");
  if (d.splits > 0) {
    p.splits = d.splits, p.tiles = d.tiles;
    AB200_CUDA(cudaFuncSetAttribute(kv8_decode_kernel<T, ROWS, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long)p.r.S * p.c.H * d.tiles * d.splits));
    cfg.blockDim = dim3(KD_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = d.splits, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    AB200_CUDA(cudaLaunchKernelEx(&cfg, kv8_decode_kernel<T, ROWS, true>, p));
    return AB200_OK;
  }
  AB200_CUDA(cudaFuncSetAttribute(kv8_decode_kernel<T, ROWS, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  AB200_CUDA(launch_pdl(kv8_decode_kernel<T, ROWS, false>, dim3(d.ctas), dim3(KD_THREADS), smem, stream, p));
  AB200_CUDA(launch_pdl(kv8_join_kernel<T, ROWS>, dim3((d.ctas + KJ_WARPS - 1) / KJ_WARPS, ROWS), dim3(KJ_THREADS), 0, stream, p, d.ctas));
  return AB200_OK;
}

// Which kernels serve a call goes by the width of its page table, the most positions that its sequences can have: their lengths are
// on the device.  A table much wider than its sequences are long costs the cluster form: one request of 384 positions and 32 heads, step /
// attention 8.5 / 6.7 us with 64 pages of 64 rows in its row, 11.0 / 9.6 with 512 or 2000.
//
// Sequences of up to KD_FEW packed rows go through the kernel above, longer ones through the prompt kernel where rows of heads
// times the positions that the pages hold are more than KD_PROMPT_WORK.  us, above / prompt kernel, rows of heads x positions:
//   500 x 2600 (one kv head) 13.5 / 24.6     2240 x 570 14.1 / 18.3     4096 x 128 7.2 / 11.5     2048 x 64 12.2 / 10.3
//   4800 x 650 28.6 / 23.4     2500 x 3000 (one kv head) 86 / 27     4000 x 2000 32 / 26     4096 x 4100 71 / 31     16384 x 4500 308 / 67
constexpr int KD_FEW = 64;
constexpr long KD_PROMPT_WORK = 2500000;
struct AttendPlan {
  bool prompts, few;  // which kernels run
  DecodePlan d;
  Kv8PrefillParams p;
  size_t bytes;       // of workspace: the prompt kernel's, then the other's (they may run side by side)
};
struct NewRows {
  const void *k, *v;
  long k_stride, v_stride;
};
static int attend_plan(const Kv8Cache &c, const Kv8Rows &r, int max_rows, int Hq, int dtype, bool rotate, AttendPlan *a) {
  const int group = Hq / c.H;
  const long capacity = (long)r.max_pages << c.shift, most = r.cu ? max_rows : r.n;
  a->prompts = most * group > KD_FEW && (long)r.T * Hq * capacity > KD_PROMPT_WORK && !rotate;
  a->few = !a->prompts || r.cu != nullptr;
  a->d = decode_plan(r.S, r.T, a->few && a->prompts ? std::max(KD_FEW / group, 1) : (int)most, Hq, c.H, r.cu == nullptr, capacity, dtype);
  a->p = Kv8PrefillParams{};
  a->p.c = c, a->p.r = r, a->p.group = group;
  size_t prompt_bytes = 0;
  if (a->prompts) {
    const int rc = kv8_prefill_plan(&a->p, dtype, capacity, &prompt_bytes);
    if (rc) return rc;
  }
  a->bytes = prompt_bytes + a->d.bytes;
  return AB200_OK;
}
static int attend(const char *who, const Kv8Cache &c, const Kv8Rows &r, const void *q, long q_stride, void *out, int max_rows, int Hq, float scale, int dtype, const float *inv_freq,
                  NewRows new_rows, bool appending, int zero_rest, void *workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (r.T == 0 || r.S == 0) return AB200_OK;
  AttendPlan a;
  int rc = attend_plan(c, r, max_rows, Hq, dtype, inv_freq != nullptr, &a);
  if (rc) return rc;
  AB200_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= a.bytes, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, a.bytes, workspace_bytes);
  int *status = kernel_error_ptr();
  AB200_REQUIRE(status != nullptr, "%s: cannot resolve the status word", who);
  const int group = Hq / c.H;
  const float scale2 = scale * 1.4426950408889634f;
  if (a.prompts) {
    a.p.q = q, a.p.q_stride = q_stride, a.p.out = out, a.p.Hq = Hq, a.p.scale = scale2, a.p.few = a.few ? KD_FEW : 0, a.p.status = status;
    rc = kv8_prefill(a.p, dtype, workspace, stream);
    if (rc) return rc;
  }
  if (a.few) {
    char *ws = (char *)workspace + (a.bytes - a.d.bytes);
    DecodeParams p{c, r, q, q_stride, out, Hq, group, scale2, inv_freq, new_rows.k, new_rows.v, new_rows.k_stride, new_rows.v_stride, zero_rest && r.cu,
                   a.prompts ? KD_FEW : 0x7fffffff, 0, 0, a.prompts && pdl_enabled() ? KD_BESIDE_PROMPTS : appending && pdl_enabled() ? KD_BESIDE_APPEND : KD_BESIDE_NONE, (float *)ws, (int4 *)(ws + a.d.partial_bytes), status};
    if (dtype == AB200_F32) rc = a.d.rows == 8 ? decode_launch<float, 8>(p, a.d, stream) : decode_launch<float, 16>(p, a.d, stream);
    else rc = a.d.rows == 8 ? decode_launch<__half, 8>(p, a.d, stream) : decode_launch<__half, 16>(p, a.d, stream);
    if (rc) return rc;
  }
  return a.prompts ? kv8_prefill_join(a.p, dtype, workspace, stream) : AB200_OK;
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
  if (S <= 0 || T <= 0 || Hkv <= 0 || Hq < Hkv || max_rows < 0) return 0;
  // whichever kernels serve the call, however long the sequences, as many rows each or not
  size_t most = 0;
  for (int dtype = AB200_F16; dtype <= AB200_F32; ++dtype)
    for (int ragged = 0; ragged < 2; ++ragged) {
      Kv8Cache c = {};
      Kv8Rows r = {};
      c.H = Hkv, c.shift = 4;
      r.S = S, r.T = T, r.n = T / S, r.max_pages = 1 << 26;
      r.cu = ragged ? (const int32_t *)16 : nullptr;
      AttendPlan a;
      if ((!ragged && T % S) || attend_plan(c, r, max_rows, Hq, dtype, false, &a)) continue;
      if (a.bytes > most) most = a.bytes;
    }
  return most;
}

extern "C" int ab200_kv8_attention(const void *q, long q_stride, void *out, const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale, int pages,
                                   int page_rows, int Hkv, const int32_t *page_table, long table_stride, int max_pages, const int32_t *pos0_dev, const int32_t *cu_rows_dev,
                                   int S, int T, int max_rows, int Hq, int D, float scale, int zero_rest, int dtype, void *workspace, size_t workspace_bytes,
                                   void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  int rc = kv8_check("kv8_attention", false, k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, cu_rows_dev, S, T, &c, &r);
  if (!rc) rc = attention_check("kv8_attention", c, T, q, q_stride, out, Hq, D, dtype);
  if (rc) return rc;
  return attend("kv8_attention", c, r, q, q_stride, out, max_rows, Hq, scale, dtype, nullptr, NewRows{}, false, zero_rest, workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" int ab200_kv8_step(const void *q, const void *k, const void *v, long q_stride, long k_stride, long v_stride, void *out, void *k_cache, void *v_cache,
                              float *k_scale, float *v_scale, int pages, int page_rows, int Hkv, const int32_t *page_table, long table_stride, int max_pages,
                              const int32_t *pos0_dev, int S, int T, int Hq, int D, const float *inv_freq, float scale, int dtype, void *workspace, size_t workspace_bytes,
                              void *stream) {
  clear_error();
  Kv8Cache c;
  Kv8Rows r;
  int rc = kv8_check("kv8_step", true, k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, nullptr, S, T, &c, &r);
  if (!rc) rc = attention_check("kv8_step", c, T, q, q_stride, out, Hq, D, dtype);
  if (rc || S == 0 || T == 0) return rc;
  const long vec = dtype == AB200_F16 ? 8 : 4;
  AB200_REQUIRE(k && v && k_stride % vec == 0 && v_stride % vec == 0 && k_stride >= (long)Hkv * KV8_D && v_stride >= (long)Hkv * KV8_D && aligned16(k) && aligned16(v),
                "kv8_step: k and v must be 16-byte aligned rows of at least %d values, a multiple of 16 bytes apart", Hkv * KV8_D);
  AttendPlan a;
  rc = attend_plan(c, r, T / S, Hq, dtype, inv_freq != nullptr, &a);
  if (rc) return rc;
  AB200_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= a.bytes, "kv8_step: needs a 16-byte aligned workspace of %zu bytes, got %zu", a.bytes, workspace_bytes);
  // fp16 rows that fit into one tile are written by the attention kernel itself where an item is a cluster's (us, together /
  // apart: one request of 384 positions and 32 heads 9.7 / 9.7 step behind step, 13.5 / 15.2 with a read of the rows behind each; in a
  // decoder of 8 layers, 360 positions, 434.7 / 434.0 a token: it saves a launch where something waits for the step, else nothing; 48
  // ragged ones in equal shares 69 / 55: each new block's 4 us then is one CTA's, and the others wait for it at the end).  Else by
  // a launch that the attention kernel starts beside, and only waits for where it reads those rows: 51.3 for the 48, against 54.5 one
  // after the other.
  const bool together = dtype == AB200_F16 && !a.prompts && a.d.splits > 0 && a.d.tiles == 1;
  const bool beside = !together && !a.prompts;
  if (beside) rc = kv8_append_beside(c, r, k, v, k_stride, v_stride, inv_freq, dtype, (cudaStream_t)stream);
  else if (!together)
    rc = ab200_kv8_append(k_cache, v_cache, k_scale, v_scale, pages, page_rows, Hkv, page_table, table_stride, max_pages, pos0_dev, nullptr, S, T, k, v, k_stride, v_stride,
                          nullptr, 0, nullptr, 0, 0, inv_freq, 0, dtype, stream);
  if (rc) return rc;
  return attend("kv8_step", c, r, q, q_stride, out, T / S, Hq, scale, dtype, inv_freq, together ? NewRows{k, v, k_stride, v_stride} : NewRows{}, beside, 0, workspace,
                workspace_bytes, (cudaStream_t)stream);
}
