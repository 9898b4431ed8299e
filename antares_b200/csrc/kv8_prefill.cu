// Attention of many query rows over the 8-bit paged KV cache on the 5th-generation tensor cores (layout: kv8.cuh; the
// mathematics: kv8_attention.cu): x = (q . k_code) scale log2(e) ks + log2(vs), P = 2^(x - m), O += P v_code, l += sum P / vs.
// Codes are fp16 numbers without rounding.  fp32 rows: q and P as pairs of fp16, four products.  fp16 rows: q as it is, P rounded to
// one fp16, once: a weight is off by up to 2^-11 of itself, as the result is by its own rounding.  The kernel over the fp16 cache
// (attention_prefill.cu) holds a pair; here that would be a third product and half as many instructions again for the softmax warps,
// which bound it, over a cache whose codes are 2^-8 apart.  Error of 2000 rows 2.65e-4 of the result, 2.1e-4 if P were exact.
//
// A CTA has 256 packed rows of a kv head (fp32: 128) and walks over 128 keys at a time: four warps bring codes to a ring of
// raw bytes and widen them into swizzled operands, K and V in turn; a warp for each 128 rows issues its products; four warps
// for each 128 rows have a row a thread.  Scores and O lie in tensor memory, P goes back over the scores: the second operand
// of P V is V alone.  Two tiles of rows share the widened keys, and one's exponentials go on under the other's products.  (Two tiles of
// rows in turn, a maximum that is only raised past a threshold and part of the exponentials off their unit are published ideas; the
// kernel, its polynomial and its figures are this project's.)
// Where few tiles of rows would leave SMs idle their keys are cut into up to 8 shares, joined by a second launch.
//
// Bound by the softmax warps: 12 instructions an element, widening included; a fourth of the exponentials are polynomials, since
// the unit makes 16 a cycle.  128 registers, 8 bytes of them spilled.  2000 rows of 32 heads 58.7 us (559 TFLOP/s, a third of a library product's rate; 12000 cycles of a
// CTA are its start and end); 1530 rows of seven sequences, 32 heads over 8 kv heads, behind 8963
// positions 93 us.  Scores taken 32 at a time, in half the code and registers: 60.3 and 98.8; 152 registers for the softmax warps, 80 for
// the loading ones: 58.0 and 93.6.
#include <math_constants.h>

#include <type_traits>

#include "attention_mma.cuh"
#include "kv8.cuh"
#include "kv8_prefill.cuh"

namespace ab200 {

constexpr int KP_BM = 128, KP_BN = 128, KP_LOAD_WARPS = 4, KP_RING = 3, KP_RAW = 4;
constexpr int KP_HALF_BYTES = KP_BN * 128;          // 64 dims of 128 rows, fp16, 128-byte swizzle
constexpr int KP_STAGE_BYTES = 2 * KP_HALF_BYTES;   // a tile of K or of V
constexpr int KP_RAW_BYTES = KP_BN * KV8_D;         // its codes
constexpr int KP_BLOCKS = KP_BN / KV8_BLOCK;
constexpr float KP_RAISE = 8.f, KP_P_EXP = 7.f, KP_LEAST_SCALE = 0x1p-100f;  // P: a row's largest 2^6 at least, since m is raised by whole numbers, and 2^15 at most

template <int TILES, int PARTS>
struct KpShape {
  static constexpr int Q_BYTES = PARTS * KP_STAGE_BYTES;                                    // of one tile of rows
  static constexpr int SMEM = TILES * Q_BYTES + KP_RING * KP_STAGE_BYTES + KP_RAW * KP_RAW_BYTES + 1024;
  static constexpr int SOFT_WARPS = 4 * TILES, LOAD_WARP = SOFT_WARPS, MMA_WARP = SOFT_WARPS + KP_LOAD_WARPS, THREADS = (MMA_WARP + TILES) * 32;
  static constexpr int TMEM_COLS = PARTS == 1 ? 256 * TILES : 512;                          // a tile: S (P over it), O; fp32 rows: the last product too
};

struct KpPair {
  float a, b;
};
__device__ __forceinline__ uint64_t kp_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ KpPair kp_unpack(uint64_t r) {
  KpPair p;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(p.a), "=f"(p.b) : "l"(r));
  return p;
}
__device__ __forceinline__ uint64_t kp_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t kp_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Waits for a barrier's phase; gives up after a while (some milliseconds at least), or soon after another warp has.
__device__ __forceinline__ bool kp_wait(uint32_t bar, unsigned parity, const volatile int *failed) {
  for (int i = 0; i < 64; ++i) {
    if (ap_wait(bar, parity, 1u << 12)) return true;  // a poll may suspend the warp until the phase ends
    if (*failed) return false;
  }
  return false;
}
__device__ __forceinline__ uint64_t kp_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float kp_max_nan(float a, float b) {  // fmaxf would drop a NaN
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 2^a and 2^b, both below 2^127, on the fused multiply-add pipes: y = n + r with r in -1/2 .. 1/2, a polynomial for 2^r fitted for the
// least relative error (2.7e-6, a hundredth of a step of the fp16 it becomes), times 2^n.  n + 127 is what the low bits of the sum
// with `magic` hold, so a shift makes it an exponent: 0, the number 0, for y = -127, which stands for all below.  So a key that is
// masked or far below the others adds nothing, and a NaN stays one.
__device__ __forceinline__ uint64_t kp_exp2(float a, float b) {
  const uint64_t y = kp_pack(kp_max_nan(a, -127.f), kp_max_nan(b, -127.f));
  const uint64_t magic = kp_pack(12583039.f, 12583039.f), minus = kp_pack(-12583039.f, -12583039.f), neg = kp_pack(-1.f, -1.f);  // 1.5 * 2^23 + 127
  auto both = [](float c) { return kp_pack(c, c); };
  const uint64_t n = kp_add2(y, magic), r = kp_fma2(kp_add2(n, minus), neg, y);
  uint64_t e = kp_fma2(both(0.00957010195f), r, both(0.0559178616f));
  e = kp_fma2(e, r, both(0.240247448f));
  e = kp_fma2(e, r, both(0.693121815f));
  e = kp_fma2(e, r, both(0.999999261f));
  const KpPair nn = kp_unpack(n);
  return kp_mul2(e, kp_pack(__int_as_float(__float_as_int(nn.a) << 23), __int_as_float(__float_as_int(nn.b) << 23)));
}
// Nothing uses the loaded registers before this.
__device__ __forceinline__ void kp_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
template <int SEL>
__device__ __forceinline__ uint32_t kp_half2(uint32_t flipped) {  // two codes (flipped to 0 .. 255) as fp16
  return h22u(__hsub2(u2h2(__byte_perm(flipped, 0x64646464u, SEL)), u2h2(0x64806480u)));
}

// The rows of a slot, ROWS packed rows of one sequence.  Sequence s owns the slots from begin(s) group / ROWS + s on: that
// many lie before the next one's.  seq < 0: none.
struct KpRows {
  int seq, row0, rows, first;  // first row of the sequence in q, its packed rows, the slot's first of them
};
template <int ROWS, int THREADS>
__device__ __forceinline__ KpRows kp_rows(const Kv8PrefillParams &p, int slot, int *seq_s) {
  const Kv8Rows &r = p.r;
  if (threadIdx.x == 0) *seq_s = r.cu ? -1 : slot / p.slots_per_seq;
  __syncthreads();
  if (r.cu) {
    for (int s = threadIdx.x; s < r.S; s += THREADS) {
      const long at = (long)r.begin(s) * p.group / ROWS + s, next = s + 1 < r.S ? (long)r.begin(s + 1) * p.group / ROWS + s + 1 : (long)p.slots;
      if (slot >= at && slot < next) *seq_s = s;
    }
    __syncthreads();
  }
  KpRows o;
  o.seq = *seq_s;
  if (o.seq < 0 || o.seq >= r.S) return KpRows{-1, 0, 0, 0};
  o.row0 = r.begin(o.seq), o.rows = max(0, r.end(o.seq) - o.row0) * p.group;
  o.first = (int)(r.cu ? slot - ((long)o.row0 * p.group / ROWS + o.seq) : slot % p.slots_per_seq) * ROWS;
  if (o.first >= o.rows || o.rows <= p.few) o.seq = -1;
  return o;
}

// TILES: tiles of 128 packed query rows that share the CTA's keys.  PARTS: fp16 numbers that a query and a P are held in.
template <typename T, int TILES, int PARTS>
__global__ void __launch_bounds__(KpShape<TILES, PARTS>::THREADS, 1) kv8_prefill_kernel(const __grid_constant__ Kv8PrefillParams p) {
  using Z = KpShape<TILES, PARTS>;
  extern __shared__ unsigned char kp_smem_raw[];
  unsigned char *smem = kp_smem_raw + ((1024u - (ap_smem_u32(kp_smem_raw) & 1023u)) & 1023u);  // swizzle atoms need 1024-byte alignment
  // barriers: full[], empty[], then for each tile: scores of the first 64 keys, of the others, P ready, O done, the others' scores read, the end of all products
  __shared__ __align__(8) uint64_t bars[2 * KP_RING + 6 * TILES];
  __shared__ uint32_t tmem_s;
  __shared__ int fail_s, seq_s;
  __shared__ float2 scales_s[4 * TILES][2][KP_BLOCKS];  // a softmax warp's own, of two tiles: factor of the scores, log2(vs)
  __shared__ float over_s[4 * TILES][2][KP_BLOCKS];     // 1 / vs, times KV8_SUM
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Kv8Rows &r = p.r;
  pdl_wait();

  // ---- which rows
  const int hk = blockIdx.x % p.c.H, slot = p.slots - 1 - (int)(blockIdx.x / p.c.H);  // the last rows have the most keys: they start first
  if (tid == 0) fail_s = 0;
  const KpRows place = kp_rows<TILES * KP_BM, Z::THREADS>(p, slot, &seq_s);
  const int seq = place.seq, row0 = place.row0, rows = place.rows, first = place.first;
  if (seq < 0) return;
  if (PARTS == 1 && warp < Z::SOFT_WARPS) {
    // ---- the queries are on their way first: 16-byte chunk c of row i to half c / 8, chunk position (c % 8) ^ (i % 8)
    const int tile0 = first + (warp >> 2) * KP_BM, last = min(tile0 + KP_BM, rows) - 1, c = tid & 15, i0 = (tid & 127) >> 4;
    const uint32_t dst = ap_smem_u32(smem) + (warp >> 2) * Z::Q_BYTES + (c >> 3) * KP_HALF_BYTES;
    const int step_t = 8 / p.group, step_h = 8 - step_t * p.group;
    int token = (tile0 + i0) / p.group, head = tile0 + i0 - token * p.group;
#pragma unroll 4
    for (int i = i0; i < KP_BM; i += 8) {
      const bool in = tile0 + i <= last;
      const __half *src = (const __half *)p.q + (in ? (size_t)(row0 + token) * p.q_stride + (size_t)(hk * p.group + head) * KV8_D + c * 8 : 0);
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * 128 + (((c & 7) ^ (i & 7)) << 4)), "l"(src), "r"(in ? 16 : 0) : "memory");
      token += step_t, head += step_h;
      if (head >= p.group) head -= p.group, ++token;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const long pos0 = r.pos0[seq], cap = (long)r.max_pages << p.c.shift;
  auto limit_of = [&](int packed) { return (int)max(0l, min(pos0 + packed / p.group + 1, cap)); };
  // key tiles of each tile of rows; this CTA's share of them
  int n_of[TILES], any = 0;
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int f = first + t * KP_BM, lim = f < rows ? limit_of(min(f + KP_BM, rows) - 1) : 0;
    n_of[t] = (lim + KP_BN - 1) / KP_BN;
    any = max(any, lim);
  }
  const int n_all = n_of[TILES - 1] > n_of[0] ? n_of[TILES - 1] : n_of[0];
  const int j0 = p.splits == 1 ? 0 : (int)((long)n_all * blockIdx.y / p.splits), j1 = p.splits == 1 ? n_all : (int)((long)n_all * (blockIdx.y + 1) / p.splits);
#pragma unroll
  for (int t = 0; t < TILES; ++t) n_of[t] = max(0, min(n_of[t], j1) - j0);
  const int n = j1 - j0;

  const uint32_t b_full = ap_smem_u32(bars), b_empty = b_full + 8 * KP_RING, b_tile = b_empty + 8 * KP_RING;
  if (tid == 0) {
    for (int i = 0; i < KP_RING; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b_full + 8 * i), "n"(KP_LOAD_WARPS * 32));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b_empty + 8 * i), "n"(TILES));
    }
    for (int t = 0; t < TILES; ++t) {
      for (int i = 0; i < 6; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b_tile + 48 * t + 8 * i), "r"(i == 2 || i == 4 ? 128 : 1));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  float back = 1.f;  // fp32 queries: what undoes the power of two that a softmax thread's row is scaled by
  if (warp < Z::SOFT_WARPS) {
    const int t = warp >> 2, mine = tid & 127;
    unsigned char *const q_s = smem + t * Z::Q_BYTES;
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;  // a negative scale is the queries': the scores' factors are not negative
    if constexpr (PARTS == 1) {
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (flip) {  // what this thread brought in
        for (int i = mine >> 4; i < KP_BM; i += 8) {
          uint4 &v = *reinterpret_cast<uint4 *>(q_s + ((mine & 15) >> 3) * KP_HALF_BYTES + i * 128 + (((mine & 7) ^ (i & 7)) << 4));
          v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
        }
      }
    } else {
      const int tile0 = first + t * KP_BM, last = min(tile0 + KP_BM, rows) - 1;
      const int packed = tile0 + mine;
      if (packed <= last) {
        // a row a thread: scaled by a power of two, its largest to 2^13 .. 2^14, and cut into two fp16 numbers
        const int token = packed / p.group, head = hk * p.group + packed - token * p.group;
        const float4 *q = reinterpret_cast<const float4 *>((const float *)p.q + (size_t)(row0 + token) * p.q_stride + (size_t)head * KV8_D);
        uint32_t most = 0;
#pragma unroll 8
        for (int c = 0; c < KV8_D / 4; ++c) {
          const float4 v = q[c];
          most = max(max(most, __float_as_uint(v.x) & 0x7fffffffu), max(__float_as_uint(v.y) & 0x7fffffffu, max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu)));
        }
        const int e = 13 - (int)(most >> 23) + 127;  // -115 .. 140
        const float up = kv8_pow2(e >> 1) * (flip ? -1.f : 1.f), up2 = kv8_pow2(e - (e >> 1));
        back = most >= 0x7f800000u ? CUDART_NAN_F : kv8_pow2(-e);
#pragma unroll 4
        for (int c = 0; c < KV8_D / 8; ++c) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 v = q[2 * c + h];
            const float x[4] = {v.x * up * up2, v.y * up * up2, v.z * up * up2, v.w * up * up2};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const __half2 a = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
              const float2 b = __half22float2(a);
              hi[2 * h + i] = h22u(a);
              lo[2 * h + i] = h22u(__floats2half2_rn(x[2 * i] - b.x, x[2 * i + 1] - b.y));
            }
          }
          unsigned char *d = q_s + (c >> 3) * KP_HALF_BYTES + mine * 128 + (((c & 7) ^ (mine & 7)) << 4);
          *reinterpret_cast<uint4 *>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4 *>(d + KP_STAGE_BYTES) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      } else {
#pragma unroll 4
        for (int c = 0; c < KV8_D / 8; ++c) {
          unsigned char *d = q_s + (c >> 3) * KP_HALF_BYTES + mine * 128 + (((c & 7) ^ (mine & 7)) << 4);
          *reinterpret_cast<uint4 *>(d) = *reinterpret_cast<uint4 *>(d + KP_STAGE_BYTES) = make_uint4(0, 0, 0, 0);
        }
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  // ---- the loading warps' way into the cache, and their first three units
  const int32_t *const table = r.table + (size_t)seq * r.table_stride;
  const int lw = warp - Z::LOAD_WARP, row = ((lane >> 2) & 1) + ((lane >> 4) << 1) + 4 * lw, piece = (lane & 3) | (lane >> 3 & 1) << 2;
  const uint32_t sw = row & 7;
  // piece i: chunks 2 i and 2 i + 1 (8 dims each) of the row, in half i / 4
  const uint32_t put = (piece >> 2) * KP_HALF_BYTES + row * 128, c0 = ((2 * piece & 7) ^ sw) << 4, c1 = ((2 * piece + 1 & 7) ^ sw) << 4;
  int where = 0, page = 0, page_at = 0;
  auto ask = [&](int j) {  // the pages of key tile j0 + j's blocks, one a lane of the first eight
    page_at = (j0 + j) * KP_BLOCKS + (lane & 7);
    page = page_at * KV8_BLOCK < any ? table[page_at >> (p.c.shift - 4)] : -1;
  };
  auto lookup = [&](int j) {  // where the blocks lie whose pages were asked for; then asks for the next tile's
    where = -1;
    if (page_at * KV8_BLOCK < any) {
      if ((unsigned)page >= (unsigned)p.c.pages) {
        atomicExch(p.status, KV8_BAD_PAGE);
        page = 0;
      }
      where = ((page * p.c.H + hk) << (p.c.shift - 4)) + (page_at & ((1 << (p.c.shift - 4)) - 1));
    }
    ask(j + 1);
  };
  // a thread's own 16 bytes of each block of a unit: it reads back what it asked for itself
  const uint32_t raw = ap_smem_u32(smem) + TILES * Z::Q_BYTES + KP_RING * KP_STAGE_BYTES + (tid & 127) * 16;
  auto load = [&](int u) {
    if (u < 2 * n) {
      if ((u & 1) == 0) lookup(u >> 1);
      const int8_t *src = (u & 1 ? p.c.v : p.c.k) + row * KV8_D + piece * 16;
#pragma unroll
      for (int i = 0; i < KP_BLOCKS; ++i) {
        const int blk = __shfl_sync(0xffffffffu, where, i);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(raw + u % KP_RAW * KP_RAW_BYTES + i * 2048), "l"(src + (size_t)max(blk, 0) * (KV8_BLOCK * KV8_D)), "r"(blk < 0 ? 0 : 16)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if (warp >= Z::LOAD_WARP && warp < Z::MMA_WARP && n > 0) {
    ask(0);
#pragma unroll
    for (int u = 0; u < KP_RAW - 1; ++u) load(u);
  }
  if (warp == Z::MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ap_smem_u32(&tmem_s)), "n"(Z::TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  pdl_launch_dependents();  // not before the tensor memory is this CTA's: a dependent may hold some while it waits for this grid
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_s, 0);
  const uint32_t q_base = ap_smem_u32(smem), ring = q_base + TILES * Z::Q_BYTES;
  unsigned char *const ring_p = smem + TILES * Z::Q_BYTES;

  if (warp >= Z::LOAD_WARP && warp < Z::MMA_WARP) {
    // ---- K and V tiles in turn through one ring: unit 2 j is K of tile j, 2 j + 1 its V.  The codes of the next three units
    // are on their way while this one's become fp16.  A quarter of a warp stores four even pieces of two neighbouring rows: no
    // two in one bank.
    bool good = true;
    for (int u = 0; u < 2 * n; ++u) {
      asm volatile("cp.async.wait_group %0;" ::"n"(KP_RAW - 2) : "memory");
      uint4 now[KP_BLOCKS];
#pragma unroll
      for (int i = 0; i < KP_BLOCKS; ++i)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(now[i].x), "=r"(now[i].y), "=r"(now[i].z), "=r"(now[i].w) : "r"(raw + u % KP_RAW * KP_RAW_BYTES + i * 2048) : "memory");
      load(u + KP_RAW - 1);
      const int st = u % KP_RING;
      if (u >= KP_RING && !__all_sync(0xffffffffu, kp_wait(b_empty + 8 * st, (u / KP_RING - 1) & 1, &fail_s))) {
        good = false;
        break;
      }
      unsigned char *dst = ring_p + st * KP_STAGE_BYTES + put;
#pragma unroll
      for (int i = 0; i < KP_BLOCKS; ++i) {
        const uint32_t w[4] = {now[i].x ^ 0x80808080u, now[i].y ^ 0x80808080u, now[i].z ^ 0x80808080u, now[i].w ^ 0x80808080u};
        *reinterpret_cast<uint4 *>(dst + i * KV8_BLOCK * 128 + c0) = make_uint4(kp_half2<0x4140>(w[0]), kp_half2<0x4342>(w[0]), kp_half2<0x4140>(w[1]), kp_half2<0x4342>(w[1]));
        *reinterpret_cast<uint4 *>(dst + i * KV8_BLOCK * 128 + c1) = make_uint4(kp_half2<0x4140>(w[2]), kp_half2<0x4342>(w[2]), kp_half2<0x4140>(w[3]), kp_half2<0x4342>(w[3]));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      ap_arrive(b_full + 8 * st);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!good) fail_s = 1;
  } else if (warp >= Z::MMA_WARP) {
    // ---- MMA issue, a warp for each tile of rows.  Scores of a tile of keys are two products, 64 keys each, in the two
    // halves of the tile's columns; its P ends up in the half of the first 64.  The next tile's first 64 keys go where the
    // others lay, as soon as those have been read; its others wait for P's product.  (Two parts of P fill both halves: nothing goes early.)
    const int t = warp - Z::MMA_WARP, my_n = n_of[t];
    const uint32_t bar = b_tile + 48 * t, bar_p = bar + 16, bar_o = bar + 24, bar_r = bar + 32;
    constexpr uint32_t ID_S = (1u << 4) | ((uint32_t)(KP_BN / 2 >> 3) << 17) | ((uint32_t)(KP_BM >> 4) << 24);
    constexpr uint32_t ID_O = (1u << 4) | (1u << 16) | ((uint32_t)(KV8_D >> 3) << 17) | ((uint32_t)(KP_BM >> 4) << 24);  // bit 16: B is MN-major
    bool good = true;
    auto wait = [&](uint32_t b, unsigned parity) { good = good && __all_sync(0xffffffffu, kp_wait(b, parity, &fail_s)); };
    auto scores = [&](int j, int half) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t b0 = ap_desc(ring + (2 * j % KP_RING) * KP_STAGE_BYTES + half * (KP_HALF_BYTES / 2), 16);
      const uint32_t d = tmem + 256 * t + 64 * (PARTS == 1 ? (j & 1) ^ half : half);
#pragma unroll
      for (int part = PARTS - 1; part >= 0; --part) {  // the low parts first: what is cut off a sum goes by its size
        const uint64_t a0 = ap_desc(q_base + t * Z::Q_BYTES + part * KP_STAGE_BYTES, 16);
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // 16 dims further: 32 B inside a swizzled row, four steps per 64-dim half
          const uint64_t step = (uint64_t)((k >> 2) * (KP_HALF_BYTES / 16) + (k & 3) * 2);
          ap_mma_ss(d, a0 + step, b0 + step, ID_S, k > 0 || part < PARTS - 1);
        }
      }
      ap_commit(bar + 8 * half);
    };
    auto values = [&](int j) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t b0 = ap_desc(ring + ((2 * j + 1) % KP_RING) * KP_STAGE_BYTES, KP_HALF_BYTES);
      const uint32_t a0 = tmem + 256 * t + (PARTS == 1 ? 64 * (j & 1) : 0), d = tmem + 256 * t + (PARTS == 1 ? 128 : 256);
#pragma unroll
      for (int part = PARTS - 1; part >= 0; --part)
#pragma unroll
        for (int k = 0; k < 8; ++k)  // 16 keys: two swizzle atoms of V; P lies as 8 columns, of fp32 rows 16 with the first part, 16 with the second
          ap_mma_ts(d, a0 + (PARTS == 1 ? 8 * k : 32 * (k >> 1) + 16 * part + 8 * (k & 1)), b0 + (uint64_t)(k * (2048 / 16)), ID_O,
                    (PARTS == 1 && j > 0) || k > 0 || part < PARTS - 1);
      ap_commit(bar_o);
    };
    // A warp says of every unit that it is done with it, also of one that its tile has no use for: after that unit has come,
    // so that the word is for this turn of the ring.
    auto full = [&](int u) { wait(b_full + 8 * (u % KP_RING), (u / KP_RING) & 1); };
    auto done = [&](int u) { ap_commit(b_empty + 8 * (u % KP_RING)); };
    if (n > 0) {
      full(0);
      if (my_n > 0 && good) scores(0, 0), scores(0, 1);
      done(0);
    }
    for (int j = 0; j < n && good; ++j) {
      full(2 * j + 1);
      if (j + 1 < n) full(2 * j + 2);
      if (PARTS == 1 && j + 1 < my_n) {
        wait(bar_r, j & 1);
        if (good) scores(j + 1, 0);
      }
      if (j < my_n) wait(bar_p, j & 1);
      if (j < my_n && good) values(j);
      done(2 * j + 1);
      if (j + 1 == n || !good) break;
      if (j + 1 < my_n) {
        wait(bar_o, j & 1);
        if (PARTS == 2 && good) scores(j + 1, 0);
        if (good) scores(j + 1, 1);
      }
      done(2 * j + 2);
    }
    // every product and every arrival of a commit has to be over before this memory is another CTA's
    ap_commit(bar + 40);
    if (!__all_sync(0xffffffffu, ap_wait(bar + 40, 0, 1u << 18))) good = false;
    if (!good) fail_s = 1;
  } else {
    // ---- softmax: thread = packed row first + 128 t + (tid & 127); its tensor memory lanes are the warp's of its four
    const int t = warp >> 2, mine = tid & 127, tile0 = first + t * KP_BM;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + 256 * t + lanes, to = ts + 128, bar = b_tile + 48 * t, bar_p = bar + 16, bar_o = bar + 24, bar_r = bar + 32;
    unsigned char *const q_s = smem + t * Z::Q_BYTES;
    const int my_n = n_of[t], packed = tile0 + mine, last = min(tile0 + KP_BM, rows) - 1;
    const int limit = packed <= last ? limit_of(packed) : 0;
    const float scale = fabsf(p.scale);
    float ks_next = 0.f, vs_next = 1.f;
    int page = 0;
    auto block_of = [&](int j) { return (j0 + j) * KP_BLOCKS + lane; };  // a block of key tile j0 + j for each of the first eight lanes
    auto ask_page = [&](int j) { page = lane < KP_BLOCKS && block_of(j) * KV8_BLOCK < any ? table[block_of(j) >> (p.c.shift - 4)] : -1; };
    auto ask = [&](int j) {  // the scales of tile j, whose pages have come; then the pages of the next
      ks_next = 0.f, vs_next = 1.f;
      if ((unsigned)page < (unsigned)p.c.pages) {
        const size_t at = ((size_t)(page * p.c.H + hk) << (p.c.shift - 4)) + (block_of(j) & ((1 << (p.c.shift - 4)) - 1));
        ks_next = p.c.ks[at], vs_next = p.c.vs[at];
      }
      ask_page(j + 1);
    };
    if (my_n > 0) ask_page(0), ask(0);
    float m = -CUDART_INF_F, l = 0.f;
    bool good = true;
    auto scales = [&](int j) {  // of tile j, whose values have come, to shared memory; asks for the next tile's
      if (lane < KP_BLOCKS) {
        const float vs = fmaxf(vs_next, KP_LEAST_SCALE);
        scales_s[warp][j & 1][lane] = make_float2(ks_next * scale, __log2f(vs)), over_s[warp][j & 1][lane] = __fdividef(KV8_SUM, vs);
      }
      ask(j + 1);
    };
    if (my_n > 0) scales(0);
    // fp32 rows: 16 dims of O with the product of tile j, which is complete, added.  The tensor cores cut what they add to 24 bits at
    // every step, always towards zero: over 16000 keys in one sum 5e-6 of it.  So a tile's product is a sum of its own, 2e-7 at most
    // with the low parts first, and joins the others by an addition that rounds.  2000 rows of 32 heads 145 -> 158 us; 32 dims at a time 161.
    auto sum_of = [&](int d, int j, uint32_t (&o)[16]) {
      uint32_t had[16];
      ap_ld16(to + 128 + d, o);
      if (j > 0) ap_ld16(to + d, had);
      ap_wait_ld();
      if (j > 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(had[i]) + __uint_as_float(o[i]));
      }
    };
    for (int j = 0; j < my_n; ++j) {
      const float2(&sc)[KP_BLOCKS] = scales_s[warp][j & 1];
      const float(&over_vs)[KP_BLOCKS] = over_s[warp][j & 1];
      __syncwarp();
      if (PARTS == 2 && j > 0) {  // meanwhile the product of the tile before is added to O
        good = __all_sync(0xffffffffu, kp_wait(bar_o, (j - 1) & 1, &fail_s));
        if (!good) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
        for (int d = 0; d < KV8_D; d += 16) {
          uint32_t o[16];
          sum_of(d, j - 1, o);
          ap_st16(to + d, o);
        }
        ap_wait_st();
      }
      if (!__all_sync(0xffffffffu, kp_wait(bar, j & 1, &fail_s))) {
        good = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int left = limit - (j0 + j) * KP_BN;  // keys of this tile the row attends to
      const bool all = __all_sync(0xffffffffu, left >= KP_BN || packed > last);
      const uint32_t t_first = ts + (PARTS == 1 ? 64 * (j & 1) : 0), t_other = ts + (PARTS == 1 ? 64 * (j & 1 ^ 1) : 64);
      auto p_at = [&](int c) { return PARTS == 1 ? t_first + 16 * c : ts + 32 * c; };  // P of 32 keys
      // 64 keys of the row: their largest exponent, then P = 2^(x - m + 7)
      auto half = [&](int hb, auto all_keys) {
        constexpr bool ALL = decltype(all_keys)::value;
        uint32_t s0[32] = {}, s1[32] = {};
        auto s = [&](int i) { return __uint_as_float(i < 32 ? s0[i & 31] : s1[i & 31]); };
        const uint32_t at = hb ? t_other : t_first;
        ap_ld32(at, s0);
        ap_ld32(at + 32, s1);
        if (hb == 1) scales(j + 1);
        float f[4], lv[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float2 q = sc[4 * hb + b];
          f[b] = PARTS == 1 ? q.x : q.x * back, lv[b] = q.y;
        }
        const int mine = left - 64 * hb;
        kp_wait_ld(s0);
        kp_wait_ld(s1);
        if (PARTS == 1 && hb == 1) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          ap_arrive(bar_r);
        }
        float mx = -CUDART_INF_F;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int i = 16 * b; i < 16 * b + 16; i += 2) {
            const float u = ALL || i < mine ? s(i) : -CUDART_INF_F, v = ALL || i + 1 < mine ? s(i + 1) : -CUDART_INF_F;
            top[i >> 1 & 1] = fmaxf(top[i >> 1 & 1], fmaxf(u, v));
          }
          const float t = fmaxf(top[0], top[1]);
          mx = fmaxf(mx, !ALL && t == -CUDART_INF_F ? t : fmaf(t, f[b], lv[b]));
        }
        const bool raise = mx > m + KP_RAISE;
        if (__any_sync(0xffffffffu, raise)) {
          // by a whole number: O, l and what is held of P are scaled by a power of two, which rounds nothing.  From nothing to the
          // maximum itself: the largest P of a row's first keys, often its largest of all, is a power of two then.
          const float d = raise ? ceilf(mx - m) : 0.f, up = m == -CUDART_INF_F ? mx : m + d, by = d > 126.f ? 0.f : kv8_pow2(-(int)d);
          m = up;
          l *= by;
          ap_wait_st();
          if (j > 0) {  // O: the other half of these scores waits for the product of the tile before
            if (PARTS == 1 && hb == 0 && !__all_sync(0xffffffffu, kp_wait(bar_o, (j - 1) & 1, &fail_s))) fail_s = 1;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
            for (int d = 0; d < KV8_D; d += 16) {
              uint32_t o[16];
              ap_ld16(to + d, o);
              ap_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
              ap_st16(to + d, o);
            }
          }
#pragma unroll 1
          for (int c = 0; c < 2 * hb; ++c) {  // P of this tile's first keys
            uint32_t hi[16];
            [[maybe_unused]] uint32_t lo[PARTS == 1 ? 1 : 16];
            ap_ld16(p_at(c), hi);
            if constexpr (PARTS == 2) ap_ld16(p_at(c) + 16, lo);
            ap_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float2 v = __half22float2(u2h2(hi[i]));
              if constexpr (PARTS == 2) {
                const float2 w = __half22float2(u2h2(lo[i]));
                v.x = (v.x + w.x) * by, v.y = (v.y + w.y) * by;
                const __half2 h = __floats2half2_rn(v.x, v.y);
                const float2 hf = __half22float2(h);
                hi[i] = h22u(h), lo[i] = h22u(__floats2half2_rn(v.x - hf.x, v.y - hf.y));
              } else {
                hi[i] = h22u(__floats2half2_rn(v.x * by, v.y * by));
              }
            }
            ap_st16(p_at(c), hi);
            if constexpr (PARTS == 2) ap_st16(p_at(c) + 16, lo);
          }
        }
        const float shift = m == -CUDART_INF_F ? 0.f : m - KP_P_EXP;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t hi[16];
          [[maybe_unused]] uint32_t lo[PARTS == 1 ? 1 : 16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int b = 2 * c + h;
            const uint64_t f2 = kp_pack(f[b], f[b]), d2 = kp_pack(lv[b] - shift, lv[b] - shift);
            uint64_t sum = kp_pack(0.f, 0.f);
#pragma unroll
            for (int i = 8 * h; i < 8 * h + 8; ++i) {
              const int k = 32 * c + 2 * i;
              KpPair v = kp_unpack(kp_fma2(kp_pack(s(k), s(k + 1)), f2, d2));
              if constexpr (!ALL) v.a = k < mine ? v.a : -CUDART_INF_F, v.b = k + 1 < mine ? v.b : -CUDART_INF_F;
              float a, b2;
              if (PARTS == 1 && i % 4 == 3) {  // a quarter of them off the exponential unit
                const KpPair e = kp_unpack(kp_exp2(v.a, v.b));
                a = e.a, b2 = e.b;
              } else {
                a = ap_ex2(v.a), b2 = ap_ex2(v.b);
              }
              sum = kp_add2(sum, kp_pack(a, b2));
              const __half2 hh = __floats2half2_rn(a, b2);
              hi[i] = h22u(hh);
              if constexpr (PARTS == 2) {
                const float2 hf = __half22float2(hh);
                lo[i] = h22u(__floats2half2_rn(a - hf.x, b2 - hf.y));
              }
            }
            const KpPair both = kp_unpack(sum);
            l = fmaf(both.a + both.b, over_vs[4 * hb + b], l);
          }
          ap_st16(p_at(2 * hb + c), hi);
          if constexpr (PARTS == 2) ap_st16(p_at(2 * hb + c) + 16, lo);
        }
      };
#pragma unroll 1
      for (int hb = 0; hb < 2; ++hb) {
        if (hb > 0) {
          good = __all_sync(0xffffffffu, kp_wait(bar + 8, j & 1, &fail_s));
          if (!good) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        if (all) {
          half(hb, std::true_type{});
        } else if (__any_sync(0xffffffffu, left > 64 * hb)) {
          half(hb, std::false_type{});
        } else {  // no row of the warp attends to any of these keys
          const uint32_t none[16] = {};
#pragma unroll
          for (int c = 0; c < (PARTS == 1 ? 2 : 4); ++c) ap_st16((PARTS == 1 ? t_first + 32 * hb : ts + 64 * hb) + 16 * c, none);
          if (hb == 1) {
            scales(j + 1);
            if (PARTS == 1) ap_arrive(bar_r);
          }
        }
      }
      if (!good) break;
      ap_wait_st();
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      ap_arrive(bar_p);
    }
    // ---- O / l: a thread's row through its own idle query memory, then stored as whole rows; or its part, to be joined
    // The product before the last is complete: the last scores' second half was only issued after it.  A wait for it here could
    // come after the last one has ended too, whose phase looks like the one before it.
    if (good && my_n > 0) good = __all_sync(0xffffffffu, kp_wait(bar_o, (my_n - 1) & 1, &fail_s));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    auto read_o = [&](int d, uint32_t (&o)[32]) {
      if constexpr (PARTS == 1) {
        ap_ld32(to + d, o);
        ap_wait_ld();
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t part[16];
          sum_of(d + 16 * h, my_n - 1, part);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[16 * h + i] = part[i];
        }
      }
    };
    if (!good) {
      fail_s = 1;
    } else if (tile0 <= last) {
      if (p.splits > 1) {
        const size_t at = (((size_t)slot * p.c.H + hk) * p.splits + blockIdx.y) * (TILES * KP_BM) + t * KP_BM + mine;
        float *o_part = p.partial + at * KV8_D;
        if (my_n > 0) {
#pragma unroll 1
          for (int d = 0; d < KV8_D; d += 32) {
            uint32_t o[32];
            read_o(d, o);
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4 *>(o_part + d + 4 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
        p.partial_ml[at] = make_float2(my_n > 0 ? m : -CUDART_INF_F, my_n > 0 ? l : 0.f);
      } else {
        const float over = limit > 0 ? KV8_SUM / l : 0.f;
        constexpr int CHUNKS = KV8_D * sizeof(T) / 16, EACH = 16 / sizeof(T);
        unsigned char *park = q_s + mine * (KV8_D * sizeof(T));
#pragma unroll 1
        for (int d = 0; d < KV8_D; d += 32) {
          uint32_t o[32];
          if (my_n > 0) {
            read_o(d, o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
#pragma unroll
          for (int i = 0; i < 32 / EACH; ++i) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (sizeof(T) == 2) {
                const float a = __uint_as_float(o[8 * i + 2 * e]) * over, b = __uint_as_float(o[8 * i + 2 * e + 1]) * over;
                u[e] = limit > 0 ? h22u(__floats2half2_rn(a, b)) : 0u;
              } else {
                u[e] = limit > 0 ? __float_as_uint(__uint_as_float(o[4 * i + e]) * over) : 0u;
              }
            }
            *reinterpret_cast<uint4 *>(park + (((d / EACH + i) ^ (mine & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
          }
        }
        __syncwarp();
        // the warp's 32 rows, CHUNKS lanes a row
        const int c = lane % CHUNKS;
        constexpr int STEP = 32 / CHUNKS;
        const int from = (warp & 3) * 32 + lane / CHUNKS, step_t = STEP / p.group, step_h = STEP - step_t * p.group;
        int token = (tile0 + from) / p.group, head = tile0 + from - token * p.group;
#pragma unroll 4
        for (int in_tile = from; in_tile < from + 32 && tile0 + in_tile <= last; in_tile += STEP) {
          const uint4 v = *reinterpret_cast<const uint4 *>(q_s + in_tile * (KV8_D * sizeof(T)) + ((c ^ (in_tile & 7)) << 4));
          *reinterpret_cast<uint4 *>((T *)p.out + ((size_t)(row0 + token) * p.Hq + hk * p.group + head) * KV8_D + c * EACH) = v;
          token += step_t, head += step_h;
          if (head >= p.group) head -= p.group, ++token;
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == Z::MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Z::TMEM_COLS) : "memory");
  if (fail_s && tid == 0) atomicExch(p.status, 710);  // site 710: a wait of the 8-bit prompt attention ran out
}

// Joins the shares of the keys: a warp a packed row.
constexpr int KP_JOIN_WARPS = 8;
template <typename T, int ROWS>
__global__ void __launch_bounds__(KP_JOIN_WARPS * 32) kv8_prefill_join_kernel(const __grid_constant__ Kv8PrefillParams p) {
  __shared__ int seq_s;
  pdl_launch_dependents();
  pdl_wait();
  const int hk = blockIdx.x % p.c.H, slot = (int)(blockIdx.x / p.c.H), lane = threadIdx.x & 31, row = blockIdx.y * KP_JOIN_WARPS + (threadIdx.x >> 5);
  const KpRows place = kp_rows<ROWS, KP_JOIN_WARPS * 32>(p, slot, &seq_s);
  const int packed = place.first + row;
  if (place.seq < 0 || packed >= place.rows) return;
  float m = -CUDART_INF_F, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int z = 0; z < p.splits; ++z) {
    const size_t at = (((size_t)slot * p.c.H + hk) * p.splits + z) * ROWS + row;
    const float2 ml = p.partial_ml[at];
    if (ml.y == 0.f) continue;  // no key of any weight there, perhaps nothing written (a sum that is not a number is not 0)
    const float4 v = reinterpret_cast<const float4 *>(p.partial + at * KV8_D)[lane];
    const float up = fmaxf(m, ml.x), f = m == -CUDART_INF_F ? 0.f : ap_ex2(m - up), fc = ml.x == -CUDART_INF_F ? 1.f : ap_ex2(ml.x - up);
    l = l * f + ml.y * fc;
    acc.x = acc.x * f + v.x * fc, acc.y = acc.y * f + v.y * fc, acc.z = acc.z * f + v.z * fc, acc.w = acc.w * f + v.w * fc;
    m = up;
  }
  const int token = packed / p.group, head = hk * p.group + packed - token * p.group;
  T *out = (T *)p.out + ((size_t)(place.row0 + token) * p.Hq + head) * KV8_D + 4 * lane;
  const float x[4] = {acc.x, acc.y, acc.z, acc.w};
  const bool none = p.r.pos0[place.seq] + (long)(packed / p.group) < 0;  // nothing to attend to; keys whose scores are all -inf have no softmax: 0 / 0
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)(none ? 0.f : x[e] * (KV8_SUM / l));
}

template <typename T, int TILES, int PARTS>
static int prefill_launch(const Kv8PrefillParams &p, cudaStream_t stream) {
  using Z = KpShape<TILES, PARTS>;
  AB200_CUDA(cudaFuncSetAttribute(kv8_prefill_kernel<T, TILES, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::SMEM));
  AB200_CUDA(launch_pdl(kv8_prefill_kernel<T, TILES, PARTS>, dim3((unsigned)(p.slots * p.c.H), p.splits), dim3(Z::THREADS), Z::SMEM, stream, p));
  return AB200_OK;
}

// Tiles of rows, and how the keys are shared out where those alone would leave most SMs idle.
int kv8_prefill_plan(Kv8PrefillParams *p, int dtype, long capacity, size_t *bytes) {
  const int rows = dtype == AB200_F16 ? 256 : 128;
  p->slots_per_seq = (int)(((long)p->r.n * p->group + rows - 1) / rows);
  const long slots = p->r.cu ? (long)p->r.T * p->group / rows + p->r.S : (long)p->r.S * p->slots_per_seq, items = slots * p->c.H;
  AB200_REQUIRE(items < 1l << 31, "kv8_attention: %ld tiles of rows are beyond the built limits", items);
  p->slots = (int)slots;
  // each share two tiles of keys at least; at most one CTA an SM, so that the parts stay within 20 MB
  long splits = sm_count() / items;
  if (splits > 8) splits = 8;
  if (splits > capacity / (2 * KP_BN)) splits = capacity / (2 * KP_BN);
  p->splits = splits > 1 ? (int)splits : 1;
  *bytes = p->splits > 1 ? (size_t)items * p->splits * rows * (KV8_D + 2) * sizeof(float) : 0;
  return AB200_OK;
}

int kv8_prefill(Kv8PrefillParams p, int dtype, void *workspace, cudaStream_t stream) {
  p.partial = (float *)workspace;
  p.partial_ml = (float2 *)(p.partial + (size_t)p.slots * p.c.H * p.splits * (dtype == AB200_F16 ? 256 : 128) * KV8_D);
  return dtype == AB200_F16 ? prefill_launch<__half, 2, 1>(p, stream) : prefill_launch<float, 1, 2>(p, stream);
}

int kv8_prefill_join(Kv8PrefillParams p, int dtype, void *workspace, cudaStream_t stream) {
  if (p.splits == 1) return AB200_OK;
  p.partial = (float *)workspace;
  p.partial_ml = (float2 *)(p.partial + (size_t)p.slots * p.c.H * p.splits * (dtype == AB200_F16 ? 256 : 128) * KV8_D);
  if (dtype == AB200_F16)
    AB200_CUDA(launch_pdl(kv8_prefill_join_kernel<__half, 256>, dim3((unsigned)(p.slots * p.c.H), 256 / KP_JOIN_WARPS), dim3(KP_JOIN_WARPS * 32), 0, stream, p));
  else
    AB200_CUDA(launch_pdl(kv8_prefill_join_kernel<float, 128>, dim3((unsigned)(p.slots * p.c.H), 128 / KP_JOIN_WARPS), dim3(KP_JOIN_WARPS * 32), 0, stream, p));
  return AB200_OK;
}

}  // namespace ab200
