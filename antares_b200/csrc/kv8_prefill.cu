// Attention of many query rows over the 8-bit paged KV cache on the 5th-generation tensor cores (layout: kv8.cuh; the
// mathematics: kv8_attention.cu): x = (q . k_code) scale log2(e) ks + log2(vs), P = 2^(x - m), O += P v_code, l += sum P / vs.
#include <math_constants.h>

#include "attention_mma.cuh"
#include "kv8.cuh"
#include "kv8_prefill.cuh"

namespace ab200 {

constexpr int KP_BM = 128, KP_BN = 128, KP_LOAD_WARPS = 4, KP_RING = 3, KP_RAW = 4;
constexpr int KP_HALF_BYTES = KP_BN * 128;          // 64 dims of 128 rows, fp16, 128-byte swizzle
constexpr int KP_STAGE_BYTES = 2 * KP_HALF_BYTES;   // a tile of K or of V
constexpr int KP_RAW_BYTES = KP_BN * KV8_D;         // its codes
constexpr int KP_BLOCKS = KP_BN / KV8_BLOCK;
constexpr float KP_RAISE = 8.f, KP_P_EXP = 6.f, KP_LEAST_SCALE = 0x1p-100f;

template <int TILES, int PARTS>
struct KpShape {
  static constexpr int Q_BYTES = PARTS * KP_STAGE_BYTES;                                    // of one tile of rows
  static constexpr int SMEM = TILES * Q_BYTES + KP_RING * KP_STAGE_BYTES + KP_RAW * KP_RAW_BYTES + 1024;
  static constexpr int SOFT_WARPS = 4 * TILES, LOAD_WARP = SOFT_WARPS, MMA_WARP = SOFT_WARPS + KP_LOAD_WARPS, THREADS = (MMA_WARP + TILES) * 32;
  static constexpr int TMEM_COLS = 256 * TILES;                                             // a tile: S (P over it), O
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
    if (ap_wait(bar, parity, 1u << 12)) return true;
    if (*failed) return false;
  }
  return false;
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

// TILES: tiles of 128 packed query rows that share the CTA's keys.  PARTS: fp16 numbers that a query and a P are held in.
template <typename T, int TILES, int PARTS>
__global__ void __launch_bounds__(KpShape<TILES, PARTS>::THREADS, 1) kv8_prefill_kernel(const __grid_constant__ Kv8PrefillParams p) {
  using Z = KpShape<TILES, PARTS>;
  extern __shared__ unsigned char kp_smem_raw[];
  unsigned char *smem = kp_smem_raw + ((1024u - (ap_smem_u32(kp_smem_raw) & 1023u)) & 1023u);  // swizzle atoms need 1024-byte alignment
  // barriers: full[], empty[], then for each tile: scores ready, P ready, O done, the end of all its products
  __shared__ __align__(8) uint64_t bars[2 * KP_RING + 4 * TILES];
  __shared__ uint32_t tmem_s;
  __shared__ int fail_s, seq_s;
  __shared__ float4 scales_s[4 * TILES][KP_BLOCKS];  // a softmax warp's own: factor of the scores, log2(vs), 1 / vs
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Kv8Rows &r = p.r;
  pdl_wait();

  // ---- which rows: pairs of tiles of one sequence and kv head.  Sequence s owns the slots from begin(s) group / 256 + s on.
  const int hk = blockIdx.x % p.c.H, slot = p.slots - 1 - (int)(blockIdx.x / p.c.H);  // the last rows have the most keys: they start first
  constexpr int ROWS = TILES * KP_BM;
  if (tid == 0) seq_s = r.cu ? -1 : slot / p.slots_per_seq, fail_s = 0;
  __syncthreads();
  if (r.cu) {
    for (int s = tid; s < r.S; s += Z::THREADS) {
      const long at = (long)r.begin(s) * p.group / ROWS + s, next = s + 1 < r.S ? (long)r.begin(s + 1) * p.group / ROWS + s + 1 : (long)p.slots;
      if (slot >= at && slot < next) seq_s = s;
    }
    __syncthreads();
  }
  const int seq = seq_s;
  if (seq < 0 || seq >= r.S) return;
  const int row0 = r.begin(seq), rows = max(0, r.end(seq) - row0) * p.group;
  const int first = (int)(r.cu ? slot - ((long)row0 * p.group / ROWS + seq) : slot % p.slots_per_seq) * ROWS;
  if (first >= rows || rows <= p.few) return;
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
  const int j0 = (int)((long)n_all * blockIdx.y / p.splits), j1 = (int)((long)n_all * (blockIdx.y + 1) / p.splits);
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
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(b_tile + 32 * t));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 128;" ::"r"(b_tile + 32 * t + 8));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(b_tile + 32 * t + 16));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(b_tile + 32 * t + 24));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
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
  const int32_t *const table = r.table + (size_t)seq * r.table_stride;

  if (warp >= Z::LOAD_WARP && warp < Z::MMA_WARP) {
    // ---- K and V tiles in turn through one ring: unit 2 j is K of tile j, 2 j + 1 its V.  The codes of the next three units
    // are on their way while this one's become fp16.  A quarter of a warp stores four even pieces of two neighbouring rows: no
    // two in one bank.
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
    const uint32_t raw = ap_smem_u32(smem) + TILES * Z::Q_BYTES + KP_RING * KP_STAGE_BYTES + (tid - Z::LOAD_WARP * 32) * 16;
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
    bool good = true;
    if (n > 0) ask(0);
#pragma unroll
    for (int u = 0; u < KP_RAW - 1; ++u) load(u);
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
    // ---- MMA issue, a warp for each tile of rows.  Its scores go where its P lay, so they wait for that P's product;
    // meanwhile the other tile's are under way.
    const int t = warp - Z::MMA_WARP, my_n = n_of[t];
    const uint32_t bar = b_tile + 32 * t;
    constexpr uint32_t ID_S = (1u << 4) | ((uint32_t)(KP_BN >> 3) << 17) | ((uint32_t)(KP_BM >> 4) << 24);
    constexpr uint32_t ID_O = (1u << 4) | (1u << 16) | ((uint32_t)(KV8_D >> 3) << 17) | ((uint32_t)(KP_BM >> 4) << 24);  // bit 16: B is MN-major
    bool good = true;
    auto wait = [&](uint32_t b, unsigned parity) { good = good && __all_sync(0xffffffffu, kp_wait(b, parity, &fail_s)); };
    auto scores = [&](int j) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t b0 = ap_desc(ring + (2 * j % KP_RING) * KP_STAGE_BYTES, 16);
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        const uint64_t a0 = ap_desc(q_base + t * Z::Q_BYTES + part * KP_STAGE_BYTES, 16);
#pragma unroll
        for (int k = 0; k < 8; ++k) {  // 16 dims further: 32 B inside a swizzled row, four steps per 64-dim half
          const uint64_t step = (uint64_t)((k >> 2) * (KP_HALF_BYTES / 16) + (k & 3) * 2);
          ap_mma_ss(tmem + 256 * t, a0 + step, b0 + step, ID_S, k > 0 || part > 0);
        }
      }
      ap_commit(bar);
    };
    auto values = [&](int j) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t b0 = ap_desc(ring + ((2 * j + 1) % KP_RING) * KP_STAGE_BYTES, KP_HALF_BYTES);
      const uint32_t a0 = tmem + 256 * t, d = a0 + 128;
#pragma unroll
      for (int k = 0; k < 8; ++k)  // 16 keys: two swizzle atoms of V; P lies as 8 columns, of fp32 rows 16 with the first part, 16 with the second
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
          ap_mma_ts(d, a0 + (PARTS == 1 ? 8 * k : 32 * (k >> 1) + 16 * part + 8 * (k & 1)), b0 + (uint64_t)(k * (2048 / 16)), ID_O, j > 0 || k > 0 || part > 0);
      ap_commit(bar + 16);
    };
    // A warp says of every unit that it is done with it, also of one that its tile has no use for: after that unit has come,
    // so that the word is for this turn of the ring.
    auto full = [&](int u) { wait(b_full + 8 * (u % KP_RING), (u / KP_RING) & 1); };
    auto done = [&](int u) { ap_commit(b_empty + 8 * (u % KP_RING)); };
    if (n > 0) {
      if (my_n > 0) wait(bar + 8, 0);  // queries are in shared memory: the softmax warps' first arrival at "P ready"
      full(0);
      if (my_n > 0 && good) scores(0);
      done(0);
    }
    for (int j = 0; j < n && good; ++j) {
      full(2 * j + 1);
      if (j < my_n) {
        wait(bar + 8, (j + 1) & 1);
        if (good) values(j);
      }
      done(2 * j + 1);
      if (j + 1 == n || !good) break;
      full(2 * j + 2);
      if (j + 1 < my_n) {
        wait(bar + 16, j & 1);
        if (good) scores(j + 1);
      }
      done(2 * j + 2);
    }
    // every product and every arrival of a commit has to be over before this memory is another CTA's
    ap_commit(bar + 24);
    if (!__all_sync(0xffffffffu, ap_wait(bar + 24, 0, 1u << 18))) good = false;
    if (!good) fail_s = 1;
  } else {
    // ---- softmax: thread = packed row first + 128 t + (tid & 127); its tensor memory lanes are the warp's of its four
    const int t = warp >> 2, mine = tid & 127, tile0 = first + t * KP_BM;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + 256 * t + lanes, to = ts + 128, bar = b_tile + 32 * t;
    unsigned char *const q_s = smem + t * Z::Q_BYTES;
    const int my_n = n_of[t], packed = tile0 + mine, last = min(tile0 + KP_BM, rows) - 1;
    const int limit = packed <= last ? limit_of(packed) : 0;
    float back = 1.f;
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;  // a negative scale is the queries': factors below are not negative
    if (my_n > 0) {
      if constexpr (PARTS == 1) {
        // 16-byte chunk c of row i to half c / 8, chunk position (c % 8) ^ (i % 8)
        const int c = mine & 15;
#pragma unroll 4
        for (int i = mine >> 4; i < KP_BM; i += 8) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (tile0 + i <= last) {
            const int token = (tile0 + i) / p.group, head = hk * p.group + tile0 + i - token * p.group;
            v = *reinterpret_cast<const uint4 *>((const __half *)p.q + (size_t)(row0 + token) * p.q_stride + (size_t)head * KV8_D + c * 8);
          }
          v.x ^= flip, v.y ^= flip, v.z ^= flip, v.w ^= flip;
          *reinterpret_cast<uint4 *>(q_s + (c >> 3) * KP_HALF_BYTES + i * 128 + (((c & 7) ^ (i & 7)) << 4)) = v;
        }
      } else if (packed <= last) {
        // a row a thread: scaled by a power of two, its largest to 2^13 .. 2^14, and cut into two fp16 numbers
        const int token = packed / p.group, head = hk * p.group + packed - token * p.group;
        const float4 *q = reinterpret_cast<const float4 *>((const float *)p.q + (size_t)(row0 + token) * p.q_stride + (size_t)head * KV8_D);
        uint32_t most = 0;
#pragma unroll 8
        for (int c = 0; c < KV8_D / 4; ++c) {
          const float4 v = q[c];
          most = max(max(most, __float_as_uint(v.x) & 0x7fffffffu), max(__float_as_uint(v.y) & 0x7fffffffu, max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu)));
        }
        const int e = max(-100, min(100, 13 - (int)(most >> 23) + 127));
        const float up = __int_as_float((127 + e) << 23) * (flip ? -1.f : 1.f);
        back = most >= 0x7f800000u ? CUDART_NAN_F : __int_as_float((127 - e) << 23);
#pragma unroll 4
        for (int c = 0; c < KV8_D / 8; ++c) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 v = q[2 * c + h];
            const float x[4] = {v.x * up, v.y * up, v.z * up, v.w * up};
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
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      ap_arrive(bar + 8);
    }
    const float scale = fabsf(p.scale);
    float ks_next = 0.f, vs_next = 1.f;
    auto ask = [&](int j) {  // the scales of key tile j0 + j, a block each for the first eight lanes
      const int b = (j0 + j) * KP_BLOCKS + lane;
      ks_next = 0.f, vs_next = 1.f;
      if (lane < KP_BLOCKS && b * KV8_BLOCK < any) {
        const int page = table[b >> (p.c.shift - 4)];
        if ((unsigned)page < (unsigned)p.c.pages) {
          const size_t at = ((size_t)(page * p.c.H + hk) << (p.c.shift - 4)) + (b & ((1 << (p.c.shift - 4)) - 1));
          ks_next = p.c.ks[at], vs_next = p.c.vs[at];
        }
      }
    };
    if (my_n > 0) ask(0);
    float m = -CUDART_INF_F, l = 0.f;
    bool good = true;
    float4(&sc)[KP_BLOCKS] = scales_s[warp];
    for (int j = 0; j < my_n; ++j) {
      __syncwarp();
      if (lane < KP_BLOCKS) {
        const float vs = fmaxf(vs_next, KP_LEAST_SCALE);
        sc[lane] = make_float4(ks_next * scale, __log2f(vs), __fdividef(1.f, vs), 0.f);
      }
      __syncwarp();
      if (j + 1 < my_n) ask(j + 1);
      if (!__all_sync(0xffffffffu, kp_wait(bar, j & 1, &fail_s))) {
        good = false;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const int left = limit - (j0 + j) * KP_BN;  // keys of this tile the row attends to
      const bool all = __all_sync(0xffffffffu, left >= KP_BN || packed > last);
      // 32 keys of the row: y = x - m + 6, and P = 2^y where no y is above 14
      auto chunk = [&](int c, uint32_t(&s)[32], uint32_t(&next)[32]) {
        uint64_t y[16];
        float f[2], lv[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 q = sc[2 * c + h];
          f[h] = PARTS == 1 ? q.x : q.x * back, lv[h] = q.y;
        }
        auto exponents = [&](float shift) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint64_t f2 = kp_pack(f[h], f[h]), d2 = kp_pack(lv[h] - shift, lv[h] - shift);
#pragma unroll
            for (int i = 8 * h; i < 8 * h + 8; ++i) y[i] = kp_fma2(kp_pack(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), f2, d2);
          }
          if (!all) {
            const int mine = left - 32 * c;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const KpPair v = kp_unpack(y[i]);
              y[i] = kp_pack(2 * i < mine ? v.a : -CUDART_INF_F, 2 * i + 1 < mine ? v.b : -CUDART_INF_F);
            }
          }
          float top[2] = {-CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const KpPair v = kp_unpack(y[i]);
            top[i & 1] = fmaxf(top[i & 1], fmaxf(v.a, v.b));
          }
          return fmaxf(top[0], top[1]);
        };
        const bool raise = exponents(m - KP_P_EXP) > KP_P_EXP + KP_RAISE;  // m = -inf: any key raises it
        if (__any_sync(0xffffffffu, raise)) {
          const float top = exponents(0.f), up = raise ? top : m, by = up == m ? 1.f : m == -CUDART_INF_F ? 0.f : ap_ex2(m - up);
          m = up;
          l *= by;
          ap_wait_st();
          if (j > 0) {  // O: these scores waited for the product of the tile before
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
          for (int b = 0; b < c; ++b) {  // P of this tile's earlier keys
            uint32_t hi[16], lo[16];
            ap_ld16(ts + (PARTS == 1 ? 16 : 32) * b, hi);
            if constexpr (PARTS == 2) ap_ld16(ts + 32 * b + 16, lo);
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
            ap_st16(ts + (PARTS == 1 ? 16 : 32) * b, hi);
            if constexpr (PARTS == 2) ap_st16(ts + 32 * b + 16, lo);
          }
          exponents(m == -CUDART_INF_F ? 0.f : m - KP_P_EXP);
        }
        // the next 32 scores come while these become P.  Not earlier: their registers are not to be touched before they are
        // there, not even to be spilled
        if (c < 3) ap_ld32(ts + 32 * c + 32, next);
        uint32_t hi[16], lo[PARTS == 1 ? 1 : 16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint64_t sum = kp_pack(0.f, 0.f);
#pragma unroll
          for (int i = 8 * h; i < 8 * h + 8; ++i) {
            const KpPair v = kp_unpack(y[i]);
            const float a = ap_ex2(v.a), b = ap_ex2(v.b);
            sum = kp_add2(sum, kp_pack(a, b));
            const __half2 hh = __floats2half2_rn(a, b);
            hi[i] = h22u(hh);
            if constexpr (PARTS == 2) {
              const float2 hf = __half22float2(hh);
              lo[i] = h22u(__floats2half2_rn(a - hf.x, b - hf.y));
            }
          }
          const KpPair both = kp_unpack(sum);
          l = fmaf(both.a + both.b, sc[2 * c + h].z, l);
        }
        ap_st16(ts + (PARTS == 1 ? 16 : 32) * c, hi);
        if constexpr (PARTS == 2) ap_st16(ts + 32 * c + 16, lo);
      };
      uint32_t s0[32], s1[32];
      ap_ld32(ts, s0);
#pragma unroll 1
      for (int c = 0; c < 4; c += 2) {
        kp_wait_ld(s0);
        chunk(c, s0, s1);
        kp_wait_ld(s1);
        chunk(c + 1, s1, s0);
      }
      ap_wait_st();
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      ap_arrive(bar + 8);
    }
    // ---- O / l: a thread's row through its own idle query memory, then stored as whole rows; or its part, to be joined
    if (good && my_n > 1) good = __all_sync(0xffffffffu, kp_wait(bar + 16, (my_n - 2) & 1, &fail_s));
    if (good && my_n > 0) good = __all_sync(0xffffffffu, kp_wait(bar + 16, (my_n - 1) & 1, &fail_s));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (!good) {
      fail_s = 1;
    } else if (tile0 <= last) {
      if (p.splits > 1) {
        const size_t at = ((((size_t)slot * p.c.H + hk) * p.splits + blockIdx.y) * TILES + t) * KP_BM + mine;
        float *o_part = p.partial + at * KV8_D;
        if (my_n > 0) {
#pragma unroll 1
          for (int d = 0; d < KV8_D; d += 32) {
            uint32_t o[32];
            ap_ld32(to + d, o);
            ap_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4 *>(o_part + d + 4 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
        p.partial_ml[at] = make_float2(my_n > 0 ? m : -CUDART_INF_F, my_n > 0 ? l : 0.f);
      } else {
        const float over = limit > 0 ? 1.f / l : 0.f;
        constexpr int CHUNKS = KV8_D * sizeof(T) / 16, EACH = 16 / sizeof(T);
        unsigned char *park = q_s + mine * (KV8_D * sizeof(T));
#pragma unroll 1
        for (int d = 0; d < KV8_D; d += 32) {
          uint32_t o[32];
          if (my_n > 0) {
            ap_ld32(to + d, o);
            ap_wait_ld();
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
#pragma unroll 4
        for (int i = lane / CHUNKS; i < 32; i += 32 / CHUNKS) {
          const int in_tile = (warp & 3) * 32 + i, pk = tile0 + in_tile;
          if (pk > last) break;
          const uint4 v = *reinterpret_cast<const uint4 *>(q_s + in_tile * (KV8_D * sizeof(T)) + ((c ^ (in_tile & 7)) << 4));
          const int token = pk / p.group, head = hk * p.group + pk - token * p.group;
          *reinterpret_cast<uint4 *>((T *)p.out + ((size_t)(row0 + token) * p.Hq + head) * KV8_D + c * EACH) = v;
        }
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == Z::MMA_WARP) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Z::TMEM_COLS) : "memory");
  if (fail_s && tid == 0) atomicExch(p.status, 710);  // site 710: a wait of the 8-bit prompt attention ran out
}

template <typename T, int TILES, int PARTS>
static int prefill_launch(Kv8PrefillParams p, long slots, cudaStream_t stream) {
  p.slots = (int)slots;
  using Z = KpShape<TILES, PARTS>;
  AB200_CUDA(cudaFuncSetAttribute(kv8_prefill_kernel<T, TILES, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::SMEM));
  AB200_REQUIRE(slots * p.c.H < 1l << 31, "kv8_attention: %ld tiles of rows are beyond the built limits", slots * p.c.H);
  AB200_CUDA(launch_pdl(kv8_prefill_kernel<T, TILES, PARTS>, dim3((unsigned)(slots * p.c.H), p.splits), dim3(Z::THREADS), Z::SMEM, stream, p));
  return AB200_OK;
}

int kv8_prefill(Kv8PrefillParams p, int dtype, cudaStream_t stream) {
  const int rows = dtype == AB200_F16 ? 256 : 128;
  p.slots_per_seq = (int)(((long)p.r.n * p.group + rows - 1) / rows);
  const long slots = p.r.cu ? (long)p.r.T * p.group / rows + p.r.S : (long)p.r.S * p.slots_per_seq;
  p.splits = 1;
  if (dtype == AB200_F16) return prefill_launch<__half, 2, 1>(p, slots, stream);
  return prefill_launch<float, 1, 2>(p, slots, stream);
}

}  // namespace ab200
