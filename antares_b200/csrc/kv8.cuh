// The paged KV cache held in 8 bits: what its writer and its readers share.
//
//   k, v      int8 [pages][Hkv][page_rows][128]         value = code * scale, codes -127 .. 127
//   ks, vs    fp32 [pages][Hkv][page_rows / 16]         one scale for each 16 rows (a block) and head
//   table     int32 [S][table_stride], max_pages in use; position p of sequence s is row p % page_rows of page table[s][p / page_rows];
//             table_stride 0: one row for all of them, where nothing is written
//
// A head's rows of a page lie together: a block is 2 KiB of consecutive memory and shares its scale, so a reader takes
// 16 keys and two scales at a time whatever the page size (a power of two from 16).
#pragma once
#include "common.cuh"

namespace ab200 {

constexpr int KV8_D = 128, KV8_BLOCK = 16;
constexpr int KV8_BAD_PAGE = 800;  // status word: a page table entry in use lies outside the cache

struct Kv8Cache {
  int8_t *k, *v;
  float *ks, *vs;
  int pages, shift, H;  // page_rows = 1 << shift
};

// The new rows of a call: sequence s has rows cu[s] .. cu[s + 1] - 1 of T (cu == nullptr: n rows each) at the positions
// pos0[s], pos0[s] + 1, ...
struct Kv8Rows {
  const int32_t *table;
  long table_stride;
  int max_pages;
  const int32_t *pos0, *cu;
  int S, T, n;

  __device__ __forceinline__ int begin(int s) const { return cu ? min(max(cu[s], 0), T) : s * n; }
  __device__ __forceinline__ int end(int s) const { return cu ? min(max(cu[s + 1], 0), T) : s * n + n; }
};

// A row's sum of P / vs is held times this: beside values of scale 0, which counts as 2^-100, P is up to 2^15, so a key adds up to 2^115 and
// some thousands of them would be infinite; with it 2^22 keys are not, and a scale of 2^118 still leaves 2^-122.
constexpr float KV8_SUM = 0x1p-10f;

// 2^e, exact: -149 <= e <= 127.  A query's largest value can lie at either end of fp32, and 2^e that brings it to a fixed size beyond
// both: that one goes in two steps.
__device__ __forceinline__ float kv8_pow2(int e) { return __int_as_float(e >= -126 ? (127 + e) << 23 : 1 << (149 + e)); }

// First element of head h in the page that holds position p of sequence s; -1 where the table names no page of the cache.
__device__ __forceinline__ long kv8_page(const Kv8Cache &c, const Kv8Rows &r, int s, int p, int *status) {
  const int page = r.table[(size_t)s * r.table_stride + (p >> c.shift)];
  if ((unsigned)page >= (unsigned)c.pages) {
    if (status) atomicExch(status, KV8_BAD_PAGE);
    return -1;
  }
  return page;
}

// Rows of k and v into the cache, by a kernel that lets the one behind it start once what came before has ended: that one
// waits for it before it reads a block from pos0 / 16 on (kv8_append.cu).
int kv8_append_beside(const Kv8Cache &c, const Kv8Rows &r, const void *k, const void *v, long k_stride, long v_stride, const float *inv_freq, int dtype, cudaStream_t stream);

// Host: checks what every entry point checks of a cache and its rows.  `writes`: a table row is one sequence's alone.
inline int kv8_check(const char *who, bool writes, const void *k, const void *v, const void *ks, const void *vs, int pages, int page_rows, int Hkv, const void *table,
                     long table_stride, int max_pages, const void *pos0, const void *cu, int S, int T, Kv8Cache *c, Kv8Rows *r) {
  int shift = 0;
  while (shift < 30 && (1 << shift) < page_rows) ++shift;
  AB200_REQUIRE(page_rows >= KV8_BLOCK && (1 << shift) == page_rows, "%s: page_rows=%d must be a power of two from %d", who, page_rows, KV8_BLOCK);
  AB200_REQUIRE(pages > 0 && Hkv > 0 && Hkv <= 65535, "%s: bad cache, pages=%d heads=%d", who, pages, Hkv);
  AB200_REQUIRE((long)pages * Hkv << (shift - 4) < 1l << 31, "%s: %d pages of %d heads and %d rows are more blocks than the built 2^31", who, pages, Hkv, page_rows);
  AB200_REQUIRE(S >= 0 && T >= 0 && max_pages > 0 && (table_stride >= max_pages || (table_stride == 0 && !writes)), "%s: bad shape S=%d T=%d max_pages=%d table_stride=%ld", who, S, T, max_pages, table_stride);
  AB200_REQUIRE((long)max_pages << shift <= 1l << 30, "%s: %d pages of %d rows are more positions than the built 2^30", who, max_pages, page_rows);
  AB200_REQUIRE(T <= 1 << 28 && S <= 1 << 20, "%s: T=%d rows of S=%d sequences are beyond the built limits", who, T, S);
  AB200_REQUIRE(cu != nullptr || S == 0 || T % S == 0, "%s: %d rows do not divide into %d sequences (cu_rows says how many each has)", who, T, S);
  if (T > 0 && S > 0) {
    AB200_REQUIRE(k && v && ks && vs && table && pos0, "%s: null pointer", who);
    AB200_REQUIRE(aligned16(k) && aligned16(v), "%s: the cache must be 16-byte aligned", who);
  }
  *c = Kv8Cache{(int8_t *)k, (int8_t *)v, (float *)ks, (float *)vs, pages, shift, Hkv};
  *r = Kv8Rows{(const int32_t *)table, table_stride, max_pages, (const int32_t *)pos0, (const int32_t *)cu, S, T, S > 0 ? T / S : 0};
  return AB200_OK;
}

}  // namespace ab200
