// The 8-bit key and value cache as its kernels see it.
//
// A sequence's tokens lie in pages, named in order by its row of `table`; a page holds page / 16 blocks of 16
// tokens for each head, and a block of one head is 16 D bytes of keys, 16 D of values and one scale for each: a
// power of two 2^E, as the byte E + 127.  Keys are rows of D bytes, one a token; values are D rows of 16 bytes, the
// block's tokens side by side, so that a lane of the product with the weights reads its column's 16 tokens in one
// load.  Both kinds of block are at 16 D times the same index.
#pragma once

#include "pnfx_common.h"

namespace pnfx {

constexpr int BLOCK = 16;      // tokens that share a scale
constexpr int RAW = 16;        // keys before the FIR that are kept of each sequence and head
constexpr int E_LOWEST = -100; // smallest scale: 2^E_LOWEST

struct Cache {
  uint8_t *k, *v, *k_scale, *v_scale;
  void* raw;
  const int* table;
  int64_t table_rs;
  int B, H, d, D, page, page_shift, pages, width;  // width: pages a sequence
  __host__ __device__ int64_t capacity() const { return (int64_t)width << page_shift; }
  // Index of the block at position pos of sequence b, head h; -1 where the table names no page.
  __device__ __forceinline__ int64_t block_at(int b, int h, int64_t pos) const {
    const int id = table[b * table_rs + (pos >> page_shift)];
    if ((unsigned)id >= (unsigned)pages) return -1;
    return ((int64_t)id * H + h) * (page >> 4) + ((pos & (page - 1)) >> 4);
  }
};

// Where the call's tokens of each sequence begin, and how many it has of them (null: the same for all).
struct Span {
  const int *start, *counts;
  int start_all, N;
  __device__ __forceinline__ int64_t first(int b) const { return start ? start[b] : start_all; }
  __device__ __forceinline__ int count(int b) const { return counts ? min(max(counts[b], 0), N) : N; }
};

__device__ __forceinline__ float two_to(int e) {  // -126 <= e <= 127
  return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
}

// The caller's description, checked.
inline int cache_of(const pnfx_cache* c, const char* what, Cache* out) {
  PNFX_REQUIRE(c && c->k && c->v && c->k_scale && c->v_scale && c->table, "%s: null pointer in the cache", what);
  PNFX_REQUIRE(c->B >= 1 && c->H >= 1 && c->pages >= 1 && c->width >= 1 && c->B < (1 << 24) && c->H < (1 << 20) &&
                   c->B * c->H < (1ll << 31) && c->pages < (1ll << 31) && c->width < (1ll << 31),
               "%s: cache of B=%lld H=%lld pages=%lld width=%lld", what, (long long)c->B, (long long)c->H,
               (long long)c->pages, (long long)c->width);
  PNFX_REQUIRE(c->d >= 1 && c->d <= PNFX_CACHE_MAX_HEAD && c->D == (c->d + 15) / 16 * 16,
               "%s: head size %lld in rows of %lld", what, (long long)c->d, (long long)c->D);
  PNFX_REQUIRE(c->page >= BLOCK && c->page <= (1 << 16) && (c->page & (c->page - 1)) == 0,
               "%s: pages of %lld tokens (a power of two from 16 to 65536)", what, (long long)c->page);
  PNFX_REQUIRE(c->table_rs >= c->width, "%s: table's row stride %lld", what, (long long)c->table_rs);
  PNFX_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) == 0,
               "%s: keys and values must be 16-byte aligned", what);
  *out = Cache{c->k, c->v, c->k_scale, c->v_scale, c->raw, c->table, c->table_rs,
               (int)c->B, (int)c->H, (int)c->d, (int)c->D, (int)c->page, __builtin_ctz((unsigned)c->page),
               (int)c->pages, (int)c->width};
  PNFX_REQUIRE(c->pages * c->H * (c->page / BLOCK) < (1ll << 31), "%s: %lld pages of %lld tokens and %lld heads", what,
               (long long)c->pages, (long long)c->page, (long long)c->H);
  PNFX_REQUIRE(out->capacity() <= (1ll << 30), "%s: %lld tokens a sequence", what, (long long)out->capacity());
  return PNFX_OK;
}

}  // namespace pnfx
