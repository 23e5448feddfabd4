// What the paged cache's kernels (paged_cache.hip, tree_attention.hip) share: the cache as they
// take it, and where its tokens lie.  The index arithmetic compiles for the host too.
#ifndef CUGO_PAGED_H_
#define CUGO_PAGED_H_

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/cugo_hip.h"

namespace cugo_amd {
namespace paged {

typedef int64_t i64;

constexpr i64 kMostTokens = ((i64)1 << 31) - (1 << 16);  // of a row: positions fit 32 bits

struct Cache {
  char* k;
  char* v;
  int32_t* table;
  i64* length;
  int32_t* refs;
  unsigned long long* free;
  i64 rows;
  i64 page_bytes;   // of one page of one layer: kv_heads * page * token_bytes
  i64 layer_bytes;  // pages * page_bytes
  int width, pages, layers, kv_heads;
  int page_shift;   // page = 1 << page_shift
  int token_bytes;  // of one head's token: dh elements
};

// A sum that stops at 2^32 - 1.
__host__ __device__ inline unsigned plus(unsigned a, unsigned b) { return __builtin_elementwise_add_sat(a, b); }

// The tokens of a row, whatever its length says.
__host__ __device__ inline int row_length(const Cache& c, i64 length) {
  const i64 most = (i64)c.width << c.page_shift;
  return (int)(length < 0 ? 0 : length > most ? most : length);
}

__host__ __device__ inline int pages_of(const Cache& c, int tokens) {
  return (tokens + (1 << c.page_shift) - 1) >> c.page_shift;
}

// A table entry as a page of the pool, or -1.
__host__ __device__ inline int page_of(const Cache& c, int32_t entry) {
  return entry >= 0 && entry < c.pages ? entry : -1;
}

// Bytes from the start of a layer's k or v to a head's slot of a page of the pool.
__host__ __device__ inline i64 slot_offset(const Cache& c, int page, int head, int slot) {
  return (i64)page * c.page_bytes + ((((i64)head << c.page_shift) + slot) * c.token_bytes);
}

// Bytes to segment s = (layer * 2 + which) * kv_heads + head of a page: a head's slots of one
// layer, which = 0 in k and 1 in v.
__host__ __device__ inline char* segment(const Cache& c, int s, int page) {
  const int head = s % c.kv_heads, rest = s / c.kv_heads;
  return (rest & 1 ? c.v : c.k) + (i64)(rest >> 1) * c.layer_bytes + slot_offset(c, page, head, 0);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int element_size(int dtype) { return dtype == CUGO_DTYPE_F32 ? 4 : 2; }

// Checks a cache as the calls' documentation says and gives the kernels' view of it.
inline int view(const CugoPagedCache* p, Cache* c) {
  if (!p || p->layers <= 0 || p->pages <= 0 || p->kv_heads <= 0 || p->rows <= 0 || p->width <= 0)
    return -1;
  if (!p->k || !p->v || !p->table || !p->length || !p->refs || !p->free) return -1;
  if (p->dtype != CUGO_DTYPE_F32 && p->dtype != CUGO_DTYPE_F16 && p->dtype != CUGO_DTYPE_BF16)
    return -2;
  if (p->dh != 32 && p->dh != 64 && p->dh != 128 && p->dh != 256) return -3;
  int shift = 4;
  while (shift < 9 && ((i64)1 << shift) != p->page) ++shift;
  if (shift > 8) return -3;
  if (p->pages > INT32_MAX / 2 || p->kv_heads > 4096 || p->layers > 4096) return -1;
  if (p->rows > INT32_MAX || p->width > kMostTokens / p->page) return -1;
  if (!aligned16(p->k) || !aligned16(p->v)) return -4;
  c->k = static_cast<char*>(p->k);
  c->v = static_cast<char*>(p->v);
  c->table = p->table;
  c->length = p->length;
  c->refs = p->refs;
  c->free = reinterpret_cast<unsigned long long*>(p->free);
  c->rows = p->rows;
  c->width = (int)p->width;
  c->pages = (int)p->pages;
  c->layers = (int)p->layers;
  c->kv_heads = (int)p->kv_heads;
  c->page_shift = shift;
  c->token_bytes = (int)p->dh * element_size(p->dtype);
  c->page_bytes = p->kv_heads * p->page * (i64)c->token_bytes;
  if (p->pages > INT64_MAX / 4 / p->layers / c->page_bytes) return -1;
  c->layer_bytes = p->pages * c->page_bytes;
  return 0;
}

}  // namespace paged
}  // namespace cugo_amd

#endif  // CUGO_PAGED_H_
