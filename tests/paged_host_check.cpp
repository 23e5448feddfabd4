// The paged cache's index arithmetic (cugo_amd/csrc/paged.h) on the host: whatever lengths and
// table entries hold, what the kernels would read or write lies in the pool.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "paged.h"

using namespace cugo_amd::paged;

#define CHECK(x)                                              \
  if (!(x)) {                                                 \
    std::printf("failed: %s (line %d)\n", #x, __LINE__);      \
    return 1;                                                 \
  }

int main() {
  std::mt19937_64 rng(7);
  alignas(16) static char pool[2][16];
  for (int round = 0; round < 400; ++round) {
    CugoPagedCache p{};
    const int64_t dhs[] = {32, 64, 128, 256};
    p.k = pool[0], p.v = pool[1];
    p.layers = 1 + rng() % 3, p.pages = 1 + rng() % 9, p.kv_heads = 1 + rng() % 5;
    p.page = 16ll << rng() % 5, p.dh = dhs[rng() % 4], p.rows = 1 + rng() % 4;
    p.width = 1 + rng() % 6, p.dtype = (int)(rng() % 3);
    std::vector<int32_t> table(p.rows * p.width), refs(p.pages);
    std::vector<int64_t> length(p.rows);
    uint64_t bits = 0;
    p.table = table.data(), p.length = length.data(), p.refs = refs.data(), p.free = &bits;
    Cache c;
    CHECK(view(&p, &c) == 0);
    const i64 bytes = p.layers * p.pages * p.kv_heads * p.page * p.dh * element_size(p.dtype);
    CHECK(c.layer_bytes * p.layers == bytes);
    for (int i = 0; i < 50; ++i) {
      const i64 len = (i64)rng() >> rng() % 64;
      const int tokens = row_length(c, len);
      CHECK(tokens >= 0 && tokens <= p.width * p.page && pages_of(c, tokens) <= c.width);
      CHECK(len < 0 || len > p.width * p.page || tokens == len);
      const int page = page_of(c, (int32_t)rng() >> rng() % 32);
      CHECK(page >= -1 && page < p.pages);
      if (page < 0) continue;
      const int head = (int)(rng() % p.kv_heads), slot = (int)(rng() % p.page);
      const i64 at = (p.layers - 1) * c.layer_bytes + slot_offset(c, page, head, slot);
      CHECK(at >= 0 && at + c.token_bytes <= bytes);
    }
    // every segment of every page, each byte once, in k or in v
    std::vector<char> seen(2 * bytes);
    const i64 each = p.page * c.token_bytes;
    for (int page = 0; page < p.pages; ++page)
      for (int s = 0; s < p.layers * 2 * p.kv_heads; ++s) {
        const char* at = segment(c, s, page);
        const bool in_v = (s / p.kv_heads) & 1;
        const i64 from = at - (in_v ? c.v : c.k);
        CHECK(from >= 0 && from + each <= bytes);
        for (i64 b = from; b < from + each; ++b) {
          char& x = seen[(in_v ? bytes : 0) + b];
          CHECK(!x);
          x = 1;
        }
      }
    for (char x : seen) CHECK(x);
  }
  std::printf("inside\n");
  return 0;
}
