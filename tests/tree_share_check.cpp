// How the attention of drafted tokens shares out its work (cugo_amd/csrc/tree_share.h), on the host: for any
// offsets, and whatever the workspace held before, workgroups' parts lie inside it, a launch that
// joins follows only parts that were written for the item it joins, and of sequences that do not
// overlap every tile of tokens is done once.
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "tree_share.h"

using namespace cugo_amd::paged;

#define CHECK(x)                                              \
  if (!(x)) {                                                 \
    std::printf("failed: %s (line %d)\n", #x, __LINE__);      \
    return 1;                                                 \
  }

struct Part {
  int sequence, item, from, to;
};

// Where queries' positions end, near the longest row too.
int ends_fit() {
  std::mt19937_64 rng(12);
  for (int i = 0; i < 200000; ++i) {
    Sequence s{};
    s.length = (int)(kMostTokens - 1) >> (rng() % 2 ? 0 : rng() % 31);
    s.prefix = rng() % 2 ? s.length - (int)(rng() % (1 + (s.length >> rng() % 31))) : s.length;
    s.queries = 1 + (int)(rng() % (1 << 24) >> rng() % 24);
    const i64 whole = (i64)s.prefix + s.queries;
    s.end = (int)(whole < s.length ? whole : s.length);
    const int index = (int)(rng() % s.queries);
    const i64 want = (i64)s.prefix + index + 1;
    CHECK(end_of(s, index) == (want < s.end ? want : s.end));
  }
  return 0;
}

int main() {
  if (ends_fit()) return 1;
  std::mt19937_64 rng(11);
  int too_much = 0, cut = 0, served = 0;
  for (int round = 0; round < 3000; ++round) {
    const bool falling = rng() % 2, vast = rng() % 4 == 0;
    Call a{};
    a.c.page_shift = vast ? 8 : 4;
    a.c.rows = 5;
    a.c.kv_heads = 1 + (int)(rng() % 4);
    a.c.width = vast ? 1 << 20 : 300 + (int)(rng() % 4000);
    std::vector<i64> length(a.c.rows);
    for (i64& x : length) x = (i64)(rng() % ((u64)a.c.width << a.c.page_shift)) >> (vast ? 0 : rng() % 12);
    a.c.length = length.data();
    a.n = 1 + (int)(rng() % (falling ? 200 : 40));
    a.group = 1 + (int)(rng() % 4);
    a.tokens = 1 + (int)(rng() % 400);
    const int rows = rng() % 2 ? 16 : 128, tile = rng() % 2 ? 32 : 64;
    if (vast) a.c.kv_heads = 1, a.n = 40 + (int)(rng() % 20), a.tokens = 60 * rows / a.group;
    std::vector<i64> offsets(a.n + 1), prefix(a.n), which(a.n);
    for (i64& x : offsets) x = (i64)(rng() % (a.tokens + 1));
    if (!falling) {
      for (int i = 1; i <= a.n; ++i)
        for (int j = i; j > 0 && offsets[j] < offsets[j - 1]; --j) std::swap(offsets[j], offsets[j - 1]);
    } else {
      for (int i = 0; i <= a.n; ++i) {
        if (vast) offsets[i] = i % 2 ? a.tokens : 0;
        if (rng() % 20 == 0) offsets[i] = (i64)rng() >> rng() % 60;
      }
    }
    for (int i = 0; i < a.n; ++i) which[i] = (i64)(rng() % 7) - 1;
    for (i64& x : prefix) x = (i64)(rng() >> rng() % 64) * (rng() % 8 ? 1 : -1);
    if (vast && round % 2) {  // all of them over the longest rows that there are
      for (int i = 0; i < a.n; ++i) which[i] = i % 5, prefix[i] = INT64_MAX;
      for (i64& x : length) x = INT64_MAX;
    }
    a.offsets = offsets.data(), a.prefix = prefix.data(), a.rows = which.data();
    a.items = (a.tokens * a.group / rows + a.n) * a.c.kv_heads;
    const i64 longest = (i64)a.c.width << a.c.page_shift;
    const i64 most = a.items * ((longest + 15) / 16);
    if (most >= (i64)1 << 31) {  // the host does not share out such a call
      --round;
      continue;
    }
    const int groups = 1 + (int)(rng() % 64);
    std::vector<unsigned> before(a.n + 1);
    unsigned sum = 0;
    u64 real = 0;
    for (int i = 0; i < a.n; ++i) {
      const unsigned x = work_of(a, i, rows, tile);
      CHECK((u64)x <= (u64)most);
      sum = plus(sum, x), real += x;
      before[i] = sum - x;
    }
    before[a.n] = sum;
    if (!falling) CHECK(real <= (u64)most);
    too_much += real >= kTooMuch;

    std::vector<int> begun(a.items), ended(groups);
    std::vector<int2> left(groups);
    for (int& x : begun) x = (int)(rng() % 2 ? rng() : rng() % (groups + 3));
    for (int& x : ended) x = (int)rng();
    a.begun = begun.data(), a.ended = ended.data(), a.left = left.data();
    std::vector<Part> part(2 * groups, Part{-1, -1, 0, 0});
    std::vector<std::vector<unsigned>> done(a.n);  // tiles of tokens done of each item of a sequence
    const i64 origin = origin_of(a);
    for (int g = 0; g < groups; ++g) {
      note_none(a, g);
      Share share = share_of(a, before.data(), g, groups, 4);
      Job job;
      int jobs = 0;
      while (share.next(a, rows, tile, job)) {
        CHECK(++jobs <= a.items * 300);
        CHECK(job.sequence >= 0 && job.sequence < a.n && job.head >= 0 && job.head < a.c.kv_heads);
        CHECK(job.tile >= 0 && job.tile < tiles_of(a, job.s, rows));
        CHECK(job.from >= 0 && job.from < job.to && job.to <= work_each(job.s, tile));
        const int item = (tiles_before(a, job.sequence, rows, origin) + job.tile) * a.c.kv_heads + job.head;
        CHECK(item >= 0 && item < a.items);
        if (job.slot >= 0) part[2 * g + job.slot] = Part{job.sequence, item, job.from, job.to};
        auto& d = done[job.sequence];
        d.resize((size_t)tiles_of(a, job.s, rows) * a.c.kv_heads);
        d[(size_t)job.head * tiles_of(a, job.s, rows) + job.tile] += job.to - job.from;
        note(a, g, job, rows);
        if (real > 200000 && jobs > 2000) break;  // the rest is the same
      }
      if (real >= kTooMuch) CHECK(jobs == 0);
    }
    if (real > 200000) continue;
    // every (sequence, tile) that the joining launch may take an item for
    for (int i = 0; i < a.n; ++i) {
      const Sequence s = sequence_at(a, i);
      const int tiles = tiles_of(a, s, rows), each = work_each(s, tile);
      if (tiles > 0) CHECK((int)done[i].size() == tiles * a.c.kv_heads);
      for (int t = 0; t < tiles; ++t)
        for (int h = 0; h < a.c.kv_heads; ++h) {
          CHECK((int)done[i][(size_t)h * tiles + t] == each);
          ++served;
          const int item = (tiles_before(a, i, rows, origin) + t) * a.c.kv_heads + h;
          const int g = begun_by(a, item, groups);
          CHECK(g >= -1 && g < groups);
          if (g < 0 || !did_begin(a, g, item, i)) continue;
          ++cut;
          int to = 0, k = g;
          for (bool ends = false; !ends; ++k) {
            CHECK(k < groups);
            const Part& p = part[2 * k + (k == g)];
            CHECK(p.sequence == i && p.item == item && p.from == to);
            to = p.to;
            ends = k > g && ended[k];
          }
          CHECK(to == each);
        }
    }
  }
  std::printf("%d with too much, %d items cut, %d done\n", too_much, cut, served);
  CHECK(too_much > 20 && cut > 1000 && served > 10000);
  std::printf("inside\n");
  return 0;
}
