// The attention of drafted tokens (tree_attention.hip): a call as its kernels take it, its sequences,
// and how workgroups share out their work.  Compiles for the host too.
#ifndef CUGO_TREE_SHARE_H_
#define CUGO_TREE_SHARE_H_

#include "paged.h"

namespace cugo_amd {
namespace paged {

typedef unsigned long long u64;

struct Call {
  Cache c;
  i64 layer_offset;
  const char* q;
  i64 q_stride;  // bytes
  i64 mask_rows;
  const i64* prefix;
  const i64* rows;
  const i64* offsets;
  const u64* mask;
  char* out;
  float* part_o;   // shared-out items' parts: [workgroups, 2, rows, dh]
  float* part_ml;  // [workgroups, 2, rows, 2]: maximum (base 2) and sum
  int2* left;      // [workgroups]: the item (and its sequence) that it began and others went on with, or -1
  int* begun;      // [items]: 1 + the workgroup that began an item others went on with, or 0; anything for
                   // items that nobody did
  int* ended;      // [workgroups]: whether it ended an item that others began
  int tokens, n, each;  // each: queries a sequence without offsets
  int heads, group, words;
  int items;       // (tile of rows, key head), at most so many
  float scale_log2;  // > 0: a negative scale turns q's signs
  uint32_t flip;
};

// What is the same in every lane, in scalar registers.
__host__ __device__ __forceinline__ int same(int x) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_readfirstlane(x);
#else
  return x;
#endif
}
__host__ __device__ __forceinline__ i64 same(i64 x) {
  return (i64)((u64)(unsigned)same((int)(x >> 32)) << 32 | (unsigned)same((int)x));
}

// A sequence as its wavefronts see it.
struct Sequence {
  int first, queries;  // its queries
  i64 row;
  bool exists;  // the row
  int length, prefix;
  int end;  // positions that some query may attend lie before it
};
__host__ __device__ __forceinline__ Sequence sequence_at(const Call& a, int i) {
  Sequence s;
  s.first = i * a.each;
  s.queries = a.each;
  if (a.offsets != nullptr) {
    const i64 first = a.offsets[i], end = a.offsets[i + 1];
    const bool fine = first >= 0 && end <= a.tokens && first < end;
    s.first = fine ? (int)first : 0;
    s.queries = fine ? (int)(end - first) : 0;
  }
  s.row = a.rows ? a.rows[i] : i;
  s.exists = s.row >= 0 && s.row < a.c.rows;
  s.length = s.exists ? row_length(a.c, a.c.length[s.row]) : 0;
  const i64 given = a.prefix[i];
  s.prefix = (int)(given < 0 ? 0 : given > s.length ? s.length : given);
  const i64 behind = a.mask ? (i64)64 * a.words : (i64)s.queries;
  s.end = (int)(s.prefix + behind < s.length ? s.prefix + behind : s.length);
  return s;
}
// Without a mask: where what query `index` may attend ends (a sum of two of these numbers may not fit).
__host__ __device__ __forceinline__ int end_of(const Sequence& s, int index) {
  return s.end - s.prefix > index ? s.prefix + index + 1 : s.end;
}
__host__ __device__ __forceinline__ Sequence same(Sequence s) {
  s.first = same(s.first), s.queries = same(s.queries), s.row = same(s.row);
  s.length = same(s.length), s.prefix = same(s.prefix), s.end = same(s.end);
  s.exists = same((int)s.exists);
  return s;
}

// Tiles of rows over all sequences.  With offsets, sequence i's begin at floor((offsets[i] - origin)
// group / rows a tile) + i, origin = offsets[0], which leaves room for what each needs: for any
// offsets, those of a sequence that is one (0 <= offsets[i] < offsets[i + 1] <= tokens) end before
// floor(tokens group / rows) + n, since the origin is not negative.
__host__ __device__ __forceinline__ i64 origin_of(const Call& a) {
  return a.offsets == nullptr || a.offsets[0] < 0 ? 0 : a.offsets[0];
}
__host__ __device__ __forceinline__ int tiles_before(const Call& a, int i, int rows, i64 origin) {
  if (a.offsets == nullptr) return i * (int)(((i64)a.each * a.group + rows - 1) / rows);
  const i64 o = a.offsets[i] - origin;
  const i64 held = o < 0 ? 0 : o > a.tokens ? a.tokens : o;
  return (int)((unsigned)(held * a.group) / (unsigned)rows) + i;
}
__host__ __device__ __forceinline__ int tiles_of(const Call& a, const Sequence& s, int rows) {
  return (int)(((i64)s.queries * a.group + rows - 1) / rows);
}

// Sharing out: the work of all items (a tile of rows over one key head) in a row, an item's being its
// sequence's tiles of tokens; each of the workgroups does as much of it, in order.
// An item that a border cuts has parts, joined by a second launch.  Every workgroup sums up the
// sequences' work for itself (kMostShared of them at most).
constexpr int kMostShared = 1024;
// Sums of work stop here.  Sequences that do not overlap have less (the host sees to it); where offsets that
// fall make more of it, nothing is done.
constexpr unsigned kTooMuch = ~0u;

// Of one key head's item of a sequence.
__host__ __device__ __forceinline__ int work_each(const Sequence& s, int tokens) {
  const int each = (s.end + tokens - 1) / tokens;
  return each > 1 ? each : 1;
}
// Of sequence i (below 2^31, as the host sees to).
__host__ __device__ __forceinline__ unsigned work_of(const Call& a, int i, int rows, int tokens) {
  const Sequence s = sequence_at(a, i);
  return (unsigned)tiles_of(a, s, rows) * a.c.kv_heads * work_each(s, tokens);
}

// One workgroup's (or wavefront's) work on an item.
struct Job {
  Sequence s;
  int sequence;
  int head, tile;  // the key head; the tile of rows
  int from, to;    // tiles of tokens
  int slot;        // -1: the whole item; 0: its end or middle, 1: its beginning
  bool ends;       // to is the item's end
};

// The jobs of a workgroup in order.
struct Share {
  const unsigned* before;
  unsigned at, end;
  int n;
  __host__ __device__ __forceinline__ bool next(const Call& a, int rows, int tokens, Job& job) {
    if (at >= end) return false;
    int low = 0, high = n;  // before[low] <= at < before[high]
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (before[mid] <= at) low = mid;
      else high = mid;
    }
    low = same(low);
    job.sequence = low;
    job.s = same(sequence_at(a, low));
    const int tiles = tiles_of(a, job.s, rows);
    const int each = work_each(job.s, tokens);
    const unsigned offset = at - (unsigned)same((int)before[low]);
    const unsigned item = offset / (unsigned)each;  // (each >= 1)
    job.from = same((int)(offset - item * each));
    const unsigned left = (unsigned)job.from + (end - at);
    job.to = same((int)(left < (unsigned)each ? left : (unsigned)each));
    job.head = same((int)(item / (unsigned)(tiles > 0 ? tiles : 1)));
    job.tile = same((int)(item - (unsigned)job.head * tiles));
    // (only where lengths or offsets change while they are read)
    if (tiles <= 0 || job.head >= a.c.kv_heads) return false;
    job.ends = job.to == each;
    job.slot = job.from > 0 ? 0 : job.ends ? -1 : 1;
    at += job.to - job.from;
    return true;
  }
};

// Workgroup `group`'s share, of `groups` at most: no less than `least` tiles of tokens each, unless
// there are more items.
__host__ __device__ __forceinline__ Share share_of(const Call& a, const unsigned* before, unsigned group,
                                                   unsigned groups, int least) {
  const unsigned summed = (unsigned)same((int)before[a.n]), all = summed == kTooMuch ? 0 : summed;
  unsigned some = all / (unsigned)least;
  some = some > (unsigned)a.items ? some : (unsigned)a.items;
  some = some < groups ? some : groups;
  some = some < all ? some : all;
  groups = some > 1 ? some : 1;
  const unsigned each = all / groups, more = all - each * groups;  // the first `more` do one more
  Share s;
  s.before = before;
  s.n = a.n;
  s.at = (unsigned)same((int)(group < groups ? each * group + (group < more ? group : more) : all));
  s.end = (unsigned)same((int)(group < groups ? s.at + each + (group < more) : all));
  return s;
}

// What a workgroup tells the launch that joins: before its jobs, and of each.
__host__ __device__ __forceinline__ void note_none(const Call& a, unsigned group) {
  a.ended[group] = 0;
  a.left[group] = make_int2(-1, -1);
}
__host__ __device__ __forceinline__ void note(const Call& a, unsigned group, const Job& job, int rows) {
  if (job.slot == 0) {
    a.ended[group] = job.ends;
    return;
  }
  const int x = tiles_before(a, job.sequence, rows, origin_of(a)) + job.tile;
  const int item = x * a.c.kv_heads + job.head;
  a.begun[item] = job.slot == 1 ? (int)group + 1 : 0;
  if (job.slot == 1) a.left[group] = make_int2(item, job.sequence);
}
// The workgroup that may have begun an item which others went on with, or -1, and whether it did: a
// sequence that nobody served, or whose tiles are another's too (offsets that fall), has anything in
// `begun`.
__host__ __device__ __forceinline__ int begun_by(const Call& a, int item, int groups) {
  const int begun = a.begun[item];
  return begun > 0 && begun <= groups ? begun - 1 : -1;
}
__host__ __device__ __forceinline__ bool did_begin(const Call& a, int group, int item, int sequence) {
  const int2 left = a.left[group];
  return left.x == item && left.y == sequence;
}

}  // namespace paged
}  // namespace cugo_amd

#endif  // CUGO_TREE_SHARE_H_
