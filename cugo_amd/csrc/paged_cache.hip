// The paged key/value cache's bookkeeping and copies, for gfx950: append, branch, accept
// (include/cugo_hip.h).
//
// Pages are handed out by rule (the lowest free ones, entry after entry), not by the order in
// which wavefronts get there, so a call's result is the same every time.  What decides is computed
// in small launches of their own; what moves data follows:
//   claim    which entries name a row that another entry names too
//   branch:  release (pages given back, a wavefront an entry) -> place (one workgroup: new pages'
//            numbers) -> apply (table, references, copies of part-filled pages)
//   accept:  decide (a wavefront an entry) -> move (tokens, pages given back)
// Bound: the copies by memory (8,192 children of rows of up to 48 tokens in four layers, 540 MB: apply
// 104 us, 5.2 TB/s; append of 49,000 tokens, 100 MB: 21.2 us), moves by half lines where a token of a head
// is 64 bytes (4,096 paths: 33 us), the rest by the launches' latency (place 14 us for 8,192 entries,
// few_kernel 12.5 for 16).
#include "paged.h"

namespace cugo_amd {
namespace paged {

constexpr int kThreads = 256;   // of launches over many workgroups
constexpr int kOneGroup = 1024;  // of the launches of one workgroup

// ------------------------------------------------------------------------------ append

// One 16-byte part of a token's key and value a thread: `parts` of them a token, whose head is
// part >> head_shift.  ok (NULL: not asked): whether the token had a place.
__global__ __launch_bounds__(kThreads) void append_kernel(
    Cache c, i64 layer, const char* __restrict__ k_new, i64 k_stride,
    const char* __restrict__ v_new, i64 v_stride, const i64* __restrict__ pos_in,
    const i64* __restrict__ rows, i64 n, int parts, int head_shift, int each, uint8_t* __restrict__ ok) {
  // `each` tokens a workgroup, or one whose parts the workgroup goes through
  const int in_group = each > 1 ? threadIdx.x / parts : 0;
  const i64 i = (i64)blockIdx.x * each + in_group;
  if (in_group >= each || i >= n) return;
  const i64 row = rows ? rows[i] : i;
  const i64 pos = pos_in[i];
  int page = -1;
  if (row >= 0 && row < c.rows && pos >= 0 && pos < row_length(c, c.length[row])) {
    page = page_of(c, c.table[row * c.width + (pos >> c.page_shift)]);
    if (page >= 0 && c.refs[page] != 1) page = -1;
  }
  if (ok != nullptr && (int)threadIdx.x == in_group * parts) ok[i] = page >= 0;
  if (page < 0) return;
  const int slot = (int)(pos & ((1 << c.page_shift) - 1));
  const i64 base = layer * c.layer_bytes;
  for (int u = threadIdx.x - in_group * parts; u < parts; u += kThreads) {
    const int head = u >> head_shift, part = u & ((1 << head_shift) - 1);
    const i64 to = base + slot_offset(c, page, head, slot) + part * 16;
    const uint4 kv = *reinterpret_cast<const uint4*>(k_new + i * k_stride + (i64)u * 16);
    const uint4 vv = *reinterpret_cast<const uint4*>(v_new + i * v_stride + (i64)u * 16);
    *reinterpret_cast<uint4*>(c.k + to) = kv;
    *reinterpret_cast<uint4*>(c.v + to) = vv;
  }
}

// ------------------------------------------------------------------------------ entries

// What the launches of a call hand on of each entry.
struct alignas(16) Plan {
  int flags;    // kFine ...
  int whole;    // branch: pages kept as they are; accept: the first token that moves
  int held;     // pages the row has afterwards
  int tokens;   // branch: the row's length afterwards; accept: kept tokens
  int page;     // branch: the page in which the kept tokens end, if more follow, or -1
  int part;     // branch: its kept tokens; accept: start
  int had;      // accept: pages the row had
  int unused;
};
constexpr int kFine = 1, kSame = 2;

// bad[i] = 1 for every entry whose dst is another entry's dst or (other than that entry's own) src.
// mark[row] need not be set before: it names an entry of the row if that entry says so too.  Two
// steps, with all of the first before any of the second.
struct Claim {
  const i64 *dst, *src;  // src may be NULL: none
  i64 n, rows;
  int *mark, *bad;
  __device__ void set(i64 i) const {
    bad[i] = 0;
    const i64 d = dst[i];
    if (d >= 0 && d < rows) mark[d] = (int)i;
  }
  __device__ void check(i64 i) const {
    const i64 d = dst[i];
    if (d >= 0 && d < rows) {
      const int w = mark[d];
      if (w != (int)i) bad[i] = 1, bad[w] = 1;
    }
    if (src == nullptr) return;
    const i64 s = src[i];
    if (s != d && s >= 0 && s < rows) {
      const int w = mark[s];
      if (w >= 0 && w < n && dst[w] == s) bad[w] = 1;
    }
  }
  // Both by one workgroup.
  __device__ void all() const {
    for (i64 i = threadIdx.x; i < n; i += blockDim.x) set(i);
    __syncthreads();
    for (i64 i = threadIdx.x; i < n; i += blockDim.x) check(i);
    __syncthreads();
  }
};
__global__ __launch_bounds__(kThreads) void set_kernel(Claim c) {
  const i64 i = (i64)blockIdx.x * kThreads + threadIdx.x;
  if (i < c.n) c.set(i);
}
__global__ __launch_bounds__(kOneGroup) void claim_kernel(Claim c) { c.all(); }
__global__ __launch_bounds__(kThreads) void check_kernel(Claim c) {
  const i64 i = (i64)blockIdx.x * kThreads + threadIdx.x;
  if (i < c.n) c.check(i);
}

// One row less holds `page`; the last one sets its bit in `free`.
__device__ inline void give_back(const Cache& c, int page) {
  if (atomicSub(c.refs + page, 1) == 1) atomicOr(c.free + (page >> 6), 1ull << (page & 63));
}

// A wavefront gives back the pages of a row's table from entry `first` on.
__device__ inline void give_back_row(const Cache& c, const int32_t* row, int first, int end) {
  for (int j = first + (threadIdx.x & 63); j < end; j += 64) {
    const int page = page_of(c, row[j]);
    if (page >= 0) give_back(c, page);
  }
}

// ------------------------------------------------------------------------------ branch

struct Branch {
  Cache c;
  const i64 *dst, *src, *length;
  i64 n;
  const int* bad;
  Plan* plan;
  int2* asked;   // new pages an entry needs at most (-1: refused); the page that it keeps if no other row
                 // holds it, or -1
  int* given;    // twice the first of its new pages (counted over all entries), 1 more if it keeps that
                 // page; -1: none
  int* fresh;    // the new pages
  uint8_t* ok;

  // By a wavefront: what becomes of entry i; its old pages given back.
  __device__ void release(i64 i) const {
    const i64 d = dst[i], s = src[i], want = length[i];
    Plan p{};
    int2 ask = make_int2(-1, -1);
    p.page = -1;
    const i64 most = (i64)c.width << c.page_shift;
    if (d >= 0 && d < c.rows && s >= 0 && s < c.rows && want >= 0 && want <= most && !bad[i]) {
      const bool same = d == s;
      // a row that is another entry's src is no entry's dst: its length and table stand still
      const int have = row_length(c, c.length[s]);
      const int kept = have < (int)want ? have : (int)want;
      p.flags = kFine | (same ? kSame : 0);
      p.whole = kept >> c.page_shift;
      p.part = kept & ((1 << c.page_shift) - 1);
      p.held = pages_of(c, (int)want);
      p.tokens = (int)want;
      if (p.part > 0) {
        if ((int)want > kept) p.page = page_of(c, c.table[s * c.width + p.whole]);
        // kept as it is where nothing will be written behind the kept tokens, or is none in place
        if ((int)want == kept || (same && p.page < 0)) ++p.whole;
      }
      ask.x = p.held > p.whole ? p.held - p.whole : 0;
      if (same) ask.y = p.page;
      const int old = pages_of(c, same ? have : row_length(c, c.length[d]));
      give_back_row(c, c.table + d * c.width, same ? p.held : 0, old);
    }
    if ((threadIdx.x & 63) == 0) plan[i] = p, asked[i] = ask;
  }
};

__global__ __launch_bounds__(kThreads) void release_kernel(Branch b) {
  const i64 i = (i64)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (i < b.n) b.release(i);
}

// Inclusive sum over the wavefront's lanes (2^32 - 1 is more than there are pages).
__device__ inline unsigned wave_scan(unsigned x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned y = __shfl_up(x, off);
    if ((int)(threadIdx.x & 63) >= off) x = plus(x, y);
  }
  return x;
}
// The sum of the wavefronts' x before this one; `total` of all.  The buffer holds one a wavefront.
__device__ inline unsigned before_wave(unsigned x, unsigned* buffer, unsigned& total) {
  const int wave = threadIdx.x >> 6;
  __syncthreads();  // the buffer's last readers
  if ((threadIdx.x & 63) == 0) buffer[wave] = x;
  __syncthreads();
  unsigned before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kOneGroup / 64; ++w) {
    const unsigned y = buffer[w];
    if (w < wave) before = plus(before, y);
    total = plus(total, y);
  }
  return before;
}

// What other wavefronts' atomics wrote, past the caches that they do not reach.
template <class T>
__device__ inline T fresh_load(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kWaves = kOneGroup / 64;
constexpr int kWordsAtOnce = kOneGroup;  // words of free bits that the workgroup holds: 65,536 pages

struct PlaceShared {
  unsigned buffer[kWaves];
  unsigned long long word[kWordsAtOnce];
  unsigned before[kWordsAtOnce];
  unsigned used;
};

// A segment of free words, one a thread, to LDS with the free pages before each; their number.
__device__ inline unsigned load_words(const Cache& c, int segment, int words, unsigned before,
                                      PlaceShared& sh) {
  const int w = threadIdx.x;
  unsigned long long word = segment + w < words ? fresh_load(c.free + segment + w) : 0;
  if (segment + w == words - 1 && (c.pages & 63)) word &= (1ull << (c.pages & 63)) - 1;  // no page beyond
  const unsigned pages = __popcll(word), sum = wave_scan(pages);
  unsigned total;
  before += before_wave(__shfl(sum, 63), sh.buffer, total);
  sh.word[w] = word;
  sh.before[w] = before + sum - pages;
  __syncthreads();
  return total;
}

// New pages' numbers, by one workgroup: each entry's first among all of them, then the lowest free
// pages in order (`fresh`), as many as the entries that fit use.  A lane takes kAtOnce entries, 64
// apart, at once.  Short code counts here: one workgroup fetches each instruction from memory anew.
template <int kAtOnce>
__device__ inline void place(const Branch& b, PlaceShared& sh) {
  const Cache& c = b.c;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int words = (c.pages + 63) >> 6;
  if (threadIdx.x == 0) sh.used = 0;
  unsigned available = 0;
  for (int segment = 0; segment < words; segment += kWordsAtOnce)
    available += load_words(c, segment, words, available, sh);
  unsigned carry = 0;  // what the entries before need
  for (i64 base = 0; base < b.n; base += kOneGroup * kAtOnce) {
    const i64 first = base + wave * (kAtOnce * 64) + lane;
    int2 ask[kAtOnce];
    unsigned own = 0, end[kAtOnce], mine = 0, total, used = 0;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      ask[k] = first + k * 64 < b.n ? b.asked[first + k * 64] : make_int2(-1, -1);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (ask[k].y >= 0 && fresh_load(c.refs + ask[k].y) <= 1) own |= 1u << k, --ask[k].x;
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const unsigned sum = wave_scan(max(ask[k].x, 0));
      end[k] = plus(mine, sum);
      mine = plus(mine, __shfl(sum, 63));
    }
    const unsigned before = plus(carry, before_wave(mine, sh.buffer, total));
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (first + k * 64 >= b.n) continue;
      const unsigned to = plus(before, end[k]);
      const bool fits = ask[k].x == 0 || (ask[k].x > 0 && to <= available);
      if (fits && ask[k].x > 0) used = to;
      b.given[first + k * 64] = fits ? (ask[k].x ? (int)(to - ask[k].x) << 1 : 0) | (int)(own >> k & 1) : -1;
      b.ok[first + k * 64] = fits;
    }
    if (used > 0) atomicMax(&sh.used, used);
    carry = plus(carry, total);
  }
  __syncthreads();
  const unsigned used = sh.used;
  unsigned rank = 0;  // of the free pages before this segment
  for (int segment = 0; segment < words && rank < used; segment += kWordsAtOnce) {
    // a pool of one segment is still there
    const unsigned total = words > kWordsAtOnce ? load_words(c, segment, words, rank, sh) : available;
    const int here = min(kWordsAtOnce, words - segment);
    for (int w = threadIdx.x; w < here; w += kOneGroup) {
      unsigned long long left = sh.word[w];
      const unsigned at = sh.before[w], pages = __popcll(left);
      if (at < used && pages > 0) {  // the lowest of them are taken
        if (at + pages <= used) left = 0;
        else
          for (unsigned t = at; t < used; ++t) left &= left - 1;
        c.free[segment + w] = left;
      }
    }
    // a word a wavefront at a time, a page a lane
    for (int w = wave; w < here; w += kWaves) {
      if (sh.before[w] >= used) break;
      const unsigned long long bits = sh.word[w];
      const unsigned to = sh.before[w] + __popcll(bits & ((1ull << lane) - 1));
      if ((bits >> lane & 1) && to < used) {
        const int page = ((segment + w) << 6) + lane;
        b.fresh[to] = page;
        c.refs[page] = 1;
      }
    }
    rank += total;
    __syncthreads();  // the segment's last readers
  }
}

template <int kAtOnce>
__global__ __launch_bounds__(kOneGroup) void place_kernel(Branch b) {
  __shared__ PlaceShared sh;
  place<kAtOnce>(b, sh);
}

// Few entries: everything before apply by one workgroup.
__global__ __launch_bounds__(kOneGroup) void few_kernel(Branch b, Claim claim) {
  __shared__ PlaceShared sh;
  claim.all();
  for (i64 i = threadIdx.x >> 6; i < b.n; i += kOneGroup / 64) b.release(i);
  __threadfence();
  __syncthreads();
  place<1>(b, sh);
}

// Copies `units` 16-byte units of every segment from page `a` to page `b`, segments first, first +
// step, ... of the pages' layers * 2 * kv_heads, a power of two of lanes a segment.
__device__ inline void copy_page(const Cache& c, int a, int b, int units, int first, int step) {
  const int lane = threadIdx.x & 63;
  int log = 0;
  while (log < 6 && (1 << log) < units) ++log;
  const int sub = lane >> log, unit = lane & ((1 << log) - 1), at_once = 64 >> log;
  const int segments = c.layers * 2 * c.kv_heads;
  for (int s = first * at_once + sub; s < segments; s += step * at_once) {
    const uint4* from = reinterpret_cast<const uint4*>(segment(c, s, a));
    uint4* to = reinterpret_cast<uint4*>(segment(c, s, b));
    for (int u = unit; u < units; u += 1 << log) to[u] = from[u];
  }
}

__global__ __launch_bounds__(kThreads) void apply_kernel(Branch b) {
  const Cache& c = b.c;
  const i64 i = blockIdx.x;
  const Plan p = b.plan[i];
  const int given = b.given[i];
  if (!(p.flags & kFine)) return;
  const i64 d = b.dst[i], s = b.src[i];
  const bool same = p.flags & kSame;
  if (given < 0) {  // no pages left
    if (!same && blockIdx.y == 0 && threadIdx.x == 0) c.length[d] = 0;
    return;
  }
  const bool copy = p.page >= 0 && !(given & 1);
  const int whole = p.whole + (given & 1);
  const int* fresh = b.fresh + (given >> 1);
  if (copy)
    copy_page(c, p.page, fresh[0], p.part * c.token_bytes / 16,
              blockIdx.y * (kThreads / 64) + (threadIdx.x >> 6), gridDim.y * (kThreads / 64));
  if (blockIdx.y != 0) return;
  int32_t* row = c.table + d * c.width;
  const int32_t* from = c.table + s * c.width;
  for (int j = threadIdx.x; j < p.held; j += kThreads) {
    if (j >= whole) {
      row[j] = fresh[j - whole];
    } else if (!same) {
      const int32_t entry = from[j];
      const int page = page_of(c, entry);
      row[j] = entry;
      if (page >= 0) atomicAdd(c.refs + page, 1);
    }
  }
  if (threadIdx.x == 0) {
    if (same && copy) give_back(c, p.page);
    c.length[d] = p.tokens;
  }
}

// ------------------------------------------------------------------------------ accept

struct Accept {
  Cache c;
  const i64 *rows, *start, *keep;
  i64 keep_stride, most, n;
  const int* bad;
  Plan* plan;
  uint8_t* ok;
  __device__ void decide(i64 i) const;
};

// By a wavefront: which tokens of entry i are kept, and whether they may be.
__device__ inline void Accept::decide(i64 i) const {
  const int lane = threadIdx.x & 63;
  const i64 row = rows[i], start = this->start[i];
  Plan p{};
  bool fine = row >= 0 && row < c.rows && !bad[i];
  const int length = fine ? row_length(c, c.length[row]) : 0;
  fine = fine && start >= 0 && start <= length;
  int count = 0, moves = -1;  // kept tokens, and the first that moves
  if (fine) {
    const i64* path = keep + i * keep_stride;
    bool going = true;
    for (i64 base = 0; base < most && going; base += 64) {
      const i64 j = base + lane;
      const i64 at = j < most ? path[j] : -1;
      const unsigned long long ends = __ballot(at < 0);
      const int here = ends ? __builtin_ctzll(ends) : 64;
      const bool mine = lane < here;
      const i64 prior = j > 0 && mine ? path[j - 1] : -1;
      const bool right = !mine || (at > prior && at < length - start);
      if (__ballot(!right)) {
        fine = false;
        break;
      }
      const unsigned long long moving = __ballot(mine && at != j);
      if (moves < 0 && moving) moves = (int)base + __builtin_ctzll(moving);
      count += here;
      going = here == 64;
    }
  }
  if (fine && moves >= 0) {  // the pages that will be written are the row's alone
    const int from = (int)(start + moves) >> c.page_shift;
    const int to = (int)(start + count - 1) >> c.page_shift;
    bool shared = false;
    for (int j = from + lane; j <= to; j += 64) {
      const int page = page_of(c, c.table[row * c.width + j]);
      shared = shared || page < 0 || c.refs[page] != 1;
    }
    fine = !__ballot(shared);
  }
  if (lane == 0) {
    if (fine) {
      p.flags = kFine;
      p.whole = moves < 0 ? count : moves;
      p.tokens = count;
      p.part = (int)start;
      p.held = pages_of(c, (int)start + count);
      p.had = pages_of(c, length);
    }
    plan[i] = p;
    ok[i] = fine;
  }
}

__global__ __launch_bounds__(kThreads) void decide_kernel(Accept a) {
  const i64 i = (i64)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (i < a.n) a.decide(i);
}

// Few entries: with the claims, by one workgroup.
__global__ __launch_bounds__(kOneGroup) void few_decide_kernel(Accept a, Claim claim) {
  claim.all();
  for (i64 i = threadIdx.x >> 6; i < a.n; i += kOneGroup / 64) a.decide(i);
}

constexpr int kPathChunk = kThreads;  // kept tokens whose places a workgroup holds at once
constexpr int kInFlight = 8;     // tokens a lane reads before it writes

// Moves the kept tokens of one entry's segments.  Kept ones rise, so a token's new place is never
// behind its old one: what is read before an earlier or equal token is written is right, and lanes
// of different segments or parts never meet.
__global__ __launch_bounds__(kThreads) void move_kernel(Cache c, const i64* __restrict__ rows,
                                                        const i64* __restrict__ keep,
                                                        i64 keep_stride, i64 most,
                                                        const Plan* __restrict__ plan) {
  __shared__ i64 from[kPathChunk], to[kPathChunk];
  const i64 i = blockIdx.x;
  const Plan p = plan[i];
  const i64 row = rows[i];
  // the first kept tokens are asked for before it is known which move
  const i64 early = threadIdx.x < most ? keep[i * keep_stride + threadIdx.x] : -1;
  if (!(p.flags & kFine)) return;
  const int32_t* table = c.table + row * c.width;
  const int units = c.token_bytes / 16;  // a power of two, at most 64
  const int log = 31 - __builtin_clz(units);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int sub = lane >> log, unit = lane & (units - 1), at_once = 64 >> log;
  const int segments = c.layers * 2 * c.kv_heads;
  const auto place = [&](int at) {
    const int page = page_of(c, table[at >> c.page_shift]);
    return page < 0 ? (i64)-1 : slot_offset(c, page, 0, at & ((1 << c.page_shift) - 1));
  };
  for (int base = 0; base < p.tokens; base += kPathChunk) {
    const int skip = max(p.whole - base, 0);  // tokens that stay where they are
    const int here = min(kPathChunk, p.tokens - base);
    if (skip >= here) continue;
    __syncthreads();
    const int j = threadIdx.x;
    if (j >= skip && j < here) {
      from[j] = place(p.part + (int)(base == 0 ? early : keep[i * keep_stride + base + j]));
      to[j] = place(p.part + base + j);
    }
    __syncthreads();
    for (int s = (blockIdx.y * (kThreads / 64) + wave) * at_once + sub; s < segments;
         s += gridDim.y * (kThreads / 64) * at_once) {
      char* at = segment(c, s, 0) + unit * 16;
      for (int j = skip; j < here; j += kInFlight) {
        uint4 x[kInFlight];
#pragma unroll
        for (int q = 0; q < kInFlight; ++q)
          if (j + q < here && from[j + q] >= 0)
            x[q] = *reinterpret_cast<const uint4*>(at + from[j + q]);
#pragma unroll
        for (int q = 0; q < kInFlight; ++q)
          if (j + q < here && from[j + q] >= 0 && to[j + q] >= 0)
            *reinterpret_cast<uint4*>(at + to[j + q]) = x[q];
      }
    }
  }
  if (blockIdx.y != 0) return;
  if (wave == 0) give_back_row(c, table, p.held, p.had);
  if (threadIdx.x == 0) c.length[row] = p.part + p.tokens;
}

// ------------------------------------------------------------------------------ the host's part

// Of a call's workspace: entries' plans, then words.
inline i64 workspace_bytes(const Cache& c, i64 n, bool branch) {
  return n * (i64)(sizeof(Plan) + sizeof(int)) + c.rows * (i64)sizeof(int) +
         (branch ? n * (i64)(sizeof(int2) + sizeof(int)) + c.pages * (i64)sizeof(int) : 0);
}

struct Workspace {
  Plan* plan;
  int2* asked;
  int *bad, *mark, *given, *fresh;
  Workspace(void* at, const Cache& c, i64 n, bool branch)
      : plan(static_cast<Plan*>(at)), asked(reinterpret_cast<int2*>(plan + n)),
        bad(reinterpret_cast<int*>(asked + (branch ? n : 0))), mark(bad + n), given(mark + c.rows),
        fresh(given + n) {}
};

constexpr i64 kMostEntries = (i64)1 << 23;  // a launch has fewer than 2^32 threads in x
// Up to so many entries one workgroup does what would otherwise be launches of its own.
constexpr i64 kFew = 256;

inline unsigned groups_of(i64 n, int each) { return (unsigned)((n + each - 1) / each); }

// The claims of many entries: by one workgroup, or two launches (257 entries 2.2 us against 3.8, 8,192
// 25 against 8.5).
inline void claim(const Claim& c, hipStream_t stream) {
  if (c.n <= 2048) {
    hipLaunchKernelGGL(claim_kernel, dim3(1), dim3(kOneGroup), 0, stream, c);
    return;
  }
  hipLaunchKernelGGL(set_kernel, dim3(groups_of(c.n, kThreads)), dim3(kThreads), 0, stream, c);
  hipLaunchKernelGGL(check_kernel, dim3(groups_of(c.n, kThreads)), dim3(kThreads), 0, stream, c);
}

// Workgroups over an entry's segments: enough for 2,048 in all, at most one for each four
// wavefronts' worth.
inline unsigned slices(const Cache& c, i64 n, int at_once) {
  const i64 most = (c.layers * 2 * (i64)c.kv_heads + 4 * at_once - 1) / (4 * at_once);
  const i64 want = (2048 + n - 1) / n;
  return (unsigned)(want < 1 ? 1 : want > most ? most : want);
}

}  // namespace paged
}  // namespace cugo_amd

extern "C" {

int cugo_paged_append(const CugoPagedCache* cache, int64_t layer, const void* k_new,
                      int64_t k_stride, const void* v_new, int64_t v_stride, const int64_t* pos,
                      const int64_t* rows, int64_t n, hipStream_t stream) {
  return cugo_paged_append_ok(cache, layer, k_new, k_stride, v_new, v_stride, pos, rows, n, nullptr, stream);
}

int cugo_paged_append_ok(const CugoPagedCache* cache, int64_t layer, const void* k_new,
                         int64_t k_stride, const void* v_new, int64_t v_stride, const int64_t* pos,
                         const int64_t* rows, int64_t n, uint8_t* ok, hipStream_t stream) {
  using namespace cugo_amd::paged;
  Cache c;
  if (const int bad = view(cache, &c)) return bad;
  const int64_t size = element_size(cache->dtype), token = cache->kv_heads * cache->dh;
  if (n < 0 || layer < 0 || layer >= cache->layers || k_stride < token || v_stride < token)
    return -1;
  if (n > 0 && (!k_new || !v_new || !pos)) return -1;
  if (!aligned16(k_new) || !aligned16(v_new) || k_stride * size % 16 != 0 || v_stride * size % 16 != 0)
    return -4;
  if (n == 0) return 0;
  const int parts = (int)(token * size / 16);
  const int each = parts >= kThreads ? 1 : kThreads / parts;
  const int64_t groups = (n + each - 1) / each;
  if (groups >= (int64_t)1 << 24) return -1;  // a launch has fewer than 2^32 threads in x
  hipLaunchKernelGGL(append_kernel, dim3((unsigned)groups), dim3(kThreads), 0, stream, c, layer,
                     static_cast<const char*>(k_new), k_stride * size,
                     static_cast<const char*>(v_new), v_stride * size, pos, rows, n, parts,
                     31 - __builtin_clz(c.token_bytes / 16), each, ok);
  return (int)hipGetLastError();
}

int64_t cugo_paged_branch_workspace(const CugoPagedCache* cache, int64_t n) {
  using namespace cugo_amd::paged;
  Cache c;
  if (view(cache, &c) || n <= 0 || n > kMostEntries) return 0;
  return workspace_bytes(c, n, true);
}

int cugo_paged_branch(const CugoPagedCache* cache, const int64_t* dst, const int64_t* src,
                      const int64_t* length, int64_t n, uint8_t* ok, void* workspace,
                      int64_t workspace_size, hipStream_t stream) {
  using namespace cugo_amd::paged;
  Cache c;
  if (const int bad = view(cache, &c)) return bad;
  if (n < 0 || n > kMostEntries || (n > 0 && (!dst || !src || !length || !ok || !workspace)))
    return -1;
  if (n == 0) return 0;
  if (!aligned16(workspace)) return -4;
  if (workspace_size < workspace_bytes(c, n, true)) return -5;
  const Workspace w(workspace, c, n, true);
  const Claim named{dst, src, n, c.rows, w.mark, w.bad};
  const Branch b{c, dst, src, length, n, w.bad, w.plan, w.asked, w.given, w.fresh, ok};
  if (n <= kFew) {
    hipLaunchKernelGGL(few_kernel, dim3(1), dim3(kOneGroup), 0, stream, b, named);
  } else {
    claim(named, stream);
    hipLaunchKernelGGL(release_kernel, dim3(groups_of(n, kThreads / 64)), dim3(kThreads), 0, stream, b);
    if (n <= kOneGroup)
      hipLaunchKernelGGL(place_kernel<1>, dim3(1), dim3(kOneGroup), 0, stream, b);
    else
      hipLaunchKernelGGL(place_kernel<8>, dim3(1), dim3(kOneGroup), 0, stream, b);
  }
  hipLaunchKernelGGL(apply_kernel, dim3((unsigned)n, slices(c, n, 1)), dim3(kThreads), 0, stream, b);
  return (int)hipGetLastError();
}

int64_t cugo_paged_accept_workspace(const CugoPagedCache* cache, int64_t n) {
  using namespace cugo_amd::paged;
  Cache c;
  if (view(cache, &c) || n <= 0 || n > kMostEntries) return 0;
  return workspace_bytes(c, n, false);
}

int cugo_paged_accept(const CugoPagedCache* cache, const int64_t* rows, const int64_t* start,
                      const int64_t* keep, int64_t keep_stride, int64_t most, int64_t n,
                      uint8_t* ok, void* workspace, int64_t workspace_size, hipStream_t stream) {
  using namespace cugo_amd::paged;
  Cache c;
  if (const int bad = view(cache, &c)) return bad;
  if (n < 0 || n > kMostEntries || most < 0 || most > kMostTokens || keep_stride < 0) return -1;
  if (n > 0 && (!rows || !start || (most > 0 && !keep) || !ok || !workspace)) return -1;
  if (n == 0) return 0;
  if (!aligned16(workspace)) return -4;
  if (workspace_size < workspace_bytes(c, n, false)) return -5;
  const Workspace w(workspace, c, n, false);
  const Claim named{rows, nullptr, n, c.rows, w.mark, w.bad};
  const Accept a{c, rows, start, keep, keep_stride, most, n, w.bad, w.plan, ok};
  if (n <= kFew) {
    hipLaunchKernelGGL(few_decide_kernel, dim3(1), dim3(kOneGroup), 0, stream, a, named);
  } else {
    claim(named, stream);
    hipLaunchKernelGGL(decide_kernel, dim3(groups_of(n, kThreads / 64)), dim3(kThreads), 0, stream, a);
  }
  hipLaunchKernelGGL(move_kernel, dim3((unsigned)n, slices(c, n, 1024 / c.token_bytes)),
                     dim3(kThreads), 0, stream, c, rows, keep, keep_stride, most, w.plan);
  return (int)hipGetLastError();
}

}  // extern "C"
