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
// Bound: the copies by memory; the rest by the launches' latency.
#include "paged.h"

namespace cugo_amd {
namespace paged {

constexpr int kThreads = 256;   // of launches over many workgroups
constexpr int kOneGroup = 1024;  // of the launches of one workgroup

// ------------------------------------------------------------------------------ append

// One 16-byte part of a token's key and value a thread: `parts` of them a token, whose head is
// part >> head_shift.
__global__ __launch_bounds__(kThreads) void append_kernel(
    Cache c, i64 layer, const char* __restrict__ k_new, i64 k_stride,
    const char* __restrict__ v_new, i64 v_stride, const i64* __restrict__ pos_in,
    const i64* __restrict__ rows, i64 n, int parts, int head_shift, int each) {
  // `each` tokens a workgroup, or one whose parts the workgroup goes through
  const int in_group = each > 1 ? threadIdx.x / parts : 0;
  const i64 i = (i64)blockIdx.x * each + in_group;
  if (in_group >= each || i >= n) return;
  const i64 row = rows ? rows[i] : i;
  if (row < 0 || row >= c.rows) return;
  const i64 pos = pos_in[i];
  if (pos < 0 || pos >= row_length(c, c.length[row])) return;
  const int page = page_of(c, c.table[row * c.width + (pos >> c.page_shift)]);
  if (page < 0 || c.refs[page] != 1) return;
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
  int first;    // branch: the first of its new pages, counted over all entries
  int had;      // accept: pages the row had
};
constexpr int kFine = 1, kSame = 2, kCopy = 4, kLacking = 8;

// bad[i] = 1 for every entry whose dst is another entry's dst or (other than that entry's own) src.
// mark[row] need not be set before: it names an entry of the row if that entry says so too.
__global__ __launch_bounds__(kOneGroup) void claim_kernel(const i64* __restrict__ dst,
                                                          const i64* __restrict__ src, i64 n,
                                                          i64 rows, int* __restrict__ mark,
                                                          int* __restrict__ bad) {
  for (i64 i = threadIdx.x; i < n; i += kOneGroup) {
    bad[i] = 0;
    const i64 d = dst[i];
    if (d >= 0 && d < rows) __hip_atomic_store(mark + d, (int)i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  }
  __syncthreads();
  for (i64 i = threadIdx.x; i < n; i += kOneGroup) {
    const i64 d = dst[i];
    if (d >= 0 && d < rows) {
      const int w = __hip_atomic_load(mark + d, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      if (w != (int)i) bad[i] = 1, bad[w] = 1;
    }
    if (src == nullptr) continue;
    const i64 s = src[i];
    if (s != d && s >= 0 && s < rows) {
      const int w = __hip_atomic_load(mark + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      if (w >= 0 && w < n && dst[w] == s) bad[w] = 1;
    }
  }
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

__global__ __launch_bounds__(kThreads) void release_kernel(
    Cache c, const i64* __restrict__ dst, const i64* __restrict__ src,
    const i64* __restrict__ length, i64 n, const int* __restrict__ bad, Plan* __restrict__ plan) {
  const i64 i = (i64)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (i >= n) return;
  const i64 d = dst[i], s = src[i], want = length[i];
  Plan p{};
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
    if (p.part > 0 && (int)want > kept)
      p.page = page_of(c, c.table[s * c.width + p.whole]);
    else if (p.part > 0)
      ++p.whole;  // nothing will be written behind the kept tokens
    const int old = pages_of(c, same ? have : row_length(c, c.length[d]));
    give_back_row(c, c.table + d * c.width, same ? p.held : 0, old);
  }
  if ((threadIdx.x & 63) == 0) plan[i] = p;
}

// Inclusive sum over the workgroup's threads; `total` of all.  The buffer holds one a wavefront.
__device__ inline i64 group_scan(i64 x, i64* buffer, i64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const i64 y = __shfl_up(x, off);
    if (lane >= off) x += y;
  }
  __syncthreads();  // the buffer's last readers
  if (lane == 63) buffer[wave] = x;
  __syncthreads();
  i64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kOneGroup / 64; ++w) {
    const i64 y = buffer[w];
    before += w < wave ? y : 0;
    total += y;
  }
  return x + before;
}

// New pages' numbers: each entry's first among all of them, then the lowest free pages in order
// (`fresh`), as many as the entries that fit use.
__global__ __launch_bounds__(kOneGroup) void place_kernel(Cache c, i64 n, Plan* __restrict__ plan,
                                                          int* __restrict__ fresh,
                                                          uint8_t* __restrict__ ok) {
  __shared__ i64 buffer[kOneGroup / 64];
  __shared__ int last_used;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int kWaves = kOneGroup / 64;
  if (threadIdx.x == 0) last_used = 0;
  // the free pages, a run of words a wavefront
  const int words = (c.pages + 63) >> 6;
  const int run = (words + kWaves - 1) / kWaves;
  const int from = min(wave * run, words), to = min(from + run, words);
  i64 count = 0, available;
  for (int w = from + lane; w < to; w += 64) count += __popcll(c.free[w]);
  const i64 upto = group_scan(count, buffer, available);
  // the free pages before this wavefront's run: its last lane's sum less its lanes' counts
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) count += __shfl_xor(count, off);
  int rank = (int)(__shfl(upto, 63) - count);
  i64 before = 0;
  for (i64 base = 0; base < n; base += kOneGroup) {
    const i64 i = base + threadIdx.x;
    Plan p{};
    int need = 0;
    if (i < n) {
      p = plan[i];
      if (p.flags & kFine) {
        // the part-filled page is copied unless it is the row's own already
        const bool ends = p.part > 0 && p.whole < p.held && p.page != -1;
        const bool gap = p.part > 0 && p.whole < p.held && p.page == -1;  // a table entry that is none
        if (ends && (p.flags & kSame) && c.refs[p.page] <= 1) ++p.whole;
        else if (ends) p.flags |= kCopy;
        else if (gap && (p.flags & kSame)) ++p.whole;
        need = p.held > p.whole ? p.held - p.whole : 0;
      }
    }
    i64 total;
    const i64 sum = group_scan(need, buffer, total);
    if (i < n) {
      const i64 end = before + sum;
      const bool fine = (p.flags & kFine) && (need == 0 || end <= available);
      if (fine && need > 0) atomicMax(&last_used, (int)end);
      p.first = fine ? (int)(end - need) : 0;
      if (!fine && (p.flags & kFine)) p.flags = (p.flags & kSame) | kLacking;
      plan[i] = p;
      ok[i] = fine;
    }
    before += total;
  }
  __syncthreads();
  const int used = last_used;
  for (int w = from; w < to && rank < used; w += 64) {
    const unsigned long long mine = w + lane < to ? c.free[w + lane] : 0;
    for (int k = 0; k < 64 && w + k < to && rank < used; ++k) {
      const unsigned long long bits = __shfl(mine, k);
      const int at = rank + __popcll(bits & ((1ull << lane) - 1));
      const bool take = (bits >> lane & 1) && at < used;
      if (take) {
        const int page = ((w + k) << 6) + lane;
        fresh[at] = page;
        c.refs[page] = 1;
      }
      const unsigned long long gone = __ballot(take);
      if (lane == 0 && gone) c.free[w + k] = bits & ~gone;
      rank += __popcll(bits);
    }
  }
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

__global__ __launch_bounds__(kThreads) void apply_kernel(Cache c, const i64* __restrict__ dst,
                                                         const i64* __restrict__ src, i64 n,
                                                         const Plan* __restrict__ plan,
                                                         const int* __restrict__ fresh) {
  const i64 i = blockIdx.x;
  const Plan p = plan[i];
  if (!(p.flags & (kFine | kLacking))) return;  // refused from the start
  const i64 d = dst[i], s = src[i];
  if (p.flags & kLacking) {
    if (!(p.flags & kSame) && blockIdx.y == 0 && threadIdx.x == 0) c.length[d] = 0;
    return;
  }
  const int wave = threadIdx.x >> 6;
  if (p.flags & kCopy) {
    const int units = p.part * c.token_bytes / 16;
    copy_page(c, p.page, fresh[p.first], units, blockIdx.y * (kThreads / 64) + wave,
              gridDim.y * (kThreads / 64));
  }
  if (blockIdx.y != 0) return;
  int32_t* row = c.table + d * c.width;
  const int32_t* from = c.table + s * c.width;
  const bool same = p.flags & kSame;
  for (int j = threadIdx.x; j < p.held; j += kThreads) {
    if (j >= p.whole) {
      row[j] = fresh[p.first + j - p.whole];
    } else if (!same) {
      const int32_t entry = from[j];
      const int page = page_of(c, entry);
      row[j] = entry;
      if (page >= 0) atomicAdd(c.refs + page, 1);
    }
  }
  if (threadIdx.x == 0) {
    if (same && (p.flags & kCopy)) give_back(c, p.page);
    c.length[d] = p.tokens;
  }
}

// ------------------------------------------------------------------------------ accept

// A wavefront an entry: which tokens are kept, and whether they may be.
__global__ __launch_bounds__(kThreads) void decide_kernel(
    Cache c, const i64* __restrict__ rows, const i64* __restrict__ start_in,
    const i64* __restrict__ keep, i64 keep_stride, i64 most, i64 n, const int* __restrict__ bad,
    Plan* __restrict__ plan, uint8_t* __restrict__ ok) {
  const i64 i = (i64)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (i >= n) return;
  const int lane = threadIdx.x & 63;
  const i64 row = rows[i], start = start_in[i];
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

constexpr int kPathChunk = 256;  // kept tokens whose places a workgroup holds at once
constexpr int kInFlight = 8;     // tokens a lane reads before it writes

// Moves the kept tokens of one entry's segments.  Kept ones rise, so a token's new place is never
// behind its old one: what is read before an earlier or equal token is written is right, and lanes
// of different segments or parts never meet.
__global__ __launch_bounds__(kThreads) void move_kernel(Cache c, const i64* __restrict__ rows,
                                                        const i64* __restrict__ keep,
                                                        i64 keep_stride,
                                                        const Plan* __restrict__ plan) {
  __shared__ i64 from[kPathChunk], to[kPathChunk];
  const i64 i = blockIdx.x;
  const Plan p = plan[i];
  if (!(p.flags & kFine)) return;
  const i64 row = rows[i];
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
  for (int base = p.whole; base < p.tokens; base += kPathChunk) {
    const int here = min(kPathChunk, p.tokens - base);
    __syncthreads();
    for (int j = threadIdx.x; j < here; j += kThreads) {
      from[j] = place(p.part + (int)keep[i * keep_stride + base + j]);
      to[j] = place(p.part + base + j);
    }
    __syncthreads();
    for (int s = (blockIdx.y * (kThreads / 64) + wave) * at_once + sub; s < segments;
         s += gridDim.y * (kThreads / 64) * at_once) {
      char* at = segment(c, s, 0) + unit * 16;
      for (int j = 0; j < here; j += kInFlight) {
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
inline i64 workspace_bytes(const Cache& c, i64 n, bool fresh) {
  return n * (i64)(sizeof(Plan) + sizeof(int)) + c.rows * (i64)sizeof(int) +
         (fresh ? c.pages * (i64)sizeof(int) : 0);
}

struct Workspace {
  Plan* plan;
  int *bad, *mark, *fresh;
  Workspace(void* at, const Cache& c, i64 n)
      : plan(static_cast<Plan*>(at)), bad(reinterpret_cast<int*>(plan + n)), mark(bad + n),
        fresh(mark + c.rows) {}
};

constexpr i64 kMostEntries = (i64)1 << 23;  // a launch has fewer than 2^32 threads in x

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
                     31 - __builtin_clz(c.token_bytes / 16), each);
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
  const Workspace w(workspace, c, n);
  const unsigned waves = (unsigned)((n + kThreads / 64 - 1) / (kThreads / 64));
  hipLaunchKernelGGL(claim_kernel, dim3(1), dim3(kOneGroup), 0, stream, dst, src, n, c.rows, w.mark,
                     w.bad);
  hipLaunchKernelGGL(release_kernel, dim3(waves), dim3(kThreads), 0, stream, c, dst, src, length, n,
                     w.bad, w.plan);
  hipLaunchKernelGGL(place_kernel, dim3(1), dim3(kOneGroup), 0, stream, c, n, w.plan, w.fresh, ok);
  hipLaunchKernelGGL(apply_kernel, dim3((unsigned)n, slices(c, n, 1)), dim3(kThreads), 0, stream, c,
                     dst, src, n, w.plan, w.fresh);
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
  const Workspace w(workspace, c, n);
  const unsigned waves = (unsigned)((n + kThreads / 64 - 1) / (kThreads / 64));
  hipLaunchKernelGGL(claim_kernel, dim3(1), dim3(kOneGroup), 0, stream, rows,
                     static_cast<const int64_t*>(nullptr), n, c.rows, w.mark, w.bad);
  hipLaunchKernelGGL(decide_kernel, dim3(waves), dim3(kThreads), 0, stream, c, rows, start, keep,
                     keep_stride, most, n, w.bad, w.plan, ok);
  hipLaunchKernelGGL(move_kernel, dim3((unsigned)n, slices(c, n, 1024 / c.token_bytes)),
                     dim3(kThreads), 0, stream, c, rows, keep, keep_stride, w.plan);
  return (int)hipGetLastError();
}

}  // extern "C"
