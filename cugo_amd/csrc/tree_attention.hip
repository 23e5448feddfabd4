// Attention of drafted tokens over a paged key/value cache, for gfx950 (include/cugo_hip.h,
// cugo_tree_attention):
//
//   out[i, h, :] = sum_t softmax_t(q[i, h, :] . K[t] scale) V[t]
//
// over the positions t of the query's row that lie before its sequence's prefix or whose bit is
// set in its mask.  A wavefront serves one query and head, its lanes a token's elements; softmax
// is online.
#include "paged.h"

namespace cugo_amd {
namespace paged {

struct BF16 {
  using storage = __bf16;
};
struct F16 {
  using storage = _Float16;
};
struct F32 {
  using storage = float;
};

struct Call {
  Cache c;
  i64 layer_offset;
  const char* q;
  i64 q_stride;  // elements
  i64 tokens, n, each;  // each: queries a sequence without offsets
  int heads, group;
  const i64* prefix;
  const i64* rows;
  const i64* offsets;
  const unsigned long long* mask;
  i64 mask_rows;
  int words;
  float scale_log2;
  char* out;
};

// The sequence whose queries `token` is among, or -1.
__device__ inline i64 sequence_of(const Call& a, i64 token, i64& first) {
  if (a.offsets == nullptr) {
    const i64 i = token / a.each;
    first = i * a.each;
    return i;
  }
  i64 low = 0, high = a.n;  // offsets[low] <= token < offsets[high], once both are known
  while (high - low > 1) {
    const i64 mid = (low + high) >> 1;
    if (a.offsets[mid] <= token) low = mid;
    else high = mid;
  }
  first = a.offsets[low];
  return token >= first && token < a.offsets[low + 1] ? low : -1;
}

template <class T, int DH>
__global__ __launch_bounds__(64) void simple_kernel(Call a) {
  using S = typename T::storage;
  constexpr int kEach = DH > 64 ? DH / 64 : 1;
  const Cache& c = a.c;
  const i64 token = blockIdx.x;
  const int head = blockIdx.y, lane = threadIdx.x;
  i64 first;
  const i64 i = sequence_of(a, token, first);
  if (i < 0) return;
  const bool mine = lane * kEach < DH;
  S* out = reinterpret_cast<S*>(a.out) + (token * a.heads + head) * DH + lane * kEach;
  const i64 row = a.rows ? a.rows[i] : i;
  if (row < 0 || row >= c.rows) {
    for (int e = 0; e < kEach; ++e)
      if (mine) out[e] = (S)__builtin_nanf("");
    return;
  }
  const int length = row_length(c, c.length[row]);
  const i64 p = a.prefix[i];
  const int prefix = (int)(p < 0 ? 0 : p > length ? length : p);
  const i64 j = token - first;
  const i64 span = a.mask ? (i64)a.words * 64 : j + 1;
  const int end = (int)(prefix + span < length ? prefix + span : length);
  const unsigned long long* mask = a.mask + (a.mask_rows == a.tokens ? token : j) * a.words;
  float q[kEach], acc[kEach] = {};
  for (int e = 0; e < kEach; ++e)
    q[e] = mine ? (float)reinterpret_cast<const S*>(a.q)[token * a.q_stride + head * DH + lane * kEach + e] : 0.f;
  float top = -__builtin_inff(), sum = 0.f;
  for (int t = 0; t < end; ++t) {
    const int b = t - prefix;
    if (b >= 0 && a.mask && !(mask[b >> 6] >> (b & 63) & 1)) continue;
    const int page = page_of(c, c.table[row * c.width + (t >> c.page_shift)]);
    const i64 at = a.layer_offset + slot_offset(c, page < 0 ? 0 : page, head / a.group, t & ((1 << c.page_shift) - 1));
    float s = 0.f, v[kEach];
    for (int e = 0; e < kEach; ++e) {
      s += mine ? q[e] * (float)reinterpret_cast<const S*>(c.k + at)[lane * kEach + e] : 0.f;
      v[e] = mine ? (float)reinterpret_cast<const S*>(c.v + at)[lane * kEach + e] : 0.f;
    }
    for (int off = 1; off < 64; off <<= 1) s += __shfl_xor(s, off);
    s *= a.scale_log2;
    if (page < 0) s = __builtin_nanf("");
    if (s == -__builtin_inff()) continue;
    const float now = fmaxf(top, s);
    const float less = top == now ? 1.f : __builtin_amdgcn_exp2f(top - now);
    const float w = s == now ? 1.f : __builtin_amdgcn_exp2f(s - now);
    top = now;
    sum = sum * less + w;
    for (int e = 0; e < kEach; ++e) acc[e] = acc[e] * less + w * v[e];
  }
  for (int e = 0; e < kEach; ++e)
    if (mine) out[e] = (S)(sum == 0.f ? 0.f : acc[e] / sum);
}

template <class T>
int by_dh(const Call& a, int dh, hipStream_t stream) {
  const dim3 grid((unsigned)a.tokens, (unsigned)a.heads);
  switch (dh) {
    case 32:
      hipLaunchKernelGGL((simple_kernel<T, 32>), grid, dim3(64), 0, stream, a);
      break;
    case 64:
      hipLaunchKernelGGL((simple_kernel<T, 64>), grid, dim3(64), 0, stream, a);
      break;
    case 128:
      hipLaunchKernelGGL((simple_kernel<T, 128>), grid, dim3(64), 0, stream, a);
      break;
    default:
      hipLaunchKernelGGL((simple_kernel<T, 256>), grid, dim3(64), 0, stream, a);
  }
  return (int)hipGetLastError();
}

// Checks a call as its documentation says and gives the kernels' view of it.
inline int view(const CugoTreeAttention* p, Call* a) {
  if (!p) return -1;
  if (const int bad = view(p->cache, &a->c)) return bad;
  if (p->layer < 0 || p->layer >= p->cache->layers || p->tokens < 0 || p->n < 0) return -1;
  if (p->heads <= 0 || p->heads > 65535 || p->heads % p->cache->kv_heads != 0) return -1;
  if (p->tokens >= (i64)1 << 24 || p->n >= (i64)1 << 24) return -1;
  if (p->q_stride < p->heads * p->cache->dh || p->words < 0 || p->words > (1 << 16)) return -1;
  if (p->tokens > 0 && (p->n == 0 || !p->q || !p->prefix || !p->out)) return -1;
  if (!p->offsets && p->n > 0 && p->tokens % p->n != 0) return -1;
  if (p->mask && p->mask_rows != p->tokens &&
      (p->offsets || p->n == 0 || p->mask_rows != p->tokens / p->n))
    return -1;
  const int size = element_size(p->cache->dtype);
  if (!aligned16(p->q) || !aligned16(p->out) || p->q_stride * size % 16 != 0) return -4;
  a->layer_offset = p->layer * a->c.layer_bytes;
  a->q = static_cast<const char*>(p->q);
  a->q_stride = p->q_stride;
  a->tokens = p->tokens;
  a->n = p->n;
  a->each = p->n > 0 ? p->tokens / p->n : 0;
  a->heads = (int)p->heads;
  a->group = (int)(p->heads / p->cache->kv_heads);
  a->prefix = p->prefix;
  a->rows = p->rows;
  a->offsets = p->offsets;
  a->mask = reinterpret_cast<const unsigned long long*>(p->mask);
  a->mask_rows = p->mask_rows;
  a->words = (int)p->words;
  a->scale_log2 = p->scale * 1.4426950408889634f;  // softmax in base 2
  a->out = static_cast<char*>(p->out);
  return 0;
}

}  // namespace paged
}  // namespace cugo_amd

extern "C" {

int64_t cugo_tree_attention_workspace(const CugoTreeAttention* call) {
  using namespace cugo_amd::paged;
  Call a;
  (void)view(call, &a);
  return 0;
}

int cugo_tree_attention(const CugoTreeAttention* call, void* workspace, int64_t workspace_bytes,
                        hipStream_t stream) {
  using namespace cugo_amd::paged;
  (void)workspace;
  (void)workspace_bytes;
  Call a;
  if (const int bad = view(call, &a)) return bad;
  if (a.tokens == 0) return 0;
  switch (call->cache->dtype) {
    case CUGO_DTYPE_BF16:
      return by_dh<BF16>(a, (int)call->cache->dh, stream);
    case CUGO_DTYPE_F16:
      return by_dh<F16>(a, (int)call->cache->dh, stream);
    default:
      return by_dh<F32>(a, (int)call->cache->dh, stream);
  }
}

}  // extern "C"
