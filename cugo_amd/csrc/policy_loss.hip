// The clipped policy loss with its KL term, entropy bonus and value loss, and its gradients.
//
// A row is one decision: its logits z, the legal actions, the action a that was taken, the
// log-probability it had then, its advantage A and weight w.  Over the legal actions,
//   l_j = z_j - log sum_k e^{z_k},  p_j = e^{l_j},  r = e^{l_a - old}
//   loss = sum_rows w [ -min(r A, clip(r, 1 - c_low, 1 + c_high) A)
//                       + c_v (V - R)^2 / 2 + c_k sum_j p_j (l_j - l'_j) + c_e sum_j p_j l_j ]
// with l' the log-probabilities of another policy's logits over the same actions.  With
// H = -sum_j p_j l_j, K = sum_j p_j (l_j - l'_j), and G = r A, or 0 where the clip cut it off:
//   d loss / d z_j = w [ G (p_j - [j = a]) + c_k p_j (l_j - l'_j - K) + c_e p_j (l_j + H) ]
//   d loss / d V = w c_v (V - R)
// The loss and both gradients come from one reading of the logits: the gradient for a factor
// of one on the loss needs nothing that the loss does not.
//
// Rows the sums leave out: w = 0 leaves out everything (whatever the row holds, its gradients
// are zeros); a row without a legal action, or whose legal logits are all -inf, has the value
// term alone.  An action that is illegal, outside the row or at a logit of -inf has
// probability 0: log-probability -inf, ratio 0, no gradient through the ratio.
// A logit whose exponential is 0 beside the row's largest (-inf, the type's lowest value) has
// p l = 0, as the limit is.
#include "learner.h"

#include <math.h>

namespace cugo_amd {
namespace learner {
namespace loss {

constexpr int kThreads = 256;
constexpr int kStats = 6;  // policy, value, kl, entropy, cut, drift: the sums' order
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxGroups = CUGO_POLICY_LOSS_PARTIALS / kStats;

struct LossArgs {
  const void* logits;
  const void* ref;
  const uint8_t* legal;
  i64 logits_stride, ref_stride, legal_stride, d_stride;
  const i64* action;
  const float* old_logp;
  const float* advantage;
  const float* weight;
  const void* value;
  const float* returns;
  const float* scale;
  i64 n;
  int actions, value_dtype;
  float even;  // the weight of every row where there is no list of them
  float least, most;  // the ratio's bounds
  float kl_coef, entropy_coef, value_coef;
  void* d_logits;
  void* d_value;
  float* logp;
  double* partials;
};

__device__ inline float load_value(const void* p, int dtype, i64 i) {
  if (dtype == CUGO_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == CUGO_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}

__device__ inline void store_value(void* p, int dtype, i64 i, float x) {
  if (dtype == CUGO_DTYPE_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == CUGO_DTYPE_F16) static_cast<_Float16*>(p)[i] = (_Float16)x;
  else static_cast<__bf16*>(p)[i] = (__bf16)x;
}

// A row's terms from the sums over its actions.  Every lane that serves the row computes them.
struct RowTerms {
  float a, b, c;   // d loss / d z_j = e_j (a + b d_j + c t_j) - [j = action] pull, with
  float pull;      // t_j = z_j - top, e_j = e^{t_j}, d_j = t_j - t'_j
  float stat[kStats];
  float logp, d_value;
  bool live;       // the row has policy terms and a weight
};

// top: the row's largest legal logit; s = sum e; u = sum e t; ref_log = log s'; ds = sum e d;
// at: the action's t, or -inf.
template <bool kRef>
__device__ inline RowTerms row_terms(const LossArgs& g, i64 r, bool some, float s, float u,
                                     float ds, float ref_log, float at) {
  RowTerms x;
  const float w = g.weight ? g.weight[r] : g.even;
  const float old = g.old_logp[r], adv = g.advantage[r];
  const float inv = some ? 1.0f / s : 0.0f;
  const float ls = some ? __builtin_amdgcn_logf(s) * kLn2 : 0.0f;  // v_log_f32: base 2
  const float entropy = ls - u * inv;
  const float shift = ls - ref_log;  // l_j - l'_j = d_j - shift
  const float kl = kRef ? ds * inv - shift : 0.0f;
  x.logp = some ? at - ls : 0.0f;
  const float drift = x.logp - old;
  const float ratio = x.logp == -INFINITY ? 0.0f : expf(drift);
  const float bound = fminf(fmaxf(ratio, g.least), g.most);
  const bool cut = ratio * adv > bound * adv;
  const float gain = cut ? bound * adv : ratio * adv;
  x.live = some && w != 0.0f;
  const float wp = x.live ? w : 0.0f;
  x.stat[0] = x.live ? -gain * wp : 0.0f;
  x.stat[2] = x.live ? kl * wp : 0.0f;
  x.stat[3] = x.live ? entropy * wp : 0.0f;
  x.stat[4] = cut ? wp : 0.0f;
  x.stat[5] = x.live ? (ratio - 1.0f - drift) * wp : 0.0f;
  const float unit = g.scale ? *g.scale : 1.0f;
  const float pull = cut ? 0.0f : ratio * adv;
  const float per = wp * unit * inv;
  x.a = per * (pull + g.entropy_coef * (entropy - ls) - (kRef ? g.kl_coef * (shift + kl) : 0.0f));
  x.b = kRef ? per * g.kl_coef : 0.0f;
  x.c = per * g.entropy_coef;
  x.pull = wp * unit * pull;
  x.stat[1] = x.d_value = 0.0f;
  if (g.value && w != 0.0f) {
    const float err = load_value(g.value, g.value_dtype, r) - g.returns[r];
    x.stat[1] = w * 0.5f * err * err;
    x.d_value = w * unit * g.value_coef * err;
  }
  return x;
}

__device__ inline float exp_of(float t) { return __builtin_amdgcn_exp2f(t * kLog2e); }

// A workgroup's sums (kStats of each of its 256 / G groups of lanes, in acc of the group's lane
// j = the sum's place) to its partials: in a fixed order, so a call's results are the same
// every time.
template <int G>
__device__ inline void write_partials(double acc, int j, double* partials) {
  __shared__ double sums[kThreads / G][kStats];
  if (j < kStats) sums[threadIdx.x / G][j] = acc;
  __syncthreads();
  if (threadIdx.x < kStats) {
    double total = 0.0;
    for (int k = 0; k < kThreads / G; ++k) total += sums[k][threadIdx.x];
    partials[(i64)blockIdx.x * kStats + threadIdx.x] = total;
  }
}

// Rows of up to 4 V G actions (V in 1..4): G lanes a row, vector i of E elements of lane j at
// action (i G + j) E, so that the row's lanes read one run of memory an instruction; the row
// stays in registers.  The last vector of a row that ends inside it is moved back to end with
// the row, where it repeats elements of other lanes: those (`mine` false) are left out of the
// sums, and their gradients stored twice, the same value.
template <class T, int G, int V, int E, bool kRef>
__global__ __launch_bounds__(kThreads) void loss_rows_kernel(const LossArgs g) {
  using S = typename T::storage;
  const int j = threadIdx.x & (G - 1);
  const int at = ((V - 1) * G + j) * E;  // the last vector's first action, where it fits
  const int last = min(at, g.actions - E);
  bool mine[E];
#pragma unroll
  for (int e = 0; e < E; ++e) mine[e] = last + e >= at;
  const bool any_mine = at < g.actions;
  constexpr int kRows = kThreads / G;
  const i64 tiles = (g.n + kRows - 1) / kRows;
  double acc = 0.0;
  for (i64 tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const i64 row = tile * kRows + threadIdx.x / G;
    const bool ok = row < g.n;
    const i64 r = ok ? row : g.n - 1;  // loads are unconditional; the sums leave it out
    const S* zs = static_cast<const S*>(g.logits) + r * g.logits_stride;
    const S* qs = static_cast<const S*>(g.ref) + (kRef ? r * g.ref_stride : 0);
    const uint8_t* ls = g.legal ? g.legal + r * g.legal_stride : nullptr;
    Any<S, E> zv[V], qv[V];
    Any<uint8_t, E> lv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int k = i + 1 < V ? (i * G + j) * E : last;
      zv[i] = *reinterpret_cast<const Any<S, E>*>(zs + k);
      if constexpr (kRef) qv[i] = *reinterpret_cast<const Any<S, E>*>(qs + k);
      if (ls) lv[i] = *reinterpret_cast<const Any<uint8_t, E>*>(ls + k);
      else
#pragma unroll
        for (int e = 0; e < E; ++e) lv[i].v[e] = 1;
    }
    const i64 act = g.action[r];
    const bool inside = act >= 0 && act < g.actions;
    const i64 ac = inside ? act : 0;
    const bool taken = inside && (!ls || ls[ac]);
    const float za = T::to_float(zs[ac]);
    float t[V * E], d[kRef ? V * E : 1];
    float top = -INFINITY, top_ref = -INFINITY;
#pragma unroll
    for (int i = 0; i < V * E; ++i) {
      const bool on = lv[i / E].v[i % E] != 0;
      t[i] = on ? T::to_float(zv[i / E].v[i % E]) : -INFINITY;
      top = fmaxf(top, t[i]);
      if constexpr (kRef) {
        d[i] = on ? T::to_float(qv[i / E].v[i % E]) : -INFINITY;
        top_ref = fmaxf(top_ref, d[i]);
      }
    }
    top = group_max<G>(top);
    const bool some = top > -INFINITY;
    top = some ? top : 0.0f;
    if constexpr (kRef) {
      top_ref = group_max<G>(top_ref);
      top_ref = top_ref > -INFINITY ? top_ref : 0.0f;
    }
    float s = 0.0f, u = 0.0f, sr = 0.0f, ds = 0.0f, p[V * E];
#pragma unroll
    for (int i = 0; i < V * E; ++i) {
      const bool here = i / E + 1 < V || mine[i % E];
      t[i] -= top;
      p[i] = exp_of(t[i]);
      const bool has = !(p[i] == 0.0f);
      const float ps = here ? p[i] : 0.0f;
      if constexpr (kRef) {
        const float q = d[i] - top_ref;
        sr += here ? exp_of(q) : 0.0f;
        d[i] = has ? t[i] - q : 0.0f;
        ds = __builtin_fmaf(ps, d[i], ds);
      }
      t[i] = has ? t[i] : 0.0f;
      s += ps;
      u = __builtin_fmaf(ps, t[i], u);
    }
    s = group_sum<G>(s);
    u = group_sum<G>(u);
    float ref_log = 0.0f;
    if constexpr (kRef) {
      ds = group_sum<G>(ds);
      ref_log = __builtin_amdgcn_logf(group_sum<G>(sr)) * kLn2;
    }
    const RowTerms x = row_terms<kRef>(g, r, some, s, u, ds, ref_log,
                                       taken ? za - top : -INFINITY);
    float stat = x.stat[5];
#pragma unroll
    for (int k = 0; k < kStats - 1; ++k) stat = j == k ? x.stat[k] : stat;
    acc += ok ? (double)stat : 0.0;
    if (!ok) continue;
    if (j == 0) {
      g.logp[r] = x.logp;
      if (g.d_value) store_value(g.d_value, g.value_dtype, r, x.d_value);
    }
    if (g.d_logits) {
      S* out = static_cast<S*>(g.d_logits) + r * g.d_stride;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int k = i + 1 < V ? (i * G + j) * E : last;
        Any<S, E> o;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int m = i * E + e;
          float h = __builtin_fmaf(x.c, t[m], x.a);
          if constexpr (kRef) h = __builtin_fmaf(x.b, d[m], h);
          const float hit = act == k + e ? x.pull : 0.0f;
          const float f = __builtin_fmaf(p[m], h, -hit);
          o.v[e] = T::from_float(x.live ? f : 0.0f);
        }
        if (i + 1 < V || any_mine) *reinterpret_cast<Any<S, E>*>(out + k) = o;
      }
    }
  }
  write_partials<G>(acc, j, g.partials);
}

// Longer rows: a workgroup a row, in two passes over it.  The first keeps each thread's
// running maximum and the sums under it, moved along with the maximum; the second reads the
// row again, from the caches, for the gradient.

// The factor that a move of the maximum by `move` (<= 0) puts on sums of e^t, and a sum of
// e^t t moved so; s is the sum of e^t.  What underflows is dropped, whatever it was: logits of
// the type's lowest value make infinities of such a sum until an ordinary one comes.
__device__ inline float moved(float f, float u, float s, float move) {
  return f == 0.0f ? 0.0f : f * __builtin_fmaf(s, move, u);
}

template <class T, bool kRef>
__global__ __launch_bounds__(kThreads) void loss_wide_kernel(const LossArgs g) {
  using S = typename T::storage;
  constexpr int E = 16 / sizeof(S);
  constexpr int kWaves = kThreads / 64;
  __shared__ float shared[kWaves][6];
  double acc = 0.0;
  for (i64 r = blockIdx.x; r < g.n; r += gridDim.x) {
    const S* zs = static_cast<const S*>(g.logits) + r * g.logits_stride;
    const S* qs = static_cast<const S*>(g.ref) + (kRef ? r * g.ref_stride : 0);
    const uint8_t* ls = g.legal ? g.legal + r * g.legal_stride : nullptr;
    float top = -INFINITY, s = 0.0f, u = 0.0f, top_ref = -INFINITY, sr = 0.0f, ds = 0.0f;
    // E elements from action c on, or the row's last E where it ends before c + E
    auto read = [&](int c, int& k, float (&z)[E], float (&q)[E]) {
      k = min(c, g.actions - E);
      const Any<S, E> zv = *reinterpret_cast<const Any<S, E>*>(zs + k);
      Any<S, E> qv;
      if constexpr (kRef) qv = *reinterpret_cast<const Any<S, E>*>(qs + k);
      Any<uint8_t, E> lv;
      if (ls) lv = *reinterpret_cast<const Any<uint8_t, E>*>(ls + k);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool on = !ls || lv.v[e] != 0;
        z[e] = on ? T::to_float(zv.v[e]) : -INFINITY;
        if constexpr (kRef) q[e] = on ? T::to_float(qv.v[e]) : -INFINITY;
      }
    };
    for (int c = threadIdx.x * E; c < g.actions; c += kThreads * E) {
      int k;
      float z[E], q[E];
      read(c, k, z, q);
      float most = top, most_ref = top_ref;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        most = fmaxf(most, z[e]);
        if constexpr (kRef) most_ref = fmaxf(most_ref, q[e]);
      }
      const float base = most > -INFINITY ? most : 0.0f;
      const float f = exp_of(top - base);
      float base_ref = 0.0f;
      if constexpr (kRef) {
        base_ref = most_ref > -INFINITY ? most_ref : 0.0f;
        ds = moved(f, ds, s, (top - base) - (top_ref - base_ref));
        sr *= exp_of(top_ref - base_ref);
        top_ref = most_ref;
      }
      u = moved(f, u, s, top - base);
      s *= f;
      top = most;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool here = k + e >= c;
        const float t = z[e] - base;
        const float p = here ? exp_of(t) : 0.0f;
        const bool has = !(p == 0.0f);
        s += p;
        u = __builtin_fmaf(p, has ? t : 0.0f, u);
        if constexpr (kRef) {
          const float tr = q[e] - base_ref;
          sr += here ? exp_of(tr) : 0.0f;
          ds = __builtin_fmaf(p, has ? t - tr : 0.0f, ds);
        }
      }
    }
    // the threads' sums under the row's maximum
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    __syncthreads();  // the last row's values have been read
    float all = group_max<64>(top), all_ref = kRef ? group_max<64>(top_ref) : 0.0f;
    if (lane == 0) shared[wave][0] = all, shared[wave][1] = all_ref;
    __syncthreads();
    for (int k = 0; k < kWaves; ++k) {
      all = fmaxf(all, shared[k][0]);
      all_ref = fmaxf(all_ref, shared[k][1]);
    }
    const bool some = all > -INFINITY;
    all = some ? all : 0.0f;
    const float f = exp_of(top - all);
    u = group_sum<64>(moved(f, u, s, top - all));
    if constexpr (kRef) {
      all_ref = all_ref > -INFINITY ? all_ref : 0.0f;
      ds = group_sum<64>(moved(f, ds, s, (top - all) - (top_ref - all_ref)));
      sr = group_sum<64>(sr * exp_of(top_ref - all_ref));
    }
    s = group_sum<64>(s * f);
    if (lane == 0) shared[wave][2] = s, shared[wave][3] = u, shared[wave][4] = ds, shared[wave][5] = sr;
    __syncthreads();
    s = u = ds = sr = 0.0f;
    for (int k = 0; k < kWaves; ++k) {
      s += shared[k][2];
      u += shared[k][3];
      ds += shared[k][4];
      sr += shared[k][5];
    }
    const float ref_log = kRef ? __builtin_amdgcn_logf(sr) * kLn2 : 0.0f;
    const i64 act = g.action[r];
    const bool inside = act >= 0 && act < g.actions;
    const bool taken = inside && (!ls || ls[act]);
    const float za = T::to_float(zs[inside ? act : 0]);
    const RowTerms x = row_terms<kRef>(g, r, some, s, u, ds, ref_log,
                                       taken ? za - all : -INFINITY);
    float stat = x.stat[5];
#pragma unroll
    for (int k = 0; k < kStats - 1; ++k) stat = (int)threadIdx.x == k ? x.stat[k] : stat;
    acc += (double)stat;
    if (threadIdx.x == 0) {
      g.logp[r] = x.logp;
      if (g.d_value) store_value(g.d_value, g.value_dtype, r, x.d_value);
    }
    if (g.d_logits) {
      S* out = static_cast<S*>(g.d_logits) + r * g.d_stride;
      for (int c = threadIdx.x * E; c < g.actions; c += kThreads * E) {
        int k;
        float z[E], q[E];
        read(c, k, z, q);
        Any<S, E> o;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float t = z[e] - all;
          const float p = exp_of(t);
          const bool has = !(p == 0.0f);
          float h = __builtin_fmaf(x.c, has ? t : 0.0f, x.a);
          if constexpr (kRef) h = __builtin_fmaf(x.b, has ? t - (q[e] - all_ref) : 0.0f, h);
          const float hit = act == k + e ? x.pull : 0.0f;
          const float v = __builtin_fmaf(p, h, -hit);
          o.v[e] = T::from_float(x.live ? v : 0.0f);
        }
        *reinterpret_cast<Any<S, E>*>(out + k) = o;
      }
    }
  }
  // lanes 0 .. kStats - 1 of the workgroup hold its sums
  if (threadIdx.x < kStats) g.partials[(i64)blockIdx.x * kStats + threadIdx.x] = acc;
}

// The workgroups' sums added up, and the loss of them.  One workgroup of kTotalThreads (a
// multiple of kStats, so that a thread's loads are of one sum, and the whole grid's partials are
// a few loads in flight for each thread): 3 us behind 2,048 workgroups, where a wavefront for each
// sum took 10.
constexpr int kTotalThreads = 960;
static_assert(kTotalThreads % kStats == 0 && kTotalThreads % 64 == 0, "one sum a thread");
__global__ __launch_bounds__(kTotalThreads) void loss_total_kernel(
    const double* partials, int groups, double kl_coef, double entropy_coef, double value_coef,
    const float* scale, float* out) {
  constexpr int kEach = kTotalThreads / kStats;  // threads a sum
  __shared__ double sums[kTotalThreads];
  __shared__ double totals[kStats];
  const int count = groups * kStats;
  double total = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < count; i += kTotalThreads) total += partials[i];
  sums[threadIdx.x] = total;
  __syncthreads();
  const int k = threadIdx.x / 64, lane = threadIdx.x % 64;
  if (k < kStats) {
    total = 0.0;
    for (int i = lane; i < kEach; i += 64) total += sums[i * kStats + k];
    for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off);
    if (lane == 0) {
      totals[k] = total;
      out[1 + k] = (float)total;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const double loss = totals[0] + value_coef * totals[1] + kl_coef * totals[2] -
                        entropy_coef * totals[3];
    out[0] = (float)(loss * (scale ? (double)*scale : 1.0));
  }
}

// x times *factor in place, for a factor other than 1 (whose gradients are right already).
template <class T>
__device__ inline void scale_all(void* data, i64 count, float factor) {
  using S = typename T::storage;
  S* x = static_cast<S*>(data);
  const i64 stride = (i64)gridDim.x * kThreads;
  for (i64 i = (i64)blockIdx.x * kThreads + threadIdx.x; i < count; i += stride)
    x[i] = T::from_float(T::to_float(x[i]) * factor);
}

__device__ inline void scale_any(int dtype, void* data, i64 count, float factor) {
  if (dtype == CUGO_DTYPE_F32) scale_all<F32>(data, count, factor);
  else if (dtype == CUGO_DTYPE_F16) scale_all<F16>(data, count, factor);
  else scale_all<BF16>(data, count, factor);
}

__global__ __launch_bounds__(kThreads) void scale_kernel(int a_dtype, void* a, i64 a_count,
                                                         int b_dtype, void* b, i64 b_count,
                                                         const float* factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  scale_any(a_dtype, a, a_count, f);
  scale_any(b_dtype, b, b_count, f);
}

// The workgroups of a launch over `tiles` pieces of work: as many as are resident at once.
inline int groups_for(i64 tiles) {
  const i64 most = (i64)compute_units() * 8;
  const i64 cap = most < kMaxGroups ? most : kMaxGroups;
  return (int)(tiles < cap ? tiles : cap);
}

template <class T, bool kRef>
int launch_loss(const LossArgs& g, hipStream_t stream) {
  const auto rows = [&](auto kernel, int lanes) {
    const int per = kThreads / lanes;
    const int groups = groups_for((g.n + per - 1) / per);
    kernel<<<groups, kThreads, 0, stream>>>(g);
    return groups;
  };
  const int a = g.actions;
  if (a < 4) return rows(loss_rows_kernel<T, 16, 1, 1, kRef>, 16);
  if (a <= 64) return rows(loss_rows_kernel<T, 16, 1, 4, kRef>, 16);
  if (a <= 128) return rows(loss_rows_kernel<T, 16, 2, 4, kRef>, 16);
  if (a <= 192) return rows(loss_rows_kernel<T, 16, 3, 4, kRef>, 16);
  if (a <= 256) return rows(loss_rows_kernel<T, 16, 4, 4, kRef>, 16);
  if (a <= 512) return rows(loss_rows_kernel<T, 64, 2, 4, kRef>, 64);
  if (a <= 768) return rows(loss_rows_kernel<T, 64, 3, 4, kRef>, 64);
  if (a <= 1024) return rows(loss_rows_kernel<T, 64, 4, 4, kRef>, 64);
  return rows(loss_wide_kernel<T, kRef>, kThreads);
}

}  // namespace loss
}  // namespace learner
}  // namespace cugo_amd

using namespace cugo_amd::learner;
using namespace cugo_amd::learner::loss;

extern "C" {

int cugo_policy_loss(const CugoPolicyLoss* p, hipStream_t stream) {
  if (!p || p->n < 0 || p->actions < 1 || p->actions > (1 << 30) || !p->out || !p->partials)
    return -1;
  if (!dtype_known(p->logits_dtype) || (p->value && !dtype_known(p->value_dtype))) return -2;
  if (p->n > 0 && (!p->logits || !p->action || !p->old_logp || !p->advantage || !p->logp))
    return -1;
  if ((p->value != nullptr) != (p->returns != nullptr) || (p->d_value && !p->value)) return -1;
  LossArgs g{};
  g.logits = p->logits, g.ref = p->ref_logits, g.legal = p->legal;
  g.logits_stride = p->logits_stride, g.ref_stride = p->ref_stride;
  g.legal_stride = p->legal_stride, g.d_stride = p->d_logits_stride;
  g.action = p->action, g.old_logp = p->old_logp, g.advantage = p->advantage;
  g.weight = p->weight, g.value = p->value, g.returns = p->returns, g.scale = p->scale;
  g.n = p->n, g.actions = (int)p->actions, g.value_dtype = p->value_dtype;
  g.even = p->n > 0 ? (float)(1.0 / (double)p->n) : 0.0f;
  g.least = (float)(1.0 - p->clip_low), g.most = (float)(1.0 + p->clip_high);
  g.kl_coef = (float)p->kl_coef, g.entropy_coef = (float)p->entropy_coef;
  g.value_coef = (float)p->value_coef;
  g.d_logits = p->d_logits, g.d_value = p->d_value, g.logp = p->logp, g.partials = p->partials;
  int groups = 0;
  if (p->n > 0) {
    const bool ref = p->ref_logits != nullptr;
    if (p->logits_dtype == CUGO_DTYPE_F32)
      groups = ref ? launch_loss<F32, true>(g, stream) : launch_loss<F32, false>(g, stream);
    else if (p->logits_dtype == CUGO_DTYPE_F16)
      groups = ref ? launch_loss<F16, true>(g, stream) : launch_loss<F16, false>(g, stream);
    else
      groups = ref ? launch_loss<BF16, true>(g, stream) : launch_loss<BF16, false>(g, stream);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
  }
  loss_total_kernel<<<1, kTotalThreads, 0, stream>>>(p->partials, groups, p->kl_coef,
                                                   p->entropy_coef, p->value_coef, p->scale,
                                                   p->out);
  return (int)hipGetLastError();
}

int cugo_scale_gradients(int a_dtype, void* a, int64_t a_count, int b_dtype, void* b,
                         int64_t b_count, const float* factor, hipStream_t stream) {
  if (a_count < 0 || b_count < 0 || (a_count > 0 && !a) || (b_count > 0 && !b) || !factor)
    return -1;
  if (!dtype_known(a_dtype) || !dtype_known(b_dtype)) return -2;
  const int64_t most = a_count > b_count ? a_count : b_count;
  if (most == 0) return 0;
  const int groups = groups_for((most + kThreads - 1) / kThreads);
  scale_kernel<<<groups, kThreads, 0, stream>>>(a_dtype, a, a_count, b_dtype, b, b_count, factor);
  return (int)hipGetLastError();
}

}  // extern "C"
