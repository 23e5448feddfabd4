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
// The loss and both gradients come from one reading of the logits (two, where a row is too long to
// be held): the gradient for a factor of one on the loss needs nothing that the loss does not.
//
// Rows the sums leave out: w = 0 leaves out everything (whatever the row holds, its gradients
// are zeros); a row without a legal action, or whose legal logits are all -inf, has the value
// term alone.  An action that is illegal, outside the row or at a logit of -inf has
// probability 0: log-probability -inf, ratio 0, no gradient through the ratio.
// A logit whose exponential is 0 beside the row's largest (-inf, the type's lowest value) has
// p l = 0, as the limit is, and p times the row's terms 0 where those are infinite or NaN: what is
// illegal has no gradient whatever the rest of the row holds.
#include "learner.h"

#include <math.h>

#include <type_traits>

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

// The address of value r.
__device__ inline const void* at_row(const void* p, int dtype, i64 r) {
  return static_cast<const char*>(p) + r * (dtype == CUGO_DTYPE_F32 ? 4 : 2);
}

__device__ inline float load_value(const void* p, int dtype, uint32_t i) {
  if (dtype == CUGO_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == CUGO_DTYPE_F16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}

__device__ inline void store_value(void* p, int dtype, uint32_t i, float x) {
  if (dtype == CUGO_DTYPE_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == CUGO_DTYPE_F16) static_cast<_Float16*>(p)[i] = (_Float16)x;
  else static_cast<__bf16*>(p)[i] = (__bf16)x;
}

// What a row's terms need beside its logits, read ahead of them.
struct RowInputs {
  float w, old, adv, value, returns;
};

// Row r + i; r is the same for the workgroup, so that a lane's addresses are scalars and 32 bits.
__device__ inline RowInputs row_inputs(const LossArgs& g, i64 r, uint32_t i) {
  RowInputs in;
  in.w = g.weight ? (g.weight + r)[i] : g.even;
  in.old = (g.old_logp + r)[i];
  in.adv = (g.advantage + r)[i];
  in.value = in.returns = 0.0f;
  if (g.value) {
    in.value = load_value(at_row(g.value, g.value_dtype, r), g.value_dtype, i);
    in.returns = (g.returns + r)[i];
  }
  return in;
}

// Exponents are in base 2: x = (z - top) log2 e, so that e^(z - top) = 2^x.  The difference comes
// first: the largest logit has x = 0 exactly, and a row's only action the log-probability 0 (as one
// multiply-add, z k - top k, x would keep the rounding of top k).
struct Scale {
  float top;
  __device__ float operator()(float z) const { return (z - top) * kLog2e; }
};
__device__ inline Scale scale_for(float top) { return Scale{top == -INFINITY ? 0.0f : top}; }
__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's terms from the sums over its actions.  Every lane that serves the row computes them.
struct RowTerms {
  float a, b, c;   // d loss / d z_j = 2^x_j (a + b d_j + c x_j) - [j = action] pull, with
  float pull;      // d_j = x_j - x'_j
  float stat[kStats];
  float logp, d_value;
  bool live;       // the row has policy terms and a weight
};

// s = sum 2^x; u = sum 2^x x; ds = sum 2^x d; sr = sum 2^x'; at: the action's x, or -inf.
// A row with an action above -inf has a sum of 1 and more, or NaN for a NaN among its logits,
// which the largest logit does not show.
template <bool kRef>
__device__ inline RowTerms row_terms(const LossArgs& g, const RowInputs& in, float s, float u,
                                     float ds, float sr, float at) {
  RowTerms x;
  const bool some = !(s == 0.0f);
  const float inv = some ? __builtin_amdgcn_rcpf(s) : 0.0f;
  const float ls = some ? __builtin_amdgcn_logf(s) : 0.0f;  // v_log_f32: base 2
  const float mean = u * inv;
  const float entropy = (ls - mean) * kLn2;
  const float shift = kRef ? ls - __builtin_amdgcn_logf(sr) : 0.0f;  // l_j - l'_j = (d_j - shift) ln 2
  const float kl2 = ds * inv;
  const float kl = kRef ? (kl2 - shift) * kLn2 : 0.0f;
  x.logp = some ? (at - ls) * kLn2 : 0.0f;
  const float drift = x.logp - in.old;
  const float ratio = x.logp == -INFINITY ? 0.0f : exp2_of(drift * kLog2e);
  const float bound = fminf(fmaxf(ratio, g.least), g.most);
  const bool cut = ratio * in.adv > bound * in.adv;
  const float gain = (cut ? bound : ratio) * in.adv;
  x.live = some && in.w != 0.0f;
  x.stat[0] = x.live ? -gain * in.w : 0.0f;
  x.stat[2] = x.live ? kl * in.w : 0.0f;
  x.stat[3] = x.live ? entropy * in.w : 0.0f;
  x.stat[4] = x.live && cut ? in.w : 0.0f;
  x.stat[5] = x.live ? (ratio - 1.0f - drift) * in.w : 0.0f;
  const float wu = in.w * (g.scale ? *g.scale : 1.0f);
  const float pull = cut || x.logp == -INFINITY ? 0.0f : ratio * in.adv;
  const float per = wu * inv;
  // c_e p (l + H) = c_e p ln 2 (x - mean);  c_k p (l - l' - K) = c_k p ln 2 (d - kl2)
  x.c = per * (g.entropy_coef * kLn2);
  x.b = kRef ? per * (g.kl_coef * kLn2) : 0.0f;
  x.a = per * pull - x.c * mean - (kRef ? x.b * kl2 : 0.0f);
  x.pull = wu * pull;
  x.stat[1] = x.d_value = 0.0f;
  if (g.value && in.w != 0.0f) {
    const float err = in.value - in.returns;
    x.stat[1] = in.w * 0.5f * err * err;
    x.d_value = wu * g.value_coef * err;
  }
  return x;
}

// A workgroup's sums to its partials: lane j of each of its 256 / G groups of lanes holds sum j in
// acc[0] (and sum j + G in acc[1], for G = 4).  In a fixed order, so a call's results are the same
// every time.
template <int G>
constexpr int kHeld = (kStats + G - 1) / G;  // sums a lane holds
template <int G>
__device__ inline void write_partials(const double (&acc)[kHeld<G>], int j, double* partials) {
  __shared__ double sums[kThreads / G][kStats];
#pragma unroll
  for (int h = 0; h < kHeld<G>; ++h)
    if (j + h * G < kStats) sums[threadIdx.x / G][j + h * G] = acc[h];
  __syncthreads();
  if (threadIdx.x < kStats) {
    double total = 0.0;
    for (int k = 0; k < kThreads / G; ++k) total += sums[k][threadIdx.x];
    partials[(i64)blockIdx.x * kStats + threadIdx.x] = total;
  }
}

// Element i from a base that is the same for the wavefront: a scalar address and 32 bits of
// offset, where 64-bit addresses of every access would hold twice the registers.
template <class S>
__device__ inline S* element(S* base, uint32_t i) {
  return reinterpret_cast<S*>(reinterpret_cast<uintptr_t>(base) + i * (uint32_t)sizeof(S));
}

// What one lane wrote to LDS before is what another lane of the wavefront reads after.
__device__ inline void wavefront_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// What a row has besides its logits, for the rows of 16 lanes and more: lane 0 of 16 reads the old
// log-probability, lane 1 the advantage and so on, one access instead of six (the addresser, not
// memory, is what short rows keep busy), and all take the values from those lanes.
struct RowReader {
  const char* base;
  int shift;  // of the row's number

  __device__ explicit RowReader(const LossArgs& g) {
    const int k = threadIdx.x & 15;
    const void* p = k == 1 ? g.advantage : g.old_logp;
    p = k == 2 && g.returns ? static_cast<const void*>(g.returns) : p;
    p = k == 3 && g.weight ? static_cast<const void*>(g.weight) : p;
    p = k == 4 && g.value && g.value_dtype == CUGO_DTYPE_F32 ? g.value : p;
    p = k == 5 ? static_cast<const void*>(g.action) : p;
    p = k == 6 ? static_cast<const void*>(reinterpret_cast<const int32_t*>(g.action) + 1) : p;
    base = static_cast<const char*>(p);
    shift = k == 5 || k == 6 ? 3 : 2;
  }
  template <int kLane>
  __device__ static int from(int x) {
    return __builtin_amdgcn_update_dpp(0, x, 0x150 + kLane, 0xf, 0xf, false);
  }
  // Row r; lane's part of it, to be passed to inputs() once the row's logits are asked for too.
  __device__ int read(i64 r) const { return *reinterpret_cast<const int*>(base + (r << shift)); }
  __device__ RowInputs inputs(const LossArgs& g, int x, i64 r0, uint32_t i0, i64& act) const {
    RowInputs in;
    in.old = __int_as_float(from<0>(x));
    in.adv = __int_as_float(from<1>(x));
    in.w = g.weight ? __int_as_float(from<3>(x)) : g.even;
    in.value = in.returns = 0.0f;
    if (g.value) {
      in.returns = __int_as_float(from<2>(x));
      in.value = g.value_dtype == CUGO_DTYPE_F32
                     ? __int_as_float(from<4>(x))
                     : load_value(at_row(g.value, g.value_dtype, r0), g.value_dtype, i0);
    }
    act = (i64)(((uint64_t)(uint32_t)from<6>(x) << 32) | (uint32_t)from<5>(x));
    return in;
  }
};

// Rows of up to E V G actions (V in 1..4): G lanes a row, vector i of E elements of lane j at
// action (i G + j) E, so that the row's lanes read one run of memory an instruction.  The last
// vector of a row that ends inside it is read moved back, to end with the row; the elements that
// it repeats of other lanes count as illegal here, and their gradients are stored twice, the same.
// The row goes through LDS as it was read, in slots: an action's slot is its number, but in the
// moved vector.  From there it is gone through for its largest logit, for its sums and for its
// gradient, a vector of each lane at a time: kept in registers for that, a row of 179 actions
// took 96 to 112 of them and left four wavefronts a SIMD.
// A game's row has about ten legal actions of 179, and an exponential or a product for each action
// takes longer than memory does: where each row of a wavefront of 16-lane rows has at most two legal
// actions a lane, a list of their slots is made, a lane computes two of them, and the gradient is put
// together in LDS.  1,048,576 x 179 bf16 with a KL term, 10 legal actions a row: 298 us (4.5 TB/s;
// the arithmetic is half of that), with 63, where the list does not hold them, 416.
template <class T, int G, int V, int E, bool kRef>
__global__ __launch_bounds__(kThreads) void loss_rows_kernel(const LossArgs g) {
  using S = typename T::storage;
  constexpr int kBytes = E * sizeof(S);
  using Slots = Vec<S, E>;
  constexpr int kRows = kThreads / G;
  constexpr int kSlots = V * G * E;
  // A slot of 16 lanes fits a byte, and their counts one DPP row; on fewer lanes rows are too short
  // for a list to pay.
  constexpr bool kList = G == 16;
  __shared__ __align__(16) S z_slots[kRows][kSlots];
  __shared__ __align__(16) S q_slots[kRef ? kRows : 1][kRef ? kSlots : E];
  __shared__ uint8_t lists[kList ? kRows : 1][2 * G];
  const int j = threadIdx.x & (G - 1), row = threadIdx.x / G;
  const int at = ((V - 1) * G + j) * E;  // the last vector's first action, where it fits
  const int last = min(at, g.actions - E);
  // the bits of the lane's elements (element e of vector i at bit E i + e) that are its own
  uint32_t own = (1u << (E * (V - 1))) - 1u;
#pragma unroll
  for (int e = 0; e < E; ++e) own |= (last + e >= at ? 1u : 0u) << (E * (V - 1) + e);
  S* zl = z_slots[row];
  S* ql = q_slots[kRef ? row : 0];
  const RowReader reader(g);
  const i64 tiles = (g.n + kRows - 1) / kRows;
  double acc[kHeld<G>] = {};
  for (i64 tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const i64 r0 = tile * kRows;
    const bool ok = r0 + row < g.n;
    // loads are unconditional, of a row that exists; the sums leave it out
    const uint32_t i0 = (uint32_t)(ok ? row : (int)(g.n - 1 - r0));
    int part = 0;
    if constexpr (G >= 16) part = reader.read(r0 + i0);
    uint32_t bits = own;
    {
      const S* zb = static_cast<const S*>(g.logits) + r0 * g.logits_stride;
      const S* qb = static_cast<const S*>(g.ref) + (kRef ? r0 * g.ref_stride : 0);
      const uint32_t z_at = i0 * (uint32_t)g.logits_stride;
      const uint32_t q_at = kRef ? i0 * (uint32_t)g.ref_stride : 0u;
      Raw<kBytes> z[V], q[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint32_t k = (uint32_t)(i + 1 < V ? (i * G + j) * E : last);
        z[i] = reinterpret_cast<const RawAny<kBytes>*>(element(zb, z_at + k))->v;
        if constexpr (kRef)
          q[i] = reinterpret_cast<const RawAny<kBytes>*>(element(qb, q_at + k))->v;
      }
      if (g.legal) {
        const uint8_t* lb = g.legal + r0 * g.legal_stride;
        const uint32_t l_at = i0 * (uint32_t)g.legal_stride;
        uint32_t legal = 0;
        if constexpr (E == 4) {
          uint32_t w[V];
#pragma unroll
          for (int i = 0; i < V; ++i)
            w[i] = reinterpret_cast<const RawAny<4>*>(
                       lb + (l_at + (uint32_t)(i + 1 < V ? (i * G + j) * E : last)))->v;
          // a byte that is not 0 sets its upper bit, and a product of bytes gathers those
          uint32_t low = 0, high = 0;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const uint32_t set = (((w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[i]) & 0x80808080u;
            uint32_t& sum = i < 2 ? low : high;
            sum = __builtin_amdgcn_udot4(set, i % 2 ? 0x80402010u : 0x08040201u, sum, false);
          }
          legal = (low >> 7) | (high << 1);
        } else {
          legal = lb[l_at + (uint32_t)last] != 0;
        }
        bits &= legal;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int k = (i * G + j) * E;
        *reinterpret_cast<Raw<kBytes>*>(zl + k) = z[i];
        if constexpr (kRef) *reinterpret_cast<Raw<kBytes>*>(ql + k) = q[i];
      }
    }
    i64 act;
    RowInputs in;
    if constexpr (G >= 16) {
      in = reader.inputs(g, part, r0, i0, act);
    } else {
      in = row_inputs(g, r0, i0);
      act = (g.action + r0)[i0];
    }
    // the action's slot, where the row has it
    const int moved_from = g.actions & ~(E - 1);
    const int slot_of_act = act < 0 || act >= g.actions ? -1
                            : (int)act >= moved_from   ? (int)act + E - (g.actions & (E - 1))
                                                       : (int)act;
    int count = 0, upto = 0, total = 2 * G + 1;
    if constexpr (kList) {
      count = upto = __popc(bits);  // summed up over the lanes of the row up to this one
      upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xf, 0xf, false);
      upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xf, 0xf, false);
      upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xf, 0xf, false);
      upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xf, 0xf, false);
      total = __builtin_amdgcn_update_dpp(0, upto, 0x15f, 0xf, 0xf, false);  // lane 15's
    }
    const bool listed = kList && __all(total <= 2 * G);
    float top = -INFINITY, top_ref = -INFINITY, s = 0.0f, u = 0.0f, sr = 0.0f, ds = 0.0f;
    float xa = -INFINITY;
    RowTerms x;
    if (listed) {
      uint8_t* list = lists[kList ? row : 0];
      for (int to = upto - count; bits; ++to) {
        const int k = __builtin_ctz(bits);
        bits &= bits - 1;
        list[to] = (uint8_t)(k / E * (G * E) + j * E + k % E);
      }
      wavefront_sync();
      int slot[2];
      float t[2], d[2], p[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool there = j + G * h < total;
        slot[h] = there ? list[j + G * h] : -2;
        t[h] = there ? T::to_float(zl[slot[h]]) : -INFINITY;
        top = fmaxf(top, t[h]);
        if constexpr (kRef) {
          d[h] = there ? T::to_float(ql[slot[h]]) : -INFINITY;
          top_ref = fmaxf(top_ref, d[h]);
        }
      }
      top = group_max<G>(top);
      const Scale scale = scale_for(top);
      Scale scale_ref{};
      if constexpr (kRef) scale_ref = scale_for(group_max<G>(top_ref));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        t[h] = scale(t[h]);
        xa = slot[h] == slot_of_act ? t[h] : xa;
        p[h] = exp2_of(t[h]);
        const bool has = !(p[h] == 0.0f);
        if constexpr (kRef) {
          const float tr = scale_ref(d[h]);
          sr += exp2_of(tr);
          d[h] = has ? t[h] - tr : 0.0f;
          ds = __builtin_fmaf(p[h], d[h], ds);
        }
        t[h] = has ? t[h] : 0.0f;
        s += p[h];
        u = __builtin_fmaf(p[h], t[h], u);
      }
      s = group_sum<G>(s);
      u = group_sum<G>(u);
      xa = group_max<G>(xa);
      if constexpr (kRef) {
        ds = group_sum<G>(ds);
        sr = group_sum<G>(sr);
      }
      x = row_terms<kRef>(g, in, s, u, ds, sr, xa);
      if (g.d_logits) {
        wavefront_sync();
#pragma unroll
        for (int i = 0; i < V; ++i)
          *reinterpret_cast<Raw<kBytes>*>(zl + (i * G + j) * E) = Raw<kBytes>{};
        wavefront_sync();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float f = __builtin_fmaf(x.c, t[h], x.a);
          if constexpr (kRef) f = __builtin_fmaf(x.b, d[h], f);
          f = p[h] == 0.0f ? 0.0f : f;
          f = __builtin_fmaf(p[h], f, -(slot[h] == slot_of_act ? x.pull : 0.0f));
          if (slot[h] >= 0 && x.live) zl[slot[h]] = T::from_float(f);
        }
        wavefront_sync();
      }
    } else {
      wavefront_sync();
      // vector i of the lane, illegal elements at -inf
      const auto logits = [&](int i, float (&z)[E], float (&q)[E]) {
        const Slots zv = *reinterpret_cast<const Slots*>(zl + (i * G + j) * E);
        Slots qv;
        if constexpr (kRef) qv = *reinterpret_cast<const Slots*>(ql + (i * G + j) * E);
        const uint32_t on = bits >> (E * i);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          z[e] = on >> e & 1 ? T::to_float(zv.v[e]) : -INFINITY;
          q[e] = kRef && on >> e & 1 ? T::to_float(qv.v[e]) : -INFINITY;
        }
      };
      float z[E], q[E];
#pragma unroll 1
      for (int i = 0; i < V; ++i) {
        logits(i, z, q);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          top = fmaxf(top, z[e]);
          if constexpr (kRef) top_ref = fmaxf(top_ref, q[e]);
        }
      }
      top = group_max<G>(top);
      const Scale scale = scale_for(top);
      Scale scale_ref{};
      if constexpr (kRef) scale_ref = scale_for(group_max<G>(top_ref));
#pragma unroll 1
      for (int i = 0; i < V; ++i) {
        logits(i, z, q);
        const int k = (i * G + j) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float t = scale(z[e]);
          xa = k + e == slot_of_act ? t : xa;
          const float p = exp2_of(t);
          const bool has = !(p == 0.0f);
          if constexpr (kRef) {
            const float tr = scale_ref(q[e]);
            sr += exp2_of(tr);
            ds = __builtin_fmaf(p, has ? t - tr : 0.0f, ds);
          }
          s += p;
          u = __builtin_fmaf(p, has ? t : 0.0f, u);
        }
      }
      s = group_sum<G>(s);
      u = group_sum<G>(u);
      xa = group_max<G>(xa);
      if constexpr (kRef) {
        ds = group_sum<G>(ds);
        sr = group_sum<G>(sr);
      }
      x = row_terms<kRef>(g, in, s, u, ds, sr, xa);
      if (g.d_logits) {
#pragma unroll 1
        for (int i = 0; i < V; ++i) {
          logits(i, z, q);
          const int k = (i * G + j) * E;
          Slots o;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float t = scale(z[e]);
            const float p = exp2_of(t);
            const bool has = !(p == 0.0f);
            float h = __builtin_fmaf(x.c, t, x.a);
            if constexpr (kRef) h = __builtin_fmaf(x.b, t - scale_ref(q[e]), h);
            h = has ? h : 0.0f;
            // the pull, whatever p is: an action so far below the others that p is 0 has a ratio
            const float f = __builtin_fmaf(p, h, -(k + e == slot_of_act ? x.pull : 0.0f));
            o.v[e] = T::from_float(x.live ? f : 0.0f);
          }
          *reinterpret_cast<Slots*>(zl + k) = o;  // where this lane alone has read
        }
        wavefront_sync();
      }
    }
    if (g.d_logits && ok) {
      S* ob = static_cast<S*>(g.d_logits) + r0 * g.d_stride;
      const uint32_t o_at = i0 * (uint32_t)g.d_stride;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int k = (i * G + j) * E;
        Raw<kBytes> o = *reinterpret_cast<const Raw<kBytes>*>(zl + k);
        if (i + 1 == V && k < g.actions && k > last) {
          // the moved vector again: what it repeats lies in those elements' own slots
          Slots m;
#pragma unroll
          for (int e = 0; e < E; ++e) m.v[e] = zl[last + e < at ? last + e : k + e];
          o = __builtin_bit_cast(Raw<kBytes>, m);
        }
        if (k < g.actions)
          reinterpret_cast<RawAny<kBytes>*>(element(ob, o_at + (uint32_t)(i + 1 < V ? k : last)))->v = o;
      }
    }
    wavefront_sync();  // the next rows' logits come after these reads
#pragma unroll
    for (int h = 0; h < kHeld<G>; ++h) {
      float stat = x.stat[kStats - 1];
#pragma unroll
      for (int k = 0; k < kStats - 1; ++k) stat = j + h * G == k ? x.stat[k] : stat;
      acc[h] += ok ? (double)stat : 0.0;
    }
    if (ok && j == 0) {
      (g.logp + r0)[i0] = x.logp;
      if (g.d_value)
        store_value(const_cast<void*>(at_row(g.d_value, g.value_dtype, r0)), g.value_dtype, i0,
                    x.d_value);
    }
  }
  write_partials<G>(acc, j, g.partials);
}

// Longer rows: a workgroup a row.

// E actions from action c on as a thread holds them, as they were read: from c, or where the row
// ends before c + E its last E, of which those before c are another thread's.  Those and the
// illegal ones are put to -inf.
template <class T, bool kRef>
struct Piece {
  using S = typename T::storage;
  static constexpr int E = 16 / sizeof(S);
  static constexpr int kPer = E / 4;  // elements a word
  Words4 z, q;

  // Element e of w at -inf.
  __device__ static void drop(Words4& w, int e) {
    constexpr uint32_t kOnes = sizeof(S) == 4 ? 0xffffffffu : 0xffffu;
    const int at = sizeof(S) == 4 ? 0 : 16 * (e % kPer);
    w[e / kPer] = (w[e / kPer] & ~(kOnes << at)) | (T::kNone << at);
  }
  // first: where the E elements start, min(c, actions - E).
  __device__ void read(const S* zs, const S* qs, const uint8_t* ls, int c, int first) {
    z = reinterpret_cast<const RawAny<16>*>(element(zs, (uint32_t)first))->v;
    if constexpr (kRef) q = reinterpret_cast<const RawAny<16>*>(element(qs, (uint32_t)first))->v;
    uint32_t gone = (1u << (c - first)) - 1u;  // elements to drop
    if (ls) {
      const Raw<E> on = reinterpret_cast<const RawAny<E>*>(ls + (uint32_t)first)->v;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        uint32_t word;
        if constexpr (E == 4) word = on;
        else word = on[e / 4];
        gone |= (word & (0xffu << (8 * (e % 4))) ? 0u : 1u) << e;
      }
    }
    if (gone == 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!(gone >> e & 1)) continue;
      drop(z, e);
      if constexpr (kRef) drop(q, e);
    }
  }
  __device__ void values(float (&zf)[E], float (&qf)[E]) const {
    unpack<T>(z, zf);
    if constexpr (kRef) unpack<T>(q, qf);
  }
  // The values are unpacked again where they are used next, and not kept instead.
  __device__ void forget() {
    asm volatile("" : "+v"(z));
    if constexpr (kRef) asm volatile("" : "+v"(q));
  }
};

// The largest of each of kN numbers over the workgroup, in every thread.
template <int kWide, int kN>
__device__ inline void workgroup_max(float (&x)[kN], float (*shared)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) x[i] = group_max<64>(x[i]);
  if (threadIdx.x % 64 == 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) shared[threadIdx.x / 64][i] = x[i];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kWide / 64; ++k) {
#pragma unroll
    for (int i = 0; i < kN; ++i) x[i] = fmaxf(x[i], shared[k][i]);
  }
}

template <int kWide>
__device__ inline void workgroup_sums(float (&x)[4], float (*shared)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = group_sum<64>(x[i]);
  if (threadIdx.x % 64 == 0)
    *reinterpret_cast<float4*>(shared[threadIdx.x / 64]) = make_float4(x[0], x[1], x[2], x[3]);
  __syncthreads();
  x[0] = x[1] = x[2] = x[3] = 0.0f;
#pragma unroll
  for (int k = 0; k < kWide / 64; ++k) {
    const float4 w = *reinterpret_cast<const float4*>(shared[k]);
    x[0] += w.x, x[1] += w.y, x[2] += w.z, x[3] += w.w;
  }
}

// A row's terms and its outputs other than the gradient of the logits.  sums: of 2^x, 2^x x,
// 2^x d and 2^x'.
template <class T, bool kRef>
__device__ inline RowTerms finish_row(const LossArgs& g, i64 r, i64 act, const RowInputs& in,
                                      const Scale& scale, const float (&sums)[4], double& acc) {
  using S = typename T::storage;
  const S* zs = static_cast<const S*>(g.logits) + r * g.logits_stride;
  const bool inside = act >= 0 && act < g.actions;
  const bool taken = inside && (!g.legal || g.legal[r * g.legal_stride + act]);
  const float za = T::to_float(zs[inside ? act : 0]);
  const RowTerms x = row_terms<kRef>(g, in, sums[0], sums[1], sums[2], sums[3],
                                     taken ? scale(za) : -INFINITY);
  float stat = x.stat[5];
#pragma unroll
  for (int k = 0; k < kStats - 1; ++k) stat = (int)threadIdx.x == k ? x.stat[k] : stat;
  acc += (double)stat;
  if (threadIdx.x == 0) {
    g.logp[r] = x.logp;
    if (g.d_value)
      store_value(const_cast<void*>(at_row(g.d_value, g.value_dtype, r)), g.value_dtype, 0,
                  x.d_value);
  }
  return x;
}

// The sums over a piece: of 2^x, 2^x x, 2^x d and 2^x'.  kFinite: no x or x' is -inf or so far
// from the others that its difference is (see loss_held_kernel).
template <bool kRef, bool kFinite, int E>
__device__ inline void add_sums(const float (&z)[E], const float (&q)[E], const Scale& scale,
                                const Scale& scale_ref, float (&sums)[4]) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float t = scale(z[e]);
    const float p = exp2_of(t);
    const bool has = kFinite || !(p == 0.0f);
    sums[0] += p;
    sums[1] = __builtin_fmaf(p, has ? t : 0.0f, sums[1]);
    if constexpr (kRef) {
      const float tr = scale_ref(q[e]);
      sums[2] = __builtin_fmaf(p, has ? t - tr : 0.0f, sums[2]);
      sums[3] += exp2_of(tr);
    }
  }
}

// The gradients of a piece's actions.
template <class T, bool kRef, bool kFinite, int E>
__device__ inline void store_gradients(const LossArgs& g, typename T::storage* out, int c, i64 act,
                                       const RowTerms& x, const float (&z)[E],
                                       const float (&q)[E], const Scale& scale,
                                       const Scale& scale_ref, int first) {
  using S = typename T::storage;
  float f[E];
  const float bc = x.b + x.c;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float t = scale(z[e]);
    const float p = exp2_of(t);
    float h;
    if constexpr (kFinite) {
      h = __builtin_fmaf(bc, t, x.a);  // a + b (t - t') + c t
      if constexpr (kRef) h = __builtin_fmaf(-x.b, scale_ref(q[e]), h);
    } else {
      h = __builtin_fmaf(x.c, t, x.a);
      if constexpr (kRef) h = __builtin_fmaf(x.b, t - scale_ref(q[e]), h);
      h = p == 0.0f ? 0.0f : h;
    }
    f[e] = p * h;
  }
  const i64 at = act - first;
  if (at >= 0 && at < E) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] -= at == e ? x.pull : 0.0f;
  }
  if (!x.live) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = 0.0f;
  }
  Vec<S, E> o;
#pragma unroll
  for (int e = 0; e < E; ++e) o.v[e] = T::from_float(f[e]);
  if (c == first) {
    reinterpret_cast<RawAny<16>*>(element(out, (uint32_t)c))->v = __builtin_bit_cast(Words4, o);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (first + e >= c) out[first + e] = o.v[e];
  }
}

// Rows of up to kWide P E actions: the row stays in registers, as it was read, through a pass
// for the largest logit, one for the sums and one for the gradient; so memory sees it once.
// 4,096 x 32,000 bf16 with a KL term: 186 us, 4.2 TB/s, where two passes over memory
// (loss_long_kernel) took 244.  Arithmetic comes next to memory in what bounds it (about 27
// instructions an action with a KL term, three of them exponentials at a quarter of the rate), so a
// row whose logits are all within 2^100 of its largest, as a row without masked entries is, leaves
// out the tests for 0 times infinity: with a mask 248 us.  A last piece that is read moved back (a
// row whose length is no multiple of 16 bytes) counts as masked: 32,001 actions take 226.
// Registers for two workgroups of 512 threads a compute unit, so that one reads while the other
// computes; with 8 pieces and a reference the 128 of them are four too few (20 bytes of scratch).
template <class T, int kWide, int P, bool kRef>
__global__ __launch_bounds__(kWide) __attribute__((amdgpu_waves_per_eu(4))) void loss_held_kernel(
    const LossArgs g) {
  using S = typename T::storage;
  constexpr int E = Piece<T, kRef>::E;
  __shared__ float tops[kWide / 64][4];
  __shared__ __align__(16) float totals[kWide / 64][4];
  double acc = 0.0;
  for (i64 r = blockIdx.x; r < g.n; r += gridDim.x) {
    const S* zs = static_cast<const S*>(g.logits) + r * g.logits_stride;
    const S* qs = static_cast<const S*>(g.ref) + (kRef ? r * g.ref_stride : 0);
    const uint8_t* ls = g.legal ? g.legal + r * g.legal_stride : nullptr;
    // strips of kWide E actions: whole ones, and a last one that may end inside
    constexpr int kStrip = kWide * E;
    const int whole = min(g.actions / kStrip, P - 1);
    const int mine = (int)threadIdx.x * E;
    const int tail_at = whole * kStrip + mine, tail_first = min(tail_at, g.actions - E);
    const bool in_tail = tail_at < g.actions;
    Piece<T, kRef> piece[P - 1], tail;
#pragma unroll
    for (int i = 0; i < P - 1; ++i)
      if (i < whole)
        piece[i].read(zs + i * kStrip, qs + (kRef ? i * kStrip : 0), ls ? ls + i * kStrip : ls, mine,
                      mine);
    if (in_tail) tail.read(zs, qs, ls, tail_at, tail_first);
    const i64 act = g.action[r];
    const RowInputs in = row_inputs(g, r, 0);
    float z[E], q[E];
    // the largest logits, and the smallest with their signs turned
    float ends[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    const auto find_ends = [&](Piece<T, kRef>& held) {
      held.values(z, q);
      float low = INFINITY, low_ref = INFINITY;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        ends[0] = fmaxf(ends[0], z[e]);
        low = fminf(low, z[e]);
        if constexpr (kRef) {
          ends[1] = fmaxf(ends[1], q[e]);
          low_ref = fminf(low_ref, q[e]);
        }
      }
      ends[2] = fmaxf(ends[2], -low);
      if constexpr (kRef) ends[3] = fmaxf(ends[3], -low_ref);
      held.forget();
    };
#pragma unroll
    for (int i = 0; i < P - 1; ++i)
      if (i < whole) find_ends(piece[i]);
    if (in_tail) find_ends(tail);
    workgroup_max<kWide, 4>(ends, tops);
    const bool finite = ends[0] + ends[2] < 0x1p100f && (!kRef || ends[1] + ends[3] < 0x1p100f);
    const Scale scale = scale_for(ends[0]), scale_ref = scale_for(ends[1]);
    float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const auto add = [&](auto is_finite) {
      const auto of = [&](Piece<T, kRef>& held) {
        held.values(z, q);
        add_sums<kRef, decltype(is_finite)::value, E>(z, q, scale, scale_ref, sums);
        held.forget();
      };
#pragma unroll
      for (int i = 0; i < P - 1; ++i)
        if (i < whole) of(piece[i]);
      if (in_tail) of(tail);
    };
    if (finite) add(std::true_type{});
    else add(std::false_type{});
    workgroup_sums<kWide>(sums, totals);
    const RowTerms x = finish_row<T, kRef>(g, r, act, in, scale, sums, acc);
    if (!g.d_logits) continue;
    S* out = static_cast<S*>(g.d_logits) + r * g.d_stride;
    const auto store = [&](auto is_finite) {
      constexpr bool kFinite = decltype(is_finite)::value;
#pragma unroll
      for (int i = 0; i < P - 1; ++i) {
        if (i >= whole) continue;
        piece[i].values(z, q);
        store_gradients<T, kRef, kFinite, E>(g, out + i * kStrip, mine, act - i * kStrip, x, z, q,
                                             scale, scale_ref, mine);
      }
      if (in_tail) {
        tail.values(z, q);
        store_gradients<T, kRef, kFinite, E>(g, out, tail_at, act, x, z, q, scale, scale_ref,
                                             tail_first);
      }
    };
    if (finite) store(std::true_type{});
    else store(std::false_type{});
  }
  // lanes 0 .. kStats - 1 of the workgroup hold its sums
  if (threadIdx.x < kStats) g.partials[(i64)blockIdx.x * kStats + threadIdx.x] = acc;
}

// Rows of any length, in two passes over memory (2,048 x 65,536 bf16 with a KL term: 239 us, 3.4 TB/s
// counted once).  The first keeps each thread's running maximum
// and the sums under it, moved along with the maximum; the second reads the row again for the
// gradient.

// A sum of 2^x y moved by a change of maximum that puts the factor f on 2^x and adds `by` to y;
// s is the sum of 2^x.  What underflows is dropped, whatever it was: logits of the type's lowest
// value make infinities of such a sum until an ordinary one comes.
__device__ inline float moved(float f, float sum, float s, float by) {
  return f == 0.0f ? 0.0f : f * __builtin_fmaf(s, by, sum);
}

template <class T, int kWide, bool kRef>
__global__ __launch_bounds__(kWide) void loss_long_kernel(const LossArgs g) {
  using S = typename T::storage;
  constexpr int E = Piece<T, kRef>::E;
  __shared__ float tops[kWide / 64][2];
  __shared__ __align__(16) float totals[kWide / 64][4];
  double acc = 0.0;
  for (i64 r = blockIdx.x; r < g.n; r += gridDim.x) {
    const S* zs = static_cast<const S*>(g.logits) + r * g.logits_stride;
    const S* qs = static_cast<const S*>(g.ref) + (kRef ? r * g.ref_stride : 0);
    const uint8_t* ls = g.legal ? g.legal + r * g.legal_stride : nullptr;
    const i64 act = g.action[r];
    const RowInputs in = row_inputs(g, r, 0);
    float top = -INFINITY, s = 0.0f, u = 0.0f, top_ref = -INFINITY, sr = 0.0f, ds = 0.0f;
    Piece<T, kRef> piece;
    float z[E], q[E];
    for (int c = threadIdx.x * E; c < g.actions; c += kWide * E) {
      const int first = min(c, g.actions - E);
      piece.read(zs, qs, ls, c, first);
      piece.values(z, q);
      float most = top, most_ref = top_ref;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        most = fmaxf(most, z[e]);
        if constexpr (kRef) most_ref = fmaxf(most_ref, q[e]);
      }
      const Scale now = scale_for(most), now_ref = scale_for(most_ref);
      const float by = now(top), f = exp2_of(by);
      if constexpr (kRef) {
        const float by_ref = now_ref(top_ref);
        ds = moved(f, ds, s, by - by_ref);
        sr *= exp2_of(by_ref);
        top_ref = most_ref;
      }
      u = moved(f, u, s, by);
      s *= f;
      top = most;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float t = now(z[e]);
        const float p = exp2_of(t);
        const bool has = !(p == 0.0f);
        s += p;
        u = __builtin_fmaf(p, has ? t : 0.0f, u);
        if constexpr (kRef) {
          const float tr = now_ref(q[e]);
          sr += exp2_of(tr);
          ds = __builtin_fmaf(p, has ? t - tr : 0.0f, ds);
        }
      }
    }
    // the threads' sums under the row's maximum
    float all[2] = {top, top_ref};
    workgroup_max<kWide, 2>(all, tops);
    const Scale scale = scale_for(all[0]), scale_ref = scale_for(all[1]);
    const float by = scale(top), f = exp2_of(by);
    float sums[4] = {s * f, moved(f, u, s, by), 0.0f, 0.0f};
    if constexpr (kRef) {
      const float by_ref = scale_ref(top_ref);
      sums[2] = moved(f, ds, s, by - by_ref);
      sums[3] = sr * exp2_of(by_ref);
    }
    workgroup_sums<kWide>(sums, totals);
    const RowTerms x = finish_row<T, kRef>(g, r, act, in, scale, sums, acc);
    if (!g.d_logits) continue;
    S* out = static_cast<S*>(g.d_logits) + r * g.d_stride;
    for (int c = threadIdx.x * E; c < g.actions; c += kWide * E) {
      const int first = min(c, g.actions - E);
      piece.read(zs, qs, ls, c, first);
      piece.values(z, q);
      store_gradients<T, kRef, false, E>(g, out, c, act, x, z, q, scale, scale_ref, first);
    }
  }
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
    const float* scale, float* loss_out, float* stats_out) {
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
      stats_out[k] = (float)total;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const double loss = totals[0] + value_coef * totals[1] + kl_coef * totals[2] -
                        entropy_coef * totals[3];
    *loss_out = (float)(loss * (scale ? (double)*scale : 1.0));
  }
}

// x times *factor in place, for a factor other than 1 (whose gradients are right already); x is
// read 16 bytes at a time from its first 16-byte boundary on.
template <class T>
__device__ inline void scale_all(void* data, i64 count, float factor) {
  using S = typename T::storage;
  constexpr int E = 16 / sizeof(S);
  S* x = static_cast<S*>(data);
  const i64 stride = (i64)gridDim.x * kThreads, me = (i64)blockIdx.x * kThreads + threadIdx.x;
  const i64 ahead = min((i64)((16 - (uintptr_t)x % 16) % 16 / sizeof(S)), count);
  const i64 vectors = (count - ahead) / E, done = ahead + vectors * E;
  for (i64 i = me; i < vectors; i += stride) {
    Vec<S, E>* at = reinterpret_cast<Vec<S, E>*>(x + ahead) + i;
    Vec<S, E> v = *at;
#pragma unroll
    for (int e = 0; e < E; ++e) v.v[e] = T::from_float(T::to_float(v.v[e]) * factor);
    *at = v;
  }
  if (me < ahead) x[me] = T::from_float(T::to_float(x[me]) * factor);
  if (me < count - done) x[done + me] = T::from_float(T::to_float(x[done + me]) * factor);
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

// A workgroup for each of `pieces` of work, or as many as a device holds of that many threads, which
// then go round (fewer, only as many as their registers leave resident, took the same time).
template <auto kKernel>
int launch_rows(const LossArgs& g, i64 pieces, int threads, hipStream_t stream) {
  const i64 most = (i64)compute_units() * (2048 / threads);
  const i64 cap = most < kMaxGroups ? most : kMaxGroups;
  const int groups = (int)(pieces < cap ? pieces : cap);
  kKernel<<<groups, threads, 0, stream>>>(g);
  return groups;
}

// Rows of up to kRowsMost actions are addressed by 32 bits within a workgroup's rows: 64 at most, so
// that the last of kStrideMost float32 elements apart begins below 2^32 bytes.
constexpr int kRowsMost = 1024;
constexpr i64 kStrideMost = (i64)1 << 24;

template <class T, bool kRef>
int launch_loss(const LossArgs& g, hipStream_t stream) {
  constexpr int E = 16 / sizeof(typename T::storage);
  const int a = g.actions;
#define CUGO_LOSS_ROWS(G, V, E)                                             \
  launch_rows<loss_rows_kernel<T, G, V, E, kRef>>(                          \
      g, (g.n + kThreads / G - 1) / (kThreads / G), kThreads, stream)
#define CUGO_LOSS_HELD(THREADS, P) \
  launch_rows<loss_held_kernel<T, THREADS, P, kRef>>(g, g.n, THREADS, stream)
  // Lanes, vectors and threads by what a row needs; us of 2^27 bf16 logits with a KL term on both
  // sides of the lines: 256 actions 230, 257 348 (16 lanes against 32; 541 on 64 lanes), 512 225, 513
  // 356, 1,024 230 and 1,025 316 (a workgroup of 64 threads: 199 and 562 of 256), 2,048 170, 4,096
  // 178, 8,192 167 and 8,193 276, 32,768 184 and 32,769 265.  Rows of 768 take 245 on 64 lanes and 253
  // as a workgroup of 64 threads, with a mask 249 and 353.
  // Just above a line much of what a row's lanes hold is empty, and is gone through all the same:
  // 257 to 264 actions 354 to 346, 320 287, 384 240; 1,032 255, 1,536 182, 2,048 170; 8,200 221,
  // 12,288 190.  An odd length costs nothing in itself, but rows of over 1,024 actions pay for the
  // last piece moved back (see loss_held_kernel): 1,025 323, 8,193 285.
  // Few actions, us of 2^21 rows (2^26 logits, where those are fewer) against 16 lanes: 4 actions 89
  // and 261, 16 89 and 251, 32 143 and 272, 48 125 and 228; 64 on 8 lanes 142 and 174 (133 on 4,
  // which float32 rows take 224 for, and 172 on 8, 182 on 16), with 10 of them legal 147 and 141.
  // Rows of 96 take 372 a 2^27 logits on 16 lanes and 247 on 8, but with 10 legal 227 and 255.
  if (a < 4) return CUGO_LOSS_ROWS(4, 1, 1);
  if (a <= 16) return CUGO_LOSS_ROWS(4, 1, 4);
  if (a <= 32) return CUGO_LOSS_ROWS(4, 2, 4);
  if (a <= 48) return CUGO_LOSS_ROWS(4, 3, 4);
  if (a <= 64) return CUGO_LOSS_ROWS(8, 2, 4);
  if (a <= 128) return CUGO_LOSS_ROWS(16, 2, 4);
  if (a <= 192) return CUGO_LOSS_ROWS(16, 3, 4);
  if (a <= 256) return CUGO_LOSS_ROWS(16, 4, 4);
  if (a <= 384) return CUGO_LOSS_ROWS(32, 3, 4);
  if (a <= 512) return CUGO_LOSS_ROWS(32, 4, 4);
  if (a <= 768) return CUGO_LOSS_ROWS(64, 3, 4);
  if (a <= kRowsMost) return CUGO_LOSS_ROWS(64, 4, 4);
  if (a <= 64 * 4 * E) return CUGO_LOSS_HELD(64, 4);
  if (a <= 128 * 4 * E) return CUGO_LOSS_HELD(128, 4);
  if (a <= 256 * 4 * E) return CUGO_LOSS_HELD(256, 4);
  if (a <= 512 * 4 * E) return CUGO_LOSS_HELD(512, 4);
  if (a <= 512 * 8 * E) return CUGO_LOSS_HELD(512, 8);
#undef CUGO_LOSS_ROWS
#undef CUGO_LOSS_HELD
  return launch_rows<loss_long_kernel<T, 1024, kRef>>(g, g.n, 1024, stream);
}

}  // namespace loss
}  // namespace learner
}  // namespace cugo_amd

using namespace cugo_amd::learner;
using namespace cugo_amd::learner::loss;

extern "C" {

int cugo_policy_loss(const CugoPolicyLoss* p, hipStream_t stream) {
  if (!p || p->n < 0 || p->actions < 1 || p->actions > (1 << 30) || !p->loss || !p->stats || !p->partials)
    return -1;
  if (!dtype_known(p->logits_dtype) || (p->value && !dtype_known(p->value_dtype))) return -2;
  if (p->n > 0 && (!p->logits || !p->action || !p->old_logp || !p->advantage || !p->logp))
    return -1;
  if ((p->value != nullptr) != (p->returns != nullptr) || (p->d_value && !p->value)) return -1;
  // (one row has no next one: its stride multiplies 0)
  if (p->actions <= kRowsMost && p->n > 1 &&
      (p->logits_stride >= kStrideMost || p->ref_stride >= kStrideMost ||
       p->legal_stride >= kStrideMost || p->d_logits_stride >= kStrideMost))
    return -4;
  if (p->logits_stride < 0 || p->ref_stride < 0 || p->legal_stride < 0 ||
      (p->d_logits && p->n > 1 && p->d_logits_stride < p->actions))
    return -4;
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
                                                   p->loss, p->stats);
  return (int)hipGetLastError();
}

int cugo_scale_gradients(int a_dtype, void* a, int64_t a_count, int b_dtype, void* b,
                         int64_t b_count, const float* factor, hipStream_t stream) {
  if (a_count < 0 || b_count < 0 || (a_count > 0 && !a) || (b_count > 0 && !b) || !factor)
    return -1;
  if (!dtype_known(a_dtype) || !dtype_known(b_dtype)) return -2;
  const int64_t most = a_count > b_count ? a_count : b_count;
  if (most == 0) return 0;
  // Two workgroups a compute unit: a factor of 1, which a backward pass from the loss itself has,
  // costs the launch of the grid alone (1.9 us, 3.9 us of one that fills the device).
  const int64_t needed = (most + 4 * kThreads - 1) / (4 * kThreads);
  const int64_t cap = 2 * (int64_t)compute_units();
  const int groups = (int)(needed < cap ? needed : cap);
  scale_kernel<<<groups, kThreads, 0, stream>>>(a_dtype, a, a_count, b_dtype, b, b_count, factor);
  return (int)hipGetLastError();
}

}  // extern "C"
