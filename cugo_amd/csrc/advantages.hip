// Generalised advantage estimation over a horizon of two-player games.
//
// With s_t = 1 where player 0 moves and -1 where player 1 does, everything is seen from
// player 0's side:
//   d_t = reward_t + [not done_t] gamma s_(t+1) V_(t+1) - s_t V_t
//   a_t = d_t + c_t a_(t+1),  c_t = gamma lam, or 0 at a done step
// and a mover's advantage is s_t a_t.  a_t is an affine map of a_(t+1), and maps compose:
// (D, C) after (D', C') is (D + C D', C C').  So the steps are split: a lane takes 4 or 8
// consecutive steps of one game in registers and composes their maps, lanes and wavefronts
// compose theirs (a suffix scan in the wavefront, then over the wavefronts in LDS), and each
// lane runs its own steps again from the value that follows them.  The data is read once, or twice
// where the steps are split over workgroups.
//
// What bounds it is memory, 16 to 18 bytes a step of a game and 8 to 10 more where it is read twice
// (128 steps of 65,536 games in 29 us, 5.2 TB/s), and below about a million steps the two or three
// rounds of latency of a launch (5 us for 64 x 300).  A wavefront's 64 lanes are
// `columns` games times 64 / columns runs of steps, the fewest columns (a power of two) that
// hold the games up to 64, so that few games still fill wavefronts; where the workgroups of
// one run over the steps would leave compute units idle, the steps are also split over
// workgroups, in two launches: the first composes each chunk's map (the first chunk's with the
// others', though no chunk lies before it), the second starts each chunk from the maps of those
// behind it.
#include "learner.h"

namespace cugo_amd {
namespace learner {
namespace gae {

constexpr int kMostWaves = 16; // wavefronts a workgroup, at most

struct GaeArgs {
  const float* reward;
  const void* value;
  const uint8_t* done;
  const uint8_t* player;
  const void* bootstrap;
  const uint8_t* last_player;
  i64 steps, batch;
  i64 chunk;    // steps a workgroup takes: a multiple of the steps of one pass over its lanes
  int chunks;
  int columns;
  float gamma, decay;
  float* advantage;
  float* returns;
  float2* maps;  // [chunks, batch]: the chunks' maps (chunks > 1)
};

// m applied to the value a that follows it, which a factor of 0 (a done step, or lam = 0) does not
// read: a NaN of the next game stays there.
__device__ inline float apply(float2 m, float a) {
  return m.y == 0.0f ? m.x : __builtin_fmaf(m.y, a, m.x);
}
// The product of two factors in [0, 1]: 0 only where one of them is, and not where it underflows,
// so that a NaN or an infinity far behind in the same game shows in every step before it.
__device__ inline float product(float a, float b) {
  return a == 0.0f || b == 0.0f ? 0.0f : fmaxf(a * b, 0x1p-149f);
}
__device__ inline float2 after(float2 m, float2 later) {
  return make_float2(apply(m, later.x), product(m.y, later.y));
}

// kSteps: the steps a lane holds.
template <class T, int kSteps, bool kMapsOnly>
__global__ __launch_bounds__(64 * kMostWaves) void gae_kernel(const GaeArgs g) {
  using S = typename T::storage;
  __shared__ float2 wave_map[kMostWaves][64];
  __shared__ float behind[2][64];  // a of the step behind a pass, for each column, in turn
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int column = lane & (g.columns - 1), run = lane / g.columns;
  const int runs = 64 / g.columns, waves = (int)blockDim.x >> 6;
  const i64 game = (i64)blockIdx.x * g.columns + column;
  const bool ok = game < g.batch;
  const i64 b = ok ? game : g.batch - 1;
  const int chunk = blockIdx.y;
  const i64 first = (i64)chunk * g.chunk;
  const i64 end = min(first + g.chunk, g.steps);
  const S* value = static_cast<const S*>(g.value);
  const i64 pass = (i64)waves * runs * kSteps;
  float carry = 0.0f;
  if (!kMapsOnly && chunk + 1 < g.chunks) {
    // The maps of the chunks behind this one: each wavefront composes a run of them (its loads
    // do not wait for one another), and every lane applies the runs.
    const int behind_it = g.chunks - 1 - chunk;
    const int each = (behind_it + waves - 1) / waves;
    const int from = chunk + 1 + wave * each, to = min(from + each, g.chunks);
    float2 m = make_float2(0.0f, 1.0f);
#pragma unroll 4
    for (int k = from; k < to; ++k) m = after(m, g.maps[(i64)k * g.batch + b]);
    if (run == 0) wave_map[wave][column] = m;
    __syncthreads();
    for (int k = waves - 1; k >= 0; --k) carry = apply(wave_map[k][column], carry);
    __syncthreads();
  }
  float2 total = make_float2(0.0f, 1.0f);  // kMapsOnly: the map of the passes so far
  int turn = 0;
  // passes from the chunk's last steps back
  for (i64 at = first + (end - first - 1) / pass * pass; at >= first; at -= pass, turn ^= 1) {
    const i64 t0 = at + ((i64)wave * runs + run) * kSteps;
    float d[kSteps], v[kSteps + 1], sign[kSteps + 1];
    bool over[kSteps];
#pragma unroll
    for (int i = 0; i <= kSteps; ++i) {
      // steps behind the horizon's end: the bootstrap's place, read by the last step alone
      const i64 t = min(t0 + i, g.steps);
      const bool boot = t == g.steps;
      const i64 at_v = boot ? b : t * g.batch + b;
      const S* from = boot ? static_cast<const S*>(g.bootstrap) : value;
      const uint8_t* who = boot ? g.last_player : g.player;
      v[i] = T::to_float(from[at_v]);
      sign[i] = who && who[at_v] ? -1.0f : 1.0f;
      if (i < kSteps) {
        const i64 at_r = min(t, g.steps - 1) * g.batch + b;
        d[i] = g.reward[at_r];
        over[i] = g.done[at_r] != 0;
      }
    }
    float2 map = make_float2(0.0f, 1.0f);
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      if (t0 + i < end) {
        const float next = over[i] ? 0.0f : g.gamma * (sign[i + 1] * v[i + 1]);
        d[i] = d[i] + next - sign[i] * v[i];
        over[i] = over[i] || g.decay == 0.0f;  // from here on: nothing is read from behind
        map.x = over[i] ? d[i] : __builtin_fmaf(g.decay, map.x, d[i]);
        map.y = over[i] ? 0.0f : product(g.decay, map.y);
      }
    }
    // each lane's map and those of the later runs of its column, then of the later runs alone
    for (int off = g.columns; off < 64; off <<= 1) {
      const float2 next = make_float2(__shfl_down(map.x, off), __shfl_down(map.y, off));
      if (lane + off < 64) map = after(map, next);
    }
    float2 later = make_float2(__shfl_down(map.x, g.columns), __shfl_down(map.y, g.columns));
    if (run == runs - 1) later = make_float2(0.0f, 1.0f);
    if (run == 0) wave_map[wave][column] = map;
    __syncthreads();
    if (kMapsOnly) {
      if (wave == 0 && run == 0) {
        float2 all = wave_map[0][column];
        for (int k = 1; k < waves; ++k) all = after(all, wave_map[k][column]);
        total = after(all, total);
      }
      __syncthreads();
      continue;
    }
    float a = at + pass >= end ? carry : behind[turn ^ 1][column];
    for (int k = waves - 1; k > wave; --k) a = apply(wave_map[k][column], a);
    if (wave == 0 && run == 0) behind[turn][column] = apply(map, a);
    a = apply(later, a);
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      if (t0 + i < end) {
        a = over[i] ? d[i] : __builtin_fmaf(g.decay, a, d[i]);
        if (ok) {
          const i64 to = (t0 + i) * g.batch + b;
          const float mine = sign[i] * a;
          g.advantage[to] = mine;
          g.returns[to] = mine + v[i];
        }
      }
    }
    __syncthreads();  // wave_map and behind[turn ^ 1] are free again
  }
  if (kMapsOnly && wave == 0 && run == 0 && ok) g.maps[(i64)chunk * g.batch + b] = total;
}

// How a call is laid out: the columns of a wavefront, the steps a lane holds and the wavefronts of
// a workgroup, and the chunks that the steps are split into.
// One or two passes are not split: the second pass costs less than a second launch and a second
// reading.  Their lanes hold 4 steps, in as many wavefronts as the steps need (16 at most).  More
// passes are split into as many chunks as give the launch two workgroups of 8 wavefronts a compute
// unit; lanes then hold 8 steps, or 4 where games do not fill a wavefront's lanes.  us, 4 steps and up
// to 16 wavefronts / 8 steps and 8 wavefronts: unsplit 128 x 32,768 16.3 / 18.0, 128 x 512 7.7 / 8.4,
// 16 x 65,536 5.9 / 10.7; split 20,001 x 45 17.9 / 15.2, 1,024 x 4,096 28.5 / 29.7; 4 steps and 8
// wavefronts / 8 and 8: 70,000 x 1 11.1 / 19.2, 1,000 x 10 8.7 / 10.0, 20,001 x 45 17.0 / 15.2.
// Unsplit / one / two / four workgroups a compute unit: 128 x 8,192 (two passes) 9.7 / 11.3 / 11.4 /
// 11.3, 256 x 1,024 (four) 15.0 / 10.1 / 10.1 / 10.1, 1,024 x 4,096 80 / 43.5 / 30.3 / 31.2.
struct GaeLayout {
  int columns, steps, waves, chunks;
  i64 groups, chunk;
};

inline GaeLayout gae_layout(i64 steps, i64 batch) {
  GaeLayout l;
  l.columns = 64;
  while (l.columns > 1 && l.columns / 2 >= batch) l.columns /= 2;
  l.groups = (batch + l.columns - 1) / l.columns;
  const int runs = 64 / l.columns;
  const i64 lanes = (steps + runs * 4 - 1) / (runs * 4);  // wavefronts that hold all of the steps
  i64 chunks = 2 * (i64)compute_units() / l.groups;
  if (lanes <= 2 * kMostWaves || chunks < 2) {
    l.steps = 4;
    l.waves = (int)(lanes < kMostWaves ? lanes : kMostWaves);
    l.chunks = 1;
    l.chunk = steps;
    return l;
  }
  l.steps = l.columns == 64 ? 8 : 4;
  l.waves = 8;
  const i64 pass = (i64)l.waves * runs * l.steps;
  const i64 passes = (steps + pass - 1) / pass;
  if (chunks > passes) chunks = passes;
  const i64 each = (passes + chunks - 1) / chunks;
  l.chunk = each * pass;
  l.chunks = (int)((passes + each - 1) / each);
  return l;
}

template <class T, int kSteps>
int launch_gae(const GaeArgs& g, const GaeLayout& l, hipStream_t stream) {
  const dim3 grid((unsigned)l.groups, (unsigned)l.chunks);
  if (l.chunks > 1) {
    gae_kernel<T, kSteps, true><<<grid, 64 * l.waves, 0, stream>>>(g);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
  }
  gae_kernel<T, kSteps, false><<<grid, 64 * l.waves, 0, stream>>>(g);
  return (int)hipGetLastError();
}

template <class T>
int launch_gae(const GaeArgs& g, const GaeLayout& l, hipStream_t stream) {
  return l.steps == 4 ? launch_gae<T, 4>(g, l, stream) : launch_gae<T, 8>(g, l, stream);
}

}  // namespace gae
}  // namespace learner
}  // namespace cugo_amd

using namespace cugo_amd::learner;
using namespace cugo_amd::learner::gae;

extern "C" {

int64_t cugo_advantages_workspace(int64_t steps, int64_t batch) {
  if (steps < 1 || batch < 1) return 0;
  const GaeLayout l = gae_layout(steps, batch);
  return l.chunks > 1 ? (int64_t)sizeof(float2) * l.chunks * batch : 0;
}

int cugo_advantages(int value_dtype, const float* reward, const void* value,
                    const uint8_t* done, const uint8_t* player, const void* bootstrap,
                    const uint8_t* last_player, int64_t steps, int64_t batch, double gamma,
                    double lam, float* advantage, float* returns, void* workspace,
                    int64_t workspace_bytes, hipStream_t stream) {
  if (steps < 0 || batch < 0 || batch > ((int64_t)1 << 36)) return -1;
  if (!dtype_known(value_dtype)) return -2;
  if (steps == 0 || batch == 0) return 0;
  if (!reward || !value || !done || !bootstrap || !advantage || !returns ||
      (player != nullptr) != (last_player != nullptr))
    return -1;
  const GaeLayout l = gae_layout(steps, batch);
  if (l.chunks > 1 &&
      (!workspace || workspace_bytes < (int64_t)sizeof(float2) * l.chunks * batch))
    return -3;
  GaeArgs g{};
  g.reward = reward, g.value = value, g.done = done, g.player = player;
  g.bootstrap = bootstrap, g.last_player = last_player;
  g.steps = steps, g.batch = batch, g.chunk = l.chunk, g.chunks = l.chunks;
  g.columns = l.columns;
  g.gamma = (float)gamma, g.decay = (float)(gamma * lam);
  g.advantage = advantage, g.returns = returns, g.maps = static_cast<float2*>(workspace);
  if (value_dtype == CUGO_DTYPE_F32) return launch_gae<F32>(g, l, stream);
  if (value_dtype == CUGO_DTYPE_F16) return launch_gae<F16>(g, l, stream);
  return launch_gae<BF16>(g, l, stream);
}

}  // extern "C"
