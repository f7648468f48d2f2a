// Routing of rows to experts: top-k softmax routing with its gradient, grouping of the places by expert (a stable
// counting sort), and the weighted sum that brings the experts' rows back together, with its gradient.
//
//   route    p_t = softmax(z_t); the k largest z of a row (ties: the lowest expert; -inf never): experts, and
//            w_tj = exp(z_t,ej - m) / sum over the chosen (or over all experts: `normalize` off); load_e = mean_t p_te
//   group    offsets[e] = places with an expert < e; order[] = the places sorted by (expert, place); position[] its inverse
//   combine  out_t = residual_t + sum_j w_tj y[position_tj]
//
// All of it is bound by memory at large sizes and by launches and dependent loads at small ones: the arithmetic of a
// row is E exponentials and k selections.  Statistics, weights and sums are fp32; nothing is added with floating-point
// atomics, so results do not depend on the schedule.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "numeric.hpp"

using namespace dimo;

namespace {

constexpr int ROUTE_THREADS = 256;
constexpr int ROUTE_MAX_E = DIMO_MAX_EXPERTS;
// Workgroups of a routing launch that also sums the load (a row of partial sums each): 131072 rows of 128 take 38 us in 512
// of them, 32 in 1024, 29 in 2048, the sums of the rows 4.0, 4.3, 7.3.
constexpr int ROUTE_MAX_BLOCKS = 1024;

// ---- routing ---------------------------------------------------------------------------------------------------
// A row lies in L neighbouring lanes (a power of two up to 64), V consecutive logits in each: sixteen-byte loads, and few
// exchanges -- a selection round is V comparisons in a lane and log2(L) exchanges of (value, index) between lanes, most of
// them DPP moves.  V = 16 from 9 experts on: 131072 rows of 128, k = 8, took 215 us with V = 4 (five exchanges a round,
// through LDS) and 54 us this way (bf16; less since: `Keys`).
struct RouteArgs {
  int T, E, k, normalize, wide;
  const void *logits;
  int64_t ld;
  const uint8_t *row_mask;
  float *weights;
  int32_t *experts;
  float *partial;  // [gridDim.x, E] sums of p over the workgroup's rows, or null
  float load_scale;
};

// The value of a lane of the other half of 2 M lanes whose halves are each uniform (the M-th step of a reduction).
template <int M>
__device__ __forceinline__ int from_other_half(int v) {
  if constexpr (M == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false);   // quad_perm [1, 0, 3, 2]
  else if constexpr (M == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false);   // quad_perm [2, 3, 0, 1]
  else if constexpr (M == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false);  // row_half_mirror
  else if constexpr (M == 8) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, false);  // row_mirror
  else return __shfl_xor(v, M);
}
template <int M>
__device__ __forceinline__ float from_other_half(float v) {
  return __int_as_float(from_other_half<M>(__float_as_int(v)));
}
template <int L, int M = 1, class F>
__device__ __forceinline__ void halving_steps(F &&f) {
  if constexpr (M < L) {
    f(std::integral_constant<int, M>{});
    halving_steps<L, 2 * M>(f);
  }
}
// exp on the hardware's exponential: off by 2^-23 and the argument's rounding, |v| 2^-24 (logits within 30 of the row's
// largest: 2e-6 of a probability of 1e-13; what is small is off most).  expf's sixteen instructions times V values were a
// third of the kernel.
__device__ __forceinline__ float exp_fast(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896340736f); }

template <int L>
__device__ __forceinline__ float row_sum(float v) {
  halving_steps<L>([&](auto m) { v += from_other_half<decltype(m)::value>(v); });
  return v;
}
template <int L>
__device__ __forceinline__ float row_max(float v) {
  halving_steps<L>([&](auto m) { v = fmaxf(v, from_other_half<decltype(m)::value>(v)); });
  return v;
}

// this lane's V logits (first .. first + V - 1 of the row at `src`), -inf where there are none
template <class T, int V>
__device__ __forceinline__ void load_row(const typename T::store *src, int first, int E, bool live, bool wide, float (&z)[V]) {
  if (wide) {
    constexpr int N = Vec16<T>::N, G = V < N ? 1 : V / N;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float q[N];
      const bool in = live && first + g * N < E;
      load_vec<T, N>(src + (in ? first + g * N : 0), q);
#pragma unroll
      for (int e = 0; e < N && g * N + e < V; ++e) z[g * N + e] = in ? q[e] : -INFINITY;
    }
  } else {
#pragma unroll
    for (int c = 0; c < V; ++c) z[c] = (live && first + c < E) ? T::load(src[first + c]) : -INFINITY;
  }
}

// A lane's V logits that are not chosen yet; next() finds the row's largest of them (ties: the lowest index) and takes it out;
// at = -1: a row without any (-inf and NaN never are).
// fp32: comparisons of (value, index).
template <class T, int V>
struct Candidates {
  float z[V];
  int first;
  uint32_t left = (1u << V) - 1u;  // (V <= 16)
  __device__ __forceinline__ Candidates(const float (&v)[V], int first_) : first(first_) {
#pragma unroll
    for (int c = 0; c < V; ++c) z[c] = v[c];
  }
  template <int L>
  __device__ __forceinline__ float next(int &at) {
    float best = -INFINITY;
    at = ROUTE_MAX_E;
#pragma unroll
    for (int c = 0; c < V; ++c)  // (ascending index: the first of equals stays)
      if (((left >> c) & 1u) && z[c] > best) best = z[c], at = first + c;
    halving_steps<L>([&](auto m) {
      const float ob = from_other_half<decltype(m)::value>(best);
      const int oa = from_other_half<decltype(m)::value>(at);
      if (ob > best || (ob == best && oa < at)) best = ob, at = oa;
    });
    const int own = at - first;
    if (own >= 0 && own < V) left &= ~(1u << own);
    if (!(best > -INFINITY)) at = -1;
    return best;
  }
};
// 16 bits: value and index fit one word that sorts like the pair -- the value's bits in ascending order, behind them the
// index, the lowest largest; 0 = none -- so a choice is a maximum (two values per instruction) and an equality.  131072 rows of
// 128 in bf16, k = 8: 54 us by comparisons, 38 this way.
template <class T, int V>
struct Keys {
  uint32_t key[V];
  __device__ __forceinline__ Keys(const float (&v)[V], int first) {
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const uint32_t bits = (uint32_t)T::save(v[c] + 0.f) << 16;  // (-0 counts as 0)
      const uint32_t up = bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
      key[c] = v[c] > -INFINITY ? (up & 0xffff0000u) | (0xffffu - (uint32_t)(first + c)) : 0u;
    }
  }
  template <int L>
  __device__ __forceinline__ float next(int &at) {
    uint32_t best = 0u;
#pragma unroll
    for (int c = 0; c < V; ++c) best = max(best, key[c]);
    halving_steps<L>([&](auto m) { best = max(best, (uint32_t)from_other_half<decltype(m)::value>((int)best)); });
#pragma unroll
    for (int c = 0; c < V; ++c) key[c] = key[c] == best ? 0u : key[c];
    at = best ? (int)(0xffffu - (best & 0xffffu)) : -1;
    return T::load((typename T::store)((best >> 16) ^ (best >> 31 ? 0x8000u : 0xffffu)));
  }
};
template <int V>
struct Candidates<BF16, V> : Keys<BF16, V> {
  using Keys<BF16, V>::Keys;
};
template <int V>
struct Candidates<F16, V> : Keys<F16, V> {
  using Keys<F16, V>::Keys;
};

template <class T, int L, int V>
__global__ __launch_bounds__(ROUTE_THREADS) void route_forward_kernel(RouteArgs a) {
  constexpr int ROWS = ROUTE_THREADS / L, KEPT = L < 8 ? 8 / L : 1;
  const int lane = threadIdx.x % L, sub = threadIdx.x / L, first = lane * V;
  float mine[V];  // sums of p over this lane's rows
#pragma unroll
  for (int c = 0; c < V; ++c) mine[c] = 0.f;
  const int rounds = (a.T + ROWS * (int)gridDim.x - 1) / (ROWS * (int)gridDim.x);
  for (int it = 0; it < rounds; ++it) {  // (the same number of rounds for every lane: the exchanges need the whole wave)
    const int64_t row = ((int64_t)it * gridDim.x + blockIdx.x) * ROWS + sub;
    const bool in = row < a.T;
    const bool live = in && (!a.row_mask || a.row_mask[in ? row : 0] != 0);
    float z[V];
    load_row<T, V>(static_cast<const typename T::store *>(a.logits) + (in ? row : 0) * a.ld, first, a.E, live, a.wide, z);
    bool nan = false;
#pragma unroll
    for (int c = 0; c < V; ++c) nan |= z[c] != z[c];
    // a NaN is never chosen; the row's weights and probabilities are NaN by the formula
    const float poison = row_max<L>(nan ? 1.f : 0.f) > 0.f ? NAN : 0.f;
    Candidates<T, V> candidates(z, first);
    float top = 0.f;      // the row's largest logit
    float chosen = 0.f;   // sum of exp over the chosen
    float kept[KEPT] = {};  // the lane of place j keeps its share until the sum is known (place j: kept[j / L]) ...
    int count = 0;
    for (int j = 0; j < a.k; ++j) {
      int at;
      const float best = candidates.template next<L>(at);
      const bool found = at >= 0;
      if (j == 0) top = found ? best : 0.f;
      const float share = found ? exp_fast(best - top) : 0.f;
      chosen += share;
      count += found;
      if (in && j % L == lane) {
#pragma unroll
        for (int i = 0; i < KEPT; ++i) kept[i] = j / L == i ? share : kept[i];
        if (j >= KEPT * L) a.weights[row * a.k + j] = share;  // ... or writes it and reads it again
        a.experts[row * a.k + j] = at;
      }
    }
    float all = 0.f, p[V];
#pragma unroll
    for (int c = 0; c < V; ++c) p[c] = exp_fast(z[c] - top), all += z[c] == z[c] ? p[c] : 0.f;
    all = row_sum<L>(all);
    const float inv_all = (all > 0.f ? 1.f / all : 0.f) + poison;
    const float inv = a.normalize ? (count ? 1.f / chosen : 0.f) + poison : inv_all;
    if (in) {
#pragma unroll
      for (int i = 0; i < KEPT; ++i)
        if (i * L + lane < a.k) a.weights[row * a.k + i * L + lane] = i * L + lane < count ? kept[i] * inv : 0.f;
      for (int j = KEPT * L + lane; j < a.k; j += L) a.weights[row * a.k + j] = j < count ? a.weights[row * a.k + j] * inv : 0.f;
    }
    if (live)
#pragma unroll
      for (int c = 0; c < V; ++c) mine[c] += p[c] * inv_all;
  }
  if (!a.partial) return;
  // the workgroup's rows one after the other, in a fixed order
  __shared__ float sums[ROUTE_THREADS * V];
#pragma unroll
  for (int c = 0; c < V; ++c) sums[sub * (L * V) + first + c] = mine[c];
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += ROUTE_THREADS) {
    float s = 0.f;
    for (int r = 0; r < ROWS; ++r) s += sums[r * (L * V) + e];
    a.partial[(size_t)blockIdx.x * a.E + e] = s * a.load_scale;
  }
}

// load[e] = sum over the workgroups' partial sums: sixteen threads per expert, theirs summed in a fixed order
__global__ __launch_bounds__(256) void route_load_kernel(int E, int blocks, const float *__restrict__ partial,
                                                         float *__restrict__ load) {
  __shared__ float s[16][17];
  const int e = blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
  float v = 0.f;
  if (e < E)
#pragma unroll 8
    for (int b = part; b < blocks; b += 16) v += partial[(size_t)b * E + e];
  s[part][threadIdx.x & 15] = v;
  __syncthreads();
  if (part == 0 && e < E) {
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) sum += s[q][threadIdx.x];
    load[e] = sum;
  }
}

// Backward: the chosen experts' share arrives in LDS (one row of E per row of logits), the rest is per element.
//   normalize:  g_ej = w_j (gw_j - sum_i w_i gw_i)         otherwise  p_e (g_e - sum p g), g_ej = gw_j
//   load:       + p_e (gl_e - sum p gl) / T
struct RouteBwdArgs {
  int T, E, k, normalize, wide;
  const void *logits;
  int64_t ld;
  const uint8_t *row_mask;
  const float *weights;
  const int32_t *experts;
  const float *g_weights, *g_load;
  void *g_logits;
  float load_scale;
  int64_t first;  // first workgroup of this launch
};

template <class T, int L, int V>
__global__ __launch_bounds__(ROUTE_THREADS) void route_backward_kernel(RouteBwdArgs a) {
  constexpr int ROWS = ROUTE_THREADS / L, PAD = 1;  // (rows of L V + 1 words: a lane's V words then lie on other banks)
  __shared__ float sparse[ROWS * (L * V + PAD)];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L, first = lane * V;
  const int64_t row = (a.first + blockIdx.x) * ROWS + sub;
  const bool in = row < a.T;
  const bool live = in && (!a.row_mask || a.row_mask[in ? row : 0] != 0);
  float *g_row = sparse + sub * (L * V + PAD);
#pragma unroll
  for (int c = 0; c < V; ++c) g_row[first + c] = 0.f;
  __syncthreads();
  float inner = 0.f;
  if (live && a.g_weights && a.normalize)
    for (int j = lane; j < a.k; j += L)
      if (a.experts[row * a.k + j] >= 0) inner += a.weights[row * a.k + j] * a.g_weights[row * a.k + j];
  inner = row_sum<L>(inner);
  if (live && a.g_weights)
    for (int j = lane; j < a.k; j += L) {
      const int e = a.experts[row * a.k + j];
      if (e < 0 || e >= a.E) continue;
      const float g = a.g_weights[row * a.k + j];
      g_row[e] = a.normalize ? a.weights[row * a.k + j] * (g - inner) : g;
    }
  __syncthreads();
  float out[V];
#pragma unroll
  for (int c = 0; c < V; ++c) out[c] = g_row[first + c];
  if (a.g_load || !a.normalize) {
    float z[V], p[V], g[V];
    load_row<T, V>(static_cast<const typename T::store *>(a.logits) + (in ? row : 0) * a.ld, first, a.E, live, a.wide, z);
    float m = -INFINITY, all = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) m = fmaxf(m, z[c]);
    m = row_max<L>(m);
    if (!(m > -INFINITY)) m = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) p[c] = exp_fast(z[c] - m), all += p[c];
    all = row_sum<L>(all);
    const float inv = all > 0.f ? 1.f / all : (all == 0.f ? 0.f : all);  // (NaN stays NaN)
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < V; ++c) {
      const int e = first + c;
      p[c] *= inv;
      g[c] = (a.g_load && e < a.E) ? a.g_load[e] * a.load_scale : 0.f;
      if (!a.normalize) g[c] += out[c], out[c] = 0.f;
      dot += e < a.E ? p[c] * g[c] : 0.f;
    }
    dot = row_sum<L>(dot);
#pragma unroll
    for (int c = 0; c < V; ++c) out[c] += p[c] * (g[c] - dot);
  }
  if (!in) return;
#pragma unroll
  for (int c = 0; c < V; ++c) out[c] = live ? out[c] : 0.f;
  typename T::store *dst = static_cast<typename T::store *>(a.g_logits) + row * a.E;
  constexpr int N = Vec16<T>::N;
  if (V >= N && a.wide) {
#pragma unroll
    for (int g = 0; g < V / N; ++g) {
      float q[N];
#pragma unroll
      for (int e = 0; e < N; ++e) q[e] = out[(g * N + e) % V];
      if (first + g * N < a.E) store_vec<T, N>(dst + first + g * N, q);
    }
  } else {
#pragma unroll
    for (int c = 0; c < V; ++c)
      if (first + c < a.E) dst[first + c] = T::save(out[c]);
  }
}

// lanes per row and values per lane for E experts
inline int route_values(int E) { return E <= 4 ? 4 : E <= 8 ? 8 : 16; }
inline int route_lanes(int E) {
  int L = 1;
  while (L * route_values(E) < E) L *= 2;
  return L;
}
inline int route_blocks(int T, int E) {
  const int rows = ROUTE_THREADS / route_lanes(E);
  return (T + rows - 1) / rows;
}
// rows that sixteen-byte loads can take: whole, and on their boundaries
inline bool route_wide(int dtype, int E, const void *p, int64_t ld) {
  const int64_t n = 16 / (int64_t)dtype_bytes(dtype);
  return E % n == 0 && ld % n == 0 && aligned16(p);
}

// f(lanes, values) as constants
template <class F>
void with_route_shape(int E, F &&f) {
  const auto go = [&](auto l, auto v) { f(l, v); };
#define DIMO_ROUTE_SHAPE(l, v) go(std::integral_constant<int, l>{}, std::integral_constant<int, v>{})
  if (E <= 4) DIMO_ROUTE_SHAPE(1, 4);
  else if (E <= 8) DIMO_ROUTE_SHAPE(1, 8);
  else if (E <= 16) DIMO_ROUTE_SHAPE(1, 16);
  else if (E <= 32) DIMO_ROUTE_SHAPE(2, 16);
  else if (E <= 64) DIMO_ROUTE_SHAPE(4, 16);
  else if (E <= 128) DIMO_ROUTE_SHAPE(8, 16);
  else if (E <= 256) DIMO_ROUTE_SHAPE(16, 16);
  else if (E <= 512) DIMO_ROUTE_SHAPE(32, 16);
  else DIMO_ROUTE_SHAPE(64, 16);
#undef DIMO_ROUTE_SHAPE
}

// ---- grouping --------------------------------------------------------------------------------------------------
// A stable counting sort of the places by expert.  A workgroup owns GROUP_CHUNK consecutive places, a wave of it 256
// of them (four rounds of 64): per-wave counts in LDS, an exclusive scan over (expert, workgroup, wave), then every
// round ranks its 64 places among equals with one ballot per bit of the expert's number.  A place without an expert
// (any value outside 0 .. E-1) is sorted behind the last group and gets order = -1 there, position = -1.
constexpr int GROUP_THREADS = 1024, GROUP_WAVES = GROUP_THREADS / 64, GROUP_CHUNK = 4096;
constexpr int GROUP_ROUNDS = GROUP_CHUNK / GROUP_THREADS;
// Up to twice that many places are one workgroup's, with twice the rounds and no counts to exchange: one launch instead of two.
// One / two launches (places, experts; us on the GPU, and a call from Python one after another):
//   4098, 8    8.9, 12.8 / 10.0, 16.6      6000, 8    9.6, 13.0 / 10.2, 17.1      8192, 8     10.9, 13.0 / 10.5, 17.0
//   4098, 128  11.1, 12.9 / 11.2, 17.2     8192, 128  13.1, 13.1 / 11.8, 17.2     8192, 1000  15.3, 14.7 / 13.6, 17.2
constexpr int GROUP_ALONE = 2 * GROUP_CHUNK;
// Few workgroups sum the counts of all of them each for itself; that work grows with the square of the places, so from some
// number of them on a launch of its own does it once.  In-kernel sums / scan, us for all launches (workgroups, experts):
//   8, 8     10.7 / 12.7      256, 8    13.5 / 15.6     1024, 8    49 / 39
//   8, 128   12.7 / 14.7      128, 128  17.0 / 18.2     256, 128   22.9 / 23.0     1024, 128  117 / 60
//   8, 1000  14.4 / 16.4      32, 1000  16.8 / 17.5      64, 1000  20.1 / 19.0      256, 1000  48 / 36
inline bool group_scanned(int64_t blocks, int E) { return blocks > 256 || blocks * (E + 1) > 40000; }

__device__ __forceinline__ int group_key(const int32_t *experts, int64_t S, int64_t at, int E) {
  if (at >= S) return -1;
  const int e = experts[at];
  return (e >= 0 && e < E) ? e : E;
}

__global__ __launch_bounds__(GROUP_THREADS) void group_count_kernel(int64_t S, int E, const int32_t *__restrict__ experts,
                                                                    int32_t *__restrict__ counts) {
  __shared__ int hist[ROUTE_MAX_E + 1];
  for (int e = threadIdx.x; e <= E; e += GROUP_THREADS) hist[e] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < GROUP_ROUNDS; ++r) {
    const int key = group_key(experts, S, (int64_t)blockIdx.x * GROUP_CHUNK + r * GROUP_THREADS + threadIdx.x, E);
    if (key >= 0) atomicAdd(&hist[key], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += GROUP_THREADS) counts[(size_t)blockIdx.x * (E + 1) + e] = hist[e];
}

// Many workgroups: their counts become what lies before each (in place), and behind them the totals, once for all of them.
// Sixteen experts per workgroup, 64 threads each over a contiguous share of the workgroups.
__global__ __launch_bounds__(GROUP_THREADS) void group_scan_kernel(int E1, int blocks, int32_t *__restrict__ counts) {
  __shared__ int sums[64][17];
  const int col = threadIdx.x & 15, part = threadIdx.x >> 4, e = blockIdx.x * 16 + col;
  const int share = (blocks + 63) / 64, begin = min(part * share, blocks), end = min(begin + share, blocks);
  int sum = 0;
  if (e < E1)
#pragma unroll 8
    for (int b = begin; b < end; ++b) sum += counts[(size_t)b * E1 + e];
  sums[part][col] = sum;
  __syncthreads();
  int before = 0;
  for (int p = 0; p < part; ++p) before += sums[p][col];
  if (e >= E1) return;
#pragma unroll 8
  for (int b = begin; b < end; ++b) {
    const int n = counts[(size_t)b * E1 + e];
    counts[(size_t)b * E1 + e] = before;
    before += n;
  }
  if (part == 63) counts[(size_t)blocks * E1 + e] = before;
}

template <int ROUNDS>
__global__ __launch_bounds__(GROUP_THREADS) void group_place_kernel(int64_t S, int E, int bits,
                                                                    const int32_t *__restrict__ experts,
                                                                    const int32_t *__restrict__ counts, int blocks, int scanned,
                                                                    int32_t *__restrict__ offsets,
                                                                    int32_t *__restrict__ order,
                                                                    int32_t *__restrict__ position, int places,
                                                                    int32_t *__restrict__ rows) {
  HIP_DYNAMIC_SHARED(int, base)  // [GROUP_WAVES][E + 1]
  __shared__ int wave_total[GROUP_WAVES], tallies[2 * (ROUTE_MAX_E + 1)];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, E1 = E + 1;
  for (int i = t; i < GROUP_WAVES * E1; i += GROUP_THREADS) base[i] = 0;
  __syncthreads();
  int key[ROUNDS];
  const int64_t first = (int64_t)blockIdx.x * (ROUNDS * GROUP_THREADS) + wave * (64 * ROUNDS) + lane;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    key[r] = group_key(experts, S, first + 64 * r, E);
    if (key[r] >= 0) atomicAdd(&base[wave * E1 + key[r]], 1);
  }
  __syncthreads();
  if (scanned) {
    for (int e = t; e < E1; e += GROUP_THREADS)
      tallies[e] = counts[(size_t)blockIdx.x * E1 + e], tallies[E1 + e] = counts[(size_t)blocks * E1 + e];
    __syncthreads();
  } else if (counts) {
    // the workgroups' counts: `parts` threads per expert, eight loads in flight each
    for (int i = t; i < 2 * E1; i += GROUP_THREADS) tallies[i] = 0;
    __syncthreads();
    int wide = 64;
    while (wide < E1) wide *= 2;
    const int parts = wide < GROUP_THREADS ? GROUP_THREADS / wide : 1, part = t / wide;
    for (int e = t % wide; e < E1 && part < parts; e += (wide < GROUP_THREADS ? wide : GROUP_THREADS)) {
      int before = 0, total = 0;
#pragma unroll 8
      for (int b = part; b < blocks; b += parts) {
        const int n = counts[(size_t)b * E1 + e];
        total += n;
        before += b < (int)blockIdx.x ? n : 0;
      }
      atomicAdd(&tallies[e], before);
      atomicAdd(&tallies[E1 + e], total);
    }
    __syncthreads();
  }
  // exclusive scan over the experts: thread t owns expert t (the last thread's round also the places without one)
  int running = 0;
  for (int e0 = 0; e0 < E1; e0 += GROUP_THREADS) {
    const int e = e0 + t;
    int before = 0, total = 0;
    if (e < E1) {
      if (counts)
        before = tallies[e], total = tallies[E1 + e];
      else
        for (int w = 0; w < GROUP_WAVES; ++w) total += base[w * E1 + e];
    }
    int scan = total;  // inclusive over the wave
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(scan, d);
      if (lane >= d) scan += o;
    }
    if (lane == 63) wave_total[wave] = scan;
    __syncthreads();
    int ahead = running, sum = 0;
    for (int w = 0; w < GROUP_WAVES; ++w) {
      if (w < wave) ahead += wave_total[w];
      sum += wave_total[w];
    }
    running += sum;
    if (e < E1) {
      const int start = ahead + scan - total;
      if (blockIdx.x == 0) offsets[e] = start;  // offsets[E] = places that have an expert
      int at = start + before;
      for (int w = 0; w < GROUP_WAVES; ++w) {
        const int n = base[w * E1 + e];
        base[w * E1 + e] = at;
        at += n;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    unsigned long long peers = __ballot(key[r] >= 0);
    for (int b = 0; b < bits; ++b) {
      const bool bit = (key[r] >> b) & 1;
      const unsigned long long set = __ballot(bit && key[r] >= 0);
      peers &= bit ? set : ~set;
    }
    // the first of the equals takes the places of all of them from the wave's counter
    const int leader = (key[r] >= 0) ? __ffsll((long long)peers) - 1 : lane;
    int start = 0;
    if (key[r] >= 0 && leader == lane) {
      start = base[wave * E1 + key[r]];
      base[wave * E1 + key[r]] = start + __popcll(peers);
    }
    start = __shfl(start, leader);
    const int64_t place = first + 64 * r;
    if (key[r] >= 0) {
      const int at = start + __popcll(peers & ((1ull << lane) - 1ull));
      const bool has = key[r] < E;
      if (order) order[at] = has ? (int32_t)place : -1;
      if (rows) rows[at] = has ? (int32_t)place / places : -1;
      position[place] = has ? at : -1;
    }
  }
}

// ---- bringing rows together ------------------------------------------------------------------------------------
// out[t] = residual[t] + sum_j w[t, j] y[position[t, j]]: VEC consecutive elements per thread, the k loads of a thread
// independent of each other.
struct CombineArgs {
  int T, k, N;
  Divide chunks;  // N / VEC
  int64_t S;
  const void *y;
  int64_t ldy;
  const float *weights;      // [T, k] or null (all 1)
  const int32_t *position;   // [T, k]
  const void *residual;      // [T, N] rows at ld_res, or null
  int64_t ld_res;
  void *out;                 // [T, N]
  int64_t first;             // first row of this launch
};
template <class T, int VEC>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a) {
  typedef typename T::store E;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, local = a.chunks(i);
  const int64_t t = a.first + local;
  if (t >= a.T) return;
  const int n = (int)(i - local * a.chunks.d) * VEC;
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.f;
  if (a.residual) load_vec<T, VEC>(static_cast<const E *>(a.residual) + t * a.ld_res + n, acc);
  for (int j = 0; j < a.k; ++j) {
    const int32_t p = a.position[t * a.k + j];
    if (p < 0 || p >= a.S) continue;
    const float w = a.weights ? a.weights[t * a.k + j] : 1.f;
    float y[VEC];
    load_vec<T, VEC>(static_cast<const E *>(a.y) + (int64_t)p * a.ldy + n, y);
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] += w * y[v];
  }
  store_vec<T, VEC>(static_cast<E *>(a.out) + t * a.N + n, acc);
}

// Backward, a wave per row: gy[position_tj] = w_tj g_t, gw_tj = <g_t, y[position_tj]>; the rows of gy behind the last
// group, which no place points to, are cleared (wave t looks after rows t k .. t k + k - 1).
struct CombineBwdArgs {
  int T, k, N, E;
  int64_t S;
  const void *g, *y;
  int64_t ldg, ldy;
  const float *weights;
  const int32_t *position, *offsets;
  void *g_y;         // [S, N] or null
  float *g_weights;  // [T, k] or null
  int64_t first;     // first workgroup of this launch
};
template <class T, int VEC>
__global__ __launch_bounds__(256) void combine_backward_kernel(CombineBwdArgs a) {
  typedef typename T::store E;
  const int lane = threadIdx.x & 63;
  const int64_t t = (a.first + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  for (int j = 0; j < a.k; ++j) {
    const int32_t p = a.position[t * a.k + j];
    const bool has = p >= 0 && p < a.S;
    const float w = a.weights ? a.weights[t * a.k + j] : 1.f;
    float dot = 0.f;
    if (has)
      for (int n = lane * VEC; n < a.N; n += 64 * VEC) {
        float g[VEC], v[VEC];
        load_vec<T, VEC>(static_cast<const E *>(a.g) + t * a.ldg + n, g);
        if (a.g_weights) {
          load_vec<T, VEC>(static_cast<const E *>(a.y) + (int64_t)p * a.ldy + n, v);
#pragma unroll
          for (int q = 0; q < VEC; ++q) dot += g[q] * v[q];
        }
        if (a.g_y) {
#pragma unroll
          for (int q = 0; q < VEC; ++q) v[q] = w * g[q];
          store_vec<T, VEC>(static_cast<E *>(a.g_y) + (int64_t)p * a.N + n, v);
        }
      }
    if (a.g_weights) {
      dot = row_sum<64>(dot);
      if (lane == 0) a.g_weights[t * a.k + j] = has ? dot : 0.f;
    }
  }
  if (!a.g_y) return;
  const int64_t used = a.offsets[a.E];
  const float zero[VEC] = {};
  for (int64_t r = t * a.k; r < (t + 1) * a.k; ++r)
    if (r >= used)
      for (int n = lane * VEC; n < a.N; n += 64 * VEC) store_vec<T, VEC>(static_cast<E *>(a.g_y) + r * a.N + n, zero);
}

}  // namespace

extern "C" size_t dimo_route_workspace_bytes(int T, int E) {
  if (T <= 0 || E <= 0) return 0;
  const int blocks = route_blocks(T, E);
  if (blocks == 1) return 0;  // (one workgroup's sums are the load)
  return align_up((size_t)(blocks < ROUTE_MAX_BLOCKS ? blocks : ROUTE_MAX_BLOCKS) * E * sizeof(float));
}

extern "C" int dimo_route_topk_forward(int T, int E, int k, int dtype, const void *logits, int64_t ld,
                                       const uint8_t *row_mask, int normalize, float *weights, int32_t *experts,
                                       float *load, void *workspace, size_t workspace_bytes, void *stream) {
  if (T < 0 || T > DIMO_MAX_SIZE || E < 1 || E > ROUTE_MAX_E || k < 1 || k > E || !known_dtype(dtype) || ld < E) return DIMO_E_ARG;
  if (T > 0 && (!logits || !weights || !experts)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_ROUTE, s);
  const int64_t most = launch_groups(ROUTE_THREADS);  // (the kernel goes over the rows in rounds)
  int grid = T > 0 ? route_blocks(T, E) : 0;
  if (grid > most) grid = (int)most;
  if (load) {
    const size_t need = dimo_route_workspace_bytes(T, E);
    if (workspace_bytes < need || (need && !workspace)) return DIMO_E_WORKSPACE;
    if (grid > ROUTE_MAX_BLOCKS) grid = ROUTE_MAX_BLOCKS;
  }
  float *partial = static_cast<float *>(workspace);
  if (T > 0) {
    const RouteArgs a{T, E, k, normalize, route_wide(dtype, E, logits, ld), logits, ld, row_mask, weights, experts,
                      load ? (grid == 1 ? load : partial) : nullptr, 1.0f / (float)T};
    with_dtype(dtype, [&](auto tag) {
      with_route_shape(E, [&](auto l, auto v) {
        hipLaunchKernelGGL((route_forward_kernel<decltype(tag), decltype(l)::value, decltype(v)::value>), dim3(grid),
                           dim3(ROUTE_THREADS), 0, s, a);
      });
    });
  }
  if (load && grid != 1)
    hipLaunchKernelGGL(route_load_kernel, dim3((E + 15) / 16), dim3(256), 0, s, E, grid, partial, load);
  return check_launch();
}

extern "C" int dimo_route_topk_backward(int T, int E, int k, int dtype, const void *logits, int64_t ld,
                                        const uint8_t *row_mask, int normalize, const float *weights,
                                        const int32_t *experts, const float *g_weights, const float *g_load,
                                        void *g_logits, void *stream) {
  if (T < 0 || T > DIMO_MAX_SIZE || E < 1 || E > ROUTE_MAX_E || k < 1 || k > E || !known_dtype(dtype) || ld < E) return DIMO_E_ARG;
  if (T == 0) return DIMO_OK;
  if (!logits || !weights || !experts || !g_logits) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_ROUTE, s);
  RouteBwdArgs a{T, E, k, normalize, route_wide(dtype, E, logits, ld) && route_wide(dtype, E, g_logits, E), logits, ld,
                 row_mask, weights, experts, g_weights, g_load, g_logits, 1.0f / (float)T, 0};
  return for_launches(route_blocks(T, E), ROUTE_THREADS, [&](int64_t first, unsigned grid) {
    a.first = first;
    with_dtype(dtype, [&](auto tag) {
      with_route_shape(E, [&](auto l, auto v) {
        hipLaunchKernelGGL((route_backward_kernel<decltype(tag), decltype(l)::value, decltype(v)::value>), dim3(grid),
                           dim3(ROUTE_THREADS), 0, s, a);
      });
    });
  });
}

extern "C" size_t dimo_group_rows_workspace_bytes(int64_t S, int E) {
  if (S <= GROUP_ALONE || E <= 0) return 0;
  const int64_t blocks = (S + GROUP_CHUNK - 1) / GROUP_CHUNK;
  return align_up((size_t)(blocks + group_scanned(blocks, E)) * (E + 1) * sizeof(int32_t));
}

extern "C" int dimo_group_rows(int64_t S, int E, int places, const int32_t *experts, int32_t *offsets, int32_t *order,
                               int32_t *position, int32_t *rows, void *workspace, size_t workspace_bytes, void *stream) {
  if (S < 0 || S > DIMO_MAX_SIZE || E < 1 || E > ROUTE_MAX_E || places < 1 || !offsets) return DIMO_E_ARG;
  if (S > 0 && (!experts || !position)) return DIMO_E_ARG;
  if (workspace_bytes < dimo_group_rows_workspace_bytes(S, E) || (S > GROUP_ALONE && !workspace)) return DIMO_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_ROUTE, s);
  int bits = 1;
  while ((1 << bits) <= E) ++bits;
  const int blocks = S > GROUP_ALONE ? (int)((S + GROUP_CHUNK - 1) / GROUP_CHUNK) : 1;
  int32_t *counts = blocks > 1 ? static_cast<int32_t *>(workspace) : nullptr;
  const int scanned = group_scanned(blocks, E);
  if (counts)
    hipLaunchKernelGGL(group_count_kernel, dim3(blocks), dim3(GROUP_THREADS), 0, s, S, E, experts, counts);
  if (scanned)
    hipLaunchKernelGGL(group_scan_kernel, dim3((E + 16) / 16), dim3(GROUP_THREADS), 0, s, E + 1, blocks, counts);
  const size_t lds = (size_t)GROUP_WAVES * (E + 1) * sizeof(int);
  auto place = S > GROUP_CHUNK && S <= GROUP_ALONE ? group_place_kernel<2 * GROUP_ROUNDS> : group_place_kernel<GROUP_ROUNDS>;
  if (lds > 32768) {  // (1024 experts: 65 600 bytes and 8 KB of tallies; a workgroup has 160 KB)
    if (hipFuncSetAttribute(reinterpret_cast<const void *>(place), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) !=
        hipSuccess)
      return check_launch();
  }
  hipLaunchKernelGGL(place, dim3(blocks), dim3(GROUP_THREADS), lds, s, S, E, bits, experts, counts, blocks, scanned, offsets,
                     order, position, places, rows);
  return check_launch();
}

extern "C" int dimo_combine_rows_forward(int T, int k, int N, int64_t S, int dtype, const void *y, int64_t ldy,
                                         const float *weights, const int32_t *position, const void *residual,
                                         int64_t ld_residual, void *out, void *stream) {
  if (T < 0 || T > DIMO_MAX_SIZE || k < 1 || N < 0 || N > DIMO_MAX_SIZE || S < 0 || S > DIMO_MAX_SIZE || !known_dtype(dtype) || ldy < N || (residual && ld_residual < N))
    return DIMO_E_ARG;
  if (T == 0 || N == 0) return DIMO_OK;
  if ((S > 0 && !y) || !position || !out) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_COMBINE, s);
  const int vec = 16 / (int)dtype_bytes(dtype);
  const bool wide = N % vec == 0 && ldy % vec == 0 && aligned16(y) && aligned16(out) &&
                    (!residual || (ld_residual % vec == 0 && aligned16(residual)));
  CombineArgs a{T, k, N, Divide((uint32_t)(wide ? N / vec : N)), S, y, ldy, weights, position, residual, ld_residual, out, 0};
  // (bands of rows whose chunks a launch can count in 31 bits)
  const int64_t most = (0x7fffffffLL - 255) / a.chunks.d;
  for (; a.first < T; a.first += most) {
    const int64_t units = (T - a.first < most ? T - a.first : most) * a.chunks.d;
    with_dtype(dtype, [&](auto tag) {
      typedef decltype(tag) Tag;
      if (wide)
        hipLaunchKernelGGL((combine_kernel<Tag, Vec16<Tag>::N>), dim3((unsigned)((units + 255) / 256)), dim3(256), 0, s, a);
      else
        hipLaunchKernelGGL((combine_kernel<Tag, 1>), dim3((unsigned)((units + 255) / 256)), dim3(256), 0, s, a);
    });
    const int rc = check_launch();
    if (rc) return rc;
  }
  return DIMO_OK;
}

extern "C" int dimo_combine_rows_backward(int T, int k, int N, int64_t S, int E, int dtype, const void *g_out,
                                          int64_t ldg, const void *y, int64_t ldy, const float *weights,
                                          const int32_t *position, const int32_t *offsets, void *g_y,
                                          float *g_weights, void *stream) {
  if (T < 0 || k < 1 || N < 0 || N > DIMO_MAX_SIZE || E < 1 || S != (int64_t)T * k || S > DIMO_MAX_SIZE || !known_dtype(dtype) || ldg < N || (g_weights && ldy < N))
    return DIMO_E_ARG;
  if (T == 0) return DIMO_OK;
  if ((N > 0 && (!g_out || (g_weights && !y))) || !position || !offsets) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_COMBINE, s);
  const int vec = 16 / (int)dtype_bytes(dtype);
  const bool wide = N % vec == 0 && ldg % vec == 0 && aligned16(g_out) && (!g_y || aligned16(g_y)) &&
                    (!g_weights || (ldy % vec == 0 && aligned16(y)));
  CombineBwdArgs a{T, k, N, E, S, g_out, y, ldg, ldy, weights, position, offsets, g_y, g_weights, 0};
  return for_launches(((int64_t)T + 3) / 4, 256, [&](int64_t first, unsigned grid) {
    a.first = first;
    with_dtype(dtype, [&](auto tag) {
      typedef decltype(tag) Tag;
      if (wide)
        hipLaunchKernelGGL((combine_backward_kernel<Tag, Vec16<Tag>::N>), dim3(grid), dim3(256), 0, s, a);
      else
        hipLaunchKernelGGL((combine_backward_kernel<Tag, 1>), dim3(grid), dim3(256), 0, s, a);
    });
  });
}
