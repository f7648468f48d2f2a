// Matrix products grouped by expert, with groups of any size:
//   forward  y_r = act(W_e x_src(r) + b_e)             rows r of [offsets[e], offsets[e + 1])
//   dgrad    gx_r = gz_r W_e
//   wgrad    gW_e = sum_r gz_r x_src(r)^T, gb_e = sum_r gz_r
// x may be read through the grouping's order (src(r) = order[r] / places: the gather of the rows is free), the sizes of
// the groups stay on the device: a launch has one workgroup per possible tile, and a workgroup finds its (expert, rows)
// by a scan over the offsets.  Rows behind the last group are written as zeros.
//
// Products run on the 16-bit matrix instructions with fp32 sums; fp32 operands as three bf16 pieces each, six
// products (matrix_ops.hpp).
#include <hip/hip_runtime.h>

#include "matrix_ops.hpp"
#include "row_tiles.hpp"

using namespace dimo;

namespace {

// ---- the general kernel: any size, stride and alignment ----------------------------------------------------------
// 64 x 64 outputs per workgroup, 32 x 32 per wave, 32 deep stages through registers into LDS as [row][k] (40 elements
// apart: sixteen-byte reads of 32 consecutive rows then spread over all banks).
constexpr int GM = 64, GN = 64, GK = 32, GLD = 40;

template <class T>
struct Planes {
  static constexpr int N = 1;
  typedef T Tag;
};
template <>
struct Planes<F32> {
  static constexpr int N = 3;
  typedef BF16 Tag;
};

struct GroupedArgs {
  int R, E, K, N;          // rows, experts, width of x, width of y
  int places;              // > 0: x rows are order[r] / places
  const void *x;           // [., K] rows at ldx
  int64_t ldx;
  const int32_t *order, *offsets;
  const void *w;           // [E, N, K]
  const void *bias;        // [E, N] or null
  int act;                 // DIMO_ACT_*
  void *y, *z;             // [R, N]; z: before the activation, or null
  const void *g;           // [R, N] (dgrad, wgrad)
  void *gx;                // [R, K]
  void *gw, *gb;           // [E, N, K], [E, N] or null
};

__device__ __forceinline__ int64_t source_row(const GroupedArgs &a, int r) {
  return a.places > 0 ? a.order[r] / a.places : r;
}

// eight elements of an operand's stage as fp32, `ok` of them inside
template <class T>
__device__ __forceinline__ void stage_elements(const typename T::store *p, int ok, bool wide, typename T::store (&v)[8]) {
  if (wide && ok >= 8) {
    constexpr int Q = sizeof(typename T::store) == 4 ? 2 : 1;
    uint4 q[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) q[i] = reinterpret_cast<const uint4 *>(p)[i];
    __builtin_memcpy(v, q, sizeof(v));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < ok ? p[i] : typename T::store(0);
}

template <class T>
__device__ __forceinline__ void split_store(uint16_t (*S)[GM][GLD], int i, int k, typename T::store v) {
  if constexpr (Planes<T>::N == 3) {
    const Split3 s = split3(v);
    S[0][i][k] = s.hi, S[1][i][k] = s.mid, S[2][i][k] = s.lo;
  } else {
    S[0][i][k] = v;
  }
}

// k contiguous: thread t brings row t / 4, eight k from 8 (t % 4);  row contiguous (transposed on its way into LDS):
// k = t / 8, eight rows from 8 (t % 8)
template <class T, bool KC>
__device__ __forceinline__ void stage_store(uint16_t (*S)[GM][GLD], const typename T::store (&v)[8]) {
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (KC)
      split_store<T>(S, t >> 2, 8 * (t & 3) + i, v[i]);
    else
      split_store<T>(S, 8 * (t & 7) + i, t >> 3, v[i]);
  }
}

template <class T>
__device__ __forceinline__ void stage_multiply(uint16_t (*A)[GM][GLD], uint16_t (*B)[GN][GLD], f32x16 &acc, f32x16 *ones_acc) {
  constexpr int P = Planes<T>::N;
  typedef typename Planes<T>::Tag Tag;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = (wave >> 1) * 32 + (lane & 31), j = (wave & 1) * 32 + (lane & 31);
#pragma unroll
  for (int ks = 0; ks < GK; ks += 16) {
    const int k = ks + 8 * (lane >> 5);
    uint4 a[P], b[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      a[p] = *reinterpret_cast<const uint4 *>(&A[p][i][k]);
      b[p] = *reinterpret_cast<const uint4 *>(&B[p][j][k]);
    }
#pragma unroll
    for (int d = P - 1; d >= 0; --d)  // the smallest products first
#pragma unroll
      for (int p = 0; p <= d; ++p) acc = mfma_32x32x16(Tag{}, a[p], b[d - p], acc);
    if (ones_acc) {
      const uint32_t w = (uint32_t)Tag::save(1.0f) * 0x10001u;
      const uint4 ones = make_uint4(w, w, w, w);
#pragma unroll
      for (int p = P - 1; p >= 0; --p) *ones_acc = mfma_32x32x16(Tag{}, a[p], ones, *ones_acc);
    }
  }
}

enum { FORWARD = 0, DGRAD = 1 };

template <class T, int MODE>
__global__ __launch_bounds__(256) void grouped_rows_general_kernel(GroupedArgs a, bool wide_a, bool wide_b) {
  typedef typename T::store E;
  __shared__ __attribute__((aligned(16))) uint16_t As[Planes<T>::N][GM][GLD], Bs[Planes<T>::N][GN][GLD];
  const RowTile tile = find_row_tile(a.offsets, a.E, a.R, GM, (int)blockIdx.x);
  if (tile.expert < 0) return;
  const int cols = MODE == FORWARD ? a.N : a.K, red = MODE == FORWARD ? a.K : a.N;
  const int n0 = blockIdx.y * GN, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  E *out = static_cast<E *>(MODE == FORWARD ? a.y : a.gx);
  if (tile.expert == a.E) {  // behind the last group
    for (int i = t; i < GM * GN; i += 256) {
      const int r = tile.begin + i / GN, c = n0 + i % GN;
      if (r < tile.end && c < cols) {
        out[(int64_t)r * cols + c] = E(0);
        if (MODE == FORWARD && a.z) static_cast<E *>(a.z)[(int64_t)r * cols + c] = E(0);
      }
    }
    return;
  }
  const E *W = static_cast<const E *>(a.w) + (int64_t)tile.expert * a.N * a.K;
  // this thread's row of A (k contiguous)
  const int ra = min(tile.begin + (t >> 2), tile.end - 1);
  const E *A = MODE == FORWARD ? static_cast<const E *>(a.x) + source_row(a, ra) * a.ldx
                               : static_cast<const E *>(a.g) + (int64_t)ra * a.N;
  const int ka = 8 * (t & 3);
  f32x16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int k0 = 0; k0 < red; k0 += GK) {
    E va[8], vb[8];
    stage_elements<T>(A + min(k0 + ka, red), red - k0 - ka, wide_a, va);
    if (MODE == FORWARD) {  // row n0 + t / 4 of W
      const int n = n0 + (t >> 2);
      stage_elements<T>(W + (int64_t)min(n, a.N - 1) * a.K + min(k0 + ka, red), n < a.N ? red - k0 - ka : 0, wide_b, vb);
    } else {  // row k0 + t / 8 of W, eight columns
      const int n = k0 + (t >> 3), c = n0 + 8 * (t & 7);
      stage_elements<T>(W + (int64_t)min(n, a.N - 1) * a.K + min(c, a.K), n < a.N ? a.K - c : 0, wide_b, vb);
    }
    __syncthreads();
    stage_store<T, true>(As, va);
    stage_store<T, MODE == FORWARD>(Bs, vb);
    __syncthreads();
    stage_multiply<T>(As, Bs, acc, nullptr);
  }
  const int c = n0 + (wave & 1) * 32 + (lane & 31);
  if (c >= cols) return;
  const float bias = MODE == FORWARD && a.bias ? T::load(static_cast<const E *>(a.bias)[(int64_t)tile.expert * a.N + c]) : 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = tile.begin + (wave >> 1) * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
    if (row >= tile.end) continue;
    const float v = acc[r] + bias;
    if (MODE == FORWARD && a.z) static_cast<E *>(a.z)[(int64_t)row * cols + c] = T::save(v);
    out[(int64_t)row * cols + c] = T::save(MODE == FORWARD ? activate(v, a.act) : v);
  }
}

// one workgroup per 64 x 64 block of an expert's gradient, the rows of the group one stage after the other
template <class T>
__global__ __launch_bounds__(256) void grouped_wgrad_general_kernel(GroupedArgs a, bool wide_a, bool wide_b) {
  typedef typename T::store E;
  __shared__ __attribute__((aligned(16))) uint16_t As[Planes<T>::N][GM][GLD], Bs[Planes<T>::N][GN][GLD];
  const int e = blockIdx.y, tiles_k = (a.K + GN - 1) / GN;
  const int n0 = (blockIdx.x / tiles_k) * GM, k0 = (blockIdx.x % tiles_k) * GN;
  const int begin = clamp_offset(a.offsets, e, a.R), end = max(begin, clamp_offset(a.offsets, e + 1, a.R));
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  f32x16 acc, sums;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f, sums[i] = 0.f;
  const bool with_bias = a.gb && k0 == 0;
  for (int r0 = begin; r0 < end; r0 += GK) {
    const int r = r0 + (t >> 3), c = 8 * (t & 7), rc = min(r, end - 1);
    E va[8], vb[8];
    stage_elements<T>(static_cast<const E *>(a.g) + (int64_t)rc * a.N + min(n0 + c, a.N), r < end ? a.N - n0 - c : 0, wide_a, va);
    stage_elements<T>(static_cast<const E *>(a.x) + source_row(a, rc) * a.ldx + min(k0 + c, a.K), r < end ? a.K - k0 - c : 0, wide_b, vb);
    __syncthreads();
    stage_store<T, false>(As, va);
    stage_store<T, false>(Bs, vb);
    __syncthreads();
    stage_multiply<T>(As, Bs, acc, with_bias ? &sums : nullptr);
  }
  const int k = k0 + (wave & 1) * 32 + (lane & 31);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = n0 + (wave >> 1) * 32 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
    if (n >= a.N) continue;
    if (k < a.K) static_cast<E *>(a.gw)[((int64_t)e * a.N + n) * a.K + k] = T::save(acc[i]);
    if (with_bias && (wave & 1) == 0 && (lane & 31) == 0) static_cast<E *>(a.gb)[(int64_t)e * a.N + n] = T::save(sums[i]);
  }
}

// gz = gy act'(s): s is the activation's output for relu (positive exactly where its input is) and its input for silu
template <class T, int VEC>
__global__ __launch_bounds__(256) void activation_backward_kernel(int64_t n, int act, const typename T::store *__restrict__ g,
                                                                  const typename T::store *__restrict__ s,
                                                                  typename T::store *__restrict__ out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
  if (i >= n) return;
  float gv[VEC], sv[VEC];
  load_vec<T, VEC>(g + i, gv);
  load_vec<T, VEC>(s + i, sv);
#pragma unroll
  for (int v = 0; v < VEC; ++v) gv[v] *= activation_slope(sv[v], act);
  store_vec<T, VEC>(out + i, gv);
}

template <class T>
bool aligned_rows(const void *p, int64_t ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * (int64_t)sizeof(typename T::store) % 16 == 0;
}

bool bad_shape(int dtype, int R, int E, int K, int N) {
  return !known_dtype(dtype) || R < 0 || E < 1 || E > DIMO_MAX_EXPERTS || K < 1 || N < 1;
}

}  // namespace

extern "C" int dimo_grouped_linear_forward(int dtype, int R, int E, int K, int N, const void *x, int64_t ldx, int places,
                                           const int32_t *order, const int32_t *offsets, const void *w,
                                           const void *bias, int act, void *y, void *z, void *stream) {
  if (bad_shape(dtype, R, E, K, N) || ldx < K || places < 0 || act < DIMO_ACT_NONE || act > DIMO_ACT_SILU) return DIMO_E_ARG;
  if (R == 0) return DIMO_OK;
  if (!x || !offsets || !w || !y || (places > 0 && !order)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_GROUPED, s);
  GroupedArgs a{};
  a.R = R, a.E = E, a.K = K, a.N = N, a.places = places, a.x = x, a.ldx = ldx, a.order = order, a.offsets = offsets;
  a.w = w, a.bias = bias, a.act = act, a.y = y, a.z = z;
  const dim3 grid(row_tile_count(R, E, GM), (N + GN - 1) / GN);
  if (grid.y > 65535) return DIMO_E_ARG;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) Tag;
    hipLaunchKernelGGL((grouped_rows_general_kernel<Tag, FORWARD>), grid, dim3(256), 0, s, a, aligned_rows<Tag>(x, ldx),
                       aligned_rows<Tag>(w, K));
  });
  return check_launch();
}

extern "C" int dimo_grouped_linear_dgrad(int dtype, int R, int E, int K, int N, const void *g, const int32_t *offsets,
                                         const void *w, void *gx, void *stream) {
  if (bad_shape(dtype, R, E, K, N)) return DIMO_E_ARG;
  if (R == 0) return DIMO_OK;
  if (!g || !offsets || !w || !gx) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_GROUPED, s);
  GroupedArgs a{};
  a.R = R, a.E = E, a.K = K, a.N = N, a.offsets = offsets, a.w = w, a.g = g, a.gx = gx;
  const dim3 grid(row_tile_count(R, E, GM), (K + GN - 1) / GN);
  if (grid.y > 65535) return DIMO_E_ARG;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) Tag;
    hipLaunchKernelGGL((grouped_rows_general_kernel<Tag, DGRAD>), grid, dim3(256), 0, s, a, aligned_rows<Tag>(g, N),
                       aligned_rows<Tag>(w, K));
  });
  return check_launch();
}

extern "C" int dimo_grouped_linear_wgrad(int dtype, int R, int E, int K, int N, const void *g, const void *x, int64_t ldx,
                                         int places, const int32_t *order, const int32_t *offsets, void *gw, void *gb,
                                         void *stream) {
  if (bad_shape(dtype, R, E, K, N) || ldx < K || places < 0 || !offsets || !gw) return DIMO_E_ARG;
  if (R > 0 && (!g || !x || (places > 0 && !order))) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_GROUPED, s);
  GroupedArgs a{};
  a.R = R, a.E = E, a.K = K, a.N = N, a.places = places, a.x = x, a.ldx = ldx, a.order = order, a.offsets = offsets;
  a.g = g, a.gw = gw, a.gb = gb;
  const int64_t tiles = (int64_t)((N + GM - 1) / GM) * ((K + GN - 1) / GN);
  if (tiles > 0x7fffffffLL) return DIMO_E_ARG;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) Tag;
    hipLaunchKernelGGL((grouped_wgrad_general_kernel<Tag>), dim3((unsigned)tiles, E), dim3(256), 0, s, a,
                       aligned_rows<Tag>(g, N), aligned_rows<Tag>(x, ldx));
  });
  return check_launch();
}

extern "C" int dimo_activation_backward(int dtype, int act, int64_t n, const void *g, const void *saved, void *out,
                                        void *stream) {
  if (!known_dtype(dtype) || n < 0 || (act != DIMO_ACT_RELU && act != DIMO_ACT_SILU)) return DIMO_E_ARG;
  if (n == 0) return DIMO_OK;
  if (!g || !saved || !out) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_GROUPED, s);
  const int vec = 16 / (int)dtype_bytes(dtype);
  const bool wide = n % vec == 0 && ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(saved) |
                                      reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int64_t blocks = (n / (wide ? vec : 1) + 255) / 256;
  if (blocks > 0x7fffffffLL) return DIMO_E_ARG;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) Tag;
    typedef typename Tag::store E;
    if (wide)
      hipLaunchKernelGGL((activation_backward_kernel<Tag, Vec16<Tag>::N>), dim3((unsigned)blocks), dim3(256), 0, s, n, act,
                         static_cast<const E *>(g), static_cast<const E *>(saved), static_cast<E *>(out));
    else
      hipLaunchKernelGGL((activation_backward_kernel<Tag, 1>), dim3((unsigned)blocks), dim3(256), 0, s, n, act,
                         static_cast<const E *>(g), static_cast<const E *>(saved), static_cast<E *>(out));
  });
  return check_launch();
}
