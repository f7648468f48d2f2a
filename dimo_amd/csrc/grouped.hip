// Matrix products grouped by expert, with groups of any size:
//   forward  y_r = act(W_e x_src(r) + b_e)             rows r of [offsets[e], offsets[e + 1])
//   dgrad    gx_r = (gz_r W_e) act'(saved_r)           (the slope of the activation that made this product's input)
//   wgrad    gW_e = sum_r gz_r x_src(r)^T, gb_e = sum_r gz_r
// x may be read through the grouping (src(r) = rows[r]: the gather of the rows is free), the sizes of
// the groups stay on the device: a launch has one workgroup per possible tile, and a workgroup finds its (expert, rows)
// by a scan over the offsets.  Rows behind the last group are written as zeros.
//
// Products run on the 16-bit matrix instructions with fp32 sums; fp32 operands as three bf16 pieces each, six
// products (matrix_ops.hpp).
#include <hip/hip_runtime.h>

#include "row_tiles.hpp"
#include "tile_product.hpp"

using namespace dimo;

namespace {

struct GroupedArgs {
  int R, E, K, N;          // rows, experts, width of x, width of y
  const void *x;           // [., K] rows at ldx
  int64_t ldx;
  const int32_t *rows, *offsets;  // rows: x's row of row r, or null
  const void *w;           // [E, N, K]
  const void *bias;        // [E, N] or null
  int act;                 // DIMO_ACT_*
  void *y, *z;             // [R, N]; z: before the activation, or null
  const void *g;           // [R, N] (dgrad, wgrad)
  const void *saved;       // [R, K] (dgrad, with act): output (relu) or input (silu) of the activation
  void *gx;                // [R, K]
  void *gw, *gb;           // [E, N, K], [E, N] or null
  int wide;                // sixteen bytes of an output row may be written at once
  int split_rows, chunks;  // wgrad: > 0: partial sums over that many rows at a time, `chunks` of them at most
  float *partial;          // [chunks, N, K], then [chunks, N]
  int first;               // first workgroup of this launch
};

__device__ __forceinline__ int64_t source_row(const GroupedArgs &a, int r) {
  return a.rows ? max(a.rows[r], 0) : r;  // (no row stands behind the last group: offsets that reach there read row 0)
}

enum { FORWARD = 0, DGRAD = 1 };

template <class T, int MODE, int HOW, class C>
__global__ __launch_bounds__(C::THREADS, 2) void grouped_rows_kernel(GroupedArgs a) {
  typedef typename T::store E;
  constexpr int BK = Planes<T>::DEPTH;
  const int columns = MODE == FORWARD ? a.N : a.K, reduction = MODE == FORWARD ? a.K : a.N;
  int ct = 0;
  const RowTile tile = find_row_tile<HALVES<C>>(a.offsets, a.E, a.R, C::TJ, (columns + C::TI - 1) / C::TI, a.first + (int)blockIdx.x, &ct);
  if (tile.expert < 0) return;
  const int c0 = ct * C::TI;
  E *out = static_cast<E *>(MODE == FORWARD ? a.y : a.gx);
  if (tile.expert == a.E) {  // behind the last group
    for (int i = threadIdx.x; i < C::TJ * C::TI; i += C::THREADS) {
      const int r = tile.begin + i / C::TI, c = c0 + i % C::TI;
      if (r < tile.end && c < columns) {
        out[(int64_t)r * columns + c] = E(0);
        if (MODE == FORWARD && a.z) static_cast<E *>(a.z)[(int64_t)r * columns + c] = E(0);
      }
    }
    return;
  }
  const E *W = static_cast<const E *>(a.w) + (int64_t)tile.expert * a.N * a.K;
  Staging<T, LINES, C::TJ, BK, C::THREADS> sj;
  sj.init_lines([&](int i) {
    const int r = min(tile.begin + i, tile.end - 1);
    return MODE == FORWARD ? static_cast<const E *>(a.x) + source_row(a, r) * a.ldx
                           : static_cast<const E *>(a.g) + (int64_t)r * a.N;
  });
  Staging<T, MODE == FORWARD ? LINES : COLUMNS, C::TI, BK, C::THREADS> si;
  if constexpr (MODE == FORWARD)
    si.init_lines([&](int i) { return W + (int64_t)min(c0 + i, a.N - 1) * a.K; });
  else
    si.init_columns(W + c0, a.K, a.K - c0);
  Accumulators<C::NJ, C::NI> acc;
  acc.clear();
  DIMO_STAGE_BUFFERS(T, C, HOW);
  run_stages<T, C, LINES, MODE == FORWARD ? LINES : COLUMNS, HOW, false>(sj, si, 0, reduction, SameRow{}, SameRow{}, acc, false, SJ0,
                                                                            SI0, SJ1, SI1, idle_wave<C>(tile));
  __syncthreads();
  const E *bias = MODE == FORWARD && a.bias ? static_cast<const E *>(a.bias) + (int64_t)tile.expert * a.N : nullptr;
  const auto add_bias = [&](int i, float (&v)[4]) {
    if (MODE != FORWARD || !bias) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += T::load(bias[min(c0 + i + e, columns - 1)]);
  };
  const auto out_row = [&](E *matrix) {
    return [=](int j) { return tile.begin + j < tile.end ? matrix + (int64_t)(tile.begin + j) * columns : nullptr; };
  };
  if constexpr (MODE == FORWARD) {
    if (a.z) write_outputs<T, C, (int)sizeof(SJ0)>(acc, SJ0, c0, columns, a.wide, out_row(static_cast<E *>(a.z)), add_bias, NoSlope{});
    write_outputs<T, C, (int)sizeof(SJ0)>(acc, SJ0, c0, columns, a.wide, out_row(out), [&](int i, float (&v)[4]) {
      add_bias(i, v);
      if (a.act != DIMO_ACT_NONE)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = activate(v[e], a.act);
    }, NoSlope{});
  } else if (a.act == DIMO_ACT_NONE) {
    write_outputs<T, C, (int)sizeof(SJ0)>(acc, SJ0, c0, columns, a.wide, out_row(out), add_bias, NoSlope{});
  } else {
    const int64_t away = static_cast<const E *>(a.saved) - out;  // (both [R, K])
    if (a.act == DIMO_ACT_RELU)
      write_outputs<T, C, (int)sizeof(SJ0)>(acc, SJ0, c0, columns, a.wide, out_row(out), add_bias, ReluSlope{away});
    else
      write_outputs<T, C, (int)sizeof(SJ0)>(acc, SJ0, c0, columns, a.wide, out_row(out), add_bias, SiluSlope{away});
  }
}

// WHOLE: the reduction is whole chunks of eight (then no load needs a branch: what is behind the end is read from the last
// chunk and cleared)
template <class T, bool WHOLE>
__device__ __forceinline__ void thin_chunk(const typename T::store *line, int k, int K, typename T::store (&v)[8]) {
  typedef typename T::store E;
  if constexpr (WHOLE) {
    __builtin_memcpy(v, line + min(k, K - 8), sizeof(v));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k < K ? v[e] : E(0);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < K ? line[k + e] : E(0);
  }
}
template <class T>
__device__ __forceinline__ void thin_operand(const typename T::store (&v)[8], uint4 (&out)[Planes<T>::N]) {
  if constexpr (Planes<T>::N == 1) {
    __builtin_memcpy(&out[0], v, 16);
  } else {
    uint32_t w[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const Split3 a = split3(v[2 * e]), b = split3(v[2 * e + 1]);
      w[0][e] = a.hi | (uint32_t)b.hi << 16, w[1][e] = a.mid | (uint32_t)b.mid << 16, w[2][e] = a.lo | (uint32_t)b.lo << 16;
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) out[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
  }
}

template <class T, bool WHOLE>
__global__ __launch_bounds__(64 * THIN_WAVES) void grouped_thin_kernel(GroupedArgs a) {
  typedef typename T::store E;
  constexpr int P = Planes<T>::N, STEPS = 128 / (16 * (int)sizeof(E));  // sixteens of the reduction in a line of memory
  typedef typename Planes<T>::Tag Tag;
  __shared__ float4 buffer[THIN_WAVES][4][64];
  int ct = 0;
  const RowTile tile = find_row_tile<false>(a.offsets, a.E, a.R, 32, (a.N + 31) / 32, a.first + (int)blockIdx.x, &ct);
  if (tile.expert < 0) return;
  const int lane = threadIdx.x & 63, c0 = 32 * ct;
  E *out = static_cast<E *>(a.y);
  f32x16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  const bool behind = tile.expert == a.E;  // the last group: zeros
  if (!behind) {
    const E *w = static_cast<const E *>(a.w) + ((int64_t)tile.expert * a.N + min(c0 + (lane & 31), a.N - 1)) * a.K;
    const E *x = static_cast<const E *>(a.x) + source_row(a, min(tile.begin + (lane & 31), tile.end - 1)) * a.ldx;
    for (int k1 = 0; k1 < a.K; k1 += 16 * STEPS * THIN_WAVES) {  // (the same count for every wave: behind the end are zeros)
      const int k0 = k1 + 16 * STEPS * wave_number();
      E vw[STEPS][8], vx[STEPS][8];
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        thin_chunk<T, WHOLE>(w, k0 + 16 * s + 8 * (lane >> 5), a.K, vw[s]);
        thin_chunk<T, WHOLE>(x, k0 + 16 * s + 8 * (lane >> 5), a.K, vx[s]);
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        uint4 ow[P], ox[P];
        thin_operand<T>(vw[s], ow);
        thin_operand<T>(vx[s], ox);
#pragma unroll
        for (int d = P - 1; d >= 0; --d)
#pragma unroll
          for (int p = 0; p <= d; ++p) acc = mfma_32x32x16(Tag{}, ow[p], ox[d - p], acc);
      }
    }
  }
  sum_over_waves(acc, buffer, [&](float (&v)[4], int j, int i) {
    const int r = tile.begin + j, c = c0 + i;
    if (r >= tile.end || c >= a.N) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (a.bias && !behind) v[e] += T::load(static_cast<const E *>(a.bias)[(int64_t)tile.expert * a.N + min(c + e, a.N - 1)]);
    if (a.z) store_quad<T>(static_cast<E *>(a.z) + (int64_t)r * a.N, c, a.N, a.wide, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = behind ? 0.f : activate(v[e], a.act);
    store_quad<T>(out + (int64_t)r * a.N, c, a.N, a.wide, v);
  });
}

// gW[e]: rows n (from g) x columns k (from x), summed over the group's rows -- all of them, or split_rows of them at a time:
// a group of more rows than that is cut into slices, whose sums go to `partial` and are added in their order by the next
// kernel (the result does not depend on the schedule).
//
// Slices of the expert's group (0 or 1: it is not cut) and the number of slices of cut groups before it.
__device__ __forceinline__ int cut_slices(const GroupedArgs &a, int expert, int *before) {
  int count = 0;
  *before = 0;
  for (int e0 = 0; e0 <= expert; e0 += 64) {
    RowTileScan s;
    s.step(a.offsets, a.E, a.R, a.split_rows, e0);
    const int lane = threadIdx.x & 63;
    int cut = e0 + lane < expert && s.mine > 1 ? s.mine : 0;
#pragma unroll
    for (int d = 32; d; d /= 2) cut += __shfl_xor(cut, d);
    *before += cut;
    if (expert - e0 < 64) count = __shfl(s.mine, expert - e0);
  }
  return __builtin_amdgcn_readfirstlane(count);
}
// The n-th slice of all groups, whole ones first, so that no long piece of work is left for the end; -1: there are fewer.
__device__ __forceinline__ int find_slice(const GroupedArgs &a, int n, int *begin, int *end) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int rest = 0; rest < 2; ++rest)
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int e = e0 + lane;
      const int lo = e < a.E ? clamp_offset(a.offsets, e, a.R) : 0;
      const int size = e < a.E ? max(lo, clamp_offset(a.offsets, e + 1, a.R)) - lo : 0, whole = size / a.split_rows;
      const int mine = rest ? size > whole * a.split_rows : whole;
      int scan = mine;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(scan, d);
        if (lane >= d) scan += o;
      }
      const unsigned long long past = __ballot(before + scan > n);
      if (past) {
        const int f = __ffsll((long long)past) - 1;
        const int at = rest ? whole : n - (before + scan - mine);
        *begin = __builtin_amdgcn_readlane(lo + (lane == f ? at : 0) * a.split_rows, f);
        *end = min(*begin + a.split_rows, __builtin_amdgcn_readlane(lo + size, f));
        return e0 + f;
      }
      before += __builtin_amdgcn_readlane(scan, 63);
    }
  return -1;
}
template <class T, int HOW, class C, class Row>
__global__ __launch_bounds__(C::THREADS, 2) void grouped_wgrad_kernel(GroupedArgs a) {
  typedef typename T::store E;
  constexpr int BK = Planes<T>::DEPTH;
  const int tiles_k = (a.K + C::TI - 1) / C::TI, tiles_n = (a.N + C::TJ - 1) / C::TJ;
  const int workgroup = a.first + (int)blockIdx.x;
  int expert, begin, end, chunk = -1, block;  // chunk: the slice's place in `partial`
  if (a.split_rows) {
    int before = 0;
    block = workgroup % (tiles_k * tiles_n);
    expert = find_slice(a, workgroup / (tiles_k * tiles_n), &begin, &end);
    if (expert < 0) return;
    if (cut_slices(a, expert, &before) > 1) {
      chunk = __builtin_amdgcn_readfirstlane(before) + (begin - clamp_offset(a.offsets, expert, a.R)) / a.split_rows;
      if (chunk >= a.chunks) return;  // (only where bad offsets make the groups overlap)
    }
  } else {
    expert = largest_first(a.offsets, a.E, a.R, workgroup / (tiles_k * tiles_n)), block = workgroup % (tiles_k * tiles_n);
    begin = clamp_offset(a.offsets, expert, a.R), end = max(begin, clamp_offset(a.offsets, expert + 1, a.R));
  }
  const int n0 = block / tiles_k * C::TJ, k0 = block % tiles_k * C::TI;
  Staging<T, COLUMNS, C::TJ, BK, C::THREADS> sj;
  Staging<T, COLUMNS, C::TI, BK, C::THREADS> si;
  sj.init_columns(static_cast<const E *>(a.g) + n0, a.N, a.N - n0);
  si.init_columns(static_cast<const E *>(a.x) + k0, a.ldx, a.K - k0);
  Accumulators<C::NJ, C::NI> acc;
  acc.clear();
  const bool sums = a.gb && k0 == 0 && wave_number() % C::WI == 0;  // (one of the waves that read a row)
  DIMO_STAGE_BUFFERS(T, C, HOW);
  Row row;
  if constexpr (Row::AHEAD) row.rows = a.rows;
  if (begin < end)
    run_stages<T, C, COLUMNS, COLUMNS, HOW, true>(sj, si, begin, end, SameRow{}, row, acc, sums, SJ0, SI0, SJ1, SI1);
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = wave_number();
  const int64_t slice = max(chunk, 0);
  float *pw = a.partial + slice * a.N * a.K, *pb = a.partial + (int64_t)a.chunks * a.N * a.K + slice * a.N;
  E *gw = static_cast<E *>(a.gw) + (int64_t)expert * a.N * a.K, *gb = static_cast<E *>(a.gb) + (int64_t)expert * a.N;
  const auto as_it_is = [](int, float (&)[4]) {};
  if (chunk >= 0)
    write_outputs<F32, C, (int)sizeof(SJ0)>(acc, SJ0, k0, a.K, a.wide,
                                            [&](int j) { return n0 + j < a.N ? pw + (int64_t)(n0 + j) * a.K : nullptr; }, as_it_is, NoSlope{});
  else
    write_outputs<T, C, (int)sizeof(SJ0)>(acc, SJ0, k0, a.K, a.wide,
                                          [&](int j) { return n0 + j < a.N ? gw + (int64_t)(n0 + j) * a.K : nullptr; }, as_it_is, NoSlope{});
  if (sums) {
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) {
      const float v = acc.sums[j] + __shfl_xor(acc.sums[j], 32);
      const int n = n0 + (wave / C::WI) * 32 * C::NJ + 32 * j + lane;
      if (lane >= 32 || n >= a.N) continue;
      if (chunk >= 0)
        pb[n] = v;
      else
        gb[n] = T::save(v);
    }
  }
}

// gW[e], gb[e] of the experts whose group is cut (the sums of its slices) or empty (zeros)
template <class T>
__global__ __launch_bounds__(256) void grouped_wgrad_sum_kernel(GroupedArgs a) {
  typedef typename T::store E;
  const int e = blockIdx.y;
  int first;
  int count = cut_slices(a, e, &first);
  if (count == 1) return;
  count = min(count, max(0, a.chunks - first));
  const int64_t size = (int64_t)a.N * a.K, stride = (int64_t)gridDim.x * 256, t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const float *pw = a.partial + (int64_t)first * size, *pb = a.partial + (int64_t)a.chunks * size + (int64_t)first * a.N;
  E *gw = static_cast<E *>(a.gw) + (int64_t)e * size, *gb = static_cast<E *>(a.gb) + (int64_t)e * a.N;
  const int64_t quads = a.wide ? size / 4 : 0;
  for (int64_t i = 4 * t; i < 4 * quads; i += 4 * stride) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int c = 0; c < count; ++c) {
      const float4 p = *reinterpret_cast<const float4 *>(pw + c * size + i);
      v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
    }
    store_quad<T>(gw + i, 0, 4, true, v);
  }
  const auto sum = [&](const float *p, int64_t step) {
    float v = 0.f;
#pragma unroll 4
    for (int c = 0; c < count; ++c) v += p[c * step];
    return T::save(v);
  };
  for (int64_t i = 4 * quads + t; i < size; i += stride) gw[i] = sum(pw + i, size);
  if (a.gb)
    for (int64_t i = t; i < a.N; i += stride) gb[i] = sum(pb + i, a.N);
}

// gz = gy act'(s): s is the activation's output for relu (positive exactly where its input is) and its input for silu
template <class T, int VEC>
__global__ __launch_bounds__(256) void activation_backward_kernel(int64_t n, int act, const typename T::store *__restrict__ g,
                                                                  const typename T::store *__restrict__ s,
                                                                  typename T::store *__restrict__ out, int64_t first) {
  const int64_t i = ((first + blockIdx.x) * 256 + threadIdx.x) * VEC;
  if (i >= n) return;
  float gv[VEC], sv[VEC];
  load_vec<T, VEC>(g + i, gv);
  load_vec<T, VEC>(s + i, sv);
#pragma unroll
  for (int v = 0; v < VEC; ++v) gv[v] *= activation_slope(sv[v], act);
  store_vec<T, VEC>(out + i, gv);
}

bool bad_shape(int dtype, int R, int E, int K, int N) {
  return !known_dtype(dtype) || R < 0 || R > DIMO_MAX_SIZE || E < 1 || E > DIMO_MAX_EXPERTS || K < 1 ||
         K > DIMO_MAX_SIZE || N < 1 || N > DIMO_MAX_SIZE;
}

typedef Tile<64, 64, 2, 2> Small;
typedef Tile<128, 128, 2, 2> Medium;
typedef Tile<256, 256, 2, 4> Large;

// rows on 16-byte boundaries, their ends on whole chunks
bool whole_chunks(int dtype, const void *p, int64_t ld, int64_t width) {
  return aligned16(p) && ld % (16 / (int64_t)dtype_bytes(dtype)) == 0 && width % 8 == 0;
}
bool wide_output(int dtype, const void *p, int64_t columns) {
  return columns % (16 / (int64_t)dtype_bytes(dtype)) == 0 && aligned16(p);
}

template <class T, int MODE, int HOW, class C>
int launch_rows(GroupedArgs a, hipStream_t s) {
  const int64_t groups = row_tile_workgroups<HALVES<C>>(row_tile_count<HALVES<C>>(a.R, a.E, C::TJ), ((MODE == FORWARD ? a.N : a.K) + C::TI - 1) / C::TI);
  if (groups > 0x7fffffffLL) return DIMO_E_ARG;
  return for_launches(groups, C::THREADS, [&](int64_t first, unsigned count) {
    a.first = (int)first;
    hipLaunchKernelGGL((grouped_rows_kernel<T, MODE, HOW, C>), dim3(count), dim3(C::THREADS), 0, s, a);
  });
}
template <class T, int HOW, class C>
int launch_wgrad(GroupedArgs a, hipStream_t s) {
  const int64_t tiles = (int64_t)((a.N + C::TJ - 1) / C::TJ) * ((a.K + C::TI - 1) / C::TI);
  const int64_t groups = tiles * (a.split_rows ? row_tile_count(a.R, a.E, a.split_rows) : a.E);
  if (groups > 0x7fffffffLL || tiles > 0x7fffffffLL) return DIMO_E_ARG;
  return for_launches(groups, C::THREADS, [&](int64_t first, unsigned count) {
    a.first = (int)first;
    if (a.rows)
      hipLaunchKernelGGL((grouped_wgrad_kernel<T, HOW, C, SourceRow>), dim3(count), dim3(C::THREADS), 0, s, a);
    else
      hipLaunchKernelGGL((grouped_wgrad_kernel<T, HOW, C, SameRow>), dim3(count), dim3(C::THREADS), 0, s, a);
  });
}

// Up to this many rows in all a forward takes the thin kernel: it reads each weight once per 32 rows of a group like the
// tiles, but spreads the reduction over a workgroup's waves.  Measured, thin / 64 x 64 tile (experts, N x K; us):
//                        1 row        8           16          32          256         512
//   bf16  8, 2048^2      9.5 / 11.7   15 / 19     16 / 19     17 / 19     28 / 18
//        16, 2048^2      8.7 / 11.4   15 / 19     15 / 19     22 / 19     30 / 20
//        64,  512^2      6.4 / 6.9    6.5 / 7.0   6.8 / 7.2   7.9 / 7.3   13 / 9
//   fp32 16, 2048^2      17 / 47      30 / 52     31 / 52     43 / 63     58 / 63     102 / 69
//         1, 1024^2      10 / 26      11 / 26     11 / 26     12 / 26     13 / 27     23 / 27
//        64,  512^2      8.5 / 17     8.6 / 17    8.9 / 17    12 / 18     22 / 24     23 / 24
// (fp32: the tile's stages are long and few workgroups run them)
inline int thin_rows(int dtype) { return dtype == DIMO_F32 ? 256 : 16; }

template <int MODE>
int run_rows(int dtype, GroupedArgs a, bool whole, hipStream_t s) {
  if (MODE == FORWARD && a.R <= thin_rows(dtype)) {
    const int64_t groups = row_tile_workgroups(row_tile_count(a.R, a.E, 32), (a.N + 31) / 32);
    if (groups > 0x7fffffffLL) return DIMO_E_ARG;
    return for_launches(groups, 64 * THIN_WAVES, [&](int64_t first, unsigned count) {
      a.first = (int)first;
      with_dtype(dtype, [&](auto tag) {
        typedef decltype(tag) T;
        if (a.K % 8 == 0)
          hipLaunchKernelGGL((grouped_thin_kernel<T, true>), dim3(count), dim3(64 * THIN_WAVES), 0, s, a);
        else
          hipLaunchKernelGGL((grouped_thin_kernel<T, false>), dim3(count), dim3(64 * THIN_WAVES), 0, s, a);
      });
    });
  }
  const int64_t per_group = (a.R + a.E - 1) / a.E;
  const int tile = choose_tile(per_group, (a.R + per_group - 1) / per_group, MODE == FORWARD ? a.N : a.K,
                               whole && dtype != DIMO_F32);
  int rc = DIMO_OK;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) T;
    constexpr int BEST = sizeof(typename T::store) == 2 ? DIRECT : WHOLE;
    if (!whole)
      rc = tile == SMALL ? launch_rows<T, MODE, ANY, Small>(a, s) : launch_rows<T, MODE, ANY, Medium>(a, s);
    else if (tile == SMALL)
      rc = launch_rows<T, MODE, BEST, Small>(a, s);
    else if (tile == MEDIUM)
      rc = launch_rows<T, MODE, BEST, Medium>(a, s);
    else if constexpr (BEST == DIRECT)
      rc = launch_rows<T, MODE, BEST, Large>(a, s);
  });
  return rc;
}

// wgrad: the tile, and rows per slice (0: groups stay whole).  Measured in bf16 / fp32, uneven groups drawn from a
// lognormal distribution (rows, groups, N x K; us; "cut at 2": groups of more than twice the mean are cut):
//                                  64 tile          128 tile                      256 tile
//   8192, 8, 256 x 256     even    10 / 23          17 / 27                       -       the 64s whole; 14 cut to 256 slices
//                          uneven  15 / 25          18 / 27                       -       the 64s cut to 256 / 512; > 18 whole
//   65536, 4, 256 x 256    even    38 / 89          33 / 65                       39      256 / 512 slices; 128s whole 61 / -
//   65536, 1, 2048 x 256   even    154 / 590        122 / 402                     107     cut to 256 / 512; 64s whole 684 / -
//   32768, 8, 1024 x 1024  even    131 / 532        96 whole, 101 cut at 2 / 380  99
//                          uneven  150 / 552        181, 117 / 847, 519           133
//   32768, 32, 1024 x 512  uneven  99 / 280         82, 82 / 350, 267             98
//   4096, 8, 2048 x 512    uneven  29 / 76          29, 28 / 115, 79              -
//   32768, 16, 4096 x 1024 even    - / -            401 / -                       313 whole, 330 cut at 2
//                          uneven  - / -            393 / -                       306 whole, 366 cut at 2
// So: the largest tile whose products last long enough to fill the chip in slices; slices where there are fewer workgroups
// than CUs (fp32, whose stages take six times as long: than twice that), of 256 rows or more; with as many
// 128 tiles as that, the groups of more than twice the mean are cut; with as many 256 tiles, taking the largest groups first
// serves better, because slices are written and read once more in fp32.  64 tiles whose stages go through registers (fp32;
// 16-bit rows that are no whole chunks) take a microsecond or two per stage, and the largest group's are one chain: groups of
// more than the mean are cut (whole / cut at 1; us):
//    5003, 13, 257 x 360   uneven 62 / 28, fp16 35 / 21        5008, 13, 256 x 360   uneven 41 / 28, even 23 / 26
//    4096, 16, 256 x 256   uneven 43 / 21                      2048, 16, 512 x 256   uneven 27 / 20, even 12 / 15
//    8192, 32, 256 x 256   uneven 45 / 27, fp16 in whole chunks 14 / 17
// 16-bit rows that are no whole chunks, of sizes for which this asks 256 tiles, run 128 tiles in the slices of that plan, which
// cuts them finer than a plan for 128 tiles does (256's / 128's slices, even; uneven; us):
//    32768, 8, 1020 x 1020    265 / 271; 274 / 494         65536, 1, 2044 x 257    324 / 698
//    32768, 32, 1020 x 516    150 / 150; 190 / 192         32768, 16, 1021 x 2043  409 / 412; 917 / 492 (whole / cut at 2)
struct WgradPlan {
  int tile, split_rows, chunks;
  size_t bytes;
};
WgradPlan wgrad_plan(int dtype, int R, int E, int K, int N) {
  WgradPlan p{SMALL, 0, 0, 0};
  const int64_t per_group = R > 0 ? (R + E - 1) / E : 1;
  const auto blocks = [&](int64_t t) { return (int64_t)E * ((N + t - 1) / t) * ((K + t - 1) / t); };
  const bool f32 = dtype == DIMO_F32;
  if (!f32 && N >= 192 && K >= 192 && blocks(256) * per_group >= 512 * 1024)
    p.tile = LARGE;
  else if (N >= 96 && K >= 96 && blocks(128) * per_group >= (f32 ? 128 : 256) * 1024)
    p.tile = MEDIUM;
  const int64_t have = blocks(p.tile == LARGE ? 256 : p.tile == MEDIUM ? 128 : 64), enough = f32 ? 512 : 256;
  int64_t rows = 0;
  if (per_group >= 512 && have < enough) {
    const int64_t splits = (enough + have - 1) / have;
    rows = (per_group + splits - 1) / splits;
  } else if (per_group >= 512 && p.tile == MEDIUM) {
    rows = 2 * per_group;
  } else if (per_group >= 128 && p.tile == SMALL && (f32 || N % 8 || K % 8)) {
    rows = per_group;
  }
  if (rows) rows = rows < 256 ? 256 : (rows + 63) / 64 * 64;
  if (rows && rows < R) {
    // a group of r > rows rows is cut into fewer than 2 r / rows slices
    const int64_t cut = 2 * (int64_t)R / rows, slices = row_tile_count(R, E, (int)rows);
    p.split_rows = (int)rows, p.chunks = (int)(cut < slices ? cut : slices);
    p.bytes = align_up((size_t)p.chunks * ((size_t)N * K + N) * sizeof(float));
  }
  return p;
}

}  // namespace

extern "C" int dimo_grouped_linear_forward(int dtype, int R, int E, int K, int N, const void *x, int64_t ldx,
                                           const int32_t *rows, const int32_t *offsets, const void *w, const void *bias, int act, void *y, void *z, void *stream) {
  if (bad_shape(dtype, R, E, K, N) || ldx < K || act < DIMO_ACT_NONE || act > DIMO_ACT_SILU) return DIMO_E_ARG;
  if (R == 0) return DIMO_OK;
  if (!x || !offsets || !w || !y) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_GROUPED, s);
  GroupedArgs a{};
  a.R = R, a.E = E, a.K = K, a.N = N, a.x = x, a.ldx = ldx, a.rows = rows, a.offsets = offsets;
  a.w = w, a.bias = bias, a.act = act, a.y = y, a.z = z;
  a.wide = wide_output(dtype, y, N) && (!z || wide_output(dtype, z, N));
  return run_rows<FORWARD>(dtype, a, whole_chunks(dtype, x, ldx, K) && whole_chunks(dtype, w, K, K), s);
}

extern "C" int dimo_grouped_linear_dgrad(int dtype, int R, int E, int K, int N, const void *g, const int32_t *offsets,
                                         const void *w, int act, const void *saved, void *gx, void *stream) {
  if (bad_shape(dtype, R, E, K, N) || act < DIMO_ACT_NONE || act > DIMO_ACT_SILU) return DIMO_E_ARG;
  if (R == 0) return DIMO_OK;
  if (!g || !offsets || !w || !gx || (act != DIMO_ACT_NONE && !saved)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_GROUPED, s);
  GroupedArgs a{};
  a.R = R, a.E = E, a.K = K, a.N = N, a.offsets = offsets, a.w = w, a.g = g, a.gx = gx;
  a.act = act, a.saved = saved;
  a.wide = wide_output(dtype, gx, K) && (act == DIMO_ACT_NONE || wide_output(dtype, saved, K));
  return run_rows<DGRAD>(dtype, a, whole_chunks(dtype, g, N, N) && whole_chunks(dtype, w, K, K), s);
}

extern "C" size_t dimo_grouped_linear_wgrad_workspace_bytes(int dtype, int R, int E, int K, int N) {
  return bad_shape(dtype, R, E, K, N) ? 0 : wgrad_plan(dtype, R, E, K, N).bytes;
}

extern "C" int dimo_grouped_linear_wgrad(int dtype, int R, int E, int K, int N, const void *g, const void *x, int64_t ldx,
                                         const int32_t *rows, const int32_t *offsets, void *gw, void *gb,
                                         void *workspace, size_t workspace_bytes, void *stream) {
  if (bad_shape(dtype, R, E, K, N) || ldx < K || !offsets || !gw) return DIMO_E_ARG;
  if (R > 0 && (!g || !x)) return DIMO_E_ARG;
  const WgradPlan plan = wgrad_plan(dtype, R, E, K, N);
  if (workspace_bytes < plan.bytes || (plan.bytes && (!workspace || !aligned16(workspace)))) return DIMO_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_GROUPED, s);
  GroupedArgs a{};
  a.R = R, a.E = E, a.K = K, a.N = N, a.x = x, a.ldx = ldx, a.rows = rows, a.offsets = offsets;
  a.g = g, a.gw = gw, a.gb = gb, a.wide = wide_output(dtype, gw, K);
  a.split_rows = plan.split_rows, a.chunks = plan.chunks, a.partial = static_cast<float *>(workspace);
  const bool whole = whole_chunks(dtype, g, N, N) && whole_chunks(dtype, x, ldx, K);
  int rc = DIMO_OK;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) T;
    constexpr int BEST = sizeof(typename T::store) == 2 ? DIRECT : WHOLE;
    if (!whole)
      rc = plan.tile == SMALL ? launch_wgrad<T, ANY, Small>(a, s) : launch_wgrad<T, ANY, Medium>(a, s);
    else if (plan.tile == SMALL)
      rc = launch_wgrad<T, BEST, Small>(a, s);
    else if (plan.tile == MEDIUM)
      rc = launch_wgrad<T, BEST, Medium>(a, s);
    else if constexpr (BEST == DIRECT)
      rc = launch_wgrad<T, BEST, Large>(a, s);
    if (!rc && a.split_rows) {
      // (most experts' workgroups may find nothing to do: few each, unless there are few experts)
      const int64_t blocks = ((int64_t)N * K / (a.wide ? 4 : 1) + 255) / 256, most = E < 16 ? 4096 / E : 256;
      hipLaunchKernelGGL((grouped_wgrad_sum_kernel<T>), dim3((unsigned)(blocks < most ? blocks : most), E), dim3(256), 0, s, a);
      rc = check_launch();
    }
  });
  return rc;
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
  return for_launches((n / (wide ? vec : 1) + 255) / 256, 256, [&](int64_t first, unsigned count) {
    with_dtype(dtype, [&](auto tag) {
      typedef decltype(tag) Tag;
      typedef typename Tag::store E;
      if (wide)
        hipLaunchKernelGGL((activation_backward_kernel<Tag, Vec16<Tag>::N>), dim3(count), dim3(256), 0, s, n, act,
                           static_cast<const E *>(g), static_cast<const E *>(saved), static_cast<E *>(out), first);
      else
        hipLaunchKernelGGL((activation_backward_kernel<Tag, 1>), dim3(count), dim3(256), 0, s, n, act,
                           static_cast<const E *>(g), static_cast<const E *>(saved), static_cast<E *>(out), first);
    });
  });
}
