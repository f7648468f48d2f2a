// Microscaled 4-bit floating point: blocks of 32 values along a row share one power-of-two scale (a byte, 2^(byte - 127);
// 255 = NaN), elements are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, low four bits first.
//   quantise   scale = 2^(floor(log2 max|x|) - 2), element = x / scale to the nearest e2m1 value, ties to the even code,
//              beyond 6 to 6; a block with an infinite or NaN value becomes NaN as a whole
//   product    y_rn = act(sum_k x_rk w_e,nk + b_e,n), rows in groups as in grouped.hip, on the matrix cores' scaled
//              4-bit instruction: products of elements and scales are exact, sums are fp32.
// The rounding to 4 bits is the only loss, and it happens in `quantise`, where the caller asked for it.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "row_tiles.hpp"
#include "tile_product.hpp"

using namespace dimo;

namespace {

// Values of a scale byte; 255 = NaN.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}

// Four lanes per block, eight values each: 16 bytes of 16-bit input (32 of fp32) and 4 bytes of codes per lane, so a
// wave reads and writes whole lines; the block's largest magnitude takes two exchanges.  The rounding is the hardware's
// conversion (nearest, ties to the even code, beyond 6 to 6: compared with the comparisons it stands for on every border);
// spelled out as comparisons the kernel was bound by them, 113 us instead of 67 for 32768 x 4096 in bf16.
struct QuantArgs {
  int64_t rows;
  int K, blocks;           // blocks of 32 per row
  const void *x;
  int64_t ldx;
  const int32_t *from;     // x's row of row r (negative: zeros), or null
  uint8_t *codes, *scales; // [rows, 16 blocks], [rows, blocks]
  Divide per_row;          // 4 blocks
  int64_t first;           // first row of this launch
};
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(QuantArgs a) {
  typedef typename T::store E;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, local = a.per_row(i);
  const int64_t row = a.first + local;
  const bool in = row < a.rows;
  const int col = 8 * (int)(i - local * a.per_row.d);
  const int64_t src = a.from ? (in ? a.from[row] : -1) : row;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = 0.f;
  if (in && src >= 0) {
    const E *p = static_cast<const E *>(a.x) + src * a.ldx + col;
    if (WIDE && col + 8 <= a.K) {
      constexpr int N = Vec16<T>::N;
#pragma unroll
      for (int h = 0; h < 8 / N; ++h) {
        float q[N];
        load_vec<T, N>(p + h * N, q);
#pragma unroll
        for (int e = 0; e < N; ++e) v[h * N + e] = q[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < a.K) v[e] = T::load(p[e]);
    }
  }
  uint32_t big = 0;  // bits of the largest magnitude (an infinity or NaN is larger than any number)
#pragma unroll
  for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(v[e]) & 0x7fffffffu);
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0xB1, 0xf, 0xf, false));  // quad_perm [1, 0, 3, 2]
  big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0x4E, 0xf, 0xf, false));  // quad_perm [2, 3, 0, 1]
  const uint32_t exponent = big >> 23;
  const uint32_t byte = exponent == 255u ? 255u : exponent > 2u ? exponent - 2u : 0u;
  const float scale = e8m0_value(byte);
  uint32_t word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
  if (!in) return;
  const int64_t at = a.first * a.per_row.d + i;
  reinterpret_cast<uint32_t *>(a.codes)[at] = word;
  if ((i & 3) == 0) a.scales[at >> 2] = (uint8_t)byte;
}

// Values of the codes, eight per thread.
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <class T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(int64_t first, int64_t rows, int K, Divide per_row,
                                                             const uint8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales, typename T::store *__restrict__ out,
                                                             bool wide) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x, local = per_row(i);
  const int64_t row = first + local, at = first * per_row.d + i;
  if (row >= rows) return;
  const int col = 8 * (int)(i - local * per_row.d);
  const uint32_t word = reinterpret_cast<const uint32_t *>(codes)[at];
  const float scale = e8m0_value(scales[at >> 2]);
  const f32x2 q0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 0), q1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 1);
  const f32x2 q2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 2), q3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 3);
  const float v[8] = {q0[0], q0[1], q1[0], q1[1], q2[0], q2[1], q3[0], q3[1]};
  typename T::store *p = out + row * K + col;
  if (wide && col + 8 <= K) {
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
      float q[N];
#pragma unroll
      for (int e = 0; e < N; ++e) q[e] = v[h * N + e];
      store_vec<T, N>(p + h * N, q);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < K) p[e] = T::save(v[e]);
  }
}

// ---- the product -------------------------------------------------------------------------------------------------
// The tiles and LDS stages of tile_product.hpp with codes as elements: a stage of 64 16-bit words per line is 256 values of
// k, eight blocks, and a lane's sixteen bytes are exactly one block.  The scale bytes come
// through LDS too; a byte permutation leaves those of a lane's half of the wave (blocks 2 s + l / 32), one per instruction.
struct Mx4Args {
  int R, E, K, N, blocks;
  const uint8_t *xc, *xs, *wc, *ws;
  const int32_t *offsets;  // null: one group of all rows
  const void *bias;
  int act, wide;
  void *y;
  int first;               // first workgroup of this launch
};

// Scale bytes of blocks b0 .. b0 + 7 of a line; what is behind its end counts as 2^0 (its codes are zero: a NaN scale must
// not meet them).  Without a branch: the eight bytes are read from where the line still has eight and shifted down (a
// branch here would split the stage, and the compiler then moves the stage's matrix instructions behind the next barrier,
// its operands into scratch).  SHORT: lines of fewer than eight blocks.
template <bool SHORT>
__device__ __forceinline__ uint2 load_scales(const uint8_t *line, int b0, int blocks) {
  if constexpr (!SHORT) {
    const int from = min(b0, blocks - 8), bytes = b0 - from;
    uint64_t w;
    __builtin_memcpy(&w, line + from, 8);
    const uint64_t ones = 0x7f7f7f7f7f7f7f7full;
    w = bytes >= 8 ? ones : w >> (8 * bytes) | (ones << 1 << (63 - 8 * bytes));
    return make_uint2((uint32_t)w, (uint32_t)(w >> 32));
  } else {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t byte = line[min(b0 + e, blocks - 1)];
      w[e >> 2] |= (b0 + e < blocks ? byte : 0x7fu) << (8 * (e & 3));
    }
    return make_uint2(w[0], w[1]);
  }
}
// bytes half, half + 2, half + 4, half + 6
__device__ __forceinline__ uint32_t own_scales(uint2 v, int half) {
  return __builtin_amdgcn_perm(v.y, v.x, half ? 0x07050301u : 0x06040200u);
}

template <class C>
__device__ __forceinline__ void multiply_codes(const uint16_t *SJ, const uint16_t *SI,
                                               const Reader<LINES, C::TJ, 64, C::NJ> &rj, const Reader<LINES, C::TI, 64, C::NI> &ri,
                                               const uint32_t (&sj)[C::NJ], const uint32_t (&si)[C::NI],
                                               Accumulators<C::NJ, C::NI> &acc) {
  uint4 a[2][C::NI], b[2][C::NJ];
  const auto read = [&](int s) {
#pragma unroll
    for (int i = 0; i < C::NI; ++i) a[s & 1][i] = ri.read(SI, i, s);
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) b[s & 1][j] = rj.read(SJ, j, s);
  };
  const auto step = [&](auto byte) {
    constexpr int S = decltype(byte)::value;
    if (S < 3) read(S + 1);
#pragma unroll
    for (int j = 0; j < C::NJ; ++j)
#pragma unroll
      for (int i = 0; i < C::NI; ++i) acc.v[j][i] = mfma_mx4_32x32x64<S>(a[S & 1][i], si[i], b[S & 1][j], sj[j], acc.v[j][i]);
    interleave<C::NI + C::NJ, C::NI * C::NJ>(S < 3);
    __builtin_amdgcn_sched_barrier(0);  // (or the compiler reads the whole stage first, into registers that are not there)
  };
  read(0);
  __builtin_amdgcn_sched_barrier(0);
  step(std::integral_constant<int, 0>{});
  step(std::integral_constant<int, 1>{});
  step(std::integral_constant<int, 2>{});
  step(std::integral_constant<int, 3>{});
}

template <class T, class C, bool SHORT>
__global__ __launch_bounds__(C::THREADS, 2) void mx4_rows_kernel(Mx4Args a) {
  typedef typename T::store E;
  constexpr int BK = 64;  // 16-bit words of codes per stage
  __shared__ __attribute__((aligned(1024))) uint16_t SJ0[C::TJ * BK], SI0[C::TI * BK], SJ1[C::TJ * BK], SI1[C::TI * BK];
  __shared__ uint2 scales[2][C::TJ + C::TI][2];  // [pairs of stages in turn][line][stage of the pair]
  int ct = 0;
  const RowTile tile = find_row_tile<HALVES<C>>(a.offsets, a.E, a.R, C::TJ, (a.N + C::TI - 1) / C::TI, a.first + (int)blockIdx.x, &ct);
  if (tile.expert < 0) return;
  const int c0 = ct * C::TI;
  E *out = static_cast<E *>(a.y);
  if (tile.expert == a.E) {  // behind the last group
    for (int i = threadIdx.x; i < C::TJ * C::TI; i += C::THREADS) {
      const int r = tile.begin + i / C::TI, c = c0 + i % C::TI;
      if (r < tile.end && c < a.N) out[(int64_t)r * a.N + c] = E(0);
    }
    return;
  }
  const int end = 8 * a.blocks, lane = threadIdx.x & 63, wave = wave_number();
  const int j0 = (wave / C::WI) * 32 * C::NJ, i0 = (wave % C::WI) * 32 * C::NI;
  const auto x_line = [&](int i) { return (int64_t)min(tile.begin + i, tile.end - 1); };
  const auto w_line = [&](int i) { return (int64_t)tile.expert * a.N + min(c0 + i, a.N - 1); };
  Staging<BF16, LINES, C::TJ, BK, C::THREADS> sj;  // (any 16-bit type: words of codes)
  Staging<BF16, LINES, C::TI, BK, C::THREADS> si;
  sj.init_lines([&](int i) { return reinterpret_cast<const uint16_t *>(a.xc) + x_line(i) * end; });
  si.init_lines([&](int i) { return reinterpret_cast<const uint16_t *>(a.wc) + w_line(i) * end; });
  // a thread brings one line's scales, two stages of them at a time, into LDS (as many requests as the codes themselves, since
  // a request brings 16 bytes of a line; each wave reading those of its lines from memory took three times as many)
  const int mine = threadIdx.x % (C::TJ + C::TI);
  const uint8_t *line = mine < C::TJ ? a.xs + x_line(mine) * a.blocks : a.ws + w_line(mine - C::TJ) * a.blocks;
  const auto fetch = [&](int b0) {
    const uint2 lo = load_scales<SHORT>(line, b0, a.blocks), hi = load_scales<SHORT>(line, b0 + 8, a.blocks);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  const Reader<LINES, C::TJ, BK, C::NJ> rj(j0);
  const Reader<LINES, C::TI, BK, C::NI> ri(i0);
  Accumulators<C::NJ, C::NI> acc;
  acc.clear();
  uint32_t cj[C::NJ], ci[C::NI];
  const SameRow same;
  const auto request = [&](uint16_t *SJ, uint16_t *SI, int k0) {
    sj.load_direct(SJ, k0, end, same);
    si.load_direct(SI, k0, end, same);
  };
  const auto take = [&](const uint2 (*S)[2], int which) {
#pragma unroll
    for (int j = 0; j < C::NJ; ++j) cj[j] = own_scales(S[j0 + 32 * j + (lane & 31)][which], lane >> 5);
#pragma unroll
    for (int i = 0; i < C::NI; ++i) ci[i] = own_scales(S[C::TJ + i0 + 32 * i + (lane & 31)][which], lane >> 5);
  };
  const auto put = [&](uint2 (*S)[2], uint4 v) {
    S[mine][0] = make_uint2(v.x, v.y), S[mine][1] = make_uint2(v.z, v.w);
  };
  const int stages = (end + BK - 1) / BK;
  request(SJ0, SI0, 0);
  put(scales[0], fetch(0));
  uint4 next = fetch(16);
  int k0 = 0;
  const bool idle = idle_wave<C>(tile);
  if (idle) {  // (as in run_stages)
    for (int n = 1; n < stages; n += 2, k0 += 2 * BK) {
      __syncthreads();
      request(SJ1, SI1, k0 + BK);
      __syncthreads();
      put(scales[((n >> 1) + 1) & 1], next);
      next = fetch((k0 + 4 * BK) / 8);
      request(SJ0, SI0, k0 + 2 * BK);
    }
    if (stages & 1) __syncthreads();
  }
  for (int n = idle ? stages : 1; n < stages; n += 2, k0 += 2 * BK) {
    __syncthreads();  // this stage is there, and everyone is done with the other buffer
    take(scales[(n >> 1) & 1], 0);
    request(SJ1, SI1, k0 + BK);
    __builtin_amdgcn_sched_barrier(0);
    multiply_codes<C>(SJ0, SI0, rj, ri, cj, ci, acc);
    acc.hold();
    __syncthreads();
    take(scales[(n >> 1) & 1], 1);
    put(scales[((n >> 1) + 1) & 1], next);
    next = fetch((k0 + 4 * BK) / 8);
    request(SJ0, SI0, k0 + 2 * BK);  // (behind the end: zeros)
    __builtin_amdgcn_sched_barrier(0);
    multiply_codes<C>(SJ1, SI1, rj, ri, cj, ci, acc);
    acc.hold();
  }
  if (!idle && (stages & 1)) {
    __syncthreads();
    take(scales[(stages >> 1) & 1], 0);
    multiply_codes<C>(SJ0, SI0, rj, ri, cj, ci, acc);
  }
  const E *bias = a.bias ? static_cast<const E *>(a.bias) + (int64_t)tile.expert * a.N : nullptr;
  __syncthreads();
  write_outputs<T, C, (int)sizeof(SJ0)>(
      acc, SJ0, c0, a.N, a.wide, [&](int j) { return tile.begin + j < tile.end ? out + (int64_t)(tile.begin + j) * a.N : nullptr; },
      [&](int i, float (&v)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = activate(v[e] + (bias ? T::load(bias[min(c0 + i + e, a.N - 1)]) : 0.f), a.act);
      },
      NoSlope{});
}

// Few rows (tile_product.hpp): a line of a column is eight blocks, four instructions.
template <class T, bool SHORT>
__global__ __launch_bounds__(64 * THIN_WAVES) void mx4_thin_kernel(Mx4Args a) {
  typedef typename T::store E;
  __shared__ float4 buffer[THIN_WAVES][4][64];
  int ct = 0;
  const RowTile tile = find_row_tile<false>(a.offsets, a.E, a.R, 32, (a.N + 31) / 32, a.first + (int)blockIdx.x, &ct);
  if (tile.expert < 0) return;
  const int lane = threadIdx.x & 63, half = lane >> 5, c0 = 32 * ct;
  E *out = static_cast<E *>(a.y);
  f32x16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  const bool behind = tile.expert == a.E;  // the last group: zeros
  if (!behind) {
    const int64_t wl = (int64_t)tile.expert * a.N + min(c0 + (lane & 31), a.N - 1), xl = min(tile.begin + (lane & 31), tile.end - 1);
    const uint4 *w = reinterpret_cast<const uint4 *>(a.wc) + wl * a.blocks, *x = reinterpret_cast<const uint4 *>(a.xc) + xl * a.blocks;
    const uint8_t *ws = a.ws + wl * a.blocks, *xs = a.xs + xl * a.blocks;
    for (int b1 = 0; b1 < a.blocks; b1 += 8 * THIN_WAVES) {  // (the same count for every wave: behind the end are zeros)
      const int b0 = b1 + 8 * wave_number();
      uint4 vw[4], vx[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int b = b0 + 2 * s + half, at = min(b, a.blocks - 1);
        const uint4 zero = make_uint4(0, 0, 0, 0), lw = w[at], lx = x[at];
        vw[s] = b < a.blocks ? lw : zero, vx[s] = b < a.blocks ? lx : zero;
      }
      const uint32_t sw = own_scales(load_scales<SHORT>(ws, b0, a.blocks), half), sx = own_scales(load_scales<SHORT>(xs, b0, a.blocks), half);
      acc = mfma_mx4_32x32x64<0>(vw[0], sw, vx[0], sx, acc);
      acc = mfma_mx4_32x32x64<1>(vw[1], sw, vx[1], sx, acc);
      acc = mfma_mx4_32x32x64<2>(vw[2], sw, vx[2], sx, acc);
      acc = mfma_mx4_32x32x64<3>(vw[3], sw, vx[3], sx, acc);
    }
  }
  sum_over_waves(acc, buffer, [&](float (&v)[4], int j, int i) {
    const int r = tile.begin + j, c = c0 + i;
    if (r >= tile.end || c >= a.N) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.bias && !behind) v[e] += T::load(static_cast<const E *>(a.bias)[(int64_t)tile.expert * a.N + min(c + e, a.N - 1)]);
      v[e] = behind ? 0.f : activate(v[e], a.act);
    }
    store_quad<T>(out + (int64_t)r * a.N, c, a.N, a.wide, v);
  });
}

typedef Tile<64, 64, 2, 2> Small;
typedef Tile<128, 128, 2, 2> Medium;
typedef Tile<256, 256, 2, 4> Large;

template <class T, class C, bool SHORT>
int launch_mx4(Mx4Args a, hipStream_t s) {
  const int64_t groups = row_tile_workgroups<HALVES<C>>(row_tile_count<HALVES<C>>(a.R, a.E, C::TJ), (a.N + C::TI - 1) / C::TI);
  if (groups > 0x7fffffffLL) return DIMO_E_ARG;
  return for_launches(groups, C::THREADS, [&](int64_t first, unsigned count) {
    a.first = (int)first;
    hipLaunchKernelGGL((mx4_rows_kernel<T, C, SHORT>), dim3(count), dim3(C::THREADS), 0, s, a);
  });
}

// launch(first row, workgroups) for bands of rows whose units (`per_row` to a row, one per thread) a launch can count in
// 31 bits
template <class F>
int for_row_bands(int64_t rows, uint32_t per_row, F &&launch) {
  const int64_t most = (0x7fffffffLL - 255) / per_row;  // (K <= 2^30: at least 15 rows)
  for (int64_t first = 0; first < rows; first += most) {
    const int64_t units = (rows - first < most ? rows - first : most) * per_row;
    launch(first, (unsigned)((units + 255) / 256));
    const int rc = check_launch();
    if (rc) return rc;
  }
  return DIMO_OK;
}

}  // namespace

extern "C" int dimo_mx4_quantize(int dtype, int64_t rows, int K, const void *x, int64_t ldx,
                                 const int32_t *from, uint8_t *codes, uint8_t *scales, void *stream) {
  if (!known_dtype(dtype) || rows < 0 || K < 1 || K > DIMO_MAX_SIZE || ldx < K) return DIMO_E_ARG;
  if (rows == 0) return DIMO_OK;
  if (!x || !codes || !scales || (reinterpret_cast<uintptr_t>(codes) & 3)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_MX4, s);
  QuantArgs a{rows, K, (K + 31) / 32, x, ldx, from, codes, scales, Divide((uint32_t)(4 * ((K + 31) / 32))), 0};
  return for_row_bands(rows, a.per_row.d, [&](int64_t first, unsigned grid) {
    a.first = first;
    with_dtype(dtype, [&](auto tag) {
      typedef decltype(tag) Tag;
      if (aligned16(x) && ldx * (int64_t)dtype_bytes(dtype) % 16 == 0)
        hipLaunchKernelGGL((mx4_quantize_kernel<Tag, true>), dim3(grid), dim3(256), 0, s, a);
      else
        hipLaunchKernelGGL((mx4_quantize_kernel<Tag, false>), dim3(grid), dim3(256), 0, s, a);
    });
  });
}

extern "C" int dimo_mx4_dequantize(int dtype, int64_t rows, int K, const uint8_t *codes, const uint8_t *scales, void *out,
                                   void *stream) {
  if (!known_dtype(dtype) || rows < 0 || K < 1 || K > DIMO_MAX_SIZE) return DIMO_E_ARG;
  if (rows == 0) return DIMO_OK;
  if (!codes || !scales || !out || (reinterpret_cast<uintptr_t>(codes) & 3)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_MX4, s);
  const Divide per_row((uint32_t)(4 * ((K + 31) / 32)));
  return for_row_bands(rows, per_row.d, [&](int64_t first, unsigned grid) {
    with_dtype(dtype, [&](auto tag) {
      typedef decltype(tag) Tag;
      const bool wide = aligned16(out) && K * (int64_t)dtype_bytes(dtype) % 16 == 0;
      hipLaunchKernelGGL((mx4_dequantize_kernel<Tag>), dim3(grid), dim3(256), 0, s, first, rows, K, per_row, codes, scales,
                         static_cast<typename Tag::store *>(out), wide);
    });
  });
}

extern "C" int dimo_mx4_linear(int dtype, int R, int E, int K, int N, const uint8_t *x_codes, const uint8_t *x_scales,
                               const int32_t *offsets, const uint8_t *w_codes, const uint8_t *w_scales, const void *bias,
                               int act, void *y, void *stream) {
  if (!known_dtype(dtype) || R < 0 || R > DIMO_MAX_SIZE || E < 1 || E > DIMO_MAX_EXPERTS || K < 1 || K > DIMO_MAX_SIZE ||
      N < 1 || N > DIMO_MAX_SIZE || act < DIMO_ACT_NONE || act > DIMO_ACT_SILU || (!offsets && E != 1))
    return DIMO_E_ARG;
  if (R == 0) return DIMO_OK;
  if (!x_codes || !x_scales || !w_codes || !w_scales || !y || !aligned16(x_codes) || !aligned16(w_codes)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_MX4, s);
  const bool wide = N % (16 / (int)dtype_bytes(dtype)) == 0 && aligned16(y);
  Mx4Args a{R, E, K, N, (K + 31) / 32, x_codes, x_scales, w_codes, w_scales, offsets, bias, act, wide, y, 0};
  // few rows, as in grouped.hip: 16 experts of 2048 x 2048, 1 / 8 / 16 / 32 / 256 rows: 6.2 / 7.5 / 7.6 / 9.4 / 12 us, the
  // 64 x 64 tile 8.1 / 8.4 / 8.4 / 9.5 / 9.7
  if (R <= 16) {
    const int64_t groups = row_tile_workgroups(row_tile_count(R, E, 32), (N + 31) / 32);
    if (groups > 0x7fffffffLL) return DIMO_E_ARG;
    return for_launches(groups, 64 * THIN_WAVES, [&](int64_t first, unsigned count) {
      a.first = (int)first;
      with_dtype(dtype, [&](auto tag) {
        if (a.blocks < 8)
          hipLaunchKernelGGL((mx4_thin_kernel<decltype(tag), true>), dim3(count), dim3(64 * THIN_WAVES), 0, s, a);
        else
          hipLaunchKernelGGL((mx4_thin_kernel<decltype(tag), false>), dim3(count), dim3(64 * THIN_WAVES), 0, s, a);
      });
    });
  }
  const int64_t per_group = (R + E - 1) / E;
  const int tile = choose_tile(per_group, (R + per_group - 1) / per_group, N, true);
  int rc = DIMO_OK;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) T;
    if (a.blocks < 8)
      rc = tile == SMALL ? launch_mx4<T, Small, true>(a, s) : launch_mx4<T, Medium, true>(a, s);
    else
      rc = tile == LARGE ? launch_mx4<T, Large, false>(a, s) : tile == MEDIUM ? launch_mx4<T, Medium, false>(a, s)
                                                                        : launch_mx4<T, Small, false>(a, s);
  });
  return rc;
}
