// Microscaled 4-bit floating point: blocks of 32 values along a row share one power-of-two scale (a byte, 2^(byte - 127);
// 255 = NaN), elements are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, low four bits first.
//   quantise   scale = 2^(floor(log2 max|x|) - 2), element = x / scale to the nearest e2m1 value, ties to the even code,
//              beyond 6 to 6; a block with an infinite or NaN value becomes NaN as a whole
//   product    y_rn = act(sum_k x_rk w_e,nk + b_e,n), rows in groups as in grouped.hip, on the matrix cores' scaled
//              4-bit instruction: products of elements and scales are exact, sums are fp32.
// The rounding to 4 bits is the only loss, and it happens in `quantise`, where the caller asked for it.
#include <hip/hip_runtime.h>

#include "matrix_ops.hpp"
#include "row_tiles.hpp"

using namespace dimo;

namespace {

// |v| as a scaled magnitude -> e2m1 code: the number of rounding borders below it; a border itself goes to the even code
__device__ __forceinline__ uint32_t e2m1_code(float a) {
  return (uint32_t)(a > 0.25f) + (uint32_t)(a >= 0.75f) + (uint32_t)(a > 1.25f) + (uint32_t)(a >= 1.75f) +
         (uint32_t)(a > 2.5f) + (uint32_t)(a >= 3.5f) + (uint32_t)(a > 5.0f);
}
__device__ __forceinline__ float e2m1_value(uint32_t code) {
  const uint32_t m = code & 7u;
  const float v = m < 2u ? 0.5f * (float)m : (1.f + 0.5f * (float)(m & 1u)) * (float)(1u << ((m >> 1) - 1u));
  return (code & 8u) ? -v : v;
}
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x00400000u : byte == 255u ? 0x7fc00000u : byte << 23);
}

// Four lanes per block, eight values each: 16 bytes of 16-bit input (32 of fp32) and 4 bytes of codes per lane, so a
// wave reads and writes whole lines; the block's largest magnitude takes two exchanges.
struct QuantArgs {
  int64_t rows;
  int K, blocks, places;   // blocks of 32 per row; places > 0: row r is order[r] / places of x (-1: zeros)
  const void *x;
  int64_t ldx;
  const int32_t *order;
  uint8_t *codes, *scales; // [rows, 16 blocks], [rows, blocks]
};
template <class T, bool WIDE>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(QuantArgs a) {
  typedef typename T::store E;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t total = a.rows * a.blocks * 4;
  const bool in = i < total;
  const int64_t row = in ? i / (4 * a.blocks) : 0;
  const int col = in ? 8 * (int)(i % (4 * a.blocks)) : 0;
  int64_t src = row;
  if (a.places > 0) {
    const int32_t o = in ? a.order[row] : -1;
    src = o < 0 ? -1 : o / a.places;
  }
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
  big = max(big, (uint32_t)__shfl_xor((int)big, 1));
  big = max(big, (uint32_t)__shfl_xor((int)big, 2));
  const uint32_t exponent = big >> 23;
  const uint32_t byte = exponent == 255u ? 255u : exponent > 2u ? exponent - 2u : 0u;
  const float inverse = __uint_as_float((254u - min(byte, 253u)) << 23);  // 2^(127 - byte); byte <= 252 for numbers
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t u = __float_as_uint(v[e]);
    word |= (e2m1_code(fabsf(v[e]) * inverse) | (u >> 31 << 3)) << (4 * e);
  }
  if (!in) return;
  reinterpret_cast<uint32_t *>(a.codes)[i] = word;
  if ((i & 3) == 0) a.scales[i >> 2] = (uint8_t)byte;
}

// Values of the codes, eight per thread.
template <class T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(int64_t rows, int K, int blocks, const uint8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales, typename T::store *__restrict__ out,
                                                             bool wide) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * blocks * 4) return;
  const int64_t row = i / (4 * blocks);
  const int col = 8 * (int)(i % (4 * blocks));
  const uint32_t word = reinterpret_cast<const uint32_t *>(codes)[i];
  const float scale = e8m0_value(scales[i >> 2]);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e2m1_value(word >> (4 * e)) * scale;
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

// ---- the product, general form: 64 x 64 outputs per workgroup, 32 x 32 per wave, operands straight from memory (16
// bytes of codes per lane are exactly one block of 32) ---------------------------------------------------------------
struct Mx4Args {
  int R, E, K, N, blocks;
  const uint8_t *xc, *xs, *wc, *ws;
  const int32_t *offsets;  // null: one group of all rows
  const void *bias;
  int act;
  void *y;
};

template <class T>
__global__ __launch_bounds__(256) void mx4_rows_general_kernel(Mx4Args a) {
  typedef typename T::store E;
  int ct = 0;
  const RowTile tile = find_row_tile(a.offsets, a.E, a.R, 64, (a.N + 63) / 64, (int)blockIdx.x, &ct);
  if (tile.expert < 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int n0 = ct * 64 + (wave & 1) * 32, r0 = tile.begin + (wave >> 1) * 32;
  E *out = static_cast<E *>(a.y);
  const int n = n0 + (lane & 31);
  if (tile.expert == a.E) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int row = r0 + 2 * i + half;
      if (row < tile.end && n < a.N) out[(int64_t)row * a.N + n] = E(0);
    }
    return;
  }
  const int64_t xr = min(r0 + (lane & 31), tile.end - 1), wr = (int64_t)tile.expert * a.N + min(n, a.N - 1);
  const uint4 *xc = reinterpret_cast<const uint4 *>(a.xc) + xr * a.blocks, *wc = reinterpret_cast<const uint4 *>(a.wc) + wr * a.blocks;
  const uint8_t *xs = a.xs + xr * a.blocks, *ws = a.ws + wr * a.blocks;
  f32x16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int b0 = 0; b0 < a.blocks; b0 += 2) {
    const int b = min(b0 + half, a.blocks - 1);
    const bool in = b0 + half < a.blocks;
    uint4 x = xc[b], w = wc[b];
    const int sx = xs[b], sw = ws[b];
    if (!in) x = make_uint4(0, 0, 0, 0), w = x;  // (both zero under the scales of the last block, a NaN scale among them)
    acc = mfma_mx4_32x32x64(x, sx, w, sw, acc);
  }
  if (n >= a.N) return;
  const float bias = a.bias ? T::load(static_cast<const E *>(a.bias)[(int64_t)tile.expert * a.N + n]) : 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = r0 + 8 * (i >> 2) + 4 * half + (i & 3);
    if (row < tile.end) out[(int64_t)row * a.N + n] = T::save(activate(acc[i] + bias, a.act));
  }
}

}  // namespace

extern "C" int dimo_mx4_quantize(int dtype, int64_t rows, int K, const void *x, int64_t ldx, int places,
                                 const int32_t *order, uint8_t *codes, uint8_t *scales, void *stream) {
  if (!known_dtype(dtype) || rows < 0 || K < 1 || ldx < K || places < 0) return DIMO_E_ARG;
  if (rows == 0) return DIMO_OK;
  if (!x || !codes || !scales || (places > 0 && !order) || (reinterpret_cast<uintptr_t>(codes) & 3)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_MX4, s);
  const QuantArgs a{rows, K, (K + 31) / 32, places, x, ldx, order, codes, scales};
  const int64_t grid = (rows * a.blocks * 4 + 255) / 256;
  if (grid > 0x7fffffffLL) return DIMO_E_ARG;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) Tag;
    if (aligned16(x) && ldx * (int64_t)dtype_bytes(dtype) % 16 == 0)
      hipLaunchKernelGGL((mx4_quantize_kernel<Tag, true>), dim3((unsigned)grid), dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((mx4_quantize_kernel<Tag, false>), dim3((unsigned)grid), dim3(256), 0, s, a);
  });
  return check_launch();
}

extern "C" int dimo_mx4_dequantize(int dtype, int64_t rows, int K, const uint8_t *codes, const uint8_t *scales, void *out,
                                   void *stream) {
  if (!known_dtype(dtype) || rows < 0 || K < 1) return DIMO_E_ARG;
  if (rows == 0) return DIMO_OK;
  if (!codes || !scales || !out || (reinterpret_cast<uintptr_t>(codes) & 3)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_MX4, s);
  const int blocks = (K + 31) / 32;
  const int64_t grid = (rows * blocks * 4 + 255) / 256;
  if (grid > 0x7fffffffLL) return DIMO_E_ARG;
  with_dtype(dtype, [&](auto tag) {
    typedef decltype(tag) Tag;
    const bool wide = aligned16(out) && K * (int64_t)dtype_bytes(dtype) % 16 == 0;
    hipLaunchKernelGGL((mx4_dequantize_kernel<Tag>), dim3((unsigned)grid), dim3(256), 0, s, rows, K, blocks, codes, scales,
                       static_cast<typename Tag::store *>(out), wide);
  });
  return check_launch();
}

extern "C" int dimo_mx4_linear(int dtype, int R, int E, int K, int N, const uint8_t *x_codes, const uint8_t *x_scales,
                               const int32_t *offsets, const uint8_t *w_codes, const uint8_t *w_scales, const void *bias,
                               int act, void *y, void *stream) {
  if (!known_dtype(dtype) || R < 0 || E < 1 || E > DIMO_MAX_EXPERTS || K < 1 || N < 1 || act < DIMO_ACT_NONE ||
      act > DIMO_ACT_SILU || (!offsets && E != 1))
    return DIMO_E_ARG;
  if (R == 0) return DIMO_OK;
  if (!x_codes || !x_scales || !w_codes || !w_scales || !y || !aligned16(x_codes) || !aligned16(w_codes)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_MX4, s);
  const Mx4Args a{R, E, K, N, (K + 31) / 32, x_codes, x_scales, w_codes, w_scales, offsets, bias, act, y};
  const int64_t grid = row_tile_workgroups(row_tile_count(R, E, 64), (N + 63) / 64);
  if (grid > 0x7fffffffLL) return DIMO_E_ARG;
  with_dtype(dtype, [&](auto tag) {
    hipLaunchKernelGGL((mx4_rows_general_kernel<decltype(tag)>), dim3((unsigned)grid), dim3(256), 0, s, a);
  });
  return check_launch();
}
