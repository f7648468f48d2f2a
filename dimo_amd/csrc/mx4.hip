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
  int K, blocks;           // blocks of 32 per row
  const void *x;
  int64_t ldx;
  const int32_t *from;     // x's row of row r (negative: zeros), or null
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
  const RowTile tile = find_row_tile(a.offsets, a.E, a.R, C::TJ, (a.N + C::TI - 1) / C::TI, (int)blockIdx.x, &ct);
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
  // a thread brings one line's scales, two stages of them at a time, into LDS (each wave reading those of its lines from
  // memory took three times the requests of the codes themselves)
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
  const auto same = [](int r) { return (int64_t)r; };
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
  for (int n = 1; n < stages; n += 2, k0 += 2 * BK) {
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
  if (stages & 1) {
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

typedef Tile<64, 64, 2, 2> Small;
typedef Tile<128, 128, 2, 2> Medium;
typedef Tile<256, 256, 2, 4> Large;

template <class T, class C, bool SHORT>
int launch_mx4(const Mx4Args &a, hipStream_t s) {
  const int64_t groups = row_tile_workgroups(row_tile_count(a.R, a.E, C::TJ), (a.N + C::TI - 1) / C::TI);
  if (groups > 0x7fffffffLL) return DIMO_E_ARG;
  hipLaunchKernelGGL((mx4_rows_kernel<T, C, SHORT>), dim3((unsigned)groups), dim3(C::THREADS), 0, s, a);
  return check_launch();
}

}  // namespace

extern "C" int dimo_mx4_quantize(int dtype, int64_t rows, int K, const void *x, int64_t ldx,
                                 const int32_t *from, uint8_t *codes, uint8_t *scales, void *stream) {
  if (!known_dtype(dtype) || rows < 0 || K < 1 || ldx < K) return DIMO_E_ARG;
  if (rows == 0) return DIMO_OK;
  if (!x || !codes || !scales || (reinterpret_cast<uintptr_t>(codes) & 3)) return DIMO_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  clear_errors();
  ScopedTimer timer(T_MX4, s);
  const QuantArgs a{rows, K, (K + 31) / 32, x, ldx, from, codes, scales};
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
  const bool wide = N % (16 / (int)dtype_bytes(dtype)) == 0 && aligned16(y);
  const Mx4Args a{R, E, K, N, (K + 31) / 32, x_codes, x_scales, w_codes, w_scales, offsets, bias, act, wide, y};
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
