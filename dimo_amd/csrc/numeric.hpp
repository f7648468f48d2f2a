// Element types of the expert operators (fp32, bf16, fp16): conversions between the stored form and fp32.
#pragma once
#include "common.hpp"

namespace dimo {

// A type's tag: `store` is what an element is in memory.  Every conversion to 16 bits rounds to nearest, ties to even
// (half a step: 2^-8 relative in bf16, 2^-11 in fp16), and happens once, when a kernel writes its result.
struct F32 {
  typedef float store;
  static __device__ __forceinline__ float load(float v) { return v; }
  static __device__ __forceinline__ float save(float v) { return v; }
};
struct BF16 {
  typedef uint16_t store;
  static __device__ __forceinline__ float load(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t save(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
struct F16 {
  typedef uint16_t store;
  static __device__ __forceinline__ float load(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t save(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

inline bool known_dtype(int dtype) { return dtype == DIMO_F32 || dtype == DIMO_BF16 || dtype == DIMO_F16; }
inline size_t dtype_bytes(int dtype) { return dtype == DIMO_F32 ? 4 : 2; }

// calls f(tag) with the tag of `dtype`
template <class F>
inline void with_dtype(int dtype, F &&f) {
  if (dtype == DIMO_F32)
    f(F32{});
  else if (dtype == DIMO_BF16)
    f(BF16{});
  else
    f(F16{});
}

// 16 / sizeof(element) consecutive elements as fp32
template <class T>
struct Vec16 {
  static constexpr int N = 16 / (int)sizeof(typename T::store);
  uint4 raw;
  __device__ __forceinline__ void get(float (&v)[N]) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (N == 4)
        v[i] = __builtin_bit_cast(float, w[i % 4]);
      else
        v[i] = T::load((typename T::store)(w[(i / 2) % 4] >> (16 * (i & 1))));
    }
  }
  __device__ __forceinline__ void put(const float (&v)[N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (N == 4)
        w[i] = __builtin_bit_cast(uint32_t, v[i % N]);
      else
        w[i] = (uint32_t)bits16(v[(2 * i) % N]) | ((uint32_t)bits16(v[(2 * i + 1) % N]) << 16);
    }
    raw = make_uint4(w[0], w[1], w[2], w[3]);
  }

 private:
  static __device__ __forceinline__ uint16_t bits16(float v) { return (uint16_t)T::save(v); }
};

// Division of 0 <= n < 2^31 by a number the host knows: a multiplication instead of the ~20 (32-bit) or ~60 (64-bit)
// instructions of a division.  q = n * ceil(2^(31 + l) / d) >> (31 + l) with l = ceil(log2 d) is exact there.
struct Divide {
  uint32_t d, m, s;
  Divide() = default;
  explicit Divide(uint32_t by) : d(by), m(0), s(0) {
    uint32_t l = 0;
    while ((1ull << l) < by) ++l;
    if (l) m = (uint32_t)(((1ull << (31 + l)) + by - 1) / by), s = l - 1;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return m ? __umulhi(n, m) >> s : n; }
};

// VEC consecutive elements: one, or sixteen bytes at a sixteen-byte boundary
template <class T, int VEC>
__device__ __forceinline__ void load_vec(const typename T::store *src, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = T::load(*src);
  } else {
    Vec16<T> q;
    q.raw = *reinterpret_cast<const uint4 *>(src);
    q.get(v);
  }
}
template <class T, int VEC>
__device__ __forceinline__ void store_vec(typename T::store *dst, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    *dst = T::save(v[0]);
  } else {
    Vec16<T> q;
    q.put(v);
    *reinterpret_cast<uint4 *>(dst) = q.raw;
  }
}

// A launch takes fewer than 2^32 threads: launch(first, count) for `total` workgroups of `threads`, as many at a time as fit
// (a multiple of eight, so that every band begins on the first XCD).
inline int64_t launch_groups(int threads) { return 0xffffffffLL / threads / 8 * 8; }
template <class F>
inline int for_launches(int64_t total, int threads, F &&launch) {
  const int64_t most = launch_groups(threads);
  for (int64_t first = 0; first < total; first += most) {
    launch(first, (unsigned)(total - first < most ? total - first : most));
    const int rc = check_launch();
    if (rc) return rc;
  }
  return DIMO_OK;
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// (relu keeps a NaN)
__device__ __forceinline__ float activate(float v, int act) {
  if (act == DIMO_ACT_RELU) return v > 0.f ? v : (v != v ? v : 0.f);
  if (act == DIMO_ACT_SILU) return v / (1.f + expf(-v));
  return v;
}

// slope of an activation: from its output for relu (positive exactly where its input is), from its input for silu
__device__ __forceinline__ float activation_slope(float s, int act) {
  if (act == DIMO_ACT_RELU) return s > 0.f ? 1.f : (s != s ? s : 0.f);
  const float q = 1.f / (1.f + expf(-s));
  return q * (1.f + s * (1.f - q));
}

}  // namespace dimo
