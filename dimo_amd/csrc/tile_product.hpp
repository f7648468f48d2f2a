// One output tile of a product on the 16-bit matrix instructions: out[row][col] = sum over the reduction of
// ROW[row][.] COL[col][.], ROW and COL being any mix of
//   LINES    the operand's lines lie along the reduction in memory (x, weights [N, K] of the forward)
//   COLUMNS  its lines lie across it (the weights of dgrad, both operands of wgrad): reduction step r is one row of
//            memory, the tile's lines are neighbours in it
// A workgroup owns TJ x TI outputs, a wave WJ x WI of them as 32 x 32 blocks of v_mfma_f32_32x32x16 with the ROW operand
// in the instruction's j (lane) and the COL operand in its i (register) dimension: a lane then holds four consecutive
// columns of one output row.
//
// A stage is BK steps of the reduction.  In LDS it lies as it lies in memory -- LINES: [line][BK], COLUMNS: [step][TILE]
// --, cut into chunks of 16 bytes whose place inside a row is permuted so that the operand reads (ds_read_b128 for
// LINES, the transposing ds_read_b64_tr_b16 for COLUMNS) spread over all banks (`lines_place`, `columns_place`).
#pragma once
#include "matrix_ops.hpp"
#include "row_tiles.hpp"

#include <type_traits>

namespace dimo {

constexpr bool LINES = true, COLUMNS = false;

// (a scalar: what it leads to stays out of the vector registers)
__device__ __forceinline__ int wave_number() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// a chunk of zeros: what lies behind the end of the reduction is read from here
__device__ const uint4 zero_chunk[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};

// Place (in chunks) of logical chunk c of LDS row `row`; `per_row` chunks in a row.  Eight neighbouring rows' chunk c
// fall on eight different 16-byte columns of the banks, sixteen on sixteen of a bank row twice as wide.
template <int PER_ROW>
__device__ __forceinline__ int lines_place(int row, int c) {
  static_assert(PER_ROW == 8 || PER_ROW == 4, "stages are 64 or 32 deep");
  return PER_ROW == 8 ? c ^ ((row & 7) ^ ((row >> 3) & 1)) : c ^ (((row >> 1) & 3) ^ ((row >> 3) & 1));
}
// ... of a COLUMNS row: a transposing read takes 32 bytes of each of four neighbouring rows per 16 lanes.
template <int PER_ROW>
__device__ __forceinline__ int columns_place(int row, int c) {
  return c ^ (((row & 3) << 1) | (PER_ROW >= 16 ? (row & 1) << 3 : 0));
}

// ---- operand reads -----------------------------------------------------------------------------------------------
// Where in a stage lane l of the matrix instruction finds its eight values of the reduction, for NB blocks of 32 lines: the
// permutation of a lane's row does not change from block to block (LINES) or from step to step (COLUMNS), so a few
// offsets serve all reads, the rest is the instructions' constant offset.
template <bool ORDER, int TILE, int BK, int NB>
struct Reader {
  static constexpr int READS = ORDER == LINES ? 1 : 2;  // instructions per read()
  int at[ORDER == LINES ? BK / 16 : NB];
  __device__ __forceinline__ explicit Reader(int line0) {
    const int lane = threadIdx.x & 63;
    if constexpr (ORDER == LINES) {
      const int row = line0 + (lane & 31);
#pragma unroll
      for (int s = 0; s < BK / 16; ++s) at[s] = row * BK + lines_place<BK / 8>(row, 2 * s + (lane >> 5)) * 8;
    } else {
      // 16 lanes read four steps of 16 lines and get, lane by lane, one line's four steps
      const int g = lane >> 4, j = lane & 15, row = 8 * (g >> 1) + (j >> 2);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int line = line0 + 32 * b + 16 * (g & 1) + 4 * (j & 3);
        at[b] = row * TILE + columns_place<TILE / 8>(row, line >> 3) * 8 + (line & 7);
      }
    }
  }
  // block b, steps 16 s ..+ 15 of the stage
  __device__ __forceinline__ uint4 read(const uint16_t *S, int b, int s) const {
    if constexpr (ORDER == LINES) {
      return *reinterpret_cast<const uint4 *>(S + at[s] + 32 * b * BK);
    } else {
      const uint2 lo = read_transposed(S + at[b] + 16 * s * TILE), hi = read_transposed(S + at[b] + (16 * s + 4) * TILE);
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  }
};

// Which memory row a step of the reduction is (COLUMNS).  AHEAD: finding it takes a load, done a stage early -- behind it the
// operand's own load would wait out two round trips per stage (a weight gradient of 32768 gathered rows, 16 x 4096 x 1024 in
// bf16: 515 us, so 375; of rows in their order 330).
struct SameRow {
  static constexpr bool AHEAD = false;
  __device__ __forceinline__ int operator()(int r) const { return r; }
};
struct SourceRow {
  static constexpr bool AHEAD = true;
  const int32_t *rows;
  __device__ __forceinline__ int load(int r) const { return load_global(rows + r); }
  // (nothing is done with what was loaded before it is needed: it would be waited for)
  __device__ __forceinline__ uint32_t operator()(int, int loaded) const { return max(loaded, 0); }
};

// ---- staging -----------------------------------------------------------------------------------------------------
// A thread brings CHUNKS chunks of 8 elements of an operand per stage.  Chunk q of thread t is number q * THREADS + t of the
// stage in LDS order, so that the 64 lanes of a wave write 1024 consecutive bytes (what a load straight into LDS does).
// For LINES a thread keeps its lines (and their addresses) from stage to stage, for COLUMNS its column.
template <class T, bool ORDER, int TILE, int BK, int THREADS>
struct Staging {
  typedef typename T::store E;
  static constexpr int CHUNKS = TILE * BK / 8 / THREADS;
  static constexpr int PER_ROW = ORDER == LINES ? BK / 8 : TILE / 8;
  static constexpr int ROW_STEP = THREADS / PER_ROW;  // LDS rows between two chunks of a thread
  static_assert(CHUNKS >= 1 && THREADS % PER_ROW == 0, "whole chunks");
  static_assert(ORDER == LINES ? ROW_STEP % 16 == 0 : ROW_STEP % 4 == 0, "a thread's chunks share their permutation");
  const E *base[ORDER == LINES ? CHUNKS : 1];  // LINES: each line's first element of this thread's chunk
  int64_t ld;                                  // COLUMNS: elements between two steps
  int col;                                     // this thread's first element: LINES along the reduction, COLUMNS across
  int limit;                                   // COLUMNS: elements of a row from `col` on that exist (<= 0: none)
  int ahead[ORDER == LINES ? 1 : CHUNKS];      // COLUMNS, rows AHEAD: what row.load() gave for the stage that is loaded next

  static __device__ __forceinline__ int lds_row(int q) { return (int)threadIdx.x / PER_ROW + q * ROW_STEP; }
  // (the permutations are their own inverse: the logical chunk at this thread's place)
  static __device__ __forceinline__ int logical_chunk() {
    const int place = (int)threadIdx.x % PER_ROW;
    if constexpr (ORDER == LINES)
      return lines_place<PER_ROW>((int)threadIdx.x / PER_ROW, place);
    else
      return columns_place<PER_ROW>((int)threadIdx.x / PER_ROW, place);
  }
  // line(i) -> pointer to the first element of line i of the tile (always a readable line)
  template <class F>
  __device__ __forceinline__ void init_lines(F &&line) {
    col = 8 * logical_chunk();
#pragma unroll
    for (int q = 0; q < CHUNKS; ++q) base[q] = line(lds_row(q)) + col;
  }
  // p: the matrix's first element of the tile's first column, `columns` of them exist
  __device__ __forceinline__ void init_columns(const E *p, int64_t ld_, int columns) {
    col = 8 * logical_chunk();
    ld = ld_, limit = columns - col;
    base[0] = p + (limit > 0 ? col : 0);
  }
  // the stage that begins at step k0 is loaded next
  template <class F>
  __device__ __forceinline__ void look_ahead(int k0, int end, F &&row) {
    if constexpr (ORDER == COLUMNS && std::decay_t<F>::AHEAD)
#pragma unroll
      for (int q = 0; q < CHUNKS; ++q) ahead[q] = row.load(min(k0 + lds_row(q), end - 1));
  }
  template <class F>
  __device__ __forceinline__ auto memory_row(int q, int r, F &&row) const {
    if constexpr (std::decay_t<F>::AHEAD)
      return row(r, ahead[q]);
    else
      return row(r);
  }
  // address of chunk q of the stage that begins at step k0 (the reduction ends at `end`), row(r) -> memory row of step r;
  // what lies behind the end comes from the zero chunk
  template <class F>
  __device__ __forceinline__ const E *address(int q, int k0, int end, F &&row) const {
    if constexpr (ORDER == LINES) {
      return k0 + col < end ? base[q] + k0 : reinterpret_cast<const E *>(zero_chunk);
    } else {
      const int r = k0 + lds_row(q);
      const E *p = base[0] + memory_row(q, min(r, end - 1), row) * ld;
      return r < end ? p : reinterpret_cast<const E *>(zero_chunk);
    }
  }
  // straight into LDS (16-bit elements, everything on 16-byte boundaries and the rows' ends too)
  template <class F>
  __device__ __forceinline__ void load_direct(uint16_t *S, int k0, int end, F &&row) const {
#pragma unroll
    for (int q = 0; q < CHUNKS; ++q)
      load_to_lds(address(q, k0, end, row), S + (q * THREADS + 64 * wave_number()) * 8);
  }
  // through registers; whole: chunks are inside or outside as a whole, so that no load needs a branch
  typedef E Chunk[8];
  template <bool WHOLE, class F>
  __device__ __forceinline__ void load(Chunk (&v)[CHUNKS], int k0, int end, F &&row) const {
#pragma unroll
    for (int q = 0; q < CHUNKS; ++q) {
      if constexpr (WHOLE) {
        const char *from = reinterpret_cast<const char *>(address(q, k0, end, row));
        uint4 w[sizeof(Chunk) / 16];
#pragma unroll
        for (int h = 0; h < (int)sizeof(Chunk) / 16; ++h) w[h] = load_global(from + 16 * h);
        __builtin_memcpy(v[q], w, sizeof(Chunk));
        continue;
      }
      const E *p;
      int ok;
      if constexpr (ORDER == LINES) {
        ok = end - k0 - col, p = base[q] + (ok > 0 ? k0 : 0);
      } else {
        const int r = k0 + lds_row(q);
        ok = r < end ? limit : 0, p = base[0] + memory_row(q, min(r, end - 1), row) * ld;
      }
      if (ok >= 8) {
        __builtin_memcpy(v[q], p, sizeof(Chunk));  // (one or two 16-byte loads; the hardware takes any alignment)
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[q][e] = e < ok ? p[e] : E(0);
      }
    }
  }
  // into the planes of LDS (three for fp32, one otherwise), `plane` elements apart
  __device__ __forceinline__ void store(const Chunk (&v)[CHUNKS], uint16_t *S, int plane) const {
#pragma unroll
    for (int q = 0; q < CHUNKS; ++q) {
      uint16_t *dst = S + (q * THREADS + (int)threadIdx.x) * 8;
      if constexpr (sizeof(E) == 4) {
        uint32_t h[4], m[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Split3 a = split3(v[q][2 * e]), b = split3(v[q][2 * e + 1]);
          h[e] = a.hi | (uint32_t)b.hi << 16, m[e] = a.mid | (uint32_t)b.mid << 16, l[e] = a.lo | (uint32_t)b.lo << 16;
        }
        *reinterpret_cast<uint4 *>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4 *>(dst + plane) = make_uint4(m[0], m[1], m[2], m[3]);
        *reinterpret_cast<uint4 *>(dst + 2 * plane) = make_uint4(l[0], l[1], l[2], l[3]);
      } else {
        uint4 w;
        __builtin_memcpy(&w, v[q], 16);
        *reinterpret_cast<uint4 *>(dst) = w;
      }
    }
  }
};

template <class T>
struct Planes {
  static constexpr int N = 1, DEPTH = 64;
  typedef T Tag;
};
template <>
struct Planes<F32> {  // (three planes: half the depth keeps a stage of 128 + 128 lines at 48 KB)
  static constexpr int N = 3, DEPTH = 32;
  typedef BF16 Tag;
};

// TJ rows x TI columns per workgroup, WJ x WI waves.
template <int TJ_, int TI_, int WJ_, int WI_>
struct Tile {
  static constexpr int TJ = TJ_, TI = TI_, WJ = WJ_, WI = WI_, THREADS = 64 * WJ * WI;
  static constexpr int NJ = TJ / WJ / 32, NI = TI / WI / 32;
};

// ---- a wave's share ------------------------------------------------------------------------------------------------
template <int NJ, int NI>
struct Accumulators {
  f32x16 v[NJ][NI];
  float sums[NJ];  // with_sums: the ROW operand's sums along the reduction, this lane's share of line l % 32
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) v[j][i][r] = 0.f;
      sums[j] = 0.f;
    }
  }
  // Ends a stage: the sums are taken to be used here, so the compiler cannot move the stage's matrix instructions (pure to
  // it) behind the next barrier, where their operands would have to wait in registers that are not there.
  __device__ __forceinline__ void hold() {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < NI; ++i) asm volatile("" : "+v"(v[j][i]));
  }
};

// Asks the scheduler for one LDS read behind each matrix instruction while there are any (READS of them for PRODUCTS
// instructions).
template <int READS, int PRODUCTS>
__device__ __forceinline__ void interleave(bool reads) {
#pragma unroll
  for (int p = 0; p < PRODUCTS; ++p) {
    constexpr int EACH = (READS + PRODUCTS - 1) / PRODUCTS;
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (reads && p * EACH < READS) __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
  }
}

// One stage of a wave's 32 NJ x 32 NI outputs: the operands of the next sixteen steps are read while these are multiplied
// (a read between two matrix instructions: issued all at once they would leave the matrix pipe waiting for them).
template <class T, class C, int BK, bool SUMS, class RJ, class RI>
__device__ __forceinline__ void multiply_stage(const uint16_t *SJ, const uint16_t *SI, const RJ &rj, const RI &ri,
                                               Accumulators<C::NJ, C::NI> &acc, bool with_sums) {
  constexpr int P = Planes<T>::N, NJ = C::NJ, NI = C::NI, STEPS = BK / 16;
  typedef typename Planes<T>::Tag Tag;
  uint4 a[2][P][NI], b[2][P][NJ];
  const auto read = [&](int s) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
#pragma unroll
      for (int i = 0; i < NI; ++i) a[s & 1][p][i] = ri.read(SI + p * C::TI * BK, i, s);
#pragma unroll
      for (int j = 0; j < NJ; ++j) b[s & 1][p][j] = rj.read(SJ + p * C::TJ * BK, j, s);
    }
  };
  read(0);
  if constexpr (!SUMS) __builtin_amdgcn_sched_group_barrier(0x100, P * (NI * RI::READS + NJ * RJ::READS), 0);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    if (s + 1 < STEPS) read(s + 1);
#pragma unroll
    for (int d = P - 1; d >= 0; --d)  // (fp32: the smallest products first)
#pragma unroll
      for (int p = 0; p <= d; ++p)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < NI; ++i) acc.v[j][i] = mfma_32x32x16(Tag{}, a[s & 1][p][i], b[s & 1][d - p][j], acc.v[j][i]);
    if constexpr (SUMS)
      if (with_sums) {
#pragma unroll
        for (int p = P - 1; p >= 0; --p)
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const uint4 v = b[s & 1][p][j];
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) acc.sums[j] += Tag::load((uint16_t)w[e]) + Tag::load((uint16_t)(w[e] >> 16));
          }
      }
    if constexpr (!SUMS) interleave<P * (NI * RI::READS + NJ * RJ::READS), NJ * NI * P * (P + 1) / 2>(s + 1 < STEPS);
  }
}

// The LDS of a product's stages: separate arrays, so that the compiler knows that what is on its way into one is not what is
// read from another (it would wait for every load in flight before each read otherwise).
#define DIMO_STAGE_BUFFERS(T, C, HOW)                                                                                          \
  __shared__ __attribute__((aligned(1024))) uint16_t SJ0[Planes<T>::N * C::TJ * Planes<T>::DEPTH],                             \
      SI0[Planes<T>::N * C::TI * Planes<T>::DEPTH], SJ1[HOW == DIRECT ? C::TJ * Planes<T>::DEPTH : 8],                                \
      SI1[HOW == DIRECT ? C::TI * Planes<T>::DEPTH : 8]

// How a stage gets into LDS.  DIRECT (16-bit, everything on 16-byte boundaries): two buffers, the next stage's loads go
// straight into the one while the other is multiplied, one barrier per stage.  WHOLE (fp32 on such boundaries) and ANY: the
// next stages wait in registers, one buffer, two barriers; a 64 x 64 tile has registers for two stages ahead, and needs
// them: its stage is multiplied in a fraction of a load's round trip.
enum Staged { ANY = 0, DIRECT = 1, WHOLE = 2 };

// The stages of a product, one after the other.
template <class T, class C, bool ORDER_J, bool ORDER_I, int HOW, bool SUMS, class RowJ, class RowI>
__device__ __forceinline__ void run_stages(Staging<T, ORDER_J, C::TJ, Planes<T>::DEPTH, C::THREADS> &sj,
                                           Staging<T, ORDER_I, C::TI, Planes<T>::DEPTH, C::THREADS> &si, int begin,
                                           int end, RowJ &&row_j, RowI &&row_i, Accumulators<C::NJ, C::NI> &acc,
                                           bool with_sums, uint16_t *SJ0, uint16_t *SI0, uint16_t *SJ1, uint16_t *SI1,
                                           bool idle = false) {
  constexpr int BK = Planes<T>::DEPTH;
  const int wave = wave_number();
  const Reader<ORDER_J, C::TJ, BK, C::NJ> rj((wave / C::WI) * 32 * C::NJ);
  const Reader<ORDER_I, C::TI, BK, C::NI> ri((wave % C::WI) * 32 * C::NI);
  if constexpr (HOW == DIRECT) {
    const int stages = (end - begin + BK - 1) / BK;
    const auto load = [&](uint16_t *SJ, uint16_t *SI, int k0) {
      sj.load_direct(SJ, k0, end, row_j);
      si.load_direct(SI, k0, end, row_i);
      sj.look_ahead(k0 + BK, end, row_j);
      si.look_ahead(k0 + BK, end, row_i);
    };
    sj.look_ahead(begin, end, row_j);
    si.look_ahead(begin, end, row_i);
    load(SJ0, SI0, begin);
    int k0 = begin;
    if (idle) {  // a wave whose rows are not there: its share of the loads, at the same barriers
      for (int n = 1; n < stages; n += 2, k0 += 2 * BK) {
        __syncthreads();
        load(SJ1, SI1, k0 + BK);
        __syncthreads();
        load(SJ0, SI0, k0 + 2 * BK);
      }
      if (stages & 1) __syncthreads();
      return;
    }
    for (int n = 1; n < stages; n += 2, k0 += 2 * BK) {
      __syncthreads();  // this stage is there, and everyone is done with the other buffer
      load(SJ1, SI1, k0 + BK);
      __builtin_amdgcn_sched_barrier(0);  // (the loads first: they have this stage's products to arrive under)
      multiply_stage<T, C, BK, SUMS>(SJ0, SI0, rj, ri, acc, with_sums);
      acc.hold();
      __syncthreads();
      load(SJ0, SI0, k0 + 2 * BK);  // (behind the end: zeros; a branch would split the stage)
      __builtin_amdgcn_sched_barrier(0);
      multiply_stage<T, C, BK, SUMS>(SJ1, SI1, rj, ri, acc, with_sums);
      acc.hold();
    }
    if (stages & 1) {
      __syncthreads();
      multiply_stage<T, C, BK, SUMS>(SJ0, SI0, rj, ri, acc, with_sums);
    }
  } else {
    typedef Staging<T, ORDER_J, C::TJ, BK, C::THREADS> LJ;
    typedef Staging<T, ORDER_I, C::TI, BK, C::THREADS> LI;
    constexpr int AHEAD = HOW == WHOLE && C::NJ * C::NI == 1 ? 3 : 1;
    typename LJ::Chunk vj[AHEAD][LJ::CHUNKS];
    typename LI::Chunk vi[AHEAD][LI::CHUNKS];
    const auto load = [&](int d, int k0) {
      sj.template load<HOW == WHOLE>(vj[d], k0, end, row_j);
      si.template load<HOW == WHOLE>(vi[d], k0, end, row_i);
      sj.look_ahead(k0 + BK, end, row_j);
      si.look_ahead(k0 + BK, end, row_i);
    };
    sj.look_ahead(begin, end, row_j);
    si.look_ahead(begin, end, row_i);
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) load(d, begin + d * BK);
    for (int k1 = begin; k1 < end; k1 += AHEAD * BK) {
#pragma unroll
      for (int d = 0; d < AHEAD; ++d) {
        const int k0 = k1 + d * BK;
        if (k0 >= end) break;
        __syncthreads();  // everyone is done with the last stage
        sj.store(vj[d], SJ0, C::TJ * BK);
        si.store(vi[d], SI0, C::TI * BK);
        __syncthreads();
        if (HOW == WHOLE || k0 + BK < end) load(d, k0 + AHEAD * BK);
        __builtin_amdgcn_sched_barrier(0);
        multiply_stage<T, C, BK, SUMS>(SJ0, SI0, rj, ri, acc, with_sums);
        acc.hold();
      }
    }
  }
}

// four elements of a row from column c on, `columns` exist
template <class T>
__device__ __forceinline__ void store_quad(typename T::store *row, int c, int columns, bool wide, const float (&v)[4]) {
  typedef typename T::store E;
  if (wide && c + 4 <= columns) {
    if constexpr (sizeof(E) == 4)
      *reinterpret_cast<float4 *>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
    else
      *reinterpret_cast<uint2 *>(row + c) = make_uint2((uint32_t)T::save(v[0]) | (uint32_t)T::save(v[1]) << 16,
                                                       (uint32_t)T::save(v[2]) | (uint32_t)T::save(v[3]) << 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < columns) row[c + e] = T::save(v[e]);
  }
}

// What happens to an output's sum on its way out: nothing, or the multiplication by the slope of an activation whose saved
// values lie `away` elements from the outputs.  The product is rounded once: silu's slope meets the sum in fp32; relu's is 0 or
// 1, which the sum's rounding does not see, so it is multiplied behind it, with half the LDS traffic.  (16 even groups, 32768 x
// 4096 outputs in bf16, reduction 1024: 292 us without a slope, 376 with relu's, 424 with silu's; the saved values alone are 268 MB.)
struct NoSlope {
  static constexpr int ACT = DIMO_ACT_NONE;
};
struct ReluSlope {
  static constexpr int ACT = DIMO_ACT_RELU;
  int64_t away;
};
struct SiluSlope {
  static constexpr int ACT = DIMO_ACT_SILU;
  int64_t away;
};

// Writes a wave's outputs.  A lane holds quads of 32 different rows: written as they are, an instruction would touch 32 lines
// of memory for 16 bytes each (measured: 22 us for a 256 x 256 tile, a third of its time at a reduction of 2048).  So
// blocks of 32 rows go through LDS -- 4 KB of the wave's own, chunks permuted as in a stage -- and leave as whole lines.  They
// lie there in the outputs' type, or, where silu's slope is to come, in fp32.
//   at(row of the tile) -> the output row, or null;  value(quad's column of the tile, its four sums) changes them in place
// The caller has passed a barrier behind the last stage; `buffer` holds 4 KB per wave.
template <class T, class C, int BYTES, class At, class Value, class Out>
__device__ __forceinline__ void write_outputs(const Accumulators<C::NJ, C::NI> &acc, uint16_t *buffer, int first_column,
                                              int columns, bool wide, At &&at, Value &&value, Out slope) {
  typedef typename T::store E;
  typedef std::conditional_t<Out::ACT == DIMO_ACT_SILU, F32, T> Slab;
  typedef typename Slab::store S;
  const int lane = threadIdx.x & 63, wave = wave_number();
  const int j0 = (wave / C::WI) * 32 * C::NJ, i0 = (wave % C::WI) * 32 * C::NI;
  constexpr int ROW_BYTES = (int)sizeof(S) * 32 * C::NI, MOST = C::WJ * C::WI * 32 * 128 <= BYTES ? 128 : 64;
  constexpr int SLAB_ROW = ROW_BYTES < MOST ? ROW_BYTES : MOST;  // bytes of a row that go together
  constexpr int CHUNKS = SLAB_ROW / 16, PER = 16 / (int)sizeof(S), SLABS = ROW_BYTES / SLAB_ROW;
  constexpr int PIECES = (int)(sizeof(S) / sizeof(E)), OUT = PIECES * PER;  // chunks and elements that a lane writes as 16 bytes
  constexpr int LANES = CHUNKS / PIECES;                                    // lanes to a row
  constexpr int EIGHTS = 4 * C::NI / SLABS;  // eights of columns per slab (a quad from each half of the wave)
  static_assert(C::WJ * C::WI * 32 * SLAB_ROW <= BYTES, "4 KB (2 KB) per wave");
  char *own = reinterpret_cast<char *>(buffer) + wave * 32 * SLAB_ROW;
#pragma unroll
  for (int j = 0; j < C::NJ; ++j)
#pragma unroll
    for (int s = 0; s < SLABS; ++s) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int eight = 0; eight < EIGHTS; ++eight) {
        const int in = 8 * eight + 4 * (lane >> 5), b = (s * EIGHTS + eight) / 4, q = (s * EIGHTS + eight) % 4;
        float v[4] = {acc.v[j][b][4 * q], acc.v[j][b][4 * q + 1], acc.v[j][b][4 * q + 2], acc.v[j][b][4 * q + 3]};
        value(i0 + 32 * b + 8 * q + 4 * (lane >> 5), v);
        const int place = (in / PER) ^ (lane & (CHUNKS - 1));  // (in: the column inside the slab)
        store_quad<Slab>(reinterpret_cast<S *>(own + (lane & 31) * SLAB_ROW + 16 * place) + in % PER, 0, 4, true, v);
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r = 0; r < 32; r += 64 / LANES) {
        const int row = r + lane / LANES, piece = lane % LANES;
        S e[OUT];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
          const uint4 v = *reinterpret_cast<const uint4 *>(own + row * SLAB_ROW + 16 * ((piece * PIECES + p) ^ (row & (CHUNKS - 1))));
          __builtin_memcpy(e + p * PER, &v, 16);
        }
        E *dst = at(j0 + 32 * j + row);
        const int c = first_column + i0 + 8 * EIGHTS * s + OUT * piece;
        if (!dst || c >= columns) continue;
        const bool all = wide && c + OUT <= columns;
        if constexpr (Out::ACT != DIMO_ACT_NONE) {
          const E *saved = dst + c + slope.away;
          float at_saved[OUT], f[OUT];
          if (all)
            load_vec<T, OUT>(saved, at_saved);
          else
#pragma unroll
            for (int k = 0; k < OUT; ++k) at_saved[k] = c + k < columns ? T::load(saved[k]) : 0.f;
#pragma unroll
          for (int k = 0; k < OUT; ++k) f[k] = Slab::load(e[k]) * activation_slope(at_saved[k], Out::ACT);
          if (all)
            store_vec<T, OUT>(dst + c, f);
          else
#pragma unroll
            for (int k = 0; k < OUT; ++k)
              if (c + k < columns) dst[c + k] = T::save(f[k]);
        } else if (all) {
          uint4 v;
          __builtin_memcpy(&v, e, 16);
          *reinterpret_cast<uint4 *>(dst + c) = v;
        } else {
#pragma unroll
          for (int k = 0; k < OUT; ++k)
            if (c + k < columns) dst[c + k] = e[k];
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // (block by block: all of them at once would not fit the registers)
    }
}

// ---- few rows ------------------------------------------------------------------------------------------------------
// A product of a handful of rows reads weights and does little else.  32 rows x 32 columns per workgroup: its THIN_WAVES
// waves take the reduction in turn, a line (128 bytes) of every column at a time, straight from memory into the matrix
// instruction's registers -- nothing is used twice, so nothing goes through LDS --, and add up their sums at the end.
constexpr int THIN_WAVES = 8;

// f(quad's sums, row of the tile, first of its four columns) for the workgroup's sums over its waves; `buffer`: 4 KB a wave
template <class F>
__device__ __forceinline__ void sum_over_waves(const f32x16 &acc, float4 (*buffer)[4][64], F &&f) {
  const int lane = threadIdx.x & 63, wave = wave_number();
#pragma unroll
  for (int q = 0; q < 4; ++q) buffer[wave][q][lane] = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
  __syncthreads();
  const int t = threadIdx.x;
  if (t >= 256) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < THIN_WAVES; ++w) {
    const float4 s = buffer[w][t >> 6][t & 63];
    v[0] += s.x, v[1] += s.y, v[2] += s.z, v[3] += s.w;
  }
  f(v, t & 31, 8 * (t >> 6) + 4 * ((t >> 5) & 1));
}

// 256 rows: the last tiles are halves (row_tiles.hpp), in which half of the waves have no rows
template <class C>
constexpr bool HALVES = C::TJ == 256;
template <class C>
__device__ __forceinline__ bool idle_wave(const RowTile &t) {
  return HALVES<C> && (wave_number() / C::WI) * 32 * C::NJ >= t.end - t.begin;
}

// Which tile: its size pays where there are enough of them.  Forward on 64 / 128 / 256 tiles, us (rows, groups, N x K; the
// gradient of x is within a few per cent):
//                                 bf16                              fp32
//   65536, 32, 2048 x 1024        538 / 373 / 307
//   16384,  8, 1024 x 1024        61 / 46 / 40, uneven 67 / 55 / 54   255 / 183, uneven 262 / 234
//   16384, 64, 1024 x 1024        uneven 76 / 62 / 59                 uneven 288 / 253
//    8192, 64,  512 x 512         uneven 19 / 17 / 22                 uneven 48 / 46
//    4096,  8,  512 x 2048        19 / 24 / 50                        73 / 112
//    2048, 16, 1024 x 1024        uneven 15 / 17 / 29                 uneven 52 / 61
enum { SMALL = 0, MEDIUM = 1, LARGE = 2 };
inline int choose_tile(int64_t rows_per_group, int64_t groups, int64_t columns, bool direct) {
  const auto blocks = [&](int64_t t) { return groups * ((rows_per_group + t - 1) / t) * ((columns + t - 1) / t); };
  if (direct && rows_per_group >= 192 && columns >= 192 && blocks(256) >= 224) return LARGE;
  if (rows_per_group >= 48 && columns >= 96 && blocks(128) >= 256) return MEDIUM;
  return SMALL;
}

}  // namespace dimo
