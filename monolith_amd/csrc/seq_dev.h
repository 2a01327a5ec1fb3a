// Device parts that the attention kernels (attention.hip) and the softmax cross entropy
// (softmax_ce.hip) share (gfx950 only).
//
// All of them are one scheme. A workgroup keeps a tile of rows X ("columns" of the products) in
// registers as B operands and streams rows Y through LDS. A 32x32 matrix instruction gives
// S[y][x] = Y X^T with x = lane & 31 and y = tile_row(r, lane) in accumulator r, so whatever
// belongs to a column (softmax maximum and sum, label, limit) is one register of a lane, and the
// weights P = f(S) lie in the lanes exactly as the B operand of the second product
// Z^T P = sum over y of Z[y][d] P[y][x] wants them, up to an order of the summation index y that
// the A operand Z^T follows: P never goes through LDS. Z^T comes out of the row-major LDS tile by
// the transposing LDS read.
#ifndef MONO_SEQ_DEV_H_
#define MONO_SEQ_DEV_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mono {
namespace seq {

typedef __bf16 bf16;
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef bf16 bf8 __attribute__((ext_vector_type(8)));
typedef bf16 bf4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float neg_inf() { return -__builtin_inff(); }

// x of the lane with the other bit 5 (16) or 4 of its number, and both values in every lane: the lane
// swaps and row permutations of the vector unit, not the LDS permutation that __shfl_xor takes
__device__ inline float swap32(float x, float* other) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  *other = __uint_as_float(p[1]);
  return __uint_as_float(p[0]);
}
__device__ inline float swap16(float x, float* other) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  *other = __uint_as_float(p[1]);
  return __uint_as_float(p[0]);
}
template <int CTRL>
__device__ inline float dpp(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}
struct Sum {
  static __device__ inline float of(float a, float b) { return a + b; }
};
struct Max {
  static __device__ inline float of(float a, float b) { return fmaxf(a, b); }
};
// Op over groups of lanes, the result in every lane: over lanes FROM apart and more, up to TO lanes.
// From 1 on the partners hold equal values by the time that halves and rows are mirrored; lanes that
// stay apart need the exact partner.
template <int FROM, int TO, typename Op>
__device__ inline float over_lanes(float x) {
  float y;
  if constexpr (FROM <= 1 && TO > 1) x = Op::of(x, dpp<0xB1>(x));
  if constexpr (FROM <= 2 && TO > 2) x = Op::of(x, dpp<0x4E>(x));
  if constexpr (FROM <= 4 && TO > 4) x = Op::of(x, FROM > 1 ? __shfl_xor(x, 4) : dpp<0x141>(x));
  if constexpr (FROM <= 8 && TO > 8) x = Op::of(x, FROM > 1 ? dpp<0x128>(x) : dpp<0x140>(x));
  if constexpr (FROM <= 16 && TO > 16) {
    x = swap16(x, &y);
    x = Op::of(x, y);
  }
  if constexpr (FROM <= 32 && TO > 32) {
    x = swap32(x, &y);
    x = Op::of(x, y);
  }
  return x;
}
// over the two lanes that hold one column
__device__ inline float col_max(float x) { return over_lanes<32, 64, Max>(x); }
__device__ inline float col_sum(float x) { return over_lanes<32, 64, Sum>(x); }

// Where a row of D elements starts, and how it may be read: `vec` rows start on 16 bytes and hold
// whole 16-byte chunks.
template <typename T>
__device__ inline u4 load_chunk(const T* row, int e0, int D, bool vec) {
  constexpr int E = 16 / sizeof(T);
  u4 out = {0u, 0u, 0u, 0u};
  if (e0 >= D) return out;
  if (vec) return *(const u4*)(row + e0);
  T tmp[E];
#pragma unroll
  for (int i = 0; i < E; ++i) tmp[i] = e0 + i < D ? row[e0 + i] : (T)0.0f;
  __builtin_memcpy(&out, tmp, 16);
  return out;
}

// A rows array as the tile loads see it.
template <typename T>
struct Rows {
  const T* base;    // first row
  int64_t stride;   // elements from row to row
  int D;
  bool vec;         // rows start on 16 bytes and are whole 16-byte chunks
};

// fp32 rows go through the bf16 matrix instructions as three bf16 numbers each, x = hi + mid + lo, every
// one the rounded rest of those before: 24 bits, as many as x has. Of the nine products of two such
// sums six are taken (hi hi, hi mid, mid hi, mid mid, hi lo, lo hi), at 6/16 of the fp32 matrix instructions'
// time. The three left out are 2^-27.4 of a product in the mean square of normal numbers, a tenth of one fp32
// rounding, and 2^-23 at worst: mid is up to 2^-8 of x and lo 2^-16, both at once in 1 + 2^-8 + 2^-16. (An
// infinite element gives NaN. Rows are split with LARGE: a number within 2^-9 of the largest would round to an
// infinite hi.)
template <typename T>
constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;

template <bool LARGE = false>
__device__ inline void split3(const float* x, int n, bf16* hi, bf16* mid, bf16* lo) {
  constexpr float kMost = 0x1.fep127f;  // the largest bf16
#pragma unroll
  for (int i = 0; i < n; ++i) {
    hi[i] = (bf16)(LARGE ? __builtin_amdgcn_fmed3f(x[i], -kMost, kMost) : x[i]);
    const float r = x[i] - (float)hi[i];
    mid[i] = (bf16)r;
    lo[i] = (bf16)(r - (float)mid[i]);
  }
}

// A tile of BN rows on its way from global memory to LDS: load() takes the thread's chunks into
// registers, store() writes them, one plane of bf16 behind the other. Rows outside [0, n) and rows whose
// word(row) is `dead` become zeros, so that nothing that lies in such a row reaches a product. word() is a
// plain load that nothing but store() looks at: a comparison in load() would wait for the rows there.
template <typename T, int DP, int BN, int NT>
struct Stage {
  static constexpr int E = 16 / sizeof(T);   // elements of a chunk
  static constexpr int CH = DP / E;          // chunks of a row
  static constexpr int PER = (BN * CH + NT - 1) / NT;
  static constexpr int STEP = NT / CH;       // rows between a thread's chunks
  static constexpr int LDW = DP + 8;         // LDS row: 16 bytes of padding against bank conflicts
  // (16 more elements: the transposing read of rows of 16 takes 32 columns, of which it uses 16)
  static constexpr int PLANE = BN * LDW + (DP < 32 ? 16 : 0), LDS = kPlanes<T> * PLANE;
  static_assert(NT % CH == 0 && (PER == 1 || BN * CH % NT == 0), "every thread holds one column of chunks");
  u4 r[PER];
  uint32_t words[PER];

  template <typename Word>
  __device__ inline void load(const Rows<T>& x, int row0, int n, int tid, bool filter, Word word) {
    const int row = row0 + tid / CH, e0 = tid % CH * E;
    const bool mine = (PER > 1 || tid < BN * CH) && e0 < x.D;
    const T* p = x.base + (int64_t)row * x.stride + e0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      r[i] = u4{0u, 0u, 0u, 0u};
      words[i] = 0;  // (such a row is zeros already)
    }
    if (x.vec && row0 + BN <= n) {
      if (mine)
#pragma unroll
        for (int i = 0; i < PER; ++i) r[i] = *(const u4*)(p + i * (STEP * x.stride));
    } else if (x.vec) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (mine && row + i * STEP < n) r[i] = *(const u4*)(p + i * (STEP * x.stride));
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (mine && row + i * STEP < n) r[i] = load_chunk(p + i * (STEP * x.stride) - e0, e0, x.D, false);
    }
    if (filter)
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (mine && row + i * STEP < n) words[i] = word(row + i * STEP);
  }
  __device__ inline void store(bf16* lds, int tid, bool filter, uint32_t dead) const {
    if (PER > 1 || tid < BN * CH) {
      bf16* p = lds + tid / CH * LDW + tid % CH * E;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const u4 w = filter && words[i] == dead ? u4{0u, 0u, 0u, 0u} : r[i];
        bf16* to = p + i * STEP * LDW;
        if constexpr (sizeof(T) == 2) {
          *(u4*)to = w;
        } else {
          const f4 x = __builtin_bit_cast(f4, w);
          const float v[4] = {x[0], x[1], x[2], x[3]};
          bf16 h[4], m[4], l[4];
          split3<true>(v, 4, h, m, l);
          *(bf4*)to = bf4{h[0], h[1], h[2], h[3]};
          *(bf4*)(to + PLANE) = bf4{m[0], m[1], m[2], m[3]};
          *(bf4*)(to + 2 * PLANE) = bf4{l[0], l[1], l[2], l[3]};
        }
      }
    }
  }
  // zeros in the place of a thread's chunks of the rows that are dead(row of the tile)
  template <typename Dead>
  static __device__ inline void clear(bf16* lds, int tid, Dead dead) {
    if (PER > 1 || tid < BN * CH)
      for (int i = 0; i < PER; ++i) {
        const int row = tid / CH + i * STEP;
        if (dead(row))
          for (int j = 0; j < kPlanes<T>; ++j) {
            bf16* to = lds + row * LDW + tid % CH * E + j * PLANE;
            if constexpr (sizeof(T) == 2) *(u4*)to = u4{0u, 0u, 0u, 0u};
            else *(uint64_t*)to = 0;
          }
      }
  }
};

// The 32x32 matrix instructions: a C tile gives lane l column l & 31 and, in register r, row
// tile_row(r, l). They are taken in place of the 16x16 ones of the same rate because every matrix
// instruction keeps the vector unit, which bounds these kernels, from issuing for a few cycles: on one
// SIMD with four waves 16 exponentials and 8 16x16x32 take 203 cycles, with 4 32x32x16 171.
__device__ inline int tile_row(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

// a row statistic (one float per row of a 32-row tile, in LDS) in the place of every C register
__device__ inline f16v by_rows(const float* x, int lane) {
  f16v v;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const f4 t = *(const f4*)(x + 8 * q + 4 * (lane >> 5));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[4 * q + i] = t[i];
  }
  return v;
}
__device__ inline f16v all_of(float x) {
  f16v v;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = x;
  return v;
}

// 32x32x16: the operands' 8 elements of a lane are k = 8 * (lane >> 5) + j.
template <typename T, int DP, int PLANE>
struct Mma {
  static constexpr int PL = kPlanes<T>, KF = DP / 16, NDT = (DP + 31) / 32, LDW = DP + 8;
  struct Frag {
    bf8 p[PL];
  };
  static __device__ inline f16v product(const Frag& a, const Frag& b, f16v c) {
#pragma unroll
    for (int i = PL - 1; i >= 0; --i)  // the small ones first
#pragma unroll
      for (int j = 0; j < PL; ++j)
        if (i + j < PL) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[i], b.p[j], c, 0, 0, 0);
    return c;
  }
  // s[c] = from + rows 32 rt .. of the tile times the columns' rows
  template <int NC>
  static __device__ inline void scores(const bf16* lds, int rt, const Frag (&x)[NC][KF], f16v (&s)[NC],
                                       f16v from, int lane) {
#pragma unroll
    for (int c = 0; c < NC; ++c) s[c] = from;
    const bf16* p = lds + (rt * 32 + (lane & 31)) * LDW + 8 * (lane >> 5);
#pragma unroll
    for (int k = 0; k < KF; ++k) {
      Frag a;
#pragma unroll
      for (int i = 0; i < PL; ++i) a.p[i] = *(const bf8*)(p + i * PLANE + 16 * k);
#pragma unroll
      for (int c = 0; c < NC; ++c) s[c] = product(a, x[c][k], s[c]);
    }
  }
  static __device__ inline void load_cols(Frag (&f)[KF], const T* row, bool ok, int D, bool vec, int lane) {
#pragma unroll
    for (int k = 0; k < KF; ++k) {
      const int e0 = 16 * k + 8 * (lane >> 5);
      u4 c[2] = {{0u, 0u, 0u, 0u}, {0u, 0u, 0u, 0u}};
      if (ok) c[0] = load_chunk(row, e0, D, vec);
      if constexpr (PL == 1) {
        f[k].p[0] = __builtin_bit_cast(bf8, c[0]);
      } else {
        if (ok) c[1] = load_chunk(row, e0 + 4, D, vec);
        const f4 x = __builtin_bit_cast(f4, c[0]), y = __builtin_bit_cast(f4, c[1]);
        const float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
        f[k] = frag<true>(v);
      }
    }
  }
  template <bool LARGE = false>
  static __device__ inline Frag frag(const float* v) {
    Frag f;
    if constexpr (PL == 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f.p[0][j] = (bf16)v[j];
    } else {
      bf16 h[8], m[8], l[8];
      split3<LARGE>(v, 8, h, m, l);
#pragma unroll
      for (int j = 0; j < 8; ++j) f.p[0][j] = h[j], f.p[1][j] = m[j], f.p[2][j] = l[j];
    }
    return f;
  }
  static __device__ inline float whole(const Frag& f, int j) {
    float t = (float)f.p[0][j];
#pragma unroll
    for (int i = 1; i < PL; ++i) t += (float)f.p[i][j];
    return t;
  }
  static __device__ inline float dot(const Frag (&a)[KF], const Frag (&b)[KF]) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < KF; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) t = fmaf(whole(a[k], j), whole(b[k], j), t);
    return t;
  }
  // Four rows from y on of columns d0 .. d0 + 31 of a row-major tile, transposed: in every group of 16
  // lanes, lane i addresses 8 bytes (row i / 4, columns 4 * (i % 4)..) and receives column i.
  static __device__ inline bf4 read_tr(const bf16* lds, int y, int d0, int lane) {
    const bf16* p = lds + (y + ((lane & 15) >> 2)) * LDW + d0 + (lane & 16) + 4 * (lane & 3);
    return __builtin_bit_cast(bf4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p));
  }
  // acc[dt][c] += sum over the 32 rows from 32 rt on of Z[y][32 dt + ..] P[y][x]. For bf16 rows P is
  // rounded to bf16 here, the one type that the matrix instructions multiply with the rows as they are: up to 2^-8 of
  // every weight, independent from weight to weight, beside the one rounding of the result to the same type (results
  // 2.4e-3 off 64 bits in the root mean square, of which their own rounding is 1.7e-3). A caller who wants more bits
  // takes fp32 rows.
  template <int NC>
  static __device__ inline void accumulate(const bf16* lds, int rt, const f16v (&p)[NC], f16v (&acc)[NDT][NC],
                                           int lane) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      Frag b[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p[c][8 * k + j];
        b[c] = frag(v);
      }
      const int y = 32 * rt + 16 * k + 4 * (lane >> 5);
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        Frag a;
#pragma unroll
        for (int i = 0; i < PL; ++i) {
          const bf4 l = read_tr(lds + i * PLANE, y, 32 * d, lane), h = read_tr(lds + i * PLANE, y + 8, 32 * d, lane);
          a.p[i] = bf8{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[d][c] = product(a, b[c], acc[d][c]);
      }
    }
  }
};

// four consecutive elements of a row of D
template <typename T>
__device__ inline void store4(T* row, int d0, int D, f4 v, bool vec) {
  if (vec && d0 + 4 <= D) {
    T t[4] = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    if (sizeof(T) == 4) {
      u4 w;
      __builtin_memcpy(&w, t, 16);
      *(u4*)(row + d0) = w;
    } else {
      uint64_t w;
      __builtin_memcpy(&w, t, 8);
      *(uint64_t*)(row + d0) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d0 + i < D) row[d0 + i] = (T)v[i];
  }
}

// what a value's rounding to T leaves
template <typename T>
__device__ inline f4 rest_of(f4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] -= (float)(T)v[i];
  return v;
}

// column c of acc, times f, as a row of D elements; rest (may be NULL) takes what the rounding leaves
template <typename T, int NDT, int NC>
__device__ inline void store_col(T* row, int D, const f16v (&acc)[NDT][NC], int c, float f, bool vec, int lane,
                                 T* rest = nullptr) {
#pragma unroll
  for (int d = 0; d < NDT; ++d)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d0 = 32 * d + 8 * q + 4 * (lane >> 5);
      f4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = acc[d][c][4 * q + i] * f;
      if (d0 < D) {
        store4(row, d0, D, v, vec);
        if (rest) store4(rest, d0, D, rest_of<T>(v), vec);
      }
    }
}

}  // namespace seq
}  // namespace mono

#endif  // MONO_SEQ_DEV_H_
