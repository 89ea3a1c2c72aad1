// Device helpers of the kernels that hold a vector (a head, a row) spread over
// neighbouring lanes in 16-byte pieces of fp32, bf16 or fp16 elements.
#pragma once
#include "gcnx_common.h"

namespace gcnx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// A lane's piece of a vector: 16 bytes.  Where the vector is no multiple of the
// piece, the last piece overlaps the one before it instead of reaching over the
// vector's end: a lane counts its elements `skip`.. only, and writes the others with
// the same values as their owner.  Vectors shorter than a piece take one lane and
// are read element by element (NARROW).
template <typename T> struct Piece;
template <> struct Piece<float> { typedef f32x4 raw; static constexpr int N = 4; };
template <> struct Piece<__bf16> { typedef bf16x8 raw; static constexpr int N = 8; };
template <> struct Piece<_Float16> { typedef f16x8 raw; static constexpr int N = 8; };

// Addresses are kept as numbers and turned into pointers to global memory where
// they are read: base + column * stride is one 32 x 32 + 64 bit multiply-add, and a
// choice between two addresses does not become a generic (flat) access.
typedef uint64_t Address;
#define GCNX_GLOBAL __attribute__((address_space(1)))
template <typename V>
__device__ __forceinline__ V load_at(Address a) {
  return *(const GCNX_GLOBAL V *)a;
}
__device__ __forceinline__ Address row_at(Address base, int32_t row, uint32_t stride) {
  return base + (uint64_t)(uint32_t)row * stride;
}

// What lanes without an edge read: loads are never conditional (a load under a
// branch is waited for before the next one can be issued into its registers).
__device__ const f32x4 g_zeros[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};

__device__ __forceinline__ Address at_or_zeros(Address a, bool on) { return on ? a : (Address)&g_zeros[0]; }

// One piece.  Rows need only their elements' alignment: global loads of 16 bytes
// take any address.  NARROW: `dim` < a piece, the rest repeats the last element.
template <typename T, bool NARROW>
__device__ __forceinline__ typename Piece<T>::raw load_piece(Address a, int dim) {
  typedef typename Piece<T>::raw raw;
  typedef raw anywhere __attribute__((aligned(sizeof(T))));
  if constexpr (!NARROW) {
    return load_at<anywhere>(a);
  } else {
    raw x;
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) x[i] = load_at<T>(a + sizeof(T) * (i < dim ? i : dim - 1));
    return x;
  }
}

template <typename T, bool NARROW>
__device__ __forceinline__ void store_piece(T *p, int dim, const float (&v)[Piece<T>::N]) {
  if constexpr (!NARROW) {
    typename Piece<T>::raw x;
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i) x[i] = (T)v[i];
    __builtin_memcpy(p, &x, sizeof(x));
  } else {
#pragma unroll
    for (int i = 0; i < Piece<T>::N; ++i)
      if (i < dim) p[i] = (T)v[i];
  }
}

// Sum over groups of G neighbouring lanes, the result in every lane of the group.
// Steps 1..8 are moves on the vector ALU: quad permutes, then the mirrors of 8 and
// 16 lanes (every lane of a sub-group already holds the sub-group's sum).
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#define GCNX_DPP(ctrl) __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), ctrl, 0xF, 0xF, true))
  if constexpr (G >= 2) v += GCNX_DPP(0xB1);
  if constexpr (G >= 4) v += GCNX_DPP(0x4E);
  if constexpr (G >= 8) v += GCNX_DPP(0x141);
  if constexpr (G >= 16) v += GCNX_DPP(0x140);
  if constexpr (G >= 32) v += __shfl_xor(v, 16, kWave);
  if constexpr (G >= 64) v += __shfl_xor(v, 32, kWave);
#undef GCNX_DPP
  return v;
}


typedef f32x4 f32x4_anywhere __attribute__((aligned(4)));
// N floats at an address that need not be a multiple of 16.
template <int N>
__device__ __forceinline__ void load_floats(const float *p, float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const f32x4 x = *reinterpret_cast<const f32x4_anywhere *>(p + i);
    f[i] = x[0]; f[i + 1] = x[1]; f[i + 2] = x[2]; f[i + 3] = x[3];
  }
}
template <int N>
__device__ __forceinline__ void store_floats(float *p, const float (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4_anywhere *>(p + i) = f32x4{f[i], f[i + 1], f[i + 2], f[i + 3]};
}

// e^x.  x log2(e) is rounded once, so that the result is off by |x| 2^-24 of itself beside
// the instruction's 1 ulp.  A softmax has x <= 0 and sums terms of e^x: |x| e^x <= 0.37,
// so that no term moves the sum by more than its own rounding at the row's largest.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// Nothing moves across: what is read ahead stays ahead of the sums.
__device__ __forceinline__ void read_ahead_fence() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

inline int log2_ceil(int64_t x) {
  int l = 0;
  while (((int64_t)1 << l) < x) ++l;
  return l;
}

}  // namespace gcnx
