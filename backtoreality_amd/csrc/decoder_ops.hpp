// decoder_ops.hpp -- element types, 16-byte row loads / stores and wave reductions shared by the
// decoder operators that take float32, bfloat16 and float16 (layer_norm.hip, linear.hip,
// cross_attention.hip).
#pragma once
#include "common.hpp"

namespace btr {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// kVec elements are 16 bytes.  Vec: the value in registers; VecU: the same in memory at the
// alignment of ONE element -- gfx950 serves global 16-byte accesses at any address, so rows of odd
// width or odd stride need no variant of their own.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kVec = 4;
  typedef f32x4_t Vec;
  typedef float VecU __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Elem<__bf16> {
  static constexpr int kVec = 8;
  typedef bf16x8_t Vec;
  typedef __bf16 VecU __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct Elem<_Float16> {
  static constexpr int kVec = 8;
  typedef f16x8_t Vec;
  typedef _Float16 VecU __attribute__((ext_vector_type(8), aligned(2)));
};

template <>
struct Elem<unsigned short> {   // 16 bits as they are
  static constexpr int kVec = 8;
  typedef unsigned short Vec __attribute__((ext_vector_type(8)));
  typedef unsigned short VecU __attribute__((ext_vector_type(8), aligned(2)));
};

// the elements [e0, e0 + kVec) of a row of n; beyond the row zero, and never read
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec load_row(const T *row, int e0, int n) {
  constexpr int V = Elem<T>::kVec;
  typename Elem<T>::Vec v = {};
  if (e0 + V <= n) {
    v = *reinterpret_cast<const typename Elem<T>::VecU *>(row + e0);
  } else if (e0 < n) {   // (the row's last element in place of what is beyond: the loads fly together)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const T t = row[min(e0 + j, n - 1)];
      v[j] = e0 + j < n ? t : (T)0.f;
    }
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void store_row(T *row, int e0, int n, typename Elem<T>::Vec v) {
  constexpr int V = Elem<T>::kVec;
  if (e0 + V <= n) {
    *reinterpret_cast<typename Elem<T>::VecU *>(row + e0) = v;
  } else if (e0 < n) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (e0 + j < n) row[e0 + j] = v[j];
  }
}

// workspaces are written and read in 16-byte units (NULL where none is needed)
inline bool aligned16(const void *p) { return ((unsigned long long)p & 15) == 0; }

// sum over the 64 lanes, in every lane
__device__ __forceinline__ float wave_sum_f32(float v) {
  v = row16_sum_f32(v);
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// Column c of the sum of `rows` partial rows of n floats, in a fixed order: 1 024 threads are 32 columns
// x 32 groups of rows, four loads of a thread in flight (eight groups and one load at a time made
// these launches 10 - 33 us).  Valid in threads of group 0 (threadIdx.x < 32).
__device__ __forceinline__ float column_sum(const float *part, int rows, long long n, long long c) {
  __shared__ float s[32][33];
  const int cl = threadIdx.x & 31, rg = threadIdx.x >> 5;
  float acc[4] = {};
  if (c < n) {
    int r = rg;
    for (; r + 96 < rows; r += 128) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += part[(r + 32ll * i) * n + c];
    }
    for (; r < rows; r += 32) acc[0] += part[(long long)r * n + c];
  }
  s[rg][cl] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
  __syncthreads();
  float t = 0.f;
  if (rg == 0) {
#pragma unroll
    for (int k = 0; k < 32; ++k) t += s[k][cl];
  }
  return t;
}

}  // namespace btr

// runs `CALL` (an expression that names the element type as T) for the type code `dtype`
#define BTR_DISPATCH_DTYPE(dtype, ...)                                          \
  do {                                                                          \
    if ((dtype) == BTR_F32) {                                                   \
      typedef float T;                                                          \
      __VA_ARGS__;                                                              \
    } else if ((dtype) == BTR_BF16) {                                           \
      typedef __bf16 T;                                                         \
      __VA_ARGS__;                                                              \
    } else {                                                                    \
      typedef _Float16 T;                                                       \
      __VA_ARGS__;                                                              \
    }                                                                           \
  } while (0)
