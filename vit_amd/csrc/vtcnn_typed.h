// Element types of the typed launchers (fp32, bf16, fp16) and their row accesses: eight consecutive elements a lane.
#pragma once
#include "vtcnn_common.h"

namespace vt {

using bf16_t = __bf16;
using f16_t = _Float16;

// Eight elements whose address is only as aligned as one element: rows of odd width and sliced tensors start anywhere,
// and global memory takes a 16-byte access at any element's address.
template <typename T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};
template <typename T>
using vec8 = typename Vec8<T>::type;

// p[0 .. 8) of a row with `left` elements from p on; `fill` behind its end.
template <typename T>
__device__ __forceinline__ vec8<T> load8(const T *__restrict__ p, int left, T fill) {
  if (left >= 8) return *reinterpret_cast<const vec8<T> *>(p);
  vec8<T> v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < left ? p[e] : fill;
  return v;
}
template <typename T>
__device__ __forceinline__ void store8(T *p, int left, vec8<T> v) {
  if (left >= 8) {
    *reinterpret_cast<vec8<T> *>(p) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) p[e] = v[e];
}
template <typename T>
__device__ __forceinline__ void to_f32(vec8<T> v, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
}
template <typename T>
__device__ __forceinline__ vec8<T> from_f32(const float (&f)[8]) {
  vec8<T> v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)f[e];  // round to nearest even
  return v;
}

// Makes the compiler forget what it knows of v, so that conversions and exponentials of a row held in registers are formed
// again in the next pass instead of being kept (four registers a vector of 16-bit elements, against eight).
template <typename T>
__device__ __forceinline__ void forget(vec8<T> &v) {
  typedef unsigned words __attribute__((ext_vector_type(2 * sizeof(T))));
  words w = __builtin_bit_cast(words, v);
#pragma unroll
  for (int i = 0; i < (int)(2 * sizeof(T)); ++i) {
    unsigned x = w[i];
    asm volatile("" : "+v"(x));
    w[i] = x;
  }
  v = __builtin_bit_cast(vec8<T>, w);
}

// Sum / maximum over a group of GS threads (one wave, or the whole workgroup of GS threads); every thread of the group
// receives it.  red: LDS, GS / 64 floats, used by workgroup-sized groups only; consecutive calls alternate between two
// such arrays, so that one barrier a call is enough.  Fixed order of summation.
template <int GS>
__device__ __forceinline__ float group_sum(float x, float *red) {
  x = wave_sum(x);
  if (GS == 64) return x;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < GS / 64; ++w) s += red[w];
  return s;
}
template <int GS>
__device__ __forceinline__ float group_max(float x, float *red) {
  x = wave_max(x);
  if (GS == 64) return x;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int w = 1; w < GS / 64; ++w) s = fmaxf(s, red[w]);
  return s;
}

}  // namespace vt

// Runs `...` with T the element type of VT_F32 / VT_BF16 / VT_F16.
#define VT_DISPATCH_TYPE(dtype, ...)             \
  do {                                           \
    if ((dtype) == VT_F32) {                     \
      using T = float;                           \
      __VA_ARGS__;                               \
    } else if ((dtype) == VT_BF16) {             \
      using T = vt::bf16_t;                      \
      __VA_ARGS__;                               \
    } else {                                     \
      using T = vt::f16_t;                       \
      __VA_ARGS__;                               \
    }                                            \
  } while (0)
