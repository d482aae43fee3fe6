// Tiles of the attention kernels: fragments of 32x32 matrix instructions for fp32, bf16 and fp16, and row tiles in LDS that
// are read both as rows and transposed.
//
// One step of the matrix cores here is C[32,32] += A[32,16] B[16,32].  Lane l (half = l / 32) holds
//   of A: row l % 32, eight values of the inner axis;  of B: column l % 32, the same eight;
//   of C: column l % 32, rows 8 (r / 4) + 4 half + r % 4 in register r = 0 .. 15.
// The inner axis may be numbered in any order that A and B share.  Where both come from row tiles, slot j of a half is inner
// index 8 half + j.  Where B is a C of before (P or dS), its registers 8 s .. 8 s + 7 are the B fragment of inner indices
// 16 s + {4 half .. 4 half + 3, 8 + 4 half .. 8 + 4 half + 3} as they lie, so no value crosses lanes between the two products.
// 16-bit types: one v_mfma_f32_32x32x16; fp32: eight v_mfma_f32_32x32x2_f32, exact products.
#pragma once
#include "vtcnn_typed.h"

namespace vt {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Frag {
  typedef T type __attribute__((ext_vector_type(8)));
};
template <typename T>
using frag = typename Frag<T>::type;

__device__ __forceinline__ f32x16 mma(frag<bf16_t> a, frag<bf16_t> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(frag<f16_t> a, frag<f16_t> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(frag<float> a, frag<float> b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// B fragment s of a product's C registers, rounded to the element type.
template <typename T>
__device__ __forceinline__ frag<T> c_frag(const f32x16 &c, int s) {
  frag<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)c[8 * s + j];
  return f;
}

// Eight elements of a global row from `at` on, zeros behind its d elements.
template <typename T>
__device__ __forceinline__ frag<T> row_frag(const T *row, bool ok, int at, int d) {
  frag<T> f;
  if (ok && at + 8 <= d) {
    const vec8<T> v = *reinterpret_cast<const vec8<T> *>(row + at);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = ok && at + e < d ? row[at + e] : (T)0.f;
  }
  return f;
}

// A tile of ROWS rows of D elements in LDS, in chunks of 16 bytes.  Chunk c of row r lies at place c ^ swz(r) of its row:
// eight consecutive rows put the same chunk into eight different 16-byte bank groups (the row fragments' reads), and four
// consecutive rows put a pair of chunks into four different 32-byte ones (the transposed reads).
template <typename T, int D, int ROWS>
struct Tile {
  static constexpr int EPC = 16 / (int)sizeof(T);     // elements a chunk
  static constexpr int CPR = D / EPC;                 // chunks a row
  static constexpr int BYTES = ROWS * D * (int)sizeof(T);
  char *base;

  static __device__ __forceinline__ int swz(int r) {
    if (CPR >= 8) return ((r & 3) << 1) | ((r >> 2) & 1);
    return (r & 2) | ((r >> 2) & 1);  // 64-byte rows: two rows fill the banks once
  }
  __device__ __forceinline__ char *chunk(int r, int c) const { return base + (r * CPR + (c ^ swz(r))) * 16; }

  // A fragment of rows row0 .. row0 + 31, elements 16 s .. 16 s + 15 as the inner axis.
  __device__ __forceinline__ frag<T> rows(int row0, int s) const {
    const int lane = threadIdx.x & 63, r = row0 + (lane & 31), half = lane >> 5;
    union {
      u32x4 w[sizeof(T) / 2];
      frag<T> f;
    } u;
    if constexpr (sizeof(T) == 2) {
      u.w[0] = *reinterpret_cast<const u32x4 *>(chunk(r, 2 * s + half));
    } else {
      u.w[0] = *reinterpret_cast<const u32x4 *>(chunk(r, 4 * s + 2 * half));
      u.w[1] = *reinterpret_cast<const u32x4 *>(chunk(r, 4 * s + 2 * half + 1));
    }
    return u.f;
  }
  // A fragment of the transpose: elements 32 c .. 32 c + 31 as rows, tile rows row0 .. row0 + 15 as the inner axis in the
  // order of a C's registers.
  __device__ __forceinline__ frag<T> cols(int row0, int c) const {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    frag<T> f;
    if constexpr (sizeof(T) == 2) {
      // ds_read_b64_tr_b16: sixteen lanes name four rows of sixteen elements, four lanes (8 bytes each) a row; lane i of
      // them receives element i of each of the four rows
      const int r = row0 + 4 * half + ((lane & 15) >> 2);
      const int k = 4 * c + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), b = (lane & 1) * 8;
      union {
        s16x4 w[2];
        frag<T> f;
      } u;
      u.w[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(chunk(r, k) + b));
      u.w[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(chunk(r + 8, k) + b));
      f = u.f;
    } else {
      const int k = 8 * c + ((lane & 31) >> 2), b = (lane & 3) * 4;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = *reinterpret_cast<const T *>(chunk(row0 + 4 * half + (j & 3) + 8 * (j >> 2), k) + b);
    }
    return f;
  }
};

// Sixteen bytes at an address that is only as aligned as one element.
template <typename T>
struct Chunk {
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// The share of NT threads in a tile's next rows, on its way from global memory to LDS through registers: rows row0 .. of p
// (stride elements apart), zeros from row `end` (> row0) on and behind d elements.  The loads take no branch: a chunk
// outside reads one inside instead, and is replaced by zeros on its way into LDS.
template <typename T, int D, int ROWS, int NT>
struct Stage {
  using L = Tile<T, D, ROWS>;
  static constexpr int N = ROWS * L::CPR / NT;
  static_assert(N * NT == ROWS * L::CPR, "the threads share the tile evenly");
  u32x4 w[N];
  __device__ __forceinline__ void load(const T *p, long stride, int row0, int end, int d, int tid) {
    if (d % L::EPC == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = tid + i * NT, r = min(row0 + at / L::CPR, end - 1), e0 = (at % L::CPR) * L::EPC;
        const T *src = p + (long)r * stride + (e0 < d ? e0 : 0);
        w[i] = __builtin_bit_cast(u32x4, *reinterpret_cast<const typename Chunk<T>::type *>(src));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int at = tid + i * NT, r = min(row0 + at / L::CPR, end - 1), e0 = (at % L::CPR) * L::EPC;
        const T *src = p + (long)r * stride;
        union {
          T t[16 / sizeof(T)];
          u32x4 v;
        } u;
#pragma unroll
        for (int e = 0; e < L::EPC; ++e) u.t[e] = e0 + e < d ? src[e0 + e] : (T)0.f;
        w[i] = u.v;
      }
    }
  }
  __device__ __forceinline__ void store(const L &t, int row0, int end, int d, int tid) const {
    const bool whole = row0 + ROWS <= end && d == D;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = tid + i * NT, r = at / L::CPR, c = at % L::CPR;
      u32x4 v = w[i];
      if (!whole && !(row0 + r < end && c * L::EPC < d)) v = u32x4{0, 0, 0, 0};
      *reinterpret_cast<u32x4 *>(t.chunk(r, c)) = v;
    }
  }
};

}  // namespace vt
