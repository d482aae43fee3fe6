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

// The lane's share of a global row as fragments (elements 16 s + 8 half .. + 7 of fragment s), zeros behind its d elements and
// where !ok.  load_frags issues all loads and waits for none: outside the row they read its start or, where there is no row,
// `any` (an address that holds 8 elements), and clear_frags drops them.
template <typename T, int NS>
__device__ __forceinline__ void load_frags(frag<T> (&f)[NS], const T *row, bool ok, const T *any, int d) {
  const int half = (threadIdx.x & 63) >> 5;
  if (d % 8 == 0) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int at = 16 * s + 8 * half;
      const T *p = ok ? row + (at < d ? at : 0) : any;
      f[s] = __builtin_bit_cast(frag<T>, *reinterpret_cast<const vec8<T> *>(p));
    }
  } else {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = 16 * s + 8 * half + e;
        f[s][e] = ok && at < d ? row[at] : (T)0.f;
      }
  }
}
template <typename T, int NS>
__device__ __forceinline__ void clear_frags(frag<T> (&f)[NS], bool ok, int d) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < NS; ++s)
    if (!(ok && 16 * s + 8 * half < d)) f[s] = frag<T>{};
}

// What that rounding left, rounded.
template <typename T>
__device__ __forceinline__ frag<T> c_rest(const f32x16 &c, int s, const frag<T> &f) {
  frag<T> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)(c[8 * s + j] - (float)f[j]);
  return r;
}

typedef __attribute__((address_space(3))) char lds_char;

// A tile of ROWS rows of D elements in LDS, in chunks of 16 bytes.  Chunk c of row r lies at place c ^ swz(r) of its row:
// eight consecutive rows put the same chunk into eight different 16-byte bank groups (the row fragments' reads), and four
// consecutive rows put a pair of chunks into four different 32-byte ones (the transposed reads).
// swz(r) depends on r mod 8 and touches only the address bits XM, so a fragment's address is (lane part ^ constant) + constant:
// two to four registers for all fragments of a tile, of which the rest is the instruction's offset.
template <typename T, int D, int ROWS>
struct Tile {
  static constexpr int EPC = 16 / (int)sizeof(T);     // elements a chunk
  static constexpr int CPR = D / EPC;                 // chunks a row
  static constexpr int RB = D * (int)sizeof(T);       // bytes a row
  static constexpr int BYTES = ROWS * RB;
  static constexpr unsigned XM = CPR >= 8 ? 0x70 : 0x30;
  lds_char *base;  // a multiple of 128 bytes

  static __device__ __forceinline__ int swz(int r) {
    if (CPR >= 8) return ((r & 3) << 1) | ((r >> 2) & 1);
    return (r & 2) | ((r >> 2) & 1);  // 64-byte rows: two rows fill the banks once
  }
  __device__ __forceinline__ lds_char *chunk(int r, int c) const { return base + r * RB + ((c ^ swz(r)) << 4); }

  // A (or B) fragment of rows row0 .. row0 + 31 (row0 a multiple of 8), elements 16 s .. 16 s + 15 as the inner axis.
  __device__ __forceinline__ frag<T> rows(int row0, int s) const {
    const int lane = threadIdx.x & 63, r = lane & 31, half = lane >> 5;
    union {
      u32x4 w[sizeof(T) / 2];
      frag<T> f;
    } u;
    const unsigned part = r * RB + (((half * (int)sizeof(T) / 2) ^ swz(r)) << 4);
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
      const unsigned at = 16 * (int)sizeof(T) * s + 16 * j;
      u.w[j] = *(const __attribute__((address_space(3))) u32x4 *)(base + (part ^ (at & XM)) + (at & ~XM) + row0 * RB);
    }
    return u.f;
  }
  // A fragment of the transpose: elements 32 c .. 32 c + 31 as rows, tile rows row0 .. row0 + 15 (row0 a multiple of 8) as the
  // inner axis in the order of a C's registers.
  __device__ __forceinline__ frag<T> cols(int row0, int c) const {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    frag<T> f;
    if constexpr (sizeof(T) == 2) {
      // ds_read_b64_tr_b16: sixteen lanes name four rows of sixteen elements, four lanes (8 bytes each) a row; lane i of
      // them receives element i of each of the four rows
      const int r = 4 * half + ((lane & 15) >> 2);
      const unsigned part = r * RB + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ swz(r)) << 4) + (lane & 1) * 8, at = 64 * c;
      lds_char *p = base + (part ^ (at & XM)) + (at & ~XM) + row0 * RB;
      union {
        s16x4 w[2];
        frag<T> f;
      } u;
      u.w[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
      u.w[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p + 8 * RB));
      f = u.f;
    } else {
      const unsigned part = 4 * half * RB + ((((lane & 31) >> 2) ^ half) << 4) + (lane & 3) * 4;
#pragma unroll
      for (int j = 0; j < 8; ++j)  // row 4 half + (j & 3) + 8 (j >> 2): swz is 2 (j & 3) + half
        f[j] = *(const __attribute__((address_space(3))) T *)(base + (part ^ ((j & 3) << 5)) + 128 * c + ((j & 3) + 8 * (j >> 2) + row0) * RB);
    }
    return f;
  }
};

// Sixteen bytes at an address that is only as aligned as one element.
template <typename T>
struct Chunk {
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// Sixteen bytes a lane from global memory (g uniform in the wave, plus a lane's byte offset) straight into LDS, at l + 16 * lane
// (l uniform).  Written out because the compiler, which knows the builtin to write LDS, would wait for it before every
// transposed read of another buffer.  It has no result register; arrive() below waits for it.  The address pair comes from
// v_readfirstlane: a vector instruction's write to a scalar register needs five wait states before a vector memory instruction
// reads it, and the compiler, which sees to that for its own loads, does not look in here.  m0 is reserved to the compiler, which
// keeps no value in it and takes no declaration of its loss: it writes it directly before each use of its own.
__device__ __forceinline__ void async16(const void *g, unsigned offset, lds_char *l) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)l);
  const unsigned long u = (unsigned long)g;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
  const unsigned long uni = ((unsigned long)hi << 32) | lo;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(uni), "s"(at) : "memory");
}
// All of the wave's loads have arrived.
__device__ __forceinline__ void arrive() { asm volatile("s_waitcnt vmcnt(0)" : : : "memory"); }
// All but the newest `newer` tiles' loads (N a tile and wave) have arrived; loads arrive in order, and others in flight make
// the wait longer, never shorter.
template <int N>
__device__ __forceinline__ void arrive_but(int newer) {
  static_assert(2 * N < 64, "the counter's range");
  if (newer >= 2)
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * N) : "memory");
  else if (newer == 1)
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
  else
    arrive();
}
// The workgroup's barrier for LDS alone: loads on their way from global memory stay on their way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

// The share of NT threads in filling a tile with rows row0 .. row0 + ROWS - 1 of p (stride elements apart; p, row0 uniform).
// Rows from `end` (> row0) on repeat row end - 1, and places behind d elements repeat the row's first chunk: what they meet
// in a product is zero, or its result is not kept, and they are as finite as the row they repeat.
// direct: rows start on 16-byte boundaries, hold whole chunks and lie within 2^31 bytes a tile (the host's check): loads
// into LDS that pass no registers.
template <typename T, int D, int ROWS, int NT>
__device__ __forceinline__ void fill(const Tile<T, D, ROWS> &t, bool direct, const T *p, long stride, int row0, int end, int d,
                                     int tid) {
  using L = Tile<T, D, ROWS>;
  constexpr int TOTAL = ROWS * L::CPR, N = TOTAL < NT ? 1 : TOTAL / NT, STEP = NT / L::CPR;
  static_assert(TOTAL % 64 == 0 && (TOTAL < NT || N * NT == TOTAL) && NT % L::CPR == 0, "whole waves share the tile evenly");
  if (TOTAL < NT && tid >= TOTAL) return;
  const T *g = p + (long)row0 * stride;
  const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~63);
  if (direct && STEP % 8 == 0 && row0 + ROWS <= end) {
    const int r = tid / L::CPR, e0 = ((tid % L::CPR) ^ L::swz(r)) * L::EPC;
    const unsigned at = (unsigned)(r * (int)stride + (D == d || e0 < d ? e0 : 0)) * (unsigned)sizeof(T);
#pragma unroll
    for (int i = 0; i < N; ++i) async16(g + (long)i * STEP * stride, at, t.base + (i * NT + wave0) * 16);
  } else if (direct) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (tid + i * NT) / L::CPR, e0 = ((tid % L::CPR) ^ L::swz(r)) * L::EPC;
      const unsigned at = (unsigned)(min(r, end - 1 - row0) * (int)stride + (D == d || e0 < d ? e0 : 0)) * (unsigned)sizeof(T);
      async16(g, at, t.base + (i * NT + wave0) * 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (tid + i * NT) / L::CPR, e0 = (tid % L::CPR) * L::EPC;
      const T *src = g + (long)min(r, end - 1 - row0) * stride;
      union {
        T t[16 / sizeof(T)];
        u32x4 v;
      } u;
      if (e0 + L::EPC <= d) {
        u.v = __builtin_bit_cast(u32x4, *reinterpret_cast<const typename Chunk<T>::type *>(src + e0));
      } else {
#pragma unroll
        for (int e = 0; e < L::EPC; ++e) u.t[e] = e0 + e < d ? src[e0 + e] : (T)0.f;
      }
      *(__attribute__((address_space(3))) u32x4 *)t.chunk(r, tid % L::CPR) = u.v;
    }
  }
}

}  // namespace vt
