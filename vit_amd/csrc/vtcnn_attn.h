// What the attention kernels' forward and backward files share: arguments, the bias by distance, masks, stores of C blocks.
#pragma once
#include "vtcnn_attn_tiles.h"

namespace vt {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int BK = 64;  // keys (forward, dq) or queries (dk, dv) of a tile in LDS

struct AttnArgs {
  const void *q, *k, *v, *o, *o_lo, *dout;
  void *out, *out_lo, *dq, *dk, *dv;
  vt_strides sq, sk, sv, so, sdo, sdq, sdk, sdv;
  const int *map, *q_start, *q_len, *k_len;
  const float *table;
  float *stats, *delta, *hist, *part;
  double *dist;
  float *dtable;
  int B, Tq, Tk, Hq, Hk, d, G, causal, nb, M;
  int splits, pack;  // few-row kernel: pieces of the keys, query heads packed into a workgroup's rows
  int hist_rows, share, direct;
  float scale;
};

__device__ __forceinline__ int length_of(const int *p, int b, int most) { return p ? min(max(p[b], 0), most) : most; }
__device__ __forceinline__ int start_of(const AttnArgs &a, int b) {
  return a.q_start ? min(max(a.q_start[b], -(1 << 29)), 1 << 29) : 0;  // positions stay within int
}
// The wave's number in its workgroup, known to be the same in all lanes: what depends on it alone decides branches.
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }
// A value that the compiler takes for new: sixteen distances derived from it are formed where they are used, not kept in
// sixteen registers over the whole loop.
__device__ __forceinline__ int afresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}
// Bias of map entry i, base 2.
__device__ __forceinline__ float bias_at(const AttnArgs &a, int i, int h) {
  const int b = a.map[i];
  if (b < 0 || b >= a.nb) return 0.f;
  const float t = a.table[(long)b * a.Hq + h], x = t * LOG2E;
  // a table that masks by the type's lowest value keeps a finite bias: a row of nothing else is uniform, not empty
  return x == -INFINITY && t != -INFINITY ? -3.4028234663852886e38f : x;
}
// A head's bias by distance in LDS: entry `away` of the returned array for -M - PAD <= away <= M + PAD.  A block that is not
// wholly beyond M on one side (64 keys, 32 queries) reaches less than 95 distances beyond it, so its reads need no clamp, only constant offsets.
constexpr int PAD = 96;
__host__ __device__ __forceinline__ int bias_floats(int M) { return 2 * M + 1 + 2 * PAD; }
__device__ __forceinline__ const float *load_bias(const AttnArgs &a, float *bias, int h, int tid, int nt) {
  for (int i = tid; i < bias_floats(a.M); i += nt) bias[i] = bias_at(a, min(max(i - PAD, 0), 2 * a.M), h);
  return bias + PAD + a.M;
}

// Scores of a 32-key block and the wave's 32 queries (lane: one query, at position pos) to base 2 with bias and mask.
// first: the block's first key; NEAR: the bias is looked up by distance, otherwise it is `flat`.
template <bool NEAR, bool MASK>
__device__ __forceinline__ void finish_scores(f32x16 &s, float c, const float *bias, float flat, int first, int pos, int kend, bool causal) {
  const int half = (threadIdx.x & 63) >> 5, at = afresh(first + 4 * half - pos);
  const int last = MASK ? min(kend - pos, causal ? 1 : kend - pos) : 0;  // distances from here on are not seen
  const float *b = bias + at;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    float x = fmaf(s[r], c, NEAR ? b[8 * (r >> 2) + (r & 3)] : flat);
    if (MASK && at + 8 * (r >> 2) + (r & 3) >= last) x = -INFINITY;
    s[r] = x;
  }
}
// A block's place: wave-uniform.
struct Place {
  bool near, mask;
  int side;  // distance whose bias the block has where it is not near: M or -M
};
__device__ __forceinline__ Place place_of(int key0, int keys, int pos0, int queries, int M, int kend, bool causal) {
  Place p;
  const int lo = key0 - (pos0 + queries - 1), hi = key0 + keys - 1 - pos0;
  p.near = lo < M && hi > -M;
  p.side = lo >= M ? M : -M;
  p.mask = key0 + keys > kend || (causal && hi > 0);
  return p;
}
__device__ __forceinline__ void scores(f32x16 &s, const Place &p, float c, const float *bias, float flat, int first, int pos, int kend,
                                       bool causal) {
  if (p.near) {
    if (p.mask)
      finish_scores<true, true>(s, c, bias, flat, first, pos, kend, causal);
    else
      finish_scores<true, false>(s, c, bias, flat, first, pos, kend, causal);
  } else {
    if (p.mask)
      finish_scores<false, true>(s, c, bias, flat, first, pos, kend, causal);
    else
      finish_scores<false, false>(s, c, bias, flat, first, pos, kend, causal);
  }
}

__device__ __forceinline__ float max16(const f32x16 &s) {
  float m = s[0];
#pragma unroll
  for (int r = 1; r < 16; ++r) m = fmaxf(m, s[r]);
  return m;
}

__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// Four elements r4 of a C block as one row's elements at .. at + 3.
template <typename T>
__device__ __forceinline__ void store4(T *row, int at, int d, float a, float b, float c, float e) {
  typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (at + 4 <= d) {
    *reinterpret_cast<four *>(row + at) = four{(T)a, (T)b, (T)c, (T)e};
  } else {
    if (at < d) row[at] = (T)a;
    if (at + 1 < d) row[at + 1] = (T)b;
    if (at + 2 < d) row[at + 2] = (T)c;
  }
}
// C blocks [D, 32] times f as rows (one a lane column).
template <typename T, int NDB>
__device__ __forceinline__ void store_rows(T *row, int d, const f32x16 (&o)[NDB], float f) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int b = 0; b < NDB; ++b)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      store4<T>(row, 32 * b + 2 * r + 4 * half, d, o[b][r] * f, o[b][r + 1] * f, o[b][r + 2] * f, o[b][r + 3] * f);
}
template <typename T, int NDB>
__device__ __forceinline__ void residues(f32x16 (&o)[NDB], float f) {
#pragma unroll
  for (int b = 0; b < NDB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = o[b][r] * f;
      o[b][r] = x - (float)(T)x;
    }
}

// Runs FN<T, D, DC> for the element type and the width of a head: D elements a row in LDS, DC of them in the products.
#define VT_WIDTH(FN, ...)                                             \
  VT_DISPATCH_TYPE(a->dtype, {                                        \
    if (a->d <= 32) return (FN<T, 32, 32>(__VA_ARGS__));              \
    if (a->d <= 64) return (FN<T, 64, 64>(__VA_ARGS__));              \
    if (a->d <= 96) return (FN<T, 128, 96>(__VA_ARGS__));             \
    return (FN<T, 128, 128>(__VA_ARGS__));                            \
  })
template <typename F>
inline int set_lds(F *f, int bytes) {
  return bytes > 65536 ? (int)hipFuncSetAttribute((const void *)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) : 0;
}

constexpr int LDS_BYTES = 160 * 1024;
// The backward pass's launches (vtcnn_attn_bwd.hip), and how it cuts its work: pieces of a head's keys a workgroup takes, key
// splits of dq, whether query heads have workgroups of their own.
struct BwdPlan {
  int split_q, split_k, key_tile, key_tiles, share;
};
BwdPlan attn_bwd_plan(const vt_relpos_attention *a);
int attn_bwd_launch(const vt_relpos_attention *a, const AttnArgs &k, const BwdPlan &p, hipStream_t s);

}  // namespace vt
