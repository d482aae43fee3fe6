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
  float *stats, *hist, *part;
  float4 *rec;  // [B, Hq, rec_rows]: maximum (+inf: no keys), log2 of the sum, D, unused
  double *dist;
  float *dtable;
  int B, Tq, Tk, Hq, Hk, d, G, causal, nb, M;
  int splits, pack;  // few-row kernel: pieces of the keys, query heads packed into a workgroup's rows
  int hist_rows, share, direct, stages, rec_rows, fine;
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
// A table entry, base 2.  The type's lowest and highest values keep a finite bias: a row of nothing else is uniform, not empty
// or NaN.
__device__ __forceinline__ float bias_of(float t) {
  constexpr float MOST = 3.4028234663852886e38f;
  return fabsf(t) <= MOST ? fminf(fmaxf(t * LOG2E, -MOST), MOST) : t;
}
// Bias of map entry i; entries outside the table have none.
__device__ __forceinline__ float bias_at(const AttnArgs &a, int i, int h) {
  const int b = a.map[i];
  return b >= 0 && b < a.nb ? bias_of(a.table[(long)b * a.Hq + h]) : 0.f;
}
// A head's bias by distance in LDS: entry `away` of the returned array for -M - PAD <= away <= M + PAD.  A block that is not
// wholly beyond M on one side (64 keys, 32 queries) reaches less than 95 distances beyond it, so its reads need no clamp, only constant offsets.
constexpr int PAD = 96;
__host__ __device__ __forceinline__ int bias_floats(int M) { return 2 * M + 1 + 2 * PAD; }
// A prologue's loads are few and each waits a microsecond or more for memory, so they are issued together: map() first, what
// else the kernel loads next, table() then, and store() last.
struct BiasLoad {
  const AttnArgs &a;
  float *bias;  // `heads` arrays of bias_floats(M), heads h ..
  int h, tid, nt, size, total, b[4], at[4];
  float t[4];
  __device__ __forceinline__ BiasLoad(const AttnArgs &a, float *bias, int h, int heads, int tid, int nt)
      : a(a), bias(bias), h(h), tid(tid), nt(nt), size(bias_floats(a.M)), total(heads * size) {}
  __device__ __forceinline__ bool has(int x) const { return b[x] >= 0 && b[x] < a.nb; }
  __device__ __forceinline__ void map(int first = 0) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int e = min(first + tid + x * nt, total - 1), head = e / size;
      at[x] = h + head;
      b[x] = a.map[min(max(e - head * size - PAD, 0), 2 * a.M)];
    }
  }
  __device__ __forceinline__ void table() {
#pragma unroll
    for (int x = 0; x < 4; ++x) t[x] = a.table[(long)(has(x) ? b[x] : 0) * a.Hq + at[x]];
  }
  __device__ __forceinline__ const float *store() {
    for (int first = 0; first < total; first += 4 * nt) {
      if (first > 0) {
        map(first);
        table();
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (first + tid + x * nt < total) bias[first + tid + x * nt] = has(x) ? bias_of(t[x]) : 0.f;
    }
    return bias + PAD + a.M;
  }
};
// The same for one head, entry by entry: where registers are short.
__device__ __forceinline__ const float *load_bias(const AttnArgs &a, float *bias, int h, int tid, int nt) {
#pragma unroll 1
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

// Waves of a workgroup that shares a ring, and its buffers: at most 64 KB with 16-bit types, so that two workgroups lie on a compute
// unit (fp32: 128 KB at most and one workgroup).  Eight waves of one workgroup, or more buffers in place of the second
// workgroup, gained nothing (2 x 4096 causal, heads of 128).
template <typename T, int D>
struct RingShape {
  static constexpr int WAVES = 4;
  static constexpr int STAGES = sizeof(T) == 2 ? (D == 128 ? 2 : D == 64 ? 3 : 4) : (D == 32 ? 4 : 2);
  static constexpr int BYTES = STAGES * 2 * Tile<T, D, BK>::BYTES;
};

// Keys and values of a head on their way through a ring of LDS buffers: tile t in buffer t % STAGES, STAGES - 1 tiles ahead, so
// that a tile has that many tiles' work to arrive in.
template <typename T, int D, int NT>
struct KeyRing {
  using L = Tile<T, D, BK>;
  static constexpr int LOADS = 2 * (BK * L::CPR < NT ? 1 : BK * L::CPR / NT);
  const AttnArgs &a;
  lds_char *base;
  const T *kp, *vp;
  static constexpr int STAGES = RingShape<T, D>::STAGES;
  int kend, n, tid, slot;
  __device__ __forceinline__ KeyRing(const AttnArgs &a, lds_char *base, const T *kp, const T *vp, int kend, int tid)
      : a(a), base(base), kp(kp), vp(vp), kend(kend), n((kend + BK - 1) / BK), tid(tid), slot(0) {
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t)
      if (t < n) fetch(t, t);
  }
  __device__ __forceinline__ void fetch(int t, int to) {
    fill<T, D, BK, NT>(L{base + to * 2 * L::BYTES}, a.direct, kp, a.sk.t, t * BK, kend, a.d, tid);
    fill<T, D, BK, NT>(L{base + (to * 2 + 1) * L::BYTES}, a.direct, vp, a.sv.t, t * BK, kend, a.d, tid);
  }
  // Waits for tile t and starts the one that takes the place of tile t - 1; all threads call it for t = 0, 1, .. n - 1.
  __device__ __forceinline__ void step(int t, L &keys, L &values) {
    if (STAGES == 2)
      arrive();
    else
      arrive_but<LOADS>(min(STAGES - 2, n - 1 - t));
    lds_barrier();
    const int last = slot == 0 ? STAGES - 1 : slot - 1;
    if (t + STAGES - 1 < n) fetch(t + STAGES - 1, last);
    keys.base = base + slot * 2 * L::BYTES;
    values.base = base + (slot * 2 + 1) * L::BYTES;
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
};
// Runs FN<T, D, DC> for the element type and the width of a head: D elements a row in LDS, DC of them in the products.
#define VT_WIDTH(FN, ...)                                             \
  VT_DISPATCH_TYPE(a->dtype, {                                        \
    if (a->d <= 32) return (FN<T, 32, 32>(__VA_ARGS__));              \
    if (a->d <= 64) return (FN<T, 64, 64>(__VA_ARGS__));              \
    if (a->d <= 96) return (FN<T, 128, 96>(__VA_ARGS__));             \
    return (FN<T, 128, 128>(__VA_ARGS__));                            \
  })
// fp16 ends at 2^-24 (2^-14 with all its bits): probabilities of long rows and ds of small output gradients lie below.  They are
// scaled by powers of two before they are rounded, and the sums scaled back: forward p by 2^13 (with which it reaches 2^15),
// backward p by 2^14 (it reaches 1), ds by a factor of its own for each of the wave's rows (fit_half).  (2 x 4096 causal, 16 heads of
// 128 over 4: backward pass 648 -> 694 us.)  bf16 and fp32 have the range.
template <typename T>
constexpr bool HALF_RANGE = __is_same(T, f16_t);
template <typename T>
constexpr float FWD_MOST = HALF_RANGE<T> ? 15.f : 8.f;  // log2 of the largest p
// The softmax's reference for a row whose maximum is t.  Large t (tables that mask by finite values) keep no lift: t - 13 would be
// rounded there, by more than 2 beyond 2^25.
template <typename T>
__device__ __forceinline__ float reference(float t) {
  return HALF_RANGE<T> && fabsf(t) < 1024.f ? t - 13.f : t;
}
constexpr float BWD_LIFT = 16384.f, DS_LIFT = 1.099511627776e12f;  // 2^40: lowered by the first block that exceeds the range
// Scales a C block of ds by its column's factor w.  Where that would exceed 2^14 the factor is lowered first, to a block's largest
// value below 2^12, and with it the sums o that the column has so far.
template <int NDB>
__device__ __forceinline__ void fit_half(f32x16 &s, f32x16 (&o)[NDB], float &w) {
  float t = fabsf(s[0]);
#pragma unroll
  for (int r = 1; r < 16; ++r) t = fmaxf(t, fabsf(s[r]));
  t = fmaxf(t, __shfl_xor(t, 32)) * w;
  if (__any(t > BWD_LIFT)) {
    const float f = t > BWD_LIFT && t < INFINITY ? __builtin_ldexpf(1.f, 12 - __builtin_amdgcn_frexp_expf(t)) : 1.f;
    w *= f;
#pragma unroll
    for (int b = 0; b < NDB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] *= f;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] *= w;
}
template <int NDB>
__device__ __forceinline__ void scale_all(f32x16 (&o)[NDB], float f) {
#pragma unroll
  for (int b = 0; b < NDB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[b][r] *= f;
}
template <typename F>
inline int set_lds(F *f, int bytes) {
  return bytes > 65536 ? (int)hipFuncSetAttribute((const void *)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) : 0;
}

constexpr int LDS_BYTES = 160 * 1024;
// Whether two waves share a block of 32 rows: where workgroups of 128 rows, of which two (fp32: one) lie on a compute unit, leave
// compute units idle.  Many causal rows are uneven in length and share on.  Wide 16-bit heads read twice the fragments a product
// where they share, which their dk, dv pass pays first.  The host cannot see whether given lengths are full: where sharing
// costs full ones little and helps uneven ones much (causal or fp32 heads of at most 64), they take a third of the blocks to be
// empty, elsewhere none.
// Measured at T = 2048, alone and shared, us; full lengths, then lengths from T / 3 to T in brackets, of 256, 512, 640, 768 blocks:
//   bf16, 64 wide    forward 60 47 [57 45], 79 81 [74 77], 102 97 [91 83], 110 113 [91 93]
//     causal         forward 57 37 [57 36], 59 49 [57 46], 61 58 [58 43], 66 66 [61 51]; dk, dv shared -38 [-38], -27 [-27], -1 [-26], +11 [-9]
//     dk, dv         256 to 768, and 320, 384: shared -33 [-33], +14 [+15], -27 [-14], -11 [-18], +4 [-15], +2 [-2]
//   bf16, 128 wide   forward 82 69 [80 66], 120 129 [104 124], 179 170 [143 137]; dk, dv shared +45 [+46] of 235, +213 [+214] of 303
//     causal         forward 79 57 [78 56], 85 78 [81 75], 91 100 [83 76], 102 114 [83 92]; dk, dv shared -34 [-32], 320 +6 [-29], 384 +22 [-8]
//   fp32, 64 wide    forward 162 151 [161 149], 287 297 [283 294], 430 375 [381 302], 434 440 [471 381]
//     causal         forward 161 118 [160 116], 214 174 [211 172], 227 207 [226 147], 252 243 [235 184]
//   fp32, 128 wide   forward 384 568 468 [482 438], 512 575 625 [565 621]; causal 284 174 [283 173], 313 337 [310 335], 438 438 [327 316]
// Backward pass with p and ds in two parts: dq in the shared form, dk and dv, where the second wave of a pair would have no
// queries if they are at most 32, in the other.  fp32 queries of at most 32 rows share up to 512 blocks, causal 1024.
inline bool attn_fine(const vt_relpos_attention *a) { return a->dtype != VT_F32 && (a->Tq <= 32 || a->precise); }
inline bool attn_split(const vt_relpos_attention *a, int heads, int rows, bool keys, bool fine = false) {
  if (fine) return !keys;
  const int tiles = (rows + 127) / 128;
  const bool narrow = a->dtype == VT_F32 || a->d <= 64, lengths = (keys ? a->k_len : a->q_len) != nullptr;
  long blocks = (long)a->B * heads * tiles;
  if (lengths && a->d <= 64 && (a->causal || a->dtype == VT_F32)) blocks -= blocks / 3;
  const bool uneven = a->causal && tiles >= 8;
  if (a->Tq <= 32) return blocks < (a->causal ? 1024 : 512);
  if (narrow) return blocks < (uneven ? 576 : keys ? 352 : 448);
  return blocks < (keys ? (uneven ? 320 : 160) : (uneven ? 576 : 288));
}
// The backward pass's launches (vtcnn_attn_bwd.hip), and how it cuts its work: whether waves share rows (queries, keys), the
// workgroups a head's keys take, their buffers and LDS, and how many workgroups share a key head's query heads (1 or G).
struct BwdPlan {
  int split_q, split_k, key_tiles, key_stages, key_bytes, share;
};
BwdPlan attn_bwd_plan(const vt_relpos_attention *a);
int attn_bwd_launch(const vt_relpos_attention *a, const AttnArgs &k, const BwdPlan &p, hipStream_t s);

}  // namespace vt
