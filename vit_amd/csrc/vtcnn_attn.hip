// Attention with a learned relative position bias by buckets, forward and backward (vt_relpos_attention_*).
//
//   s_ij = scale q_i . k_j + table[map[clamp(j - i - start)]][h],  p = softmax over the visible j,  o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i;  dp_ij = do_i . v_j;  D_i = sum_j p_ij dp_ij = do_i . o_i;  ds = p (dp - D);
//   dq_i = scale sum_j ds_ij k_j;  dk_j = scale sum_i ds_ij q_i;  dtable[b][h] = sum of ds over the pairs of bucket b
//
// One pass over the keys with the running maximum and sum of the softmax (base 2); scores and probabilities stay in registers.
// The scores are formed transposed (keys x queries): a lane then holds scores of one query only, so maximum and sum need one
// exchange between the wave's halves, and p is the second product's operand as it lies (vtcnn_attn_tiles.h).
// The bias depends on the distance alone: a workgroup lays its head's bias out by distance in LDS once; tiles that lie
// wholly beyond max_distance on one side, which is nearly all of them in a long row, take a single value instead.
// Its gradient is gathered the same way: by distance in LDS arrays of one wave each (a wave's additions have one order),
// registers for the tiles beyond max_distance; the workgroups' arrays are added in double in their order and only then
// folded into buckets.  No atomics between waves: the same call gives the same bytes.
// p and ds are rounded to the inputs' type for the second products (fp32: not at all); the softmax's sum takes p before.
#include "vtcnn_attn_tiles.h"

namespace vt {
namespace {

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
__device__ __forceinline__ int bias_floats(int M) { return 2 * M + 1 + 2 * PAD; }
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

// One key tile's step of the running softmax: the scores s c + f (base 2; c > 0) become p.  m is a reference near the maximum
// rather than the maximum: o and l are brought to a new one only where a score exceeds it by more than 8, so p reaches up to
// 2^8, which costs neither fp32 sums nor a rounded p anything, and most tiles rescale nothing.
template <int NKB, int NDB>
__device__ __forceinline__ void online(f32x16 (&s)[NKB], f32x16 (&o)[NDB], float c, float f, float &m, float &l) {
  float t = max16(s[0]);
#pragma unroll
  for (int b = 1; b < NKB; ++b) t = fmaxf(t, max16(s[b]));
  t = fmaf(fmaxf(t, __shfl_xor(t, 32)), c, f);
  if (__any(t > m + 8.f)) {
    const float mn = fmaxf(m, t), w = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
    l *= w;
#pragma unroll
    for (int b = 0; b < NDB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] *= w;
    m = mn;
  }
  f -= m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int b = 0; b < NKB; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], c, f));
      sum += s[b][r];
    }
  l += sum;
}

// o += v^T p over a block of 32 keys.  LO: p as a high and a low part, for a forward pass that will be differentiated.
template <typename T, int NDB, bool LO, typename L>
__device__ __forceinline__ void add_values(const L &v, int row0, const f32x16 &p, f32x16 (&o)[NDB]) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const frag<T> pf = c_frag<T>(p, t);
    frag<T> lf;
    if (LO)
#pragma unroll
      for (int j = 0; j < 8; ++j) lf[j] = (T)(p[8 * t + j] - (float)pf[j]);
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const frag<T> vf = v.cols(row0 + 16 * t, db);
      o[db] = mma(vf, pf, o[db]);
      if (LO) o[db] = mma(vf, lf, o[db]);
    }
  }
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

// Statistics of a row: its maximum and log2 of its sum, apart, so that 2^(x - max - log2 sum) loses nothing to a large maximum.
__device__ __forceinline__ void store_stats(const AttnArgs &a, int b, int h, int i, float m, float l) {
  const float2 st = {l == 0.f ? -INFINITY : m, l == 0.f ? 0.f : __builtin_amdgcn_logf(l)};
  *reinterpret_cast<float2 *>(a.stats + 2 * (((long)b * a.Hq + h) * a.Tq + i)) = st;
}
// Output of the lane's query from its accumulators: o / l, zeros for a query without keys (l = 0) or outside its sequence.
template <typename T, int NDB>
__device__ __forceinline__ void finish_rows(const AttnArgs &a, f32x16 (&o)[NDB], float m, float l, bool ok, int b, int h, int i) {
  if (!ok) l = 0.f;
  const float f = l == 0.f ? 0.f : 1.f / l;
  if (l == 0.f)
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db] = f32x16{};
  const long at = b * a.so.b + (long)i * a.so.t + h * a.so.h;
  store_rows<T>((T *)a.out + at, a.d, o, f);
  if (a.out_lo) {
    residues<T>(o, f);
    store_rows<T>((T *)a.out_lo + at, a.d, o, 1.f);
  }
  if (a.stats && (threadIdx.x & 32) == 0) store_stats(a, b, h, i, m, l);
}

// ---------------------------------------------------------------------------------------------------------------------
// Forward, many rows: a workgroup takes 128 queries of one head, a wave 32 of them; the waves share the key tiles.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int D, bool LO>
__global__ __launch_bounds__(256) void k_attn_fwd(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  lds_char *tiles = (lds_char *)lds;
  using L = Tile<T, D, BK>;
  float *bias_lds = (float *)(lds + 4 * L::BYTES);
  constexpr int NS = D / 16, NDB = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int pairs = a.B * a.Hk, grp = blockIdx.x % pairs, b = grp / a.Hk, hk = grp % a.Hk, h = hk * a.G + blockIdx.x / pairs;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * 128, qw = q0 + wave_of() * 32, i = qw + (lane & 31);
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  const int pos0 = start + qw, pos = start + i;
  // keys beyond the last query's own are seen by none of the workgroup's
  const int kend = q0 >= qlen ? 0 : a.causal ? min(klen, max(0, start + min(q0 + 128, qlen))) : klen;
  const T *kp = (const T *)a.k + b * a.sk.b + hk * a.sk.h, *vp = (const T *)a.v + b * a.sv.b + hk * a.sv.h;
  const T *qp = (const T *)a.q + b * a.sq.b + h * a.sq.h;

  const float *bias = load_bias(a, bias_lds, h, tid, 256);
  frag<T> qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = row_frag<T>(qp + (long)i * a.sq.t, i < qlen, 16 * s + 8 * half, a.d);
  f32x16 o[NDB] = {};
  float m = -INFINITY, l = 0.f;
  const float c = a.scale * LOG2E;

  // two tiles of keys and of values in turn: one is read while the other one is on its way
  if (kend > 0) {
    fill<T, D, BK, 256>(L{tiles}, a.direct, kp, a.sk.t, 0, kend, a.d, tid);
    fill<T, D, BK, 256>(L{tiles + L::BYTES}, a.direct, vp, a.sv.t, 0, kend, a.d, tid);
  }
  int turn = 0;
  for (int key0 = 0; key0 < kend; key0 += BK, turn ^= 1) {
    const L kt = {tiles + turn * 2 * L::BYTES}, vt_ = {tiles + (turn * 2 + 1) * L::BYTES};
    arrive();
    __syncthreads();
    if (key0 + BK < kend) {
      lds_char *next = tiles + (turn ^ 1) * 2 * L::BYTES;
      fill<T, D, BK, 256>(L{next}, a.direct, kp, a.sk.t, key0 + BK, kend, a.d, tid);
      fill<T, D, BK, 256>(L{next + L::BYTES}, a.direct, vp, a.sv.t, key0 + BK, kend, a.d, tid);
    }
    if (qw >= qlen || (a.causal && key0 > pos0 + 31)) continue;
    f32x16 s[2] = {};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < NS; ++e) s[kb] = mma(kt.rows(32 * kb, e), qf[e], s[kb]);
    const Place p = place_of(key0, BK, pos0, 32, a.M, kend, a.causal);
    const float flat = p.near ? 0.f : bias[p.side];
    float cs = c, fs = flat;
    // a bias that swallows the scores (a table that masks by the type's lowest value) is added before the maximum is taken off
    if (p.near || p.mask || !(c > 0.f) || !__all(fabsf(flat) < 1e30f)) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) scores(s[kb], p, c, bias, flat, key0 + 32 * kb, pos, kend, a.causal);
      cs = 1.f;
      fs = 0.f;
    }
    online(s, o, cs, fs, m, l);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) add_values<T, NDB, LO>(vt_, 32 * kb, s[kb], o);
  }
  if (i >= a.Tq) return;
  l += __shfl_xor(l, 32);
  finish_rows<T>(a, o, m, l, i < qlen, b, h, i);
}

// ---------------------------------------------------------------------------------------------------------------------
// Forward, few rows (at most 32): the rows of `pack` query heads that share keys and values lie in one wave's 32 columns.
// The waves of a workgroup take the keys' tiles in turn, each with LDS of its own, and join at the end; long keys are also
// cut over workgroups (splits), joined by k_attn_join.
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
template <typename T, int D, int NWV>
__global__ __launch_bounds__(64 * NWV) void k_attn_few(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  using L = Tile<T, D, 32>;
  constexpr int NS = D / 16, NDB = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, w = wave_of();
  lds_char *own = (lds_char *)lds + w * 4 * L::BYTES;
  float *bias = (float *)(lds + NWV * 4 * L::BYTES);
  const int per_b = a.Hq / a.pack, b = blockIdx.x / per_b, h0 = (blockIdx.x % per_b) * a.pack, hk = h0 / a.G;
  const int row = lane & 31, hh = row / a.Tq, i = row - hh * a.Tq, h = h0 + hh;
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  const bool ok = hh < a.pack && i < qlen;
  const int pos = start + i;
  const int seen = qlen == 0 ? 0 : a.causal ? min(klen, max(0, start + qlen)) : klen;
  // equal shares of whole tiles
  const int tiles = (seen + 31) / 32, share = (tiles + a.splits - 1) / a.splits;
  const int t0 = min(tiles, (int)blockIdx.y * share), t1 = min(tiles, t0 + share);
  const T *kp = (const T *)a.k + b * a.sk.b + hk * a.sk.h, *vp = (const T *)a.v + b * a.sv.b + hk * a.sv.h;
  const T *qp = (const T *)a.q + b * a.sq.b + (long)i * a.sq.t + h * a.sq.h;

  // the bias by distance only where a tile of this piece lies within max_distance
  const Place whole = place_of(t0 * 32, (t1 - t0) * 32, start, a.Tq, a.M, seen, a.causal);
  if (whole.near)
    for (int x = 0; x < a.pack; ++x) load_bias(a, bias + x * bias_floats(a.M), h0 + x, tid, 64 * NWV);
  const float far_behind = ok ? bias_at(a, 0, h) : 0.f, far_ahead = ok ? bias_at(a, 2 * a.M, h) : 0.f;
  __syncthreads();
  const float *own_bias = bias + (ok ? hh : 0) * bias_floats(a.M) + PAD + a.M;
  frag<T> qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = row_frag<T>(qp, ok, 16 * s + 8 * half, a.d);
  f32x16 o[NDB] = {};
  float m = -INFINITY, l = 0.f;
  const float c = a.scale * LOG2E;
  int t = t0 + w, turn = 0;
  if (t < t1) {
    fill<T, D, 32, 64>(L{own}, a.direct, kp, a.sk.t, t * 32, seen, a.d, lane);
    fill<T, D, 32, 64>(L{own + L::BYTES}, a.direct, vp, a.sv.t, t * 32, seen, a.d, lane);
  }
  for (; t < t1; t += NWV, turn ^= 1) {
    const int key0 = t * 32;
    const L kt = {own + turn * 2 * L::BYTES}, vt_ = {own + (turn * 2 + 1) * L::BYTES};
    arrive();
    wave_sync();
    if (t + NWV < t1) {
      lds_char *next = own + (turn ^ 1) * 2 * L::BYTES;
      fill<T, D, 32, 64>(L{next}, a.direct, kp, a.sk.t, key0 + 32 * NWV, seen, a.d, lane);
      fill<T, D, 32, 64>(L{next + L::BYTES}, a.direct, vp, a.sv.t, key0 + 32 * NWV, seen, a.d, lane);
    }
    f32x16 s[1] = {};
#pragma unroll
    for (int e = 0; e < NS; ++e) s[0] = mma(kt.rows(0, e), qf[e], s[0]);
    const Place p = place_of(key0, 32, start, a.Tq, a.M, seen, a.causal);
    const float flat = p.side > 0 ? far_ahead : far_behind;
    float cs = c, fs = flat;
    if (p.near || p.mask || !(c > 0.f) || !__all(fabsf(flat) < 1e30f)) {
      if (p.near)
        finish_scores<true, true>(s[0], c, own_bias, 0.f, key0, pos, seen, a.causal);
      else
        finish_scores<false, true>(s[0], c, own_bias, flat, key0, pos, seen, a.causal);
      cs = 1.f;
      fs = 0.f;
    }
    online(s, o, cs, fs, m, l);
    if (a.out_lo)
      add_values<T, NDB, sizeof(T) == 2>(vt_, 0, s[0], o);
    else
      add_values<T, NDB, false>(vt_, 0, s[0], o);
  }
  l += __shfl_xor(l, 32);
  if (NWV > 1) {
    // the waves' results in LDS: m and l [NWV][32], o [NWV][D][32]
    __syncthreads();
    float *wm = (float *)lds, *wl = wm + NWV * 32, *wo = wl + NWV * 32;
    if (half == 0) {
      wm[w * 32 + row] = m;
      wl[w * 32 + row] = l;
    }
    if (w > 0)
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) wo[((w - 1) * D + 32 * db + 8 * (r >> 2) + 4 * half + (r & 3)) * 32 + row] = o[db][r];
    __syncthreads();
    if (w > 0) return;
    float mn = m;
#pragma unroll
    for (int x = 1; x < NWV; ++x) mn = fmaxf(mn, wm[x * 32 + row]);
    const float ref = mn == -INFINITY ? 0.f : mn;
    float f = __builtin_amdgcn_exp2f(m - ref);
    l *= f;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= f;
#pragma unroll
    for (int x = 1; x < NWV; ++x) {
      f = __builtin_amdgcn_exp2f(wm[x * 32 + row] - ref);
      l += f * wl[x * 32 + row];
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] += f * wo[((x - 1) * D + 32 * db + 8 * (r >> 2) + 4 * half + (r & 3)) * 32 + row];
    }
    m = mn;
  }
  if (hh >= a.pack) return;
  if (a.splits > 1) {
    float *p = a.part + (((long)b * a.Hq + h) * a.Tq + i) * a.splits * (D + 2) + (long)blockIdx.y * (D + 2);
    if (half == 0) {
      p[0] = ok ? m : -INFINITY;
      p[1] = ok ? l : 0.f;
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) p[2 + 32 * db + 8 * (r >> 2) + 4 * half + (r & 3)] = o[db][r];
    return;
  }
  finish_rows<T>(a, o, m, l, ok, b, h, i);
}

// One row's pieces: D threads.
template <typename T, int D>
__global__ __launch_bounds__(D < 64 ? 64 : D) void k_attn_join(AttnArgs a) {
  const long n = blockIdx.x;  // (b, h, i)
  const int b = (int)(n / ((long)a.Hq * a.Tq)), h = (int)(n / a.Tq % a.Hq), i = (int)(n % a.Tq), e = threadIdx.x;
  const float *p = a.part + n * a.splits * (D + 2);
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, p[(long)s * (D + 2)]);
  if (m != -INFINITY)
    for (int s = 0; s < a.splits; ++s) {
      const float ms = p[(long)s * (D + 2)];
      if (ms == -INFINITY) continue;
      const float f = __builtin_amdgcn_exp2f(ms - m);
      l += f * p[(long)s * (D + 2) + 1];
      if (e < D) o += f * p[(long)s * (D + 2) + 2 + e];
    }
  const float x = l == 0.f ? 0.f : o / l;
  if (e < a.d) {
    ((T *)a.out)[b * a.so.b + (long)i * a.so.t + h * a.so.h + e] = (T)x;
    if (a.out_lo) ((T *)a.out_lo)[b * a.so.b + (long)i * a.so.t + h * a.so.h + e] = (T)(x - (float)(T)x);
  }
  if (a.stats && e == 0) store_stats(a, b, h, i, m, l);
}

// ---------------------------------------------------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------------------------------------------------
// dq and D_i: as the forward pass, 128 queries of one head a workgroup.  dq takes D_i = do_i . (o_i + what its rounding left);
// the pass that follows takes the sum of p dp over the row, which this one forms anyway from unrounded p.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attn_dq(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  lds_char *tiles = (lds_char *)lds;
  using L = Tile<T, D, BK>;
  float *bias_lds = (float *)(lds + 4 * L::BYTES);
  constexpr int NS = D / 16, NDB = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int pairs = a.B * a.Hk, grp = blockIdx.x % pairs, b = grp / a.Hk, hk = grp % a.Hk, h = hk * a.G + blockIdx.x / pairs;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * 128, qw = q0 + wave_of() * 32, i = qw + (lane & 31);
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  const int pos0 = start + qw, pos = start + i;
  const int kend = q0 >= qlen ? 0 : a.causal ? min(klen, max(0, start + min(q0 + 128, qlen))) : klen;
  const T *kp = (const T *)a.k + b * a.sk.b + hk * a.sk.h, *vp = (const T *)a.v + b * a.sv.b + hk * a.sv.h;
  const bool ok = i < qlen;

  const float *bias = load_bias(a, bias_lds, h, tid, 256);
  const T *qp = (const T *)a.q + b * a.sq.b + (long)i * a.sq.t + h * a.sq.h;
  const T *dop = (const T *)a.dout + b * a.sdo.b + (long)i * a.sdo.t + h * a.sdo.h;
  const T *op = (const T *)a.o + b * a.so.b + (long)i * a.so.t + h * a.so.h;
  const T *lop = a.o_lo ? (const T *)a.o_lo + b * a.so.b + (long)i * a.so.t + h * a.so.h : nullptr;
  frag<T> qf[NS], df[NS];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int at = 16 * s + 8 * half;
    qf[s] = row_frag<T>(qp, ok, at, a.d);
    df[s] = row_frag<T>(dop, ok, at, a.d);
    const frag<T> of = row_frag<T>(op, ok, at, a.d);
    frag<T> lf = {};
    if (lop) lf = row_frag<T>(lop, ok, at, a.d);
#pragma unroll
    for (int e = 0; e < 8; ++e) delta += (float)df[s][e] * ((float)of[e] + (float)lf[e]);
  }
  delta += __shfl_xor(delta, 32);
  float2 st = {INFINITY, 0.f};  // p = 0 where there are no keys
  if (ok) {
    const long n = ((long)b * a.Hq + h) * a.Tq + i;
    st = *reinterpret_cast<const float2 *>(a.stats + 2 * n);
    if (st.x == -INFINITY) st.x = INFINITY;
  }
  f32x16 acc[NDB] = {};
  float pdp = 0.f;
  const float c = a.scale * LOG2E;
  // two tiles of keys and of values in turn: one is read while the other one is on its way
  if (kend > 0) {
    fill<T, D, BK, 256>(L{tiles}, a.direct, kp, a.sk.t, 0, kend, a.d, tid);
    fill<T, D, BK, 256>(L{tiles + L::BYTES}, a.direct, vp, a.sv.t, 0, kend, a.d, tid);
  }
  int turn = 0;
  for (int key0 = 0; key0 < kend; key0 += BK, turn ^= 1) {
    const L kt = {tiles + turn * 2 * L::BYTES}, vt_ = {tiles + (turn * 2 + 1) * L::BYTES};
    arrive();
    __syncthreads();
    if (key0 + BK < kend) {
      lds_char *next = tiles + (turn ^ 1) * 2 * L::BYTES;
      fill<T, D, BK, 256>(L{next}, a.direct, kp, a.sk.t, key0 + BK, kend, a.d, tid);
      fill<T, D, BK, 256>(L{next + L::BYTES}, a.direct, vp, a.sv.t, key0 + BK, kend, a.d, tid);
    }
    if (qw >= qlen || (a.causal && key0 > pos0 + 31)) continue;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int first = key0 + 32 * kb;
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        s = mma(kt.rows(32 * kb, e), qf[e], s);
        dp = mma(vt_.rows(32 * kb, e), df[e], dp);
      }
      const Place p = place_of(first, 32, pos0, 32, a.M, kend, a.causal);
      scores(s, p, c, bias, p.near ? 0.f : bias[p.side], first, pos, kend, a.causal);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p1 = __builtin_amdgcn_exp2f(s[r] - st.x - st.y);
        pdp = fmaf(p1, dp[r], pdp);
        s[r] = p1 * (dp[r] - delta);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const frag<T> sf = c_frag<T>(s, t);
#pragma unroll
        for (int db = 0; db < NDB; ++db) acc[db] = mma(kt.cols(32 * kb + 16 * t, db), sf, acc[db]);
      }
    }
  }
  if (i < a.Tq) {
    if (!ok)
#pragma unroll
      for (int db = 0; db < NDB; ++db) acc[db] = f32x16{};
    store_rows<T>((T *)a.dq + b * a.sdq.b + (long)i * a.sdq.t + h * a.sdq.h, a.d, acc, a.scale);
  }
  pdp += __shfl_xor(pdp, 32);
  if (ok && half == 0) a.delta[((long)b * a.Hq + h) * a.Tq + i] = pdp;
}

// Scores of a block of 32 queries and the wave's 32 keys (lane: one key) to base 2 with bias and mask; base: distance of row 0.
template <bool NEAR, bool MASK>
__device__ __forceinline__ void finish_back(f32x16 &s, float c, float flat, const float *bias, int base) {
  const int half = (threadIdx.x & 63) >> 5, at = afresh(base - 4 * half - 31);
  const float *b = bias + at;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int away = 31 - (8 * (r >> 2) + (r & 3));
    s[r] = fmaf(s[r], c, NEAR ? b[away] : flat);
    if (MASK && at + away > 0) s[r] = -INFINITY;
  }
}

// Rotation by N lanes inside each half of the wave: lane c receives lane (c + N) % 32.
template <int N>
__device__ __forceinline__ float rotate32(float x) {
  if (N == 0) return x;
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, x), 0xC000 | (N << 5)));
}
template <int R>
__device__ __forceinline__ void diagonal(const f32x16 &s, int col, float &here, float &below) {
  constexpr int N = 8 * (R >> 2) + (R & 3);
  const float v = rotate32<N>(s[R]), in = col + N < 32 ? v : 0.f;
  here += in;
  below += v - in;
  if constexpr (R < 15) diagonal<R + 1>(s, col, here, below);
}

// dk, dv and the bias gradient by distance: a workgroup takes 128 keys of one key head, a wave 32 of them, and walks over the
// queries of the heads that share it (share == 1: of all G of them; share == G: of one, leaving fp32 parts for k_attn_dkv_sum).
// The bias gradient: with its registers rotated by their row, a block's ds of one distance lie in one lane; the sums of the
// block's lower 32 distances are the next block's upper ones and move on in registers, the upper ones are done and added to
// the wave's array.  (One addition in LDS a block; added one by one, sixteen a block, they took two thirds of the kernel's
// time where all tiles are near: 16 x 196 tokens, 48 us of which 30.)
// Widths of 256 bytes: the keys' fragments are read from LDS, which leaves two waves a SIMD.
template <typename T, int D>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void k_attn_dkv(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  lds_char *tiles = (lds_char *)lds;
  constexpr int BQ = 32, NS = D / 16, NDB = D / 32;
  using L = Tile<T, D, BQ>;
  const int W = 2 * a.M + 1;
  constexpr bool KEYS_IN_LDS = sizeof(T) == 2 && D == 128;
  using LK = Tile<T, D, KEYS_IN_LDS ? 128 : 32>;
  const LK kt = {tiles + 4 * L::BYTES};
  float *rows = (float *)(lds + 4 * L::BYTES + (KEYS_IN_LDS ? LK::BYTES : 0));  // [2][3][BQ]: maximum, log2 of the sum, D
  float *bias_lds = rows + 6 * BQ, *hist_all = bias_lds + W + 2 * PAD, *hist = hist_all + (threadIdx.x >> 6) * W;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int pairs = a.B * a.Hk, grp = blockIdx.x % pairs, b = grp / a.Hk, hk = grp % a.Hk, part = blockIdx.x / pairs;
  const int k0 = blockIdx.y * 128, kw = k0 + wave_of() * 32, key = kw + (lane & 31);
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  // queries before the first key's own place see none of the workgroup's keys
  const int qfirst = (a.causal ? min(max(0, k0 - start), a.Tq) : 0) & ~(BQ - 1), qend = k0 < klen ? qlen : 0;
  const bool ok = key < klen;
  const T *kp = (const T *)a.k + b * a.sk.b + (long)key * a.sk.t + hk * a.sk.h;
  const T *vp = (const T *)a.v + b * a.sv.b + (long)key * a.sv.t + hk * a.sv.h;
  frag<T> kf[KEYS_IN_LDS ? 1 : NS], vf[NS];
  if constexpr (KEYS_IN_LDS) {
    if (k0 < klen) {
      fill<T, D, 128, 256>(kt, a.direct, (const T *)a.k + b * a.sk.b + hk * a.sk.h, a.sk.t, k0, klen, a.d, tid);
      if (a.d < D) {  // the queries' tiles repeat a chunk behind d elements: here they must meet zeros
        arrive();
        __syncthreads();
        constexpr int EPC = LK::EPC, CPR = LK::CPR;
        const int c0 = (a.d + EPC - 1) / EPC;
        for (int x = tid; x < 128 * (CPR - c0); x += 256)
          *(__attribute__((address_space(3))) u32x4 *)kt.chunk(x / (CPR - c0), c0 + x % (CPR - c0)) = u32x4{0, 0, 0, 0};
      }
    }
  } else {
#pragma unroll
    for (int s = 0; s < NS; ++s) kf[s] = row_frag<T>(kp, ok, 16 * s + 8 * half, a.d);
  }
#pragma unroll
  for (int s = 0; s < NS; ++s) vf[s] = row_frag<T>(vp, ok, 16 * s + 8 * half, a.d);
  f32x16 dk[NDB] = {}, dv[NDB] = {};
  const float c = a.scale * LOG2E;
  const int heads = a.G / a.share;
  for (int g = part * heads; g < (part + 1) * heads; ++g) {
    const int h = hk * a.G + g;
    const T *qp = (const T *)a.q + b * a.sq.b + h * a.sq.h, *dop = (const T *)a.dout + b * a.sdo.b + h * a.sdo.h;
    const float2 *statp = reinterpret_cast<const float2 *>(a.stats) + ((long)b * a.Hq + h) * a.Tq;
    const float *deltap = a.delta + ((long)b * a.Hq + h) * a.Tq;
    float behind = 0.f, ahead = 0.f, carry = 0.f;
    const auto add_distance = [&](int away, float x) {
      if (away <= -a.M)
        behind += x;
      else if (away >= a.M)
        ahead += x;
      else
        unsafeAtomicAdd(hist + away + a.M, x);
    };
    __syncthreads();
    const float *bias = load_bias(a, bias_lds, h, tid, 256);
    if (a.hist)
      for (int x = tid; x < 4 * W; x += 256) hist_all[x] = 0.f;
    float2 st = {INFINITY, 0.f};  // p = 0 where there are no keys
    float de = 0.f;
    const auto stats_of = [&](int r0) {
      st = float2{INFINITY, 0.f};
      de = 0.f;
      if (tid < BQ && r0 + tid < qend) {
        st = statp[r0 + tid];
        de = deltap[r0 + tid];
        if (st.x == -INFINITY) st.x = INFINITY;
      }
    };
    if (qfirst < qend) {
      fill<T, D, BQ, 256>(L{tiles}, a.direct, qp, a.sq.t, qfirst, qend, a.d, tid);
      fill<T, D, BQ, 256>(L{tiles + L::BYTES}, a.direct, dop, a.sdo.t, qfirst, qend, a.d, tid);
      stats_of(qfirst);
    }
    int turn = 0;
    for (int r0 = qfirst; r0 < qend; r0 += BQ, turn ^= 1) {
      const L qt = {tiles + turn * 2 * L::BYTES}, dt = {tiles + (turn * 2 + 1) * L::BYTES};
      const float *row_max = rows + turn * 3 * BQ;
      if (tid < BQ) {
        float *r = rows + turn * 3 * BQ + tid;
        r[0] = st.x;
        r[BQ] = st.y;
        r[2 * BQ] = de;
      }
      arrive();
      __syncthreads();
      if (r0 + BQ < qend) {
        lds_char *next = tiles + (turn ^ 1) * 2 * L::BYTES;
        fill<T, D, BQ, 256>(L{next}, a.direct, qp, a.sq.t, r0 + BQ, qend, a.d, tid);
        fill<T, D, BQ, 256>(L{next + L::BYTES}, a.direct, dop, a.sdo.t, r0 + BQ, qend, a.d, tid);
        stats_of(r0 + BQ);
      }
      if (kw >= klen || (a.causal && kw > start + r0 + BQ - 1)) continue;
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        if constexpr (KEYS_IN_LDS)
          s = mma(qt.rows(0, e), kt.rows(32 * wave_of(), e), s);
        else
          s = mma(qt.rows(0, e), kf[e], s);
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // no more fragments in flight than registers hold
      }
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        dp = mma(dt.rows(0, e), vf[e], dp);
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_sched_barrier(0);
      // distance of register r: key - start - query; its bounds over the block decide the variant
      const int base = key - start - r0, lo = kw - start - r0 - 31, hi = kw + 31 - start - r0;
      const bool near = lo < a.M && hi > -a.M;
      const float flat = bias[lo >= a.M ? a.M : -a.M];
      const bool mask = a.causal && hi > 0;
      if (near) {
        if (mask)
          finish_back<true, true>(s, c, 0.f, bias, base);
        else
          finish_back<true, false>(s, c, 0.f, bias, base);
      } else {
        if (mask)
          finish_back<false, true>(s, c, flat, bias, base);
        else
          finish_back<false, false>(s, c, flat, bias, base);
      }
      f32x16 p;
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        __builtin_amdgcn_sched_barrier(0);  // the next rows' statistics are not read before these are used
        const float *row = row_max + 8 * r4 + 4 * half;
        const float4 mx = *reinterpret_cast<const float4 *>(row), lg = *reinterpret_cast<const float4 *>(row + BQ);
        const float4 dd = *reinterpret_cast<const float4 *>(row + 2 * BQ);
        const float mv[4] = {mx.x, mx.y, mx.z, mx.w}, lv[4] = {lg.x, lg.y, lg.z, lg.w}, ev[4] = {dd.x, dd.y, dd.z, dd.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * r4 + j;
          p[r] = __builtin_amdgcn_exp2f(s[r] - mv[j] - lv[j]);
          s[r] = p[r] * (dp[r] - ev[j]);
        }
      }
      if (near) {
        if (a.hist) {
          if (!ok)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
          float here = carry, below = 0.f;
          diagonal<0>(s, lane & 31, here, below);
          add_distance(kw - start - r0 + (lane & 31) - 4 * half, here);
          carry = below;
        }
      } else {
        float all = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) all += s[r];
        if (!ok) all = 0.f;
        if (lo >= a.M)
          ahead += all;
        else
          behind += all + carry;  // what a near block before left lies behind, too
        carry = 0.f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        const frag<T> pf = c_frag<T>(p, t), sf = c_frag<T>(s, t);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          dv[db] = mma(dt.cols(16 * t, db), pf, dv[db]);
          dk[db] = mma(qt.cols(16 * t, db), sf, dk[db]);
        }
      }
    }
    if (a.hist) {
      add_distance(kw - start - (qfirst + (max(qend - qfirst, 0) + BQ - 1) / BQ * BQ) + (lane & 31) - 4 * half, carry);
      behind = wave_sum(behind);
      ahead = wave_sum(ahead);
      wave_sync();
      if (lane == 0) {
        hist[0] += behind;
        hist[2 * a.M] += ahead;
      }
      __syncthreads();
      // rows of one head lie together: [Hq][B * key tiles][W]
      float *out = a.hist + ((long)h * a.hist_rows + (long)b * gridDim.y + blockIdx.y) * W;
      for (int x = tid; x < W; x += 256) out[x] = (hist_all[x] + hist_all[W + x]) + (hist_all[2 * W + x] + hist_all[3 * W + x]);
    }
  }
  if (key >= a.Tk) return;
  if (!ok)
#pragma unroll
    for (int db = 0; db < NDB; ++db) dk[db] = dv[db] = f32x16{};
  if (a.share > 1) {
    float *p = a.part + ((((long)part * a.B + b) * a.Hk + hk) * a.Tk + key) * 2 * a.d;
    store_rows<float>(p, a.d, dk, a.scale);
    store_rows<float>(p + a.d, a.d, dv, 1.f);
    return;
  }
  store_rows<T>((T *)a.dk + b * a.sdk.b + (long)key * a.sdk.t + hk * a.sdk.h, a.d, dk, a.scale);
  store_rows<T>((T *)a.dv + b * a.sdv.b + (long)key * a.sdv.t + hk * a.sdv.h, a.d, dv, 1.f);
}

// dk and dv from the query heads' parts, [G][B][Hk][Tk][2][d].
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_sum(AttnArgs a) {
  const long rows = (long)a.B * a.Hk * a.Tk, n = (long)blockIdx.x * 256 + threadIdx.x;
  if (n >= rows * 2 * a.d) return;
  float t = 0.f;
  for (int g = 0; g < a.share; ++g) t += a.part[g * rows * 2 * a.d + n];
  const long row = n / (2 * a.d);
  const int e = (int)(n - row * 2 * a.d), b = (int)(row / ((long)a.Hk * a.Tk)), hk = (int)(row / a.Tk % a.Hk), key = (int)(row % a.Tk);
  if (e < a.d)
    ((T *)a.dk)[b * a.sdk.b + (long)key * a.sdk.t + hk * a.sdk.h + e] = (T)t;
  else
    ((T *)a.dv)[b * a.sdv.b + (long)key * a.sdv.t + hk * a.sdv.h + e - a.d] = (T)t;
}

// The bias gradient of one distance and head: the workgroups' sums, in double and in order.
__global__ __launch_bounds__(1024) void k_attn_distances(AttnArgs a) {
  __shared__ double s[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, W = 2 * a.M + 1, x = blockIdx.x * 64 + lane, h = blockIdx.y;
  double t = 0;
  if (x < W)
    for (int r = w; r < a.hist_rows; r += 16) t += a.hist[((long)h * a.hist_rows + r) * W + x];
  s[w][lane] = t;
  __syncthreads();
  if (w == 0 && x < W) {
    t = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) t += s[j][lane];
    a.dist[(long)h * W + x] = t;
  }
}
// The distances of one bucket.
__global__ __launch_bounds__(64) void k_attn_buckets(AttnArgs a) {
  const int bucket = blockIdx.x, h = blockIdx.y, W = 2 * a.M + 1;
  double t = 0;
  for (int x = threadIdx.x; x < W; x += 64)
    if (a.map[x] == bucket) t += a.dist[(long)h * W + x];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
  if (threadIdx.x == 0) a.dtable[(long)bucket * a.Hq + h] = (float)t;
}

// ---------------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------------
int check_args(const vt_relpos_attention *a) {
  if (!a || a->B < 1 || a->Tq < 1 || a->Tk < 1 || a->Hq < 1 || a->Hk < 1 || a->d < 1 || a->num_buckets < 1 || a->max_distance < 0 ||
      !a->map || !a->table || !a->q || !a->k || !a->v || !(a->scale > -INFINITY && a->scale < INFINITY))
    return VT_EINVAL;
  if (a->dtype != VT_F32 && a->dtype != VT_BF16 && a->dtype != VT_F16) return VT_EUNSUPPORTED;
  if (a->d > 128 || a->max_distance > 2048 || a->Hq % a->Hk != 0) return VT_EUNSUPPORTED;
  // grids, and positions within int
  if (a->Tq > 65535 * 128 || a->Tk > (1 << 29) || (long)a->B * a->Hq * (a->Tq <= 32 ? a->Tq : 1) >= (1L << 31)) return VT_EUNSUPPORTED;
  return 0;
}
// Whether rows start on 16-byte boundaries, hold whole chunks of 16 bytes and lie within 2^31 bytes a tile of 128.
bool aligned(const vt_relpos_attention *a, const void *p, const vt_strides &s) {
  const long e = a->dtype == VT_F32 ? 4 : 8;
  return a->d % e == 0 && s.b % e == 0 && s.t % e == 0 && s.h % e == 0 && ((uintptr_t)p & 15) == 0 && s.t >= 0 && s.t < (1L << 22);
}
AttnArgs kernel_args(const vt_relpos_attention *a) {
  AttnArgs k = {};
  k.direct = aligned(a, a->q, a->sq) && aligned(a, a->k, a->sk) && aligned(a, a->v, a->sv);
  k.q = a->q;
  k.k = a->k;
  k.v = a->v;
  k.sq = a->sq;
  k.sk = a->sk;
  k.sv = a->sv;
  k.map = a->map;
  k.table = a->table;
  k.q_start = a->q_start;
  k.q_len = a->q_len;
  k.k_len = a->k_len;
  k.B = a->B;
  k.Tq = a->Tq;
  k.Tk = a->Tk;
  k.Hq = a->Hq;
  k.Hk = a->Hk;
  k.d = a->d;
  k.G = a->Hq / a->Hk;
  k.causal = a->causal != 0;
  k.nb = a->num_buckets;
  k.M = a->max_distance;
  k.scale = a->scale;
  return k;
}
int width_of(const vt_relpos_attention *a) { return a->d <= 32 ? 32 : a->d <= 64 ? 64 : 128; }
int size_of(const vt_relpos_attention *a) { return a->dtype == VT_F32 ? 4 : 2; }

// At most 32 rows of queries share one read of the keys: all heads of a key head where they and their bias fit.
struct Few {
  bool use;
  int pack, waves, splits, lds;
};
Few few_of(const vt_relpos_attention *a) {
  Few f = {};
  if (a->Tq > 32) return f;
  f.use = true;
  const int G = a->Hq / a->Hk, W = 2 * a->max_distance + 1 + 2 * PAD;
  f.pack = G * a->Tq <= 32 && (long)G * W <= 8192 ? G : 1;
  const int tiles = (a->Tk + 31) / 32;
  f.waves = tiles == 1 ? 1 : a->dtype == VT_F32 && a->d > 64 ? 2 : 4;  // what LDS holds
  const long groups = (long)a->B * (a->Hq / f.pack);
  // pieces of at least one tile a wave, as many as bring four workgroups to a compute unit
  long splits = (1024 + groups - 1) / groups, most = (tiles + f.waves - 1) / f.waves;
  f.splits = (int)(splits < most ? splits : most);
  if (f.splits > 256) f.splits = 256;
  const int D = width_of(a), tile = 32 * D * size_of(a), join = 4 * (2 * f.waves * 32 + (f.waves - 1) * D * 32);
  f.lds = 4 * f.waves * tile + 4 * f.pack * W;
  if (f.lds < join) f.lds = join;
  return f;
}
long few_floats(const vt_relpos_attention *a) {
  const Few f = few_of(a);
  return f.use && f.splits > 1 ? (long)a->B * a->Hq * a->Tq * f.splits * (width_of(a) + 2) : 0;
}

template <typename F>
int set_lds(F *f, int bytes) {
  return bytes > 65536 ? (int)hipFuncSetAttribute((const void *)f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) : 0;
}

template <typename T, int D>
int launch_fwd(const vt_relpos_attention *a, const AttnArgs &k, hipStream_t s) {
  const Few f = few_of(a);
  if (f.use) {
    AttnArgs n = k;
    n.splits = f.splits;
    n.pack = f.pack;
    const dim3 grid(a->B * (a->Hq / f.pack), f.splits);
#define VT_FEW(NWV)                                                                    \
  if (f.waves == (NWV)) {                                                              \
    if (int rc = set_lds(k_attn_few<T, D, NWV>, f.lds)) return rc;                     \
    hipLaunchKernelGGL((k_attn_few<T, D, NWV>), grid, dim3(64 * (NWV)), f.lds, s, n);  \
  }
    VT_FEW(1)
    if constexpr (sizeof(T) == 4 && D == 128) {
      VT_FEW(2)
    } else {
      VT_FEW(4)
    }
#undef VT_FEW
    if (f.splits > 1)
      hipLaunchKernelGGL((k_attn_join<T, D>), dim3((unsigned)((long)a->B * a->Hq * a->Tq)), dim3(D < 64 ? 64 : D), 0, s, n);
  } else {
    const int lds = 4 * Tile<T, D, BK>::BYTES + 4 * (2 * a->max_distance + 1 + 2 * PAD);
    const dim3 grid(a->B * a->Hq, (a->Tq + 127) / 128);
    if (k.out_lo) {
      if (int rc = set_lds(k_attn_fwd<T, D, sizeof(T) == 2>, lds)) return rc;
      hipLaunchKernelGGL((k_attn_fwd<T, D, sizeof(T) == 2>), grid, dim3(256), lds, s, k);
    } else {
      if (int rc = set_lds(k_attn_fwd<T, D, false>, lds)) return rc;
      hipLaunchKernelGGL((k_attn_fwd<T, D, false>), grid, dim3(256), lds, s, k);
    }
  }
  VT_CHECK_LAUNCH();
  return 0;
}

template <typename T, int D>
int launch_bwd(const vt_relpos_attention *a, const AttnArgs &k, hipStream_t s) {
  const int W = 2 * a->max_distance + 1;
  const int lds_q = 4 * Tile<T, D, BK>::BYTES + 4 * (W + 2 * PAD), keys = sizeof(T) == 2 && D == 128 ? Tile<T, D, 128>::BYTES : 0;
  const int lds_k = 4 * Tile<T, D, 32>::BYTES + keys + 4 * (6 * 32 + 5 * W + 2 * PAD);
  if (int rc = set_lds(k_attn_dq<T, D>, lds_q)) return rc;
  if (int rc = set_lds(k_attn_dkv<T, D>, lds_k)) return rc;
  hipLaunchKernelGGL((k_attn_dq<T, D>), dim3(a->B * a->Hq, (a->Tq + 127) / 128), dim3(256), lds_q, s, k);
  hipLaunchKernelGGL((k_attn_dkv<T, D>), dim3(a->B * a->Hk * k.share, (a->Tk + 127) / 128), dim3(256), lds_k, s, k);
  if (k.share > 1) {
    const long n = (long)a->B * a->Hk * a->Tk * 2 * a->d;
    hipLaunchKernelGGL((k_attn_dkv_sum<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, k);
  }
  if (k.dtable) {
    hipLaunchKernelGGL(k_attn_distances, dim3((W + 63) / 64, a->Hq), dim3(1024), 0, s, k);
    hipLaunchKernelGGL(k_attn_buckets, dim3(a->num_buckets, a->Hq), dim3(64), 0, s, k);
  }
  VT_CHECK_LAUNCH();
  return 0;
}

#define VT_WIDTH(FN)                                            \
  VT_DISPATCH_TYPE(a->dtype, {                                  \
    if (a->d <= 32) return (FN<T, 32>(a, k, (hipStream_t)s));   \
    if (a->d <= 64) return (FN<T, 64>(a, k, (hipStream_t)s));   \
    return (FN<T, 128>(a, k, (hipStream_t)s));                  \
  })

// Scratch of the backward pass: delta [B, Hq, Tq], distances in double [Hq, W], the workgroups' sums [Hq, rows, W].
struct BwdScratch {
  long delta, dist, hist, part, total;
  int rows, share;
};
BwdScratch bwd_scratch(const vt_relpos_attention *a) {
  BwdScratch b;
  const long W = 2L * a->max_distance + 1;
  b.rows = a->B * ((a->Tk + 127) / 128);
  b.delta = 0;
  b.dist = ((long)a->B * a->Hq * a->Tq + 3) & ~3L;
  b.hist = b.dist + ((2 * a->Hq * W + 3) & ~3L);
  b.part = b.hist + (((long)a->Hq * b.rows * W + 3) & ~3L);
  // a workgroup a query head where the key heads alone would not give every compute unit four: their parts cost a write and a
  // read in fp32, the walk over all G heads leaves compute units idle (and, causal, waiting for the longest)
  b.share = a->Hq / a->Hk > 1 && (long)a->Hk * b.rows < 1024 ? a->Hq / a->Hk : 1;
  b.total = b.part + (b.share > 1 ? (long)b.share * a->B * a->Hk * a->Tk * 2 * a->d : 0);
  return b;
}

}  // namespace
}  // namespace vt

using namespace vt;

extern "C" int vt_relpos_buckets(int num_buckets, int max_distance, int bidirectional, int *map) {
  const int side = bidirectional ? num_buckets / 2 : num_buckets, single = side / 2, ranges = side - single;
  if (!map || num_buckets < (bidirectional ? 4 : 2) || num_buckets > 256 || (bidirectional && num_buckets % 2) || max_distance < single ||
      max_distance > 2048)
    return VT_EINVAL;
  // whole numbers of as many 32-bit words as (2^11 + 1)^ranges needs: ranges <= 128
  constexpr int WORDS = 64;
  struct Big {
    uint32_t w[WORDS] = {1};
    void times(uint32_t f) {
      uint64_t c = 0;
      for (int i = 0; i < WORDS; ++i) {
        c += (uint64_t)w[i] * f;
        w[i] = (uint32_t)c;
        c >>= 32;
      }
    }
    bool at_least(const Big &o) const {
      for (int i = WORDS - 1; i >= 0; --i)
        if (w[i] != o.w[i]) return w[i] > o.w[i];
      return true;
    }
  };
  int m = 0;  // ranges whose lower border lies at or below the distance
  for (int n = 0; n <= max_distance; ++n) {
    int bucket = n;
    if (n >= single) {
      for (; m + 1 < ranges; ++m) {
        Big l, r;
        for (int i = 0; i < ranges; ++i) {
          l.times((uint32_t)n);
          r.times((uint32_t)(i < m + 1 ? max_distance : single));
        }
        if (!l.at_least(r)) break;
      }
      bucket = single + m;
    }
    map[max_distance - n] = bucket;
    if (n > 0) map[max_distance + n] = bidirectional ? bucket + side : 0;
  }
  return 0;
}

extern "C" long vt_relpos_attention_fwd_scratch_floats(const vt_relpos_attention *a) {
  return check_args(a) != 0 ? 0 : few_floats(a);
}

extern "C" int vt_relpos_attention_fwd(const vt_relpos_attention *a, void *out, vt_strides so, void *out_lo, float *stats,
                                       float *scratch, long scratch_floats, vt_stream s) {
  const int rc = check_args(a);
  if (rc != 0) return rc;
  if (!out || (out_lo && !stats) || ((uintptr_t)stats & 7)) return VT_EINVAL;
  if (scratch_floats < few_floats(a)) return VT_ELIMIT;
  if (few_floats(a) > 0 && !scratch) return VT_EINVAL;
  AttnArgs k = kernel_args(a);
  k.out = out;
  k.out_lo = a->dtype == VT_F32 ? nullptr : out_lo;
  k.so = so;
  k.stats = stats;
  k.part = scratch;
  VT_WIDTH(launch_fwd);
  return 0;
}

extern "C" long vt_relpos_attention_bwd_scratch_floats(const vt_relpos_attention *a) {
  return check_args(a) != 0 ? 0 : bwd_scratch(a).total;
}

extern "C" int vt_relpos_attention_bwd(const vt_relpos_attention *a, const void *out, vt_strides so, const void *out_lo,
                                       const float *stats, const void *dout, vt_strides sdo, void *dq, vt_strides sdq, void *dk,
                                       vt_strides sdk, void *dv, vt_strides sdv, float *dtable, float *scratch,
                                       long scratch_floats, vt_stream s) {
  const int rc = check_args(a);
  if (rc != 0) return rc;
  if (!out || !stats || ((uintptr_t)stats & 7) || !dout || !dq || !dk || !dv || !scratch || ((uintptr_t)scratch & 15) || (a->dtype != VT_F32 && !out_lo))
    return VT_EINVAL;
  if (a->Tk > 65535 * 128) return VT_EUNSUPPORTED;
  const BwdScratch b = bwd_scratch(a);
  if (scratch_floats < b.total) return VT_ELIMIT;
  AttnArgs k = kernel_args(a);
  k.o = out;
  k.o_lo = a->dtype == VT_F32 ? nullptr : out_lo;
  k.so = so;
  k.stats = const_cast<float *>(stats);
  k.dout = dout;
  k.sdo = sdo;
  k.dq = dq;
  k.sdq = sdq;
  k.dk = dk;
  k.sdk = sdk;
  k.dv = dv;
  k.sdv = sdv;
  k.dtable = dtable;
  k.delta = scratch + b.delta;
  k.dist = reinterpret_cast<double *>(scratch + b.dist);
  k.hist = dtable ? scratch + b.hist : nullptr;
  k.hist_rows = b.rows;
  k.share = b.share;
  k.part = scratch + b.part;
  k.direct = k.direct && aligned(a, dout, sdo);
  VT_WIDTH(launch_bwd);
  return 0;
}
