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
// The forward pass multiplies p with v in two parts, its value rounded to the inputs' type and what that left (2^-17 in bf16;
// fp32: exact products): the output is off by its own rounding alone, the same bytes for training and inference, and
// D = do . o carries no error of p into every gradient.  The backward pass rounds p and ds to the inputs' type for the second
// products where queries are more than 32 and the caller does not ask for more, which adds to a gradient as much as its own
// rounding does (bf16, 2 x 4096 causal: 2.4e-3 from 64 bits against 1.7e-3); in two parts the pass takes 901 us instead of 629
// (16 x 196: 44 instead of 41).
#include "vtcnn_attn.h"

namespace vt {
namespace {

// A tile beyond max_distance keeps its scores apart from its one bias, which is taken off together with the maximum.  That is
// more exact than adding the bias to each score, as tiles within max_distance and the backward pass do, and so only done where
// the addition rounds by no more than the scores' own size costs (2^-18): a finite bias that masks (-1e4, -1e9) swallows the
// scores' low bits, and the tiles of a row that sees nothing else have to agree on what is left.
constexpr float FLAT_MAX = 128.f;

// One key tile's step of the running softmax: the scores s c + f (base 2; c > 0) become p.  m is a reference near the maximum
// rather than the maximum: o and l are brought to a new one only where a score exceeds it by more than 8 (fp16, whose reference is
// set 13 below: 15), so p reaches up to 2^8 (2^15), which costs neither fp32 sums nor a rounded p anything, and most tiles rescale nothing.
template <typename T, int NKB, int NDB>
__device__ __forceinline__ void online(f32x16 (&s)[NKB], f32x16 (&o)[NDB], float c, float f, float &m, float &l) {
  float t = max16(s[0]);
#pragma unroll
  for (int b = 1; b < NKB; ++b) t = fmaxf(t, max16(s[b]));
  t = fmaf(fmaxf(t, __shfl_xor(t, 32)), c, f);
  if (__any(t - m > FWD_MOST<T>)) {
    const float mn = fmaxf(m, reference<T>(t)), w = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
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

// o += v^T p over a block of 32 keys, p of 16 bits in two parts.
template <typename T, int NDB, typename L>
__device__ __forceinline__ void add_values(const L &v, int row0, const f32x16 &p, f32x16 (&o)[NDB]) {
  constexpr bool LO = sizeof(T) == 2;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const frag<T> pf = c_frag<T>(p, t);
    frag<T> lf;
    if (LO) lf = c_rest<T>(p, t, pf);
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const frag<T> vf = v.cols(row0 + 16 * t, db);
      o[db] = mma(vf, pf, o[db]);
      if (LO) o[db] = mma(vf, lf, o[db]);
    }
  }
}

// Statistics of a row: its reference (at most 8 below its maximum, fp16 15) and log2 of the sum of 2^(x - reference), apart, so
// that 2^(x - reference - log2 sum) loses nothing to a large maximum.
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

// Joins the partial softmaxes of N waves a group (wave w: part w / GROUPS of group w % GROUPS) over the same queries in part 0's
// registers.  f: LDS, every wave of the workgroup being done with what it held.  All waves call it.
template <int NDB, int N, int GROUPS>
__device__ __forceinline__ void join_waves(float *f, int w, f32x16 (&o)[NDB], float &m, float &l) {
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, part = w / GROUPS, g = w % GROUPS;
  float *wm = f, *wl = f + N * GROUPS * 32, *wo = wl + N * GROUPS * 32;
  if (half == 0) {
    wm[w * 32 + col] = m;
    wl[w * 32 + col] = l;
  }
  if (part > 0)
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) wo[((((part - 1) * GROUPS + g) * NDB + db) * 16 + r) * 64 + lane] = o[db][r];
  __syncthreads();
  if (part > 0) return;
  float mn = m;
#pragma unroll
  for (int x = 1; x < N; ++x) mn = fmaxf(mn, wm[(x * GROUPS + g) * 32 + col]);
  const float ref = mn == -INFINITY ? 0.f : mn;
  float k = __builtin_amdgcn_exp2f(m - ref);
  l *= k;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] *= k;
#pragma unroll
  for (int x = 1; x < N; ++x) {
    k = __builtin_amdgcn_exp2f(wm[(x * GROUPS + g) * 32 + col] - ref);
    l += k * wl[(x * GROUPS + g) * 32 + col];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] += k * wo[((((x - 1) * GROUPS + g) * NDB + db) * 16 + r) * 64 + lane];
  }
  m = mn;
}

// ---------------------------------------------------------------------------------------------------------------------
// Forward, many rows: a wave takes 32 queries of one head; a workgroup's waves share the key tiles.  SPLIT 1: every wave has
// queries of its own and takes all 64 keys of a tile.  SPLIT 2: two waves take 32 keys each of every tile for the same queries
// and join at the end: half the time of a tile's chain of dependent steps, for grids that leave compute units idle or wait for
// their longest row.  (2 x 4096 causal, 16 heads of 128 over 4, bf16: 234 us, 206 GFLOP of products, p in two parts, at
// 880 TFLOP/s; a large library product reaches 1171.)
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int D, int DC, int SPLIT>
__global__ __launch_bounds__((64 * RingShape<T, D>::WAVES), sizeof(T) == 2 ? 2 : 1) void k_attn_fwd(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  lds_char *tiles = (lds_char *)lds;
  using L = Tile<T, D, BK>;
  constexpr int NW = RingShape<T, D>::WAVES, NT = 64 * NW;
  float *bias_lds = (float *)(lds + RingShape<T, D>::BYTES);
  constexpr int NS = DC / 16, NDB = DC / 32, NKB = 2 / SPLIT, ROWS = 32 * NW / SPLIT;
  const int tid = threadIdx.x, lane = tid & 63;
  const int pairs = a.B * a.Hk, grp = blockIdx.x % pairs, b = grp / a.Hk, hk = grp % a.Hk, h = hk * a.G + blockIdx.x / pairs;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * ROWS, w = wave_of(), qw = q0 + (w % (NW / SPLIT)) * 32, i = qw + (lane & 31);
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  const int pos0 = start + qw, pos = start + i;
  // keys beyond the last query's own are seen by none of the workgroup's
  const int kend = q0 >= qlen ? 0 : a.causal ? min(klen, max(0, start + min(q0 + ROWS, qlen))) : klen;
  const T *kp = (const T *)a.k + b * a.sk.b + hk * a.sk.h, *vp = (const T *)a.v + b * a.sv.b + hk * a.sv.h;
  const T *qp = (const T *)a.q + b * a.sq.b + h * a.sq.h;

  KeyRing<T, D, NT> ring(a, tiles, kp, vp, kend, tid);
  BiasLoad bl(a, bias_lds, h, 1, tid, NT);
  frag<T> qf[NS];
  bl.map();
  load_frags<T, NS>(qf, qp + (long)i * a.sq.t, i < qlen, (const T *)a.q, a.d);
  bl.table();
  const float *bias = bl.store();
  clear_frags<T, NS>(qf, i < qlen, a.d);
  f32x16 o[NDB] = {};
  float m = -INFINITY, l = 0.f;
  const float c = a.scale * LOG2E;

  for (int t = 0; t < ring.n; ++t) {
    const int key0 = t * BK;
    L kt, vt_;
    ring.step(t, kt, vt_);
    if (qw >= qlen || (a.causal && key0 > pos0 + 31)) continue;
    const int kb0 = SPLIT == 1 ? 0 : w / (NW / SPLIT), first = key0 + 32 * kb0;
    if (SPLIT > 1 && (first >= kend || (a.causal && first > pos0 + 31))) continue;
    f32x16 s[NKB] = {};
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int e = 0; e < NS; ++e) s[kb] = mma(kt.rows(32 * (kb0 + kb), e), qf[e], s[kb]);
    const Place p = place_of(first, 32 * NKB, pos0, 32, a.M, kend, a.causal);
    const float flat = p.near ? 0.f : bias[p.side];
    float cs = c, fs = flat;
    if (p.near || p.mask || !(c > 0.f) || !__all(fabsf(flat) < FLAT_MAX)) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) scores(s[kb], p, c, bias, flat, first + 32 * kb, pos, kend, a.causal);
      cs = 1.f;
      fs = 0.f;
    }
    online<T>(s, o, cs, fs, m, l);
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) add_values<T, NDB>(vt_, 32 * (kb0 + kb), s[kb], o);
  }
  l += __shfl_xor(l, 32);
  if constexpr (SPLIT > 1) {
    __syncthreads();
    join_waves<NDB, 2, NW / 2>((float *)lds, w, o, m, l);
    if (w >= NW / 2) return;
  }
  if (i >= a.Tq) return;
  finish_rows<T>(a, o, m, l, i < qlen, b, h, i);
}

// ---------------------------------------------------------------------------------------------------------------------
// Forward, few rows (at most 32): the rows of `pack` query heads that share keys and values lie in one wave's 32 columns.
// The waves of a workgroup take the keys' tiles in turn, each with LDS of its own, and join at the end; long keys are also
// cut over workgroups (splits), joined by k_attn_join.  (One token behind 16 caches of up to 8192 keys, 8 key heads of 128, bf16:
// 357 MB in 83 us, 4.3 TB/s; a large copy reaches 4.8.)
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int D, int DC, int NWV>
__global__ __launch_bounds__(64 * NWV) void k_attn_few(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  using L = Tile<T, D, 32>;
  constexpr int NS = DC / 16, NDB = DC / 32;
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

  int t = t0 + w, turn = 0;
  if (t < t1) {
    fill<T, D, 32, 64>(L{own}, a.direct, kp, a.sk.t, t * 32, seen, a.d, lane);
    fill<T, D, 32, 64>(L{own + L::BYTES}, a.direct, vp, a.sv.t, t * 32, seen, a.d, lane);
  }
  frag<T> qf[NS];
  load_frags<T, NS>(qf, qp, ok, (const T *)a.q, a.d);
  // the bias by distance only where a tile of this piece lies within max_distance
  const Place whole = place_of(t0 * 32, (t1 - t0) * 32, start, a.Tq, a.M, seen, a.causal);
  const float far_behind = ok ? bias_at(a, 0, h) : 0.f, far_ahead = ok ? bias_at(a, 2 * a.M, h) : 0.f;
  if (whole.near) {
    BiasLoad bl(a, bias, h0, a.pack, tid, 64 * NWV);
    bl.map();
    bl.table();
    bl.store();
  }
  clear_frags<T, NS>(qf, ok, a.d);
  __syncthreads();
  const float *own_bias = bias + (ok ? hh : 0) * bias_floats(a.M) + PAD + a.M;
  f32x16 o[NDB] = {};
  float m = -INFINITY, l = 0.f;
  const float c = a.scale * LOG2E;
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
    if (p.near || p.mask || !(c > 0.f) || !__all(fabsf(flat) < FLAT_MAX)) {
      if (p.near)
        finish_scores<true, true>(s[0], c, own_bias, 0.f, key0, pos, seen, a.causal);
      else
        finish_scores<false, true>(s[0], c, own_bias, flat, key0, pos, seen, a.causal);
      cs = 1.f;
      fs = 0.f;
    }
    online<T>(s, o, cs, fs, m, l);
    add_values<T, NDB>(vt_, 0, s[0], o);
  }
  l += __shfl_xor(l, 32);
  if (NWV > 1) {
    __syncthreads();
    join_waves<NDB, NWV, 1>((float *)lds, w, o, m, l);
    if (w > 0) return;
  }
  if (hh >= a.pack) return;
  if (a.splits > 1) {
    float *p = a.part + (((long)b * a.Hq + h) * a.Tq + i) * a.splits * (DC + 2) + (long)blockIdx.y * (DC + 2);
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
template <typename T, int DC>
__global__ __launch_bounds__(DC < 64 ? 64 : DC) void k_attn_join(AttnArgs a) {
  const long n = blockIdx.x;  // (b, h, i)
  const int b = (int)(n / ((long)a.Hq * a.Tq)), h = (int)(n / a.Tq % a.Hq), i = (int)(n % a.Tq), e = threadIdx.x;
  const float *p = a.part + n * a.splits * (DC + 2);
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, p[(long)s * (DC + 2)]);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int s = 0; s < a.splits; ++s) {
    const float ls = p[(long)s * (DC + 2) + 1];
    if (ls == 0.f) continue;  // a piece without keys; one whose scores are NaN has no maximum but a sum
    const float f = __builtin_amdgcn_exp2f(p[(long)s * (DC + 2)] - ref);
    l += f * ls;
    if (e < DC) o += f * p[(long)s * (DC + 2) + 2 + e];
  }
  const float x = l == 0.f ? 0.f : o / l;
  if (e < a.d) {
    ((T *)a.out)[b * a.so.b + (long)i * a.so.t + h * a.so.h + e] = (T)x;
    if (a.out_lo) ((T *)a.out_lo)[b * a.so.b + (long)i * a.so.t + h * a.so.h + e] = (T)(x - (float)(T)x);
  }
  if (a.stats && e == 0) store_stats(a, b, h, i, m, l);
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
  // grids (a launch's threads, 256 a head and block, 64 a bucket, are counted in 32 bits), and positions within int
  if (a->num_buckets >= (1 << 26) || a->Tq > 65535 * 64 || a->Tk > (1 << 29) || a->Hq > 65535 || (long)a->B * a->Hq >= (1L << 24)) return VT_EUNSUPPORTED;
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
int compute_width(const vt_relpos_attention *a) { return a->d > 64 && a->d <= 96 ? 96 : width_of(a); }
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
  const int G = a->Hq / a->Hk, W = bias_floats(a->max_distance);
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
  return f.use && f.splits > 1 ? (long)a->B * a->Hq * a->Tq * f.splits * (compute_width(a) + 2) : 0;
}

template <typename T, int D, int DC>
int launch_fwd(const vt_relpos_attention *a, const AttnArgs &k, hipStream_t s) {
  const Few f = few_of(a);
  if (f.use) {
    AttnArgs n = k;
    n.splits = f.splits;
    n.pack = f.pack;
    const dim3 grid(a->B * (a->Hq / f.pack), f.splits);
#define VT_FEW(NWV)                                                                    \
  if (f.waves == (NWV)) {                                                              \
    if (int rc = set_lds(k_attn_few<T, D, DC, NWV>, f.lds)) return rc;                     \
    hipLaunchKernelGGL((k_attn_few<T, D, DC, NWV>), grid, dim3(64 * (NWV)), f.lds, s, n);  \
  }
    VT_FEW(1)
    if constexpr (sizeof(T) == 4 && D == 128) {
      VT_FEW(2)
    } else {
      VT_FEW(4)
    }
#undef VT_FEW
    if (f.splits > 1)
      hipLaunchKernelGGL((k_attn_join<T, DC>), dim3((unsigned)((long)a->B * a->Hq * a->Tq)), dim3(DC < 64 ? 64 : DC), 0, s, n);
  } else {
    using S = RingShape<T, D>;
    const int lds = S::BYTES + 4 * bias_floats(a->max_distance);
#define VT_FWD(SPLIT)                                                                      \
  {                                                                                        \
    constexpr int ROWS = 32 * S::WAVES / (SPLIT);                                          \
    if (int rc = set_lds(k_attn_fwd<T, D, DC, SPLIT>, lds)) return rc;                     \
    const dim3 grid(a->B * a->Hq, (a->Tq + ROWS - 1) / ROWS);                              \
    hipLaunchKernelGGL((k_attn_fwd<T, D, DC, SPLIT>), grid, dim3(64 * S::WAVES), lds, s, k); \
  }
    if (attn_split(a, a->Hq, a->Tq, false)) VT_FWD(2) else VT_FWD(1)
#undef VT_FWD
  }
  VT_CHECK_LAUNCH();
  return 0;
}

// Scratch of the backward pass: records [B, Hq, rows], distances in double [Hq, W], the workgroups' sums [Hq, rows, W].
struct BwdScratch {
  long dist, hist, part, total;
  int rows, rec_rows;
};
BwdScratch bwd_scratch(const vt_relpos_attention *a, const BwdPlan &p) {
  BwdScratch b;
  const long W = 2L * a->max_distance + 1;
  b.rows = a->B * p.key_tiles;
  b.rec_rows = (a->Tq + 255) & ~255;  // whole workgroups' rows: the records behind the last query are written, too
  b.dist = 4L * a->B * a->Hq * b.rec_rows;
  b.hist = b.dist + ((2 * a->Hq * W + 3) & ~3L);
  b.part = b.hist + (((long)a->Hq * b.rows * W + 3) & ~3L);
  b.total = b.part + (p.share > 1 ? (long)p.share * a->B * a->Hk * a->Tk * 2 * a->d : 0);
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
  VT_WIDTH(launch_fwd, a, k, (hipStream_t)s);
  return 0;
}

extern "C" long vt_relpos_attention_bwd_scratch_floats(const vt_relpos_attention *a) {
  return check_args(a) != 0 ? 0 : bwd_scratch(a, attn_bwd_plan(a)).total;
}

extern "C" int vt_relpos_attention_bwd(const vt_relpos_attention *a, const void *out, vt_strides so, const void *out_lo,
                                       const float *stats, const void *dout, vt_strides sdo, void *dq, vt_strides sdq, void *dk,
                                       vt_strides sdk, void *dv, vt_strides sdv, float *dtable, float *scratch,
                                       long scratch_floats, vt_stream s) {
  const int rc = check_args(a);
  if (rc != 0) return rc;
  if (!out || !stats || ((uintptr_t)stats & 7) || !dout || !dq || !dk || !dv || !scratch || ((uintptr_t)scratch & 15) || (a->dtype != VT_F32 && !out_lo))
    return VT_EINVAL;
  if (a->Tk > 65535 * 64) return VT_EUNSUPPORTED;
  const BwdPlan p = attn_bwd_plan(a);
  const BwdScratch b = bwd_scratch(a, p);
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
  k.rec = reinterpret_cast<float4 *>(scratch);
  k.rec_rows = b.rec_rows;
  k.dist = reinterpret_cast<double *>(scratch + b.dist);
  k.hist = dtable ? scratch + b.hist : nullptr;
  k.hist_rows = b.rows;
  k.share = p.share;
  k.fine = attn_fine(a);
  k.part = scratch + b.part;
  k.direct = k.direct && aligned(a, dout, sdo);
  return attn_bwd_launch(a, k, p, (hipStream_t)s);
}
