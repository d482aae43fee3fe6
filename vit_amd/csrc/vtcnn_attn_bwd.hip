// Backward pass of the attention with a learned relative position bias (vt_relpos_attention_bwd; formulas in vtcnn_attn.hip):
// dq and D_i by query blocks, then dk, dv and the bias gradient by key blocks.
#include "vtcnn_attn.h"

namespace vt {
namespace {

// dq and D_i: as the forward pass (SPLIT as there: two waves a query block add their shares at the end).  dq takes
// D_i = do_i . (o_i + what its rounding left); the pass that follows takes the sum of p dp over the row, which this one forms anyway from unrounded p.  (2 x 4096 causal, 16
// heads of 128 over 4, bf16: 206 GFLOP, 274 us under a kernel trace; the whole backward pass, with its 275 GFLOP of dk, dv, takes
// 629 us without one, 765 TFLOP/s.)
template <typename T, int D, int DC, int SPLIT>
__global__ __launch_bounds__((64 * RingShape<T, D>::WAVES), sizeof(T) == 2 ? 2 : 1) void k_attn_dq(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  lds_char *tiles = (lds_char *)lds;
  using L = Tile<T, D, BK>;
  constexpr int NW = RingShape<T, D>::WAVES, NT = 64 * NW, HALF = NW / 2;
  float *bias_lds = (float *)(lds + RingShape<T, D>::BYTES);
  constexpr int NS = DC / 16, NDB = DC / 32, NKB = 2 / SPLIT, ROWS = 32 * NW / SPLIT;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int pairs = a.B * a.Hk, grp = blockIdx.x % pairs, b = grp / a.Hk, hk = grp % a.Hk, h = hk * a.G + blockIdx.x / pairs;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * ROWS, w = wave_of(), qw = q0 + (w % (NW / SPLIT)) * 32, i = qw + (lane & 31);
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  const int pos0 = start + qw, pos = start + i;
  const int kend = q0 >= qlen ? 0 : a.causal ? min(klen, max(0, start + min(q0 + ROWS, qlen))) : klen;
  const T *kp = (const T *)a.k + b * a.sk.b + hk * a.sk.h, *vp = (const T *)a.v + b * a.sv.b + hk * a.sv.h;
  const bool ok = i < qlen;

  KeyRing<T, D, NT> ring(a, tiles, kp, vp, kend, tid);
  BiasLoad bl(a, bias_lds, h, 1, tid, NT);
  bl.map();
  const T *qp = (const T *)a.q + b * a.sq.b + (long)i * a.sq.t + h * a.sq.h;
  const T *dop = (const T *)a.dout + b * a.sdo.b + (long)i * a.sdo.t + h * a.sdo.h;
  const T *op = (const T *)a.o + b * a.so.b + (long)i * a.so.t + h * a.so.h;
  frag<T> qf[NS], df[NS];
  float delta = 0.f;
  load_frags<T, NS>(qf, qp, ok, (const T *)a.q, a.d);
  load_frags<T, NS>(df, dop, ok, (const T *)a.dout, a.d);
  {
    frag<T> of[NS], lf[NS] = {};
    load_frags<T, NS>(of, op, ok, (const T *)a.o, a.d);
    if (sizeof(T) == 2)
      load_frags<T, NS>(lf, (const T *)a.o_lo + b * a.so.b + (long)i * a.so.t + h * a.so.h, ok, (const T *)a.o_lo, a.d);
    bl.table();
    clear_frags<T, NS>(qf, ok, a.d);
    clear_frags<T, NS>(df, ok, a.d);
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta += (float)df[s][e] * ((float)of[s][e] + (float)lf[s][e]);
  }
  const float *bias = bl.store();
  delta += __shfl_xor(delta, 32);
  float2 st = {INFINITY, 0.f};  // p = 0 where there are no keys
  if (ok) {
    const long n = ((long)b * a.Hq + h) * a.Tq + i;
    st = *reinterpret_cast<const float2 *>(a.stats + 2 * n);
    if (st.x == -INFINITY) st.x = INFINITY;
  }
  f32x16 acc[NDB] = {};
  float pdp = 0.f, lift = DS_LIFT;
  const float c = a.scale * LOG2E;
  for (int t = 0; t < ring.n; ++t) {
    const int key0 = t * BK;
    L kt, vt_;
    ring.step(t, kt, vt_);
    if (qw >= qlen || (a.causal && key0 > pos0 + 31)) continue;
#pragma unroll
    for (int x = 0; x < NKB; ++x) {
      const int kb = SPLIT == 1 ? x : w / (NW / SPLIT), first = key0 + 32 * kb;
      if (first >= kend || (a.causal && first > pos0 + 31)) continue;
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
      if constexpr (HALF_RANGE<T>) fit_half(s, acc, lift);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const frag<T> sf = c_frag<T>(s, t);
#pragma unroll
        for (int db = 0; db < NDB; ++db) acc[db] = mma(kt.cols(32 * kb + 16 * t, db), sf, acc[db]);
        if (SPLIT > 1 && sizeof(T) == 2 && a.fine) {
          const frag<T> lf = c_rest<T>(s, t, sf);
#pragma unroll
          for (int db = 0; db < NDB; ++db) acc[db] = mma(kt.cols(32 * kb + 16 * t, db), lf, acc[db]);
        }
      }
    }
  }
  pdp += __shfl_xor(pdp, 32);
  if constexpr (HALF_RANGE<T>) scale_all(acc, 1.f / lift);
  if constexpr (SPLIT > 1) {
    float *f = (float *)lds;
    __syncthreads();
    if (w >= HALF) {
      f[(w - HALF) * 64 + lane] = pdp;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) f[HALF * 64 + (((w - HALF) * NDB + db) * 16 + r) * 64 + lane] = acc[db][r];
    }
    __syncthreads();
    if (w >= HALF) return;
    pdp += f[w * 64 + lane];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] += f[HALF * 64 + ((w * NDB + db) * 16 + r) * 64 + lane];
  }
  if (i < a.Tq) {
    if (!ok)
#pragma unroll
      for (int db = 0; db < NDB; ++db) acc[db] = f32x16{};
    store_rows<T>((T *)a.dq + b * a.sdq.b + (long)i * a.sdq.t + h * a.sdq.h, a.d, acc, a.scale);
  }
  if (half == 0) a.rec[((long)b * a.Hq + h) * a.rec_rows + i] = float4{st.x, st.y, ok ? pdp : 0.f, 0.f};
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
  if constexpr (R % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // no more rotated values at once than registers hold
  if constexpr (R < 15) diagonal<R + 1>(s, col, here, below);
}

// dk, dv and the bias gradient by distance: a workgroup takes 128 keys of one key head, a wave 32 of them, and walks over the
// queries of the heads that share it (share == 1: of all G of them; share == G: of one, leaving fp32 parts for k_attn_dkv_sum).
// The bias gradient: with its registers rotated by their row, a block's ds of one distance lie in one lane; the sums of the
// block's lower 32 distances are the next block's upper ones and move on in registers, the upper ones are done and added to
// the wave's array.  (One addition in LDS a block; added one by one, sixteen a block, they took two thirds of the kernel's
// time where all tiles are near: 16 x 196 tokens, 48 us of which 30.)
// FINE: p and ds in two parts, where the caller asks for it, and where queries are at most 32 and few terms average a rounding: one
// tile a head, so that the second products cost little (whole backward pass in bf16 with dq so, too: 2 x 32 queries, 4096 keys, 16 heads of 128 170 us against 166
// in one part, 64 x 32 tokens 68 against 58).
// Widths of 256 bytes: the keys' fragments are read from LDS, which leaves two waves a SIMD.  (2 x 4096 causal, 16 heads of 128
// over 4, bf16: 275 GFLOP, 447 us under a kernel trace.)
template <typename T, int D, int DC, int SPLIT, bool FINE>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void k_attn_dkv(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  lds_char *tiles = (lds_char *)lds;
  constexpr int NW = 4, NT = 64 * NW, HALF = NW / 2, BQ = 32 * SPLIT, KEYS = 32 * NW / SPLIT, NS = DC / 16, NDB = DC / 32;
  using L = Tile<T, D, BQ>;
  const int W = 2 * a.M + 1;
  constexpr bool KEYS_IN_LDS = sizeof(T) == 2 && D == 128;
  using LK = Tile<T, D, KEYS_IN_LDS ? KEYS : 32>;
  const LK kt = {tiles};
  constexpr int STAGE = 2 * L::BYTES + 16 * BQ;  // queries, output gradients, records
  lds_char *ring = tiles + (KEYS_IN_LDS ? LK::BYTES : 0);
  float *bias_lds = (float *)(lds + (KEYS_IN_LDS ? LK::BYTES : 0) + a.stages * STAGE), *hist_all = bias_lds + W + 2 * PAD, *hist = hist_all + (threadIdx.x >> 6) * W;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int pairs = a.B * a.Hk, grp = blockIdx.x % pairs, b = grp / a.Hk, hk = grp % a.Hk, part = blockIdx.x / pairs;
  const int w = wave_of(), k0 = blockIdx.y * KEYS, kw = k0 + (w % (NW / SPLIT)) * 32, key = kw + (lane & 31);
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  // queries before the first key's own place see none of the workgroup's keys
  const int qfirst = (a.causal ? min(max(0, k0 - start), a.Tq) : 0) & ~(BQ - 1), qend = k0 < klen ? qlen : 0;
  const bool ok = key < klen;
  const T *kp = (const T *)a.k + b * a.sk.b + (long)key * a.sk.t + hk * a.sk.h;
  const T *vp = (const T *)a.v + b * a.sv.b + (long)key * a.sv.t + hk * a.sv.h;
  frag<T> kf[KEYS_IN_LDS ? 1 : NS], vf[NS];
  if constexpr (KEYS_IN_LDS) {
    if (k0 < klen) {
      fill<T, D, KEYS, NT>(kt, a.direct, (const T *)a.k + b * a.sk.b + hk * a.sk.h, a.sk.t, k0, klen, a.d, tid);
      if (a.d < D) {  // the queries' tiles repeat a chunk behind d elements: here they must meet zeros
        arrive();
        __syncthreads();
        constexpr int EPC = LK::EPC, CPR = LK::CPR;
        const int c0 = (a.d + EPC - 1) / EPC;
        for (int x = tid; x < KEYS * (CPR - c0); x += NT)
          *(__attribute__((address_space(3))) u32x4 *)kt.chunk(x / (CPR - c0), c0 + x % (CPR - c0)) = u32x4{0, 0, 0, 0};
      }
    }
  } else {
    load_frags<T, NS>(kf, kp, ok, (const T *)a.k, a.d);
  }
  load_frags<T, NS>(vf, vp, ok, (const T *)a.v, a.d);
  if constexpr (!KEYS_IN_LDS) clear_frags<T, NS>(kf, ok, a.d);
  clear_frags<T, NS>(vf, ok, a.d);
  f32x16 dk[NDB] = {}, dv[NDB] = {};
  float lift = DS_LIFT;
  const float c = a.scale * LOG2E;
  const int heads = a.G / a.share;
  for (int g = part * heads; g < (part + 1) * heads; ++g) {
    const int h = hk * a.G + g;
    const T *qp = (const T *)a.q + b * a.sq.b + h * a.sq.h, *dop = (const T *)a.dout + b * a.sdo.b + h * a.sdo.h;
    const float4 *recp = a.rec + ((long)b * a.Hq + h) * a.rec_rows;
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
    const float *bias = load_bias(a, bias_lds, h, tid, NT);
    if (a.hist)
      for (int x = tid; x < NW * W; x += NT) hist_all[x] = 0.f;
    const int n = qfirst < qend ? (qend - qfirst + BQ - 1) / BQ : 0;
    if (n == 0) __syncthreads();  // without a tile no barrier of the loop stands between the clearing and the sums' last additions
    const auto fetch = [&](int t, int to) {
      lds_char *s = ring + to * STAGE;
      const int r0 = qfirst + t * BQ;
      fill<T, D, BQ, NT>(L{s}, a.direct, qp, a.sq.t, r0, qend, a.d, tid);
      fill<T, D, BQ, NT>(L{s + L::BYTES}, a.direct, dop, a.sdo.t, r0, qend, a.d, tid);
      if (tid < BQ) async16(recp + r0, tid * 16, s + 2 * L::BYTES);
    };
    constexpr int LOADS = 2 * (BQ * L::CPR < NT ? 1 : BQ * L::CPR / NT);
    for (int t = 0; t < a.stages - 1 && t < n; ++t) fetch(t, t);
    int slot = 0;
    for (int t = 0; t < n; ++t) {
      const int r0 = qfirst + t * BQ;
      arrive_but<LOADS>(min(a.stages - 2, n - 1 - t));
      lds_barrier();
      if (t + a.stages - 1 < n) fetch(t + a.stages - 1, slot == 0 ? a.stages - 1 : slot - 1);
      const L qt = {ring + slot * STAGE}, dt = {ring + slot * STAGE + L::BYTES};
      const __attribute__((address_space(3))) float4 *rec = (const __attribute__((address_space(3))) float4 *)(ring + slot * STAGE + 2 * L::BYTES);
      slot = slot + 1 == a.stages ? 0 : slot + 1;
      // the wave's 32 queries of the tile, from row rb on
      const int rb = SPLIT == 1 ? 0 : (w / HALF) * 32, rw = r0 + rb;
      if (kw >= klen || rw >= qend || (a.causal && kw > start + rw + 31)) continue;
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        if constexpr (KEYS_IN_LDS)
          s = mma(qt.rows(rb, e), kt.rows(kw - k0, e), s);
        else
          s = mma(qt.rows(rb, e), kf[e], s);
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // no more fragments in flight than registers hold
      }
#pragma unroll
      for (int e = 0; e < NS; ++e) {
        dp = mma(dt.rows(rb, e), vf[e], dp);
        if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_sched_barrier(0);
      // distance of register r: key - start - query; its bounds over the block decide the variant
      const int base = key - start - rw, lo = kw - start - rw - 31, hi = kw + 31 - start - rw;
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
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * r4 + j;
          const float x = rec[rb + 8 * r4 + 4 * half + j].x, y = rec[rb + 8 * r4 + 4 * half + j].y, z = rec[rb + 8 * r4 + 4 * half + j].z;
          p[r] = __builtin_amdgcn_exp2f(s[r] - x - y);
          s[r] = p[r] * (dp[r] - z);
        }
      }
      if (near) {
        if (a.hist) {
          if (!ok)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 0.f;
          float here = carry, below = 0.f;
          diagonal<0>(s, lane & 31, here, below);
          const int away = kw - start - rw + (lane & 31) - 4 * half;
          add_distance(away, here);
          if (SPLIT == 1)
            carry = below;
          else  // the next block of this wave is 64 queries on
            add_distance(away - 32, below);
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
      if constexpr (HALF_RANGE<T>) {
        fit_half(s, dk, lift);
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] *= BWD_LIFT;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        const frag<T> pf = c_frag<T>(p, t), sf = c_frag<T>(s, t);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          dv[db] = mma(dt.cols(rb + 16 * t, db), pf, dv[db]);
          dk[db] = mma(qt.cols(rb + 16 * t, db), sf, dk[db]);
        }
        if (FINE) {
          const frag<T> pl = c_rest<T>(p, t, pf), sl = c_rest<T>(s, t, sf);
#pragma unroll
          for (int db = 0; db < NDB; ++db) {
            dv[db] = mma(dt.cols(rb + 16 * t, db), pl, dv[db]);
            dk[db] = mma(qt.cols(rb + 16 * t, db), sl, dk[db]);
          }
        }
      }
    }
    if (a.hist) {
      if (SPLIT == 1) add_distance(kw - start - (qfirst + n * BQ) + (lane & 31) - 4 * half, carry);
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
      for (int x = tid; x < W; x += NT) {
        float t = 0.f;
#pragma unroll
        for (int y = 0; y < NW; ++y) t += hist_all[y * W + x];
        out[x] = t;
      }
    }
  }
  if constexpr (HALF_RANGE<T>) {
    scale_all(dk, 1.f / lift);
    scale_all(dv, 1.f / BWD_LIFT);
  }
  if constexpr (SPLIT > 1) {
    float *f = (float *)lds;
    __syncthreads();
    if (w >= HALF)
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          f[((((w - HALF) * 2) * NDB + db) * 16 + r) * 64 + lane] = dk[db][r];
          f[((((w - HALF) * 2 + 1) * NDB + db) * 16 + r) * 64 + lane] = dv[db][r];
        }
    __syncthreads();
    if (w >= HALF) return;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        dk[db][r] += f[(((w * 2) * NDB + db) * 16 + r) * 64 + lane];
        dv[db][r] += f[(((w * 2 + 1) * NDB + db) * 16 + r) * 64 + lane];
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

// dk and dv from the query heads' parts, [G][B][Hk][Tk][2][d]: eight elements of a row a thread.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_dkv_sum(AttnArgs a) {
  const int per = (a.d + 7) / 8;
  const long rows = (long)a.B * a.Hk * a.Tk * 2, n = (long)blockIdx.x * 256 + threadIdx.x;
  if (n >= rows * per) return;
  const long row = n / per;
  const int at = (int)(n - row * per) * 8;
  float t[8] = {};
  for (int g = 0; g < a.share; ++g) {
    float f[8];
    to_f32<float>(load8<float>(a.part + (g * rows + row) * a.d + at, a.d - at, 0.f), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] += f[e];
  }
  const long key_row = row >> 1;
  const int b = (int)(key_row / ((long)a.Hk * a.Tk)), hk = (int)(key_row / a.Tk % a.Hk), key = (int)(key_row % a.Tk);
  T *out = row & 1 ? (T *)a.dv + b * a.sdv.b + (long)key * a.sdv.t + hk * a.sdv.h : (T *)a.dk + b * a.sdk.b + (long)key * a.sdk.t + hk * a.sdk.h;
  store8<T>(out + at, a.d - at, from_f32<T>(t));
}

// The bias gradient by distance: the workgroups' sums, in double and in order (64 distances of head blockIdx.y a workgroup).
__device__ __forceinline__ double distance_sum(const AttnArgs &a, int h, int x, int w, int lane, double (&s)[16][64]) {
  const int W = 2 * a.M + 1;
  double t = 0;
  if (x < W)
    for (int r = w; r < a.hist_rows; r += 16) t += a.hist[((long)h * a.hist_rows + r) * W + x];
  __syncthreads();
  s[w][lane] = t;
  __syncthreads();
  t = 0;
  if (w == 0)
#pragma unroll
    for (int j = 0; j < 16; ++j) t += s[j][lane];
  return t;
}
__global__ __launch_bounds__(1024) void k_attn_distances(AttnArgs a) {
  __shared__ double s[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, x = blockIdx.x * 64 + lane, h = blockIdx.y, W = 2 * a.M + 1;
  const double t = distance_sum(a, h, x, w, lane, s);
  if (w == 0 && x < W) a.dist[(long)h * W + x] = t;
}
// The distances of one bucket and head, by one wave.
__device__ __forceinline__ void bucket_sum(const AttnArgs &a, int bucket, int h, const double *dist, int lane) {
  double t = 0;
  for (int x = lane; x < 2 * a.M + 1; x += 64)
    if (a.map[x] == bucket) t += dist[x];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
  if (lane == 0) a.dtable[(long)bucket * a.Hq + h] = (float)t;
}
__global__ __launch_bounds__(64) void k_attn_buckets(AttnArgs a) {
  bucket_sum(a, blockIdx.x, blockIdx.y, a.dist + (long)blockIdx.y * (2 * a.M + 1), threadIdx.x);
}
// Both for one head in one launch, the distances staying in LDS: as many groups of threads as a workgroup holds take the rows in
// turn, a thread one distance (lds: a double a group and distance).
__host__ __device__ __forceinline__ int table_groups(int W) { return W >= 512 ? 1 : 1024 / ((W + 63) & ~63); }
__global__ __launch_bounds__(1024) void k_attn_table(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  double *dist = (double *)lds;
  const int W = 2 * a.M + 1, groups = table_groups(W), width = groups == 1 ? 1024 : (W + 63) & ~63;
  const int h = blockIdx.x, g = threadIdx.x / width, x0 = threadIdx.x % width;
  if (g < groups)
    for (int x = x0; x < W; x += width) {
      const float *p = a.hist + (long)h * a.hist_rows * W + x;
      double t = 0;
      int r = g;
      for (; r + 3 * groups < a.hist_rows; r += 4 * groups) {
        float f[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = p[(long)(r + k * groups) * W];
#pragma unroll
        for (int k = 0; k < 4; ++k) t += f[k];
      }
      for (; r < a.hist_rows; r += groups) t += p[(long)r * W];
      dist[(long)g * W + x] = t;
    }
  __syncthreads();
  if (g == 0)
    for (int x = x0; x < W; x += width) {
      double t = dist[x];
      for (int k = 1; k < groups; ++k) t += dist[(long)k * W + x];
      dist[x] = t;
    }
  __syncthreads();
  for (int b = threadIdx.x >> 6; b < a.nb; b += 16) bucket_sum(a, b, h, dist, threadIdx.x & 63);
}

// ---------------------------------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int D>
constexpr int dkv_lds(int split, int stages, int M) {
  const int W = 2 * M + 1, keys = sizeof(T) == 2 && D == 128 ? 128 / split * 256 : 0, bq = 32 * split;
  return keys + stages * (2 * bq * D * (int)sizeof(T) + 16 * bq) + 4 * (W + 2 * PAD + 4 * W);
}
// Buffers and LDS of a dk, dv workgroup for a split; buffers 0: no room.
struct KeyShape {
  int stages, bytes;
};
template <typename T, int D, int DC>
KeyShape key_shape(int split, int M) {
  // two workgroups a compute unit where they fit, or one with what it needs at least
  for (int stages = 4; stages >= 2; --stages)
    if (dkv_lds<T, D>(split, stages, M) <= (stages > 2 ? LDS_BYTES / 2 : LDS_BYTES))
      return KeyShape{stages, dkv_lds<T, D>(split, stages, M)};
  return KeyShape{0, 0};
}
KeyShape key_shape_of(const vt_relpos_attention *a, int split) {
  VT_WIDTH(key_shape, split, a->max_distance);
  return KeyShape{0, 0};
}

template <typename T, int D, int DC, int SPLIT>
int launch_dq(const vt_relpos_attention *a, const AttnArgs &k, hipStream_t s) {
  using S = RingShape<T, D>;
  const int lds = S::BYTES + 4 * bias_floats(a->max_distance);
  if (int rc = set_lds(k_attn_dq<T, D, DC, SPLIT>, lds)) return rc;
  constexpr int ROWS = 32 * S::WAVES / SPLIT;
  hipLaunchKernelGGL((k_attn_dq<T, D, DC, SPLIT>), dim3(a->B * a->Hq, (a->Tq + ROWS - 1) / ROWS), dim3(64 * S::WAVES), lds, s, k);
  return 0;
}
template <typename T, int D, int DC, int SPLIT, bool FINE>
int launch_dkv(const vt_relpos_attention *a, const AttnArgs &k, const BwdPlan &p, hipStream_t s) {
  if (int rc = set_lds(k_attn_dkv<T, D, DC, SPLIT, FINE>, p.key_bytes)) return rc;
  hipLaunchKernelGGL((k_attn_dkv<T, D, DC, SPLIT, FINE>), dim3(a->B * a->Hk * k.share, p.key_tiles), dim3(256), p.key_bytes, s, k);
  return 0;
}
template <typename T, int D, int DC>
int launch_bwd(const vt_relpos_attention *a, AttnArgs k, const BwdPlan &p, hipStream_t s) {
  if (int rc = p.split_q == 2 ? launch_dq<T, D, DC, 2>(a, k, s) : launch_dq<T, D, DC, 1>(a, k, s)) return rc;
  k.stages = p.key_stages;
  int rc;
  if (p.split_k == 2)
    rc = launch_dkv<T, D, DC, 2, false>(a, k, p, s);
  else if (sizeof(T) == 2 && k.fine)
    rc = launch_dkv<T, D, DC, 1, sizeof(T) == 2>(a, k, p, s);
  else
    rc = launch_dkv<T, D, DC, 1, false>(a, k, p, s);
  if (rc) return rc;
  if (k.share > 1) {
    const long n = (long)a->B * a->Hk * a->Tk * 2 * ((a->d + 7) / 8);
    hipLaunchKernelGGL((k_attn_dkv_sum<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, k);
  }
  if (k.dtable) {
    const int W = 2 * a->max_distance + 1;
    // one workgroup a head while its sums are read in a few microseconds
    if ((long)W * k.hist_rows <= 32768) {
      hipLaunchKernelGGL(k_attn_table, dim3(a->Hq), dim3(1024), 8 * W * table_groups(W), s, k);
      VT_CHECK_LAUNCH();
      return 0;
    }
    hipLaunchKernelGGL(k_attn_distances, dim3((W + 63) / 64, a->Hq), dim3(1024), 0, s, k);
    hipLaunchKernelGGL(k_attn_buckets, dim3(a->num_buckets, a->Hq), dim3(64), 0, s, k);
  }
  VT_CHECK_LAUNCH();
  return 0;
}

}  // namespace

BwdPlan attn_bwd_plan(const vt_relpos_attention *a) {
  BwdPlan p;
  const int G = a->Hq / a->Hk;
  p.split_q = attn_split(a, a->Hq, a->Tq, false, attn_fine(a)) ? 2 : 1;
  const long tiles = (long)a->B * a->Hk * ((a->Tk + 127) / 128);
  // a workgroup a query head where the key heads alone would not give every compute unit four: their parts cost a write and a
  // read in fp32, the walk over all G heads leaves compute units idle (and, causal, waiting for the longest)
  p.share = G > 1 && tiles < 1024 ? G : 1;
  p.split_k = attn_split(a, a->Hk * p.share, a->Tk, true, attn_fine(a)) && key_shape_of(a, 2).stages > 0 ? 2 : 1;
  const KeyShape k = key_shape_of(a, p.split_k);
  p.key_stages = k.stages;
  p.key_bytes = k.bytes;
  const int keys = 128 / p.split_k;
  p.key_tiles = (a->Tk + keys - 1) / keys;
  return p;
}
int attn_bwd_launch(const vt_relpos_attention *a, const AttnArgs &k, const BwdPlan &p, hipStream_t s) {
  VT_WIDTH(launch_bwd, a, k, p, s);
  return 0;
}

}  // namespace vt
