// Backward pass of the attention with a learned relative position bias (vt_relpos_attention_bwd; formulas in vtcnn_attn.hip):
// dq and D_i by query blocks, then dk, dv and the bias gradient by key blocks.
#include "vtcnn_attn.h"

namespace vt {
namespace {

// dq and D_i: as the forward pass (SPLIT as there: two waves a query block add their shares at the end).  dq takes D_i = do_i . (o_i + what its rounding left);
// the pass that follows takes the sum of p dp over the row, which this one forms anyway from unrounded p.
template <typename T, int D, int DC, int SPLIT>
__global__ __launch_bounds__(256) void k_attn_dq(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  lds_char *tiles = (lds_char *)lds;
  using L = Tile<T, D, BK>;
  float *bias_lds = (float *)(lds + 4 * L::BYTES);
  constexpr int NS = DC / 16, NDB = DC / 32, NKB = 2 / SPLIT, ROWS = 128 / SPLIT;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int pairs = a.B * a.Hk, grp = blockIdx.x % pairs, b = grp / a.Hk, hk = grp % a.Hk, h = hk * a.G + blockIdx.x / pairs;
  const int q0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * ROWS, w = wave_of(), qw = q0 + (w % (4 / SPLIT)) * 32, i = qw + (lane & 31);
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  const int pos0 = start + qw, pos = start + i;
  const int kend = q0 >= qlen ? 0 : a.causal ? min(klen, max(0, start + min(q0 + ROWS, qlen))) : klen;
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
    for (int x = 0; x < NKB; ++x) {
      const int kb = SPLIT == 1 ? x : w / 2, first = key0 + 32 * kb;
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
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const frag<T> sf = c_frag<T>(s, t);
#pragma unroll
        for (int db = 0; db < NDB; ++db) acc[db] = mma(kt.cols(32 * kb + 16 * t, db), sf, acc[db]);
      }
    }
  }
  pdp += __shfl_xor(pdp, 32);
  if constexpr (SPLIT > 1) {
    float *f = (float *)lds;
    __syncthreads();
    if (w >= 2) {
      f[(w - 2) * 64 + lane] = pdp;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) f[128 + (((w - 2) * NDB + db) * 16 + r) * 64 + lane] = acc[db][r];
    }
    __syncthreads();
    if (w >= 2) return;
    pdp += f[w * 64 + lane];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] += f[128 + ((w * NDB + db) * 16 + r) * 64 + lane];
  }
  if (i < a.Tq) {
    if (!ok)
#pragma unroll
      for (int db = 0; db < NDB; ++db) acc[db] = f32x16{};
    store_rows<T>((T *)a.dq + b * a.sdq.b + (long)i * a.sdq.t + h * a.sdq.h, a.d, acc, a.scale);
  }
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
template <typename T, int D, int DC, int SPLIT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void k_attn_dkv(AttnArgs a) {
  extern __shared__ __align__(128) char lds[];
  lds_char *tiles = (lds_char *)lds;
  constexpr int BQ = 32 * SPLIT, KEYS = 128 / SPLIT, NS = DC / 16, NDB = DC / 32;
  using L = Tile<T, D, BQ>;
  const int W = 2 * a.M + 1;
  constexpr bool KEYS_IN_LDS = sizeof(T) == 2 && D == 128;
  using LK = Tile<T, D, KEYS_IN_LDS ? KEYS : 32>;
  const LK kt = {tiles + 4 * L::BYTES};
  float *rows = (float *)(lds + 4 * L::BYTES + (KEYS_IN_LDS ? LK::BYTES : 0));  // [2][3][BQ]: maximum, log2 of the sum, D
  float *bias_lds = rows + 6 * BQ, *hist_all = bias_lds + W + 2 * PAD, *hist = hist_all + (threadIdx.x >> 6) * W;
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int pairs = a.B * a.Hk, grp = blockIdx.x % pairs, b = grp / a.Hk, hk = grp % a.Hk, part = blockIdx.x / pairs;
  const int w = wave_of(), k0 = blockIdx.y * KEYS, kw = k0 + (w % (4 / SPLIT)) * 32, key = kw + (lane & 31);
  const int qlen = length_of(a.q_len, b, a.Tq), klen = length_of(a.k_len, b, a.Tk), start = start_of(a, b);
  // queries before the first key's own place see none of the workgroup's keys
  const int qfirst = (a.causal ? min(max(0, k0 - start), a.Tq) : 0) & ~(BQ - 1), qend = k0 < klen ? qlen : 0;
  const bool ok = key < klen;
  const T *kp = (const T *)a.k + b * a.sk.b + (long)key * a.sk.t + hk * a.sk.h;
  const T *vp = (const T *)a.v + b * a.sv.b + (long)key * a.sv.t + hk * a.sv.h;
  frag<T> kf[KEYS_IN_LDS ? 1 : NS], vf[NS];
  if constexpr (KEYS_IN_LDS) {
    if (k0 < klen) {
      fill<T, D, KEYS, 256>(kt, a.direct, (const T *)a.k + b * a.sk.b + hk * a.sk.h, a.sk.t, k0, klen, a.d, tid);
      if (a.d < D) {  // the queries' tiles repeat a chunk behind d elements: here they must meet zeros
        arrive();
        __syncthreads();
        constexpr int EPC = LK::EPC, CPR = LK::CPR;
        const int c0 = (a.d + EPC - 1) / EPC;
        for (int x = tid; x < KEYS * (CPR - c0); x += 256)
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
      // the wave's 32 queries of the tile, from row rb on
      const int rb = SPLIT == 1 ? 0 : (w / 2) * 32, rw = r0 + rb;
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
        const float *row = row_max + rb + 8 * r4 + 4 * half;
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
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        const frag<T> pf = c_frag<T>(p, t), sf = c_frag<T>(s, t);
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          dv[db] = mma(dt.cols(rb + 16 * t, db), pf, dv[db]);
          dk[db] = mma(qt.cols(rb + 16 * t, db), sf, dk[db]);
        }
      }
    }
    if (a.hist) {
      if (SPLIT == 1) add_distance(kw - start - (qfirst + (max(qend - qfirst, 0) + BQ - 1) / BQ * BQ) + (lane & 31) - 4 * half, carry);
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
  if constexpr (SPLIT > 1) {
    float *f = (float *)lds;
    __syncthreads();
    if (w >= 2)
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          f[((((w - 2) * 2) * NDB + db) * 16 + r) * 64 + lane] = dk[db][r];
          f[((((w - 2) * 2 + 1) * NDB + db) * 16 + r) * 64 + lane] = dv[db][r];
        }
    __syncthreads();
    if (w >= 2) return;
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
template <typename T, int D>
constexpr int dkv_lds(int split, int M) {
  const int W = 2 * M + 1, keys = sizeof(T) == 2 && D == 128 ? 128 / split * 256 : 0;
  return 4 * 32 * split * D * (int)sizeof(T) + keys + 4 * (6 * 32 * split + W + 2 * PAD + 4 * W);
}
template <typename T, int D, int DC>
int dkv_bytes(int split, int M) {
  return dkv_lds<T, D>(split, M);
}
int dkv_lds_of(const vt_relpos_attention *a, int split) { VT_WIDTH(dkv_bytes, split, a->max_distance); }

template <typename T, int D, int DC, int SPLIT>
int launch_dq(const vt_relpos_attention *a, const AttnArgs &k, hipStream_t s) {
  const int lds = 4 * Tile<T, D, BK>::BYTES + 4 * bias_floats(a->max_distance);
  if (int rc = set_lds(k_attn_dq<T, D, DC, SPLIT>, lds)) return rc;
  constexpr int ROWS = 128 / SPLIT;
  hipLaunchKernelGGL((k_attn_dq<T, D, DC, SPLIT>), dim3(a->B * a->Hq, (a->Tq + ROWS - 1) / ROWS), dim3(256), lds, s, k);
  return 0;
}
template <typename T, int D, int DC, int SPLIT>
int launch_dkv(const vt_relpos_attention *a, const AttnArgs &k, const BwdPlan &p, hipStream_t s) {
  const int lds = dkv_lds<T, D>(SPLIT, a->max_distance);
  if (int rc = set_lds(k_attn_dkv<T, D, DC, SPLIT>, lds)) return rc;
  hipLaunchKernelGGL((k_attn_dkv<T, D, DC, SPLIT>), dim3(a->B * a->Hk * k.share, p.key_tiles), dim3(256), lds, s, k);
  return 0;
}
template <typename T, int D, int DC>
int launch_bwd(const vt_relpos_attention *a, const AttnArgs &k, const BwdPlan &p, hipStream_t s) {
  if (int rc = p.split_q == 2 ? launch_dq<T, D, DC, 2>(a, k, s) : launch_dq<T, D, DC, 1>(a, k, s)) return rc;
  if (int rc = p.split_k == 2 ? launch_dkv<T, D, DC, 2>(a, k, p, s) : launch_dkv<T, D, DC, 1>(a, k, p, s)) return rc;
  if (k.share > 1) {
    const long n = (long)a->B * a->Hk * a->Tk * 2 * a->d;
    hipLaunchKernelGGL((k_attn_dkv_sum<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, k);
  }
  if (k.dtable) {
    const int W = 2 * a->max_distance + 1;
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
  p.split_q = (long)a->B * a->Hq * ((a->Tq + 127) / 128) < 1024 ? 2 : 1;
  const long tiles = (long)a->B * a->Hk * ((a->Tk + 127) / 128);
  // a workgroup a query head where the key heads alone would not give every compute unit four: their parts cost a write and a
  // read in fp32, the walk over all G heads leaves compute units idle (and, causal, waiting for the longest)
  p.share = G > 1 && tiles < 1024 ? G : 1;
  p.split_k = tiles * p.share < 1024 && dkv_lds_of(a, 2) <= LDS_BYTES ? 2 : 1;
  p.key_tile = 128 / p.split_k;
  p.key_tiles = (a->Tk + p.key_tile - 1) / p.key_tile;
  return p;
}
int attn_bwd_launch(const vt_relpos_attention *a, const AttnArgs &k, const BwdPlan &p, hipStream_t s) {
  VT_WIDTH(launch_bwd, a, k, p, s);
  return 0;
}

}  // namespace vt
