// The norms around a block, its gate and its residual scale, forward and backward (vt_block_norms_*).
//
//   u = norm(y; w_post, b_post),  r = x + s u with s = res_scale * gate,  h = norm(r; w_pre, b_pre)
//   norm(t) = (t - mean) rstd w + b, mean = 0 for the RMS kind;  norm'(g) = rstd (g - mean(g) - t^ mean(g t^)), t^ = (t - mean) rstd
//
// Bound by memory: the forward pass reads x, y, gate and writes r, h; the backward pass reads x, y, gate, dr, dh and writes
// dx, dy, dgate (r is formed again in fp32 from x and y, which have to be read anyway, so its rounding enters no gradient).
// A row lies in the registers of one wave (D <= 512) or one workgroup (D <= 8192); the variance is summed around the mean
// from those registers.  In the backward pass a workgroup walks over a range of rows and keeps the weight gradients of its
// columns in registers; the ranges' partial sums are added by a second launch in their order, so there are no atomics.
#include "vtcnn_typed.h"

namespace vt {
namespace {

struct NormArgs {
  const void *x, *y, *gate, *dr, *dh;
  void *r, *h, *dx, *dy, *dgate;
  const float *scale, *w_post, *b_post, *w_pre, *b_pre;
  float *stats, *part, *gate_part;
  float eps, inv_d;
  int N, D, R;            // R: rows per gate row
  int pieces, piece_rows; // pieces of a gate row's rows (backward), and the rows of one
  long units, per_unit;   // pieces in all, and pieces a workgroup (or wave) walks over
  int layer;
  float *out[5];
};

// fp32 weights of eight columns; absent ones read as `fill`.
__device__ __forceinline__ void load_w(const float *w, int at, int D, float fill, float (&f)[8]) {
  if (w && at < D) {
    to_f32<float>(load8<float>(w + at, D - at, 0.f), f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fill;
  }
}
template <typename T>
__device__ __forceinline__ void load_row(const void *p, long n, int at, int D, float (&f)[8]) {
  if (p && at < D) {
    to_f32<T>(load8<T>((const T *)p + n * D + at, D - at, (T)0.f), f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_row(void *p, long n, int at, int D, const float (&f)[8]) {
  if (at < D) store8<T>((T *)p + n * D + at, D - at, from_f32<T>(f));
}

// Mean and 1 / sqrt(var + eps) of the group's row (zeros behind its end).
template <int GS, bool LAYER>
__device__ __forceinline__ void row_stats(const float (&t)[8], int at, int D, float inv_d, float eps, float *red, float &mean,
                                          float &rstd) {
  mean = 0.f;
  if (LAYER) {
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += t[e];
    mean = group_sum<GS>(s, red) * inv_d;
  }
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = !LAYER || at + e < D ? t[e] - mean : 0.f;
    q += d * d;
  }
  rstd = 1.f / sqrtf(group_sum<GS>(q, red + GS / 64) * inv_d + eps);
}

// A group of GS threads a row, eight columns a thread (D <= 8 GS); groups of one wave lie four to a workgroup.  (8192 x 4096 bf16
// with a gate row a token: 335 MB in 72 us, 4.6 TB/s; a large copy reaches 4.8.)
template <typename T, int GS, bool LAYER>
__global__ __launch_bounds__(GS == 64 ? 256 : GS) void k_norms_fwd(NormArgs a) {
  __shared__ float red[GS == 64 ? 1 : 4 * (GS / 64)];
  const int tid = GS == 64 ? (threadIdx.x & 63) : threadIdx.x, at = tid * 8;
  const long n = GS == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  if (n >= a.N) return;  // whole waves, which meet no barrier, or whole workgroups
  const int D = a.D;
  float x[8], y[8], w[8], b[8], s[8], g[8];
  load_row<T>(a.y, n, at, D, y);
  load_row<T>(a.x, n, at, D, x);
  load_w(a.w_post, at, D, 1.f, w);
  load_w(a.b_post, at, D, 0.f, b);
  load_w(a.scale, at, D, 1.f, s);
  if (a.gate) {
    load_row<T>(a.gate, n / a.R, at, D, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] *= g[e];
  }
  float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
  if (a.w_post) row_stats<GS, LAYER>(y, at, D, a.inv_d, a.eps, red, m1, r1);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] += s[e] * ((y[e] - m1) * r1 * w[e] + b[e]);
    if (at + e >= D) x[e] = 0.f;
  }
  store_row<T>(a.r, n, at, D, x);
  if (a.w_pre) {
    load_w(a.w_pre, at, D, 1.f, w);
    load_w(a.b_pre, at, D, 0.f, b);
    row_stats<GS, LAYER>(x, at, D, a.inv_d, a.eps, red + 2 * (GS / 64), m2, r2);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (x[e] - m2) * r2 * w[e] + b[e];
    store_row<T>(a.h, n, at, D, y);
  }
  if (tid == 0) {
    const float4 q = {m1, r1, m2, r2};
    *reinterpret_cast<float4 *>(a.stats + 4 * n) = q;
  }
}

// What a row of the backward pass reads, as it lies in memory: on its way while the row before is worked on.
template <typename T>
struct RowIn {
  vec8<T> x, y, dr, dh, gate;
  __device__ __forceinline__ void load(const NormArgs &a, long n, long grow, int at) {
    if (at >= a.D) return;
    const long p = n * a.D + at;
    const int left = a.D - at;
    y = load8<T>((const T *)a.y + p, left, (T)0.f);
    x = load8<T>((const T *)a.x + p, left, (T)0.f);
    if (a.dr) dr = load8<T>((const T *)a.dr + p, left, (T)0.f);
    if (a.dh) dh = load8<T>((const T *)a.dh + p, left, (T)0.f);
    if (a.gate) gate = load8<T>((const T *)a.gate + grow * a.D + at, left, (T)0.f);
  }
};
// The weights of eight columns; absent ones are 1, absent shifts 0.
template <bool LAYER>
struct ColumnWeights {
  float post[8], shift[8], scale[8], pre[8];
  __device__ __forceinline__ void load(const NormArgs &a, int at) {
    load_w(a.w_post, at, a.D, 1.f, post);
    load_w(LAYER ? a.b_post : nullptr, at, a.D, 0.f, shift);
    load_w(a.scale, at, a.D, 1.f, scale);
    load_w(a.w_pre, at, a.D, 1.f, pre);
  }
};

// A unit (wave of its own, or workgroup) walks over pieces [unit * per_unit, ...); a piece is a range of rows that share a
// row of the gate.  A thread has NC chunks of eight columns, GS * 8 apart.  Weight gradients: acc[k] = res_scale, w_post,
// b_post, w_pre, b_pre.  With one chunk the weights and the next row lie in registers beside the row (8192 x 4096 bf16: 243 us
// without either, 148 with both, at 3.6 TB/s); with two there is room for neither, and three of the five sums lie in LDS.
template <typename T, int GS, int NC, bool LAYER>
__global__ __launch_bounds__(GS == 64 ? 256 : GS) void k_norms_bwd(NormArgs a) {
  __shared__ float red[GS == 64 ? 1 : 4 * (GS / 64)];
  __shared__ float join[GS == 64 ? 4 * 512 : 1];
  constexpr bool HOLD = NC == 1;
  const int tid = GS == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const long unit = GS == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  const int D = a.D;
  constexpr bool IN_LDS = NC > 1;
  extern __shared__ __align__(16) char lds[];
  float4 *far = (float4 *)lds;  // [3][NC * 2][GS]: sums 0, 1 and 3
  float acc[5][NC][8] = {};
  if (IN_LDS)
#pragma unroll
    for (int i = 0; i < 3 * NC * 2; ++i) far[i * GS + tid] = float4{0.f, 0.f, 0.f, 0.f};
  const auto add = [&](int k, int c, const float (&v)[8]) {
    if (IN_LDS && k != 2 && k != 4) {
      float4 *p = far + ((k == 3 ? 2 : k) * NC * 2 + c * 2) * GS + tid;
      float4 lo = p[0], hi = p[GS];
      lo.x += v[0], lo.y += v[1], lo.z += v[2], lo.w += v[3];
      hi.x += v[4], hi.y += v[5], hi.z += v[6], hi.w += v[7];
      p[0] = lo;
      p[GS] = hi;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[k][c][e] += v[e];
    }
  };
  ColumnWeights<LAYER> held;
  if (HOLD) held.load(a, tid * 8);

  const long first = unit * a.per_unit, last = min(a.units, first + a.per_unit);
  // rows of a piece; pieces behind the last row are empty
  const auto range = [&](long p, long &grow, long &lo, long &hi) {
    grow = p / a.pieces;
    lo = grow * a.R + (p - grow * a.pieces) * a.piece_rows;
    hi = min((long)a.N, min(lo + a.piece_rows, (grow + 1) * a.R));
  };
  RowIn<T> in[NC] = {};
  float4 st = {}, st_next = {};
  const auto fetch = [&](long n, long grow) {
    st_next = *reinterpret_cast<const float4 *>(a.stats + 4 * n);
#pragma unroll
    for (int c = 0; c < NC; ++c) in[c].load(a, n, grow, (c * GS + tid) * 8);
  };
  long grow = 0, lo = 0, hi = 0;
  if (first < last) {
    range(first, grow, lo, hi);
    if (HOLD && lo < hi) fetch(lo, grow);
  }
  for (long p = first; p < last; ++p) {
    float dg[NC][8] = {};
    const long g0 = grow;
    long next_grow = 0, next_lo = 0, next_hi = 0;
    if (p + 1 < last) range(p + 1, next_grow, next_lo, next_hi);
    for (long n = lo; n < hi; ++n) {
      float yh[NC][8], rh[NC][8], g[NC][8], dx[NC][8], gt[NC][8];
      if (!HOLD) fetch(n, g0);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        to_f32<T>(in[c].y, yh[c]);
        to_f32<T>(in[c].x, rh[c]);
        to_f32<T>(in[c].dr, dx[c]);
        to_f32<T>(in[c].dh, g[c]);
        if (a.gate) {
          to_f32<T>(in[c].gate, gt[c]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) gt[c][e] = 1.f;
        }
      }
      st = st_next;
      if (HOLD) {
        if (n + 1 < hi)
          fetch(n + 1, g0);
        else if (next_lo < next_hi)
          fetch(next_lo, next_grow);
      }
      float sum = 0.f, dot = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        ColumnWeights<LAYER> w = held;
        if (!HOLD) w.load(a, at);
        float t3[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool inside = at + e < D;
          yh[c][e] = inside ? (yh[c][e] - st.x) * st.y : 0.f;
          const float r = rh[c][e] + w.scale[e] * gt[c][e] * (yh[c][e] * w.post[e] + w.shift[e]);
          rh[c][e] = inside ? (r - st.z) * st.w : 0.f;
          t3[e] = g[c][e] * rh[c][e];
          if (LAYER) acc[4][c][e] += g[c][e];
          g[c][e] *= w.pre[e];
          sum += g[c][e];
          dot += g[c][e] * rh[c][e];
        }
        add(3, c, t3);
      }
      if (a.w_pre) {
        sum = LAYER ? group_sum<GS>(sum, red) * a.inv_d : 0.f;
        dot = group_sum<GS>(dot, red + GS / 64) * a.inv_d;
      }
      float sum2 = 0.f, dot2 = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        ColumnWeights<LAYER> w = held;
        if (!HOLD) w.load(a, at);
        float t0[8], t1[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (a.w_pre) dx[c][e] += st.w * (g[c][e] - sum - rh[c][e] * dot);
          const bool inside = at + e < D;
          const float u = yh[c][e] * w.post[e] + w.shift[e], dxu = inside ? dx[c][e] * u : 0.f;
          t0[e] = dxu * gt[c][e];
          dg[c][e] += dxu * w.scale[e];
          const float du = inside ? dx[c][e] * w.scale[e] * gt[c][e] : 0.f;
          t1[e] = du * yh[c][e];
          if (LAYER) acc[2][c][e] += du;
          g[c][e] = du * w.post[e];
          sum2 += g[c][e];
          dot2 += g[c][e] * yh[c][e];
        }
        add(0, c, t0);
        add(1, c, t1);
        store_row<T>(a.dx, n, at, D, dx[c]);
      }
      if (a.w_post) {
        sum2 = LAYER ? group_sum<GS>(sum2, red + 2 * (GS / 64)) * a.inv_d : 0.f;
        dot2 = group_sum<GS>(dot2, red + 3 * (GS / 64)) * a.inv_d;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) g[c][e] = st.y * (g[c][e] - sum2 - yh[c][e] * dot2);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) store_row<T>(a.dy, n, (c * GS + tid) * 8, D, g[c]);
      // with a single reduction a row the next row's would overwrite the array that slower waves still read
      if (GS != 64 && !LAYER && !(a.w_pre && a.w_post)) __syncthreads();
    }
    if (a.gate && lo < hi)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        if (a.pieces == 1)
          store_row<T>(a.dgate, g0, at, D, dg[c]);
        else if (at < D)
          store8<float>(a.gate_part + p * D + at, D - at, from_f32<float>(dg[c]));
      }
    grow = next_grow;
    lo = next_lo;
    hi = next_hi;
  }
  // the unit's partial sums; the four waves of a workgroup of waves are added first, in order
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    if (!LAYER && (k == 2 || k == 4)) continue;  // the RMS kind has no shifts
    if (GS == 64) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) join[(threadIdx.x >> 6) * 512 + tid * 8 + e] = acc[k][0][e];
      __syncthreads();
      for (int i = threadIdx.x; i < D; i += 256)
        a.part[((long)blockIdx.x * 5 + k) * D + i] = join[i] + join[512 + i] + join[1024 + i] + join[1536 + i];
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        if (IN_LDS && k != 2 && k != 4) {  // a thread's own sums: no barrier between
          const float4 *q = far + ((k == 3 ? 2 : k) * NC * 2 + c * 2) * GS + tid;
          const float4 lo = q[0], hi = q[GS];
          const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          if (at < D) store8<float>(a.part + ((long)blockIdx.x * 5 + k) * D + at, D - at, from_f32<float>(v));
        } else if (at < D) {
          store8<float>(a.part + ((long)blockIdx.x * 5 + k) * D + at, D - at, from_f32<float>(acc[k][c]));
        }
      }
    }
  }
}

// Column sums of partial sums, sixteen rows of threads a workgroup: weight gradient blockIdx.y over the workgroups (below 5), or
// gate row blockIdx.y - 5 over its pieces.
template <typename T>
__global__ __launch_bounds__(1024) void k_norms_sums(NormArgs a, int blocks) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = blockIdx.x * 64 + lane, k = blockIdx.y;
  if (k < 5 && !a.out[k]) return;
  const long g = k - 5;
  // a short last gate row: pieces behind the last row hold nothing
  const int rows = k < 5 ? blocks : (int)min((long)a.pieces, (a.N - g * a.R + a.piece_rows - 1) / a.piece_rows);
  const float *p = k < 5 ? a.part + (long)k * a.D : a.gate_part + g * a.pieces * a.D;
  const long step = k < 5 ? 5L * a.D : a.D;
  float t = 0.f;
  if (i < a.D)
    for (int r = w; r < rows; r += 16) t += p[r * step + i];
  s[w][lane] = t;
  __syncthreads();
  if (w == 0 && i < a.D) {
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) x += s[j][lane];
    if (k < 5)
      a.out[k][i] = x;
    else
      ((T *)a.dgate)[g * a.D + i] = (T)x;
  }
}

// Rows that share a row of the gate.
long gate_rows(const vt_block_norms *a) { return a->gate && a->rows_per_gate < a->N ? a->rows_per_gate : a->N; }

int group_size(int D) { return D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }

struct Plan {
  int gs, pieces, piece_rows, blocks;
  long units, per_unit;
};
Plan plan_of(const vt_block_norms *a) {
  Plan p;
  p.gs = group_size(a->D);
  const int per_block = p.gs == 64 ? 4 : 1;
  // units that fill the chip: eight waves a compute unit, sixteen where they need not share a row
  const long target = p.gs == 64 ? 2048 : p.gs == 128 ? 1024 : p.gs == 256 ? 512 : 256;
  const long R = gate_rows(a), G = ((long)a->N + R - 1) / R;
  const long rows = ((long)a->N + target - 1) / target;
  if (R <= rows || R == 1) {
    p.pieces = 1;
    p.piece_rows = (int)R;
  } else {
    p.pieces = (int)((R + rows - 1) / rows);
    p.piece_rows = (int)rows;
  }
  p.units = G * p.pieces;
  p.per_unit = (p.units + target - 1) / target;
  const long n = (p.units + p.per_unit - 1) / p.per_unit;
  p.blocks = (int)((n + per_block - 1) / per_block);
  return p;
}

int check_args(const vt_block_norms *a) {
  if (!a || a->N < 1 || a->D < 1 || (a->gate && a->rows_per_gate < 1) || !(a->eps >= 0.f)) return VT_EINVAL;
  if (a->dtype != VT_F32 && a->dtype != VT_BF16 && a->dtype != VT_F16) return VT_EUNSUPPORTED;
  if (a->kind != VT_NORM_RMS && a->kind != VT_NORM_LAYER) return VT_EUNSUPPORTED;
  if (a->kind == VT_NORM_RMS && (a->b_post || a->b_pre)) return VT_EINVAL;
  if ((a->b_post && !a->w_post) || (a->b_pre && !a->w_pre)) return VT_EINVAL;
  // a launch's threads are counted in 32 bits
  if (a->D > 8192 || (long)a->N * group_size(a->D) > 0xffffff00L) return VT_EUNSUPPORTED;
  return 0;
}

NormArgs kernel_args(const vt_block_norms *a) {
  NormArgs k = {};
  k.gate = a->gate;
  k.scale = a->res_scale;
  k.w_post = a->w_post;
  k.b_post = a->b_post;
  k.w_pre = a->w_pre;
  k.b_pre = a->b_pre;
  k.eps = a->eps;
  k.inv_d = 1.f / (float)a->D;
  k.N = a->N;
  k.D = a->D;
  k.R = (int)gate_rows(a);
  k.layer = a->kind == VT_NORM_LAYER;
  return k;
}

template <typename T, bool LAYER, bool BWD>
int launch(const Plan &p, const NormArgs &k, hipStream_t s) {
#define VT_NORM(GS)                                                                                                            \
  if (p.gs == (GS)) {                                                                                                          \
    constexpr int BGS = (GS) == 1024 ? 512 : (GS), NC = (GS) / BGS;                                                            \
    if constexpr (BWD) {                                                                                                       \
      const int lds = NC > 1 ? 3 * NC * 2 * BGS * 16 : 0;                                                                      \
      if (lds > 65536)                                                                                                         \
        if (hipError_t e = hipFuncSetAttribute((const void *)&k_norms_bwd<T, BGS, NC, LAYER>,                                  \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds))                               \
          return (int)e;                                                                                                       \
      hipLaunchKernelGGL((k_norms_bwd<T, BGS, NC, LAYER>), dim3(p.blocks), dim3(BGS == 64 ? 256 : BGS), lds, s, k);            \
    } else {                                                                                                                   \
      hipLaunchKernelGGL((k_norms_fwd<T, GS, LAYER>), dim3((GS) == 64 ? (unsigned)((k.N + 3L) / 4) : k.N),                     \
                         dim3((GS) == 64 ? 256 : (GS)), 0, s, k);                                                              \
    }                                                                                                                          \
  }
  VT_NORM(64)
  VT_NORM(128)
  VT_NORM(256)
  VT_NORM(512)
  VT_NORM(1024)
#undef VT_NORM
  return 0;
}

}  // namespace
}  // namespace vt

using namespace vt;

extern "C" int vt_block_norms_fwd(const vt_block_norms *a, const void *x, const void *y, void *r, void *h, float *stats,
                                  vt_stream s) {
  const int rc = check_args(a);
  if (rc != 0) return rc;
  if (!x || !y || !r || (a->w_pre && !h) || !stats || ((uintptr_t)stats & 15)) return VT_EINVAL;
  NormArgs k = kernel_args(a);
  k.x = x;
  k.y = y;
  k.r = r;
  k.h = h;
  k.stats = stats;
  const Plan p = plan_of(a);
  VT_DISPATCH_TYPE(a->dtype, {
    const int e = k.layer ? launch<T, true, false>(p, k, (hipStream_t)s) : launch<T, false, false>(p, k, (hipStream_t)s);
    if (e != 0) return e;
  });
  VT_CHECK_LAUNCH();
  return 0;
}

extern "C" long vt_block_norms_bwd_scratch_floats(const vt_block_norms *a) {
  if (check_args(a) != 0) return 0;
  const Plan p = plan_of(a);
  return (long)p.blocks * 5 * a->D + (a->gate && p.pieces > 1 ? p.units * a->D : 0);
}

extern "C" int vt_block_norms_bwd(const vt_block_norms *a, const void *x, const void *y, const float *stats, const void *dr,
                                  const void *dh, void *dx, void *dy, void *dgate, float *dres_scale, float *dw_post,
                                  float *db_post, float *dw_pre, float *db_pre, float *scratch, long scratch_floats,
                                  vt_stream s) {
  const int rc = check_args(a);
  if (rc != 0) return rc;
  if (!x || !y || !stats || ((uintptr_t)stats & 15) || !dx || !dy || (!dr && !dh) || (a->w_pre && !dh) || (!a->w_pre && dh) ||
      !a->gate != !dgate || !scratch || (dres_scale && !a->res_scale) || (dw_post && !a->w_post) || (db_post && !a->b_post) ||
      (dw_pre && !a->w_pre) || (db_pre && !a->b_pre))
    return VT_EINVAL;
  if (scratch_floats < vt_block_norms_bwd_scratch_floats(a)) return VT_ELIMIT;
  const Plan p = plan_of(a);
  const long G = (a->N + gate_rows(a) - 1) / gate_rows(a);  // below the units' target wherever a gate row is cut
  const bool cut = a->gate && p.pieces > 1;
  NormArgs k = kernel_args(a);
  k.x = x;
  k.y = y;
  k.stats = const_cast<float *>(stats);
  k.dr = dr;
  k.dh = dh;
  k.dx = dx;
  k.dy = dy;
  k.dgate = dgate;
  k.part = scratch;
  k.gate_part = scratch + (long)p.blocks * 5 * a->D;
  k.pieces = p.pieces;
  k.piece_rows = p.piece_rows;
  k.units = p.units;
  k.per_unit = p.per_unit;
  float *out[5] = {dres_scale, dw_post, db_post, dw_pre, db_pre};
  bool any = false;
  for (int i = 0; i < 5; ++i) {
    k.out[i] = out[i];
    any = any || out[i];
  }
  VT_DISPATCH_TYPE(a->dtype, {
    const int e = k.layer ? launch<T, true, true>(p, k, (hipStream_t)s) : launch<T, false, true>(p, k, (hipStream_t)s);
    if (e != 0) return e;
    if (any || cut)
      hipLaunchKernelGGL((k_norms_sums<T>), dim3((a->D + 63) / 64, 5 + (cut ? (unsigned)G : 0)), dim3(1024), 0, (hipStream_t)s, k,
                         p.blocks);
  });
  VT_CHECK_LAUNCH();
  return 0;
}
