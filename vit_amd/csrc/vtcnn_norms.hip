// The norms around a block, its gate and its residual scale, forward and backward (vt_block_norms_*).
//
//   u = norm(y; w_post, b_post),  r = x + s u with s = res_scale * gate,  h = norm(r; w_pre, b_pre)
//   norm(t) = (t - mean) rstd w + b, mean = 0 for the RMS kind;  norm'(g) = rstd (g - mean(g) - t^ mean(g t^)), t^ = (t - mean) rstd
//
// Bound by memory: the forward pass reads x, y, gate and writes r, h; the backward pass reads x, y, gate, dr, dh and writes
// dx, dy, dgate (r is formed again in fp32 from x and y, which have to be read anyway, so its rounding enters no gradient).
// A row lies in the registers of one wave (D <= 1024) or one workgroup (D <= 8192); the variance is summed around the mean
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
template <int GS, int NC, bool LAYER>
__device__ __forceinline__ void row_stats(const float (&t)[NC][8], int tid, int D, float inv_d, float eps, float *red, float &mean,
                                          float &rstd) {
  mean = 0.f;
  if (LAYER) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += t[c][e];
    mean = group_sum<GS>(s, red) * inv_d;
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = !LAYER || (c * GS + tid) * 8 + e < D;
      const float d = in ? t[c][e] - mean : 0.f;
      q += d * d;
    }
  rstd = 1.f / sqrtf(group_sum<GS>(q, red + GS / 64) * inv_d + eps);
}

template <typename T, int GS, int NC, bool LAYER>
__global__ __launch_bounds__(GS == 64 ? 256 : GS) void k_norms_fwd(NormArgs a) {
  __shared__ float red[GS == 64 ? 1 : 4 * (GS / 64)];
  const int tid = GS == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const long n = GS == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  if (n >= a.N) return;  // whole waves, which meet no barrier, or whole workgroups
  const int D = a.D;
  float x[NC][8], y[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int at = (c * GS + tid) * 8;
    load_row<T>(a.y, n, at, D, y[c]);
    load_row<T>(a.x, n, at, D, x[c]);
  }
  float m1 = 0.f, r1 = 1.f, m2 = 0.f, r2 = 1.f;
  if (a.w_post) row_stats<GS, NC, LAYER>(y, tid, D, a.inv_d, a.eps, red, m1, r1);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int at = (c * GS + tid) * 8;
    float w[8], b[8], s[8], g[8];
    load_w(a.w_post, at, D, 1.f, w);
    load_w(a.b_post, at, D, 0.f, b);
    load_w(a.scale, at, D, 1.f, s);
    if (a.gate) {
      load_row<T>(a.gate, n / a.R, at, D, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] *= g[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = (y[c][e] - m1) * r1 * w[e] + b[e];
      x[c][e] += s[e] * u;
      if (at + e >= D) x[c][e] = 0.f;
    }
    store_row<T>(a.r, n, at, D, x[c]);
  }
  if (a.w_pre) {
    row_stats<GS, NC, LAYER>(x, tid, D, a.inv_d, a.eps, red + 2 * (GS / 64), m2, r2);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int at = (c * GS + tid) * 8;
      float w[8], b[8], h[8];
      load_w(a.w_pre, at, D, 1.f, w);
      load_w(a.b_pre, at, D, 0.f, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = (x[c][e] - m2) * r2 * w[e] + b[e];
      store_row<T>(a.h, n, at, D, h);
    }
  }
  if (tid == 0) {
    const float4 q = {m1, r1, m2, r2};
    *reinterpret_cast<float4 *>(a.stats + 4 * n) = q;
  }
}

// A unit (wave of its own, or workgroup) walks over pieces [unit * per_unit, ...); a piece is a range of rows that share a
// row of the gate.  Weight gradients: acc[k] = res_scale, w_post, b_post, w_pre, b_pre.
template <typename T, int GS, int NC, bool LAYER>
__global__ __launch_bounds__(GS == 64 ? 256 : GS) void k_norms_bwd(NormArgs a) {
  __shared__ float red[GS == 64 ? 1 : 4 * (GS / 64)];
  __shared__ float join[GS == 64 ? 4 * NC * 512 : 1];
  const int tid = GS == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const long unit = GS == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  const int D = a.D;
  float acc[5][NC][8];
#pragma unroll
  for (int k = 0; k < 5; ++k)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[k][c][e] = 0.f;

  const long first = unit * a.per_unit, last = min(a.units, first + a.per_unit);
  for (long p = first; p < last; ++p) {
    const long grow = p / a.pieces;
    const long lo = grow * a.R + (p - grow * a.pieces) * a.piece_rows;
    const long hi = min((long)a.N, min(lo + a.piece_rows, (grow + 1) * a.R));
    float dg[NC][8];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) dg[c][e] = 0.f;
    for (long n = lo; n < hi; ++n) {
      const float4 st = *reinterpret_cast<const float4 *>(a.stats + 4 * n);
      float yh[NC][8], rh[NC][8], g[NC][8], dx[NC][8];
      float sum = 0.f, dot = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        load_row<T>(a.y, n, at, D, yh[c]);
        load_row<T>(a.x, n, at, D, rh[c]);
        load_row<T>(a.dr, n, at, D, dx[c]);
        load_row<T>(a.dh, n, at, D, g[c]);
        float w[8], b[8], s[8], gt[8];
        load_w(a.w_post, at, D, 1.f, w);
        load_w(a.b_post, at, D, 0.f, b);
        load_w(a.scale, at, D, 1.f, s);
        if (a.gate) {
          load_row<T>(a.gate, grow, at, D, gt);
#pragma unroll
          for (int e = 0; e < 8; ++e) s[e] *= gt[e];
        }
        load_w(a.w_pre, at, D, 1.f, gt);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool in = at + e < D;
          yh[c][e] = in ? (yh[c][e] - st.x) * st.y : 0.f;
          const float r = rh[c][e] + s[e] * (yh[c][e] * w[e] + b[e]);
          rh[c][e] = in ? (r - st.z) * st.w : 0.f;
          acc[3][c][e] += g[c][e] * rh[c][e];
          acc[4][c][e] += g[c][e];
          g[c][e] *= gt[e];
          sum += g[c][e];
          dot += g[c][e] * rh[c][e];
        }
      }
      if (a.w_pre) {
        sum = LAYER ? group_sum<GS>(sum, red) * a.inv_d : 0.f;
        dot = group_sum<GS>(dot, red + GS / 64) * a.inv_d;
      }
      float sum2 = 0.f, dot2 = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        float w[8], b[8], s[8], gt[8];
        load_w(a.w_post, at, D, 1.f, w);
        load_w(a.b_post, at, D, 0.f, b);
        load_w(a.scale, at, D, 1.f, s);
        if (a.gate) {
          load_row<T>(a.gate, grow, at, D, gt);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) gt[e] = 1.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (a.w_pre) dx[c][e] += st.w * (g[c][e] - sum - rh[c][e] * dot);
          const float u = yh[c][e] * w[e] + b[e], dxu = at + e < D ? dx[c][e] * u : 0.f;
          acc[0][c][e] += dxu * gt[e];
          dg[c][e] += dxu * s[e];
          const float du = at + e < D ? dx[c][e] * s[e] * gt[e] : 0.f;
          acc[1][c][e] += du * yh[c][e];
          acc[2][c][e] += du;
          g[c][e] = du * w[e];
          sum2 += g[c][e];
          dot2 += g[c][e] * yh[c][e];
        }
        store_row<T>(a.dx, n, at, D, dx[c]);
      }
      if (a.w_post) {
        sum2 = LAYER ? group_sum<GS>(sum2, red + 2 * (GS / 64)) * a.inv_d : 0.f;
        dot2 = group_sum<GS>(dot2, red + 3 * (GS / 64)) * a.inv_d;
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        if (a.w_post) {
#pragma unroll
          for (int e = 0; e < 8; ++e) g[c][e] = st.y * (g[c][e] - sum2 - yh[c][e] * dot2);
        }
        store_row<T>(a.dy, n, at, D, g[c]);
      }
      // with a single reduction a row the next row's would overwrite the array that slower waves still read
      if (GS != 64 && !LAYER && !(a.w_pre && a.w_post)) __syncthreads();
    }
    if (a.gate && lo < hi) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        if (a.pieces == 1) {
          store_row<T>(a.dgate, grow, at, D, dg[c]);
        } else if (at < D) {
          vec8<float> v;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = dg[c][e];
          store8<float>(a.gate_part + p * D + at, D - at, v);
        }
      }
    }
  }
  // the unit's partial sums; the four waves of a workgroup of waves are added first, in order
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    if (GS == 64) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) join[(threadIdx.x >> 6) * NC * 512 + (c * 64 + tid) * 8 + e] = acc[k][c][e];
      __syncthreads();
      for (int i = threadIdx.x; i < D; i += 256) {
        const float s = join[i] + join[NC * 512 + i] + join[2 * NC * 512 + i] + join[3 * NC * 512 + i];
        a.part[((long)blockIdx.x * 5 + k) * D + i] = s;
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int at = (c * GS + tid) * 8;
        if (at >= D) continue;
        vec8<float> v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = acc[k][c][e];
        store8<float>(a.part + ((long)blockIdx.x * 5 + k) * D + at, D - at, v);
      }
    }
  }
}

// Weight gradients: column i of array k = blockIdx.y over the workgroups' partial sums, 16 rows of threads a workgroup.
__global__ __launch_bounds__(1024) void k_norms_weights(NormArgs a, int blocks) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = blockIdx.x * 64 + lane, k = blockIdx.y;
  if (!a.out[k]) return;
  float t = 0.f;
  if (i < a.D)
    for (int b = w; b < blocks; b += 16) t += a.part[((long)b * 5 + k) * a.D + i];
  s[w][lane] = t;
  __syncthreads();
  if (w == 0 && i < a.D) {
    float x = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) x += s[j][lane];
    a.out[k][i] = x;
  }
}

// Gradient of a gate row whose rows were cut into pieces.
template <typename T>
__global__ __launch_bounds__(256) void k_norms_gate(NormArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  const long g = blockIdx.y;
  if (i >= a.D) return;
  float t = 0.f;
  for (int p = 0; p < a.pieces; ++p) {
    if (g * a.R + (long)p * a.piece_rows >= a.N) break;  // a short last gate row: pieces behind the last row hold nothing
    t += a.gate_part[(g * a.pieces + p) * a.D + i];
  }
  ((T *)a.dgate)[g * a.D + i] = (T)t;
}

struct Plan {
  int gs, nc, pieces, piece_rows, blocks;
  long units, per_unit;
};
Plan plan_of(const vt_block_norms *a) {
  Plan p;
  const int D = a->D;
  p.gs = D <= 1024 ? 64 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024;
  p.nc = D <= 512 || D > 1024 ? 1 : 2;
  const int per_block = p.gs == 64 ? 4 : 1;
  const long target = (p.gs == 1024 ? 256L : 512L) * per_block;  // units that fill the chip
  const long R = a->gate ? a->rows_per_gate : a->N, G = ((long)a->N + R - 1) / R;
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
  if (a->D > 8192) return VT_EUNSUPPORTED;
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
  k.R = a->gate ? a->rows_per_gate : a->N;
  k.layer = a->kind == VT_NORM_LAYER;
  return k;
}

template <typename T, bool LAYER, bool BWD>
void launch(const Plan &p, const NormArgs &k, hipStream_t s) {
#define VT_NORM(GS, NC)                                                                                      \
  if (p.gs == (GS) && p.nc == (NC)) {                                                                        \
    const dim3 block((GS) == 64 ? 256 : (GS));                                                               \
    if constexpr (BWD)                                                                                       \
      hipLaunchKernelGGL((k_norms_bwd<T, GS, NC, LAYER>), dim3(p.blocks), block, 0, s, k);                   \
    else                                                                                                     \
      hipLaunchKernelGGL((k_norms_fwd<T, GS, NC, LAYER>), dim3((GS) == 64 ? (unsigned)((k.N + 3L) / 4) : k.N), block, 0, s, k); \
  }
  VT_NORM(64, 1)
  VT_NORM(64, 2)
  VT_NORM(256, 1)
  VT_NORM(512, 1)
  VT_NORM(1024, 1)
#undef VT_NORM
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
    if (k.layer)
      launch<T, true, false>(p, k, (hipStream_t)s);
    else
      launch<T, false, false>(p, k, (hipStream_t)s);
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
  const long G = ((long)a->N + (a->gate ? a->rows_per_gate : a->N) - 1) / (a->gate ? a->rows_per_gate : a->N);
  if (a->gate && p.pieces > 1 && G > 65535) return VT_EUNSUPPORTED;
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
    if (k.layer)
      launch<T, true, true>(p, k, (hipStream_t)s);
    else
      launch<T, false, true>(p, k, (hipStream_t)s);
    if (a->gate && p.pieces > 1)
      hipLaunchKernelGGL((k_norms_gate<T>), dim3((a->D + 255) / 256, (unsigned)G), dim3(256), 0, (hipStream_t)s, k);
  });
  if (any) hipLaunchKernelGGL(k_norms_weights, dim3((a->D + 63) / 64, 5), dim3(1024), 0, (hipStream_t)s, k, p.blocks);
  VT_CHECK_LAUNCH();
  return 0;
}
