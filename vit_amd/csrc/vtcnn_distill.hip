// Distillation from a teacher's top logits (vt_distill_*).
//
//   p = softmax(t / tau) over the K valid teacher entries, q = softmax(z / tau), c = softmax(z)
//   loss = kd tau^2 sum_k p_k (log p_k - log q_k) - ce log c_label
//   dz   = dloss (kd tau ((sum p) q - sum_k p_k e_k) + ce (c - e_label))
//
// A row is bound by memory: z is read once and dz written once.  A group of threads (a wave for short rows, a workgroup of
// 256 or 512 threads for long ones) holds its row in registers, so that maximum, both sums and the gradient come from one
// read.  Rows that are too few to fill the chip, or too long for a workgroup's registers, are cut along the vocabulary:
// partial statistics, a join of one workgroup a row, and a gradient pass that reads z again.
// The K entries and the label are a correction of the dense row: the thread of an id's first entry writes that element
// again, whole, with the p of all entries of that id added in their order; no atomics.
#include "vtcnn_typed.h"

namespace vt {
namespace {

struct DistillArgs {
  const void *z;
  const float *top;
  const int *id, *label;
  const float *dloss;
  float *loss, *stats;
  void *dz;
  float *part;
  long ldz, ldd;
  int N, V, K, splits, piece;
  float tau, inv_tau, kd, ce;
};

// The exponential of the dense pass: the library's where the result is fp32, the hardware's 2^x (error of the rounded
// argument x log2 e, 2^-24 |x|) where it is rounded to 16 bits anyway.
// `k` of dexp(x, k) = e^(x k') with the base's factor in it.
template <typename T>
__device__ __forceinline__ float rate(float k) {
  return sizeof(T) == 4 ? k : k * 1.44269504088896340736f;
}
template <typename T>
__device__ __forceinline__ float dexp(float x, float k) {
  return sizeof(T) == 4 ? expf(x * k) : __builtin_amdgcn_exp2f(x * k);
}

template <int GS>
__device__ __forceinline__ void group_sync() {
  if (GS == 64) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  } else {
    __syncthreads();
  }
}

// The teacher's side of one row in LDS: p, ids (-1: none) and the student's logits at them.
struct Teacher {
  float *p, *z;
  int *id;
  int *label_hit;
};
__device__ __forceinline__ Teacher teacher_lds(char *base, int K) {
  Teacher t;
  t.p = (float *)base;
  t.z = t.p + K;
  t.id = (int *)(t.z + K);
  t.label_hit = t.id + K;
  return t;
}
constexpr int TEACHER_BYTES(int K) { return (12 * K + 4 + 15) & ~15; }

// Fills t and returns (sum of p, the group's sum of p log p); the student's logits at ids in [lo, hi) only.  red: two arrays of
// GS / 64 floats.
template <typename T, int GS>
__device__ __forceinline__ void teacher_load(const DistillArgs &a, const Teacher &t, const T *row, long n, int lo, int hi, int label,
                                             int tid, float *red, float &psum, float &plogp) {
  const float *top = a.top + n * a.K;
  const int *id = a.id + n * a.K;
  float m = -INFINITY;
  for (int k = tid; k < a.K; k += GS) {
    const int i = id[k];
    const bool ok = i >= 0 && i < a.V;
    const float v = ok ? top[k] : -INFINITY;
    t.id[k] = ok ? i : -1;
    t.p[k] = v;
    t.z[k] = ok && i >= lo && i < hi ? (float)row[i] : 0.f;
    m = v > m || v != v ? v : m;
  }
  if (tid == 0) *t.label_hit = 0;
  m = group_max<GS>(m, red);
  float s = 0.f;
  for (int k = tid; k < a.K; k += GS) {
    // entries whose logit is -inf have p = 0; where nothing else is there, the row has no teacher's term
    const float e = m == -INFINITY ? 0.f : expf((t.p[k] - m) * a.inv_tau);
    s += t.id[k] >= 0 ? e : 0.f;
  }
  s = group_sum<GS>(s, red + GS / 64);
  const float rs = s == 0.f ? 0.f : 1.f / s, ls = s == 0.f ? 0.f : logf(s);
  float pl = 0.f;
  for (int k = tid; k < a.K; k += GS) {
    const float x = (t.p[k] - m) * a.inv_tau;
    const float p = m == -INFINITY || t.id[k] < 0 ? 0.f : expf(x) * rs;
    if (p != 0.f) pl += p * (x - ls);
    t.p[k] = p;
    if (t.id[k] == label) *t.label_hit = 1;  // id -1 never equals a valid label
  }
  psum = s == 0.f ? 0.f : (s != s ? s : 1.f);
  plogp = pl;
  group_sync<GS>();
}

// loss of a row from its statistics; plogp and the sum over k are still per thread.
template <int GS>
__device__ __forceinline__ float row_loss(const DistillArgs &a, const Teacher &t, float m, float st, float s1, float psum,
                                          float plogp, int label, float zlabel, int tid, float *red) {
  float kl = plogp;
  for (int k = tid; k < a.K; k += GS) {
    const float p = t.p[k];
    if (p != 0.f) kl -= p * ((t.z[k] - m) * a.inv_tau);
  }
  kl = group_sum<GS>(kl, red);
  float loss = a.kd == 0.f ? 0.f : a.kd * a.tau * a.tau * (kl + (psum == 0.f ? 0.f : psum * logf(st)));
  if (label >= 0 && a.ce != 0.f) loss += a.ce * (logf(s1) - (zlabel - m));
  return loss;
}

// What the gradient of a row needs besides z.
struct RowGrad {
  float m, wq, wc;  // dz = wq exp((z - m) / tau) + wc exp(z - m), then the corrections
};
// A term that the row has not (no valid entry, no label, weight 0) is 0 whatever the logits hold: rows of padding may be NaN
// or wholly -inf.
__device__ __forceinline__ RowGrad row_grad(const DistillArgs &a, float m, float st, float s1, float psum, float dl, int label) {
  return RowGrad{m, psum == 0.f || a.kd == 0.f ? 0.f : dl * a.kd * a.tau * psum / st, label < 0 || a.ce == 0.f ? 0.f : dl * a.ce / s1};
}
template <typename T>
__device__ __forceinline__ float dense_grad(const DistillArgs &a, const RowGrad &g, float z) {
  float d = 0.f;
  if (g.wq != 0.f) d = g.wq * dexp<T>(z - g.m, rate<T>(a.inv_tau));
  if (g.wc != 0.f) d += g.wc * dexp<T>(z - g.m, rate<T>(1.f));
  return d;
}

// The elements of [lo, hi) that the teacher's entries or the label touch.
template <typename T, int GS>
__device__ __forceinline__ void correct(const DistillArgs &a, const Teacher &t, const RowGrad &g, T *out, float dl, int label,
                                        float zlabel, int lo, int hi, int tid) {
  for (int k = tid; k < a.K; k += GS) {
    const int i = t.id[k];
    if (i < lo || i >= hi) continue;
    float ps = 0.f;
    bool first = true;
    for (int j = 0; j < a.K; ++j)
      if (t.id[j] == i) {
        if (j < k) first = false;
        ps += t.p[j];
      }
    if (!first) continue;
    float d = dense_grad<T>(a, g, t.z[k]);
    if (a.kd != 0.f) d -= dl * a.kd * a.tau * ps;
    if (i == label && a.ce != 0.f) d -= dl * a.ce;
    out[i] = (T)d;
  }
  if (tid == 0 && label >= lo && label < hi && a.ce != 0.f && !*t.label_hit)
    out[label] = (T)(dense_grad<T>(a, g, zlabel) - dl * a.ce);
}

__device__ __forceinline__ int row_label(const DistillArgs &a, long n) {
  const int l = a.label ? a.label[n] : -1;
  return l >= 0 && l < a.V ? l : -1;
}

// One row a group of GS threads, held in registers: V <= GS * 8 * NC.
template <typename T, int GS, int NC, bool GRAD>
__global__ __launch_bounds__(GS == 64 ? 256 : GS) void k_distill_row(DistillArgs a) {
  extern __shared__ char lds[];
  __shared__ float red_all[GS == 64 ? 1 : 8 * (GS / 64)];
  const int tid = GS == 64 ? (threadIdx.x & 63) : threadIdx.x;
  const long n = GS == 64 ? (long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long)blockIdx.x;
  if (n >= a.N) return;  // whole groups only: a wave of its own needs no barrier, a workgroup has one row
  float *red[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) red[i] = GS == 64 ? red_all : red_all + i * (GS / 64);
  const Teacher t = teacher_lds(lds + (GS == 64 ? (threadIdx.x >> 6) * TEACHER_BYTES(a.K) : 0), a.K);
  const T *row = (const T *)a.z + n * a.ldz;
  vec8<T> v[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const unsigned at = (c * GS + tid) * 8;
    if ((c + 1) * GS * 8 <= a.V)  // the same for the whole group: all chunks but the last ones
      v[c] = *reinterpret_cast<const vec8<T> *>(row + at);
    else if ((int)at < a.V)
      v[c] = load8<T>(row + at, a.V - (int)at, (T)(-INFINITY));
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = (T)(-INFINITY);
  }
  const int label = row_label(a, n);
  const float zlabel = label >= 0 ? (float)row[label] : 0.f;
  float psum, plogp;
  teacher_load<T, GS>(a, t, row, n, 0, a.V, label, tid, red[0], psum, plogp);
  float m = -INFINITY;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, (float)v[c][e]);
  }
  m = group_max<GS>(m, red[2]);
  const bool two = a.tau != 1.f;
  float st = 0.f, s1 = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    __builtin_amdgcn_sched_barrier(0);
    forget<T>(v[c]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      st += dexp<T>((float)v[c][e] - m, rate<T>(a.inv_tau));
    }
  }
  if (two)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      __builtin_amdgcn_sched_barrier(0);
      forget<T>(v[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s1 += dexp<T>((float)v[c][e] - m, rate<T>(1.f));
    }
  st = group_sum<GS>(st, red[3]);
  s1 = two ? group_sum<GS>(s1, red[4]) : st;
  const float loss = row_loss<GS>(a, t, m, st, s1, psum, plogp, label, zlabel, tid, red[5]);
  if (tid == 0) {
    a.loss[n] = loss;
    if (!GRAD) {
      float4 q = {m, st, s1, 0.f};
      *reinterpret_cast<float4 *>(a.stats + 4 * n) = q;
    }
  }
  if (!GRAD) return;
  const float dl = a.dloss[n];
  const RowGrad g = row_grad(a, m, st, s1, psum, dl, label);
  T *out = (T *)a.dz + n * a.ldd;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    __builtin_amdgcn_sched_barrier(0);
    forget<T>(v[c]);
    if (c * GS * 8 >= a.V) break;
    const unsigned at = (c * GS + tid) * 8;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = dense_grad<T>(a, g, (float)v[c][e]);
    if ((c + 1) * GS * 8 <= a.V)
      *reinterpret_cast<vec8<T> *>(out + at) = from_f32<T>(f);
    else if ((int)at < a.V)
      store8<T>(out + at, a.V - (int)at, from_f32<T>(f));
  }
  group_sync<GS>();
  correct<T, GS>(a, t, g, out, dl, label, zlabel, 0, a.V, tid);
}

// Partial statistics of a piece of a row (workgroup n * splits + piece): part[n][piece] = (max, sum at tau, sum at 1).
template <typename T>
__global__ __launch_bounds__(256) void k_distill_part(DistillArgs a) {
  __shared__ float red[3][4];
  const int tid = threadIdx.x;
  const long n = blockIdx.x / a.splits;
  const T *row = (const T *)a.z + n * a.ldz;
  const int split = blockIdx.x - n * a.splits, lo = split * a.piece, hi = min(a.V, lo + a.piece);
  const bool two = a.tau != 1.f;
  float m = -INFINITY;
  for (int at = lo + tid * 8; at < hi; at += 2048) {
    const vec8<T> v = load8<T>(row + at, hi - at, (T)(-INFINITY));
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, (float)v[e]);
  }
  m = group_max<256>(m, red[0]);
  const float base = m == -INFINITY ? 0.f : m;
  float st = 0.f, s1 = 0.f;
  for (int at = lo + tid * 8; at < hi; at += 2048) {
    const vec8<T> v = load8<T>(row + at, hi - at, (T)(-INFINITY));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (float)v[e] - base;
      st += dexp<T>(x, rate<T>(a.inv_tau));
      if (two) s1 += dexp<T>(x, rate<T>(1.f));
    }
  }
  st = group_sum<256>(st, red[1]);
  s1 = two ? group_sum<256>(s1, red[2]) : st;
  if (tid == 0) {
    float *p = a.part + (long)blockIdx.x * 3;
    p[0] = m;
    p[1] = st;
    p[2] = s1;
  }
}

// Joins a row's partial statistics and forms its loss.
template <typename T>
__global__ __launch_bounds__(256) void k_distill_join(DistillArgs a) {
  extern __shared__ char lds[];
  __shared__ float red[8][4];
  const int tid = threadIdx.x;
  const long n = blockIdx.x;
  const Teacher t = teacher_lds(lds, a.K);
  const T *row = (const T *)a.z + n * a.ldz;
  const int label = row_label(a, n);
  const float zlabel = label >= 0 ? (float)row[label] : 0.f;
  float psum, plogp;
  teacher_load<T, 256>(a, t, row, n, 0, a.V, label, tid, red[0], psum, plogp);
  const float *part = a.part + n * a.splits * 3;
  float m = -INFINITY;
  for (int i = tid; i < a.splits; i += 256) m = fmaxf(m, part[3 * i]);
  m = group_max<256>(m, red[2]);
  float st = 0.f, s1 = 0.f;
  for (int i = tid; i < a.splits; i += 256) {
    const float x = part[3 * i] - m;  // a piece of nothing but -inf has sums of 0, one with NaN beside them sums that count
    st += part[3 * i + 1] * expf(x * a.inv_tau);
    s1 += part[3 * i + 2] * expf(x);
  }
  st = group_sum<256>(st, red[3]);
  s1 = group_sum<256>(s1, red[4]);
  const float loss = row_loss<256>(a, t, m, st, s1, psum, plogp, label, zlabel, tid, red[5]);
  if (tid == 0) {
    a.loss[n] = loss;
    float4 q = {m, st, s1, 0.f};
    *reinterpret_cast<float4 *>(a.stats + 4 * n) = q;
  }
}

// Gradient of a piece of a row (workgroup n * splits + piece) from the row's statistics.
template <typename T>
__global__ __launch_bounds__(256) void k_distill_bwd(DistillArgs a) {
  extern __shared__ char lds[];
  __shared__ float red[2][4];
  const int tid = threadIdx.x;
  const long n = blockIdx.x / a.splits;
  const Teacher t = teacher_lds(lds, a.K);
  const T *row = (const T *)a.z + n * a.ldz;
  const int label = row_label(a, n);
  const int lo = (int)(blockIdx.x - n * a.splits) * a.piece, hi = min(a.V, lo + a.piece);
  // another workgroup may already have replaced z by dz outside [lo, hi): only elements inside are read
  const bool mine = label >= lo && label < hi;
  const float zlabel = mine ? (float)row[label] : 0.f;
  float psum, plogp;
  teacher_load<T, 256>(a, t, row, n, lo, hi, label, tid, red[0], psum, plogp);
  const float4 q = *reinterpret_cast<const float4 *>(a.stats + 4 * n);
  const float dl = a.dloss[n];
  const RowGrad g = row_grad(a, q.x, q.y, q.z, psum, dl, label);
  T *out = (T *)a.dz + n * a.ldd;
  for (int at = lo + tid * 8; at < hi; at += 2048) {
    float f[8];
    to_f32<T>(load8<T>(row + at, hi - at, (T)0.f), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = dense_grad<T>(a, g, f[e]);
    store8<T>(out + at, hi - at, from_f32<T>(f));
  }
  __syncthreads();
  correct<T, 256>(a, t, g, out, dl, label, zlabel, lo, hi, tid);
}

// Elements of a row that one workgroup takes where rows are cut: 8192, fewer while the grid would not fill the chip.
int piece_of(const vt_distill *a) {
  int piece = 8192;
  while (piece > 2048 && (long)a->N * ((a->V + piece - 1) / piece) < 512) piece /= 2;
  return piece;
}
// The widest instances hold a row in 512 threads' registers, 128 elements of 16 bits or 64 of fp32 each.
int row_limit(int dtype) { return dtype == VT_F32 ? 32768 : 65536; }
bool cut_rows(const vt_distill *a) { return a->V > row_limit(a->dtype) || (a->N < 128 && a->V > 8192); }
long part_floats(const vt_distill *a) {
  const int piece = piece_of(a);
  return (3L * a->N * ((a->V + piece - 1) / piece) + 3) & ~3L;
}

int check_args(const vt_distill *a) {
  if (!a || !a->z || !a->top_logit || !a->top_id || a->N < 1 || a->V < 1 || a->K < 1 || a->K > a->V || a->ldz < a->V ||
      !(a->tau > 0.f) || !(a->tau < INFINITY))
    return VT_EINVAL;
  if (a->dtype != VT_F32 && a->dtype != VT_BF16 && a->dtype != VT_F16) return VT_EUNSUPPORTED;
  // columns are counted in int, a launch's threads (256 a piece of a row at most) in 32 bits
  if (a->K > 1024 || a->V > (1 << 30) || (long)a->N * ((a->V + 2047) / 2048) >= (1L << 24)) return VT_EUNSUPPORTED;
  return 0;
}

// Whether dz's rows lie apart from z's, or are z's own: between the two matrices, beside each other in one, or in place.
bool rows_apart(const vt_distill *a, const void *dz) {
  const long size = a->dtype == VT_F32 ? 4 : 2, v = a->V * size;
  const long zspan = ((a->N - 1L) * a->ldz + a->V) * size, dspan = ((a->N - 1L) * a->ldd + a->V) * size;
  const uintptr_t z = (uintptr_t)a->z, d = (uintptr_t)dz;
  if (d >= z + zspan || z >= d + dspan) return true;
  if (a->ldz != a->ldd) return false;
  if (d == z) return true;
  const long row = a->ldz * size, off = (long)((d > z ? d - z : z - d) % row);
  return off >= v && off <= row - v;
}

DistillArgs kernel_args(const vt_distill *a) {
  DistillArgs k = {};
  k.z = a->z;
  k.top = a->top_logit;
  k.id = a->top_id;
  k.label = a->labels;
  k.ldz = a->ldz;
  k.ldd = a->ldd;
  k.N = a->N;
  k.V = a->V;
  k.K = a->K;
  k.piece = piece_of(a);
  k.splits = (a->V + k.piece - 1) / k.piece;
  k.tau = a->tau;
  k.inv_tau = 1.f / a->tau;
  k.kd = a->kd_weight;
  k.ce = a->ce_weight;
  return k;
}

template <typename T, bool GRAD>
int launch_rows(const DistillArgs &k, hipStream_t s) {
  const int V = k.V, tb = TEACHER_BYTES(k.K);
#define VT_ROW(GS, NC)                                                                                                   \
  if (V <= (GS) * 8 * (NC)) {                                                                                            \
    hipLaunchKernelGGL((k_distill_row<T, GS, NC, GRAD>), dim3((GS) == 64 ? (unsigned)((k.N + 3L) / 4) : (unsigned)k.N),   \
                       dim3((GS) == 64 ? 256 : (GS)), (GS) == 64 ? 4 * tb : tb, s, k);                                   \
    VT_CHECK_LAUNCH();                                                                                                   \
    return 0;                                                                                                            \
  }
  // eight columns a thread and chunk; four workgroups a compute unit up to 32768 columns of 16 bits (16384 of fp32), so that
  // one row's loads run beside another's reductions (4096 x 32000 bf16: 199 us with one workgroup of 1024
  // threads, 135 to 140 with four of 256, 524 MB at 3.8 TB/s)
  VT_ROW(64, 1)
  VT_ROW(64, 2)
  VT_ROW(256, 1)
  VT_ROW(256, 2)
  VT_ROW(256, 4)
  VT_ROW(256, 8)
  if constexpr (sizeof(T) == 2) {
    VT_ROW(256, 16)
    VT_ROW(512, 16)
  } else {
    VT_ROW(512, 8)
  }
#undef VT_ROW
  return VT_EUNSUPPORTED;
}

}  // namespace
}  // namespace vt

using namespace vt;

extern "C" long vt_distill_scratch_floats(const vt_distill *a) {
  if (check_args(a) != 0) return 0;
  return cut_rows(a) ? part_floats(a) + 4L * a->N : 0;
}

extern "C" int vt_distill_fwd(const vt_distill *a, float *loss, float *stats, float *scratch, long scratch_floats, vt_stream s) {
  const int rc = check_args(a);
  if (rc != 0) return rc;
  if (!loss || !stats || ((uintptr_t)stats & 15)) return VT_EINVAL;
  DistillArgs k = kernel_args(a);
  k.loss = loss;
  k.stats = stats;
  if (!cut_rows(a)) {
    VT_DISPATCH_TYPE(a->dtype, return (launch_rows<T, false>(k, (hipStream_t)s)));
    return 0;
  }
  if (scratch_floats < vt_distill_scratch_floats(a)) return VT_ELIMIT;
  if (!scratch || ((uintptr_t)scratch & 15)) return VT_EINVAL;
  k.part = scratch;
  VT_DISPATCH_TYPE(a->dtype, {
    hipLaunchKernelGGL((k_distill_part<T>), dim3((unsigned)k.splits * k.N), dim3(256), 0, (hipStream_t)s, k);
    hipLaunchKernelGGL((k_distill_join<T>), dim3(k.N), dim3(256), TEACHER_BYTES(k.K), (hipStream_t)s, k);
  });
  VT_CHECK_LAUNCH();
  return 0;
}

extern "C" int vt_distill_bwd(const vt_distill *a, const float *dloss, const float *stats, void *dz, vt_stream s) {
  const int rc = check_args(a);
  if (rc != 0) return rc;
  if (!dloss || !stats || !dz || ((uintptr_t)stats & 15) || a->ldd < a->V || !rows_apart(a, dz)) return VT_EINVAL;
  DistillArgs k = kernel_args(a);
  k.dloss = dloss;
  k.stats = const_cast<float *>(stats);
  k.dz = dz;
  VT_DISPATCH_TYPE(a->dtype,
                   hipLaunchKernelGGL((k_distill_bwd<T>), dim3((unsigned)k.splits * k.N), dim3(256), TEACHER_BYTES(k.K), (hipStream_t)s, k));
  VT_CHECK_LAUNCH();
  return 0;
}

extern "C" int vt_distill_fwd_bwd(const vt_distill *a, const float *dloss, float *loss, void *dz, float *scratch,
                                  long scratch_floats, vt_stream s) {
  const int rc = check_args(a);
  if (rc != 0) return rc;
  if (!dloss || !loss || !dz || a->ldd < a->V || !rows_apart(a, dz)) return VT_EINVAL;
  if (cut_rows(a)) {
    if (scratch_floats < vt_distill_scratch_floats(a)) return VT_ELIMIT;
    if (!scratch || ((uintptr_t)scratch & 15)) return VT_EINVAL;
    float *stats = scratch + part_floats(a);
    const int rf = vt_distill_fwd(a, loss, stats, scratch, scratch_floats, s);
    return rf != 0 ? rf : vt_distill_bwd(a, dloss, stats, dz, s);
  }
  DistillArgs k = kernel_args(a);
  k.dloss = dloss;
  k.loss = loss;
  k.dz = dz;
  VT_DISPATCH_TYPE(a->dtype, return (launch_rows<T, true>(k, (hipStream_t)s)));
  return 0;
}
