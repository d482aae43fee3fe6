"""Operators of larger transformers over torch tensors, on top of the C ABI: attention with a learned relative position
bias, the norms around a block and distillation from a teacher's top logits (include/vtcnn_hip.h, "Operators of larger transformers").

Every function checks its arguments on the host (ValueError), runs on the current stream of its tensors' device and
allocates results and scratch as torch tensors on that stream; nothing is kept between calls, so calls from several
streams or captured graphs do not share memory.  There is no CPU path and no autograd: `*_fwd` and `*_bwd` pairs, like the
launchers below them.  Tensors made on another stream are ordered and kept alive by the caller, as for any torch operator.
"""
import ctypes as C

import torch

from ._lib import VtBlockNorms, VtDistill, VtRelposAttention, VtStrides, check, lib

VT_F32, VT_BF16, VT_F16 = 0, 1, 2
_DTYPE = {torch.float32: VT_F32, torch.bfloat16: VT_BF16, torch.float16: VT_F16}
VT_NORM_RMS, VT_NORM_LAYER = 0, 1
_KIND = {"rms": VT_NORM_RMS, "layer": VT_NORM_LAYER}


def _need(ok, text, *args):
    if not ok:
        raise ValueError(text % args)


def _typed(t, what):
    """Element type code of the call's leading tensor."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, "%s: a tensor on a HIP device is needed", what)
    _need(t.dtype in _DTYPE, "%s: element type %s is not one of float32, bfloat16, float16", what, t.dtype)
    return _DTYPE[t.dtype]


def _tensor(t, what, lead, dtype, shape):
    """A contiguous tensor of the given type and shape on the leading tensor's device."""
    _need(isinstance(t, torch.Tensor) and t.device == lead.device, "%s: a tensor on %s is needed", what, lead.device)
    _need(t.dtype == dtype, "%s: element type %s, %s is needed", what, t.dtype, dtype)
    _need(tuple(t.shape) == tuple(shape), "%s: shape %s, %s is needed", what, tuple(t.shape), tuple(shape))
    _need(t.is_contiguous(), "%s: not contiguous", what)
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


class _Call:
    """The leading tensor's device made current for a call, and its current stream."""

    __slots__ = ("device", "guard", "stream")

    def __init__(self, lead):
        self.device = lead.device
        self.guard = None if lead.device.index == torch.cuda.current_device() else torch.cuda.device(lead.device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        self.stream = torch.cuda.current_stream(self.device).cuda_stream
        return self

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _scratch(floats, lead):
    return torch.empty(floats, dtype=torch.float32, device=lead.device) if floats > 0 else None


# ---------------------------------------------------------------------------------------------
# Distillation
# ---------------------------------------------------------------------------------------------
def _distill_args(logits, top_logit, top_id, labels, tau, kd_weight, ce_weight, out=None):
    code = _typed(logits, "logits")
    _need(logits.dim() == 2 and logits.shape[0] >= 1 and logits.shape[1] >= 1, "logits: shape %s, [N, V] is needed", tuple(logits.shape))
    n, v = logits.shape
    _need(v == 1 or logits.stride(1) == 1, "logits: the elements of a row are not adjacent")
    _need(n == 1 or logits.stride(0) >= v, "logits: rows overlap")
    _need(isinstance(top_logit, torch.Tensor) and top_logit.dim() == 2, "top_logit: [N, K] is needed")
    k = top_logit.shape[1]
    _need(1 <= k <= min(v, 1024), "top_logit: %d entries a row, 1 to min(V, 1024) are needed", k)
    _tensor(top_logit, "top_logit", logits, torch.float32, (n, k))
    _tensor(top_id, "top_id", logits, torch.int32, (n, k))
    if labels is not None:
        _tensor(labels, "labels", logits, torch.int32, (n,))
    _need(0.0 < tau < float("inf"), "tau: %r is not a positive number", tau)
    a = VtDistill(code, n, v, k, logits.stride(0) if n > 1 else v, v, tau, kd_weight, ce_weight, logits.data_ptr(),
                  top_logit.data_ptr(), top_id.data_ptr(), _ptr(labels))
    if out is not None:
        _need(out.device == logits.device and out.dtype == logits.dtype and out.shape == logits.shape,
              "out: a tensor like logits is needed")
        _need((v == 1 or out.stride(1) == 1) and (n == 1 or out.stride(0) >= v), "out: rows must not overlap, their elements be adjacent")
        a.ldd = out.stride(0) if n > 1 else v
    return a, n


def distill_fwd(logits, top_logit, top_id, labels=None, tau=1.0, kd_weight=1.0, ce_weight=0.0):
    """Loss of each row of the student's logits [N, V] against the teacher's best K logits (top_logit float32, top_id
    int32, both [N, K]; ids outside [0, V) are ignored) and, where labels (int32 [N]) are given and inside [0, V), the
    cross-entropy of the label: kd_weight tau^2 KL(teacher || student) + ce_weight CE (vt_distill_fwd).  The rows of
    logits may be strided.  Returns (loss [N], stats [N, 4]); stats goes to distill_bwd."""
    a, n = _distill_args(logits, top_logit, top_id, labels, tau, kd_weight, ce_weight)
    with _Call(logits) as c:
        loss = torch.empty(n, dtype=torch.float32, device=logits.device)
        stats = torch.empty((n, 4), dtype=torch.float32, device=logits.device)
        floats = lib.vt_distill_scratch_floats(a)
        scratch = _scratch(floats, logits)
        check(lib.vt_distill_fwd(a, loss.data_ptr(), stats.data_ptr(), _ptr(scratch), floats, c.stream), "vt_distill_fwd")
    return loss, stats


def distill_bwd(logits, top_logit, top_id, dloss, stats, labels=None, tau=1.0, kd_weight=1.0, ce_weight=0.0, out=None):
    """Gradient of the logits from the gradient dloss [N] of each row's loss and distill_fwd's stats (vt_distill_bwd).
    out: a tensor like logits to write it to, logits itself among them."""
    a, n = _distill_args(logits, top_logit, top_id, labels, tau, kd_weight, ce_weight, out)
    _tensor(dloss, "dloss", logits, torch.float32, (n,))
    _tensor(stats, "stats", logits, torch.float32, (n, 4))
    with _Call(logits) as c:
        dz = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if out is None else out
        check(lib.vt_distill_bwd(a, dloss.data_ptr(), stats.data_ptr(), dz.data_ptr(), c.stream), "vt_distill_bwd")
    return dz


def distill_fwd_bwd(logits, top_logit, top_id, dloss, labels=None, tau=1.0, kd_weight=1.0, ce_weight=0.0, out=None):
    """Loss and gradient in one call, for a step that knows dloss [N] beforehand (1 / N for a mean): the logits are read
    once where a row fits a workgroup's registers (vt_distill_fwd_bwd).  Returns (loss, dlogits)."""
    a, n = _distill_args(logits, top_logit, top_id, labels, tau, kd_weight, ce_weight, out)
    _tensor(dloss, "dloss", logits, torch.float32, (n,))
    with _Call(logits) as c:
        loss = torch.empty(n, dtype=torch.float32, device=logits.device)
        dz = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device) if out is None else out
        floats = lib.vt_distill_scratch_floats(a)
        scratch = _scratch(floats, logits)
        check(lib.vt_distill_fwd_bwd(a, dloss.data_ptr(), loss.data_ptr(), dz.data_ptr(), _ptr(scratch), floats, c.stream),
              "vt_distill_fwd_bwd")
    return loss, dz


# ---------------------------------------------------------------------------------------------
# The norms around a block
# ---------------------------------------------------------------------------------------------
def _norm_args(x, y, gate, rows_per_gate, res_scale, w_post, b_post, w_pre, b_pre, kind, eps):
    code = _typed(x, "x")
    _need(x.dim() == 2 and x.shape[0] >= 1 and x.shape[1] >= 1, "x: shape %s, [N, D] is needed", tuple(x.shape))
    n, d = x.shape
    _need(d <= 8192, "x: rows of %d elements, at most 8192 are supported", d)
    _need(x.is_contiguous(), "x: not contiguous")
    _tensor(y, "y", x, x.dtype, (n, d))
    _need(kind in _KIND, "kind: %r is not one of 'rms', 'layer'", kind)
    _need(eps >= 0.0, "eps: %r is negative", eps)
    _need(rows_per_gate >= 1, "rows_per_gate: %r is not positive", rows_per_gate)
    if gate is not None:
        _tensor(gate, "gate", x, x.dtype, ((n + rows_per_gate - 1) // rows_per_gate, d))
    for name, w in (("res_scale", res_scale), ("w_post", w_post), ("b_post", b_post), ("w_pre", w_pre), ("b_pre", b_pre)):
        if w is not None:
            _tensor(w, name, x, torch.float32, (d,))
    for b, w, at in ((b_post, w_post, "post"), (b_pre, w_pre, "pre")):
        _need(b is None or (kind == "layer" and w is not None), "b_%s: only beside w_%s and with kind 'layer'", at, at)
    return VtBlockNorms(code, _KIND[kind], n, d, min(rows_per_gate, n), eps, _ptr(gate), _ptr(res_scale), _ptr(w_post), _ptr(b_post),
                        _ptr(w_pre), _ptr(b_pre))


def block_norms_fwd(x, y, gate=None, rows_per_gate=1, res_scale=None, w_post=None, b_post=None, w_pre=None, b_pre=None, kind="rms",
                    eps=1e-6):
    """From a block's output y to the next block's input: r = x + res_scale * gate * norm(y; w_post, b_post) and
    h = norm(r; w_pre, b_pre) (vt_block_norms_fwd).  x, y [N, D] of one element type; gate [ceil(N / rows_per_gate), D] of
    that type, each row for rows_per_gate rows of x; res_scale and the norms' weights float32 [D].  Any of gate, res_scale,
    w_post, w_pre may be None (without w_post there is no norm on y, without w_pre no h).  Returns (r, h or None, stats);
    stats goes to block_norms_bwd."""
    a = _norm_args(x, y, gate, rows_per_gate, res_scale, w_post, b_post, w_pre, b_pre, kind, eps)
    with _Call(x) as c:
        r = torch.empty_like(x)
        h = torch.empty_like(x) if w_pre is not None else None
        stats = torch.empty((a.N, 4), dtype=torch.float32, device=x.device)
        check(lib.vt_block_norms_fwd(a, x.data_ptr(), y.data_ptr(), r.data_ptr(), _ptr(h), stats.data_ptr(), c.stream),
              "vt_block_norms_fwd")
    return r, h, stats


def block_norms_bwd(dr, dh, x, y, stats, gate=None, rows_per_gate=1, res_scale=None, w_post=None, b_post=None, w_pre=None, b_pre=None,
                    kind="rms", eps=1e-6):
    """Gradients of block_norms_fwd from those of r (dr, may be None where dh is given) and of h (dh, None without w_pre)
    (vt_block_norms_bwd).  Returns a dict with dx, dy and, for each argument that is given (None otherwise), dgate,
    dres_scale, dw_post, db_post, dw_pre, db_pre."""
    a = _norm_args(x, y, gate, rows_per_gate, res_scale, w_post, b_post, w_pre, b_pre, kind, eps)
    _need(dr is not None or dh is not None, "dr, dh: one of them is needed")
    _need((dh is None) == (w_pre is None), "dh: given exactly with w_pre")
    for name, t in (("dr", dr), ("dh", dh)):
        if t is not None:
            _tensor(t, name, x, x.dtype, x.shape)
    _tensor(stats, "stats", x, torch.float32, (a.N, 4))
    with _Call(x) as c:
        g = {"dx": torch.empty_like(x), "dy": torch.empty_like(x), "dgate": None if gate is None else torch.empty_like(gate)}
        weights = [w for w in (res_scale, w_post, b_post, w_pre, b_pre)]
        rows = iter(torch.empty((max(1, sum(w is not None for w in weights)), a.D), dtype=torch.float32, device=x.device))
        for name, w in zip(("dres_scale", "dw_post", "db_post", "dw_pre", "db_pre"), weights):
            g[name] = None if w is None else next(rows)
        floats = lib.vt_block_norms_bwd_scratch_floats(a)
        scratch = _scratch(floats, x)
        check(lib.vt_block_norms_bwd(a, x.data_ptr(), y.data_ptr(), stats.data_ptr(), _ptr(dr), _ptr(dh), g["dx"].data_ptr(),
                                     g["dy"].data_ptr(), _ptr(g["dgate"]), _ptr(g["dres_scale"]), _ptr(g["dw_post"]), _ptr(g["db_post"]),
                                     _ptr(g["dw_pre"]), _ptr(g["db_pre"]), _ptr(scratch), floats, c.stream), "vt_block_norms_bwd")
    return g


# ---------------------------------------------------------------------------------------------
# Attention with a learned relative position bias
# ---------------------------------------------------------------------------------------------
def relpos_buckets(num_buckets=32, max_distance=128, bidirectional=True, device=None):
    """Bucket of each distance key - query from -max_distance to max_distance as an int32 tensor [2 max_distance + 1] for
    relpos_attention_fwd (vt_relpos_buckets): half of a side's buckets hold single distances, the others ranges that grow
    geometrically up to max_distance; bidirectional=False is the scheme of causal attention."""
    m = torch.empty(2 * max(int(max_distance), 0) + 1, dtype=torch.int32)
    check(lib.vt_relpos_buckets(int(num_buckets), int(max_distance), int(bool(bidirectional)), m.data_ptr()), "vt_relpos_buckets")
    return m if device is None else m.to(device)


def _strides(t):
    return VtStrides(t.stride(0), t.stride(1), t.stride(2))


def _heads(t, what, lead, shape):
    """[B, T, H, d] of the leading tensor's type and device; any strides for B, T and H."""
    _need(isinstance(t, torch.Tensor) and t.device == lead.device, "%s: a tensor on %s is needed", what, lead.device)
    _need(t.dtype == lead.dtype, "%s: element type %s, %s is needed", what, t.dtype, lead.dtype)
    _need(tuple(t.shape) == tuple(shape), "%s: shape %s, %s is needed", what, tuple(t.shape), tuple(shape))
    _need(t.shape[3] == 1 or t.stride(3) == 1, "%s: the elements of a head are not adjacent", what)
    return t


def _attention_args(q, k, v, table, buckets, scale, causal, q_start, q_len, k_len):
    code = _typed(q, "q")
    _need(q.dim() == 4 and min(q.shape) >= 1, "q: shape %s, [B, Tq, Hq, d] is needed", tuple(q.shape))
    b, tq, hq, d = q.shape
    _need(d <= 128, "q: heads of %d elements, at most 128 are supported", d)
    _heads(q, "q", q, q.shape)
    _need(isinstance(k, torch.Tensor) and k.dim() == 4 and min(k.shape) >= 1, "k: [B, Tk, Hk, d] is needed")
    tk, hk = k.shape[1], k.shape[2]
    _need(hq % hk == 0, "k: %d heads do not divide the %d of q", hk, hq)
    _heads(k, "k", q, (b, tk, hk, d))
    _heads(v, "v", q, (b, tk, hk, d))
    _need(isinstance(table, torch.Tensor) and table.dim() == 2 and table.shape[0] >= 1, "table: [num_buckets, Hq] is needed")
    nb = table.shape[0]
    _tensor(table, "table", q, torch.float32, (nb, hq))
    _need(isinstance(buckets, torch.Tensor) and buckets.dim() == 1 and buckets.numel() % 2 == 1 and buckets.numel() <= 4097,
          "buckets: [2 max_distance + 1] with max_distance at most 2048 is needed")
    _tensor(buckets, "buckets", q, torch.int32, (buckets.numel(),))
    for name, t in (("q_start", q_start), ("q_len", q_len), ("k_len", k_len)):
        if t is not None:
            _tensor(t, name, q, torch.int32, (b,))
    scale = d ** -0.5 if scale is None else float(scale)
    _need(-float("inf") < scale < float("inf"), "scale: %r is not finite", scale)
    return VtRelposAttention(code, b, tq, tk, hq, hk, d, int(bool(causal)), nb, buckets.numel() // 2, scale, buckets.data_ptr(),
                             table.data_ptr(), _ptr(q_start), _ptr(q_len), _ptr(k_len), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                             _strides(q), _strides(k), _strides(v))


def relpos_attention_fwd(q, k, v, table, buckets, scale=None, causal=False, q_start=None, q_len=None, k_len=None, training=False):
    """Attention with a learned bias by the bucket of the distance key - query (vt_relpos_attention_fwd).

    q [B, Tq, Hq, d], k and v [B, Tk, Hk, d] of one element type, Hk dividing Hq, the elements of a head adjacent and any
    other strides; table float32 [num_buckets, Hq]; buckets int32 [2 max_distance + 1] on the device (relpos_buckets, or
    the caller's own scheme); scale defaults to d ** -0.5.  q_len and k_len (int32 [B]): queries and keys in use of each
    sequence of a padded batch; q_start (int32 [B]): place of query 0 among the keys, for a prompt or a token behind a
    cache; with causal, query i sees keys up to q_start + i.  A query that sees no key has output 0, and so have queries
    behind q_len.  Returns out [B, Tq, Hq, d], and with training=True (out, saved) for relpos_attention_bwd."""
    a = _attention_args(q, k, v, table, buckets, scale, causal, q_start, q_len, k_len)
    with _Call(q) as c:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        stats = out_lo = None
        if training:
            stats = torch.empty((a.B, a.Hq, a.Tq, 2), dtype=torch.float32, device=q.device)
            if a.dtype != VT_F32:
                out_lo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        floats = lib.vt_relpos_attention_fwd_scratch_floats(a)
        scratch = _scratch(floats, q)
        check(lib.vt_relpos_attention_fwd(a, out.data_ptr(), _strides(out), _ptr(out_lo), _ptr(stats), _ptr(scratch), floats, c.stream),
              "vt_relpos_attention_fwd")
    return (out, (stats, out_lo)) if training else out


def relpos_attention_bwd(dout, q, k, v, out, saved, table, buckets, scale=None, causal=False, q_start=None, q_len=None, k_len=None):
    """Gradients (dq, dk, dv, dtable) of relpos_attention_fwd(..., training=True) from the gradient of its output and what
    it returned (vt_relpos_attention_bwd); the other arguments as there.  Padded rows of dq, dk, dv are 0."""
    a = _attention_args(q, k, v, table, buckets, scale, causal, q_start, q_len, k_len)
    _heads(dout, "dout", q, q.shape)
    _need(isinstance(out, torch.Tensor) and out.is_contiguous(), "out: the forward call's result is needed")
    _heads(out, "out", q, q.shape)
    _need(isinstance(saved, tuple) and len(saved) == 2, "saved: what the forward call returned with training=True is needed")
    stats, out_lo = saved
    _tensor(stats, "saved", q, torch.float32, (a.B, a.Hq, a.Tq, 2))
    if a.dtype != VT_F32:
        _tensor(out_lo, "saved", q, q.dtype, q.shape)
    with _Call(q) as c:
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk = torch.empty(k.shape, dtype=q.dtype, device=q.device)
        dv = torch.empty(k.shape, dtype=q.dtype, device=q.device)
        dtable = torch.empty(table.shape, dtype=torch.float32, device=q.device)
        floats = lib.vt_relpos_attention_bwd_scratch_floats(a)
        scratch = _scratch(floats, q)
        check(lib.vt_relpos_attention_bwd(a, out.data_ptr(), _strides(out), _ptr(out_lo), stats.data_ptr(), dout.data_ptr(), _strides(dout),
                                          dq.data_ptr(), _strides(dq), dk.data_ptr(), _strides(dk), dv.data_ptr(), _strides(dv),
                                          dtable.data_ptr(), _ptr(scratch), floats, c.stream), "vt_relpos_attention_bwd")
    return dq, dk, dv, dtable
