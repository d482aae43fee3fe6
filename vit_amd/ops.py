"""Operators of larger transformers over torch tensors, on top of the C ABI: attention with a learned relative position
bias, the norms around a block and distillation from a teacher's top logits (include/vtcnn_hip.h, "Operators of larger
transformers").

Every function checks its arguments on the host (ValueError), runs on the current stream of its tensors' device and
allocates results and scratch as torch tensors on that stream; nothing is kept between calls, so calls from several
streams or captured graphs do not share memory.  There is no CPU path and no autograd: `*_fwd` and `*_bwd` pairs, like the
launchers below them; while gradients are recorded, inputs that require one are refused (call under torch.no_grad(), in a
torch.autograd.Function or on detached tensors), since theirs would be lost without a word.  Tensors made on another stream
are ordered and kept alive by the caller, as for any torch operator.

A call of the smallest sizes costs what its checks and allocations cost the host (10 to 20 us), not what its kernels take:
descriptors are packed as bytes, and messages are formed only when they are raised.
"""
import struct

import torch

from ._lib import VtBlockNorms, VtDistill, VtRelposAttention, VtStrides, check, lib

VT_F32, VT_BF16, VT_F16 = 0, 1, 2
_DTYPE = {torch.float32: VT_F32, torch.bfloat16: VT_BF16, torch.float16: VT_F16}
VT_NORM_RMS, VT_NORM_LAYER = 0, 1
_KIND = {"rms": VT_NORM_RMS, "layer": VT_NORM_LAYER}
_F32, _I32 = torch.float32, torch.int32
_recording = torch.is_grad_enabled
_F32_MIN, _F32_MAX = 2.0 ** -126, (2.0 - 2.0 ** -23) * 2.0 ** 127  # normal numbers
# the descriptors of include/vtcnn_hip.h as bytes; None pointers are packed as 0
_DISTILL = struct.Struct("@4i2q3f4x4P")
_NORMS = struct.Struct("@5if6P")
_ATTENTION = struct.Struct("@10if4x8P9qi4x")


def _bad(text, *args):
    raise ValueError(text % args)


def _lost(what):
    _bad("%s requires a gradient, which this call does not record: call it under torch.no_grad() or on detached tensors", what)


def _beyond(e):
    raise ValueError("a size beyond 32 bits: %s" % e) from None


def _lead(t, what):
    """(element type code, device index) of the call's leading tensor."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _bad("%s: a tensor on a HIP device is needed", what)
    code = _DTYPE.get(t.dtype)
    if code is None:
        _bad("%s: element type %s is not one of float32, bfloat16, float16", what, t.dtype)
    if t.requires_grad and _recording():
        _lost(what)
    return code, t.get_device()


def _ptr(t, what, dev, dtype, shape):
    """Address of a contiguous tensor of the given type and shape on the leading tensor's device."""
    if not isinstance(t, torch.Tensor) or t.get_device() != dev:  # -1 on the host
        _bad("%s: a tensor on HIP device %d is needed", what, dev)
    if t.dtype != dtype:
        _bad("%s: element type %s, %s is needed", what, t.dtype, dtype)
    if t.shape != shape:
        _bad("%s: shape %s, %s is needed", what, tuple(t.shape), tuple(shape))
    if not t.is_contiguous():
        _bad("%s: not contiguous", what)
    if t.requires_grad and _recording():
        _lost(what)
    return t.data_ptr()


def _opt(t, what, dev, dtype, shape):
    return 0 if t is None else _ptr(t, what, dev, dtype, shape)


def _on(dev, call, *args):
    """call(current stream of device dev, *args) with that device current."""
    if dev == torch._C._cuda_getDevice():
        return call(torch._C._cuda_getCurrentRawStream(dev), *args)
    with torch.cuda.device(dev):
        return call(torch._C._cuda_getCurrentRawStream(dev), *args)


def _scratch(floats, lead):
    """Scratch of a call as (tensor or None, its address): kept by the caller's frame until the call is issued."""
    if floats <= 0:
        return None, None
    t = lead.new_empty(floats, dtype=_F32)
    return t, t.data_ptr()


# ---------------------------------------------------------------------------------------------
# Distillation
# ---------------------------------------------------------------------------------------------
def _rows(t, what, v):
    """Elements from row to row of a matrix whose rows may be strided."""
    s0, s1 = t.stride()
    if s1 != 1 and v > 1:
        _bad("%s: the elements of a row are not adjacent", what)
    if t.shape[0] == 1:
        return v
    if s0 < v:
        _bad("%s: rows overlap", what)
    return s0


def _distill_args(logits, top_logit, top_id, labels, tau, kd_weight, ce_weight, out=None):
    code, dev = _lead(logits, "logits")
    if logits.dim() != 2 or logits.numel() == 0:
        _bad("logits: shape %s, [N, V] is needed", tuple(logits.shape))
    n, v = logits.shape
    ldz = _rows(logits, "logits", v)
    if not isinstance(top_logit, torch.Tensor) or top_logit.dim() != 2 or not 1 <= top_logit.shape[1] <= min(v, 1024):
        _bad("top_logit: [N, K] with K from 1 to min(V, 1024) is needed")
    k = top_logit.shape[1]
    if not _F32_MIN <= tau <= _F32_MAX:
        _bad("tau: %r is not a positive number of float32", tau)
    if not (-_F32_MAX <= kd_weight <= _F32_MAX and -_F32_MAX <= ce_weight <= _F32_MAX):
        _bad("kd_weight, ce_weight: %r, %r are not finite numbers of float32", kd_weight, ce_weight)
    ldd = v
    if out is not None:
        if not isinstance(out, torch.Tensor) or out.device != logits.device or out.dtype != logits.dtype or out.shape != logits.shape:
            _bad("out: a tensor like logits is needed")
        ldd = _rows(out, "out", v)
    fields = (code, n, v, k, ldz, ldd, tau, kd_weight, ce_weight, logits.data_ptr(), _ptr(top_logit, "top_logit", dev, _F32, (n, k)),
              _ptr(top_id, "top_id", dev, _I32, (n, k)), _opt(labels, "labels", dev, _I32, (n,)))
    try:
        return VtDistill.from_buffer_copy(_DISTILL.pack(*fields)), dev, n
    except struct.error as e:
        _beyond(e)


def distill_fwd(logits, top_logit, top_id, labels=None, tau=1.0, kd_weight=1.0, ce_weight=0.0):
    """Loss of each row of the student's logits [N, V] against the teacher's best K logits (top_logit float32, top_id
    int32, both [N, K]; ids outside [0, V) are ignored) and, where labels (int32 [N]) are given and inside [0, V), the
    cross-entropy of the label: kd_weight tau^2 KL(teacher || student) + ce_weight CE (vt_distill_fwd).  The rows of
    logits may be strided.  Returns (loss [N], stats [N, 4]); stats goes to distill_bwd."""
    a, dev, n = _distill_args(logits, top_logit, top_id, labels, tau, kd_weight, ce_weight)

    def call(stream):
        loss, stats = logits.new_empty(n, dtype=_F32), logits.new_empty((n, 4), dtype=_F32)
        floats = lib.vt_distill_scratch_floats(a)
        scratch, at = _scratch(floats, logits)
        check(lib.vt_distill_fwd(a, loss.data_ptr(), stats.data_ptr(), at, floats, stream), "vt_distill_fwd")
        return loss, stats

    return _on(dev, call)


def distill_bwd(logits, top_logit, top_id, dloss, stats, labels=None, tau=1.0, kd_weight=1.0, ce_weight=0.0, out=None):
    """Gradient of the logits from the gradient dloss [N] of each row's loss and distill_fwd's stats (vt_distill_bwd).
    out: a tensor like logits to write it to, logits itself among them."""
    a, dev, n = _distill_args(logits, top_logit, top_id, labels, tau, kd_weight, ce_weight, out)
    dl, st = _ptr(dloss, "dloss", dev, _F32, (n,)), _ptr(stats, "stats", dev, _F32, (n, 4))

    def call(stream):
        dz = logits.new_empty(logits.shape) if out is None else out
        check(lib.vt_distill_bwd(a, dl, st, dz.data_ptr(), stream), "vt_distill_bwd")
        return dz

    return _on(dev, call)


def distill_fwd_bwd(logits, top_logit, top_id, dloss, labels=None, tau=1.0, kd_weight=1.0, ce_weight=0.0, out=None):
    """Loss and gradient in one call, for a step that knows dloss [N] beforehand (1 / N for a mean): the logits are read
    once where a row fits a workgroup's registers (vt_distill_fwd_bwd).  Returns (loss, dlogits)."""
    a, dev, n = _distill_args(logits, top_logit, top_id, labels, tau, kd_weight, ce_weight, out)
    dl = _ptr(dloss, "dloss", dev, _F32, (n,))

    def call(stream):
        loss, dz = logits.new_empty(n, dtype=_F32), logits.new_empty(logits.shape) if out is None else out
        floats = lib.vt_distill_scratch_floats(a)
        scratch, at = _scratch(floats, logits)
        check(lib.vt_distill_fwd_bwd(a, dl, loss.data_ptr(), dz.data_ptr(), at, floats, stream), "vt_distill_fwd_bwd")
        return loss, dz

    return _on(dev, call)


# ---------------------------------------------------------------------------------------------
# The norms around a block
# ---------------------------------------------------------------------------------------------
def _norm_args(x, y, gate, rows_per_gate, res_scale, w_post, b_post, w_pre, b_pre, kind, eps):
    """(descriptor, device index, addresses of x and y)."""
    code, dev = _lead(x, "x")
    if x.dim() != 2 or x.numel() == 0:
        _bad("x: shape %s, [N, D] is needed", tuple(x.shape))
    n, d = x.shape
    if d > 8192:
        _bad("x: rows of %d elements, at most 8192 are supported", d)
    if kind not in _KIND:
        _bad("kind: %r is not one of 'rms', 'layer'", kind)
    if not 0.0 <= eps <= _F32_MAX:
        _bad("eps: %r is negative or not finite", eps)
    if rows_per_gate < 1:
        _bad("rows_per_gate: %r is not positive", rows_per_gate)
    if (b_post is not None and (kind != "layer" or w_post is None)) or (b_pre is not None and (kind != "layer" or w_pre is None)):
        _bad("b_post, b_pre: only beside w_post, w_pre and with kind 'layer'")
    ty, row = x.dtype, (d,)
    xp, yp = _ptr(x, "x", dev, ty, (n, d)), _ptr(y, "y", dev, ty, (n, d))
    fields = (code, _KIND[kind], n, d, min(rows_per_gate, n), eps, _opt(gate, "gate", dev, ty, ((n + rows_per_gate - 1) // rows_per_gate, d)),
              _opt(res_scale, "res_scale", dev, _F32, row), _opt(w_post, "w_post", dev, _F32, row), _opt(b_post, "b_post", dev, _F32, row),
              _opt(w_pre, "w_pre", dev, _F32, row), _opt(b_pre, "b_pre", dev, _F32, row))
    try:
        return VtBlockNorms.from_buffer_copy(_NORMS.pack(*fields)), dev, xp, yp
    except struct.error as e:
        _beyond(e)


def block_norms_fwd(x, y, gate=None, rows_per_gate=1, res_scale=None, w_post=None, b_post=None, w_pre=None, b_pre=None, kind="rms",
                    eps=1e-6):
    """From a block's output y to the next block's input: r = x + res_scale * gate * norm(y; w_post, b_post) and
    h = norm(r; w_pre, b_pre) (vt_block_norms_fwd).  x, y [N, D] of one element type; gate [ceil(N / rows_per_gate), D] of
    that type, each row for rows_per_gate rows of x; res_scale and the norms' weights float32 [D].  Any of gate, res_scale,
    w_post, w_pre may be None (without w_post there is no norm on y, without w_pre no h).  Returns (r, h or None, stats);
    stats goes to block_norms_bwd."""
    a, dev, xp, yp = _norm_args(x, y, gate, rows_per_gate, res_scale, w_post, b_post, w_pre, b_pre, kind, eps)

    def call(stream):
        r = torch.empty_like(x)
        h = None if w_pre is None else torch.empty_like(x)
        stats = x.new_empty((x.shape[0], 4), dtype=_F32)
        check(lib.vt_block_norms_fwd(a, xp, yp, r.data_ptr(), None if h is None else h.data_ptr(), stats.data_ptr(), stream),
              "vt_block_norms_fwd")
        return r, h, stats

    return _on(dev, call)


def block_norms_bwd(dr, dh, x, y, stats, gate=None, rows_per_gate=1, res_scale=None, w_post=None, b_post=None, w_pre=None, b_pre=None,
                    kind="rms", eps=1e-6):
    """Gradients of block_norms_fwd from those of r (dr, may be None where dh is given) and of h (dh, None without w_pre)
    (vt_block_norms_bwd).  Returns a dict with dx, dy and, for each argument that is given (None otherwise), dgate,
    dres_scale, dw_post, db_post, dw_pre, db_pre."""
    a, dev, xp, yp = _norm_args(x, y, gate, rows_per_gate, res_scale, w_post, b_post, w_pre, b_pre, kind, eps)
    if dr is None and dh is None:
        _bad("dr, dh: one of them is needed")
    if (dh is None) != (w_pre is None):
        _bad("dh: given exactly with w_pre")
    drp, dhp = _opt(dr, "dr", dev, x.dtype, x.shape), _opt(dh, "dh", dev, x.dtype, x.shape)
    sp = _ptr(stats, "stats", dev, _F32, (x.shape[0], 4))

    def call(stream):
        g = {"dx": torch.empty_like(x), "dy": torch.empty_like(x), "dgate": None if gate is None else torch.empty_like(gate)}
        weights = (("dres_scale", res_scale), ("dw_post", w_post), ("db_post", b_post), ("dw_pre", w_pre), ("db_pre", b_pre))
        # one allocation for the weights' gradients
        rows = iter(x.new_empty((5, x.shape[1]), dtype=_F32).unbind(0))
        at = []
        for name, w in weights:
            g[name] = t = None if w is None else next(rows)
            at.append(None if t is None else t.data_ptr())
        floats = lib.vt_block_norms_bwd_scratch_floats(a)
        scratch, sat = _scratch(floats, x)
        check(lib.vt_block_norms_bwd(a, xp, yp, sp, drp, dhp, g["dx"].data_ptr(), g["dy"].data_ptr(),
                                     None if gate is None else g["dgate"].data_ptr(), *at, sat, floats, stream), "vt_block_norms_bwd")
        return g

    return _on(dev, call)


# ---------------------------------------------------------------------------------------------
# Attention with a learned relative position bias
# ---------------------------------------------------------------------------------------------
def relpos_buckets(num_buckets=32, max_distance=128, bidirectional=True, device=None):
    """Bucket of each distance key - query from -max_distance to max_distance as an int32 tensor [2 max_distance + 1] for
    relpos_attention_fwd (vt_relpos_buckets): half of a side's buckets hold single distances, the others ranges that grow
    geometrically up to max_distance; bidirectional=False is the scheme of causal attention."""
    # within the library's own int, where it refuses them
    num_buckets, max_distance = (max(-1, min(int(x), 1 << 30)) for x in (num_buckets, max_distance))
    m = torch.empty(2 * min(max(max_distance, 0), 2048) + 1, dtype=torch.int32)
    check(lib.vt_relpos_buckets(num_buckets, max_distance, int(bool(bidirectional)), m.data_ptr()), "vt_relpos_buckets")
    return m if device is None else m.to(device)


def _heads(t, what, dev, dtype, shape):
    """(address, strides of B, T, H) of a [B, T, H, d] tensor of the leading one's type and device."""
    if not isinstance(t, torch.Tensor) or t.get_device() != dev:  # -1 on the host
        _bad("%s: a tensor on HIP device %d is needed", what, dev)
    if t.dtype != dtype:
        _bad("%s: element type %s, %s is needed", what, t.dtype, dtype)
    if t.shape != shape:
        _bad("%s: shape %s, %s is needed", what, tuple(t.shape), tuple(shape))
    b, s, h, e = t.stride()
    if e != 1 and shape[3] != 1:
        _bad("%s: the elements of a head are not adjacent", what)
    if t.requires_grad and _recording():
        _lost(what)
    return t.data_ptr(), b, s, h


def _attention_args(q, k, v, table, buckets, scale, causal, q_start, q_len, k_len, precise=0):
    """(descriptor, device index)."""
    code, dev = _lead(q, "q")
    if q.dim() != 4 or q.numel() == 0:
        _bad("q: shape %s, [B, Tq, Hq, d] is needed", tuple(q.shape))
    b, tq, hq, d = q.shape
    if d > 128:
        _bad("q: heads of %d elements, at most 128 are supported", d)
    if not isinstance(k, torch.Tensor) or k.dim() != 4 or k.numel() == 0:
        _bad("k: [B, Tk, Hk, d] is needed")
    tk, hk = k.shape[1], k.shape[2]
    if hq % hk:
        _bad("k: %d heads do not divide the %d of q", hk, hq)
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.shape[0] < 1:
        _bad("table: [num_buckets, Hq] is needed")
    nb = table.shape[0]
    if not isinstance(buckets, torch.Tensor) or buckets.dim() != 1 or buckets.shape[0] % 2 != 1 or buckets.shape[0] > 4097:
        _bad("buckets: [2 max_distance + 1] with max_distance at most 2048 is needed")
    width = buckets.shape[0]
    scale = d ** -0.5 if scale is None else float(scale)
    if not -_F32_MAX <= scale <= _F32_MAX:
        _bad("scale: %r is not a finite number of float32", scale)
    ty, keys, row = q.dtype, (b, tk, hk, d), (b,)
    qp, qb, qt, qh = _heads(q, "q", dev, ty, q.shape)
    kp, kb, kt, kh = _heads(k, "k", dev, ty, keys)
    vp, vb, vt, vh = _heads(v, "v", dev, ty, keys)
    fields = (code, b, tq, tk, hq, hk, d, 1 if causal else 0, nb, width // 2, scale, _ptr(buckets, "buckets", dev, _I32, (width,)),
              _ptr(table, "table", dev, _F32, (nb, hq)), _opt(q_start, "q_start", dev, _I32, row), _opt(q_len, "q_len", dev, _I32, row),
              _opt(k_len, "k_len", dev, _I32, row), qp, kp, vp, qb, qt, qh, kb, kt, kh, vb, vt, vh, precise)
    try:
        return VtRelposAttention.from_buffer_copy(_ATTENTION.pack(*fields)), dev
    except struct.error as e:
        _beyond(e)


def _packed(t, h, d):
    """Strides of a contiguous [B, t, h, d] tensor."""
    return VtStrides(t * h * d, h * d, d)


def relpos_attention_fwd(q, k, v, table, buckets, scale=None, causal=False, q_start=None, q_len=None, k_len=None, training=False):
    """Attention with a learned bias by the bucket of the distance key - query (vt_relpos_attention_fwd).

    q [B, Tq, Hq, d], k and v [B, Tk, Hk, d] of one element type, Hk dividing Hq, the elements of a head adjacent and any
    other strides; table float32 [num_buckets, Hq]; buckets int32 [2 max_distance + 1] on the device (relpos_buckets, or
    the caller's own scheme); scale defaults to d ** -0.5.  q_len and k_len (int32 [B]): queries and keys in use of each
    sequence of a padded batch; q_start (int32 [B]): place of query 0 among the keys, for a prompt or a token behind a
    cache; with causal, query i sees keys up to q_start + i.  A query that sees no key has output 0, and so have queries
    behind q_len.  Returns out [B, Tq, Hq, d], and with training=True (out, saved) for relpos_attention_bwd."""
    a, dev = _attention_args(q, k, v, table, buckets, scale, causal, q_start, q_len, k_len)

    def call(stream):
        b, tq, hq, d = shape = q.shape
        out = q.new_empty(shape)
        stats = lo = sp = lp = None
        if training:
            stats = q.new_empty((b, hq, tq, 2), dtype=_F32)
            sp = stats.data_ptr()
            if q.dtype != _F32:
                lo = q.new_empty(shape)
                lp = lo.data_ptr()
        floats = lib.vt_relpos_attention_fwd_scratch_floats(a)
        scratch, at = _scratch(floats, q)
        check(lib.vt_relpos_attention_fwd(a, out.data_ptr(), _packed(tq, hq, d), lp, sp, at, floats, stream), "vt_relpos_attention_fwd")
        return (out, (stats, lo)) if training else out

    return _on(dev, call)


def relpos_attention_bwd(dout, q, k, v, out, saved, table, buckets, scale=None, causal=False, q_start=None, q_len=None, k_len=None,
                         precise=False):
    """Gradients (dq, dk, dv, dtable) of relpos_attention_fwd(..., training=True) from the gradient of its output and what
    it returned (vt_relpos_attention_bwd); the other arguments as there.  Padded rows of dq, dk, dv are 0.  With 16-bit
    types and more than 32 queries the probabilities and score gradients are rounded to the type once on their way (1.4 times
    the error of the results' own rounding); precise=True takes them in two parts instead (2 x 4096 tokens, 16 heads of 128 in bf16: 901
    us instead of 629)."""
    a, dev = _attention_args(q, k, v, table, buckets, scale, causal, q_start, q_len, k_len, 1 if precise else 0)
    b, tq, hq, d = shape = q.shape
    tk, hk = k.shape[1], k.shape[2]
    dp, db, dt, dh = _heads(dout, "dout", dev, q.dtype, shape)
    op = _ptr(out, "out", dev, q.dtype, shape)
    if not isinstance(saved, tuple) or len(saved) != 2:
        _bad("saved: what the forward call returned with training=True is needed")
    sp = _ptr(saved[0], "saved", dev, _F32, (b, hq, tq, 2))
    lp = None if q.dtype == _F32 else _ptr(saved[1], "saved", dev, q.dtype, shape)

    def call(stream):
        dq, dk, dv = q.new_empty(shape), q.new_empty((b, tk, hk, d)), q.new_empty((b, tk, hk, d))
        dtable = torch.empty_like(table)
        floats = lib.vt_relpos_attention_bwd_scratch_floats(a)
        scratch, at = _scratch(floats, q)
        of_q, of_k = _packed(tq, hq, d), _packed(tk, hk, d)
        check(lib.vt_relpos_attention_bwd(a, op, of_q, lp, sp, dp, VtStrides(db, dt, dh), dq.data_ptr(), of_q, dk.data_ptr(), of_k,
                                          dv.data_ptr(), of_k, dtable.data_ptr(), at, floats, stream), "vt_relpos_attention_bwd")
        return dq, dk, dv, dtable

    return _on(dev, call)
