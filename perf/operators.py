"""Attention with a learned relative position bias, the norms around a block, and distillation from a teacher's top logits:
the calls that a training step, a prompt and a token of a served model make of them, at the sizes of this repository's
own configurations (16 and 196 tokens, widths 32 and 512, 8 and 10 classes) and at those of larger transformers.

`run` with `own` false is the plain form in elementary tensor operations, in 32 bits with one rounding at the end; with
`own` true it makes the calls of `vit_amd`.  `exact` states the same operators in 64 bits, one head or one operator at a time.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one training step of the attention of the 16-token, 32-channel, two-head transformer at a batch of 32
        attention("attn_16_tokens", "train", "f32", 32, 16, 16, 2, 2, 16, 32, 128),
        # the wide configuration: 196 tokens of 512 channels in 8 heads, a batch of 16
        attention("attn_196_tokens", "train", "bf16", 16, 196, 196, 8, 8, 64, 32, 128),
        # a causal decoder trained on long rows, keys and values shared by four query heads
        attention("attn_4096_causal", "train", "bf16", 2, 4096, 4096, 16, 4, 128, 32, 128, causal=True),
        # a padded batch of prompts of uneven lengths, one of them empty, an odd head width
        attention("attn_prompts", "fwd", "f16", 6, 1023, 1023, 12, 4, 80, 48, 200, causal=True, ragged=True),
        # one token a sequence against long caches of uneven fill
        attention("attn_token_long", "token", "bf16", 16, 1, 8192, 32, 8, 128, 32, 128, causal=True, ragged=True),
        # one token of one short sequence: latency
        attention("attn_token_short", "token", "f16", 1, 1, 777, 8, 8, 64, 32, 128, causal=True),
        # the small transformer's block in training, one gate row a sequence
        norms("norms_16_tokens", "train", "f32", 32 * 16, 32, "layer", 16),
        # a wide decoder's block in training, every token with a gate of its own
        norms("norms_8192_rows", "train", "bf16", 8192, 4096, "rms", 1),
        # a served prompt, odd sizes, no gate
        norms("norms_prompt", "fwd", "f16", 3137, 1001, "rms", 0),
        # the ten-class classifier taught by another one's four best classes
        distill("distill_classes", "both", "f32", 1024, 10, 4, 2.0),
        # a language model's loss and gradient in one call
        distill("distill_32000", "both", "bf16", 4096, 32000, 64, 1.0),
        # a few rows of a large odd vocabulary, loss first and gradient later
        distill("distill_few_rows", "split", "f16", 7, 131071, 100, 3.0),
    ]


def attention(name, way, dtype, b, tq, tk, hq, hk, d, buckets, reach, causal=False, ragged=False):
    c = dict(op="attention", way=way, dtype=dtype, b=b, tq=tq, tk=tk, hq=hq, hk=hk, d=d, buckets=buckets, reach=reach,
             causal=causal, ragged=ragged)
    return dict(c, name=name) if name else c


def norms(name, way, dtype, rows, width, kind, per_gate):
    """per_gate: rows that share a row of the gate; 0: no gate."""
    c = dict(op="norms", way=way, dtype=dtype, rows=rows, width=width, kind=kind, per_gate=per_gate)
    return dict(c, name=name) if name else c


def distill(name, way, dtype, rows, vocab, top, tau):
    c = dict(op="distill", way=way, dtype=dtype, rows=rows, vocab=vocab, top=top, tau=tau)
    return dict(c, name=name) if name else c


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    op = rng.choice(["train", "fwd", "token", "norms", "distill"])
    if op in ("train", "fwd", "token"):
        hk, share = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4])
        d = rng.choice([16, 32, 40, 64, 64, 80, 96, 128, 128])
        buckets, reach = rng.choice([(32, 128), (32, 128), (16, 64), (48, 200), (64, 512)])
        causal, ragged = rng.random() < 0.5, rng.random() < 0.4
        if op == "token":
            b, tk = log(1, 32), log(16, 32768)
            while b * tk * hk > (1 << 20):
                tk //= 2
            return attention(None, "token", dtype, b, rng.choice([1, 1, 1, 2, 4]), tk, hk * share, hk, d, buckets, reach, True, ragged)
        t = log(1, 4096)
        tk = t if causal or rng.random() < 0.7 else log(1, 4096)
        b = log(1, 64)
        # no more scores than the largest listed case computes; products in 32 bits cost many times those in 16
        room = 2 * 16 * 4096 * 4096 // (1 if causal else 2) // (8 if dtype == "f32" else 1)
        while b * t * tk * hk * share > room:
            if b > 1:
                b = (b + 1) // 2
            else:
                t, tk = (t + 1) // 2, (tk + 1) // 2
        return attention(None, op, dtype, b, t, tk, hk * share, hk, d, buckets, reach, causal, ragged)
    if op == "norms":
        width, rows = log(16, 8192), log(1, 16384)
        while rows * width * SIZE[dtype] > 8192 * 4096 * 2:
            rows = (rows + 1) // 2
        per = rng.choice([0, 1, 1, 7, 196])
        if per > 1:
            rows = max(per, rows // per * per)
            if rows * width * SIZE[dtype] > 8192 * 4096 * 2:
                per = 1
                rows //= 2
        return norms(None, rng.choice(["train", "train", "fwd"]), dtype, rows, width, rng.choice(["rms", "layer"]), per)
    vocab, rows, way = log(8, 150000), log(1, 8192), rng.choice(["both", "both", "split"])
    while rows * vocab * SIZE[dtype] * (2 if way == "split" else 1) > 4096 * 32000 * 2:
        rows = (rows + 1) // 2
    return distill(None, way, dtype, rows, vocab, min(vocab, rng.choice([1, 4, 20, 64, 100, 256])),
                   rng.choice([1.0, 2.0, 4.0]))


# ---------------------------------------------------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------------------------------------------------
def lengths(case):
    """Keys in use of each sequence: uneven, and with three sequences or more the last one empty."""
    b, t = case["b"], case["tk"]
    if not case["ragged"]:
        return [t] * b
    return [0 if i == b - 1 and b > 2 else t - (i * 2 * t) // (3 * b) for i in range(b)]


def bucket_map(case):
    """Bucket of each distance key - query from -reach to reach: half of a side's buckets for single distances, the other
    half for ranges whose borders grow geometrically up to reach; two sides, or for causal attention the past alone."""
    nb, reach = case["buckets"], case["reach"]
    side = nb if case["causal"] else nb // 2
    single = side // 2
    ranges = side - single

    def of(n):
        if n < single:
            return n
        # the largest m with n >= single * (reach / single) ** (m / ranges), in whole numbers
        m = sum(n ** ranges >= single ** (ranges - j) * reach ** j for j in range(1, ranges))
        return single + m

    if case["causal"]:
        return [of(max(-r, 0)) for r in range(-reach, reach + 1)]
    return [of(abs(r)) + (side if r > 0 else 0) for r in range(-reach, reach + 1)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    st = {"case": case}
    if case["op"] == "attention":
        b, tq, tk, hq, hk, d = (case[n] for n in ("b", "tq", "tk", "hq", "hk", "d"))
        st["q"], st["k"], st["v"] = normal(b, tq, hq, d), normal(b, tk, hk, d), normal(b, tk, hk, d)
        st["table"] = normal(case["buckets"], hq, scale=0.5, dtype=torch.float32)
        st["map"] = torch.tensor(bucket_map(case), dtype=torch.int32, device="cuda")
        lens = lengths(case)
        st["k_len"] = torch.tensor(lens, dtype=torch.int32, device="cuda") if case["ragged"] else None
        st["q_len"] = st["k_len"] if case["ragged"] and case["way"] != "token" and tq == tk else None
        # the tokens of a decode step are the last ones in the cache
        st["q_start"] = torch.tensor([n - tq for n in lens], dtype=torch.int32, device="cuda") if case["way"] == "token" else None
        if case["way"] == "train":
            st["dout"] = normal(b, tq, hq, d)
    elif case["op"] == "norms":
        n, w, per = case["rows"], case["width"], case["per_gate"]
        st["x"], st["y"] = normal(n, w, scale=2.0), normal(n, w, scale=0.7)
        st["gate"] = torch.sigmoid(torch.randn((n + per - 1) // per, w, device="cuda", generator=g)).to(dt) if per else None
        st["scale"] = normal(w, scale=0.1, dtype=torch.float32) + 0.5
        bias = case["kind"] == "layer"
        for at in ("post", "pre"):
            st["w_" + at] = normal(w, scale=0.2, dtype=torch.float32) + 1
            st["b_" + at] = normal(w, scale=0.1, dtype=torch.float32) if bias else None
        if case["way"] == "train":
            st["dr"], st["dh"] = normal(n, w), normal(n, w)
    else:
        n, v, top = case["rows"], case["vocab"], case["top"]
        st["logits"] = normal(n, v, scale=2.0)
        # the teacher's best classes: distinct ones, spread over the vocabulary, their logits in falling order
        first = torch.randint(0, v, (n, 1), device="cuda", generator=g)
        st["top_id"] = ((first + torch.arange(top, device="cuda") * (v // top)) % v).to(torch.int32)
        st["top_logit"] = torch.sort(torch.randn(n, top, device="cuda", generator=g) * 2 + 4, dim=1, descending=True)[0]
        st["label"] = torch.where(torch.rand(n, device="cuda", generator=g) < 0.1, -1,
                                  torch.randint(0, v, (n,), device="cuda", generator=g)).to(torch.int32)
        st["dloss"] = torch.rand(n, device="cuda", generator=g) + 0.5
    return st


# ---------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------
KD, CE = 0.7, 0.3  # weights of the teacher's term and of the labels' term
EPS = 1e-6


def run(st):
    case = st["case"]
    if own:
        return {"attention": own_attention, "norms": own_norms, "distill": own_distill}[case["op"]](st, case)
    return {"attention": plain_attention, "norms": plain_norms, "distill": plain_distill}[case["op"]](st, case)


def own_attention(st, case):
    import vit_amd
    how = dict(causal=case["causal"], q_start=st["q_start"], q_len=st["q_len"], k_len=st["k_len"])
    if case["way"] != "train":
        return {"out": vit_amd.relpos_attention_fwd(st["q"], st["k"], st["v"], st["table"], st["map"], **how)}
    out, saved = vit_amd.relpos_attention_fwd(st["q"], st["k"], st["v"], st["table"], st["map"], training=True, **how)
    dq, dk, dv, dtable = vit_amd.relpos_attention_bwd(st["dout"], st["q"], st["k"], st["v"], out, saved, st["table"], st["map"], **how)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable}


def own_norms(st, case):
    import vit_amd
    how = dict(gate=st["gate"], rows_per_gate=max(case["per_gate"], 1), res_scale=st["scale"], w_post=st["w_post"], b_post=st["b_post"],
               w_pre=st["w_pre"], b_pre=st["b_pre"], kind=case["kind"], eps=EPS)
    r, h, stats = vit_amd.block_norms_fwd(st["x"], st["y"], **how)
    if case["way"] != "train":
        return {"r": r, "h": h}
    g = vit_amd.block_norms_bwd(st["dr"], st["dh"], st["x"], st["y"], stats, **how)
    return {"r": r, "h": h, **{n: t for n, t in g.items() if t is not None}}


def own_distill(st, case):
    import vit_amd
    how = dict(labels=st["label"], tau=case["tau"], kd_weight=KD, ce_weight=CE)
    args = (st["logits"], st["top_logit"], st["top_id"])
    if case["way"] == "both":
        loss, dlogits = vit_amd.distill_fwd_bwd(*args, st["dloss"], **how)
    else:
        loss, lse = vit_amd.distill_fwd(*args, **how)
        dlogits = vit_amd.distill_bwd(*args, st["dloss"], lse, **how)
    return {"loss": loss, "dlogits": dlogits}


def plain_attention(st, case):
    b, tq, tk, hq, hk, d = (case[n] for n in ("b", "tq", "tk", "hq", "hk", "d"))
    dt, reach, share = st["q"].dtype, case["reach"], hq // hk
    q = st["q"].float().transpose(1, 2)
    k = st["k"].float().transpose(1, 2).repeat_interleave(share, 1)
    v = st["v"].float().transpose(1, 2).repeat_interleave(share, 1)
    rows, cols = torch.arange(tq, device=q.device), torch.arange(tk, device=q.device)
    start = st["q_start"].long() if st["q_start"] is not None else torch.zeros(1, dtype=torch.long, device=q.device)
    away = cols[None, None, :] - rows[None, :, None] - start[:, None, None]  # [b or 1, tq, tk]
    seen = torch.ones_like(away, dtype=torch.bool)
    if case["causal"]:
        seen = seen & (away <= 0)
    if st["k_len"] is not None:
        seen = seen & (cols < st["k_len"][:, None])[:, None, :]
    if st["q_len"] is not None:
        seen = seen & (rows < st["q_len"][:, None])[:, :, None]
    bucket = st["map"].long()[away.clamp(-reach, reach) + reach]
    bias = st["table"][bucket].permute(0, 3, 1, 2)
    scale = 1.0 / math.sqrt(d)
    s = (q @ k.transpose(-1, -2)) * scale + bias
    s = torch.where(seen[:, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    res = {"out": out.transpose(1, 2).to(dt)}
    if case["way"] != "train":
        return res
    do = st["dout"].float().transpose(1, 2)
    dv = p.transpose(-1, -2) @ do
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q) * scale
    # the scores of one distance lie on a diagonal: with the rows turned round and each shifted by one they lie in a column
    turned = torch.nn.functional.pad(ds.sum(0).flip(1), (0, tq)).reshape(hq, -1)[:, :tq * (tk + tq - 1)]
    by_distance = turned.reshape(hq, tq, tk + tq - 1).sum(1, dtype=torch.float64)
    apart = torch.arange(-(tq - 1), tk, device=q.device).clamp(-reach, reach) + reach
    which = st["map"].long()[apart][:, None] == torch.arange(case["buckets"], device=q.device)
    res |= {"dq": dq.transpose(1, 2).to(dt), "dk": dk.reshape(b, hk, share, tk, d).sum(2).transpose(1, 2).to(dt),
            "dv": dv.reshape(b, hk, share, tk, d).sum(2).transpose(1, 2).to(dt),
            "dtable": (by_distance @ which.double()).t().float()}
    return res


def plain_norm(t, w, b, kind):
    mean = t.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(t[:, :1])
    away = t - mean
    rstd = torch.rsqrt((away * away).mean(-1, keepdim=True) + EPS)
    hat = away * rstd
    return hat, rstd, hat * w + (b if b is not None else 0.0)


def plain_norm_back(g, hat, rstd, kind):
    mean = g.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return rstd * (g - mean - hat * (g * hat).mean(-1, keepdim=True))


def plain_norms(st, case):
    dt, kind, per = st["x"].dtype, case["kind"], case["per_gate"]
    n, w = case["rows"], case["width"]
    x, y = st["x"].float(), st["y"].float()
    gate = st["gate"].float().repeat_interleave(per, 0)[:n] if per else 1.0
    y_hat, y_rstd, u = plain_norm(y, st["w_post"], st["b_post"], kind)
    r = x + st["scale"] * gate * u
    r_hat, r_rstd, h = plain_norm(r, st["w_pre"], st["b_pre"], kind)
    res = {"r": r.to(dt), "h": h.to(dt)}
    if case["way"] != "train":
        return res
    dh = st["dh"].float()
    dx = st["dr"].float() + plain_norm_back(dh * st["w_pre"], r_hat, r_rstd, kind)
    du = dx * st["scale"] * gate
    dy = plain_norm_back(du * st["w_post"], y_hat, y_rstd, kind)
    res |= {"dx": dx.to(dt), "dy": dy.to(dt)}
    if per:
        res["dgate"] = (dx * st["scale"] * u).reshape(n // per, per, w).sum(1).to(dt)
    res |= {"dres_scale": (dx * gate * u).sum(0), "dw_post": (du * y_hat).sum(0)}
    if kind == "layer":
        res["db_post"] = du.sum(0)
    res["dw_pre"] = (dh * r_hat).sum(0)
    if kind == "layer":
        res["db_pre"] = dh.sum(0)
    return res


def plain_distill(st, case):
    tau = case["tau"]
    z, ids = st["logits"].float(), st["top_id"].long()
    has = st["label"] >= 0
    label = st["label"].long().clamp(min=0)[:, None]

    def log_softmax(t):
        away = t - t.amax(-1, keepdim=True)
        return away - torch.log(torch.exp(away).sum(-1, keepdim=True))

    log_p, log_q, log_c = log_softmax(st["top_logit"] / tau), log_softmax(z / tau), log_softmax(z)
    p = torch.exp(log_p)
    kd = (p * (log_p - log_q.gather(1, ids))).sum(-1)
    ce = torch.where(has, -log_c.gather(1, label)[:, 0], 0.0)
    loss = KD * tau * tau * kd + CE * ce
    dz = KD * tau * torch.exp(log_q).scatter_add(1, ids, -p)
    dz = dz + CE * has[:, None] * torch.exp(log_c).scatter_add(1, label, torch.full_like(label, -1, dtype=torch.float32))
    return {"loss": loss, "dlogits": (st["dloss"][:, None] * dz).to(st["logits"].dtype)}


# ---------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "attention":
        b, tq, tk, hq, hk, d = (case[n] for n in ("b", "tq", "tk", "hq", "hk", "d"))
        lens = lengths(case)
        padded = case["ragged"] and case["way"] != "token" and tq == tk
        pairs = 0
        for n in lens:
            r = n if padded else tq
            start = n - tq if case["way"] == "token" else 0
            # query i sees keys 0 .. start + i of n where it is causal, all n otherwise
            pairs += sum(max(0, min(n, start + i + 1)) for i in range(r)) if case["causal"] else r * n
        q, kv = b * tq * hq * d * e, sum(lens) * hk * d * e
        bytes_, flops = 2 * q + 2 * kv, 4.0 * pairs * hq * d
        if case["way"] == "train":
            # the gradient's pass: queries, keys, values, output and its gradient in, three gradients out; five products
            bytes_, flops = bytes_ + 4 * q + 4 * kv, flops + 10.0 * pairs * hq * d
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "norms":
        n, w, per = case["rows"], case["width"], case["per_gate"]
        gate = (n + per - 1) // per * w * e if per else 0
        bytes_, flops = 4 * n * w * e + gate + 12 * w, 14.0 * n * w
        if case["way"] == "train":
            bytes_, flops = bytes_ + 6 * n * w * e + 2 * gate + 24 * w, flops + 40.0 * n * w
        return {"bytes": bytes_, "flops": flops}
    n, v, top = case["rows"], case["vocab"], case["top"]
    reads = 2 if case["way"] == "split" else 1
    return {"bytes": (reads + 1) * n * v * e + 8 * n * top * reads, "flops": 12.0 * n * v}


# ---------------------------------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": exact_attention, "norms": exact_norms, "distill": exact_distill}[case["op"]](st, case)


def exact_attention(st, case):
    b, tq, tk, hq, hk, d = (case[n] for n in ("b", "tq", "tk", "hq", "hk", "d"))
    if b * hq > 600:
        return None
    lens, train, reach = lengths(case), case["way"] == "train", case["reach"]
    f64 = dict(dtype=torch.float64, device="cuda")
    out, dq = torch.zeros(b, tq, hq, d, **f64), torch.zeros(b, tq, hq, d, **f64)
    dk, dv = torch.zeros(b, tk, hk, d, **f64), torch.zeros(b, tk, hk, d, **f64)
    dtable = torch.zeros(case["buckets"], hq, **f64)
    of = torch.tensor(bucket_map(case), device="cuda")
    padded = case["ragged"] and case["way"] != "token" and tq == tk
    for i in range(b):
        n = lens[i]
        m = n if padded else tq
        if n == 0 or m == 0:
            continue
        place = torch.arange(m, device="cuda") + (n - tq if case["way"] == "token" else 0)
        away = torch.arange(n, device="cuda")[None] - place[:, None]
        bucket = of[away.clamp(-reach, reach) + reach]
        hidden = (away > 0) if case["causal"] else None
        for h in range(hq):
            q, k, v = st["q"][i, :m, h].double(), st["k"][i, :n, h * hk // hq].double(), st["v"][i, :n, h * hk // hq].double()
            s = (q @ k.t()) / d ** 0.5 + st["table"][:, h].double()[bucket]
            if hidden is not None:
                s = s.masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1) if s.isfinite().any(-1).all() else torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            out[i, :m, h] = p @ v
            if train:
                do = st["dout"][i, :m, h].double()
                dp = do @ v.t()
                ds = p * (dp - (do * out[i, :m, h]).sum(-1, keepdim=True))
                dq[i, :m, h] = ds @ k / d ** 0.5
                dk[i, :n, h * hk // hq] += ds.t() @ q / d ** 0.5
                dv[i, :n, h * hk // hq] += p.t() @ do
                dtable[:, h] += torch.bincount(bucket.reshape(-1), ds.reshape(-1), minlength=case["buckets"])
    res = {"out": out}
    return {**res, "dq": dq, "dk": dk, "dv": dv, "dtable": dtable} if train else res


def exact_norms(st, case):
    layer, per, train = case["kind"] == "layer", case["per_gate"], case["way"] == "train"
    leaves = {n: st[n].double().requires_grad_(train) for n in ("x", "y", "gate", "scale", "w_post", "b_post", "w_pre", "b_pre")
              if st[n] is not None}

    def norm(t, at):
        t = t - t.mean(1, keepdim=True) if layer else t
        t = t / (t.square().mean(1, keepdim=True) + EPS).sqrt() * leaves["w_" + at]
        return t + leaves["b_" + at] if layer else t

    u = norm(leaves["y"], "post") * leaves["scale"]
    if per:
        u = (u.unflatten(0, (-1, per)) * leaves["gate"][:, None]).flatten(0, 1)
    r = leaves["x"] + u
    h = norm(r, "pre")
    res = {"r": r.detach(), "h": h.detach()}
    if train:
        torch.autograd.backward([r, h], [st["dr"].double(), st["dh"].double()])
        names = {"x": "dx", "y": "dy", "gate": "dgate", "scale": "dres_scale", "w_post": "dw_post", "b_post": "db_post",
                 "w_pre": "dw_pre", "b_pre": "db_pre"}
        res |= {names[n]: t.grad for n, t in leaves.items()}
    return res


def exact_distill(st, case):
    tau = case["tau"]
    z = st["logits"].double().requires_grad_()
    teacher = torch.softmax(st["top_logit"].double() / tau, 1)
    student = z / tau
    kd = (teacher * (teacher.log() - (student.gather(1, st["top_id"].long()) - student.logsumexp(1, keepdim=True)))).sum(1)
    picked = z.gather(1, st["label"].long().clamp(min=0)[:, None])[:, 0]
    ce = (z.logsumexp(1) - picked) * (st["label"] >= 0)
    loss = KD * tau ** 2 * kd + CE * ce
    (loss * st["dloss"].double()).sum().backward()
    return {"loss": loss.detach(), "dlogits": z.grad}
