"""Plain 64-bit forms of the typed operators on the CPU, with bounds of what their kernels may be off by (tests only)."""
import math

import torch

U32 = 2.0 ** -24  # half a step of fp32
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, table, buckets, scale=None, causal=False, q_start=None, q_len=None, k_len=None, dout=None):
    """(results, bounds) of relpos_attention in 64 bits; the inputs are the kernel's own (already rounded)."""
    dt = q.dtype
    u = 0.0 if dt == torch.float32 else half_step(dt)  # the rounding of p and ds
    r = half_step(dt)                                  # the rounding of a result
    b, tq, hq, d = q.shape
    tk, hk = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    reach = buckets.numel() // 2
    tab = table.double().cpu()
    mp = buckets.long().cpu()
    res = {"out": torch.zeros(b, tq, hq, d).double()}
    tol = {"out": torch.zeros(b, tq, hq, d).double()}
    if dout is not None:
        for n, t in (("dq", q), ("dk", k), ("dv", v), ("dtable", table)):
            res[n], tol[n] = torch.zeros(t.shape).double(), torch.zeros(t.shape).double()
    for i in range(b):
        n = tk if k_len is None else min(max(int(k_len[i]), 0), tk)
        m = tq if q_len is None else min(max(int(q_len[i]), 0), tq)
        st = 0 if q_start is None else int(q_start[i])
        if n == 0 or m == 0:
            continue
        away = torch.arange(n)[None] - torch.arange(m)[:, None] - st
        bk = mp[away.clamp(-reach, reach) + reach]
        has = (bk >= 0) & (bk < tab.shape[0])
        seen = (away <= 0) if causal else torch.ones_like(away, dtype=torch.bool)
        for h in range(hq):
            g = h * hk // hq
            Q, K, V = q[i, :m, h].double().cpu(), k[i, :n, g].double().cpu(), v[i, :n, g].double().cpu()
            bias = torch.where(has, tab[bk.clamp(0, tab.shape[0] - 1), h], 0.0)
            s = torch.where(seen, scale * Q @ K.t() + bias, -math.inf)
            top = s.amax(1, keepdim=True)
            e = torch.where(seen, torch.exp(s - torch.where(top.isinf(), 0.0, top)), 0.0)
            tot = e.sum(1, keepdim=True)
            p = e / torch.where(tot == 0, 1.0, tot)
            # relative error of p in fp32: the score's products and its base-2 form, the maximum's subtraction, the sum
            A = float((abs(scale) * Q.abs() @ K.abs().t()).max())
            big = float(s[seen].abs().max()) if bool((seen & s.isfinite()).any()) else 0.0
            big = big if math.isfinite(big) and big < 1e30 else float(bias[bias.isfinite() & (bias.abs() < 1e30)].abs().max()) if bool((bias.isfinite() & (bias.abs() < 1e30)).any()) else 0.0
            rho = U32 * (d * A + 8 * (big + 1) + n + 32)
            pv = p @ V.abs()
            res["out"][i, :m, h] = p @ V
            tol["out"][i, :m, h] = r * (p @ V).abs() + (u + 2 * rho) * pv
            if dout is None:
                continue
            dO = dout[i, :m, h].double().cpu()
            dp, dpa = dO @ V.t(), dO.abs() @ V.abs().t()
            D = (dO * (p @ V)).sum(1, keepdim=True)
            Da = (dO.abs() * pv).sum(1, keepdim=True)
            ds = p * (dp - D)
            # fp32 error of ds: p's, the product's d terms; the row sum D carries p's error, and 16-bit forward passes give it to
            # twice the mantissa (two roundings of p and of out)
            dsa = p * ((2 * rho + d * U32) * (dpa + Da) + 4 * rho * Da)
            dsq = dsa + p * (4 * u * u * Da)
            res["dq"][i, :m, h] = scale * ds @ K
            tol["dq"][i, :m, h] = abs(scale) * ((u + n * U32) * ds.abs() + dsq) @ K.abs()
            res["dk"][i, :n, g] += scale * ds.t() @ Q
            tol["dk"][i, :n, g] += abs(scale) * ((u + (m * hq // hk) * U32) * ds.abs() + dsa).t() @ Q.abs()
            res["dv"][i, :n, g] += p.t() @ dO
            tol["dv"][i, :n, g] += ((u + 2 * rho + (m * hq // hk) * U32) * p).t() @ dO.abs()
            one = torch.nn.functional.one_hot(torch.where(has, bk, tab.shape[0]).reshape(-1), tab.shape[0] + 1).double()[:, :-1]
            res["dtable"][:, h] += one.t() @ ds.reshape(-1)
            tol["dtable"][:, h] += one.t() @ (dsa + (128 + m) * U32 * ds.abs()).reshape(-1)
    if dout is not None:
        for name in ("dq", "dk", "dv"):
            tol[name] += r * res[name].abs()
        tol["dtable"] += U32 * res["dtable"].abs()
    return res, {n: t + 1e-30 + (2.0 ** -24 if dt == torch.float16 and n != "dtable" else 0.0) for n, t in tol.items()}


def norms(x, y, gate, per, scale, w_post, b_post, w_pre, b_pre, kind, eps, dr=None, dh=None):
    """block_norms in 64 bits by automatic differentiation: (r, h, {gradients})."""
    names = dict(x=x, y=y, gate=gate, res_scale=scale, w_post=w_post, b_post=b_post, w_pre=w_pre, b_pre=b_pre)
    leaf = {n: t.double().cpu().clone().requires_grad_() for n, t in names.items() if t is not None}

    def norm(t, at):
        if kind == "layer":
            t = t - t.mean(1, keepdim=True)
        t = t / torch.sqrt((t * t).mean(1, keepdim=True) + eps) * leaf["w_" + at]
        return t + leaf["b_" + at] if "b_" + at in leaf else t

    u = norm(leaf["y"], "post") if w_post is not None else leaf["y"]
    if scale is not None:
        u = u * leaf["res_scale"]
    if gate is not None:
        u = u * leaf["gate"].repeat_interleave(per, 0)[:x.shape[0]]
    r = leaf["x"] + u
    h = norm(r, "pre") if w_pre is not None else None
    if dr is None and dh is None:
        return r.detach(), None if h is None else h.detach(), None
    outs, grads = [], []
    for t, g in ((r, dr), (h, dh)):
        if g is not None:
            outs.append(t)
            grads.append(g.double().cpu())
    torch.autograd.backward(outs, grads)
    key = {"x": "dx", "y": "dy", "gate": "dgate", "res_scale": "dres_scale", "w_post": "dw_post", "b_post": "db_post", "w_pre": "dw_pre",
           "b_pre": "db_pre"}
    return r.detach(), None if h is None else h.detach(), {key[n]: t.grad for n, t in leaf.items()}


def distill(z, top, ids, dloss, labels, tau, kd, ce):
    """(loss, dz) in 64 bits, row by row from the formulas."""
    z, top = z.double().cpu(), top.double().cpu()
    ids = ids.long().cpu()
    n, v = z.shape
    loss, dz = torch.zeros(n).double(), torch.zeros(n, v).double()
    for i in range(n):
        ok = (ids[i] >= 0) & (ids[i] < v)
        t, k = top[i][ok] / tau, ids[i][ok]
        log_q = torch.log_softmax(z[i] / tau, 0)
        if t.numel() and bool((t > -math.inf).any()):
            p = torch.softmax(t, 0)
            live = p > 0
            loss[i] = kd * tau * tau * (p[live] * (torch.log_softmax(t, 0)[live] - log_q[k][live])).sum()
            g = torch.exp(log_q)
            for j in range(len(k)):
                g[k[j]] -= p[j]
            dz[i] = kd * tau * g
        lab = -1 if labels is None else int(labels[i])
        if 0 <= lab < v and ce != 0:
            log_c = torch.log_softmax(z[i], 0)
            loss[i] -= ce * log_c[lab]
            g = torch.exp(log_c)
            g[lab] -= 1
            dz[i] += ce * g
        dz[i] *= float(dloss[i])
    return loss, dz
