"""The typed operators together, as a training step uses them: a transformer block with biased attention, the norms around it
with gate and residual scale, a classifier and the loss of a teacher's best classes; every gradient against automatic
differentiation of the same network in 64 bits.  fp32, so the tolerance is that of the hot path: 1e-4 of the largest value."""
import math

import pytest

torch = pytest.importorskip("torch")

TOL = 1e-4


def rel(got, want):
    return float((got.double().cpu() - want).abs().max() / want.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_a_block_taught_by_another_model(causal):
    import vit_amd
    B, T, D, H, HK, K, top = 6, 49, 64, 4, 2, 10, 3
    hd = D // H
    g = torch.Generator().manual_seed(0)

    def t(*s, scale=1.0, at=0.0):
        return (torch.randn(*s, generator=g) * scale + at).cuda()

    P = dict(x=t(B * T, D), wq=t(D, D, scale=0.2), wk=t(D, HK * hd, scale=0.2), wv=t(D, HK * hd, scale=0.2), wo=t(D, D, scale=0.2), wc=t(D, K, scale=0.3),
             table=t(16, H, scale=0.5), gate=t(B, D, scale=0.3, at=0.6), res=t(D, scale=0.1, at=0.5), w0=t(D, scale=0.1, at=1), b0=t(D, scale=0.1),
             w1=t(D, scale=0.1, at=1), b1=t(D, scale=0.1), w2=t(D, scale=0.1, at=1), b2=t(D, scale=0.1))
    lens = torch.tensor([49, 1, 20, 49, 33, 7], dtype=torch.int32).cuda()
    buckets = vit_amd.relpos_buckets(16, 40, not causal, "cuda")
    ids = torch.stack([torch.randperm(K, generator=g)[:top] for _ in range(B * T)]).to(torch.int32).cuda()
    best = (torch.randn(B * T, top, generator=g) * 2).cuda()
    labels = torch.randint(0, K, (B * T,), generator=g).to(torch.int32).cuda()
    inside = (torch.arange(T).cuda()[None] < lens[:, None]).reshape(-1)
    labels[~inside] = -1
    ids[~inside] = -1
    dloss = inside.float() / float(inside.sum())
    how = dict(labels=labels, tau=2.0, kd_weight=0.6, ce_weight=0.4)
    attn = dict(causal=causal, q_len=lens, k_len=lens)

    # forward: norm into the block, attention, norms out of it, classifier, loss and its gradient
    zero = torch.zeros_like(P["x"])
    _, h, s0 = vit_amd.block_norms_fwd(P["x"], zero, w_pre=P["w0"], b_pre=P["b0"], kind="layer")
    q, k, v = (h @ P["wq"]).view(B, T, H, hd), (h @ P["wk"]).view(B, T, HK, hd), (h @ P["wv"]).view(B, T, HK, hd)
    o, saved = vit_amd.relpos_attention_fwd(q, k, v, P["table"], buckets, training=True, **attn)
    y = o.reshape(B * T, D) @ P["wo"]
    n1 = dict(gate=P["gate"], rows_per_gate=T, res_scale=P["res"], w_post=P["w1"], b_post=P["b1"], w_pre=P["w2"], b_pre=P["b2"], kind="layer")
    r, h2, s1 = vit_amd.block_norms_fwd(P["x"], y, **n1)
    loss, dz = vit_amd.distill_fwd_bwd(h2 @ P["wc"], best, ids, dloss, **how)

    # backward
    G = {"wc": h2.t() @ dz}
    gn = vit_amd.block_norms_bwd(None, dz @ P["wc"].t(), P["x"], y, s1, **n1)
    G["wo"] = o.reshape(B * T, D).t() @ gn["dy"]
    dq, dk, dv, G["table"] = vit_amd.relpos_attention_bwd((gn["dy"] @ P["wo"].t()).view(B, T, H, hd), q, k, v, o, saved, P["table"], buckets, **attn)
    dh = torch.zeros_like(h)
    for n, d in (("wq", dq), ("wk", dk), ("wv", dv)):
        d = d.reshape(B * T, -1)
        G[n] = h.t() @ d
        dh += d @ P[n].t()
    g0 = vit_amd.block_norms_bwd(gn["dx"], dh, P["x"], zero, s0, w_pre=P["w0"], b_pre=P["b0"], kind="layer")
    G.update(x=g0["dx"], w0=g0["dw_pre"], b0=g0["db_pre"], gate=gn["dgate"], res=gn["dres_scale"], w1=gn["dw_post"], b1=gn["db_post"], w2=gn["dw_pre"],
             b2=gn["db_pre"])

    # the same network in 64 bits
    W = {n: p.double().cpu().requires_grad_() for n, p in P.items()}
    nrm = lambda a, w, b: torch.nn.functional.layer_norm(a, (D,), w, b, 1e-6)  # noqa: E731
    hh = nrm(W["x"], W["w0"], W["b0"])
    qq, kk, vv = ((hh @ W[n]).view(B, T, -1, hd).transpose(1, 2) for n in ("wq", "wk", "wv"))
    away = torch.arange(T)[None] - torch.arange(T)[:, None]
    bias = W["table"][buckets.long().cpu()[away.clamp(-40, 40) + 40]].permute(2, 0, 1)
    sc = qq @ kk.repeat_interleave(H // HK, 1).transpose(-1, -2) / math.sqrt(hd) + bias
    keep = (torch.arange(T) < lens.cpu()[:, None])[:, None, None, :] & ((away <= 0) if causal else True)
    oo = torch.softmax(sc.masked_fill(~keep, -math.inf), -1) @ vv.repeat_interleave(H // HK, 1)
    oo = (oo * (torch.arange(T) < lens.cpu()[:, None])[:, None, :, None]).transpose(1, 2).reshape(B * T, D)
    u = nrm(oo @ W["wo"], W["w1"], W["b1"]) * W["res"] * W["gate"].repeat_interleave(T, 0)
    zz = nrm(W["x"] + u, W["w2"], W["b2"]) @ W["wc"]
    rows = inside.cpu()
    p = torch.softmax(best.double().cpu()[rows] / 2, 1)
    lq = torch.log_softmax(zz[rows] / 2, 1).gather(1, ids.long().cpu()[rows])
    want = 0.6 * 4 * (p * (p.log() - lq)).sum(1) + 0.4 * torch.nn.functional.cross_entropy(zz[rows], labels.long().cpu()[rows], reduction="none")
    want.mean().backward()
    assert rel(loss[inside], want.detach()) < TOL and not loss[~inside].any()
    for n, p in W.items():
        assert rel(G[n], p.grad) < TOL, (n, rel(G[n], p.grad))
