"""What relpos_attention gives without the rounding of probabilities to 16 bits: its output always, its gradients where queries
are at most 32.  The bound counts the fp32 sums, the result's one rounding and what two parts of a value leave of it: half a
step of the second part, (half a step)^2 of the value, and for fp16 2^-25 beside that, where the second part is subnormal."""
import math

import pytest

torch = pytest.importorskip("torch")
from op_refs import DTYPES, U32, attention, half_step  # noqa: E402

gpu = pytest.mark.gpu


def make(dtype, b, tq, tk, hq, hk, d, nb=16, reach=24, causal=False, seed=0):
    import vit_amd
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(*s, generator=g).to(DTYPES[dtype]).cuda() for s in ((b, tq, hq, d), (b, tk, hk, d), (b, tk, hk, d), (b, tq, hq, d)))
    return q, k, v, do, (torch.randn(nb, hq, generator=g) * 0.7).cuda(), vit_amd.relpos_buckets(nb, reach, not causal, "cuda")


def exact(q, k, v, do, table, buckets, causal, start):
    """{name: (value, bound)} in 64 bits on the GPU; query i is at place start + i."""
    b, tq, hq, d = q.shape
    tk, share, reach = k.shape[1], hq // k.shape[2], buckets.numel() // 2
    dt = q.dtype
    r, u = half_step(dt), 0.0 if dt == torch.float32 else half_step(dt)
    least = 2.0 ** -25 if dt == torch.float16 else 0.0
    Q, O = q.double().transpose(1, 2), do.double().transpose(1, 2)
    K, V = (t.double().transpose(1, 2).repeat_interleave(share, 1) for t in (k, v))
    away = torch.arange(tk, device=q.device)[None] - torch.arange(tq, device=q.device)[:, None] - start
    bias = table.double()[buckets.long()[away.clamp(-reach, reach) + reach]].permute(2, 0, 1)
    scale = d ** -0.5

    def back(t):
        return t.contiguous().transpose(-1, -2).contiguous()

    s = scale * (Q @ back(K)) + bias
    big = float(s.abs().max())
    A = float((scale * Q.abs() @ back(K.abs())).max())
    if causal:
        s = s.masked_fill(away > 0, -math.inf)
    p = torch.softmax(s, -1)
    rho = U32 * (d * A + 8 * (big + 1) + tk + 32)
    pv, out = p @ V.abs(), p @ V
    dp, dpa = O @ back(V), O.abs() @ back(V.abs())
    D, Da = (O * out).sum(-1, keepdim=True), (O.abs() * pv).sum(-1, keepdim=True)
    ds = p * (dp - D)
    dsa = p * ((2 * rho + d * U32) * (dpa + Da) + 4 * rho * Da)
    seen = (p > 0).double()
    rows = tq * share
    res = {"out": (out, r * out.abs() + p @ V.abs() * (u * u + 2 * rho) + least * seen @ V.abs()),
           "dq": (scale * ds @ K, scale * ((u * u + tk * U32) * ds.abs() + dsa + p * 4 * u * u * Da + least * seen) @ K.abs()),
           "dk": (scale * back(ds) @ Q, scale * back((u * u + rows * U32) * ds.abs() + dsa + least * seen) @ Q.abs()),
           "dv": (back(p) @ O, back((u * u + 2 * rho + rows * U32) * p + least * seen) @ O.abs())}
    for n in ("dk", "dv"):
        res[n] = tuple(t.reshape(b, hq // share, share, tk, d).sum(2) for t in res[n])
    # the least step of an fp16 result
    return {n: (w.transpose(1, 2), (t + (r * w.abs() if n != "out" else 0) + least).transpose(1, 2)) for n, (w, t) in res.items()}


def check(got, want, what):
    off = (got.double() - want[0]).abs() / (want[1] + 1e-30)
    assert float(off.max()) <= 1, (what, float(off.max()), int((off > 1).sum()))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(2, 200, 200, 4, 2, 64), (1, 140, 300, 2, 2, 128), (1, 333, 333, 3, 1, 80), (2, 70, 190, 4, 4, 24), (1, 300, 260, 384, 128, 32)])
@pytest.mark.parametrize("causal", [False, True])
def test_training_and_inference_give_one_output(dtype, shape, causal):
    import vit_amd
    q, k, v, do, table, buckets = make(dtype, *shape, causal=causal, seed=sum(shape))
    out = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, causal=causal)
    again, _ = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, causal=causal, training=True)
    assert torch.equal(out, again)
    check(out, exact(q, k, v, do, table, buckets, causal, 0)["out"], "out")


# on both sides of the sizes at which workgroups of whole rows fill the chip: by heads, by key tiles, by heads that share keys
FEW = [
    # b, tq, tk, hq, hk, d
    (2, 16, 16, 2, 2, 16), (3, 31, 200, 4, 2, 64), (1, 1, 700, 2, 1, 128), (64, 16, 24, 16, 8, 32), (40, 32, 32, 32, 32, 64), (1, 5, 300, 1024, 512, 128),
    (2, 1, 4096, 16, 16, 64), (2, 32, 2100, 32, 32, 96),
]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", FEW)
@pytest.mark.parametrize("causal", [False, True])
def test_few_queries_have_gradients_without_the_rounding_of_probabilities(dtype, shape, causal):
    import vit_amd
    b, tq, tk = shape[:3]
    q, k, v, do, table, buckets = make(dtype, *shape, causal=causal, seed=sum(shape))
    start = (tk - tq) // 2 if causal else 0
    how = dict(causal=causal, q_start=torch.full((b,), start, dtype=torch.int32, device="cuda"))
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True, **how)
    want = exact(q, k, v, do, table, buckets, causal, start)
    check(out, want["out"], "out")
    for n, t in zip(("dq", "dk", "dv"), vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, table, buckets, **how)):
        check(t, want[n], n)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(2, 200, 200, 4, 2, 64), (1, 140, 300, 2, 2, 128), (2, 70, 190, 4, 4, 24), (1, 300, 260, 384, 128, 80), (1, 16, 90, 2, 2, 32)])
@pytest.mark.parametrize("causal", [False, True])
def test_precise_gradients_of_many_queries(dtype, shape, causal):
    import vit_amd
    q, k, v, do, table, buckets = make(dtype, *shape, causal=causal, seed=sum(shape))
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, causal=causal, training=True)
    args = (do, q, k, v, out, saved, table, buckets)
    got = vit_amd.relpos_attention_bwd(*args, causal=causal, precise=True)
    want = exact(q, k, v, do, table, buckets, causal, 0)
    for n, t in zip(("dq", "dk", "dv"), got):
        check(t, want[n], n)
    plain = vit_amd.relpos_attention_bwd(*args, causal=causal)
    if dtype == "f32" or shape[1] <= 32:
        assert all(torch.equal(a, b) for a, b in zip(got, plain))
    assert all(torch.equal(a, b) for a, b in zip(got, vit_amd.relpos_attention_bwd(*args, causal=causal, precise=True)))


@gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("reach", [0, 2048])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_few_queries_with_the_smallest_and_the_largest_maps(dtype, reach, d):
    import vit_amd
    q, k, v, do, table, _ = make(dtype, 2, 32, 500, 2, 1, d, nb=8, seed=d)
    buckets = torch.arange(2 * reach + 1, device="cuda", dtype=torch.int32) % 8
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True)
    want = exact(q, k, v, do, table, buckets, False, 0)
    for n, t in zip(("dq", "dk", "dv"), vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, table, buckets)):
        check(t, want[n], n)


@gpu
@pytest.mark.parametrize("shape", [(2, 300, 300, 4, 2, 64), (1, 260, 400, 2, 1, 128), (1, 300, 260, 768, 768, 32), (1, 20, 400, 2, 2, 40)])
@pytest.mark.parametrize("power", [-16, 0, 7])
@pytest.mark.parametrize("causal", [False, True])
def test_fp16_gradients_below_and_at_the_ends_of_its_range(shape, power, causal):
    """Probabilities of 1 / 300 times output gradients of 2^-16 lie below fp16's least step, their sums over 300 rows do not; with
    2^7 the largest ds would pass its end if they were scaled by one factor."""
    import vit_amd
    q, k, v, do, table, buckets = make("f16", *shape, causal=causal, seed=sum(shape))
    do = do * 2.0 ** power
    if power > 0:  # rows of one key's weight beside even ones
        q[:, ::7] *= 8
    few = slice(0, 2) if shape[3] > 4 else slice(None)  # the 64-bit form of two heads of many
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, causal=causal, training=True)
    got = (out, *vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, table, buckets, causal=causal))
    want, bound = attention(q[:, :, few], k[:, :, few], v[:, :, few], table[:, few], buckets, causal=causal, dout=do[:, :, few])
    for n, t in zip(("out", "dq", "dk", "dv", "dtable"), got):
        t = (t[:, few] if n == "dtable" else t[:, :, few]).double().cpu()
        off = (t - want[n]).abs() / bound[n]
        assert float(off.max()) <= 1, (n, float(off.max()), int((off > 1).sum()))


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tq", [1, 40])
def test_many_keys_of_little_weight_beside_one_of_much(dtype, tq):
    """e^-17.5 each (2^-25, half of fp16's least step), 2^18 of them: 0.0066 of the weight.  The exponentials' arguments of 25
    cost 25 * 2^-24, and the result its own rounding.  Sums: terms of one size round all the same way, so their errors add.  With
    40 queries one wave adds the products of all keys one instruction after the other: 2 keys an instruction in fp32, 2^17
    roundings of 2^-24 of the sum so far, whose mean is half the last one's; 16 keys and two parts in 16 bits, 2^15.  The
    weights' sum adds 2^12 tiles to a sum near 1, whose rounding is 2^-24 each and no more."""
    import vit_amd
    n = 1 << 18
    q, k, v = (torch.zeros(1, s, 1, 32, dtype=DTYPES[dtype], device="cuda") for s in (tq, n, n))
    q[..., 0], k[0, 100, 0, 0] = 5.0, 3.5
    v += 1
    v[0, 100] = 0
    out = vit_amd.relpos_attention_fwd(q, k, v, torch.zeros(4, 1, device="cuda"), vit_amd.relpos_buckets(4, 8, True, "cuda"), scale=1.0)
    w = (n - 1) * math.exp(-17.5)
    adds = (2 ** 17 if dtype == "f32" else 2 ** 15) / 2 + 2 ** 12
    assert float((out.double() / (w / (1 + w)) - 1).abs().max()) < half_step(DTYPES[dtype]) + 2.0 ** -24 * (adds + 64) + 2.0 ** -16
