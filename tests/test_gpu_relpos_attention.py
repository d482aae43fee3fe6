"""vt_relpos_attention_fwd / _bwd through vit_amd against a plain 64-bit form: types, head layouts, lengths, masks, strides,
padding, streams, graphs; every element within a bound that counts the kernels' roundings (tests/op_refs.py)."""
import itertools

import pytest

torch = pytest.importorskip("torch")
from op_refs import DTYPES, attention  # noqa: E402

gpu = pytest.mark.gpu


def make(dtype, b, tq, tk, hq, hk, d, nb=32, reach=128, bidirectional=True, seed=0, spread=1.0):
    import vit_amd
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    q, k, v, do = ((torch.randn(*s, generator=g) * spread).to(dt).cuda() for s in
                   ((b, tq, hq, d), (b, tk, hk, d), (b, tk, hk, d), (b, tq, hq, d)))
    table = (torch.randn(nb, hq, generator=g) * 0.7).cuda()
    return q, k, v, do, table, vit_amd.relpos_buckets(nb, reach, bidirectional, "cuda")


def ints(*a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def check(got, want, bound, what):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= bound)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / bound)[bad].max()), bad.nonzero()[:4].tolist())


def run(q, k, v, do, table, buckets, **how):
    import vit_amd
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True, **how)
    plain = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, **how)
    grads = vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, table, buckets, **how)
    want, bound = attention(q, k, v, table, buckets, dout=do, **how)
    check(plain, want["out"], bound["out"], "out")
    check(out, want["out"], bound["out"], "out, training")
    for n, t in zip(("dq", "dk", "dv", "dtable"), grads):
        check(t, want[n], bound[n], n)
    return out, grads


SHAPES = [
    # b, tq, tk, hq, hk, d
    (1, 1, 1, 1, 1, 1), (2, 16, 16, 2, 2, 16), (1, 33, 33, 2, 1, 32), (2, 1, 70, 4, 2, 64), (1, 65, 129, 3, 3, 40),
    (1, 130, 63, 2, 2, 128), (1, 200, 200, 4, 1, 80), (3, 31, 257, 2, 1, 24), (1, 257, 300, 1, 1, 33), (1, 4, 515, 8, 1, 128),
]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [False, True])
def test_against_the_formula(dtype, shape, causal):
    q, k, v, do, table, buckets = make(dtype, *shape, bidirectional=not causal, reach=24 if shape[1] % 2 else 128, nb=16, seed=sum(shape))
    how = dict(causal=causal)
    if causal and shape[1] != shape[2]:
        how["q_start"] = torch.full((shape[0],), shape[2] - shape[1], dtype=torch.int32, device="cuda")
    run(q, k, v, do, table, buckets, **how)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tq,tk,d", [(150, 150, 64), (20, 90, 32), (5, 700, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batches_read_nothing_behind_their_lengths(dtype, tq, tk, d, causal):
    q, k, v, do, table, buckets = make(dtype, 5, tq, tk, 4, 2, d, seed=3)
    q_len, k_len = ints(tq, 0, 3, tq - 1, 1), ints(tk, 7, 0, tk // 2 + 1, -5)
    ql, kl = [tq, 0, 3, tq - 1, 1], [tk, 7, 0, tk // 2 + 1, 0]
    for b in range(5):
        q[b, ql[b]:], do[b, ql[b]:] = float("nan"), float("inf")
        k[b, kl[b]:], v[b, kl[b]:] = float("nan"), float("-inf")
    out, (dq, dk, dv, dtable) = run(q, k, v, do, table, buckets, causal=causal, q_len=q_len, k_len=k_len)
    for b in range(5):
        assert not out[b, ql[b]:].any() and not dq[b, ql[b]:].any() and not dk[b, kl[b]:].any() and not dv[b, kl[b]:].any()
    assert not out[2].any() and not out[4].any()  # no keys: empty rows


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_queries_placed_behind_before_and_beyond_the_keys(dtype):
    q, k, v, do, table, buckets = make(dtype, 6, 40, 90, 2, 2, 32, nb=16, reach=20, seed=5)
    for causal in (False, True):
        run(q, k, v, do, table, buckets, causal=causal, q_start=ints(0, 50, -10, -40, 1000, -2**31 + 1), k_len=ints(90, 90, 90, 90, 80, 90))
    few = [t[:, :3].contiguous() for t in (q, do)]
    for causal in (False, True):
        run(few[0], k, v, few[1], table, buckets, causal=causal, q_start=ints(0, 87, -1, -3, 2**31 - 1, 40), k_len=ints(90, 90, 90, 90, 5, 43))


@gpu
@pytest.mark.parametrize("tq", [1, 2, 3])
def test_a_token_behind_a_cache_is_the_row_of_the_whole_prompt(tq):
    import vit_amd
    q, k, v, do, table, buckets = make("bf16", 2, 300, 300, 8, 2, 64, bidirectional=False, seed=8)
    whole = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, causal=True)
    cache_k, cache_v = torch.full((2, 512, 2, 64), float("nan"), dtype=q.dtype, device="cuda"), torch.full((2, 512, 2, 64), float("nan"), dtype=q.dtype, device="cuda")
    for n in (tq, 64, 200, 300):
        cache_k[:, :n], cache_v[:, :n] = k[:, :n], v[:, :n]
        part = vit_amd.relpos_attention_fwd(q[:, n - tq:n], cache_k, cache_v, table, buckets, causal=True, q_start=ints(n - tq, n - tq),
                                            k_len=ints(n, n))
        # each is within one rounding of p (2^-9 of |p||v|) and of the result of the same value
        want, bound = attention(q[:, n - tq:n], k[:, :n], v[:, :n], table, buckets, causal=True, q_start=ints(n - tq, n - tq))
        check(part, want["out"], bound["out"], n)
        check(whole[:, n - tq:n], want["out"], bound["out"], n)


@gpu
def test_strides_of_packed_and_transposed_projections():
    import vit_amd
    g = torch.Generator().manual_seed(1)
    b, t, h, d = 2, 77, 4, 40
    qkv = torch.randn(b, t, 3, h, d, generator=g).to(torch.bfloat16).cuda()
    table, buckets = torch.randn(32, h, generator=g).cuda(), vit_amd.relpos_buckets(device="cuda")
    views = [qkv[:, :, i] for i in range(3)]
    turned = [torch.randn(b, h, t, d, generator=g).to(torch.bfloat16).cuda().transpose(1, 2) for _ in range(4)]
    odd = [torch.randn(b, t + 2, h, d + 3, generator=g).to(torch.bfloat16).cuda()[:, 1:-1, :, 1:d + 1] for _ in range(4)]
    shared = torch.randn(1, t, h, d, generator=g).to(torch.bfloat16).cuda().expand(b, t, h, d)
    dup = torch.randn(b, t, h, d, generator=g).to(torch.bfloat16).cuda()
    for q, k, v, do in ((*views, turned[3]), turned, odd, (views[0], shared, turned[1], shared), (dup, dup, dup, dup)):
        run(q, k, v, do, table, buckets)
        dense = [x.contiguous() for x in (q, k, v, do)]
        o1, s1 = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True)
        o2, s2 = vit_amd.relpos_attention_fwd(*dense[:3], table, buckets, training=True)
        assert torch.equal(o1, o2)
        for x, y in zip(vit_amd.relpos_attention_bwd(do, q, k, v, o1, s1, table, buckets),
                        vit_amd.relpos_attention_bwd(dense[3], *dense[:3], o2, s2, table, buckets)):
            assert torch.equal(x, y)


@gpu
@pytest.mark.parametrize("tq", [3, 70])
def test_tables_that_mask(tq):
    """A bias of -inf hides its keys, the type's lowest value hides them behind others and leaves a row of its own uniform."""
    import vit_amd
    q, k, v, do, table, _ = make("f32", 1, tq, 100, 2, 2, 16, nb=4, reach=8, seed=2)
    buckets = vit_amd.relpos_buckets(4, 8, True, "cuda")
    for value in (float("-inf"), torch.finfo(torch.float32).min):
        t = table.clone()
        t[1] = value
        run(q, k, v, do, t, buckets)
    t = torch.full_like(table, float("-inf"))
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, t, buckets, training=True)
    assert not out.any()
    assert all(not x.any() for x in vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, t, buckets))
    t = torch.full_like(table, torch.finfo(torch.float32).min)
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, t, buckets, training=True)
    assert float((out - v.mean(1, keepdim=True)).abs().max()) < 1e-5
    dv = vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, t, buckets)[2]
    assert float((dv - do.sum(1, keepdim=True) / 100).abs().max()) < 1e-5


@gpu
@pytest.mark.parametrize("tq", [3, 70])
def test_tables_of_the_types_highest_value(tq):
    """Buckets of it outweigh all others and are even among themselves."""
    import vit_amd
    q, k, v, do, table, _ = make("f32", 1, tq, 300, 2, 2, 16, nb=4, reach=8, seed=2)
    buckets = vit_amd.relpos_buckets(4, 8, True, "cuda")
    for part in (slice(0, 4), slice(1, 2)):
        t = table.clone()
        t[part] = torch.finfo(torch.float32).max
        away = torch.arange(300)[None] - torch.arange(tq)[:, None]
        on = (buckets.cpu().long()[away.clamp(-8, 8) + 8] >= part.start) & (buckets.cpu().long()[away.clamp(-8, 8) + 8] < part.stop)
        w = on.double() / on.sum(1, keepdim=True).clamp(min=1)
        out, saved = vit_amd.relpos_attention_fwd(q, k, v, t, buckets, training=True)
        dv = vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, t, buckets)[2]
        rows = on.any(1)
        assert bool(out.isfinite().all())
        for h in range(2):
            want = w @ v[0, :, h].double().cpu()
            assert float((out[0, :, h].double().cpu() - want)[rows].abs().max()) < 1e-5
            if bool(rows.all()):
                assert float((dv[0, :, h].double().cpu() - w.t() @ do[0, :, h].double().cpu()).abs().max()) < 1e-5


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tq", [3, 70])
@pytest.mark.parametrize("value", [-1e4, -1e6, -1e9, 1e9])
def test_tables_of_large_finite_values(dtype, tq, value):
    """Near and far tiles, and the backward pass, agree on what such a bias leaves of a score: the probabilities of every row add
    to 1 in both passes (fp32's 1000 terms, 2^-24 each and the exponential's; bf16's rounded p, 2^-8), and are the same where
    nothing is left: at 1e9 a score in base 2 is a multiple of 128."""
    import vit_amd
    q, k, v, do, table, _ = make(dtype, 1, tq, 1000, 2, 2, 16, nb=4, reach=8, seed=2)
    buckets = vit_amd.relpos_buckets(4, 8, True, "cuda")
    ones = torch.ones_like(do)
    for part in (slice(0, 4), slice(1, 2)):  # rows that see nothing else, rows that see other buckets, too
        t = table.clone()
        t[part] = value
        out, saved = vit_amd.relpos_attention_fwd(q, k, v, t, buckets, training=True)
        dv = vit_amd.relpos_attention_bwd(ones, q, k, v, out, saved, t, buckets)[2]
        tol = 1000 * 2.0 ** -24 + (2.0 ** -8 if dtype == "bf16" else 0)
        assert float((dv.double().sum(1) / tq - 1).abs().max()) < tol
        if part.start == 0:
            plain = vit_amd.relpos_attention_fwd(q, k, v, t, buckets)
        if part.start == 0 and abs(value) == 1e9:
            want = v.double().mean(1, keepdim=True)
            for got in (out, plain):
                # a sum of 1000 terms of at most |v|, p in two parts and one rounding
                assert float((got.double() - want).abs().max()) < 1000 * 2.0 ** -24 * float(v.abs().max()) + (2.0 ** -8 if dtype == "bf16" else 0) * float(want.abs().max()) + 2.0 ** -16


@gpu
@pytest.mark.parametrize("tq", [3, 70])
@pytest.mark.parametrize("size", [60.0, 700.0, 715.0, 1e4, 1e6, 1.1e7, 2.4e7, 5e7, 9e7, 2e8, 1e9, 1e30])
def test_tables_of_finite_values_in_fp16(tq, size):
    """As above where probabilities are scaled into fp16's range, around the size from which the scale is left off and at those
    where a float's steps are 1 to 64.  Probabilities and dv are rounded, 2^-11 each."""
    import vit_amd
    q, k, v, do, table, _ = make("f16", 1, tq, 1000, 2, 2, 16, nb=4, reach=8, seed=2)
    buckets = vit_amd.relpos_buckets(4, 8, True, "cuda")
    for sign in (-1, 1):
        for part in (slice(0, 4), slice(1, 2), slice(2, 4)):
            t = table.clone()
            t[part] += sign * size
            out, saved = vit_amd.relpos_attention_fwd(q, k, v, t, buckets, training=True)
            assert bool(out.isfinite().all()) and float(out.abs().max()) <= float(v.abs().max()) * (1 + 2.0 ** -10)
            got = vit_amd.relpos_attention_bwd(torch.ones_like(do), q, k, v, out, saved, t, buckets)
            assert all(bool(x.isfinite().all()) for x in got)
            assert float((got[2].double().sum(1) / tq - 1).abs().max()) < 1000 * 2.0 ** -24 + 2.0 ** -10
            if size < 1000:
                run(q, k, v, do, t, buckets)


@gpu
@pytest.mark.parametrize("reach", [0, 1, 2048])
def test_maps_of_the_callers_own(reach):
    g = torch.Generator().manual_seed(reach)
    q, k, v, do, table, _ = make("bf16", 2, 100, 140, 4, 4, 64, nb=8, seed=9)
    table = table[:7].contiguous()
    own = torch.randint(-2, 9, (2 * reach + 1,), generator=g).to(torch.int32).cuda()  # entries outside 0 .. 6 have no bias
    run(q, k, v, do, table, own)
    run(q[:, :2].contiguous(), k, v, do[:, :2].contiguous(), table, own, causal=True, q_start=ints(130, 20))


@gpu
def test_a_value_that_is_not_finite_reaches_its_own_rows_only():
    import vit_amd
    q, k, v, do, table, buckets = make("bf16", 2, 80, 80, 2, 2, 32, seed=4)
    q[0, 5, 1, 3] = float("nan")
    out = vit_amd.relpos_attention_fwd(q, k, v, table, buckets)
    bad = out.isnan().any(-1)
    assert bool(bad[0, 5, 1]) and int(bad.sum()) == 1
    few = vit_amd.relpos_attention_fwd(q[:, :8].contiguous(), k, v, table, buckets).isnan().any(-1)
    assert bool(few[0, 5, 1]) and int(few.sum()) == 1


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tk", [20, 700, 9000])
def test_a_token_with_values_that_are_not_numbers(dtype, tk):
    """A NaN query, and a NaN among the keys, in one piece of a cache that is cut or in all of them."""
    import vit_amd
    q, k, v, do, table, buckets = make(dtype, 3, 2, tk, 4, 2, 64, bidirectional=False, seed=tk)
    q[0, 1, 3, 5] = float("nan")
    k[1, tk // 2, 1, 7] = float("nan")
    how = dict(causal=True, q_start=ints(tk - 2, tk - 2, tk - 2))
    out, (stats, _) = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True, **how)
    want = torch.zeros(3, 2, 4, dtype=torch.bool)
    want[0, 1, 3] = True
    want[1, :, 2:] = True
    assert torch.equal(out.isnan().any(-1).cpu(), want) and torch.equal(out.isnan().all(-1).cpu(), want)
    assert torch.equal(stats.sum(-1).isnan().transpose(1, 2).cpu(), want)


@gpu
def test_gradients_against_differences():
    """Differences of the kernel's own fp32 forward: steps of 2^-6 leave an error of 2^-12 of the third derivative and the
    forward's 2^-20 / 2^-6."""
    import vit_amd
    q, k, v, do, table, buckets = make("f32", 2, 12, 50, 2, 1, 8, nb=8, reach=10, seed=6, spread=0.7)

    def loss(*a):
        return float((vit_amd.relpos_attention_fwd(*a, table_, buckets, causal=True, q_start=start).double() * do.double()).sum())

    start, table_ = ints(30, 10), table
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, causal=True, q_start=start, training=True)
    grads = vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, table, buckets, causal=True, q_start=start)
    step = 2.0 ** -6
    for t, g in zip((q, k, v, table), grads):
        for at in torch.randperm(t.numel(), generator=torch.Generator().manual_seed(0))[:6].tolist():
            flat, keep = t.view(-1), float(t.view(-1)[at])
            flat[at] = keep + step
            up = loss(q, k, v)
            flat[at] = keep - step
            down = loss(q, k, v)
            flat[at] = keep
            assert abs((up - down) / (2 * step) - float(g.view(-1)[at])) < 2e-3 * (1 + abs(float(g.view(-1)[at])))


# grids that fill the chip: workgroups of whole rows of 128, heads that share keys walked over by one workgroup or side by side
WIDE = [
    # b, tq, tk, hq, hk, d
    (1, 40, 70, 1024, 1024, 24), (2, 200, 150, 512, 256, 64), (1, 140, 130, 1024, 512, 128), (1, 300, 260, 384, 128, 80), (1, 129, 200, 512, 512, 33),
]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", WIDE)
@pytest.mark.parametrize("causal", [False, True])
def test_grids_that_fill_the_chip(dtype, shape, causal):
    q, k, v, do, table, buckets = make(dtype, *shape, bidirectional=not causal, reach=40, nb=16, seed=sum(shape))
    b, tq, tk = shape[:3]
    how = dict(q_start=ints(*[tk // 3] * b), q_len=ints(*[tq - 1] * b), k_len=ints(*[tk - 3] * b)) if causal else {}
    run(q, k, v, do, table, buckets, causal=causal, **how)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_far_reaching_maps_over_long_keys(dtype, d, causal):
    q, k, v, do, table, buckets = make(dtype, 2, 90, 600, 2, 1, d, nb=48, reach=2048, bidirectional=not causal, seed=d)
    run(q, k, v, do, table, buckets, causal=causal, q_start=ints(511, 100))


@gpu
def test_the_same_call_gives_the_same_bytes_on_any_stream():
    import vit_amd
    a = make("bf16", 2, 300, 300, 4, 2, 64, seed=12)
    q, k, v, do, table, buckets = a

    def once():
        out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True)
        return (out, *vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, table, buckets))

    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in streams:  # two calls at once
            with torch.cuda.stream(s):
                results.append(once())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(x, y) for x, y in zip(first, r))


# key blocks that no query sees: behind k_len (0 and 1 among the lengths), of a sequence without queries, and ahead of the last
# causal query; distance arrays of 65, 257 and 4097 entries a wave
EMPTY = [
    # tq, tk, d, reach, causal, q_len, k_len
    (200, 700, 64, 128, False, (200, 0, 77, 200), (1, 700, 0, 130)), (200, 700, 64, 2048, False, (200, 0, 77, 200), (1, 700, 0, 130)),
    (90, 1000, 128, 128, True, None, None), (90, 1000, 32, 2048, True, None, (1000, 3, 0, 90)), (20, 500, 64, 32, True, (20, 0, 1, 7), None),
]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", EMPTY)
def test_blocks_without_queries_give_the_same_bytes_on_any_stream(dtype, case):
    """Every workgroup leaves its distances' sums: those without a tile leave zeros, whatever LDS held before."""
    import vit_amd
    tq, tk, d, reach, causal, q_len, k_len = case
    q, k, v, do, table, buckets = make(dtype, 4, tq, tk, 4, 2, d, nb=16, reach=reach, bidirectional=not causal, seed=tq + d)
    how = dict(causal=causal, q_len=ints(*q_len) if q_len else None, k_len=ints(*k_len) if k_len else None)
    _, first = run(q, k, v, do, table, buckets, **how)

    def once():
        out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True, **how)
        return vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, table, buckets, **how)

    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                # LDS full of something else beforehand
                torch.nn.functional.softmax(q.float().reshape(-1, d) * 50, dim=-1)
                results.append(once())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(x, y) for x, y in zip(first, r))


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_captured_calls_follow_their_inputs(d):
    import vit_amd
    q, k, v, do, table, buckets = make("bf16", 2, 100, 100, 4, 2, d, seed=13)
    tok, start, lens = make("bf16", 2, 1, 1, 4, 2, d, seed=14)[0], ints(59, 99), ints(60, 100)

    def both():
        out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, causal=True, training=True)
        grads = vit_amd.relpos_attention_bwd(do, q, k, v, out, saved, table, buckets, causal=True)
        return (out, *grads, vit_amd.relpos_attention_fwd(tok, k, v, table, buckets, causal=True, q_start=start, k_len=lens))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    captured = []
    for g in graphs:
        with torch.cuda.graph(g):
            captured.append(both())
    for turn in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)).to(q.dtype))
        table.mul_(0.9)
        lens.copy_(torch.tensor([60 - turn, 100 - 7 * turn]))
        start.copy_(lens - 1)
        for s, g in zip((torch.cuda.Stream(), torch.cuda.Stream()), graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want = both()
        for got in captured:
            assert all(torch.equal(x, y) for x, y in zip(got, want)), turn


@gpu
@pytest.mark.parametrize("far,t", [((1 << 27) + 8, 20), (1 << 21, 1100)])
def test_offsets_beyond_32_bits(far, t):
    """Rows 2^27 and 2^21 elements apart: the last ones lie 5 GB behind the first."""
    import vit_amd
    d = 32
    store = torch.empty(far * t, dtype=torch.bfloat16, device="cuda")
    k = store.as_strided((1, t, 2, d), (0, far, d, 1))
    v = store.as_strided((1, t, 2, d), (0, far, d, 1), 2 * d)
    q, kd, vd, do, table, buckets = make("bf16", 1, 40, t, 2, 2, d, seed=15)
    k.copy_(kd)
    v.copy_(vd)
    for rows in (40, 1):
        x, y = q[:, :rows].contiguous(), do[:, :rows].contiguous()
        o1, s1 = vit_amd.relpos_attention_fwd(x, k, v, table, buckets, training=True)
        o2, s2 = vit_amd.relpos_attention_fwd(x, kd, vd, table, buckets, training=True)
        assert torch.equal(o1, o2)
        for a, b in zip(vit_amd.relpos_attention_bwd(y, x, k, v, o1, s1, table, buckets),
                        vit_amd.relpos_attention_bwd(y, x, kd, vd, o2, s2, table, buckets)):
            assert torch.equal(a, b)


@gpu
def test_refusals():
    import vit_amd
    q, k, v, do, table, buckets = make("bf16", 2, 8, 8, 4, 2, 16)
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True)
    wide = torch.zeros(2, 8, 4, 136, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(k=k[:, :, :1].expand(2, 8, 3, 16)), dict(v=v.float()), dict(v=v[:, :4]), dict(table=table[:, :3]), dict(table=table.half()),
                dict(buckets=buckets[:-1]), dict(buckets=buckets.long()), dict(q=q.cpu()), dict(q=q.double()), dict(q=wide, k=wide, v=wide),
                dict(q=q.transpose(2, 3)), dict(k_len=ints(1)), dict(q_start=torch.zeros(2, device="cuda")), dict(scale=float("nan")),
                dict(k_len=ints(1, 2).cpu()), dict(buckets=torch.zeros(4099, dtype=torch.int32, device="cuda")), dict(q=q[:0], k=k[:0], v=v[:0])):
        args = {**dict(q=q, k=k, v=v, table=table, buckets=buckets), **bad}
        with pytest.raises(ValueError):
            vit_amd.relpos_attention_fwd(**args)
    for bad in (dict(dout=do[:1]), dict(dout=do.float()), dict(saved=None), dict(saved=(saved[0][:1], saved[1])), dict(saved=(saved[0], None)),
                dict(out=out.transpose(0, 1))):
        args = {**dict(dout=do, q=q, k=k, v=v, out=out, saved=saved, table=table, buckets=buckets), **bad}
        with pytest.raises(ValueError):
            vit_amd.relpos_attention_bwd(**args)


def test_bucket_scheme_in_whole_numbers():
    import vit_amd
    for nb, reach, two in itertools.product((4, 8, 32, 48, 256), (128, 200, 2048), (False, True)):
        side = nb // 2 if two else nb
        single = side // 2
        ranges = side - single

        def of(n):
            return n if n < single else single + sum(n ** ranges >= single ** (ranges - j) * reach ** j for j in range(1, ranges))

        m = vit_amd.relpos_buckets(nb, reach, two).tolist()
        some = sorted({*range(0, min(reach, 140)), reach - 1, reach, reach // 2, reach // 4})
        for n in some:
            assert m[reach - n] == of(n)
            if n:
                assert m[reach + n] == (of(n) + side if two else 0)
    for bad in ((3, 128, True), (2, 128, True), (1, 128, False), (32, 4, True), (32, 4096, True), (258, 2048, True), (32, -1, False)):
        with pytest.raises(vit_amd._lib.VtError):
            vit_amd.relpos_buckets(*bad)


@gpu
def test_inputs_whose_gradient_would_be_lost_are_refused():
    import vit_amd
    q, k, v, do, table, buckets = make("f32", 2, 8, 8, 4, 2, 16)
    out, saved = vit_amd.relpos_attention_fwd(q, k, v, table, buckets, training=True)
    for at in range(4):
        args = [q, k, v, table]
        args[at] = args[at].clone().requires_grad_()
        with pytest.raises(ValueError):
            vit_amd.relpos_attention_fwd(*args, buckets)
        with pytest.raises(ValueError):
            vit_amd.relpos_attention_bwd(do, *args[:3], out, saved, args[3], buckets)
        with torch.no_grad():
            assert torch.equal(vit_amd.relpos_attention_fwd(*args, buckets), out)


@gpu
def test_a_scale_beyond_float32_is_refused():
    import vit_amd
    q, k, v, do, table, buckets = make("f32", 2, 8, 8, 4, 2, 16)
    for scale in (1e300, -1e39, float("inf")):
        with pytest.raises(ValueError):
            vit_amd.relpos_attention_fwd(q, k, v, table, buckets, scale=scale)


def test_bucket_sizes_beyond_32_bits_are_refused():
    import vit_amd
    for bad in ((32, (1 << 32) + 128), ((1 << 32) + 32, 128), (32, 10 ** 15), (32, -(1 << 32) + 128)):
        with pytest.raises(vit_amd._lib.VtError):
            vit_amd.relpos_buckets(*bad)


def test_the_library_refuses_before_it_launches():
    """Descriptors that must be turned down on the host; nothing here reaches a GPU."""
    from vit_amd._lib import VtRelposAttention, VtStrides, lib
    s = VtStrides(64, 16, 16)

    def desc(**kw):
        a = VtRelposAttention(1, 1, 8, 8, 2, 2, 16, 0, 32, 128, 0.25, 8, 8, None, None, None, 8, 8, 8, s, s, s)
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    def fwd(a, out=8, lo=None, stats=None, scratch=None, floats=0):
        return lib.vt_relpos_attention_fwd(a, out, s, lo, stats, scratch, floats, None)

    def bwd(a, out=8, lo=8, stats=8, dout=8, dq=8, scratch=16, floats=1 << 40):
        return lib.vt_relpos_attention_bwd(a, out, s, lo, stats, dout, s, dq, s, 8, s, 8, s, 8, scratch, floats, None)

    EINVAL, EUNSUPPORTED, ELIMIT = -1, -2, -6
    for kw, rc in ((dict(B=0), EINVAL), (dict(Tq=0), EINVAL), (dict(Tk=-1), EINVAL), (dict(d=0), EINVAL), (dict(q=None), EINVAL), (dict(map=None), EINVAL),
                   (dict(table=None), EINVAL), (dict(num_buckets=0), EINVAL), (dict(max_distance=-1), EINVAL), (dict(scale=float("inf")), EINVAL),
                   (dict(dtype=3), EUNSUPPORTED), (dict(d=129), EUNSUPPORTED), (dict(max_distance=2049), EUNSUPPORTED), (dict(Hk=3), EUNSUPPORTED),
                   (dict(Tq=1 << 24), EUNSUPPORTED), (dict(Tk=(1 << 29) + 1), EUNSUPPORTED), (dict(Hq=1 << 16), EUNSUPPORTED),
                   (dict(B=1 << 23), EUNSUPPORTED)):
        assert fwd(desc(**kw)) == rc, kw
        assert bwd(desc(**kw)) == rc, kw
        assert lib.vt_relpos_attention_fwd_scratch_floats(desc(**kw)) == 0
    assert fwd(desc(), out=None) == EINVAL and fwd(desc(), lo=8) == EINVAL and fwd(desc(), stats=4) == EINVAL
    long = desc(Tq=1, Tk=100000)
    assert lib.vt_relpos_attention_fwd_scratch_floats(long) > 0
    assert fwd(long) == ELIMIT and fwd(long, floats=1 << 40) == EINVAL
    assert bwd(desc(), lo=None) == EINVAL and bwd(desc(), stats=None) == EINVAL and bwd(desc(), scratch=None) == EINVAL
    assert bwd(desc(), floats=lib.vt_relpos_attention_bwd_scratch_floats(desc()) - 1) == ELIMIT
    assert bwd(desc(Tk=1 << 24)) == EUNSUPPORTED
    assert fwd(None) == EINVAL


def test_lengths_do_not_change_how_wide_heads_are_cut():
    """Lengths may be full: wide heads are cut as without them (the scratch has a row of distances a workgroup of keys), narrow
    causal ones as if a third of the batch were empty."""
    from vit_amd._lib import VtRelposAttention, VtStrides, lib
    s = VtStrides(64, 16, 16)

    def floats(b, h, t, d, causal, k_len):
        return lib.vt_relpos_attention_bwd_scratch_floats(VtRelposAttention(1, b, t, t, h, h, d, causal, 32, 128, 0.25, 8, 8, None, k_len, k_len, 8, 8, 8, s, s, s))

    for causal in (0, 1):
        for heads in (1, 2, 4, 5, 6, 8, 9, 10, 16):
            assert floats(4, heads, 2048, 128, causal, 8) == floats(4, heads, 2048, 128, causal, None)
    assert floats(4, 10, 2048, 64, 1, 8) > floats(4, 10, 2048, 64, 1, None)  # 640 blocks count as 427: shared
    assert floats(4, 16, 2048, 64, 1, 8) == floats(4, 16, 2048, 64, 1, None)  # 1024 as 683: not


def test_more_buckets_than_a_launch_has_threads_for_are_refused():
    from vit_amd._lib import VtRelposAttention, VtStrides, lib
    s = VtStrides(64, 16, 16)
    a = VtRelposAttention(1, 1, 8, 8, 2, 2, 16, 0, 1 << 26, 128, 0.25, 8, 8, None, None, None, 8, 8, 8, s, s, s)
    assert lib.vt_relpos_attention_fwd(a, 8, s, None, None, None, 0, None) == -2
    assert lib.vt_relpos_attention_bwd(a, 8, s, 8, 8, 8, s, 8, s, 8, s, 8, s, 8, 16, 1 << 40, None) == -2
    a.num_buckets -= 1
    assert lib.vt_relpos_attention_bwd_scratch_floats(a) > 0
