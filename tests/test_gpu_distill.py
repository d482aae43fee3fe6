"""vt_distill_fwd / _bwd / _fwd_bwd through vit_amd against the formulas in 64 bits.

Bounds.  An exponential's argument x carries its rounding, 2^-23 |x| with the base-2 form's, and a sum of V terms is a tree of
at most 80 additions, so q and c are off by rho = 2^-24 (80 + 4 max |z - top| / min(tau, 1)) of themselves; a gradient adds the
rounding to its type, a loss 80 roundings of its largest term."""
import pytest

torch = pytest.importorskip("torch")
from op_refs import DTYPES, distill, half_step  # noqa: E402

gpu = pytest.mark.gpu


def make(dtype, n, v, k, seed=0, labels=True):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(n, v, generator=g) * 2).to(DTYPES[dtype]).cuda()
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)]).to(torch.int32).cuda()
    top = (torch.randn(n, k, generator=g) * 2 + 3).sort(1, descending=True)[0].cuda()
    lab = torch.randint(-1, v, (n,), generator=g).to(torch.int32).cuda() if labels else None
    return z, top, ids, (torch.rand(n, generator=g) + 0.5).cuda(), lab


def check(z, top, ids, dl, lab, tau, kd, ce, loss, dz):
    ref_loss, ref_dz = distill(z, top, ids, dl, lab, tau, kd, ce)
    zz = z.double().cpu()
    span = float((zz.amax(1) - zz.masked_fill(zz == -float("inf"), 0).amin(1)).clamp(min=0).max())
    rho = 2.0 ** -24 * (80 + 4 * span / min(tau, 1.0))
    most = tau * tau * abs(kd) * (span / tau + 12) + abs(ce) * (span + 12)
    assert bool(((loss.double().cpu() - ref_loss).abs() <= 2.0 ** -24 * 80 * (most + ref_loss.abs())).all()), (loss.cpu() - ref_loss).abs().max()
    d = dl.double().cpu()[:, None].abs() * (abs(kd) * tau + abs(ce))
    q = torch.softmax(zz / tau, 1) + torch.softmax(zz, 1)
    p = torch.zeros_like(zz)
    ok = (ids >= 0) & (ids < z.shape[1])
    e = torch.where(ok.cpu(), 1.0, 0.0).double()
    p.scatter_add_(1, ids.long().cpu().clamp(0, z.shape[1] - 1), e)  # elements with a teacher's entry: p itself has rho
    bound = half_step(z.dtype) * ref_dz.abs() + rho * d * (q + p.clamp(max=1)) + (2.0 ** -25 if z.dtype == torch.float16 else 1e-38)
    if lab is not None:
        for i, l in enumerate(lab.tolist()):
            if 0 <= l < z.shape[1]:
                bound[i, l] += rho * float(d[i])
    bad = ~((dz.double().cpu() - ref_dz).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((dz.double().cpu() - ref_dz).abs() / bound).max()))


def run(data, tau, kd=0.7, ce=0.3):
    import vit_amd
    z, top, ids, dl, lab = data
    how = dict(labels=lab, tau=tau, kd_weight=kd, ce_weight=ce)
    loss, stats = vit_amd.distill_fwd(z, top, ids, **how)
    dz = vit_amd.distill_bwd(z, top, ids, dl, stats, **how)
    check(z, top, ids, dl, lab, tau, kd, ce, loss, dz)
    loss2, dz2 = vit_amd.distill_fwd_bwd(z, top, ids, dl, **how)
    check(z, top, ids, dl, lab, tau, kd, ce, loss2, dz2)
    return loss, dz


# widths on both sides of every variant's limit, and rows that are cut (few rows of more than 8192)
@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,v,k", [(3, 1, 1), (5, 10, 4), (9, 512, 7), (6, 513, 64), (5, 1025, 100), (4, 2049, 5), (3, 8192, 256), (3, 8193, 20),
                                   (2, 40001, 1024)])
def test_against_the_formula(dtype, n, v, k):
    run(make(dtype, n, v, k, seed=n + v), 2.0)


@gpu
@pytest.mark.parametrize("dtype,v", [("f32", 9000), ("f32", 32768), ("bf16", 33333), ("f16", 65536), ("f32", 32769), ("bf16", 65537),
                                     ("bf16", 16400), ("f16", 32000)])
def test_many_long_rows(dtype, v):
    run(make(dtype, 130, v, 6, seed=v), 1.0)


@gpu
def test_more_rows_than_a_grid_axis():
    """70000 rows, compared in all with the call that does both and in part with the formula."""
    import vit_amd
    z, top, ids, dl, lab = make("f16", 100, 20, 3, seed=4)
    n = 700
    big = [t.repeat(n, *[1] * (t.dim() - 1)) for t in (z, top, ids, dl, lab)]
    loss, dz = run((z, top, ids, dl, lab), 2.0)
    l1, stats = vit_amd.distill_fwd(big[0], big[1], big[2], labels=big[4], tau=2.0, kd_weight=0.7, ce_weight=0.3)
    d1 = vit_amd.distill_bwd(big[0], big[1], big[2], big[3], stats, labels=big[4], tau=2.0, kd_weight=0.7, ce_weight=0.3)
    assert torch.equal(l1, loss.repeat(n)) and torch.equal(d1, dz.repeat(n, 1))


@gpu
@pytest.mark.parametrize("tau", [0.5, 1.0, 4.0])
@pytest.mark.parametrize("kd,ce", [(1.0, 0.0), (0.0, 1.0), (0.5, 0.5), (0.0, 0.0)])
@pytest.mark.parametrize("v", [10, 3000, 20000])
def test_weights_and_temperatures(tau, kd, ce, v):
    data = make("f32", 4, v, 5, seed=v)
    run(data, tau, kd, ce)
    run((*data[:4], None), tau, kd, ce)


@gpu
@pytest.mark.parametrize("v", [40, 5000, 20000])
def test_entries_that_repeat_or_are_absent(v):
    z, top, ids, dl, lab = make("bf16", 8, v, 6, seed=v)
    ids[0] = ids[0, 0]                      # one class six times
    ids[1, 2], ids[1, 5] = ids[1, 0], -1
    ids[2] = -1                             # no entry: the label's term alone
    ids[3] = torch.tensor([v, v + 5, 2**31 - 1, -2**31, 0, v - 1])
    top[4, 1:] = float("-inf")              # one entry with all the weight
    top[5] = float("-inf")                  # entries without any
    lab[:] = ids[:, 0].clamp(0, v - 1)      # the label among the entries
    lab[6], lab[7] = v, -7                  # labels outside
    for tau in (1.0, 3.0):
        run((z, top, ids, dl, lab), tau)


@gpu
@pytest.mark.parametrize("v", [100, 4000, 30000])
def test_vocabulary_entries_that_are_masked(v):
    """Logits of -inf have no probability and no gradient."""
    z, top, ids, dl, lab = make("f32", 4, v, 3, seed=v)
    hidden = torch.ones(v, dtype=torch.bool, device="cuda")
    hidden[ids.long().flatten()] = False
    hidden[lab.long().clamp(min=0)] = False
    hidden[::3] = False
    z[:, hidden] = float("-inf")
    loss, dz = run((z, top, ids, dl, lab), 2.0)
    assert not dz[:, hidden].any() and bool(loss.isfinite().all())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", [500, 20000])
def test_a_logit_that_is_not_a_number_reaches_its_row_only(dtype, v):
    """Also where it stands in a part of the row that holds no finite logit."""
    import vit_amd
    z, top, ids, dl, lab = make(dtype, 5, v, 4, seed=v)
    ids[:], lab[:] = ids % 200, 0
    lo, hi = (256, 400) if v == 500 else (2048, 14000)
    z[1, lo:hi] = float("nan")
    z[2, lo:hi], z[2, (lo + hi) // 2] = float("-inf"), float("nan")
    z[3, lo:hi] = float("-inf")
    how = dict(labels=lab, tau=2.0, kd_weight=0.6, ce_weight=0.4)
    loss, stats = vit_amd.distill_fwd(z, top, ids, **how)
    dz = vit_amd.distill_bwd(z, top, ids, dl, stats, **how)
    both, dz2 = vit_amd.distill_fwd_bwd(z, top, ids, dl, **how)
    for a, b in ((loss, dz), (both, dz2)):
        assert a.isnan().tolist() == [False, True, True, False, False]
        assert bool(b[1:3].isnan().all()) and bool(b[[0, 3, 4]].isfinite().all())
    rows = [0, 3, 4]
    check(z[rows], top[rows], ids[rows], dl[rows], lab[rows], 2.0, 0.6, 0.4, loss[rows], dz[rows])


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n,v", [(6, 60), (6, 5000), (130, 9000), (6, 20000)])
def test_rows_without_a_term_have_no_gradient_whatever_they_hold(dtype, n, v):
    """Rows of padding: no valid entry and no label, logits NaN, infinite or wholly masked."""
    import vit_amd
    z, top, ids, dl, lab = make(dtype, n, v, 4, seed=v)
    ids[:4], lab[:4] = -1, -1
    lab[4:] = 3
    z[0], z[1], z[2] = float("nan"), float("-inf"), float("inf")
    z[3, ::2] = float("nan")
    for kd, ce in ((0.6, 0.4), (1.0, 0.0)):
        how = dict(labels=lab, tau=2.0, kd_weight=kd, ce_weight=ce)
        loss, stats = vit_amd.distill_fwd(z, top, ids, **how)
        dz = vit_amd.distill_bwd(z, top, ids, dl, stats, **how)
        both, dz2 = vit_amd.distill_fwd_bwd(z, top, ids, dl, **how)
        for a, b in ((loss, dz), (both, dz2)):
            assert not a[:4].any() and not b[:4].any()
            check(z[4:], top[4:], ids[4:], dl[4:], lab[4:], 2.0, kd, ce, a[4:], b[4:])
    # a weight of 0 takes its term away, too
    top[4], lab[5] = float("nan"), v
    loss, dz = vit_amd.distill_fwd_bwd(z, top, ids, dl, labels=lab, tau=2.0, kd_weight=0.0, ce_weight=1.0)
    assert bool(loss[4:].isfinite().all()) and bool(dz[4].isfinite().all()) and not dz[5].any()


@gpu
@pytest.mark.parametrize("n,v", [(7, 100), (6, 3001), (200, 9001), (3, 50001)])
def test_strided_rows_and_results_in_place(n, v):
    import vit_amd
    z, top, ids, dl, lab = make("bf16", n, v, 4, seed=n)
    how = dict(labels=lab, tau=2.0, kd_weight=0.6, ce_weight=0.4)
    loss, dz = vit_amd.distill_fwd_bwd(z, top, ids, dl, **how)
    _, stats = vit_amd.distill_fwd(z, top, ids, **how)
    dz_split = vit_amd.distill_bwd(z, top, ids, dl, stats, **how)
    wide = torch.full((n, v + 13), 7.0, dtype=z.dtype, device="cuda")
    for both in (True, False):
        view = wide[:, 5:5 + v]
        view.copy_(z)
        if both:
            got, out = vit_amd.distill_fwd_bwd(view, top, ids, dl, out=view, **how)
            assert torch.equal(got, loss)
        else:
            out = vit_amd.distill_bwd(view, top, ids, dl, stats, out=view, **how)
        assert out is view and torch.equal(view, dz if both else dz_split)
        assert bool((wide[:, :5] == 7).all()) and bool((wide[:, 5 + v:] == 7).all())


@gpu
def test_cut_rows_replaced_in_place_with_entries_in_every_part():
    import vit_amd
    z, top, ids, dl, lab = make("f16", 3, 60000, 1024, seed=11)
    how = dict(labels=lab, tau=2.0, kd_weight=0.6, ce_weight=0.4)
    _, stats = vit_amd.distill_fwd(z, top, ids, **how)
    want = vit_amd.distill_bwd(z, top, ids, dl, stats, **how)
    for _ in range(8):
        own = z.clone()
        assert torch.equal(vit_amd.distill_bwd(own, top, ids, dl, stats, out=own, **how), want)


@gpu
def test_gradient_against_differences():
    """In fp32 with steps of 2^-5: 2^-10 / 6 of the third derivative and the loss's 2^-22 / 2^-5."""
    import vit_amd
    z, top, ids, dl, lab = make("f32", 3, 50, 5, seed=1)
    how = dict(labels=lab, tau=1.5, kd_weight=0.5, ce_weight=0.5)
    _, dz = vit_amd.distill_fwd_bwd(z, top, ids, torch.ones_like(dl), **how)
    for i in range(3):
        for j in [*ids[i].tolist(), 0, 7, 49]:
            keep, vals = float(z[i, j]), []
            for s in (2.0 ** -5, -2.0 ** -5):
                z[i, j] = keep + s
                vals.append(float(vit_amd.distill_fwd(z, top, ids, **how)[0][i]))
            z[i, j] = keep
            assert abs((vals[0] - vals[1]) * 16 - float(dz[i, j])) < 1e-3


@gpu
@pytest.mark.parametrize("n,v", [(300, 12000), (4, 100000), (64, 10)])
def test_the_same_bytes_every_time_on_streams_and_in_graphs(n, v):
    import vit_amd
    z, top, ids, dl, lab = make("bf16", n, v, 5, seed=2)

    def once():
        return vit_amd.distill_fwd_bwd(z, top, ids, dl, labels=lab, tau=2.0, kd_weight=0.5, ce_weight=0.5)

    first = once()
    torch.cuda.synchronize()
    got = []
    for s in (torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(s):
            got += [once(), once()]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in got for a, b in zip(o, first))
    graphs, held = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            held.append(once())
    for turn in range(3):
        z.mul_(0.8)
        dl.add_(0.25)
        for g in graphs:
            g.replay()
        want = once()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in held for a, b in zip(o, want)), turn


@gpu
@pytest.mark.parametrize("v", [100, 9001])
def test_gradient_beside_the_logits_in_one_matrix(v):
    import vit_amd
    z, top, ids, dl, lab = make("bf16", 5, v, 4, seed=v)
    both = torch.zeros(5, 2 * v, dtype=z.dtype, device="cuda")
    both[:, :v] = z
    how = dict(labels=lab, tau=2.0, kd_weight=0.7, ce_weight=0.3)
    want = vit_amd.distill_fwd_bwd(z, top, ids, dl, **how)
    loss, dz = vit_amd.distill_fwd_bwd(both[:, :v], top, ids, dl, out=both[:, v:], **how)
    assert torch.equal(loss, want[0]) and torch.equal(dz, want[1]) and torch.equal(both[:, :v], z)
    with pytest.raises(vit_amd._lib.VtError):
        vit_amd.distill_fwd_bwd(both[:, :v], top, ids, dl, out=both[:, v - 1:-1], **how)


@gpu
def test_refusals():
    import vit_amd
    z, top, ids, dl, lab = make("bf16", 4, 40, 5)
    good = dict(logits=z, top_logit=top, top_id=ids, dloss=dl, labels=lab)
    vit_amd.distill_fwd_bwd(**good)
    for bad in (dict(logits=z.cpu()), dict(logits=z.double()), dict(logits=z[0]), dict(logits=z.t()), dict(logits=z[:1].expand(4, 40)), dict(top_logit=top.half()),
                dict(top_logit=top[:, :3]), dict(top_id=ids.long()), dict(top_id=ids[:2]), dict(labels=lab.long()), dict(labels=lab[:1]), dict(tau=0.0),
                dict(tau=-1.0), dict(tau=float("nan")), dict(tau=float("inf")), dict(dloss=dl.half()), dict(dloss=dl[:2]), dict(out=z.float()),
                dict(out=z[:2]), dict(out=z.t()), dict(logits=z[:, :4])):
        with pytest.raises(ValueError):
            vit_amd.distill_fwd_bwd(**{**good, **bad})
    _, stats = vit_amd.distill_fwd(z, top, ids)
    with pytest.raises(ValueError):
        vit_amd.distill_bwd(z, top, ids, dl, stats[:2])


@gpu
def test_inputs_whose_gradient_would_be_lost_are_refused():
    import vit_amd
    z, top, ids, dl, lab = make("bf16", 4, 40, 5)
    loss, stats = vit_amd.distill_fwd(z, top, ids)
    leaf = z.clone().requires_grad_()
    calls = (lambda a, b: vit_amd.distill_fwd(a, b, ids), lambda a, b: vit_amd.distill_fwd_bwd(a, b, ids, dl),
             lambda a, b: vit_amd.distill_bwd(a, b, ids, dl, stats))
    for call in calls:
        for a, b in ((leaf, top), (leaf * 2, top), (z, top.clone().requires_grad_())):
            with pytest.raises(ValueError):
                call(a, b)
    with torch.no_grad():
        assert torch.equal(vit_amd.distill_fwd(leaf, top, ids)[0], loss)
    assert torch.equal(vit_amd.distill_fwd(leaf.detach(), top, ids)[0], loss)

    class Taught(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            loss, ctx.d = vit_amd.distill_fwd_bwd(x, top, ids, torch.ones_like(dl))
            return loss

        @staticmethod
        def backward(ctx, g):
            return ctx.d * g[:, None]

    Taught.apply(leaf).sum().backward()
    assert torch.equal(leaf.grad, vit_amd.distill_fwd_bwd(z, top, ids, torch.ones_like(dl))[1])


@gpu
def test_numbers_beyond_float32_are_refused():
    import vit_amd
    z, top, ids, dl, lab = make("f32", 4, 40, 5)
    for bad in (dict(tau=1e300), dict(tau=1e-60), dict(tau=1e-42), dict(kd_weight=1e300), dict(ce_weight=-1e39)):
        with pytest.raises(ValueError):
            vit_amd.distill_fwd(z, top, ids, lab, **bad)


def test_the_library_refuses_before_it_launches():
    from vit_amd._lib import VtDistill, lib

    def desc(**kw):
        a = VtDistill(1, 4, 100, 5, 100, 100, 1.0, 1.0, 0.0, 16, 16, 16, None)
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    def calls(a, loss=16, stats=16, dl=16, dz=16, scratch=16, floats=1 << 40):
        return (lib.vt_distill_fwd(a, loss, stats, scratch, floats, None), lib.vt_distill_bwd(a, dl, stats, dz, None),
                lib.vt_distill_fwd_bwd(a, dl, loss, dz, scratch, floats, None))

    for kw, rc in ((dict(N=0), -1), (dict(V=0), -1), (dict(K=0), -1), (dict(K=101), -1), (dict(ldz=99), -1), (dict(tau=0.0), -1), (dict(z=None), -1),
                   (dict(top_id=None), -1), (dict(dtype=7), -2), (dict(V=5000, K=1025, ldz=5000, ldd=5000), -2),
                   (dict(V=(1 << 30) + 1, ldz=1 << 31, ldd=1 << 31), -2), (dict(N=1 << 30, V=9000, ldz=9000, ldd=9000), -2), (dict(N=1 << 24), -2)):
        assert calls(desc(**kw)) == (rc, rc, rc), kw
        assert lib.vt_distill_scratch_floats(desc(**kw)) == 0
    assert calls(desc(ldd=99))[1:] == (-1, -1)
    # rows of dz that overlap z's (2 bytes an element): shifted, of another stride, beside each other but too near
    for kw, dz in ((dict(), 18), (dict(), 16 + 2 * 300), (dict(ldd=104), 16), (dict(ldz=150, ldd=150), 16 + 2 * 99), (dict(ldz=150, ldd=150), 16 + 2 * 151),
                   (dict(z=16 + 2 * 150, ldz=150, ldd=150), 18)):
        assert calls(desc(**kw), dz=dz)[1:] == (-1, -1), (kw, dz)
    assert lib.vt_distill_fwd(desc(), None, 16, None, 0, None) == -1 and lib.vt_distill_fwd(desc(), 16, 8, None, 0, None) == -1
    assert lib.vt_distill_bwd(desc(), None, 16, 16, None) == -1 and lib.vt_distill_bwd(desc(), 16, 16, None, None) == -1
    cut = desc(V=100000, ldz=100000, ldd=100000)
    floats = lib.vt_distill_scratch_floats(cut)
    assert floats > 0
    assert lib.vt_distill_fwd(cut, 16, 16, 16, floats - 1, None) == -6 and lib.vt_distill_fwd_bwd(cut, 16, 16, 16, 16, floats - 1, None) == -6
    assert lib.vt_distill_fwd(cut, 16, 16, None, floats, None) == -1
