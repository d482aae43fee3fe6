"""vt_block_norms_fwd / _bwd through vit_amd against automatic differentiation in 64 bits.

Tolerance, relative to a result's largest value: half a step of its type for its one rounding, and 2^-24 * 256 for the fp32
sums (a thread adds at most 16 columns and its rows, then ten exchanges and 16 partial sums: some 32 roundings, through up to
eight such steps in a row).

dx and dy are differences: norm'(g) = rstd (g - mean g - t^ mean(g t^)).  Each of the three terms is as large as rstd max|g| and
rounded in fp32 before they cancel (with two columns and a layer norm they cancel to rstd g eps / (var + eps): t^ is +-1 there,
so g - mean g = t^ mean(g t^) but for eps).  Their fp32 part is therefore counted relative to rstd max|g|, if that is larger."""
import pytest

torch = pytest.importorskip("torch")
from op_refs import DTYPES, half_step, norms  # noqa: E402

gpu = pytest.mark.gpu
NAMES = ("gate", "res_scale", "w_post", "b_post", "w_pre", "b_pre")


def make(dtype, n, d, per, kind, skip=(), seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]

    def t(*s, scale=1.0, at=0.0, ty=dt):
        return (torch.randn(*s, generator=g) * scale + at).to(ty).cuda()

    w = dict(gate=t((n + per - 1) // per, d, scale=0.3, at=0.5), res_scale=t(d, scale=0.2, at=0.6, ty=torch.float32),
             w_post=t(d, scale=0.2, at=1, ty=torch.float32), b_post=t(d, scale=0.2, ty=torch.float32) if kind == "layer" else None,
             w_pre=t(d, scale=0.2, at=1, ty=torch.float32), b_pre=t(d, scale=0.2, ty=torch.float32) if kind == "layer" else None)
    for name in skip:
        w[name] = None
        if name.startswith("w_"):
            w["b_" + name[2:]] = None
    return t(n, d, scale=2.0, at=0.5), t(n, d, scale=0.7, at=-0.3), t(n, d), t(n, d), w


def near(got, want, dtype, what, terms=0.0):
    """terms: size of the terms that cancel in the result."""
    want = want.double()
    top = float(want.abs().max())
    err = float((got.double().cpu() - want).abs().max())
    assert got.dtype == dtype, what
    assert err <= half_step(dtype) * top + 2.0 ** -24 * 256 * max(top, terms) + 1e-12, (what, err, top, terms)


def run(dtype, x, y, dr, dh, w, per, kind, eps=1e-6):
    import vit_amd
    how = dict(rows_per_gate=per, kind=kind, eps=eps, **w)
    r, h, stats = vit_amd.block_norms_fwd(x, y, **how)
    dh = dh if w["w_pre"] is not None else None
    grads = vit_amd.block_norms_bwd(dr, dh, x, y, stats, **how)
    ref_r, ref_h, ref = norms(x, y, w["gate"], per, w["res_scale"], w["w_post"], w["b_post"], w["w_pre"], w["b_pre"], kind, eps, dr, dh)
    near(r, ref_r, DTYPES[dtype], "r")
    assert (h is None) == (ref_h is None)
    if h is not None:
        near(h, ref_h, DTYPES[dtype], "h")
    assert {n for n, t in grads.items() if t is not None} == set(ref)
    rstd_y, rstd_r = (stats[:, i:i + 1].double().cpu() for i in (1, 3))
    one = torch.ones(1, 1).double()
    part = {n: one if t is None else t.double().cpu() for n, t in w.items()}
    gate = part["gate"].repeat_interleave(per, 0)[:x.shape[0]] if w["gate"] is not None else one
    terms = {"dy": float((ref["dx"] * part["res_scale"] * gate * part["w_post"] * rstd_y).abs().max()) if w["w_post"] is not None else 0.0,
             "dx": float((dh.double().cpu() * part["w_pre"] * rstd_r).abs().max()) if dh is not None else 0.0}
    for n, t in ref.items():
        near(grads[n], t, DTYPES[dtype] if n in ("dx", "dy", "dgate") else torch.float32, n, terms.get(n, 0.0))
    return r, h, grads


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("n,d,per", [(1, 2, 1), (5, 7, 2), (512, 32, 16), (33, 512, 1), (70, 1001, 33), (9, 1500, 9), (40, 2048, 7), (21, 4095, 1),
                                     (6, 8192, 4), (2500, 64, 2500), (3000, 16, 1700)])
def test_against_the_formula(dtype, kind, n, d, per):
    run(dtype, *make(dtype, n, d, per, kind, seed=n + d), per, kind)


@gpu
@pytest.mark.parametrize("skip", [("gate",), ("res_scale",), ("w_post",), ("w_pre",), ("w_post", "w_pre"), ("gate", "res_scale", "w_post"),
                                  ("gate", "res_scale", "w_post", "w_pre")])
@pytest.mark.parametrize("kind,d", [("rms", 100), ("layer", 100), ("rms", 1600), ("layer", 5000)])
def test_absent_parts(skip, kind, d):
    run("f32", *make("f32", 37, d, 5, kind, skip, seed=d), 5, kind)


@gpu
def test_layer_norms_without_their_shift_and_a_row_of_one_column():
    x, y, dr, dh, w = make("bf16", 20, 96, 4, "layer")
    w["b_post"] = None
    run("bf16", x, y, dr, dh, w, 4, "layer")
    x, y, dr, dh, w = make("f32", 20, 1, 4, "rms")
    run("f32", x, y, dr, dh, w, 4, "rms", eps=0.25)


@gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_rows_far_from_zero_and_rows_of_zeros(kind):
    """The variance is taken around the mean: an offset of 64 costs the offset's own rounding, 64 * 2^-24 of the deviation."""
    x, y, dr, dh, w = make("f32", 12, 640, 1, kind, seed=3)
    y[3], x[4] = y[3] + 64, x[4] - 64
    import vit_amd
    how = dict(kind=kind, eps=1e-5, **w)
    r, h, stats = vit_amd.block_norms_fwd(x, y, **how)
    rr, hh, _ = norms(x, y, w["gate"], 1, w["res_scale"], w["w_post"], w["b_post"], w["w_pre"], w["b_pre"], kind, 1e-5)
    assert float((h.double().cpu() - hh).abs().max() / hh.abs().max()) < 64 * 2.0 ** -24 * 8
    y[5], x[5] = 0, 0
    r, h, stats = vit_amd.block_norms_fwd(x, y, **how)
    assert bool(r[5].isfinite().all()) and bool(h[5].isfinite().all())


@gpu
def test_only_one_of_the_gradients_and_results_in_place():
    import vit_amd
    from vit_amd._lib import check, lib
    from vit_amd.ops import _norm_args
    x, y, dr, dh, w = make("bf16", 50, 300, 5, "layer", seed=1)
    how = dict(rows_per_gate=5, kind="layer", **w)
    r, h, stats = vit_amd.block_norms_fwd(x, y, **how)
    a = vit_amd.block_norms_bwd(None, dh, x, y, stats, **how)
    b = vit_amd.block_norms_bwd(torch.zeros_like(dr), dh, x, y, stats, **how)
    assert all(torch.equal(a[n], b[n]) for n in a)
    want = vit_amd.block_norms_bwd(dr, dh, x, y, stats, **how)
    args, _, _, _ = _norm_args(x, y, w["gate"], 5, w["res_scale"], w["w_post"], w["b_post"], w["w_pre"], w["b_pre"], "layer", 1e-6)
    dx, dy, dg = dr.clone(), dh.clone(), torch.empty_like(w["gate"])
    floats = lib.vt_block_norms_bwd_scratch_floats(args)
    scratch = torch.empty(floats, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    check(lib.vt_block_norms_bwd(args, x.data_ptr(), y.data_ptr(), stats.data_ptr(), dx.data_ptr(), dy.data_ptr(), dx.data_ptr(), dy.data_ptr(),
                                 dg.data_ptr(), None, None, None, None, None, scratch.data_ptr(), floats, s))
    assert torch.equal(dx, want["dx"]) and torch.equal(dy, want["dy"]) and torch.equal(dg, want["dgate"])


@gpu
def test_a_gate_row_for_more_rows_than_there_are():
    """One row of the gate for all rows, by any number of rows per gate row from theirs on: the same bytes and scratch."""
    import vit_amd
    from vit_amd._lib import lib
    from vit_amd.ops import _norm_args
    x, y, dr, dh, w = make("f32", 50, 300, 50, "rms", seed=1)
    want = None
    for per in (50, 51, 2**31 - 1):
        r, h, stats = vit_amd.block_norms_fwd(x, y, rows_per_gate=per, **w)
        g = vit_amd.block_norms_bwd(dr, dh, x, y, stats, rows_per_gate=per, **w)
        got = [r, h] + [t for t in g.values() if t is not None]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    a = _norm_args(x, y, w["gate"], 50, w["res_scale"], w["w_post"], None, w["w_pre"], None, "rms", 1e-6)[0]
    floats = lib.vt_block_norms_bwd_scratch_floats(a)
    a.rows_per_gate = 2**31 - 1
    assert lib.vt_block_norms_bwd_scratch_floats(a) == floats


@gpu
def test_the_same_bytes_every_time_on_streams_and_in_graphs():
    import vit_amd
    x, y, dr, dh, w = make("bf16", 700, 1024, 100, "rms", seed=2)
    how = dict(rows_per_gate=100, kind="rms", **w)

    def once():
        r, h, stats = vit_amd.block_norms_fwd(x, y, **how)
        return [r, h] + [t for t in vit_amd.block_norms_bwd(dr, dh, x, y, stats, **how).values() if t is not None]

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
        x.mul_(1.1)
        w["w_pre"].add_(0.1)
        for g in graphs:
            g.replay()
        want = once()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in held for a, b in zip(o, want)), turn


@gpu
def test_refusals():
    import vit_amd
    x, y, dr, dh, w = make("bf16", 10, 64, 5, "layer")
    good = dict(x=x, y=y, rows_per_gate=5, kind="layer", **w)
    vit_amd.block_norms_fwd(**good)
    big = torch.zeros(2, 8193, device="cuda")
    for bad in (dict(y=y[:5]), dict(y=y.float()), dict(x=x.t()), dict(x=x[:, ::2], y=y[:, ::2]), dict(x=x.cpu()), dict(x=x.double()), dict(kind="batch"),
                dict(kind="rms"), dict(w_post=None), dict(gate=w["gate"][:1]), dict(rows_per_gate=0), dict(rows_per_gate=4), dict(eps=-1.0),
                dict(w_pre=w["w_pre"].half()), dict(res_scale=w["res_scale"][:3]), dict(x=x[:0], y=y[:0]), dict(x=big, y=big)):
        with pytest.raises(ValueError):
            vit_amd.block_norms_fwd(**{**good, **bad})
    stats = vit_amd.block_norms_fwd(**good)[2]
    for bad in (dict(dh=None), dict(dr=dr[:2]), dict(stats=stats[:3]), dict(dr=None, dh=None)):
        with pytest.raises(ValueError):
            vit_amd.block_norms_bwd(**{**dict(dr=dr, dh=dh, stats=stats), **good, **bad})


@gpu
def test_inputs_whose_gradient_would_be_lost_are_refused():
    import vit_amd
    x, y, dr, dh, w = make("f32", 10, 64, 5, "layer")
    good = dict(x=x, y=y, rows_per_gate=5, kind="layer", **w)
    r, _, stats = vit_amd.block_norms_fwd(**good)
    for name in ("x", "y", *NAMES):
        args = {**good, name: good[name].clone().requires_grad_()}
        with pytest.raises(ValueError):
            vit_amd.block_norms_fwd(**args)
        with pytest.raises(ValueError):
            vit_amd.block_norms_bwd(dr=dr, dh=dh, stats=stats, **args)
        with torch.no_grad():
            assert torch.equal(vit_amd.block_norms_fwd(**args)[0], r)


@gpu
def test_an_eps_beyond_float32_is_refused():
    import vit_amd
    x, y, dr, dh, w = make("f32", 10, 64, 5, "layer")
    for eps in (1e300, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            vit_amd.block_norms_fwd(x, y, rows_per_gate=5, kind="layer", eps=eps, **w)


def test_the_library_refuses_before_it_launches():
    from vit_amd._lib import VtBlockNorms, lib

    def desc(**kw):
        a = VtBlockNorms(1, 1, 8, 64, 2, 1e-6, 8, 8, 8, 8, 8, 8)
        for n, v in kw.items():
            setattr(a, n, v)
        return a

    def fwd(a, x=16, y=16, r=16, h=16, stats=16):
        return lib.vt_block_norms_fwd(a, x, y, r, h, stats, None)

    def bwd(a, dr=16, dh=16, dgate=16, floats=1 << 40, scratch=16, db=16, dw=16):
        return lib.vt_block_norms_bwd(a, 16, 16, 16, dr, dh, 16, 16, dgate, 16, dw, db, 16, None, scratch, floats, None)

    for kw, rc in ((dict(N=0), -1), (dict(D=0), -1), (dict(rows_per_gate=0), -1), (dict(eps=-1.0), -1), (dict(kind=0), -1), (dict(w_post=None), -1),
                   (dict(dtype=5), -2), (dict(kind=2), -2), (dict(D=8193), -2)):
        assert fwd(desc(**kw)) == rc, kw
        assert bwd(desc(**kw)) == rc, kw
        assert lib.vt_block_norms_bwd_scratch_floats(desc(**kw)) == 0
    for rows, d in ((1 << 26, 64), (1 << 22, 8192)):
        assert fwd(desc(N=rows, D=d)) == -2 and bwd(desc(N=rows, D=d)) == -2
    assert fwd(desc(), x=None) == -1 and fwd(desc(), h=None) == -1 and fwd(desc(), stats=8) == -1 and fwd(None) == -1
    assert bwd(desc(), dgate=None) == -1 and bwd(desc(gate=None)) == -1 and bwd(desc(), dh=None) == -1 and bwd(desc(w_pre=None, b_pre=None)) == -1
    assert bwd(desc(b_post=None)) == -1 and bwd(desc(res_scale=None)) == -1 and bwd(desc(), scratch=None) == -1
    assert bwd(desc(), floats=lib.vt_block_norms_bwd_scratch_floats(desc()) - 1) == -6
