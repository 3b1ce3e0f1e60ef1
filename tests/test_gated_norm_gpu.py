"""The gated norms on the GPU, forward and backward, against their formulas in 64 bits.

Tolerances. A mean of D <= 10240 squares is at most 40 additions in a lane, 8 more over lanes and a division: its relative error
is below 64 * 2^-24 = 2^-18, half of that in rstd, and a handful of products add 2^-24 each; so a value made of terms t is off
by at most 2^-18 sum |t| before it is stored, plus half a step of its type (bf16: 2^-8 |value|). Two norms in a row (the
backward) add twice: 2^-16. A column sum over R rows adds (R + 32) 2^-24 sum |t|."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6
E1, E2 = 2.0 ** -18, 2.0 ** -16


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from vpt import ops as _ops
    return _ops


def rnd(*shape, dtype=BF16, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def make(G, R, D, stream, opts, seed=0):
    """opts: letters of what is there: p post, n next norm, g / G gate of all / of each group, m / M modulation likewise."""
    vec = lambda each, s, sc: rnd(*((G, D) if each else (D,)), seed=s, scale=sc)  # noqa: E731
    kw = dict(w_post=1 + rnd(D, seed=seed + 1, scale=0.2) if "p" in opts else None,
              w_pre=1 + rnd(D, seed=seed + 2, scale=0.2) if "n" in opts else None,
              gate=vec("G" in opts, seed + 3, 0.7) if "g" in opts.lower() else None,
              scale=vec("M" in opts, seed + 4, 0.5) if "m" in opts.lower() else None,
              shift=vec("M" in opts, seed + 5, 0.5) if "m" in opts.lower() else None, groups=G, resid_scale=0.7)
    return rnd(G * R, D, seed=seed + 6, scale=3.0), rnd(G * R, D, dtype=stream, seed=seed + 7, scale=2.0), kw


def rows(v, G, R):
    """A vector of the call as f64, broadcast over rows."""
    v = v.double()
    return v if v.dim() == 1 else v.repeat_interleave(R, 0)


def half(t, ref):
    return 2.0 ** -8 * ref.abs() if t.dtype == BF16 else 2.0 ** -24 * ref.abs()


def ok(got, ref, tol, what):
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} past the bound"


def check_fwd(ops, h, x, kw):
    G = kw["groups"]
    R = h.shape[0] // G
    x_new, y, rh, rx = ops.gated_norm_fwd(h, x, eps=EPS, **kw)
    u = h.double()
    if kw["w_post"] is not None:
        r = torch.rsqrt(u.square().mean(1, keepdim=True) + EPS)
        ok(rh, r[:, 0], E1 * r[:, 0], "rstd_post")
        u = u * r * kw["w_post"].double()
    else:
        assert rh is None
    if kw["gate"] is not None:
        u = u * rows(kw["gate"], G, R)
    u = u * kw["resid_scale"]
    ref = x.double() + u
    assert x_new.dtype == x.dtype
    ok(x_new, ref, half(x_new, ref) * 1.01 + E1 * (x.double().abs() + u.abs()), "x_new")
    if kw["w_pre"] is None:
        assert y is None and rx is None
        return x_new, y, rh, rx
    n = x_new.double()
    r = torch.rsqrt(n.square().mean(1, keepdim=True) + EPS)
    ok(rx, r[:, 0], E1 * r[:, 0], "rstd_pre")
    ref = n * r * kw["w_pre"].double()
    top = ref.abs()
    if kw["scale"] is not None:
        sc, sh = rows(kw["scale"], G, R), rows(kw["shift"], G, R)
        ref, top = ref * (1 + sc) + sh, top * (1 + sc.abs()) + sh.abs()
    ok(y, ref, half(y, ref) * 1.01 + E1 * top, "y")
    return x_new, y, rh, rx


def check_bwd(ops, h, x_new, rh, rx, kw, dx_new, dy):
    G = kw["groups"]
    R = h.shape[0] // G
    D = h.shape[1]
    got = ops.gated_norm_bwd(dy, dx_new, h, x_new, rh, rx, **kw)
    s = kw["resid_scale"]
    dX = dx_new.double() if dx_new is not None else torch.zeros(h.shape, dtype=F64, device=DEV)
    top = dX.abs()
    gsum = lambda t: t.view(G, R, D).sum(1)  # noqa: E731
    es = (R + 32) * 2.0 ** -24 + E2

    def vec(name, v, terms, mags):
        if v is None:
            assert getattr(got, name) is None
            return
        t, a = gsum(terms), gsum(mags)
        if v.dim() == 1:
            t, a = t.sum(0), a.sum(0)
        g = getattr(got, name)
        assert g.dtype == F32 and g.shape == v.shape
        ok(g, t, (es + G * 2.0 ** -24) * a + 1e-30, name)

    if kw["w_pre"] is not None:
        r = torch.rsqrt(x_new.double().square().mean(1, keepdim=True) + EPS)
        n, d, w = x_new.double() * r, dy.double(), kw["w_pre"].double()
        one = 1 + rows(kw["scale"], G, R) if kw["scale"] is not None else torch.ones_like(n)
        vec("dshift", kw["shift"], d, d.abs())
        vec("dscale", kw["scale"], d * n * w, (d * n * w).abs())
        vec("dw_pre", kw["w_pre"], d * one * n, (d * one * n).abs())
        dn = d * one * w
        dX = dX + r * (dn - n * (dn * n).mean(1, keepdim=True))
        top = top + r * (dn.abs() + n.abs() * (dn * n).abs().mean(1, keepdim=True))
        ok(got.dx, dX, half(got.dx, dX) * 1.01 + E2 * top, "dx")
    else:
        assert got.dx is dx_new and got.dw_pre is None
    r = torch.rsqrt(h.double().square().mean(1, keepdim=True) + EPS) if kw["w_post"] is not None else 1.0
    v = h.double() * r
    w = kw["w_post"].double() if kw["w_post"] is not None else torch.ones(D, dtype=F64, device=DEV)
    gt = rows(kw["gate"], G, R) if kw["gate"] is not None else torch.ones_like(v)
    vec("dgate", kw["gate"], s * dX * v * w, s * top * (v * w).abs())
    vec("dw_post", kw["w_post"], s * gt * dX * v, s * top * (gt * v).abs())
    dv, A = s * gt * w * dX, s * (gt * w).abs() * top
    dh, T = dv, A
    if kw["w_post"] is not None:
        dh = r * (dv - v * (dv * v).mean(1, keepdim=True))
        T = r * (A + v.abs() * (A * v.abs()).mean(1, keepdim=True))
    ok(got.dh, dh, half(got.dh, dh) * 1.01 + E2 * T, "dh")
    return got


OPTS = ["pnGM", "pngm", "pn", "pG", "nM", "ng", "p", "g", "pnGm", "pngM"]


@pytest.mark.parametrize("opts", OPTS)
@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("G,R,D", [(1, 1, 8), (3, 5, 64), (2, 77, 640)])
def test_both_directions(ops, G, R, D, stream, opts):
    h, x, kw = make(G, R, D, stream, opts, seed=D)
    x_new, y, rh, rx = check_fwd(ops, h, x, kw)
    dxn = rnd(G * R, D, dtype=stream, seed=50)
    check_bwd(ops, h, x_new, rh, rx, kw, dxn, rnd(G * R, D, seed=51) if y is not None else None)
    if y is not None:
        check_bwd(ops, h, x_new, rh, rx, kw, None, rnd(G * R, D, seed=51))


@pytest.mark.parametrize("G,R,D", [(1, 1, 16), (1, 3, 120), (2, 1, 136), (5, 33, 256), (1, 300, 512), (2, 130, 648), (8, 131, 768),
                                   (3, 100, 1024), (4, 65, 1280), (2, 40, 1288), (1, 70, 2048), (2, 33, 2560), (1, 9, 2568),
                                   (2, 20, 4096), (1, 7, 5120), (1, 5, 10240), (300, 1, 64), (40, 9, 768)])
@pytest.mark.parametrize("stream", [BF16, F32])
def test_shapes(ops, G, R, D, stream):
    h, x, kw = make(G, R, D, stream, "pnGM", seed=G + R)
    x_new, y, rh, rx = check_fwd(ops, h, x, kw)
    check_bwd(ops, h, x_new, rh, rx, kw, rnd(G * R, D, dtype=stream, seed=50), rnd(G * R, D, seed=51))


@pytest.mark.parametrize("D", [64, 768, 1280, 2560, 4096])
def test_rows_of_zeros(ops, D):
    """A padded token (h and x zero): rstd = eps^-1/2, nothing but the modulation's shift comes out, gradients are finite."""
    h, x, kw = make(2, 6, D, BF16, "pnGM", seed=3)
    h[4] = 0
    x[4] = 0
    h[11] = 0
    x_new, y, rh, rx = check_fwd(ops, h, x, kw)
    assert not x_new[4].any() and torch.equal(y[4], kw["shift"][0]) and torch.equal(x_new[11], x[11])
    g = check_bwd(ops, h, x_new, rh, rx, kw, rnd(12, D, seed=50), rnd(12, D, seed=51))
    assert all(torch.isfinite(t.float()).all() for t in g)


@pytest.mark.parametrize("D", [768, 2048, 4096])
def test_not_finite_rows(ops, D):
    """A NaN or an infinity stays in its row forward; backward it reaches its row and its group's column sums."""
    h, x, kw = make(2, 40, D, BF16, "pnGM", seed=4)
    clean = ops.gated_norm_fwd(h, x, **kw)
    h2 = h.clone()
    h2[7, 3] = float("nan")
    h2[50, 9] = float("inf")
    got = ops.gated_norm_fwd(h2, x, **kw)
    keep = torch.ones(80, dtype=torch.bool, device=DEV)
    keep[[7, 50]] = False
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1][keep], clean[1][keep])
    assert got[1][7].isnan().all()
    dy, dxn = rnd(80, D, seed=5), rnd(80, D, seed=6)
    dy2 = dy.clone()
    dy2[7, 3] = float("nan")
    a = ops.gated_norm_bwd(dy, dxn, h, clean[0], clean[2], clean[3], **kw)
    b = ops.gated_norm_bwd(dy2, dxn, h, clean[0], clean[2], clean[3], **kw)
    keep[50] = True
    assert torch.equal(a.dx[keep], b.dx[keep]) and torch.equal(a.dh[keep], b.dh[keep]) and b.dx[7].isnan().all()
    assert torch.equal(a.dshift[1], b.dshift[1]) and torch.equal(a.dgate[1], b.dgate[1])
    assert b.dshift[0, 3].isnan() and b.dshift[0].isnan().sum() == 1 and b.dgate[0].isnan().all()


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("D", [64, 768, 4096])
def test_strides_and_in_place(ops, D, stream):
    """Rows of wider tensors, vectors that are columns of one modulation, results over their inputs; what lies around stays."""
    G, R = 3, 11
    M = G * R
    h, x, kw = make(G, R, D, stream, "pnGM", seed=9)
    mod = torch.zeros(G, 3 * D + 8, dtype=BF16, device=DEV)
    views = [mod[:, i * D:(i + 1) * D].copy_(kw[k]) for i, k in enumerate(("gate", "scale", "shift"))]
    kv = {**kw, "gate": views[0], "scale": views[1], "shift": views[2]}
    want = ops.gated_norm_fwd(h, x, **kw)

    def wide(t, fill=9.0):
        buf = torch.full((M + 2, D + 24), fill, dtype=t.dtype, device=DEV)
        return buf, buf[1:M + 1, 8:D + 8].copy_(t)
    hb, hv = wide(h)
    xb, xv = wide(x)
    yb, yv = wide(torch.zeros_like(want[1]))
    got = ops.gated_norm_fwd(hv, xv, x_out=xv, y=yv, **kv)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0] is xv and got[1] is yv
    dy, dxn = rnd(M, D, seed=50), rnd(M, D, dtype=stream, seed=51)
    gw = ops.gated_norm_bwd(dy, dxn, h, *[want[0], want[2], want[3]], **kw)
    db, dyv = wide(dy)
    nb, dxv = wide(dxn)
    gg = ops.gated_norm_bwd(dyv, dxv, hv, xv, got[2], got[3], dh=hv, dx=dxv, **kv)
    assert all(torch.equal(a, b) for a, b in zip(gg, gw)) and gg.dh is hv and gg.dx is dxv
    for buf, v in ((hb, hv), (xb, xv), (yb, yv), (db, dyv), (nb, dxv)):
        v.fill_(9.0)
        assert (buf == 9.0).all()


def test_no_rows(ops):
    h, x, kw = make(1, 0, 64, BF16, "pngm")
    x_new, y, rh, rx = ops.gated_norm_fwd(h, x, **kw)
    assert x_new.shape == y.shape == (0, 64)
    g = ops.gated_norm_bwd(y, x_new, h, x_new, rh, rx, **kw)
    assert g.dh.shape == (0, 64) and not g.dw_post.any() and not g.dgate.any()


def test_gradient_against_differences(ops):
    """Each gradient along a direction against central differences of the formula in 64 bits (their error: step^2 times the third
    derivative, here below 1e-6 of the value); the kernel's own error is the sum of the bounds above along the direction."""
    G, R, D = 2, 5, 64
    h, x, kw = make(G, R, D, F32, "pnGM", seed=13)
    x_new, y, rh, rx = ops.gated_norm_fwd(h, x, **kw)
    dy, dxn = rnd(G * R, D, seed=50), rnd(G * R, D, dtype=F32, seed=51)
    g = ops.gated_norm_bwd(dy, dxn, h, x_new, rh, rx, **kw)
    base = {k: kw[k].double() for k in ("w_post", "w_pre", "gate", "scale", "shift")}
    base.update(h=h.double(), x=x.double())
    # the stream as stored, so that the point is the kernel's: x_new = x + add(h)
    rep = lambda v: v.repeat_interleave(R, 0)  # noqa: E731
    norm = lambda t, w: t * torch.rsqrt(t.square().mean(1, keepdim=True) + EPS) * w  # noqa: E731
    off = x_new.double() - (base["x"] + 0.7 * rep(base["gate"]) * norm(base["h"], base["w_post"]))

    def loss(b):
        xn = b["x"] + 0.7 * rep(b["gate"]) * norm(b["h"], b["w_post"]) + off
        yy = norm(xn, b["w_pre"]) * (1 + rep(b["scale"])) + rep(b["shift"])
        return (xn * dxn.double()).sum() + (yy * dy.double()).sum()
    for name, grad in [("h", g.dh), ("x", g.dx), ("w_post", g.dw_post), ("w_pre", g.dw_pre), ("gate", g.dgate),
                       ("scale", g.dscale), ("shift", g.dshift)]:
        for seed in (1, 2):
            e = rnd(*base[name].shape, dtype=F32, seed=seed).double()
            st = 1e-4
            fd = (loss({**base, name: base[name] + st * e}) - loss({**base, name: base[name] - st * e})) / (2 * st)
            an = (grad.double() * e).sum()
            tol = (grad.double() * e).abs().sum() * (2.0 ** -8 if grad.dtype == BF16 else 2.0 ** -16) + 1e-3
            assert abs(an - fd) <= tol, (name, an.item(), fd.item(), tol.item())


@pytest.mark.parametrize("D", [768, 4096])
def test_streams_graphs_and_repeats(ops, D):
    G, R = 4, 70
    ins = [make(G, R, D, BF16, "pnGM", seed=100 * i) for i in range(3)]
    dys, dxns = [rnd(G * R, D, seed=60 + i) for i in range(3)], [rnd(G * R, D, seed=70 + i) for i in range(3)]

    def step(h, x, kw, dy, dxn):
        f = ops.gated_norm_fwd(h, x, **kw)
        return [*f, *ops.gated_norm_bwd(dy, dxn, h, f[0], f[2], f[3], **kw)]
    want = [step(*i, dy, dxn) for i, dy, dxn in zip(ins, dys, dxns)]
    assert all(torch.equal(a, b) for a, b in zip(step(*ins[0], dys[0], dxns[0]), want[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*ins[1], dys[1], dxns[1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    h, x, dy, dxn = (t.clone() for t in (ins[0][0], ins[0][1], dys[0], dxns[0]))
    kw = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in ins[0][2].items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(h, x, kw, dy, dxn)
    for i in (0, 1, 2, 0):
        for a, b in zip((h, x, dy, dxn), (ins[i][0], ins[i][1], dys[i], dxns[i])):
            a.copy_(b)
        for k, v in ins[i][2].items():
            if isinstance(v, torch.Tensor):
                kw[k].copy_(v)
        graph.replay()
        step(*ins[(i + 1) % 3], dys[0], dxns[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want[i]))


def test_far_offsets(ops):
    """Rows whose byte offsets pass 32 bits."""
    M, D = 40, 64
    h, x, kw = make(2, M // 2, D, BF16, "pnGM", seed=2)
    want = ops.gated_norm_fwd(h, x, **kw)
    buf = torch.zeros(M, 1 << 26, dtype=BF16, device=DEV)  # 5.4 GB
    v = [buf[:, 4096 * i:4096 * i + D] for i in range(6)]
    got = ops.gated_norm_fwd(v[0].copy_(h), v[1].copy_(x), x_out=v[2], y=v[3], **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    dy, dxn = rnd(M, D, seed=50), rnd(M, D, seed=51)
    a = ops.gated_norm_bwd(dy, dxn, h, want[0], want[2], want[3], **kw)
    b = ops.gated_norm_bwd(v[4].copy_(dy), v[5].copy_(dxn), v[0], v[2], got[2], got[3], dh=v[1], dx=v[3], **kw)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_more_rows_than_blocks(ops):
    """2^28 + 40 rows of 8 columns, 16 to a block: more than one round of them per block; sampled rows against 64 bits, the
    whole by a second half that repeats the first."""
    half_rows, D = (1 << 27) + 20, 8
    h = torch.empty(2, half_rows, D, dtype=BF16, device=DEV)
    x = torch.empty_like(h)
    g = torch.Generator(DEV).manual_seed(3)
    for t in (h, x):
        t[0].normal_(generator=g)
        t[1].copy_(t[0])
    w = 1 + rnd(D, seed=4, scale=0.2)
    x_new, y, rh, rx = ops.gated_norm_fwd(h.view(-1, D), x.view(-1, D), w_post=w, w_pre=w, eps=EPS, x_out=x.view(-1, D))
    for t in (x_new, y, rh, rx):
        a, b = t.view(2, -1)
        assert torch.equal(a, b)
    at = torch.randint(half_rows, (4096,), device=DEV, generator=g)
    u = h[0, at].double()
    r = torch.rsqrt(u.square().mean(1, keepdim=True) + EPS)
    ok(rh[:half_rows][at], r[:, 0], E1 * r[:, 0], "rstd_post")
    xs = x_new.view(2, half_rows, D)[0, at].double()
    r = torch.rsqrt(xs.square().mean(1, keepdim=True) + EPS)
    ok(rx[:half_rows][at], r[:, 0], E1 * r[:, 0], "rstd_pre")
    ref = xs * r * w.double()
    ok(y.view(2, half_rows, D)[0, at], ref, 2.0 ** -8 * ref.abs() * 1.01 + E1 * ref.abs(), "y")


@pytest.mark.parametrize("D", [8, 72, 648, 1288, 2568, 10232])
@pytest.mark.parametrize("name", ["w_post", "gate", "w_pre", "scale"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("R", [5, 1])
def test_not_finite_vectors(ops, D, name, bad, R):
    """An infinity or a NaN in a vector's last value, at widths that leave lanes behind the row: forward and backward give what
    the formula gives, finite where it is finite, a NaN where it is one, the same infinity elsewhere."""
    G = 2
    h, x, kw = make(G, R, D, F32, "pnGM", seed=5)
    kw[name] = kw[name].clone()
    kw[name][..., -1] = bad
    vec = {k: rows(kw[k], G, R) for k in ("w_post", "w_pre", "gate", "scale", "shift")}

    def same(got, ref, what):
        assert torch.equal(got.isnan().cpu(), ref.isnan().cpu()), what
        inf = ref.isinf()
        assert torch.equal(got.double()[inf], ref[inf]) and torch.isfinite(got[torch.isfinite(ref)]).all(), what
    u = h.double() * torch.rsqrt(h.double().square().mean(1, keepdim=True) + EPS) * vec["w_post"] * vec["gate"]
    xn = x.double() + 0.7 * u
    n = xn * torch.rsqrt(xn.square().mean(1, keepdim=True) + EPS)
    x_new, y, rh, rx = ops.gated_norm_fwd(h, x, eps=EPS, **kw)
    same(x_new, xn, "x_new")
    same(y, n * vec["w_pre"] * (1 + vec["scale"]) + vec["shift"], "y")
    # backward, at a finite stream
    xf = x.double()
    r, rr = torch.rsqrt(h.double().square().mean(1, keepdim=True) + EPS), torch.rsqrt(xf.square().mean(1, keepdim=True) + EPS)
    dy, dxn = rnd(G * R, D, seed=50), rnd(G * R, D, dtype=F32, seed=51)
    got = ops.gated_norm_bwd(dy, dxn, h, x, r[:, 0].float(), rr[:, 0].float(), **kw)
    n, v = xf * rr, h.double() * r
    dn = dy.double() * (1 + vec["scale"]) * vec["w_pre"]
    dX = dxn.double() + rr * (dn - n * (dn * n).mean(1, keepdim=True))
    dv = 0.7 * vec["gate"] * vec["w_post"] * dX
    same(got.dx, dX, "dx")
    same(got.dh, r * (dv - v * (dv * v).mean(1, keepdim=True)), "dh")
    P, Q = ((t * u).view(G, R, D).sum(1) for t, u in ((dy.double(), n), (dX, v)))
    wide = {k: kw[k].double() for k in ("w_post", "w_pre", "gate", "scale")}
    for k, ref in (("dscale", wide["w_pre"] * P), ("dw_pre", ((1 + wide["scale"]) * P).sum(0)), ("dgate", 0.7 * wide["w_post"] * Q),
                   ("dw_post", (0.7 * wide["gate"] * Q).sum(0)), ("dshift", dy.double().view(G, R, D).sum(1))):
        same(getattr(got, k), ref, k)


def passes(ops, G, R, D):
    """Passes of the backward's blocks over their rows, from the workspace: blocks per group x 3 sums x D x 4 bytes."""
    blocks = ops.call("vpt_gated_norm_bwd_workspace", G, R, D) // (12 * G * D)
    at_once = 16 if D <= 384 else 4 if D <= 1536 else 1
    return -(-(-(-R // blocks)) // at_once)


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("G,R,D,opts", [(1, 17000, 64, "pnGM"), (3, 11003, 136, "pngm"), (3, 1401, 768, "pnGM"), (2, 1537, 768, "pG"),
                                        (2, 1031, 1280, "pngM"), (5, 823, 1288, "nM"), (2, 1111, 2048, "pnGM"), (3, 301, 4096, "pnGm"),
                                        (1, 601, 10240, "pnGM"), (7, 601, 768, "pnGM")])
def test_blocks_of_several_passes(ops, G, R, D, stream, opts):
    """Rows enough that a block goes over several of them: sums kept from pass to pass, a last pass short of rows, groups that
    end within a block's pass; forward and backward, with and without the stream's own gradient."""
    assert passes(ops, G, R, D) >= 2
    h, x, kw = make(G, R, D, stream, opts, seed=R)
    x_new, y, rh, rx = check_fwd(ops, h, x, kw)
    dy = rnd(G * R, D, seed=51) if y is not None else None
    dxn = rnd(G * R, D, dtype=stream, seed=50)
    got = check_bwd(ops, h, x_new, rh, rx, kw, dxn, dy)
    again = ops.gated_norm_bwd(dy, dxn, h, x_new, rh, rx, **kw)
    assert all(a is b or torch.equal(a, b) for a, b in zip(got, again))
    if y is not None:
        check_bwd(ops, h, x_new, rh, rx, kw, None, dy)


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("G,R,D", [(1, 17000, 64), (3, 1401, 768), (2, 1111, 2048)])
def test_several_passes_strided_in_place(ops, G, R, D, stream):
    """The same over rows of wider tensors, results over their inputs, and what lies around stays."""
    assert passes(ops, G, R, D) >= 2
    M = G * R
    h, x, kw = make(G, R, D, stream, "pnGM", seed=9)
    want = ops.gated_norm_fwd(h, x, **kw)
    dy, dxn = rnd(M, D, seed=50), rnd(M, D, dtype=stream, seed=51)
    grads = ops.gated_norm_bwd(dy, dxn, h, want[0], want[2], want[3], **kw)

    def wide(t):
        buf = torch.full((M + 2, D + 24), 9.0, dtype=t.dtype, device=DEV)
        return buf, buf[1:M + 1, 8:D + 8].copy_(t)
    (hb, hv), (xb, xv), (db, dv), (nb, nv) = wide(h), wide(x), wide(dy), wide(dxn)
    f = ops.gated_norm_fwd(hv, xv, x_out=xv, **kw)
    assert all(torch.equal(a, b) for a, b in zip(f, want))
    got = ops.gated_norm_bwd(dv, nv, hv, xv, f[2], f[3], dh=hv, dx=nv, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    for buf, v in ((hb, hv), (xb, xv), (db, dv), (nb, nv)):
        v.fill_(9.0)
        assert (buf == 9.0).all()
