"""The new operators as they are used: one fine-tuning step of a gated block over an MXFP4 base, with its gradients clipped, and a
LoRA target on such a base."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6


@pytest.fixture(scope="module")
def m():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from vpt import mxfp4, ops, optim
    return ops, mxfp4, optim


def rnd(*shape, dtype=BF16, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


class Block:
    """h, x -> x1 = x + gate0 post0(h), y1 = pre0(x1) modulated -> silu(y1 W1 + b1) W2 -> x2, y2 likewise."""

    def __init__(self, m, G, D, F):
        self.ops, mx, self.optim = m
        self.G, self.D = G, D
        self.w = [mx.MXFP4Weight.quantize(rnd(F, D, seed=1, scale=D ** -0.5)), mx.MXFP4Weight.quantize(rnd(D, F, seed=2, scale=F ** -0.5))]
        self.b1 = rnd(F, seed=3, scale=0.1)
        mod = rnd(G, 6 * D, seed=4, scale=0.5)
        col = lambda i: mod[:, i * D:(i + 1) * D]  # noqa: E731
        self.norms = [dict(w_post=1 + rnd(D, seed=5 + i, scale=0.2), w_pre=1 + rnd(D, seed=7 + i, scale=0.2), gate=col(3 * i),
                           scale=col(3 * i + 1), shift=col(3 * i + 2), groups=G, resid_scale=0.8) for i in (0, 1)]

    def step(self, h, x, dx2, dy2, max_norm):
        ops, (n0, n1) = self.ops, self.norms
        x1, y1, *r1 = ops.gated_norm_fwd(h, x, eps=EPS, **n0)
        a = ops.linear_mxfp4(y1, self.w[0], bias=self.b1)
        s = ops.silu(a, torch.empty_like(a))
        u = ops.linear_mxfp4(s, self.w[1])
        x2, y2, *r2 = ops.gated_norm_fwd(u, x1, eps=EPS, **n1)
        g1 = ops.gated_norm_bwd(dy2, dx2, u, x2, *r2, **n1)
        ds = ops.linear_mxfp4_dgrad(g1.dh, self.w[1])
        da = ops.silu_bwd(ds, a, torch.empty_like(a))
        g0 = ops.gated_norm_bwd(ops.linear_mxfp4_dgrad(da, self.w[0]), g1.dx, h, x1, *r1, **n0)
        grads = [t for g in (g0, g1) for t in g[2:]]
        if not hasattr(self, "grads"):  # as a program keeps them: gradient buffers and the plan that clips them
            self.grads = [torch.empty_like(t) for t in grads]
            self.clip = self.optim.GradClip(self.grads)
        raw = [t.clone() for t in grads]
        for buf, t in zip(self.grads, grads):
            buf.copy_(t)
        norm = self.clip.clip(max_norm)
        return dict(x2=x2, y2=y2, dh=g0.dh, dx=g0.dx, norm=norm, clipped=[b.clone() for b in self.grads], raw=raw,
                    mid=(x1, y1, a, s, u, x2))


def norm64(t, w):
    return t * torch.rsqrt(t.square().mean(1, keepdim=True) + EPS) * w


@pytest.mark.parametrize("G,R,D,F", [(2, 33, 128, 264), (3, 170, 768, 2048)])
def test_step_against_64_bits(m, G, R, D, F):
    """The gradients of the whole chain against 64-bit autograd of its formulas, taken at the step's own values (each stored tensor
    enters as it is, the quantisation's gradient goes straight through). The five gradients stored in bf16 on the way are
    off by at most 2^-8 of their norm each, and each map between has gradients of random, uncorrelated rows, which keep
    relative norms: below 8 * 2^-8 in all."""
    blk = Block(m, G, D, F)
    h, x = rnd(G * R, D, seed=20, scale=3.0), rnd(G * R, D, seed=21, scale=2.0)
    dx2, dy2 = rnd(G * R, D, seed=22), rnd(G * R, D, seed=23)
    got = blk.step(h, x, dx2, dy2, 0.5)
    x1, y1, a, s, u, x2 = (t.double() for t in got["mid"])
    W = [w.dequantize().double() for w in blk.w]

    def at(value, stored):  # the stored value, the formula's gradient
        return value + (stored - value).detach()
    leaf = {"h": h.double().requires_grad_(), "x": x.double().requires_grad_()}
    vecs = [{k: n[k].double().requires_grad_() for k in ("w_post", "w_pre", "gate", "scale", "shift")} for n in blk.norms]
    rep = lambda v: v.repeat_interleave(R, 0)  # noqa: E731

    def gated(hh, xx, v, stored):
        xn = at(xx + 0.8 * rep(v["gate"]) * norm64(hh, v["w_post"]), stored)
        return xn, norm64(xn, v["w_pre"]) * (1 + rep(v["scale"])) + rep(v["shift"])
    x1f, y1f = gated(leaf["h"], leaf["x"], vecs[0], x1)
    af = at(at(y1f, y1) @ W[0].t() + blk.b1.double(), a)
    uf = at(torch.nn.functional.silu(af) @ W[1].t(), u)
    x2f, y2f = gated(uf, x1f, vecs[1], x2)
    order = [v[k] for v in vecs for k in ("w_post", "w_pre", "gate", "scale", "shift")]
    want = torch.autograd.grad((x2f * dx2.double()).sum() + (y2f * dy2.double()).sum(), [leaf["h"], leaf["x"], *order])
    rel = lambda p, q: ((p.double() - q).norm() / q.norm()).item()  # noqa: E731
    assert rel(got["y2"], y2f) < 2.0 ** -8 * 1.1 and rel(got["x2"], x2f) < 2.0 ** -8 * 1.1
    for p, q in zip([got["dh"], got["dx"], *got["raw"]], want):
        assert p.shape == q.shape and rel(p, q) < 8 * 2.0 ** -8
    total = torch.cat([t.double().flatten() for t in got["raw"]]).norm()
    assert abs(got["norm"].item() - total.item()) <= 2.0 ** -23 * total.item() and total > 0.5
    for p, q in zip(got["clipped"], got["raw"]):
        torch.testing.assert_close(p.double(), q.double() * (0.5 / (total + 1e-6)), rtol=2.0 ** -22, atol=0)


def test_step_captured(m):
    """The step in a graph: replays with new inputs, eager steps between them, give the eager step's bits."""
    blk = Block(m, 2, 256, 512)
    M = 2 * 150
    ins = [[rnd(M, 256, seed=30 + 4 * k + i) for i in range(4)] for k in range(3)]
    flat = lambda r: [r["x2"], r["y2"], r["dh"], r["dx"], r["norm"], *r["clipped"]]  # noqa: E731
    want = [[t.clone() for t in flat(blk.step(*i, 1.0))] for i in ins]
    buf = [t.clone() for t in ins[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = flat(blk.step(*buf, 1.0))
    for k in (1, 2, 0, 1):
        for b, t in zip(buf, ins[k]):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, want[k]))
        eager = flat(blk.step(*ins[k - 1], 1.0))
        assert all(torch.equal(p, q) for p, q in zip(eager, want[k - 1]))


def test_two_streams_at_once(m):
    """Two steps of two blocks under way on two streams share nothing."""
    blks = [Block(m, 2, 384, 768) for _ in range(2)]
    ins = [[rnd(2 * 200, 384, seed=60 + 4 * k + i) for i in range(4)] for k in range(2)]
    flat = lambda r: [r["x2"], r["y2"], r["dh"], r["dx"], r["norm"], *r["clipped"]]  # noqa: E731
    want = [[t.clone() for t in flat(b.step(*i, 1.0))] for b, i in zip(blks, ins)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        out = []
        for b, i, s in zip(blks, ins, streams):
            with torch.cuda.stream(s):
                out.append(flat(b.step(*i, 1.0)))
        torch.cuda.synchronize()
        for r, w in zip(out, want):
            assert all(torch.equal(p, q) for p, q in zip(r, w))


@pytest.mark.parametrize("N,K", [(640, 2048), (1280, 1280), (200, 264)])
def test_lora_linear_on_mxfp4(m, N, K):
    """LoRALinearNF4 over an MXFP4 base: dequantised per call and kept resident give the same bits; output and gradients against
    64 bits. Roundings to bf16 on the way: ds / vs and the result, for (200, 264), whose sizes the fused kernels do not
    take, also the LoRA term and its sum: at most 4 half steps of values no larger than the result's terms: 4 * 2^-8."""
    from vpt.sdxl import LoRALinearNF4
    ops, mx, _ = m
    w = mx.MXFP4Weight.quantize(rnd(N, K, seed=1, scale=K ** -0.5))
    down, up, bias = rnd(16, K, seed=2, scale=0.05), rnd(N, 16, seed=3, scale=0.05), rnd(N, seed=4, scale=0.1)
    x, dy = rnd(300, K, seed=5), rnd(300, N, seed=6)
    out = []
    for mode in ("dequant", "resident"):
        lin = LoRALinearNF4(w, bias, down, up, alpha=16.0, rank=16, base_mode=mode)
        out.append((lin.forward(x), lin.backward(dy), lin.g_up.clone(), lin.g_down.clone()))
    assert all(torch.equal(p, q) for p, q in zip(*out))
    W, X, DY, Dn, Up = (t.double() for t in (w.dequantize(), x, dy, down, up))
    rel = lambda p, q: ((p.double() - q).norm() / q.norm()).item()  # noqa: E731
    y, dx, gu, gd = out[0]
    assert rel(y, X @ W.t() + bias.double() + X @ Dn.t() @ Up.t()) < 4 * 2.0 ** -8
    assert rel(dx, DY @ W + DY @ Up @ Dn) < 4 * 2.0 ** -8
    assert rel(gu, DY.t() @ (X @ Dn.t())) < 4 * 2.0 ** -8 and rel(gd, (DY @ Up).t() @ X) < 4 * 2.0 ** -8
    with pytest.raises(ValueError, match="inline"):
        LoRALinearNF4(w, bias, down, up, alpha=16.0, rank=16, base_mode="inline")


def test_sdxl_block_on_mxfp4(m):
    """A transformer block whose ten bases are MXFP4 gives what it gives on resident bf16 copies of them."""
    from vpt import sdxl
    ops, mx, _ = m
    dim, heads, cdim, rank = 256, 4, 512, 16
    shapes = {t: (dim, cdim if t in ("attn2.to_k", "attn2.to_v") else dim) for t in sdxl.TARGETS}
    shapes["ff.net.0.proj"], shapes["ff.net.2"] = (8 * dim, dim), (dim, 4 * dim)
    sd = {}
    for i, (t, (n, k)) in enumerate(shapes.items()):
        sd[f"{t}.linear.weight"] = mx.MXFP4Weight.quantize(rnd(n, k, seed=100 + i, scale=k ** -0.5))
        if t not in ("attn1.to_q", "attn1.to_k", "attn1.to_v", "attn2.to_q", "attn2.to_k", "attn2.to_v"):
            sd[f"{t}.linear.bias"] = rnd(n, seed=120 + i, scale=0.1)
        sd[f"{t}.lora_down.weight"], sd[f"{t}.lora_up.weight"] = rnd(rank, k, seed=140 + i, scale=0.05), rnd(n, rank, seed=160 + i, scale=0.05)
    for k in ("norm1", "norm2", "norm3"):
        sd[f"{k}.weight"], sd[f"{k}.bias"] = torch.ones(dim, device=DEV), torch.zeros(dim, device=DEV)
    res = []
    for mode in ("dequant", "resident"):
        blk = sdxl.SDXLTransformerBlock(dim, heads, cdim, rank, 16.0, sd)
        for lin in blk.lin.values():
            lin.base_mode = mode
        y = blk.forward(rnd(2 * 80, dim, seed=1), rnd(2 * 20, cdim, seed=2), 2, 80, 20)
        dx, dctx = blk.backward(rnd(2 * 80, dim, seed=3, scale=0.1))
        res.append([y, dx, dctx] + [t.clone() for lin in blk.lin.values() for t in (lin.g_up, lin.g_down)])
    assert all(torch.isfinite(t.float()).all() and t.float().abs().max() > 0 for t in res[0])
    assert all(torch.equal(p, q) for p, q in zip(*res))


@pytest.mark.parametrize("mode", ["dequant", "resident"])
def test_lora_on_two_streams(m, mode):
    """Two LoRA targets of one size over different MXFP4 bases, forward and backward under way on two streams at once: each
    gives what it gives alone (the dequantised bases, split-K slabs and adapter-gradient slabs are a stream's own)."""
    from vpt.sdxl import LoRALinearNF4
    ops, mx, _ = m
    N, K, M = 1280, 5120, 500  # the forward splits its reduction
    lins, ins = [], []
    for k in (0, 1):
        w = mx.MXFP4Weight.quantize(rnd(N, K, seed=10 + k, scale=K ** -0.5))
        lins.append(LoRALinearNF4(w, rnd(N, seed=20 + k), rnd(16, K, seed=30 + k, scale=0.05), rnd(N, 16, seed=40 + k, scale=0.05),
                                  alpha=16.0, rank=16, base_mode=mode))
        ins.append((rnd(M, K, seed=50 + k), rnd(M, N, seed=60 + k)))

    def step(lin, x, dy):
        lin.g_up.zero_()
        lin.g_down.zero_()
        return lin.forward(x), lin.backward(dy), lin.g_up, lin.g_down
    want = [[t.clone() for t in step(lin, *i)] for lin, i in zip(lins, ins)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for lin in lins:
        lin.base.resident = None  # the first use is on the side stream, the next on another
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for lin, i, s in zip(lins, ins, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    out = step(lin, *i)
                got.append(out)
        streams.reverse()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_lora_captured_twice(m):
    """Two graphs of two LoRA targets share no scratch, and an eager call that needs a larger one takes none from them."""
    from vpt.sdxl import LoRALinearNF4
    ops, mx, _ = m
    lins, ins, want, graphs, res = [], [], [], [], []
    for k, (N, K) in enumerate([(1280, 5120), (1280, 5120), (2560, 5120)]):
        w = mx.MXFP4Weight.quantize(rnd(N, K, seed=10 + k, scale=K ** -0.5))
        lins.append(LoRALinearNF4(w, None, rnd(16, K, seed=30 + k, scale=0.05), rnd(N, 16, seed=40 + k, scale=0.05), alpha=16.0,
                                  rank=16, base_mode="dequant"))
        ins.append((rnd(400, K, seed=50 + k), rnd(400, N, seed=60 + k)))

    def step(lin, x, dy):
        lin.g_up.zero_()
        lin.g_down.zero_()
        return lin.forward(x), lin.backward(dy), lin.g_up, lin.g_down
    for lin, i in zip(lins[:2], ins):
        want.append([t.clone() for t in step(lin, *i)])
    for lin, i in zip(lins[:2], ins):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res.append(step(lin, *i))
        graphs.append(g)
    side = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        torch.cuda.synchronize()
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        step(lins[2], *ins[2])
        torch.cuda.synchronize()
        for a, b in zip(res, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
        step(lins[0], *ins[0])


def test_frozen_linear_on_mxfp4(m):
    """A frozen Linear without adapters over an MXFP4 base, both ways against 64 bits: f32 sums and one rounding to bf16."""
    from vpt.sdxl import NF4Linear
    ops, mx, _ = m
    N, K = 320, 640
    w, bias = mx.MXFP4Weight.quantize(rnd(N, K, seed=1, scale=K ** -0.5)), rnd(N, seed=2)
    x, dy = rnd(150, K, seed=3), rnd(150, N, seed=4)
    W = w.dequantize().double()
    for mode in ("dequant", "resident"):
        lin = NF4Linear(w, bias, mode)
        for got, a, b, add in ((lin.forward(x), x, W.t(), bias), (lin.backward(dy), dy, W, None)):
            ref, top = a.double() @ b, a.double().abs() @ b.abs()
            if add is not None:
                ref, top = ref + add.double(), top + add.double().abs()
            assert ((got.double() - ref).abs() <= (a.shape[1] + 3) * 2.0 ** -23 * top + 2.0 ** -8 * ref.abs()).all()


def test_stacks_on_mxfp4(m):
    """Transformer stacks of two widths whose every base is MXFP4: the stacked k / v projections against 64 bits (ds rounded to
    bf16, 2^-8 of it, f32 sums, one rounding of the result), and a step's gradients, dequantised per block and kept."""
    from vpt.sdxl_train import SDXLStacksQLoRA
    ops, mx, _ = m
    res = []
    for mode in ("dequant", "resident"):
        st = SDXLStacksQLoRA(B=2, stacks=[("a", 640, 10, 1, 16), ("b", 1280, 20, 2, 8)], n_ctx=77, seed=3)
        g = torch.Generator(device=DEV).manual_seed(9)
        st.params.copy_((torch.randn(st.params.shape, device=DEV, generator=g) * 0.03).bfloat16())
        blocks = [blk for (_, _, _, s) in st.stacks for blk in s.blocks]
        layers = [p for (_, _, _, s) in st.stacks for p in (s.proj_in, s.proj_out)] + [lin for b in blocks for lin in b.lin.values()]
        for p in layers:
            p.base = mx.MXFP4Weight.quantize(p.base.dequantize())
            p.base_mode = mode
        xs, ctx, gs = st.make_inputs(seed=4)
        st.opt.step = lambda: None
        res.append((st.step(xs, ctx, gs).clone(), st.grads.clone()))
        assert st.precompute_ctx_kv(ctx)
        X = ctx.double()
        for blk in blocks:
            for got, t in zip(blk.ctx_kv, ("attn2.to_k", "attn2.to_v")):
                lin = blk.lin[t]
                W, down, up = (v.double() for v in (lin.base.dequantize(), lin.down, lin.up))
                ds = lin.scale * (X @ down.t())
                ref = X @ W.t() + ds @ up.t()
                tol = 2.0 ** -8 * (ref.abs() + ds.abs() @ up.abs().t()) * 1.01 + \
                    (X.shape[1] + 32) * 2.0 ** -23 * (X.abs() @ W.abs().t() + lin.scale * (X.abs() @ down.abs().t()) @ up.abs().t())
                assert ((got.double() - ref).abs() <= tol).all()
    assert all(torch.equal(p, q) and torch.isfinite(p.float()).all() and p.float().abs().max() > 0 for p, q in zip(*res))


def test_sdxl_block_captured(m):
    """Two transformer blocks on MXFP4 bases, forward and backward captured each in a graph of its own, replayed at once on two
    streams with new inputs while an eager step of a third runs: the eager bits (bases, slabs and tickets are a graph's own)."""
    from vpt import sdxl
    ops, mx, _ = m
    dim, cdim, rank = 256, 512, 16
    shapes = {t: (dim, cdim if t in ("attn2.to_k", "attn2.to_v") else dim) for t in sdxl.TARGETS}
    shapes["ff.net.0.proj"], shapes["ff.net.2"] = (8 * dim, dim), (dim, 4 * dim)

    def block(seed):
        sd = {}
        for i, (t, (n, k)) in enumerate(shapes.items()):
            sd[f"{t}.linear.weight"] = mx.MXFP4Weight.quantize(rnd(n, k, seed=seed + i, scale=k ** -0.5))
            sd[f"{t}.lora_down.weight"], sd[f"{t}.lora_up.weight"] = (rnd(*s, seed=seed + 20 + i, scale=0.05) for s in ((rank, k), (n, rank)))
        for k in ("norm1", "norm2", "norm3"):
            sd[f"{k}.weight"], sd[f"{k}.bias"] = torch.ones(dim, device=DEV), torch.zeros(dim, device=DEV)
        return sdxl.SDXLTransformerBlock(dim, 4, cdim, rank, 16.0, sd)

    def inputs(seed):
        return [rnd(2 * 80, dim, seed=seed), rnd(2 * 20, cdim, seed=seed + 1), rnd(2 * 80, dim, seed=seed + 2, scale=0.1)]

    def step(blk, x, ctx, dy):
        grads = [g for lin in blk.lin.values() for g in (lin.g_up, lin.g_down)]
        for g in grads:
            g.zero_()
        y = blk.forward(x, ctx, 2, 80, 20)
        return [y, *blk.backward(dy), *grads]
    blks, ins = [block(100 * k) for k in range(3)], [[inputs(1000 * k + 10 * i) for i in range(3)] for k in range(2)]
    want = [[[t.clone() for t in step(b, *i)] for i in per] for b, per in zip(blks, ins)]
    third = [t.clone() for t in step(blks[2], *ins[0][0])]
    bufs, graphs, res = [[t.clone() for t in per[0]] for per in ins], [], []
    for b, buf in zip(blks, bufs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            res.append(step(b, *buf))
    streams = [torch.cuda.Stream() for _ in graphs]
    for k in (1, 2, 0, 1):
        for buf, per in zip(bufs, ins):
            for t, v in zip(buf, per[k]):
                t.copy_(v)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = step(blks[2], *ins[0][0])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for r, w in zip(res, want) for p, q in zip(r, w[k]))
        assert all(torch.equal(p, q) for p, q in zip(eager, third))
