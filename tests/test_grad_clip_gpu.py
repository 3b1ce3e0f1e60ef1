"""The global norm of many gradient tensors and their clipping on the GPU, against 64 bits and torch.nn.utils.

Tolerances. The squares are added in 64 bits, so the norm is off by its rounding to f32 (2^-24 relative); the coefficient by 2^-24
once more, the product by 2^-24, and storing by half a step of the type (bf16 2^-8, f16 2^-11, and half of f16's smallest
step, 2^-25, where values are that small)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
STEP = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


@pytest.fixture(scope="module")
def optim():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from vpt import optim as _optim
    return _optim


def rnd(n, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    shape = n if isinstance(n, tuple) else (n,)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def norm64(grads):
    return math.sqrt(sum(g.double().square().sum().item() for g in grads))


def check(grads, before, norm, max_norm, value=None):
    want = norm64(before)
    if norm is not None:
        assert abs(norm.item() - want) <= 2.0 ** -23 * want
    coef = 1.0 if max_norm is None else min(1.0, max_norm / (want + 1e-6))
    for g, b in zip(grads, before):
        ref = b.double() * coef
        if value is not None:
            ref = ref.clamp(-value, value)
        tol = (STEP[g.dtype] * 1.01 + 2.0 ** -22) * ref.abs() + (2.0 ** -25 if g.dtype == F16 else 1e-44)
        assert ((g.double() - ref).abs() <= tol).all()


SIZES = [[1], [7], [64, 1, 0, 3], [16384], [16385, 16383, 5], [40000, 2, 100003], [1 << 21, 33], list(range(0, 400, 3))]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("over", [True, False])
def test_clip(optim, sizes, dtype, over):
    grads = [rnd(n, dtype, seed=i) for i, n in enumerate(sizes)]
    before = [g.clone() for g in grads]
    n = norm64(before)
    limit = n / 3 if over else n * 1.5 + 1
    out = [torch.full_like(g, 9.0) for g in grads]
    norm = optim.GradClip(grads, out=out).clip(limit)
    check(out, before, norm, limit)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    again = optim.GradClip(grads).clip(limit)
    assert torch.equal(again, norm) and all(torch.equal(a, b) for a, b in zip(grads, out))
    assert over or all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("align", [0, 1, 2, 3, 4, 7])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_alignment_and_neighbours(optim, align, dtype):
    """Tensors that start anywhere; what lies before and behind them stays."""
    for n in (1, 5, 8, 255, 4099, 20001):
        buf = torch.full((n + 32,), 7.0, dtype=dtype, device=DEV)
        ob = torch.full((n + 32,), 8.0, dtype=dtype, device=DEV)
        g, o = buf[align:align + n], ob[16 - align:16 - align + n]
        g.copy_(rnd(n, dtype, seed=n))
        before = g.clone()
        norm = optim.GradClip([g], out=[o]).clip(0.5, 0.01)
        check([o], [before], norm, 0.5, 0.01)
        norm = optim.GradClip([g]).clip(0.5, 0.01)
        check([g], [before], norm, 0.5, 0.01)
        assert torch.equal(g, o)
        g.fill_(7.0)
        o.fill_(8.0)
        assert (buf == 7.0).all() and (ob == 8.0).all()


def test_mixed_types_and_layouts(optim):
    grads = [rnd((33, 20), BF16, 1), rnd((5, 7, 9), F32, 2).permute(2, 0, 1), rnd((64, 48), F16, 3).t(), rnd(0, F32),
             rnd(1, F32, 4).view(()), rnd((3, 1, 5), BF16, 5).transpose(0, 2)]
    before = [g.clone() for g in grads]
    c = optim.GradClip(grads)
    assert torch.equal(c.norm(), c.norm()) and all(torch.equal(a, b) for a, b in zip(grads, before))
    norm = c.clip(2.0, 0.05)
    check(grads, before, norm, 2.0, 0.05)
    assert c.clip(clip_value=0.01) is None
    assert all(g.abs().max() <= 0.0101 for g in grads if g.numel())


def test_value_only(optim):
    g = rnd(3001, seed=1)
    g[5], g[6], g[7] = float("inf"), float("-inf"), float("nan")
    want = g.clamp(-0.3, 0.3)
    optim.GradClip([g]).clip(clip_value=0.3)
    assert torch.equal(g.nan_to_num(9.0), want.nan_to_num(9.0)) and g[7].isnan()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_not_finite(optim, bad):
    """As torch.nn.utils.clip_grad_norm_: a NaN norm makes everything NaN; an infinite one zero, and NaN where it was infinite."""
    grads = [rnd(100, seed=1), rnd(20000, BF16, seed=2)]
    grads[1][777] = bad
    ps = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g.clone()
    want = torch.nn.utils.clip_grad_norm_(ps, 1.0)
    norm = optim.GradClip(grads).clip(1.0)
    assert torch.equal(norm.isnan(), want.isnan()) and (norm.isnan() or norm.item() == want.item())
    for p, g in zip(ps, grads):
        assert torch.equal(g.isnan(), p.grad.isnan()) and torch.equal(g.nan_to_num(5.0), p.grad.nan_to_num(5.0))
    for p, g in zip(ps, [torch.ones(100, device=DEV), torch.full((20000,), bad, dtype=BF16, device=DEV)]):
        p.grad = g
    with pytest.raises(RuntimeError, match="not finite"):
        optim.clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert torch.equal(ps[0].grad, torch.ones(100, device=DEV))


@pytest.mark.parametrize("scale", [1e-30, 1e-20, 1e18, 1e30])
def test_far_from_one(optim, scale):
    """Squares that leave the range of f32."""
    for dtype in (F32, BF16):
        grads = [rnd(5000, dtype, seed=1, scale=scale), rnd(17, dtype, seed=2, scale=scale)]
        before = [g.clone() for g in grads]
        out = [torch.zeros_like(g) for g in grads]
        n = norm64(before)
        check(out, before, optim.GradClip(grads, out=out).clip(n / 2), n / 2)


def test_as_torch(optim):
    ps = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in [(300, 70), (70,), (1,), (129, 65)]]
    ps.append(torch.nn.Parameter(torch.zeros(5, device=DEV)))  # without a gradient
    for i, p in enumerate(ps[:-1]):
        p.grad = rnd(tuple(p.shape), seed=i)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = None if p.grad is None else p.grad.clone()
    a = optim.clip_grad_norm_(ps, 1.0, clip_value=0.02)
    b = torch.nn.utils.clip_grad_norm_(qs, 1.0)
    torch.nn.utils.clip_grad_value_(qs, 0.02)
    assert abs(a.item() - b.item()) <= 1e-6 * b.item()
    for p, q in zip(ps[:-1], qs):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)
    assert ps[-1].grad is None
    one = torch.nn.Parameter(torch.zeros(3, device=DEV))
    one.grad = torch.full((3,), 2.0, device=DEV)
    optim.clip_grad_norm_(one, 1.0)
    assert abs(one.grad.norm().item() - 1.0) < 1e-5


def test_the_same_bits_streams_and_graphs(optim):
    sizes = [30000, 5, 70001, 16384, 0, 999]
    data = [[rnd(n, BF16, seed=10 * k + i) for i, n in enumerate(sizes)] for k in range(3)]
    grads = [torch.empty_like(g) for g in data[0]]
    out = [torch.empty_like(g) for g in grads]
    c = optim.GradClip(grads, out=out)

    def load(k):
        for g, d in zip(grads, data[k]):
            g.copy_(d)
    want = []
    for k in range(3):
        load(k)
        n = c.clip(1.0)
        want.append((n.clone(), [o.clone() for o in out]))
        assert all(torch.equal(c.clip(1.0), n) for _ in range(3))
    side = torch.cuda.Stream()
    load(0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n = c.clip(1.0)
    torch.cuda.synchronize()
    assert torch.equal(n, want[0][0])
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        na = c.clip(1.0)
    with torch.cuda.graph(b):
        nb = c.norm()
    for k in (1, 2, 0, 1):
        load(k)
        a.replay()
        b.replay()
        eager = optim.GradClip(data[0]).norm()
        torch.cuda.synchronize()
        assert torch.equal(na, want[k][0]) and torch.equal(nb, want[k][0]) and torch.equal(eager, want[0][0])
        assert all(torch.equal(x, y) for x, y in zip(out, want[k][1]))


def test_many_and_none(optim):
    flat = rnd(3000 * 24, BF16, seed=3)
    grads = [flat[24 * i:24 * i + 17] for i in range(3000)]
    before = [g.clone() for g in grads]
    rest = flat.view(3000, 24)[:, 17:].clone()
    check(grads, before, optim.GradClip(grads).clip(1.0), 1.0)
    assert torch.equal(flat.view(3000, 24)[:, 17:], rest)
    assert optim.GradClip([]).clip(1.0).item() == 0.0
    assert optim.GradClip([torch.empty(0, device=DEV)]).norm().item() == 0.0
    optim.GradClip([]).clip(clip_value=1.0)


def test_past_32_bits(optim):
    """One tensor of more than 2^31 values (4.4 GB)."""
    n = (1 << 31) + 12345
    g = torch.zeros(n, dtype=BF16, device=DEV)
    spots = [0, 1, (1 << 31) - 1, 1 << 31, n - 1]
    g[spots] = torch.tensor([3.0, 4.0, 12.0, 84.0, 0.0], dtype=BF16, device=DEV)
    norm = optim.GradClip([g]).clip(8.5)
    assert norm.item() == math.sqrt(9 + 16 + 144 + 84 * 84)
    assert abs(g[1 << 31].item() - 8.4) < 0.04 and abs(g[0].item() - 0.3) < 0.002 and g[2:1000].abs().max().item() == 0


def test_captured_and_the_handle_gone(optim):
    """A graph's replays after its handle went and its memory was asked for again."""
    import gc
    data = [[rnd(n, F32, seed=10 * k + i) for i, n in enumerate((20000, 3, 40001))] for k in range(2)]
    grads = [torch.empty_like(g) for g in data[0]]
    out = [torch.empty_like(g) for g in grads]
    handle = optim.GradClip(grads, out=out)
    want = []
    for d in data:
        [g.copy_(t) for g, t in zip(grads, d)]
        want.append([handle.clip(1.0).clone(), *(o.clone() for o in out)])
    size = handle._table.numel()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = handle.clip(1.0)
    del handle
    gc.collect()
    junk = [torch.full((size,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]
    for k in (0, 1, 0):
        [g.copy_(t) for g, t in zip(grads, data[k])]
        [o.zero_() for o in out]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([norm, *out], want[k]))
    assert all((j == 255).all() for j in junk)


def test_a_gradient_given_other_memory(optim):
    """A handle's table names the memory its tensors had: that stays, and what lies elsewhere is left alone."""
    g = rnd(30000, F32, seed=1)
    handle, first = optim.GradClip([g]), g.detach().clone()
    g.data = torch.full_like(g, 7.0)
    torch.cuda.empty_cache()
    others = [torch.full_like(g, 5.0) for _ in range(8)]
    norm = handle.clip(1.0)
    assert abs(norm.item() - norm64([first])) <= 2.0 ** -23 * norm64([first])
    assert (g == 7.0).all() and all((o == 5.0).all() for o in others)
