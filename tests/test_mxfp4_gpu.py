"""MXFP4 quantisation, dequantisation and products on the GPU against definitions in 64 bits.

Tolerances. Quantisation and dequantisation are exact: codes, scales and values have to be equal. A product of two codes and
scales is exact in f32, so a result differs from the 64-bit one by the f32 additions, each off by at most one unit in the last
place of the running sum (2^-23 of it, rounding or cutting off), K + 3 of them over sums that never pass
S = sum |a||b| + |bias| + |resid|: (K + 3) 2^-23 S; a bf16 output adds half a step, 2^-8 |result| (eps / 2)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64)


@pytest.fixture(scope="module")
def m():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from vpt import mxfp4, ops
    return ops, mxfp4


def rnd(*shape, dtype=BF16, seed=0, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if spread:
        x = x * torch.exp2((torch.randn(*shape, generator=g) * spread).round())
    return x.to(dtype).to(DEV)


def reference(x):
    """(codes [M, Kp] as numbers 0 .. 15, scale bytes [M, Kp / 32], values f64 [M, K]) of the definition, on the CPU."""
    x = x.detach().cpu().double()
    M, K = x.shape
    Kp = -(-K // 128) * 128
    p = torch.zeros(M, Kp, dtype=F64)
    p[:, :K] = x
    p = p.view(M, Kp // 32, 32)
    top = p.abs().amax(2, keepdim=True)  # a NaN stays a NaN
    bad = ~torch.isfinite(p).all(2, keepdim=True)
    safe = torch.where(bad | (top == 0), torch.ones_like(top), top)
    e = torch.frexp(safe).exponent - 3
    e = torch.where(top == 0, torch.full_like(e, -127), e).clamp(-127, 127)
    a = torch.where(bad, torch.zeros_like(p), p.abs()) * torch.exp2(-e.double())
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    q = (torch.round(a / step) * step).clamp(max=6)
    code = torch.searchsorted(GRID, q) + 8 * torch.signbit(p).long()
    value = torch.where(bad, torch.full_like(q, float("nan")), q * torch.exp2(e.double()) * torch.where(torch.signbit(p), -1.0, 1.0))
    s = torch.where(bad, torch.full_like(e, 255), e + 127).squeeze(2)
    return code.view(M, Kp), s, value.view(M, Kp)[:, :K], bad


def unpack(codes):
    return torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1).cpu().long()


def check_quantize(ops, x):
    codes, scales = ops.mxfp4_quantize(x)
    code, s, value, bad = reference(x)
    assert torch.equal(scales.cpu().long(), s.long())
    good = (~bad).expand(-1, -1, 32).reshape(code.shape)
    assert torch.equal(unpack(codes)[good], code[good])
    for dtype in (BF16, F32):
        back = ops.mxfp4_dequantize(codes, scales, x.shape[1], dtype=dtype).cpu().double()
        assert torch.equal(back.isnan(), value.isnan())
        assert torch.equal(back.nan_to_num(7.0), value.nan_to_num(7.0))
    return codes, scales


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 100), (7, 128), (4, 129), (64, 768), (77, 1000),
                                 (1, 5120), (129, 264)])
def test_quantize(m, dtype, M, K):
    check_quantize(m[0], rnd(M, K, dtype=dtype, seed=M + K, spread=3.0))


def test_quantize_every_bf16(m):
    """Every bf16 bit pattern, shuffled over blocks (blocks with an infinity or a NaN read back as NaN), and every pattern
    next to values that set its block's scale: all roundings, ties included, at every distance from the largest value."""
    bits = torch.arange(65536, dtype=torch.int32)
    perm = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(1))].to(torch.int16).view(BF16)
    check_quantize(m[0], perm.view(512, 128).to(DEV))
    fin = bits.to(torch.int16).view(BF16)
    fin = fin[torch.isfinite(fin.float())]
    order = fin[fin.float().abs().argsort(stable=True)]  # neighbours in size share blocks
    check_quantize(m[0], order[: len(order) // 128 * 128].view(-1, 128).to(DEV))


def test_quantize_ties_and_limits(m):
    """Midpoints of the grid and their f32 neighbours, saturation, signs, zeros, denormals, the largest finite values."""
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.99, 6.0, 0.0, -0.0, 4.0, 0.5, 1.0, 3.0])
    up, dn = torch.nextafter(mid, mid + 9), torch.nextafter(mid, mid - 9)
    row = torch.cat([mid, up[:8], dn[:8]]).clamp(-7.99, 7.99)
    row[8] = 7.99  # the block's scale is 1
    rows = torch.stack([row, -row] * 3) * torch.exp2(torch.tensor([0, 0, 100, -100, -124, 120.])).view(6, 1)
    check_quantize(m[0], rows.to(DEV))
    tiny = torch.zeros(4, 64)
    tiny[0, 3] = 2.0 ** -126
    tiny[1, 40] = -(2.0 ** -149)
    tiny[2, 0] = 1.5 * 2.0 ** -125
    tiny[3, 5] = 2.0 ** -123
    check_quantize(m[0], tiny.to(DEV))
    big = torch.full((2, 32), torch.finfo(F32).max)
    big[1] = -torch.finfo(BF16).max
    check_quantize(m[0], big.to(DEV))


def test_quantize_not_finite(m):
    x = rnd(6, 160, dtype=F32, seed=3)
    x[0, 5] = float("inf")
    x[1, 40] = float("nan")
    x[2, 159] = float("-inf")
    x[3] = float("nan")
    codes, scales = check_quantize(m[0], x)
    assert (scales == 255).sum().item() == 1 + 1 + 1 + 5


@pytest.mark.parametrize("K,pad", [(96, 8), (96, 3), (100, 1), (33, 0)])
def test_strided_and_unaligned(m, K, pad):
    """Rows in a wider buffer, at offsets that 16-byte loads cannot take; what lies around outputs stays as it was."""
    ops, _ = m
    wide = rnd(9, K + pad + 3, seed=K)
    for x in (wide[:, :K], wide[:, 1:K + 1], wide[::2, 3:K + 3], wide[4:5, 2:K + 2]):
        codes, scales = check_quantize(ops, x)
        M = x.shape[0]
        C = torch.full((M, codes.shape[1] + 32), 0xAB, dtype=torch.uint8, device=DEV)
        S = torch.full((M, scales.shape[1] + 4), 0xCD, dtype=torch.uint8, device=DEV)
        ops.mxfp4_quantize(x, C[:, 16:-16], S[:, :-4])
        assert torch.equal(C[:, 16:-16], codes) and torch.equal(S[:, :-4], scales)
        assert (C[:, :16] == 0xAB).all() and (C[:, -16:] == 0xAB).all() and (S[:, -4:] == 0xCD).all()
        for dtype in (BF16, F32):
            out = torch.full((M + 2, K + 5), 3.0, dtype=dtype, device=DEV)
            ops.mxfp4_dequantize(C[:, 16:-16], S[:, :-4], K, out=out[1:M + 1, 2:K + 2])
            assert torch.equal(out[1:M + 1, 2:K + 2], ops.mxfp4_dequantize(codes, scales, K, dtype=dtype))
            out[1:M + 1, 2:K + 2] = 3.0
            assert (out == 3.0).all()


def test_dequantize_every_code(m):
    codes = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(4, 64).repeat(64, 1).to(DEV)
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(256, 1).expand(256, 4).contiguous().to(DEV)
    got = m[0].mxfp4_dequantize(codes, scales, 128, dtype=F32).cpu()
    c = unpack(codes)
    want = GRID[c % 8] * torch.where(c >= 8, -1.0, 1.0) * torch.exp2(torch.arange(256, dtype=F64) - 127).view(256, 1)
    assert got[255].isnan().all() and torch.equal(got[:255].double(), want[:255].float().double())
    assert torch.equal(torch.signbit(got[:255]), c[:255] >= 8)
    b = m[0].mxfp4_dequantize(codes, scales, 128)
    assert torch.equal(b[:255].float().cpu(), got[:255])


def product(m, M, N, K, seed=0, bias=True, resid=True, out_dtype=BF16, spread=1.0):
    ops, mxfp4 = m
    x, wt = rnd(M, K, seed=seed, spread=spread), rnd(N, K, dtype=F32, seed=seed + 1, spread=spread)
    b = rnd(N, seed=seed + 2) if bias else None
    r = rnd(M, N, seed=seed + 3) if resid else None
    w = mxfp4.MXFP4Weight.quantize(wt)
    y = ops.linear_mxfp4(x, w, bias=b, resid=r, out_dtype=out_dtype)
    return x, wt, b, r, w, y


def close(y, x, wt, b, r):
    xv, wv = reference(x)[2].to(y.device), reference(wt)[2].to(y.device)
    ref, top = xv @ wv.t(), xv.abs() @ wv.abs().t()
    for t in (b, r):
        if t is not None:
            ref, top = ref + t.double(), top + t.double().abs()
    tol = (x.shape[1] + 3) * 2.0 ** -23 * top + (2.0 ** -8 * ref.abs() if y.dtype == BF16 else 0) + 1e-37
    bad = (y.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} past the bound, worst {((y.double() - ref).abs() / tol).max().item():.2f}"


SIZES = [(1, 1, 1), (1, 8, 32), (1, 2304, 768), (2, 7, 33), (3, 64, 128), (15, 100, 129), (16, 16, 256), (17, 130, 500),
         (33, 40, 1024), (64, 1280, 640), (65, 8, 96), (77, 640, 2048), (100, 129, 300), (128, 128, 128), (129, 127, 384),
         (200, 264, 160), (255, 256, 511), (257, 384, 640), (300, 1000, 72), (513, 136, 896)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("out_dtype", [BF16, F32])
def test_linear(m, M, N, K, out_dtype):
    x, wt, b, r, w, y = product(m, M, N, K, seed=M + N + K, out_dtype=out_dtype)
    assert y.dtype == out_dtype and tuple(y.shape) == (M, N)
    close(y, x, wt, b, r)


@pytest.mark.parametrize("M", [1, 4, 16, 17, 50, 64, 65, 300])
@pytest.mark.parametrize("bias,resid", [(False, False), (True, False), (False, True)])
def test_linear_without(m, M, bias, resid):
    x, wt, b, r, _, y = product(m, M, 96, 288, seed=9, bias=bias, resid=resid)
    close(y, x, wt, b, r)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_linear_input_types(m, dtype):
    ops, mxfp4 = m
    for M in (1, 20, 150):
        x, wt = rnd(M, 200, dtype=dtype, seed=4, spread=1.0), rnd(72, 200, dtype=dtype, seed=5)
        close(ops.linear_mxfp4(x, mxfp4.MXFP4Weight.quantize(wt)), x, wt, None, None)


@pytest.mark.parametrize("M", [1, 16, 40, 200])
def test_exact_small_integers(m, M):
    """Values of the grid under scales of one: every partial sum is a multiple of 1/4 below 2^24, so the result is exact."""
    ops, mxfp4 = m
    g = torch.Generator().manual_seed(M)
    def pick(rows, K):
        v = torch.cat([GRID, -GRID])[torch.randint(0, 16, (rows, K), generator=g)]
        v[:, ::32] = 4.0  # the block's scale
        return v.float().to(DEV)
    x, wt = pick(M, 416), pick(136, 416)
    y = ops.linear_mxfp4(x, mxfp4.MXFP4Weight.quantize(wt), out_dtype=F32)
    assert torch.equal(y.double(), x.double() @ wt.double().t())


@pytest.mark.parametrize("M", [1, 16, 33, 140])
def test_not_finite_blocks(m, M):
    """A NaN or an infinity in one row of x, or of W, reaches that row, or column, of the result and nothing else."""
    ops, mxfp4 = m
    K, N = 300, 140
    x, wt = rnd(M, K, seed=1), rnd(N, K, seed=2)
    clean = ops.linear_mxfp4(x, mxfp4.MXFP4Weight.quantize(wt))
    x2, w2 = x.clone(), wt.clone()
    x2[M // 2, 299] = float("inf")
    w2[77, 3] = float("nan")
    y = ops.linear_mxfp4(x2, mxfp4.MXFP4Weight.quantize(w2))
    mask = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    mask[M // 2] = True
    mask[:, 77] = True
    assert torch.equal(y.isnan(), mask) and torch.equal(y[~mask], clean[~mask])


@pytest.mark.parametrize("M", [1, 2, 30, 130])
@pytest.mark.parametrize("N,off", [(136, 8), (136, 1), (99, 0)])
def test_strided_operands(m, M, N, off):
    """Outputs and residuals inside wider buffers (what is around stays), codes with gaps, the residual in place."""
    ops, mxfp4 = m
    K = 160
    x, wt, b, r, w, y = product(m, M, N, K, seed=N)
    buf = torch.full((M + 2, N + 24), 5.0, dtype=BF16, device=DEV)
    out = buf[1:M + 1, off:off + N]
    rbuf = torch.zeros(M, N + 11, dtype=BF16, device=DEV)
    rr = rbuf[:, 3:N + 3].copy_(r)
    xx = torch.zeros(M, K + 7, dtype=BF16, device=DEV)[:, 5:K + 5].copy_(x)
    gap = lambda t, n: torch.zeros(t.shape[0], t.shape[1] + n, dtype=torch.uint8, device=DEV)[:, n:].copy_(t)  # noqa: E731
    w2 = mxfp4.MXFP4Weight(gap(w.codes, 48), gap(w.scales, 4), w.shape)
    assert torch.equal(ops.linear_mxfp4(xx, w2, bias=b, resid=rr, out=out), y)
    out.fill_(5.0)
    assert (buf == 5.0).all()
    assert torch.equal(ops.linear_mxfp4(x, w, bias=b, resid=r, out=r), y) and torch.equal(r, y)


def test_no_rows(m):
    ops, mxfp4 = m
    w = mxfp4.MXFP4Weight.quantize(rnd(24, 40))
    x = torch.empty(0, 40, dtype=BF16, device=DEV)
    assert ops.mxfp4_quantize(x)[0].shape == (0, 64)
    assert ops.linear_mxfp4(x, w).shape == (0, 24)
    assert ops.linear_mxfp4_dgrad(torch.empty(0, 24, dtype=BF16, device=DEV), w).shape == (0, 40)
    assert ops.mxfp4_dequantize(*ops.mxfp4_quantize(x), 40).shape == (0, 40)


@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (1, 64, 136), (5, 128, 256), (130, 264, 520), (300, 1280, 640), (1, 2304, 768),
                                   (16, 2304, 768), (3, 4096, 264), (64, 5120, 136), (129, 1032, 1000), (700, 2304, 768),
                                   (3000, 2304, 768), (40, 136, 5120)])
def test_dgrad(m, M, N, K):
    """dx = dy . W against 64 bits, bf16 inputs (the bound of the module's head with N additions)."""
    ops, mxfp4 = m
    wt, dy = rnd(N, K, seed=1), rnd(M, N, seed=2)
    w = mxfp4.MXFP4Weight.quantize(wt)
    dx = ops.linear_mxfp4_dgrad(dy, w).double()
    wv = reference(wt)[2].to(DEV)
    ref, top = dy.double() @ wv, dy.double().abs() @ wv.abs()
    assert ((dx - ref).abs() <= (N + 3) * 2.0 ** -23 * top + 2.0 ** -8 * ref.abs()).all()
    wide = torch.zeros(M + 1, N + 8, dtype=BF16, device=DEV)
    wide[:M, 8:].copy_(dy)
    assert torch.equal(ops.linear_mxfp4_dgrad(wide[:M, 8:], w).double(), dx)
    assert torch.equal(ops.linear_mxfp4_dgrad(dy, w, out=torch.empty(M, K, dtype=BF16, device=DEV)).double(), dx)
    buf = torch.full((M + 2, K + 16), 3.0, dtype=BF16, device=DEV)
    into = ops.linear_mxfp4_dgrad(dy, w, out=buf[1:M + 1, 8:K + 8]).double()
    assert ((into - ref).abs() <= (N + 3) * 2.0 ** -23 * top + 2.0 ** -8 * ref.abs()).all()
    buf[1:M + 1, 8:K + 8] = 3.0
    assert (buf == 3.0).all()


def test_dgrad_against_differences(m):
    """y is linear in an input that the quantisation keeps: with x and x + h e on the grid, (y(x + h e) - y(x)) . dy / h is
    dx . e up to the f32 sums of y and the bf16 rounding of dx."""
    ops, mxfp4 = m
    M, N, K = 3, 40, 64
    w = mxfp4.MXFP4Weight.quantize(rnd(N, K, seed=5))
    dy = rnd(M, N, seed=6)
    dx = ops.linear_mxfp4_dgrad(dy, w).double()
    x = torch.full((M, K), 4.0, dtype=BF16, device=DEV)
    x[:, 1::2] = 1.0
    y0 = ops.linear_mxfp4(x, w, out_dtype=F32).double()
    wv = w.dequantize().double()
    for k in (1, 33, 63):
        x1 = x.clone()
        x1[:, k] = 2.0
        d = (ops.linear_mxfp4(x1, w, out_dtype=F32).double() - y0) * dy.double()
        tol = 2 * (K + 3) * 2.0 ** -23 * ((4.0 * wv.abs().sum(1)) * dy.double().abs()).sum(1) + 2.0 ** -7 * dx[:, k].abs() + \
            (N + 3) * 2.0 ** -23 * (dy.double().abs() @ wv.abs())[:, k]
        assert ((d.sum(1) - dx[:, k]).abs() <= tol).all()


def test_far_offsets(m):
    """More than 2^31 values, and rows more than 2^32 bytes apart."""
    ops, mxfp4 = m
    M, K = 70001, 32768
    x = torch.zeros(M, K, dtype=BF16, device=DEV)
    rows = [0, 1, 65535, 65536, 70000]
    x[rows] = rnd(len(rows), K, seed=8, spread=2.0)
    codes, scales = ops.mxfp4_quantize(x)
    want = ops.mxfp4_quantize(x[rows].contiguous())
    assert torch.equal(codes[rows], want[0]) and torch.equal(scales[rows], want[1])
    assert not codes[2:65535].any() and not codes[65537:70000].any()
    back = ops.mxfp4_dequantize(codes, scales, K, out=x)
    assert torch.equal(back[rows], ops.mxfp4_dequantize(*want, K)) and not back[65537:70000].any()
    del codes, scales, back, x
    buf = torch.zeros(21, 1 << 28, dtype=torch.uint8, device=DEV)  # 5.6 GB
    for M in (20, 1):
        x, wt, b, _, w, y = product(m, M, 48, 256, seed=M, resid=False)
        a, s = ops.mxfp4_quantize(x)
        far, fars = buf[1:M + 1, :128].copy_(a), buf[1:M + 1, 4096:4104].copy_(s)
        out = buf[1:M + 1, 8192:8192 + 96].view(BF16)
        assert torch.equal(ops.gemm_mxfp4(far, fars, w, out, bias=b), y)
    wfar = mxfp4.MXFP4Weight(buf[:20, 256:384].copy_(w.codes[:20]), buf[:20, 512:520].copy_(w.scales[:20]), (20, 256))
    for M in (1, 40, 130):
        x = rnd(M, 256, seed=M)
        assert torch.equal(ops.linear_mxfp4(x, wfar), ops.linear_mxfp4(x, w)[:, :20])


@pytest.mark.parametrize("M", [1, 24, 200])
def test_streams_and_graphs(m, M):
    """On another stream, and captured: replays with new inputs give the eager result, the eager work between them too."""
    ops, mxfp4 = m
    N, K = 264, 640
    w = mxfp4.MXFP4Weight.quantize(rnd(N, K, seed=1))
    b = rnd(N, seed=2)
    xs = [rnd(M, K, seed=10 + i) for i in range(4)]
    dys = [rnd(M, N, seed=20 + i) for i in range(4)]
    want = [(ops.linear_mxfp4(x, w, bias=b), ops.linear_mxfp4_dgrad(dy, w)) for x, dy in zip(xs, dys)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_mxfp4(xs[0], w, bias=b)
    torch.cuda.synchronize()
    assert torch.equal(got, want[0][0])
    x, dy = xs[0].clone(), dys[0].clone()
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, dx = ops.linear_mxfp4(x, w, bias=b), ops.linear_mxfp4_dgrad(dy, w)
    with torch.cuda.graph(g2):
        y2 = ops.linear_mxfp4(x, w)
    for i in range(4):
        x.copy_(xs[i])
        dy.copy_(dys[i])
        g.replay()
        g2.replay()
        eager = ops.linear_mxfp4(xs[i - 1], w, bias=b)
        torch.cuda.synchronize()
        assert torch.equal(y, want[i][0]) and torch.equal(dx, want[i][1]) and torch.equal(eager, want[i - 1][0])
        assert torch.equal(y2, ops.linear_mxfp4(xs[i], w))


def test_repeatable(m):
    ops, mxfp4 = m
    for M in (1, 30, 300):
        x, _, b, r, w, y = product(m, M, 520, 1000, seed=M)
        assert all(torch.equal(ops.linear_mxfp4(x, w, bias=b, resid=r), y) for _ in range(5))


@pytest.mark.parametrize("M,N,K", [(M, N, K) for M, N in [(4100, 4104), (8193, 2049), (1200, 1032), (1100, 515)]
                                   for K in (100, 256, 300, 512, 600, 768, 800, 1100)] +
                         [(4000, 4000, K) for K in (2945, 3100, 3200, 3300, 3456)] + [(3900, 4001, 3100)])
def test_linear_large(m, M, N, K):
    """Grids of every tile kernel (256 x 256 from 24 steps along K on), one step to nine, edges in both directions."""
    x, wt, b, r, w, y = product(m, M, N, K, seed=K, out_dtype=F32 if K == 300 else BF16)
    close(y, x, wt, b, r)
    assert torch.equal(m[0].linear_mxfp4(x, w, bias=b, resid=r, out_dtype=y.dtype), y)


@pytest.mark.parametrize("M,N,K", [(8200, 3080, 200), (8200, 3080, 640), (8200, 3073, 640), (33000, 4100, 128), (33000, 4104, 128),
                                   (33000, 4104, 3100), (70000, 2000, 520)])
def test_linear_sampled(m, M, N, K):
    """Large results, also past what the cache holds, checked on rows of every part of them."""
    ops, mxfp4 = m
    x = rnd(512, K, seed=K, spread=1.0).repeat(-(-M // 512), 1)[:M].contiguous()
    wt, b, r = rnd(N, K, dtype=F32, seed=1), rnd(N, seed=2), rnd(M, N, seed=3)
    y = ops.linear_mxfp4(x, mxfp4.MXFP4Weight.quantize(wt), bias=b, resid=r)
    at = torch.tensor(sorted({0, 1, 15, 16, 127, 128, 255, 256, 4095, M // 2, M // 2 + 77, M - 257, M - 130, M - 17, M - 1}), device=DEV)
    close(y[at], x[at], wt, b, r[at])
    part = ops.linear_mxfp4(x[:512], mxfp4.MXFP4Weight.quantize(wt), bias=b).double()  # every row: the same product, other bits of r
    for lo in range(0, M, 512):
        n = min(512, M - lo)
        d = (y[lo:lo + n].double() - r[lo:lo + n].double() - part[:n]).abs()
        assert (d <= 2.0 ** -7 * (part[:n].abs() + r[lo:lo + n].double().abs()) + 1e-3).all()


@pytest.mark.parametrize("M", [1, 3, 8, 16, 17, 40, 64, 65, 100, 300, 1000])
@pytest.mark.parametrize("K", [96, 768, 2048])
def test_linear_is_quantize_and_gemm(m, M, K):
    ops, mxfp4 = m
    x, w, b = rnd(M, K, seed=M), mxfp4.MXFP4Weight.quantize(rnd(200, K, seed=K)), rnd(200, seed=5)
    assert torch.equal(ops.linear_mxfp4(x, w, bias=b), ops.gemm_mxfp4(*ops.mxfp4_quantize(x), w, bias=b))


def test_dgrad_refuses_far_rows(m):
    ops, mxfp4 = m
    w = mxfp4.MXFP4Weight.quantize(rnd(16, 64))
    dy = torch.zeros(2, 1 << 23, dtype=BF16, device=DEV)[:, :16]
    with pytest.raises(ValueError, match="apart"):
        ops.linear_mxfp4_dgrad(dy, w)


@pytest.mark.parametrize("M,N,K", [(300, 200, 300), (8200, 3080, 200), (4000, 4000, 3100)])
@pytest.mark.parametrize("off", [0, 1, 2, 4])
def test_bias_anywhere(m, M, N, K, off):
    """A bias that starts at any place of its buffer, at every tile kernel, the buffer ending with it."""
    ops, mxfp4 = m
    x, w = rnd(M, K, seed=1), mxfp4.MXFP4Weight.quantize(rnd(N, K, seed=2))
    b = rnd(N, seed=3)
    at = torch.empty(off + N, dtype=BF16, device=DEV)[off:].copy_(b)
    zero = ops.linear_mxfp4(x, w, out_dtype=F32)
    assert torch.equal(ops.linear_mxfp4(x, w, bias=at, out_dtype=F32), zero + b.float())


# Sizes that the dispatch sends to each kernel of many rows, the last tile 4 or 8 rows high: 128 x 128 tiles (two steps along K,
# whose scales go straight to registers, and five), 256 x 128 tiles, the 256 x 256 ring (24 steps and more).
TILES = [(260, 1000, 200), (260, 1000, 520), (8200, 3080, 648), (3848, 4000, 3100)]
GUARD = 300  # more rows than a tile has: what a tile would write behind row M lies in these


def framed(M, N, dtype, off, fill):
    """(buffer, [M, N] view of it): GUARD rows before and behind, columns beside."""
    buf = torch.full((M + 2 * GUARD, N + 24), fill, dtype=dtype, device=DEV)
    return buf, buf[GUARD:GUARD + M, off:off + N]


def only_inside(buf, M, N, off, fill):
    buf[GUARD:GUARD + M, off:off + N] = fill
    return bool((buf == fill).all())


def gaps(t, n):
    return torch.full((t.shape[0], t.shape[1] + n), 255, dtype=torch.uint8, device=DEV)[:, n:].copy_(t)


@pytest.mark.parametrize("M,N,K", TILES)
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("off", [8, 1])
def test_tiles_write_their_rows_alone(m, M, N, K, out_dtype, off):
    """16-byte stores (off 8) and element by element (off 1): the result of a dense call, nothing written behind the last row,
    before the first or beside the columns, nothing but the residual's own rows read; codes and scales with gaps; in place."""
    ops, mxfp4 = m
    x, wt, b, r, w, y = product(m, M, N, K, seed=N, out_dtype=out_dtype)
    close(y, x, wt, b, r)
    a, s = ops.mxfp4_quantize(x)
    wg = mxfp4.MXFP4Weight(gaps(w.codes, 48), gaps(w.scales, 4), w.shape)
    buf, out = framed(M, N, out_dtype, off, 5.0)
    rbuf, rr = framed(M, N, BF16, off, float("nan"))
    rr.copy_(r)
    assert torch.equal(ops.gemm_mxfp4(gaps(a, 16), gaps(s, 4), wg, out, bias=b, resid=rr), y)
    assert only_inside(buf, M, N, off, 5.0)
    assert torch.equal(ops.linear_mxfp4(x, wg, bias=b, resid=rr, out=out), y) and only_inside(buf, M, N, off, 5.0)
    rbuf.fill_(3.0)
    if out_dtype == BF16:
        rr.copy_(r)
        assert torch.equal(ops.linear_mxfp4(x, w, bias=b, resid=rr, out=rr), y)
    assert only_inside(rbuf, M, N, off, 3.0)
    y0 = ops.linear_mxfp4(x, w, out_dtype=out_dtype)
    assert torch.equal(ops.linear_mxfp4(x, w, out=out), y0) and only_inside(buf, M, N, off, 5.0)


@pytest.mark.parametrize("M,N,K", TILES)
def test_tiles_not_finite_blocks(m, M, N, K):
    """As test_not_finite_blocks: scale byte 255 in every of a row's 4-step groups, in A and in W."""
    ops, mxfp4 = m
    x, wt = rnd(M, K, seed=1), rnd(N, K, seed=2)
    clean = ops.linear_mxfp4(x, mxfp4.MXFP4Weight.quantize(wt))
    x2, w2 = x.clone(), wt.clone()
    rows = [0, 77, M // 2, M - 3, M - 1]
    cols = [3, N // 2, N - 1]
    for i, r in enumerate(rows):
        x2[r, (i * K) // len(rows) + 5] = float("inf") if i % 2 else float("nan")
    for i, c in enumerate(cols):
        w2[c, K - 1 - (i * K) // len(cols)] = float("nan") if i % 2 else float("-inf")
    y = ops.linear_mxfp4(x2, mxfp4.MXFP4Weight.quantize(w2))
    mask = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    mask[rows] = True
    mask[:, cols] = True
    assert torch.equal(y.isnan(), mask) and torch.equal(y[~mask], clean[~mask])


@pytest.mark.parametrize("M,N,K", TILES)
def test_tiles_exact_integers(m, M, N, K):
    """As test_exact_small_integers: multiples of 1/4 whose sums stay below 2^24 / 4 (36 per product, K <= 3100)."""
    ops, mxfp4 = m
    g = torch.Generator().manual_seed(M)

    def pick(rows, cols):
        v = torch.cat([GRID, -GRID])[torch.randint(0, 16, (rows, cols), generator=g)]
        v[:, ::32] = 4.0  # the block's scale
        return v.float().to(DEV)
    x, wt = pick(M, K), pick(N, K)
    y = ops.linear_mxfp4(x, mxfp4.MXFP4Weight.quantize(wt), out_dtype=F32)
    assert torch.equal(y.double(), x.double() @ wt.double().t())


@pytest.mark.parametrize("M,N,K", TILES)
@pytest.mark.parametrize("dtype", [F16, F32])
def test_tiles_input_types(m, M, N, K, dtype):
    ops, mxfp4 = m
    x, wt = rnd(M, K, dtype=dtype, seed=4, spread=1.0), rnd(N, K, dtype=dtype, seed=5)
    w = mxfp4.MXFP4Weight.quantize(wt)
    y = ops.linear_mxfp4(x, w)
    close(y, x, wt, None, None)
    assert torch.equal(y, ops.gemm_mxfp4(*ops.mxfp4_quantize(x), w))


@pytest.mark.parametrize("M,N,K", TILES)
def test_tiles_streams_and_graphs(m, M, N, K):
    """On another stream, captured twice, replayed with new inputs between eager calls: the same bits."""
    ops, mxfp4 = m
    w, b = mxfp4.MXFP4Weight.quantize(rnd(N, K, seed=1)), rnd(N, seed=2)
    xs, r = [rnd(M, K, seed=10 + i) for i in range(3)], rnd(M, N, seed=3)
    want = [ops.linear_mxfp4(x, w, bias=b, resid=r) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_mxfp4(xs[0], w, bias=b, resid=r)
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    x, graphs, res = xs[0].clone(), [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            res.append(ops.linear_mxfp4(x, w, bias=b, resid=r))
    for i in (1, 2, 0):
        x.copy_(xs[i])
        [g.replay() for g in graphs]
        eager = ops.linear_mxfp4(xs[i - 1], w, bias=b, resid=r)
        torch.cuda.synchronize()
        assert all(torch.equal(t, want[i]) for t in res) and torch.equal(eager, want[i - 1])


@pytest.mark.parametrize("what", ["out", "out f32", "resid", "codes", "scales", "W codes", "W scales"])
def test_rows_far_apart(m, what):
    """An operand whose rows lie 4 MB apart and more, at a size past the few-row kernel's: the kernel with 64-bit addresses,
    against the definition, and what lies around the result stays."""
    ops, mxfp4 = m
    M, N, K = (2000, 140, 300) if what[0] == "W" else (130, 1500, 300)
    dtype = F32 if what == "out f32" else BF16
    x, wt, b, r = rnd(M, K, seed=1, spread=1.0), rnd(N, K, dtype=F32, seed=2, spread=1.0), rnd(N, seed=3), rnd(M, N, seed=4)
    w = mxfp4.MXFP4Weight.quantize(wt)
    a, s = ops.mxfp4_quantize(x)
    c, ws = w.codes, w.scales

    def far(t, fill):
        """t in rows of 4 MB of one buffer, a row of it free before and behind."""
        buf = torch.full((t.shape[0] + 2, (1 << 22) // t.element_size()), fill, dtype=t.dtype, device=DEV)
        return buf, buf[1:-1, 64:64 + t.shape[1]].copy_(t)
    buf, out = None, None
    if what.startswith("out"):
        buf, out = far(torch.zeros(M, N, dtype=dtype, device=DEV), 5.0)
    elif what == "resid":
        _, r = far(r, float("nan"))
    elif what == "codes":
        _, a = far(a, 255)
    elif what == "scales":
        _, s = far(s, 255)
    elif what == "W codes":
        _, c = far(c, 255)
    else:
        _, ws = far(ws, 255)
    y = ops.gemm_mxfp4(a, s, mxfp4.MXFP4Weight(c, ws, (N, K)), out, bias=b, resid=r, out_dtype=dtype)
    close(y, x, wt, b, r)
    assert torch.equal(ops.gemm_mxfp4(a, s, mxfp4.MXFP4Weight(c, ws, (N, K)), out, bias=b, resid=r, out_dtype=dtype), y)
    if buf is not None:
        out.fill_(5.0)
        assert (buf == 5.0).all()


def test_more_rows_than_a_launch(m):
    """2^27 + 9 rows of 128 values: quantisation and dequantisation take several launches; the rows around their border and the
    last ones as on their own, zeros elsewhere."""
    ops, _ = m
    M, K = (1 << 27) + 9, 128
    x = torch.zeros(M, K, dtype=BF16, device=DEV)  # 34 GB
    at = torch.tensor([0, 1, (1 << 26) + 3, (1 << 27) - 2, (1 << 27) - 1, 1 << 27, (1 << 27) + 1, M - 1], device=DEV)
    x[at] = rnd(len(at), K, seed=8, spread=2.0)
    codes, scales = ops.mxfp4_quantize(x)
    want = ops.mxfp4_quantize(x[at].contiguous())
    assert torch.equal(codes[at], want[0]) and torch.equal(scales[at], want[1])
    back = ops.mxfp4_dequantize(codes, scales, K, out=x)
    assert torch.equal(back[at], ops.mxfp4_dequantize(*want, K))
    back[at], codes[at], scales[at] = 0, 0, 0
    assert not any(t.any() for part in (back, codes, scales) for t in part.split(1 << 24))


@pytest.mark.parametrize("K", [130, 3100])
def test_streamed_tiles_write_their_rows_alone(m, K):
    """Results past what the cache holds (stores that leave no copy in it), from the 256 x 128 tiles and from the ring: as above."""
    ops, mxfp4 = m
    M, N = 16392, 4104
    x, w, b = rnd(M, K, seed=1, spread=1.0), mxfp4.MXFP4Weight.quantize(rnd(N, K, dtype=F32, seed=2)), rnd(N, seed=3)
    y = ops.linear_mxfp4(x, w, bias=b, out_dtype=F32)
    at = torch.tensor([0, 15, 16, 255, 256, 4095, M // 2, M - 9, M - 8, M - 1], device=DEV)
    close(y[at], x[at], rnd(N, K, dtype=F32, seed=2), b, None)
    buf, out = framed(M, N, F32, 8, 5.0)
    assert torch.equal(ops.linear_mxfp4(x, w, bias=b, out=out), y)
    assert only_inside(buf, M, N, 8, 5.0)
