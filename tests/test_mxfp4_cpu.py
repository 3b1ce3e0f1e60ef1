"""CPU: the refusals of the MXFP4 entry points (argument checks of vpt.ops / vpt.mxfp4, and of the C ABI, which returns before
any launch)."""

import pytest
import torch

U8 = torch.uint8


@pytest.fixture(scope="module")
def m():
    from vpt import _lib, mxfp4, ops
    return ops, mxfp4, _lib


def parts(rows, K):
    c = (K + 127) // 128
    return torch.zeros(rows, 64 * c, dtype=U8), torch.zeros(rows, 4 * c, dtype=U8)


def test_shapes(m):
    ops, mxfp4, _ = m
    assert ops.mxfp4_shapes(3, 1) == ((3, 64), (3, 4))
    assert ops.mxfp4_shapes(3, 128) == ((3, 64), (3, 4))
    assert ops.mxfp4_shapes(0, 129) == ((0, 128), (0, 8))
    w = mxfp4.MXFP4Weight(*parts(5, 300), (5, 300))
    assert w.shape == (5, 300) and w.numel == 1500


@pytest.mark.parametrize("x,msg", [
    (torch.zeros(2, 3, dtype=torch.float64), "dtype"),
    (torch.zeros(2, 3, dtype=torch.int32), "dtype"),
    (torch.zeros(3), "shape"),
    (torch.zeros(2, 3, 4), "shape"),
    (torch.zeros(4, 3).t(), "contiguous"),
    (torch.zeros(1, 8).expand(4, 8), "overlap"),
    (torch.zeros(2, 0), "K >= 1"),
    (torch.zeros(2, 8), "GPU"),
])
def test_quantize_refuses(m, x, msg):
    with pytest.raises(ValueError, match=msg):
        m[0].mxfp4_quantize(x)


def test_parts_refused(m):
    ops, mxfp4, _ = m
    c, s = parts(5, 300)
    for codes, scales, msg in [(c[:, :64], s, "codes"), (c[:4], s, "codes"), (c, s[:, :4], "scales"),
                               (c.to(torch.int8), s, "dtype"), (c, s.int(), "dtype"),
                               (torch.zeros(5, 200, dtype=U8)[:, :192], s, "16 bytes"),
                               (torch.zeros(5 * 192 + 1, dtype=U8)[1:].view(5, 192), s, "16 bytes"),
                               (c, torch.zeros(5, 13, dtype=U8)[:, :12], "4 bytes"),
                               (c, torch.zeros(61, dtype=U8)[1:].view(5, 12), "4 bytes")]:
        with pytest.raises(ValueError, match=msg):
            mxfp4.MXFP4Weight(codes, scales, (5, 300))
        with pytest.raises(ValueError):
            ops.mxfp4_dequantize(codes, scales, 300, out=torch.zeros(5, 300))
    for shape in [(300,), (0, 300), (5, 0)]:
        with pytest.raises(ValueError):
            mxfp4.MXFP4Weight(c, s, shape)
    with pytest.raises(ValueError, match="codes"):
        mxfp4.MXFP4Weight.from_parts(torch.zeros(5, 149, dtype=U8), torch.zeros(5, 10, dtype=U8), (5, 300))
    with pytest.raises(ValueError, match="scales"):
        mxfp4.MXFP4Weight.from_parts(torch.zeros(5, 150, dtype=U8), torch.zeros(5, 9, dtype=U8), (5, 300))


def test_from_parts_pads(m):
    codes = torch.arange(5 * 51, dtype=torch.int32).to(U8).view(5, 51)
    scales = torch.full((5, 4), 130, dtype=U8)
    w = m[1].MXFP4Weight.from_parts(codes, scales, (5, 101))
    assert torch.equal(w.codes[:, :50], codes[:, :50]) and torch.equal(w.codes[:, 50], codes[:, 50] & 15)
    assert not w.codes[:, 51:].any() and torch.equal(w.scales, scales)
    dense = m[1].MXFP4Weight.from_parts(torch.ones(3, 64, dtype=U8), torch.ones(3, 4, dtype=U8), (3, 128))
    assert dense.codes.shape == (3, 64)


def test_linear_refuses(m):
    ops, mxfp4, _ = m
    w = mxfp4.MXFP4Weight(*parts(16, 64), (16, 64))
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    z = lambda *s, d=torch.bfloat16: torch.zeros(*s, dtype=d)  # noqa: E731
    for kw, msg in [(dict(bias=z(15)), "bias"), (dict(bias=z(16, d=torch.float32)), "bias"), (dict(bias=z(32)[::2]), "bias"),
                    (dict(resid=z(4, 15)), "resid"), (dict(resid=z(4, 16, d=torch.float32)), "resid"),
                    (dict(out=z(4, 15)), "out"), (dict(out=z(4, 16, d=torch.float16)), "out"),
                    (dict(out=z(16, 4).t()), "contiguous"), (dict(out_dtype=torch.float16), "out"), ({}, "GPU")]:
        with pytest.raises(ValueError, match=msg):
            ops.linear_mxfp4(x, w, **kw)
    with pytest.raises(ValueError, match="match"):
        ops.linear_mxfp4(z(4, 63), w)
    with pytest.raises(ValueError, match="dtype"):
        ops.linear_mxfp4(z(4, 64, d=torch.float64), w)
    with pytest.raises(ValueError, match="codes"):
        ops.gemm_mxfp4(*parts(4, 200), w)
    for dy, ww, msg in [(z(4, 15), w, "match"), (z(4, 16, d=torch.float32), w, "dtype"), (z(4, 24)[:, :16], w, "GPU"),
                        (z(4, 20)[:, :16], w, "16 bytes"),
                        (z(4, 12), mxfp4.MXFP4Weight(*parts(12, 64), (12, 64)), "multiples of 8"),
                        (z(4, 16), mxfp4.MXFP4Weight(*parts(16, 60), (16, 60)), "multiples of 8")]:
        with pytest.raises(ValueError, match=msg):
            ops.linear_mxfp4_dgrad(dy, ww)


def test_c_abi_refuses(m):
    lib = m[2].lib
    p, q = 4096, 4096 + 1  # never read: every call below is refused before a launch
    ok_q = [p, 0, 256, 4, 256, p, 128, p, 8, None]
    for i, v in [(0, None), (0, q), (1, 3), (1, -1), (2, 255), (3, -1), (4, 0), (5, None), (5, p + 8), (6, 112), (6, 136),
                 (7, None), (7, p + 2), (8, 4), (8, 10)]:
        a = list(ok_q)
        a[i] = v
        assert lib.vpt_mxfp4_quantize(*a) == 1, (i, v)
        assert b"vpt_mxfp4_quantize" in lib.vpt_last_error_string()
    ok_d = [p, 128, p, 8, 4, 256, p, 256, 0, None]
    for i, v in [(0, None), (0, p + 4), (1, 64), (2, None), (3, 4), (4, -1), (5, 0), (6, None), (6, q), (7, 255)]:
        a = list(ok_d)
        a[i] = v
        assert lib.vpt_mxfp4_dequantize(*a) == 1, (i, v)
    ok_g = [p, 128, p, 8, p, 128, p, 8, p, 64, 4, 64, 256, p, p, 64, 0, None]
    for i, v in [(0, None), (1, 64), (1, 136), (2, None), (3, 4), (4, p + 8), (5, 120), (6, p + 1), (7, 6), (8, None), (8, q),
                 (9, 63), (10, -1), (10, (1 << 30) + 1), (11, 0), (11, (1 << 30) + 1), (12, 0), (13, q), (14, q), (15, 63)]:
        a = list(ok_g)
        a[i] = v
        assert lib.vpt_gemm_mxfp4(*a) == 1, (i, v)
    ok_l = [p, 0, 256, p, 128, p, 8, p, 64, 20, 64, 256, p, p, 64, 0, p, None]
    assert lib.vpt_linear_mxfp4_workspace(20, 256) == 20 * 136 and lib.vpt_linear_mxfp4_workspace(1, 256) == 0
    for rows in (20, 2):  # the form with a workspace and the one without
        for i, v in [(0, None), (0, q), (1, 3), (2, 255), (3, None), (3, p + 8), (4, 64), (4, 136), (5, None), (6, 6), (7, None),
                     (7, q), (8, 63), (9, -1), (10, 0), (11, 0), (12, q), (13, q), (14, 63)]:
            a = list(ok_l)
            a[9] = rows
            a[i] = v
            assert lib.vpt_linear_mxfp4(*a) == 1, (rows, i, v)
    for v in (None, p + 8):
        a = list(ok_l)
        a[16] = v
        assert lib.vpt_linear_mxfp4(*a) == 1
    # nothing to do: no pointer is needed
    assert lib.vpt_mxfp4_quantize(None, 0, 256, 0, 256, None, 128, None, 8, None) == 0
    assert lib.vpt_mxfp4_dequantize(None, 128, None, 8, 0, 256, None, 256, 0, None) == 0
    assert lib.vpt_gemm_mxfp4(None, 128, None, 8, None, 128, None, 8, None, 64, 0, 64, 256, None, None, 0, 0, None) == 0


def test_limits(m):
    """Sizes beyond what a launch covers: more rows than an int holds, and more tiles than a grid."""
    ops, lib = m[0], m[2].lib
    many = torch.zeros(1, 64, dtype=torch.bfloat16, device="meta").expand((1 << 32) + 4, 64)
    for t in (many, torch.empty((1 << 31), 1, dtype=torch.bfloat16, device="meta")):
        with pytest.raises(ValueError, match=r"2\^31"):
            ops.mxfp4_quantize(t)
    p = 4096  # never read
    for M, N in [(64, (1 << 27) + 1), (1 << 30, 257), (1 << 20, 1 << 20)]:
        assert lib.vpt_gemm_mxfp4(p, 64, p, 4, p, 64, p, 4, p, N, M, N, 64, None, None, 0, 0, None) == 1
        assert lib.vpt_linear_mxfp4(p, 0, 64, p, 64, p, 4, p, N, M, N, 64, None, None, 0, 0, p, None) == 1


def test_out_is_not_x(m):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w = type("W", (), dict(shape=(64, 64), codes=torch.zeros(64, 64, dtype=torch.uint8), scales=torch.zeros(64, 4, dtype=torch.uint8)))
    with pytest.raises(ValueError, match="out is x"):
        m[0].linear_mxfp4(x, w, out=x)


def test_numbers_are_no_matrices(m):
    """A tensor without dims is refused as any other wrong shape."""
    ops, mxfp4, _ = m
    w = mxfp4.MXFP4Weight(*parts(16, 64), (16, 64))
    u8, bf = torch.zeros((), dtype=U8), torch.zeros((), dtype=torch.bfloat16)
    for call in (lambda: ops.mxfp4_dequantize(u8, u8, 64), lambda: ops.gemm_mxfp4(u8, u8, w), lambda: ops.linear_mxfp4_dgrad(bf, w),
                 lambda: ops.linear_mxfp4(bf, w), lambda: ops.mxfp4_quantize(bf), lambda: ops.gated_norm_fwd(bf, bf)):
        with pytest.raises(ValueError, match="shape"):
            call()
