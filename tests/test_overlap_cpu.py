"""CPU: results that share memory with what their call reads are refused (a block may write a row before another block has read
it), unless they are the input itself where that is offered. The bytes two strided tensors share, against a count."""

import itertools

import pytest
import torch

BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


@pytest.fixture(scope="module")
def m():
    from vpt import mxfp4, ops
    return ops, mxfp4


def z(*s, d=BF16):
    return torch.zeros(*s, dtype=d)


def test_share_counts_bytes(m):
    """Views of one buffer with equal and other row strides, against the set of their bytes."""
    buf = torch.zeros(400, dtype=U8)
    views = [buf[o:].as_strided((r, c), (s, 1)) for o, r, c, s in itertools.product(
        (0, 3, 16, 40, 111), (1, 2, 5), (1, 4, 9), (9, 16, 40))]
    spots = [{v.data_ptr() + i * v.stride(0) + j for i in range(v.shape[0]) for j in range(v.shape[1])} for v in views]
    for (a, sa), (b, sb) in itertools.product(zip(views, spots), repeat=2):
        assert m[0]._share(a, b) == bool(sa & sb), (a.shape, a.stride(), b.shape, b.stride())
    assert not m[0]._share(buf[:0].view(0, 4), buf.view(40, 10)) and m[0]._share(buf[5:6], buf.view(40, 10))
    wide = torch.zeros(64, dtype=F32)
    assert m[0]._share(wide.view(BF16)[20:24], wide[10:12]) and not m[0]._share(wide.view(BF16)[20:24], wide[12:14])


def refused(fn, what):
    with pytest.raises(ValueError, match=what):
        fn()


def test_mxfp4(m):
    ops, mxfp4 = m
    buf = z(8, 256)
    w = mxfp4.MXFP4Weight(z(64, 64, d=U8), z(64, 4, d=U8), (64, 64))
    x = buf[:, :64]
    refused(lambda: ops.linear_mxfp4(x, w, out=buf[:, 32:96]), "shares memory with x")
    refused(lambda: ops.linear_mxfp4(buf[1:5, :64], w, out=buf[:4, :64]), "shares memory with x")
    refused(lambda: ops.linear_mxfp4(x, w, out=buf[:, 64:128]), "GPU")  # columns beside it: nothing shared
    refused(lambda: ops.linear_mxfp4(x, w, resid=buf[:, 64:128], out=buf[:, 65:129]), "shares memory with resid")
    refused(lambda: ops.linear_mxfp4(x, w, resid=buf[:, 64:128], out=buf[:, 64:128]), "GPU")
    refused(lambda: ops.linear_mxfp4(x, w, bias=buf[0, 96:160], out=buf[:, 64:128]), "shares memory with bias")
    over = torch.as_strided(w.codes.view(BF16), (4, 64), (64, 1))
    refused(lambda: ops.linear_mxfp4(x[:4], w, out=over), "shares memory with W")
    bytes_ = z(16, 512, d=U8)
    a, s = bytes_[:, :64], bytes_[:, 64:68]
    refused(lambda: ops.gemm_mxfp4(a, s, w, out=bytes_.view(BF16)[:, 33:97]), "shares memory with a_scales")
    refused(lambda: ops.gemm_mxfp4(a, s, w, out=bytes_.view(BF16)[:, 16:80]), "shares memory with a_codes")
    refused(lambda: ops.gemm_mxfp4(a, s, w, out=bytes_.view(BF16)[:, 64:128]), "GPU")
    xb = bytes_.view(BF16)[:, :64]
    refused(lambda: ops.mxfp4_quantize(xb, bytes_[:, 64:128], bytes_[:, 256:260]), "shares memory with x")
    refused(lambda: ops.mxfp4_quantize(xb, bytes_[:, 128:192], bytes_[:, 160:164]), "share memory")
    refused(lambda: ops.mxfp4_quantize(xb, bytes_[:, 128:192], bytes_[:, 124:128]), "shares memory with x")
    refused(lambda: ops.mxfp4_dequantize(a, s, 64, out=bytes_.view(BF16)[:, 30:94]), "shares memory with codes")
    refused(lambda: ops.mxfp4_dequantize(a, s, 64, out=bytes_.view(BF16)[:, 33:97]), "shares memory with scales")
    refused(lambda: ops.linear_mxfp4_dgrad(buf[:, :64], w, out=buf[:, 56:120]), "shares memory with dy")
    refused(lambda: ops.linear_mxfp4_dgrad(buf[:, :64], w, out=buf[:, :64]), "shares memory with dy")


def test_gated_norm(m):
    ops = m[0]
    h, x, v = z(6, 64)[:, :16], z(6, 64)[:, :16], z(16)
    hw, xw = h._base, x._base
    ok = dict(w_post=v, w_pre=z(16), gate=z(3, 16), groups=3)
    for kw, what in [(dict(x_out=xw[:, 8:24]), "x_out shares memory with x"), (dict(x_out=x), "GPU"), (dict(x_out=h), "GPU"),
                     (dict(y=hw[:, 8:24]), "y shares memory with h"), (dict(y=h), "GPU"), (dict(x_out=x, y=x), "share memory"),
                     (dict(x_out=xw[:, 16:32], y=xw[:, 24:40]), "share memory"), (dict(x_out=xw[:, 16:32]), "GPU"),
                     (dict(x_out=xw[:, 16:32], gate=xw[:3, 16:32]), "x_out shares memory with gate"),
                     (dict(y=xw[:, 16:32], w_pre=xw[3, 24:40]), "y shares memory with w_pre")]:
        refused(lambda: ops.gated_norm_fwd(h, x, **{**ok, **kw}), what)
    dy, dxn, st = z(6, 16), z(6, 16), z(96, d=F32)
    args = (dy, dxn, h, x, st[:6], z(6, d=F32))
    ok["gate"] = None
    for kw, what in [(dict(dh=h, dx=dxn), "GPU"), (dict(dh=hw[:, 8:24]), "dh shares memory with h"), (dict(dh=dy, dx=dy), "share memory"),
                     (dict(dx=xw[:, 8:24]), "dx shares memory with x_new"), (dict(dx=dy), "GPU"),
                     (dict(dh=st.view(BF16)[:96].view(6, 16)), "dh shares memory with rstd_post"),
                     (dict(dh=hw[:, 16:32], w_post=hw[2, 16:32]), "dh shares memory with w_post")]:
        refused(lambda: ops.gated_norm_bwd(*args, **{**ok, **kw}), what)
    # without w_pre dx is dx_new itself: dh may not be written over it
    refused(lambda: ops.gated_norm_bwd(None, dxn, h, None, st[:6], None, w_post=v, dh=dxn), "share memory")
    refused(lambda: ops.gated_norm_bwd(None, dxn, h, None, st[:6], None, w_post=v, dh=h), "GPU")
    big = z(6, 64, d=F32)
    f = (dy, big[:, :16], h, big[:, 16:32], st[:6], z(6, d=F32))
    refused(lambda: ops.gated_norm_bwd(*f, **ok, dh=big.view(BF16)[:, 24:40]), "dh shares memory with dx_new")
    refused(lambda: ops.gated_norm_bwd(*f, **ok, dx=big[:, 32:48]), "GPU")
