"""CPU: the refusals of the gated norms (vpt.ops, C ABI) and of the gradient clipping (vpt.optim, C ABI), and the table of
pieces that GradClip makes."""

import pytest
import torch

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def m():
    from vpt import _lib, ops, optim
    return ops, optim, _lib


def z(*s, d=BF16):
    return torch.zeros(*s, dtype=d)


FWD = dict(h=z(6, 16), x=z(6, 16), w_post=z(16), w_pre=z(16), gate=z(3, 16), scale=z(3, 16), shift=z(16), groups=3)


@pytest.mark.parametrize("change,msg", [
    (dict(), "GPU"), (dict(h=z(6, 16, d=F32)), "dtype"), (dict(h=z(16)), "shape"), (dict(h=z(5, 16), x=z(5, 16)), "groups"),
    (dict(groups=0), "groups"), (dict(h=z(6, 12), x=z(6, 12)), "multiple of 8"),
    (dict(h=z(6, 10248), x=z(6, 10248)), "10240"), (dict(x=z(6, 24)), "shape"), (dict(x=z(6, 16, d=torch.float16)), "dtype"),
    (dict(x=z(16, 6).t()), "contiguous"), (dict(x=z(6, 20)[:, :16]), "16 bytes"), (dict(h=z(97)[1:].view(6, 16)), "16 bytes"),
    (dict(x=z(1, 16).expand(6, 16)), "overlap"), (dict(w_post=z(8)), "w_post"), (dict(w_pre=z(16, d=F32)), "w_pre"),
    (dict(w_pre=z(17)[1:]), "16 bytes"), (dict(gate=z(2, 16)), "gate"), (dict(gate=z(1, 16).expand(3, 16)), "overlap"),
    (dict(gate=z(3, 16, d=F32)), "gate"), (dict(shift=None), "go together"), (dict(w_pre=None), "modulation"),
    (dict(w_pre=None, scale=None, shift=None, y=z(6, 16)), "w_pre"), (dict(y=z(6, 8)), "y"), (dict(x_out=z(6, 16, d=F32)), "x_out"),
    (dict(scale=z(3, 20)[:, :16]), "16 bytes"),
])
def test_fwd_refuses(m, change, msg):
    a = {**FWD, **change}
    with pytest.raises(ValueError, match=msg):
        m[0].gated_norm_fwd(a.pop("h"), a.pop("x"), **a)


BWD = dict(dy=z(6, 16), dx_new=z(6, 16), h=z(6, 16), x_new=z(6, 16), rstd_post=z(6, d=F32), rstd_pre=z(6, d=F32), w_post=z(16),
           w_pre=z(16), gate=z(16), groups=3)


@pytest.mark.parametrize("change,msg", [
    (dict(), "GPU"), (dict(dy=None), "dy"), (dict(w_pre=None, dy=None, dx_new=None), "dx_new"), (dict(w_pre=None), "dy"),
    (dict(rstd_post=None), "rstd_post"), (dict(rstd_pre=None), "rstd_pre"), (dict(rstd_pre=z(6)), "rstd_pre"),
    (dict(rstd_post=z(5, d=F32)), "rstd_post"), (dict(dx_new=z(6, 16, d=F32)), "dx_new"), (dict(x_new=z(6, 8)), "x_new"),
    (dict(dy=z(6, 16, d=F32)), "dy"), (dict(dh=z(6, 16, d=F32)), "dh"), (dict(dx=z(6, 16, d=F32)), "dx"),
    (dict(w_pre=None, dy=None, dx=z(6, 16)), "dx"), (dict(scale=z(16)), "go together"), (dict(groups=4), "groups"),
])
def test_bwd_refuses(m, change, msg):
    a = {**BWD, **change}
    args = [a.pop(k) for k in ("dy", "dx_new", "h", "x_new", "rstd_post", "rstd_pre")]
    with pytest.raises(ValueError, match=msg):
        m[0].gated_norm_bwd(*args, **a)


def test_c_abi_refuses_gated(m):
    lib = m[2].lib
    p = 4096  # never read
    ok = [p, 16, p, 0, 16, p, p, p, 16, p, 16, p, 0, p, 16, p, 16, p, p, 3, 2, 16, 1.0, 1e-6, None]
    for i, v in [(0, None), (0, p + 2), (1, 8), (1, 17), (2, None), (4, 12), (5, p + 8), (7, p + 4), (8, 12), (9, None), (6, None),
                 (13, None), (14, 20), (15, None), (19, -1), (20, 1 << 30), (21, 0), (21, 12), (21, 10248)]:
        a = list(ok)
        a[i] = v
        assert lib.vpt_gated_norm_fwd(*a) == 1, (i, v)
    ok = [p, 16, p, 16, p, 16, p, 0, 16, p, p, p, p, p, 16, p, 16, p, 0, p, 16, p, 16, p, p, p, p, p, p, 3, 2, 16, 1.0, None]
    for i, v in [(0, None), (1, 12), (3, 17), (4, None), (5, 8), (6, None), (9, None), (10, None), (11, None), (12, None),
                 (13, None), (14, 4), (15, None), (19, None), (20, 12), (21, None), (28, None), (28, p + 8), (29, 0), (29, -1),
                 (30, 0), (30, 1 << 30), (31, 12), (31, 10248)]:
        a = list(ok)
        a[i] = v
        assert lib.vpt_gated_norm_bwd(*a) == 1, (i, v)
    assert lib.vpt_gated_norm_bwd_workspace(0, 4, 16) == 0 and lib.vpt_gated_norm_bwd_workspace(1, 4, 12) == 0
    assert lib.vpt_gated_norm_bwd_workspace(2, 3, 16) == 2 * 3 * 16 * 4


def test_clip_refuses(m):
    optim = m[1]
    g = z(4, 6, d=F32)
    for grads, out, msg in [([g], None, "GPU"), ([g.int()], None, "gradients"), ([g.double()], None, "gradients"),
                            ([g[:, :3]], None, "gaps"), ([g.to_sparse()], None, "dense"), ([1.0], None, "tensors"),
                            ([g, g], None, "overlap"), ([g, g[1:3]], None, "overlap"), ([g], [], "outputs"),
                            ([g], [g.half()], "another type"), ([g], [z(6, 4, d=F32)], "another type"),
                            ([g], [z(6, 4, d=F32).t()], "another type"),
                            ([g[0:2], g[2:4]], [g[2:4], g[0:2]], "overlaps another"), ([g[0:3]], [g[1:4]], "in part"),
                            ([g, g], [g, z(4, 6, d=F32)], "overlaps another")]:
        with pytest.raises(ValueError, match=msg):
            optim.GradClip(grads, out)
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([torch.nn.Parameter(g)], 0.0)
    assert optim.clip_grad_norm_([torch.nn.Parameter(g)], 1.0).item() == 0.0
    for t, want in [(g.t(), True), (g[:, :1], False), (g[1:3], True), (g.view(2, 2, 6).permute(2, 0, 1), True),
                    (z(0, 4), True), (z(1, 6, 1, 4).transpose(1, 3), True), (g.expand(2, 4, 6), False)]:
        assert optim._dense(t) == want


def test_pieces(m):
    """The table covers every value once, in pieces of at most the library's size."""
    import numpy as np
    ops, optim, _ = m
    piece = ops.call("vpt_grad_list_piece")
    sizes = [1, piece, 0, piece + 1, 3 * piece - 5, 7]
    c = optim.GradClip.__new__(optim.GradClip)
    c.grads = [z(n, d=d) for n, d in zip(sizes, [F32, BF16, F32, BF16, torch.float16, F32])]
    c.out = [g if i % 2 else g.clone() for i, g in enumerate(c.grads)]
    c.device = torch.device("cpu")
    table, count = c._pieces()
    t = table.numpy().view(optim._PIECE)
    assert len(t) == count == 1 + 1 + 2 + 3 + 1
    at = 0
    for g, o in zip(c.grads, c.out):
        done = 0
        while done < g.numel():
            r, es = t[at], g.element_size()
            assert r["g"] == g.data_ptr() + done * es and r["out"] == o.data_ptr() + done * es
            assert 0 < r["n"] <= piece and r["dtype"] == optim._CLIP_DTYPES[g.dtype]
            done += int(r["n"])
            at += 1
        assert done == g.numel()
    assert at == count and t.dtype.itemsize == 24 and isinstance(t, np.ndarray)
    c.grads = c.out = [z(0)]
    assert c._pieces() == (None, 0)


def test_c_abi_refuses_clip(m):
    lib = m[2].lib
    p = 4096
    assert lib.vpt_grad_list_norm(p, -1, p, None) == 1 and lib.vpt_grad_list_norm(None, 3, p, None) == 1
    assert lib.vpt_grad_list_norm(p, 3, None, None) == 1 and lib.vpt_grad_list_norm(p, 3, p + 4, None) == 1
    ok = [p, 3, 0, p, 3, 1.0, 0.0, p, None]
    for i, v in [(0, None), (1, -1), (3, None), (3, p + 4), (4, 0), (4, 1 << 20), (5, -1.0), (6, -1.0), (5, float("nan"))]:
        a = list(ok)
        a[i] = v
        assert lib.vpt_grad_list_clip(*a) == 1, (i, v)


def test_limits(m):
    """Sizes beyond what a launch covers, limits that f32 holds as zero."""
    ops, optim, _lib = m
    p, lib = 4096, _lib.lib  # never read
    fwd = [p, 16, p, 0, 16, p, p, p, 16, p, 16, p, 0, p, 16, p, 16, p, p, 3, 2, 16, 1.0, 1e-6, None]
    bwd = [p, 16, p, 16, p, 16, p, 0, 16, p, p, p, p, p, 16, p, 16, p, 0, p, 16, p, 16, p, p, p, p, p, p, 3, 2, 16, 1.0, None]
    for groups, rows in [(1 << 24, 1), (1, (1 << 30) + 1), (1 << 23, 129)]:
        fwd[19:21], bwd[29:31] = (groups, rows), (groups, rows)
        assert lib.vpt_gated_norm_fwd(*fwd) == 1 and lib.vpt_gated_norm_bwd(*bwd) == 1
    handle = optim.GradClip.__new__(optim.GradClip)
    for kw in (dict(max_norm=1e-50), dict(clip_value=1e-50), dict(max_norm=float("nan")), dict(clip_value=0.0), dict(max_norm=-1.0)):
        with pytest.raises(ValueError, match="must be > 0"):
            handle.clip(**kw)
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([], 1e-50)


def test_clip_grad_norm_has_torchs_positions(m, monkeypatch):
    """The third positional argument is torch's norm_type (L2 alone is offered), never the value limit."""
    optim = m[1]
    calls = []

    class Handle:
        def __init__(self, grads, out=None):
            pass

        def norm(self):
            return torch.tensor(1.0)

        def clip(self, max_norm=None, clip_value=None):
            calls.append((max_norm, clip_value))
            return torch.tensor(1.0)
    monkeypatch.setattr(optim, "GradClip", Handle)
    p = torch.nn.Parameter(z(3, d=F32))
    p.grad = z(3, d=F32)
    optim.clip_grad_norm_([p], 10.0, 2.0)
    optim.clip_grad_norm_([p], 10.0, 2, True)
    optim.clip_grad_norm_([p], 10.0, error_if_nonfinite=True, clip_value=0.5)
    assert calls == [(10.0, None), (10.0, None), (10.0, 0.5)]
    for kind in (float("inf"), 1.0, 0.02, float("nan")):
        for grads in ([p], []):
            with pytest.raises(ValueError, match="norm_type"):
                optim.clip_grad_norm_(grads, 1.0, kind)


def handle(optim, grads, out=None):
    """A GradClip without a GPU: its table on the CPU, no launch."""
    c = optim.GradClip.__new__(optim.GradClip)
    c.grads, c.out, c.device = grads, grads if out is None else out, torch.device("cpu")
    return c


def test_a_captured_table_stays(m, monkeypatch):
    """A graph reads the handle's table at every replay, also when the handle is gone by then."""
    import contextlib
    import gc
    import weakref
    ops, optim, _ = m
    state = {"capturing": False}
    monkeypatch.setattr(ops, "_on", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(ops, "_capturing", lambda: state["capturing"])
    real = ops.call
    monkeypatch.setattr(ops, "call", lambda name, *a: real(name, *a) if name.endswith(("_parts", "_piece")) else None)

    def use(capturing):
        c = handle(optim, [z(40, d=F32)])
        c._finish()
        state["capturing"] = capturing
        c.clip(1.0)
        c.clip(clip_value=1.0)
        state["capturing"] = False
        return weakref.ref(c._table)
    tables = use(False), use(True)
    gc.collect()
    assert tables[0]() is None and tables[1]() is not None


def test_the_memory_of_the_table_stays(m, monkeypatch):
    """The handle holds the memory that its table names, also when a tensor is given other memory meanwhile."""
    ops, optim, _ = m
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(ops, "_capturing", lambda: False, raising=False)
    g, o = z(40, d=F32), z(40, d=F32)
    c = handle(optim, [g], [o])
    c._finish()
    mem = [t.untyped_storage().data_ptr() for t in (g, o)]
    g.data, o.data = z(40, d=F32), z(40, d=F32)
    assert {s.data_ptr() for s in c._memory} == set(mem)


def test_no_handle_in_a_capture(m, monkeypatch):
    """Its table is copied from the host; refused before that."""
    ops, optim, _ = m
    monkeypatch.setattr(ops, "_capturing", lambda: True, raising=False)
    monkeypatch.setattr(optim.GradClip, "_pieces", lambda self: pytest.fail("a copy inside the capture"))
    with pytest.raises(RuntimeError, match="captured"):
        handle(optim, [z(4, d=F32)])._finish()


def test_streamed_by_bytes(m, monkeypatch):
    """Results go past the caches where gradients and results are more bytes than those hold, however many tensors they are."""
    ops, optim, _ = m
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(ops, "_capturing", lambda: False)

    def cached(sizes, dtype, in_place=False):
        flat = torch.empty(sum(sizes), dtype=dtype)
        grads = list(flat.split(sizes))
        c = handle(optim, grads, None if in_place else list(torch.empty_like(flat).split(sizes)))
        c._finish()
        return c._cached
    assert cached([300] * 3000, BF16) == 1  # 1.8 MB in 3000 pieces
    assert cached([16384] * 3000, BF16) == 1  # 98 MB and as much again
    assert cached([70_000_000], BF16) == 0 and cached([35_000_000], F32) == 0
    assert cached([70_000_000], BF16, in_place=True) == 1
