"""Cases that time the operators of a gated transformer block over a 4-bit base, and of clipping its gradients.

  quantize  microscaled 4-bit values (MXFP4): a tensor to codes and shared scales, and back
  linear    a Linear on a microscaled 4-bit weight: the input quantised, the product, bias and residual; with "train"
            also its input gradient
  gated     a block's output normed, gated and added to the residual stream, and the next block's norm; or its backward
  clip      the global norm of many gradient tensors, and their clipping

`own` false: plain torch in 32 bits (64 where sums are long), rounded once at the end. `own` true: the framework's calls.

The 4-bit layout both sides share: a row of K values is padded with zeros to a multiple of 128 and cut into blocks of 32;
a block has a power-of-two scale 2^e, e = clamp(floor(log2 max|x|) - 2, -127, 127), stored as the byte e + 127, and 32
codes of x / 2^e rounded to the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} (ties to the even code), two to a byte, the
first in the low half.
"""

import math
import os
import random
import sys

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # hidden activations of the feed-forward at 1024 x 1024, batch 8 (8 x 4170 tokens), and back
        {"name": "quantize_tokens", "op": "quantize", "rows": 33360, "cols": 2048, "dtype": "bfloat16"},
        # a master weight in 32 bits, its rows no multiple of a block
        {"name": "quantize_weight_odd", "op": "quantize", "rows": 1279, "cols": 1000, "dtype": "float32"},
        # the joined first products of a feed-forward, 1024 x 1024, batch 8
        {"name": "linear_1024", "op": "linear", "m": 33360, "n": 4096, "k": 768, "bias": True, "resid": False, "train": False},
        # one token's q, k and v
        {"name": "linear_one_token", "op": "linear", "m": 1, "n": 2304, "k": 768, "bias": True, "resid": False, "train": False},
        # a feed-forward's last product into the residual stream, one training step of it
        {"name": "linear_ff_train", "op": "linear", "m": 4224, "n": 1280, "k": 5120, "bias": True, "resid": True, "train": True},
        # q, k and v at 512 x 512, batch 16 (16 x 1098 tokens), one training step of it
        {"name": "linear_512_train", "op": "linear", "m": 17568, "n": 2304, "k": 768, "bias": True, "resid": False, "train": True},
        # a block's end at 1024 x 1024, batch 8: post-norm, gate, residual, the next norm and its modulation
        {"name": "gated_1024", "op": "gated", "groups": 8, "rows": 4170, "dim": 768, "stream": "bfloat16", "post": True,
         "pre": True, "mod": True, "gate": "group", "backward": False},
        # two short sequences over a 32-bit residual stream, a learned gate for all of them
        {"name": "gated_text_f32", "op": "gated", "groups": 2, "rows": 77, "dim": 640, "stream": "float32", "post": True,
         "pre": True, "mod": False, "gate": "all", "backward": False},
        # the backward of the 1024 x 1024 step
        {"name": "gated_1024_bwd", "op": "gated", "groups": 8, "rows": 4170, "dim": 768, "stream": "bfloat16", "post": True,
         "pre": True, "mod": True, "gate": "group", "backward": True},
        # the backward of a wider block with one learned gate
        {"name": "gated_wide_bwd", "op": "gated", "groups": 4, "rows": 1025, "dim": 1280, "stream": "bfloat16", "post": True,
         "pre": True, "mod": True, "gate": "all", "backward": True},
        # every gradient of a depth-12 model in 32 bits, over the limit: clipped copies for the optimizer
        {"name": "clip_model", "op": "clip", "tensors": "model", "count": 0, "total": 0, "dtype": "float32", "over": True,
         "inplace": False, "value": 0.0},
        # the gradients of 1400 adapter matrices, under the limit, in place
        {"name": "clip_adapters", "op": "clip", "tensors": "adapters", "count": 0, "total": 0, "dtype": "bfloat16",
         "over": False, "inplace": True, "value": 0.0},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "gated", "gated", "clip"])
    if op == "quantize":
        cols = _spread(rng, 32, 5120)
        return {"op": op, "rows": _spread(rng, 1, min(33360, 68_000_000 // cols)), "cols": cols,
                "dtype": rng.choice(list(TYPES))}
    if op == "linear":
        train = rng.random() < 0.3
        step = 8 if train or rng.random() < 0.5 else 1  # a gradient's rows start at multiples of 16 bytes
        n, k = (max(step, _spread(rng, 64, 5120) // step * step) for _ in range(2))
        resid = rng.random() < 0.4
        most = min(100_000_000_000 // (n * k * (2 if train else 1)), 130_000_000 // (n * (2 if resid else 1)))
        return {"op": op, "m": _spread(rng, 1, max(1, min(33360, most))), "n": n, "k": k, "bias": rng.random() < 0.6,
                "resid": resid, "train": train}
    if op == "gated":
        dim = 8 * _spread(rng, 8, 320)
        groups = _spread(rng, 1, 16)
        post = rng.random() < 0.7
        pre = not post or rng.random() < 0.8
        return {"op": op, "groups": groups, "rows": _spread(rng, 1, max(1, min(4170, 25_000_000 // (dim * groups)))), "dim": dim,
                "stream": rng.choice(["bfloat16", "bfloat16", "float32"]), "post": post, "pre": pre,
                "mod": pre and rng.random() < 0.6, "gate": rng.choice(["group", "all", "none"]), "backward": rng.random() < 0.5}
    over = rng.random() < 0.5
    total = _spread(rng, 2000, 60_000_000)
    return {"op": op, "tensors": "random", "count": _spread(rng, 1, 600), "total": total, "dtype": rng.choice(list(TYPES)),
            "over": over, "inplace": not over, "value": rng.choice([0.0, 0.0, 0.01]) if over else 0.0}


def _model_shapes(depth=12, dim=768, hidden=2048, bottleneck=128, heads=64):
    block = [(dim, dim), (dim,)] * 4 + [(heads,)] * 2 + [(dim,)] * 2 + [(hidden, dim), (hidden,)] * 2 + [(dim, hidden), (dim,)]
    ends = [(bottleneck, 768), (dim, bottleneck), (dim,), (dim, 256), (dim,), (dim, dim), (dim,), (dim,), (768, dim), (768,)]
    return block * depth + ends


def _adapter_shapes(rank=16):
    shapes = []
    for dim, blocks in ((640, 10), (1280, 60)):
        sizes = [(dim, dim)] * 4 + [(dim, dim), (dim, 2048), (dim, 2048), (dim, dim), (8 * dim, dim), (dim, 4 * dim)]
        shapes += [s for n, k in sizes for s in ((rank, k), (n, rank))] * blocks
    return shapes


def _shapes(case):
    if case["tensors"] == "model":
        return _model_shapes()
    if case["tensors"] == "adapters":
        return _adapter_shapes()
    rng = random.Random(case["total"] * 1009 + case["count"])
    cuts = sorted(rng.randrange(case["total"] + 1) for _ in range(case["count"] - 1))  # odd sizes, empty ones too
    return [(b - a,) for a, b in zip([0] + cuts, cuts + [case["total"]])]


def _split(flat, shapes):
    """The tensors of `shapes` one behind the other, each start at a multiple of 16 bytes, as views of `flat`."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += -(-n // 8) * 8
    return out


def _flat_size(shapes):
    return sum(-(-math.prod(s) // 8) * 8 for s in shapes)


# ------------------------------------------------------------------------------------------ plain forms
def _power(byte):
    """2^(byte - 127) for whole numbers 0 .. 254, exactly."""
    byte = byte.int()
    return torch.where(byte > 0, byte << 23, torch.full_like(byte, 1 << 22)).view(torch.float32)


def _quantize(x):
    """(codes [rows, 64 c] u8, scales [rows, 4 c] u8), c = ceil(cols / 128)."""
    rows, cols = x.shape
    wide = -(-cols // 128) * 128
    x = torch.nn.functional.pad(x.float(), (0, wide - cols)).view(rows, wide // 32, 32)
    top = x.abs().amax(2)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127, dtype=torch.int32)).clamp(-127, 127)
    a = x.abs() * _power(127 - e).unsqueeze(2)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
            + 8 * torch.signbit(x).to(torch.uint8)).view(rows, wide)
    return code[:, 0::2] | (code[:, 1::2] << 4), (e + 127).to(torch.uint8)


def _dequantize(codes, scales, cols):
    rows = codes.shape[0]
    code = torch.stack([codes & 15, codes >> 4], 2).view(rows, -1)
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    return (grid[code.long()] * _power(scales).repeat_interleave(32, 1))[:, :cols]


def _plain_linear(s):
    codes, scales = _quantize(s["x"])
    k = s["x"].shape[1]
    w = _dequantize(s["codes"], s["scales"], k)
    y = _dequantize(codes, scales, k) @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["resid"] is not None:
        y = y + s["resid"].float()
    out = {"y": y.to(torch.bfloat16)}
    if s["dy"] is not None:
        out["dx"] = (s["dy"].float() @ w).to(torch.bfloat16)
    return out


def _rows(v, s):
    """A vector for all groups, or one of each, as something that multiplies [groups, rows, dim]."""
    return v.float().view(-1, 1, s["h"].shape[1])


def _plain_gated(s):
    g, d = s["groups"], s["h"].shape[1]
    h, x = s["h"].float().view(g, -1, d), s["x"].float().view(g, -1, d)
    u = h
    if s["w_post"] is not None:
        u = h * torch.rsqrt(h.square().mean(2, keepdim=True) + EPS) * s["w_post"].float()
    if s["gate"] is not None:
        u = u * _rows(s["gate"], s)
    new = (x + s["resid_scale"] * u).to(s["x"].dtype)
    out = {"x": new.view(-1, d)}
    if s["w_pre"] is not None:
        f = new.float()
        y = f * torch.rsqrt(f.square().mean(2, keepdim=True) + EPS) * s["w_pre"].float()
        if s["scale"] is not None:
            y = y * (1 + _rows(s["scale"], s)) + _rows(s["shift"], s)
        out["y"] = y.to(torch.bfloat16).view(-1, d)
    return out


def _for(v, t):
    """A sum of each group as the gradient of a vector `v`: of all groups together where v is one for all."""
    return t.view(v.shape) if v.dim() == 2 else t.sum(0)


def _plain_gated_backward(s):
    g, d = s["groups"], s["h"].shape[1]
    view = lambda t: t.float().view(g, -1, d)  # noqa: E731
    h, new, dx = view(s["h"]), view(s["x_new"]), view(s["dx_new"])
    out = {}
    if s["w_pre"] is not None:
        r = s["rstd_pre"].view(g, -1, 1)
        n, dy, w = new * r, view(s["dy"]), s["w_pre"].float()
        dm = dy
        if s["scale"] is not None:
            out["dscale"] = _for(s["scale"], (dy * n * w).sum(1))
            out["dshift"] = _for(s["shift"], dy.sum(1))
            dm = dy * (1 + _rows(s["scale"], s))
        out["dw_pre"] = (dm * n).sum((0, 1))
        dn = dm * w
        dx = dx + r * (dn - n * (dn * n).mean(2, keepdim=True))
    out["dx"] = dx.to(s["x_new"].dtype).view(-1, d)
    v, w = h, None
    if s["w_post"] is not None:
        r, w = s["rstd_post"].view(g, -1, 1), s["w_post"].float()
        v = h * r
    du = dx * s["resid_scale"]
    if s["gate"] is not None:
        out["dgate"] = _for(s["gate"], (du * (v if w is None else v * w)).sum(1))
        du = du * _rows(s["gate"], s)
    if w is not None:
        out["dw_post"] = (du * v).sum((0, 1))
        dv = du * w
        du = r * (dv - v * (dv * v).mean(2, keepdim=True))
    out["dh"] = du.to(torch.bfloat16).view(-1, d)
    return out


def _plain_clip(s):
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    limit = s["value"] or math.inf
    [o.copy_((g.float() * coef).clamp(-limit, limit)) for g, o in zip(s["grads"], s["out"])]
    return {"grads": s["flat_out"], "norm": norm.float()}


# ------------------------------------------------------------------------------------------ the framework's calls
def _framework():
    path = os.path.join(os.getcwd(), "vision-pt_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vpt import mxfp4, ops, optim
    return ops, mxfp4, optim


def _own_run(s):
    ops, mxfp4, _ = _framework()
    if s["op"] == "quantize":
        codes, scales = ops.mxfp4_quantize(s["x"])
        return {"values": ops.mxfp4_dequantize(codes, scales, s["x"].shape[1]), "scales": scales}
    if s["op"] == "linear":
        w = mxfp4.MXFP4Weight(s["codes"], s["scales"], (s["codes"].shape[0], s["x"].shape[1]))
        out = {"y": ops.linear_mxfp4(s["x"], w, bias=s["bias"], resid=s["resid"])}
        if s["dy"] is not None:
            out["dx"] = ops.linear_mxfp4_dgrad(s["dy"], w)
        return out
    if s["op"] == "clip":
        return {"norm": s["clipper"].clip(s["max_norm"], s["value"] or None), "grads": s["flat_out"]}
    params = {k: s[k] for k in ("w_post", "w_pre", "gate", "scale", "shift", "groups", "resid_scale")}
    if "dx_new" not in s:
        new, y, _, _ = ops.gated_norm_fwd(s["h"], s["x"], eps=EPS, **params)
        return {"x": new} if y is None else {"x": new, "y": y}
    g = ops.gated_norm_bwd(s["dy"], s["dx_new"], s["h"], s["x_new"], s["rstd_post"], s["rstd_pre"], **params)
    return {k: v for k, v in g._asdict().items() if v is not None}


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    bf = torch.bfloat16
    if case["op"] == "quantize":
        # values of very different sizes from one channel to the next, some blocks of zeros
        x = randn(case["rows"], case["cols"]) * torch.exp2(randn(case["cols"]).mul(2).round())
        x[:: 17, : 32] = 0
        return {"op": "quantize", "x": x.to(TYPES[case["dtype"]])}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        codes, scales = _quantize(randn(n, k) * 0.02)
        return {"op": "linear", "x": (randn(m, k) * torch.exp2(randn(k).round())).to(bf), "codes": codes, "scales": scales,
                "bias": randn(n).to(bf) if case["bias"] else None, "resid": randn(m, n).to(bf) if case["resid"] else None,
                "dy": randn(m, n).to(bf) if case["train"] else None}
    if case["op"] == "clip":
        shapes, kind = _shapes(case), TYPES[case["dtype"]]
        flat = torch.zeros(_flat_size(shapes), device="cuda", dtype=kind)
        grads = _split(flat, shapes)
        noise = _split(randn(flat.numel()), shapes)
        sizes = torch.exp2(torch.randn(len(shapes), generator=torch.Generator().manual_seed(int(seed)))).tolist()
        unit = math.sqrt(sum(a * a * math.prod(s) for a, s in zip(sizes, shapes)))
        to = 7.5 if case["over"] else 0.25  # their norm, near enough; the limit is 1
        [g.copy_(z * (a * to / unit)) for g, z, a in zip(grads, noise, sizes)]
        flat_out = flat if case["inplace"] else torch.zeros_like(flat)
        s = {"op": "clip", "grads": grads, "flat": flat, "out": grads if case["inplace"] else _split(flat_out, shapes),
             "flat_out": flat_out, "max_norm": 1.0, "value": case["value"]}
        if own:
            s["clipper"] = _framework()[2].GradClip(grads, out=None if case["inplace"] else s["out"])
        return s
    g, rows, d, kind = case["groups"], case["groups"] * case["rows"], case["dim"], TYPES[case["stream"]]
    mod = randn(g, 3 * d).mul(0.5).to(bf)  # one row for each sample, as a modulation's Linear gives it
    gate = {"group": mod[:, 2 * d:], "all": (randn(d) * 0.3).to(bf), "none": None}[case["gate"]]
    s = {"op": "gated", "groups": g, "resid_scale": 0.7, "h": randn(rows, d).mul(3).to(bf),
         "w_post": (1 + 0.2 * randn(d)).to(bf) if case["post"] else None,
         "w_pre": (1 + 0.2 * randn(d)).to(bf) if case["pre"] else None, "gate": gate,
         "scale": mod[:, :d] if case["mod"] else None, "shift": mod[:, d:2 * d] if case["mod"] else None}
    x = randn(rows, d).mul(2).to(kind)
    if not case["backward"]:
        return {**s, "x": x}
    rstd = lambda t: torch.rsqrt(t.double().square().mean(1) + EPS).float()  # noqa: E731
    return {**s, "x_new": x, "dx_new": randn(rows, d).to(kind), "dy": randn(rows, d).to(bf) if case["pre"] else None,
            "rstd_post": rstd(s["h"]) if case["post"] else None, "rstd_pre": rstd(x) if case["pre"] else None}


def run(state):
    if own:
        return _own_run(state)
    if state["op"] == "quantize":
        codes, scales = _quantize(state["x"])
        return {"values": _dequantize(codes, scales, state["x"].shape[1]).to(torch.bfloat16), "scales": scales}
    if state["op"] == "linear":
        return _plain_linear(state)
    if state["op"] == "clip":
        return _plain_clip(state)
    return _plain_gated_backward(state) if "dx_new" in state else _plain_gated(state)


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        size = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
        return {"bytes": n * (size + 2 + 17 / 32), "flops": 2 * n}  # values in, values and codes out
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        b = 2 * m * k + n * k * 17 / 32 + 2 * m * n * (2 if case["resid"] else 1) + (2 * n if case["bias"] else 0)
        if case["train"]:
            b += 2 * m * n + 2 * m * k
        return {"bytes": b, "flops": 2 * m * n * k * (2 if case["train"] else 1)}
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _shapes(case))
        size = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
        return {"bytes": n * size * (2 if case["over"] else 1), "flops": 3 * n}
    n = case["groups"] * case["rows"] * case["dim"]
    size = torch.empty(0, dtype=TYPES[case["stream"]]).element_size()
    if case["backward"]:  # dy, h in, dh out; dx', x' in, dx out (x' feeds only the norm behind it)
        return {"bytes": n * ((2 if case["pre"] else 0) + 4 + size * (3 if case["pre"] else 1)), "flops": 20 * n}
    return {"bytes": n * (2 + 2 * size + (2 if case["pre"] else 0)), "flops": 12 * n}


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
def _exact_power(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_codes(x):
    """The 4-bit values of x and the bytes of their scales: the nearest multiple of the grid's step there."""
    rows, cols = x.shape
    wide = -(-cols // 128) * 128
    p = torch.zeros(rows, wide // 32, 32, dtype=torch.float64, device=x.device)
    p.view(rows, wide)[:, :cols] = x.double()
    top = p.abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -130)))
    e = e + (top >= _exact_power(e + 1)).double() - (top < _exact_power(e)).double()  # where log2 was rounded over a border
    unit = _exact_power((e - 2).clamp(-127, 127))
    unit[top == 0] = 2.0 ** -127
    a = p.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    q = torch.minimum(torch.round(a / step) * step, torch.full_like(a, 6.0)) * torch.sign(p) * unit
    return q.view(rows, wide)[:, :cols], torch.log2(unit).add(127).round().to(torch.uint8).squeeze(2)


def _exact_values(codes, scales, cols):
    mant = torch.tensor(GRID, dtype=torch.float64, device=codes.device)
    lo, hi = codes % 16, codes // 16
    half = [mant[(c % 8).long()] * (1 - 2 * (c // 8).double()) for c in (lo, hi)]
    v = torch.stack(half, -1).reshape(codes.shape[0], -1, 32) * _exact_power(scales.double() - 127).unsqueeze(-1)
    return v.reshape(codes.shape[0], -1)[:, :cols]


def _exact_norm(t, w):
    return t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * w


def _exact_gated(s):
    g, d = s["groups"], s["h"].shape[1]
    with torch.enable_grad():
        leaf = {k: s[k].double().requires_grad_() for k in ("w_post", "w_pre", "gate", "scale", "shift") if s[k] is not None}
        vec = lambda k: leaf[k].unsqueeze(1) if leaf[k].dim() == 2 else leaf[k]  # noqa: E731
        h = s["h"].double().view(g, -1, d).requires_grad_()
        add = _exact_norm(h, leaf["w_post"]) if "w_post" in leaf else h * 1.0
        if "gate" in leaf:
            add = add * vec("gate")
        add = add * s["resid_scale"]
        if "dx_new" in s:
            new = s["x_new"].double().view(g, -1, d).requires_grad_()
        else:  # the next norm reads the stream as it is stored
            exact = (s["x"].double().view(g, -1, d) + add).detach()
            new = exact.to(s["x"].dtype).double()
        y = None
        if "w_pre" in leaf:
            y = _exact_norm(new, leaf["w_pre"])
            if "scale" in leaf:
                y = y * (1 + vec("scale")) + vec("shift")
        if "dx_new" not in s:
            out = {"x": exact.view(-1, d)}
            return out if y is None else {**out, "y": y.detach().view(-1, d)}
        total, out = s["dx_new"].double().view(g, -1, d), {}
        if y is not None:
            names = [k for k in ("w_pre", "scale", "shift") if k in leaf]
            got = torch.autograd.grad(y, [new] + [leaf[k] for k in names], s["dy"].double().view(g, -1, d))
            total = total + got[0]
            out.update({"d" + k: t for k, t in zip(names, got[1:])})
        names = [k for k in ("w_post", "gate") if k in leaf]
        got = torch.autograd.grad(add, [h] + [leaf[k] for k in names], total)
        out.update({"d" + k: t for k, t in zip(names, got[1:])})
        return {**out, "dx": total.view(-1, d), "dh": got[0].view(-1, d)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        values, scales = _exact_codes(s["x"])
        return {"values": values, "scales": scales}
    if case["op"] == "linear":
        w = _exact_values(s["codes"], s["scales"], s["x"].shape[1])
        y = torch.matmul(_exact_codes(s["x"])[0], w.t())
        y = y + (0 if s["bias"] is None else s["bias"].double()) + (0 if s["resid"] is None else s["resid"].double())
        return {"y": y} if s["dy"] is None else {"y": y, "dx": torch.matmul(s["dy"].double(), w)}
    if case["op"] == "clip":
        flat = s["flat"].double()
        norm = torch.linalg.vector_norm(flat)
        new = flat * torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        return {"grads": torch.clamp(new, -s["value"], s["value"]) if s["value"] else new, "norm": norm}
    return _exact_gated(s)
