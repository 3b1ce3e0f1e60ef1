"""CPU: MXFP4 weights (and NF4 states of other classes) as frozen bases of the LoRA layers: where they are moved, which modes they
take, which launch dequantises them."""

import pytest
import torch

BF16, U8 = torch.bfloat16, torch.uint8


@pytest.fixture(scope="module")
def m():
    from vpt import mxfp4, ops, sdxl
    return ops, mxfp4, sdxl


def weight(m, N, K):
    c = -(-K // 128)
    return m[1].MXFP4Weight(torch.zeros(N, 64 * c, dtype=U8), torch.zeros(N, 4 * c, dtype=U8), (N, K))


def block_sd(m, dim=64, rank=16):
    sd = {}
    for t in m[2].TARGETS:
        n, k = {"ff.net.0.proj": (8 * dim, dim), "ff.net.2": (dim, 4 * dim)}.get(t, (dim, dim))
        sd[f"{t}.linear.weight"] = weight(m, n, k)
        sd[f"{t}.lora_down.weight"], sd[f"{t}.lora_up.weight"] = torch.zeros(rank, k), torch.zeros(n, rank)
    for k in ("norm1", "norm2", "norm3"):
        sd[f"{k}.weight"], sd[f"{k}.bias"] = torch.ones(dim), torch.zeros(dim)
    return sd


def test_block_moves_its_bases(m):
    """A state dict loaded elsewhere: bases follow the block's device as NF4 states, biases and adapters do."""
    blk = m[2].SDXLTransformerBlock(64, 1, 64, 16, 16.0, block_sd(m), device="meta")
    for t, lin in blk.lin.items():
        assert lin.down.device.type == "meta" and lin.base.codes.device.type == "meta" and lin.base.scales.device.type == "meta", t
    here = block_sd(m)
    blk = m[2].SDXLTransformerBlock(64, 1, 64, 16, 16.0, here, device="cpu")
    assert all(blk.lin[t].base is here[f"{t}.linear.weight"] for t in blk.lin)  # already there: the same weight, with what it keeps


def lora(m, base, mode=None):
    return m[2].LoRALinearNF4(base, None, torch.zeros(16, base.shape[1]), torch.zeros(base.shape[0], 16), 16.0, 16, mode)


def test_base_mode_is_checked_when_set(m):
    """The mode is assigned after construction too; "inline" reads NF4 parts, which an MXFP4 base has not."""
    lin = lora(m, weight(m, 64, 64))
    assert lin.base_mode == "dequant"
    lin.base_mode = "resident"
    for mode, what in [("inline", "inline"), ("fast", "base_mode"), (None, "base_mode")]:
        with pytest.raises(ValueError, match=what):
            lin.base_mode = mode
        assert lin.base_mode == "resident"
    with pytest.raises(ValueError, match="inline"):
        lora(m, weight(m, 64, 64), "inline")
    nf4 = m[2].NF4Weight(*[torch.zeros(1)] * 5, (64, 64))
    lin = lora(m, nf4)
    lin.base_mode = "inline"
    proj = m[2].NF4Linear(nf4, None, "inline")
    assert lin.base_mode == proj.base_mode == "inline"
    with pytest.raises(ValueError, match="base_mode"):
        proj.base_mode = "fast"
    with pytest.raises(ValueError, match="inline"):
        m[2].NF4Linear(weight(m, 64, 64), None, "inline")


def test_every_base_is_dequantised(m, monkeypatch):
    """dequant_into: MXFP4 bases by their own launch, every other one (NF4 states of any class) in the batched launches."""
    ops, _, sdxl = m
    batched, own = [], []
    monkeypatch.setattr(ops, "nf4_dequant_batch", lambda pairs: batched.append([b for b, _ in pairs]))

    class Like:  # the parts of an NF4Weight, of a class of its own
        pass
    mx = weight(m, 64, 64)
    mx.dequantize = lambda out=None: own.append(out)
    nf4, like, out = m[2].NF4Weight(*[torch.zeros(1)] * 5, (64, 64)), Like(), torch.zeros(1)
    sdxl.dequant_into([(nf4, None), (mx, out), (like, None)])
    assert batched == [[nf4, like]] and own == [out]
    like.shape, like.numel = (64, 64), 4096
    assert lora(m, like, "inline").base is like


def test_spatial_transformer_takes_them(m):
    """proj_in and proj_out too, on the stack's device."""
    sd = {f"transformer_blocks.0.{k}": v for k, v in block_sd(m).items()}
    sd.update({"norm.weight": torch.ones(64), "norm.bias": torch.zeros(64), "proj_in.weight": weight(m, 64, 64),
               "proj_in.bias": torch.zeros(64), "proj_out.weight": weight(m, 64, 64), "proj_out.bias": torch.zeros(64)})
    st = m[2].SDXLSpatialTransformer(64, 1, 1, 64, 16, 16.0, sd, device="meta")
    for p in (st.proj_in, st.proj_out):
        assert isinstance(p.base, m[1].MXFP4Weight) and p.base.codes.device.type == "meta" and p.base_mode == "dequant"
