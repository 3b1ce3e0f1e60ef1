"""CPU: which launches share a scratch buffer. A buffer is one stream's (its launches run in order); another stream has its own, and
a captured region takes a new one from its graph's memory, which neither another graph nor an eager call that lets a
buffer grow can touch."""

import pytest
import torch

BF16 = torch.bfloat16


@pytest.fixture()
def at(monkeypatch):
    """(ops, sdxl, state): state's stream and capturing are what the buffers see."""
    from vpt import ops, sdxl
    state = {"stream": 11, "capturing": False}
    monkeypatch.setattr(ops, "_here", lambda dev: (str(dev), state["stream"]), raising=False)
    monkeypatch.setattr(ops, "_capturing", lambda: state["capturing"], raising=False)
    monkeypatch.setattr(ops, "stream", lambda: state["stream"])
    return ops, sdxl, state


class Base:
    shape, numel = (8, 16), 128

    def dequantize(self, out=None):
        return torch.zeros(self.shape, dtype=BF16) if out is None else out


def takers(ops, sdxl):
    dev = torch.device("cpu")
    return {"workspace": lambda n: ops.workspace(dev, "t", n), "tickets": lambda n: ops.tickets(dev, n),
            "slabs": lambda n: ops._lora_ws(dev, "t", 4 * n), "base": lambda n: sdxl._dequant_scratch(Base(), dev)}


@pytest.mark.parametrize("what", ["workspace", "tickets", "slabs", "base"])
def test_one_stream_one_buffer(at, what):
    ops, sdxl, state = at
    take = takers(ops, sdxl)[what]
    a = take(64)
    assert take(64).data_ptr() == a.data_ptr()
    state["stream"] = 12
    b = take(64)
    assert b.data_ptr() != a.data_ptr() and take(64).data_ptr() == b.data_ptr()
    state["stream"] = 11
    assert take(64).data_ptr() == a.data_ptr()


@pytest.mark.parametrize("what", ["workspace", "tickets", "slabs", "base"])
def test_captured_regions_share_nothing(at, what):
    ops, sdxl, state = at
    take = takers(ops, sdxl)[what]
    a = take(64)
    state["capturing"] = True
    b, c = take(64), take(64)
    assert len({a.data_ptr(), b.data_ptr(), c.data_ptr()}) == 3
    if what == "tickets":
        assert not b.any() and b.numel() >= 64
    state["capturing"] = False
    assert take(64).data_ptr() == a.data_ptr()  # the capture left nothing of its graph behind


def test_block_bases(at):
    """The bases of a block's targets, dequantised side by side."""
    ops, sdxl, state = at
    from vpt.mxfp4 import MXFP4Weight
    w = MXFP4Weight(torch.zeros(64, 64, dtype=torch.uint8), torch.zeros(64, 4, dtype=torch.uint8), (64, 64))
    w.dequantize = lambda out=None: out
    lin = type("L", (), dict(base=w, fused=True, base_mode="dequant"))
    lins = {t: lin for t in sdxl.TARGETS}
    first = sdxl.dequant_bases(lins, sdxl.TARGETS, torch.device("cpu"))
    ptr = {t: v.data_ptr() for t, v in first.items()}
    state["stream"] = 12
    other = sdxl.dequant_bases(lins, sdxl.TARGETS, torch.device("cpu"))
    assert not set(ptr.values()) & {v.data_ptr() for v in other.values()}
    state["stream"] = 11
    again = sdxl.dequant_bases(lins, sdxl.TARGETS, torch.device("cpu"))
    assert {t: v.data_ptr() for t, v in again.items()} == ptr


def test_batched_slabs_are_held(at):
    """Slabs of a captured region belong to no cache: the batch holds them until its reduce is launched."""
    ops, _, state = at
    state["capturing"] = True
    b = ops._LoraBatch()
    ptrs = [b.ws(torch.device("cpu"), 4096).data_ptr() for _ in range(4)]
    assert len(set(ptrs)) == 4 and {t.data_ptr() for t in b.keep} >= set(ptrs)


class Event:
    made = []

    def __init__(self):
        self.recorded = None
        Event.made.append(self)

    def record(self, stream=None):
        self.recorded = stream


class Stream:
    def __init__(self, name):
        self.name, self.waits = name, []

    def wait_event(self, e):
        self.waits.append(e)


class Kept(torch.Tensor):
    """A tensor that notes the streams it is marked as used on."""
    def record_stream(self, s):
        self.__dict__.setdefault("used", []).append(s.name)


@pytest.mark.parametrize("attr", ["resident", "resident_qkv", "anything"])
def test_built_once_is_waited_for(at, monkeypatch, attr):
    """A base kept on the device is built on the stream of its first caller; another stream waits for that, once, and its use is
    known to the allocator; a capture keeps nothing whose values only a replay would make."""
    ops, _, state = at
    streams = {k: Stream(k) for k in (11, 12, 13)}
    monkeypatch.setattr(torch.cuda, "Event", Event)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: streams[state["stream"]])
    owner, builds = type("Owner", (), dict(resident=None, resident_qkv=None))(), []

    def build():
        builds.append(state["stream"])
        return torch.zeros(4).as_subclass(Kept)
    state["capturing"] = True
    t = ops.built_once(owner, attr, build)
    assert getattr(owner, attr, None) is None and builds == [11]
    state["capturing"] = False
    t = ops.built_once(owner, attr, build)
    assert builds == [11, 11] and getattr(owner, attr) is t and ops.built_once(owner, attr, build) is t
    assert not streams[11].waits and Event.made[-1].recorded is streams[11]
    for s in (12, 13, 12, 11):
        state["stream"] = s
        assert ops.built_once(owner, attr, build) is t
    assert [len(streams[s].waits) for s in (11, 12, 13)] == [0, 1, 1] and t.used == [12, 13] and builds == [11, 11]
    state["stream"], state["capturing"] = 14, True  # an event from outside may not enter a capture
    streams[14] = Stream(14)
    assert ops.built_once(owner, attr, build) is t and not streams[14].waits
