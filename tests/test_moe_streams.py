"""CPU test: the mixture-of-experts calls take what they allocate for the stream
that their kernels run on.  torch and the library are stand-ins that note the
stream of every allocation and of every call."""
from __future__ import annotations

import contextlib
import types

import pytest

CURRENT, OTHER = 0x100, 0x200


class Tensor:
    def __init__(self, world, shape, dtype):
        self.world, self.shape, self.dtype, self.device = world, tuple(shape), dtype, world.device
        self.used_on = []

    def dim(self):
        return len(self.shape)

    def numel(self):
        n = 1
        for s in self.shape:
            n *= s
        return n

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 0x1000

    def new_empty(self, shape, dtype=None):
        return self.world.empty(shape, dtype=dtype or self.dtype)

    def record_stream(self, stream):
        self.used_on.append(stream.cuda_stream)


class World:
    """What mlq.py uses of torch, with one device and a current stream."""

    def __init__(self):
        self.device = types.SimpleNamespace(type="cuda", index=0)
        self.now = CURRENT
        self.allocated, self.calls = [], []
        self.uint8, self.float32, self.int32 = "u8", "f32", "i32"
        self._C = types.SimpleNamespace(_cuda_getCurrentRawStream=lambda index: self.now)
        self.cuda = types.SimpleNamespace(
            current_device=lambda: 0, stream=self.on, device=lambda d: contextlib.nullcontext(),
            ExternalStream=lambda handle, device=None: types.SimpleNamespace(cuda_stream=handle),
            default_stream=lambda device=None: types.SimpleNamespace(cuda_stream=0),
            current_stream=lambda device=None: types.SimpleNamespace(cuda_stream=self.now))

    @contextlib.contextmanager
    def on(self, stream):
        before, self.now = self.now, stream.cuda_stream
        try:
            yield
        finally:
            self.now = before

    def empty(self, shape, dtype=None, device=None):
        t = Tensor(self, (shape,) if isinstance(shape, int) else shape, dtype)
        self.allocated.append((self.now, t))
        return t

    def tensor(self, *shape, dtype="f32"):
        return Tensor(self, shape, dtype)

    # the library: every function notes the stream, its last argument
    def __getattr__(self, name):
        if not name.startswith("mlq_"):
            raise AttributeError(name)
        if name.endswith("_workspace_bytes"):
            return lambda *a: 4096
        return lambda *a: self.calls.append(a[-1]) or 0


def _all_given(mlq, w, **kw):
    """Nothing is left to allocate: the handle goes to the library as it is."""
    return mlq.moe_layer(mlq.Router(w.tensor(4, 64), 2), _experts(mlq, w), w.tensor(3, 64), y=w.tensor(3, 64),
                         ids=w.tensor(3, 2, dtype="i32"), weights=w.tensor(3, 2), workspace=w.tensor(4096, dtype="u8"), **kw)


CALLS = {
    "all given": _all_given,
    "route": lambda mlq, w, **kw: mlq.moe_route(mlq.Router(w.tensor(4, 64), 2), w.tensor(3, 64), **kw),
    "experts": lambda mlq, w, **kw: mlq.moe_experts(_experts(mlq, w), w.tensor(3, 64), w.tensor(3, 2, dtype="i32"),
                                                    w.tensor(3, 2), **kw),
    "layer": lambda mlq, w, **kw: mlq.moe_layer(mlq.Router(w.tensor(4, 64), 2), _experts(mlq, w), w.tensor(3, 64), **kw),
    "epilogue": lambda mlq, w, **kw: mlq.linear_epilogue("q8_0", w.tensor(32 * 2 * 34, dtype="u8"), 32, 64,
                                                         w.tensor(3, 64), **kw),
}


def _experts(mlq, w):
    up, down = w.tensor(4 * 32 * 2 * 34, dtype="u8"), w.tensor(4 * 64 * 34, dtype="u8")
    return mlq.Experts("q8_0", up, up, down, 4, 64, 32)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("given,stream", [
    (None, CURRENT), (CURRENT, CURRENT), (OTHER, OTHER), (types.SimpleNamespace(cuda_stream=OTHER), OTHER), (0, 0)],
    ids=["none", "current", "handle", "object", "default"])
def test_a_call_allocates_for_its_stream(pkg, monkeypatch, name, given, stream):
    mlq, world = pkg.mlq, World()
    monkeypatch.setattr(mlq, "_torch", world)
    monkeypatch.setattr(mlq, "_moe_lib", lambda: world)
    out = CALLS[name](mlq, world, stream=given)
    assert world.calls == [stream] and world.now == CURRENT
    made = {"all given": 0, "route": 3, "experts": 2, "layer": 4, "epilogue": 2}[name]  # outputs and a workspace
    assert [s for s, _ in world.allocated] == [stream] * made
    # what the caller gets may be used on its own stream, and be dropped there
    for t in out if isinstance(out, tuple) else (out,):
        assert t.used_on == ([] if stream == CURRENT or name == "all given" else [CURRENT])


@pytest.mark.parametrize("name", [c for c in CALLS if c != "all given"])
def test_a_stream_of_another_device_is_refused(pkg, monkeypatch, name):
    """Under such a stream the tensors' device would have another current stream."""
    mlq, world = pkg.mlq, World()
    monkeypatch.setattr(mlq, "_torch", world)
    monkeypatch.setattr(mlq, "_moe_lib", lambda: world)
    with pytest.raises(ValueError, match="stream"):
        CALLS[name](mlq, world, stream=types.SimpleNamespace(cuda_stream=OTHER, device="cuda:1"))
    assert world.calls == [] and world.allocated == []
    CALLS[name](mlq, world, stream=types.SimpleNamespace(cuda_stream=OTHER, device=world.device))
    assert world.calls == [OTHER]
