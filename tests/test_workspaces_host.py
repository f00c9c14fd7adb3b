"""Which calls share a cached workspace, and how long it lives, without a GPU."""

import contextlib
import importlib
import types
import weakref

import pytest
import torch


@pytest.fixture
def cuda(monkeypatch):
    """A stand-in for the device: the stream, the capture it is part of (0: none), and what was
    allocated, as (capture at the time, weak reference)."""
    from m5kernels_b200 import _lib, paged

    linear = importlib.import_module("m5kernels_b200.linear")  # (the package's `linear` is the call)
    state = types.SimpleNamespace(stream=11, capture=0, made=[])
    alloc = {f: getattr(torch, f) for f in ("empty", "zeros")}

    def recorded(f):
        def make(*shape, device=None, **kw):
            t = alloc[f](*shape, **kw)
            state.made.append((state.capture, weakref.ref(t)))
            return t
        return make

    class Lib:
        def m5b_paged_attention_workspace_bytes(self, dim):
            return 8192 * dim

        def m5b_stream_capture_id(self, stream, out):
            assert stream == state.stream
            out._obj.value = state.capture
            return 0

    for f in alloc:
        monkeypatch.setattr(torch, f, recorded(f))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: state.stream, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: state.capture != 0,
                        raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream",
                        lambda d=None: types.SimpleNamespace(cuda_stream=state.stream))
    monkeypatch.setattr(torch.cuda, "device", lambda i: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "lib", lambda: Lib())
    monkeypatch.setattr(paged, "_scratch_bytes", {})
    monkeypatch.setattr(linear, "_workspaces", {})
    for module, name in ((paged, "_workspaces"), (linear, "_captured")):
        monkeypatch.setattr(module, name, linear._workspaces if module is paged else {}, raising=False)
    return state


def owner(cuda, pointer):
    """(capture, index) of the living allocation that starts at the pointer."""
    for i, (capture, ref) in enumerate(cuda.made):
        t = ref()
        if t is not None and t.data_ptr() == pointer:
            return capture, i
    raise AssertionError("no living allocation there")


def test_a_captured_attention_call_has_its_graphs_workspace(cuda):
    """A stream's buffer may be replaced by a larger one while the graph keeps its address."""
    from m5kernels_b200.paged import _scratch

    _scratch(0, 64)
    cuda.capture = 7
    first = _scratch(0, 64)
    assert owner(cuda, first[0])[0] == 7
    assert _scratch(0, 64)[0] == first[0]  # one for the calls of a capture
    cuda.capture = 8
    second = _scratch(0, 64)
    assert owner(cuda, second[0])[0] == 8 and second[0] != first[0]
    larger = _scratch(0, 128)
    assert owner(cuda, larger[0])[0] == 8 and larger[1] == 128 * 8192
    cuda.capture = 0
    eager = _scratch(0, 128)
    assert owner(cuda, eager[0])[0] == 0
    assert _scratch(0, 64)[0] == eager[0]


@pytest.mark.parametrize("name", ["workspace", "gemm_workspace", "fp32_workspace"])
def test_a_captured_product_has_its_graphs_workspaces(cuda, name):
    """Also without a first call: what a capture clears is not clear for calls beside the graph."""
    get = getattr(importlib.import_module("m5kernels_b200.linear"), name)
    dev = torch.device("cuda", 0)
    cuda.capture = 7
    owners = [owner(cuda, get(dev, 1000).data_ptr())]
    cuda.capture = 0
    first = get(dev, 1000)
    owners.append(owner(cuda, first.data_ptr()))
    cuda.capture = 8
    owners.append(owner(cuda, get(dev, 900).data_ptr()))
    assert [o[0] for o in owners] == [7, 0, 8]
    cuda.capture = 0
    assert get(dev, 1000) is first and get(dev, 2000) is not first


def test_a_workspace_lives_until_its_call_is_launched(cuda):
    """Another thread may replace the stream's buffer in between."""
    from m5kernels_b200.paged import _scratch

    mine = _scratch(0, 64)
    _scratch(0, 128)
    assert owner(cuda, mine[0])[1] == 0


def test_workspaces_of_finished_captures_are_let_go(cuda):
    from m5kernels_b200.paged import _scratch

    cuda.capture = 7
    _scratch(0, 64)
    assert cuda.made[0][1]() is not None
    cuda.capture = 0
    _scratch(0, 64)
    assert cuda.made[0][1]() is None


def test_counters_are_renewed_after_a_timeout(cuda, monkeypatch):
    """A wait that gave up may leave counters that later calls expect to be zero."""
    from m5kernels_b200 import _lib
    from m5kernels_b200.paged import _scratch

    linear = importlib.import_module("m5kernels_b200.linear")
    status = types.SimpleNamespace(value=0, cleared=0)

    class Lib(type(_lib.lib())):
        def m5b_device_status(self, out, clear):
            out._obj.value = status.value
            status.cleared += clear
            return 0

    monkeypatch.setattr(_lib, "lib", lambda: Lib())

    class Step:
        gemm_ws, device = torch.ones(4, dtype=torch.uint8), torch.device("cuda", 0)

    class Elsewhere(Step):
        gemm_ws, device = torch.ones(4, dtype=torch.uint8), torch.device("cuda", 1)

    bound = [Step(), Elsewhere()]
    monkeypatch.setattr(linear, "_bound", set(bound), raising=False)
    dev = torch.device("cuda", 0)
    get = lambda: (linear.gemm_workspace(dev, 100), _scratch(0, 64)[-1], linear.workspace(dev, 100))
    before = get()
    assert _lib.device_status() == 0
    assert all(a is b for a, b in zip(get(), before)) and bound[0].gemm_ws.all()
    status.value = 2
    assert _lib.device_status(clear=True) == 2 and status.cleared == 1
    after = get()
    assert after[0] is not before[0] and after[1] is not before[1] and after[2] is before[2]
    assert not after[0].any() and not after[1][:4096].any()
    assert not bound[0].gemm_ws.any() and bound[1].gemm_ws.all()


def test_captures_one_after_another_hold_one_workspace(cuda):
    """Graphs of one memory pool can take it in turn."""
    from m5kernels_b200.paged import _scratch

    real = torch.empty
    alive = []

    def counted(*shape, **kw):
        alive.append(sum(ref() is not None for _, ref in cuda.made))
        return real(*shape, **kw)

    torch.empty = counted
    try:
        for cuda.capture in (7, 8, 9):
            _scratch(0, 128)
    finally:
        torch.empty = real
    assert alive == [0, 0, 0]


def test_streams_have_their_own(cuda):
    from m5kernels_b200.paged import _scratch

    one = _scratch(0, 64)
    cuda.stream = 12
    assert _scratch(0, 64)[0] != one[0]
    cuda.stream = 11
    assert _scratch(0, 64)[0] == one[0]
