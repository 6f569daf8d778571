"""The stream that a backward of window attention runs on, without a GPU: streams, captures and kernels are stand-ins, the autograd
engine is torch's."""

import contextlib
import threading

import pytest
import torch

from torch_mojo_backend_b200 import _lib, tensor, window
from torch_mojo_backend_b200.flash_ops import _stream_for   # (the fixture below puts stand-ins in their places)
from torch_mojo_backend_b200.tensor import _alloc_holder

_cuda_view = tensor.TorchMojoTensor._cuda_view


class Stream:
    device = torch.device("cuda", 0)

    def __init__(self, name, capturing=False):
        self.name, self.capturing, self.waits = name, capturing, []

    def wait_stream(self, other):
        assert self.capturing or not other.capturing, f"{self.name} would be drawn into a capture"
        assert other.capturing or not self.capturing, f"{self.name} is captured and {other.name} is not"
        self.waits.append(other)


@pytest.fixture
def streams(host_backed_mojo, monkeypatch):
    """(the streams that every thread starts with, one that is being captured); the forward's is what its maker says."""
    own, captured = Stream("own"), Stream("captured", True)
    held = threading.local()
    current = lambda device=None: getattr(held, "stream", own)   # noqa: E731

    def set_stream(s):
        held.stream = s

    @contextlib.contextmanager
    def stream(s):
        before = current()
        set_stream(s)
        try:
            yield
        finally:
            set_stream(before)

    for name, f in (("current_stream", current), ("set_stream", set_stream), ("stream", stream),
                    ("is_current_stream_capturing", lambda: current().capturing)):
        monkeypatch.setattr(torch.cuda, name, f)
    ran = []   # the streams of the kernels
    monkeypatch.setattr(_lib, "window_fwd", lambda *a: _lib.OK)
    monkeypatch.setattr(_lib, "window_bwd", lambda *a: ran.append(current()) or _lib.OK)
    monkeypatch.setattr(_lib, "window_bwd_workspace_bytes", lambda *a: 256)
    monkeypatch.setattr(tensor, "_lent", {})
    captured.ran = ran
    return own, captured


class Bring(torch.autograd.Function):
    """A CPU tensor onto the device: the CPU side of its gradient is the caller's thread's, not the engine's."""

    @staticmethod
    def forward(ctx, x):
        return x.to("mojo")

    @staticmethod
    def backward(ctx, grad):
        return torch.zeros(grad.shape, dtype=grad.dtype)


class Ask(torch.autograd.Function):
    """A node that does something on the engine's thread and notes its stream."""

    @staticmethod
    def forward(ctx, x, act, note):
        ctx.how = act, note
        return x.detach()

    @staticmethod
    def backward(ctx, grad):
        act, note = ctx.how
        with contextlib.suppress(AssertionError, RuntimeError, AttributeError):   # (there is no CUDA device)
            act()
        note.append((threading.get_ident(), torch.cuda.current_stream()))
        return grad, None, None


def tensor_of(make, device="mojo"):
    t = make(1, 2, 8, 64, dtype=torch.bfloat16)
    return t.to(device) if device == "mojo" else t


def leaf(device="mojo"):
    return tensor_of(torch.zeros, device).requires_grad_()


def attend(q, on):
    out = window.window_attention(q, q, q, 3)
    out.grad_fn.stream = on   # (of a host-backed tensor there is none)
    return out


def ones():
    return tensor_of(torch.ones)


def asked(act=lambda: None):
    """(engine's thread, its current stream) behind `act` there."""
    note = []
    Ask.apply(leaf(), act, note).backward(ones())
    return note[0]


def test_a_captured_pass_runs_on_the_captured_stream_and_gives_the_threads_back(streams):
    own, captured = streams
    q, note = leaf(), []
    q.register_hook(lambda _: note.append(torch.cuda.current_stream()))
    attend(q, captured).backward(ones())
    assert captured.ran == [captured] and note == [captured]   # what the engine adds is captured too
    assert asked()[1] is own and not tensor._lent


@pytest.mark.parametrize("fails", [True, False])
@pytest.mark.parametrize("act", [None, lambda: _cuda_view(ones()), lambda: _alloc_holder(16, 0), lambda: _stream_for(0)])
def test_a_captured_pass_that_fails_or_ends_on_another_thread(streams, fails, act):
    """Nothing runs at the end of a pass that fails, and of another only on the thread that it ends on: here the caller's.  The next thing
    that the engine's thread does on the device is on its own stream again."""
    own, captured = streams
    x, threads = leaf("cpu"), []

    def hook(_):
        threads.append(threading.get_ident())
        if fails:
            raise ValueError("on purpose")

    x.register_hook(hook)
    out = attend(Ask.apply(Bring.apply(x), lambda: None, threads), captured)
    if fails:
        with pytest.raises(ValueError, match="on purpose"):
            out.backward(ones())
    else:
        out.backward(ones())
    (engine, at_that_time), caller = threads
    assert at_that_time is captured and caller == threading.get_ident()
    captured.capturing = False   # the capture is over: its stream is ordered with nothing
    if act is None:   # another backward
        q = leaf()
        attend(q, own).backward(ones())
        assert captured.ran == [captured, own]
    assert asked(act or (lambda: None)) == (engine, own)
    assert engine == caller or not tensor._lent


def test_a_pass_that_ends_on_another_thread(streams, monkeypatch):
    own, captured = streams
    ends = []

    class Engine:
        queue_callback = staticmethod(ends.append)

    monkeypatch.setattr(torch.autograd.Variable, "_execution_engine", Engine)
    with window._on_stream(captured):
        pass
    assert torch.cuda.current_stream() is captured
    other = threading.Thread(target=ends[0])
    other.start(), other.join()
    tensor.take_back_stream()
    assert torch.cuda.current_stream() is captured   # (the pass is not gone yet)
    ends.clear()
    tensor.take_back_stream()
    assert torch.cuda.current_stream() is own


def test_two_streams_of_one_capture_wait_for_one_another(streams):
    own, captured = streams
    side = Stream("side", True)
    torch.cuda.set_stream(captured)
    q = leaf()
    with torch.autograd.set_multithreading_enabled(False):
        attend(q, side).backward(ones())
    assert captured.ran == [side] and torch.cuda.current_stream() is captured
    assert side.waits == [captured, captured] and captured.waits == [side]
