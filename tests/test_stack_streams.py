"""On which stream MoeStack makes the buffers of a call (CPU: torch.cuda's streams are stand-ins, the library does nothing).  The
kernels run on the handle given; a buffer filled, or handed out again, on another stream is not ordered with them."""
import contextlib

import pytest
import torch

import checkpoint as C

H, E, I, K = 256, 8, 128, 2


class Created:
    def __init__(self, handle):
        self.cuda_stream = handle

    def wait_event(self, e):
        pass

    record = wait_event


class Streams:
    """torch.cuda's current stream as a list, and where each allocation was made."""

    def __init__(self, monkeypatch):
        self.stack, self.made = ["default"], []
        monkeypatch.setattr(torch.cuda, "ExternalStream", lambda h, device=None: Created(h))
        monkeypatch.setattr(torch.cuda, "Stream", lambda device=None: Created(9))
        monkeypatch.setattr(torch.cuda, "Event", lambda: Created(0))
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.stack[-1])
        monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: "default")
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        monkeypatch.setattr(torch.cuda, "stream", self.enter)
        for name in ("empty", "zeros"):
            monkeypatch.setattr(torch, name, self.noted(getattr(torch, name)))

    @contextlib.contextmanager
    def enter(self, s):
        self.stack.append(s)
        yield
        self.stack.pop()

    def noted(self, f):
        def make(*a, **k):
            self.made.append(self.stack[-1])
            return f(*a, **k)

        return make


class Lib:
    def __getattr__(self, name):
        return lambda *a: 4096 if name.endswith("_ws") else 0


def stack():
    s = C.MoeStack.__new__(C.MoeStack)
    s.H, s.E, s.I, s.topk, s.eps, s.fp8, s.lib = H, E, I, K, 1e-6, False, Lib()
    s.layers = [{k: torch.ones(16) for k in C._KEYS}]
    s.packed, s._gemm, s._rows_buf = [], {7: 1, 0: 1}, {}
    return s


CALLS = {
    "rows": lambda s, x, hn, st: s.rows(0, x[:3], hn[:3], stream=st),
    "forward of few rows": lambda s, x, hn, st: s.forward(x[:3], stream=st),
    "forward of many rows": lambda s, x, hn, st: s.forward(x, stream=st),
    "prefill": lambda s, x, hn, st: s.prefill(0, x[:9], hn[:9], stream=st),
}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("handle,want", [(0, "default"), (7, 7)])
def test_buffers_belong_to_the_stream_of_the_kernels(monkeypatch, call, handle, want):
    """A call with the handle of the null stream, or of a created one, while a third stream is torch's current one."""
    s, x = stack(), torch.ones(80, H)
    hn = x.to(torch.bfloat16)
    streams = Streams(monkeypatch)
    with streams.enter("third"):
        CALLS[call](s, x, hn, handle)
    assert streams.made and {getattr(m, "cuda_stream", m) for m in streams.made} == {want}


@pytest.mark.gpu
def test_first_call_on_the_null_stream(tmp_path):
    """rows and forward called first with handle 0 while another stream is the current one and busy: the bits of calls on the
    current stream alone."""
    from ckpt_helpers import write_checkpoint

    write_checkpoint(str(tmp_path), [70, 71], E=64)
    want, st = C.MoeStack(str(tmp_path)), C.MoeStack(str(tmp_path))
    torch.manual_seed(3)
    xs = {n: torch.randn(n, want.H, device="cuda") for n in (5, 100)}
    hn = torch.randn(5, want.H, device="cuda").to(torch.bfloat16)
    a, b = xs[5].clone(), xs[5].clone()
    want.rows(0, a, hn)
    ref = {n: x.clone() for n, x in xs.items()}
    for x in ref.values():
        want.forward(x)
    torch.cuda.synchronize()
    other, big = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        for _ in range(20):
            big = (big @ big).clamp_(-1, 1)
        st.rows(0, b, hn, stream=0)
        for x in xs.values():
            st.forward(x, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(a, b)
    for n in xs:
        assert torch.equal(xs[n], ref[n])
