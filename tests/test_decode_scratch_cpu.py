"""Which scratch the decode calls take, on CPU with a library that only looks at its arguments:
while a graph is captured scratch of the capture's own, otherwise the stream's kept buffer."""
import contextlib
import threading
import types

import pytest
import torch

import attnkernels as ak
from attnkernels import _native

CALLS = ["paged_decode", "paged_decode_partials", "paged_decode_weights", "kv4_decode"]


class Library:
    """The decode entry points: each notes the address of its workspace."""

    def __init__(self):
        self.seen = []

    def _decode(self, *args):
        self.seen.append(args[-3])
        return 0

    attn_paged_decode = attn_paged_decode_partials = _decode
    attn_paged_decode_weights = attn_kv4_decode = _decode

    @staticmethod
    def attn_paged_decode_workspace_bytes(*sizes):
        return 1 << 16


@pytest.fixture
def ext(monkeypatch):
    e = _native.Extension.__new__(_native.Extension)
    e.lib = Library()
    e.stream, e.capturing, e.made = 0, False, []

    def workspace(nbytes, device):
        # Held on to, so that no two have one address.
        e.made.append(torch.empty(max(nbytes, 256), dtype=torch.uint8))
        return e.made[-1]

    monkeypatch.setattr(_native, "_raw_stream", lambda dev: e.stream)
    monkeypatch.setattr(_native, "_workspace", workspace)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: e.capturing)
    ak.release_workspaces()
    yield e
    ak.release_workspaces()


def call(e, name, dev=0):
    q = torch.zeros(1, 8, 64, dtype=torch.float16)
    kc = torch.zeros(1, 8, 16, 64, dtype=torch.float16)
    t, w, sizes = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 8, 16), (1, 8, 8, 64, 16, 1, 1)
    if name.startswith("paged_decode") and name != "paged_decode_weights":
        getattr(e, name)(q, kc, kc, t, t[0], 16, 1.0, 256)
    elif name == "kv4_decode":
        e.kv4_decode(dev, q, kc, kc, t, t[0], None, sizes, 16, 1.0)
    else:
        e.paged_decode_weights(dev, q, kc, kc, t, t[0], w, sizes, 16, 1.0, 256)
    return e.lib.seen[-1]


@pytest.mark.parametrize("name", CALLS)
def test_a_capture_has_scratch_of_its_own(ext, name):
    """The kept buffer is given back by a larger call or release_workspaces(), and two graphs
    captured on one stream may replay at the same time: neither may hold it."""
    kept = call(ext, name)
    assert call(ext, name) == kept
    ext.capturing = True
    first, second = call(ext, name), call(ext, name)
    assert len({kept, first, second}) == 3
    ext.capturing = False
    assert call(ext, name) == kept


@pytest.mark.parametrize("name", CALLS)
def test_a_capture_keeps_nothing_for_later_calls(ext, name):
    """Scratch from a graph's private pool is the graph's: no eager call may use it."""
    ext.capturing = True
    captured = call(ext, name)
    ext.capturing = False
    assert call(ext, name) != captured


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("same", [False, True])
def test_calls_wait_for_their_own_stream_alone(ext, monkeypatch, name, same):
    """A launch that blocks (a full queue) holds back calls that share its scratch, and no call
    on another stream."""
    stream = threading.local()
    monkeypatch.setattr(_native, "_raw_stream", lambda dev: stream.handle)
    inside, leave, other = threading.Event(), threading.Event(), threading.Event()

    def decode(*args):
        if args[-1] == 1 and not inside.is_set():
            inside.set()
            leave.wait(20)
        return 0

    def run(handle, done=None):
        stream.handle = handle
        call(ext, name)
        if done is not None:
            done.set()

    monkeypatch.setattr(ext, "lib", types.SimpleNamespace(
        seen=[0], attn_paged_decode_workspace_bytes=Library.attn_paged_decode_workspace_bytes,
        **{"attn_" + n: decode for n in CALLS}))
    first = threading.Thread(target=run, args=(1,))
    second = threading.Thread(target=run, args=(1 if same else 2, other))
    first.start()
    assert inside.wait(20)
    second.start()
    try:
        assert other.wait(0.3 if same else 10) != same
    finally:
        leave.set()
        first.join()
        second.join()
    assert other.is_set()


@pytest.mark.parametrize("capturing", [0, 1])
@pytest.mark.parametrize("name", ["paged_decode_weights", "kv4_decode"])
def test_the_capture_that_counts_is_the_tensors_device(ext, monkeypatch, name, capturing):
    """Tensors on device 1, device 0 current: device 1's stream is asked, not device 0's."""
    at = [0]

    @contextlib.contextmanager
    def device(index):
        before, at[0] = at[0], index
        yield
        at[0] = before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    kept = call(ext, name, dev=1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: at[0] == capturing)
    assert (call(ext, name, dev=1) == kept) == (capturing == 0)
    assert at == [0]
