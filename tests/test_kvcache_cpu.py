"""Host side of the 4-bit cache and of eviction, on CPU: refusals of the Python
functions and of the C ABI, row sizes, and the oracle's packing against itself."""
import ctypes

import pytest
import torch

import attnkernels as ak
from attnkernels import _native
from oracle import kvcache as ora

P = ctypes.c_void_p(4096)


@pytest.fixture(scope="module")
def lib():
    return _native.library()


def err(lib):
    return lib.attn_last_error().decode()


def test_row_bytes(lib):
    for d in (64, 128):
        assert ak.kv4_row_bytes(d) == lib.attn_kv4_row_bytes(d) == ora.row_bytes(d)
    assert lib.attn_kv4_row_bytes(96) == 0
    with pytest.raises(ValueError):
        ak.kv4_row_bytes(96)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("value", [False, True])
def test_oracle_pack_round_trip(d, value):
    x = torch.randn(5, 3, d).half()
    code, scale, low = ora.quantise(x)
    got_code, got_scale, got_low = ora.parts(ora.pack(x, value), value)
    assert torch.equal(got_code.long(), code)
    assert torch.equal(got_scale[..., ::32], scale.double())
    assert torch.equal(got_low[..., ::32], low.double())
    # Within half a step of the input, plus what rounding the scale to fp16 loses at code 15.
    back = ora.unpack(ora.pack(x, value), value)
    step = got_scale
    assert ((back - x.double()).abs() <= step * (0.5 + 15 * 2 ** -11)).all()
    byte, shift = ora.code_places(d, value)
    assert sorted(zip(byte, shift)) == [(i, s) for i in range(d // 2) for s in (0, 4)]


def kv(t=4, h=2, d=64, dtype=torch.float16):
    return torch.zeros(t, h, d, dtype=dtype)


def cache4(blocks=3, h=2, bs=16, d=64):
    return torch.zeros(blocks, h, bs, ak.kv4_row_bytes(d), dtype=torch.uint8)


def refused(fn, *args, **kw):
    with pytest.raises(ValueError):
        fn(*args, **kw)


def test_append_refusals():
    c, s = cache4(), torch.arange(4)
    refused(ak.paged_append_kv4, kv(), kv(), c, c, s)  # CPU tensors
    refused(ak.paged_append_kv4, kv(dtype=torch.float32), kv(dtype=torch.float32), c, c, s)
    refused(ak.paged_append_kv4, kv(), kv(t=5), c, c, s)
    refused(ak.paged_append_kv4, kv(d=128), kv(d=128), c, c, s)
    refused(ak.paged_append_kv4, kv(h=3), kv(h=3), c, c, s)
    refused(ak.paged_append_kv4, kv(), kv(), c, c, s[:3])
    refused(ak.paged_append_kv4, kv(), kv(), c, c, s.float())
    refused(ak.paged_append_kv4, kv(), kv(), c.transpose(0, 1), c.transpose(0, 1), s)
    refused(ak.paged_append_kv4, kv(), kv(), c, c, s, weights=torch.zeros(3, 2, 8))
    refused(ak.paged_read_kv4, c, c, s, dtype=torch.float32)
    refused(ak.paged_read_kv4, c.float(), c.float(), s)


def test_decode_refusals():
    c = cache4()
    q, bt, lens = torch.zeros(2, 4, 64).half(), torch.zeros(2, 3).int(), torch.ones(2).int()
    refused(ak.paged_decode_kv4, q, c, c, bt, lens, 1)  # CPU tensors
    refused(ak.paged_decode_kv4, q.float(), c, c, bt, lens, 1)
    refused(ak.paged_decode_kv4, q.half()[..., :32], c, c, bt, lens, 1)
    refused(ak.paged_decode_kv4, q, cache4(d=128), cache4(d=128), bt, lens, 1)
    refused(ak.paged_decode_kv4, q, c, c, bt[:1], lens, 1)
    refused(ak.paged_decode_kv4, q, c, c, bt, lens[:1], 1)
    refused(ak.paged_decode_kv4, q[:, :, None].expand(2, 4, 2, 64), c, c, bt, lens, 1)
    kc, w = torch.zeros(3, 2, 16, 64).half(), torch.zeros(3, 2, 16)
    refused(ak.paged_decode_weights, q, kc, kc, bt, lens, 1, w)  # CPU tensors
    refused(ak.paged_decode_weights, q, kc, kc, bt, lens, 1, w.half())
    refused(ak.paged_decode_weights, q, kc, kc, bt, lens, 1, w[:2])
    refused(ak.paged_decode_weights, q.bfloat16(), kc, kc, bt, lens, 1, w)


def test_evict_refusals():
    c, w = cache4(), torch.zeros(3, 2, 16)
    bt, lens, new = torch.zeros(2, 3).int(), torch.ones(2).int(), torch.zeros(2, 1).int()
    refused(ak.paged_evict, (c,), w, bt, lens, 1, new, 4)  # CPU tensors
    refused(ak.paged_evict, (), w, bt, lens, 1, new, 4)
    refused(ak.paged_evict, (c,) * 9, w, bt, lens, 1, new, 4)
    refused(ak.paged_evict, (c[:2],), w, bt, lens, 1, new, 4)
    refused(ak.paged_evict, (c,), w.half(), bt, lens, 1, new, 4)
    refused(ak.paged_evict, (c,), w, bt, lens, 1, new, 4, recent=3, sinks=2)
    refused(ak.paged_evict, (c,), w, bt, lens, 1, new, 0)
    refused(ak.paged_evict, (c,), w, bt, lens, 1, new[:1], 4)
    refused(ak.paged_evict, (c,), w, bt, lens[:1], 1, new, 4)


def decode4(lib, **kw):
    a = dict(q=P, dtype=0, batch=2, hq=8, hkv=8, d=128, bs=16, nblk=10, maxb=5, max_ctx=80,
             ws=P, ws_bytes=1 << 30, weights=None)
    a.update(kw)
    return lib.attn_kv4_decode(a["q"], a["dtype"], P, P, P, P, P, a["weights"], a["batch"], a["hq"],
                               a["hkv"], a["d"], a["bs"], a["nblk"], a["maxb"], a["max_ctx"], 0.1,
                               a["ws"], a["ws_bytes"], None)


def test_abi_decode_refusals(lib):
    assert decode4(lib, hq=6, hkv=4) == 1 and "multiple of num_kv_heads" in err(lib)
    assert decode4(lib, hq=72, hkv=8) == 2 and "1 to 8" in err(lib)
    assert decode4(lib, d=96) == 2 and "head_dim" in err(lib)
    assert decode4(lib, dtype=2) == 2 and "dtype" in err(lib)
    assert decode4(lib, d=64, bs=15) == 2 and "even block_size" in err(lib)
    assert decode4(lib, max_ctx=81) == 1 and "max_blocks_per_seq" in err(lib)
    assert decode4(lib, nblk=0) == 1
    assert decode4(lib, q=None) == 1 and decode4(lib, q=ctypes.c_void_p(4098)) == 1
    # 4100: misaligned for 16-byte copies, fine for fp32; here as the totals.
    assert decode4(lib, weights=ctypes.c_void_p(4097)) == 1 and "weights" in err(lib)
    p4104 = ctypes.c_void_p(4104)
    assert decode4(lib, ws=p4104) == 4 and decode4(lib, ws_bytes=16) == 4 and \
        "workspace" in err(lib)
    assert decode4(lib, batch=0) == 0


def test_abi_append_and_read_refusals(lib):
    def append(k=P, dtype=0, tokens=4, hkv=2, d=64, stride=128, bs=16, nblk=3):
        return lib.attn_kv4_append(k, P, dtype, P, P, P, None, tokens, hkv, d, stride, 64, 128, 64,
                                   bs, nblk, None)

    assert append(k=None) == 1 and append(dtype=5) == 2 and append(d=80) == 2
    assert append(stride=129) == 1 and "multiples of 8" in err(lib)
    assert append(tokens=-1) == 1 and append(bs=0) == 1
    assert append(tokens=1 << 31) == 2
    assert append(tokens=0) == 0
    assert lib.attn_kv4_read(P, P, None, P, P, 0, 4, 2, 64, 16, 3, None) == 1
    assert lib.attn_kv4_read(P, P, P, P, P, 0, 0, 2, 64, 16, 3, None) == 0


def test_abi_evict_refusals(lib):
    def evict(n=1, row=80, weights=P, batch=2, hkv=2, bs=16, nblk=9, maxb=4, max_ctx=64, newb=2,
              keep=32, recent=4, sinks=4):
        k = max(1, min(n, 9))
        return lib.attn_paged_evict((ctypes.c_void_p * k)(*[4096] * k), (ctypes.c_int64 * k)(*[row] * k),
                                    n, weights, P, P, P, P, P, batch, hkv, bs, nblk, maxb, max_ctx,
                                    newb, keep, recent, sinks, None)

    assert evict(n=0) == 1 and evict(n=9) == 1 and evict(row=0) == 1 and evict(weights=None) == 1
    assert evict(recent=30, sinks=4) == 1 and "keep at most" in err(lib)
    assert evict(newb=1) == 1 and "too few" in err(lib)
    assert evict(max_ctx=65) == 1 and evict(bs=0) == 1 and evict(keep=-1) == 1
    assert evict(batch=1 << 30, hkv=4) == 2
    assert evict(batch=0) == 0


def test_abi_weights_refusals(lib):
    def weights(w=P, ws=P, ws_bytes=1 << 30, hq=8, max_ctx=80):
        return lib.attn_paged_decode_weights(P, P, P, P, P, P, w, 2, hq, 8, 128, 16, 10, 5, max_ctx,
                                             0.1, 256, ws, ws_bytes, None)

    need = lib.attn_paged_decode_weights_workspace_bytes(2, 8, 8, 128, 80, 256)
    base = lib.attn_paged_decode_workspace_bytes(2, 8, 128, 80, 256)
    assert need == base + 2 * 8 * 80 * 4
    assert weights(w=None) == 1 and weights(hq=24) == 2 and weights(max_ctx=81) == 1
    assert weights(ws_bytes=base) == 4 and "paged_decode_weights" in err(lib)


class _OneAtATime:
    """A library whose decode calls take a while and record whether two of them had
    the same workspace at once, as a second thread's launches between two of the
    first one's would."""

    def __init__(self):
        import threading
        self.inside, self.overlap, self.guard = set(), False, threading.Lock()

    def _decode(self, *args):
        import time
        ws = args[-3]
        with self.guard:
            self.overlap |= ws in self.inside
            self.inside.add(ws)
        time.sleep(0.01)
        with self.guard:
            self.inside.discard(ws)
        return 0

    attn_kv4_decode = attn_paged_decode_weights = _decode


def _fake_extension(monkeypatch):
    """An Extension over _OneAtATime: no GPU, workspaces of 1 KiB and more on the CPU."""
    ext = _native.Extension.__new__(_native.Extension)
    ext.lib = _OneAtATime()
    monkeypatch.setattr(_native, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(_native, "_workspace", lambda n, device: torch.empty(n, dtype=torch.uint8))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ak.release_workspaces()
    return ext


def test_threads_on_one_stream_take_turns(monkeypatch):
    import threading
    ext = _fake_extension(monkeypatch)
    q = torch.zeros(1, 8, 64, dtype=torch.float16)
    kc = torch.zeros(1, 8, 16, 40, dtype=torch.uint8)
    t, w = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 8, 16)
    sizes = (1, 8, 8, 64, 16, 1, 1)

    def four_bit():
        for _ in range(5):
            ext.kv4_decode(0, q, kc, kc, t, t[0], None, sizes, 16, 1.0)

    def weights():
        for _ in range(5):
            ext.paged_decode_weights(0, q, kc, kc, t, t[0], w, sizes, 16, 1.0, 128)

    threads = [threading.Thread(target=f) for f in (four_bit, weights, four_bit, weights)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    ak.release_workspaces()
    assert not ext.lib.overlap


def test_paged_decode_keeps_its_scratch(monkeypatch):
    """A captured paged_decode holds the address of its buffer."""
    ext = _fake_extension(monkeypatch)
    kept = _native._decode_ws.get(1 << 20, torch.device("cuda", 0), 0)
    q = torch.zeros(512, 8, 64, dtype=torch.float16)
    kc = torch.zeros(1, 8, 16, 40, dtype=torch.uint8)
    t = torch.zeros(512, 64, dtype=torch.int32)
    w = torch.zeros(1, 8, 16)
    ext.kv4_decode(0, q, kc, kc, t, t[:, 0], w, (512, 8, 8, 64, 16, 1, 64), 1024, 1.0)
    assert _native._workspace_bytes("attn_kv4_decode_workspace_bytes", 512, 8, 8, 64, 1024,
                                    1) > kept.numel()
    assert _native._decode_ws.kept(0, 0) is kept
    ak.release_workspaces()
    assert _native._decode_ws._bufs == {} == _native._cache_ws._bufs
