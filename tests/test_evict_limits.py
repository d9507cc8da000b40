"""Eviction at the ends of the ranges of its whole numbers."""
import pytest
import torch

import attnkernels as ak


def last_index(keep, at, step, bits):
    """The largest j of `for (j = at; j < keep; j += step)` and whether every j is an index of
    [0, keep), with j of `bits` bits, signed at 32 as in C's int."""
    n = -(-(keep - at) // step)
    after = at + n * step  # the j that ends the loop
    wraps = bits == 32 and after >= 1 << 31
    return at + (n - 1) * step, not wraps


@pytest.mark.parametrize("step", [256, 1024, 2048, 8192])
def test_filling_past_an_uncut_sequence_ends(step):
    """keep up to 2^31 - 1: a 32-bit signed index wraps below 0 before the loop ends for some
    thread of every launch shape, an unsigned one does not (2^31 - 1 + 8192 < 2^32)."""
    keep = (1 << 31) - 1
    assert not all(last_index(keep, at, step, 32)[1] for at in range(step))
    for at in range(step):
        assert last_index(keep, at, step, 33) == (keep - 1 - (keep - 1 - at) % step, True)
    assert keep + 8192 < 1 << 32


@pytest.mark.gpu
@pytest.mark.parametrize("n", [37, 20000])
def test_keep_of_any_size(n):
    """keep = 2^31 - 1 as "no limit": nothing is cut, and 8.6 GB of `kept` behind the sequence's
    own indices hold -1."""
    keep, bs = (1 << 31) - 1, 16
    blocks = -(-n // bs)
    cache = torch.randn(blocks, 1, bs, 8, device="cuda")
    before, w = cache.clone(), torch.rand(blocks, 1, bs, device="cuda")
    tables = torch.arange(blocks, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    new_lens, kept = ak.paged_evict((cache,), w, tables, lens, n, tables, keep)
    assert new_lens.tolist() == [n] and kept.shape == (1, 1, keep)
    assert torch.equal(kept[0, 0, :n], torch.arange(n, dtype=torch.int32, device="cuda"))
    tail = kept[0, 0, n:]
    assert int(tail.max()) == int(tail.min()) == -1
    assert torch.equal(cache, before)
    ak.check_device_status()
