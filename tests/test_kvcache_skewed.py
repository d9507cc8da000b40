"""One long sequence among many short ones, as continuous batching has them, with weights; and
eviction of 4-bit rows at serving sizes. Bounds: tests/test_kvcache.py."""
import pytest
import torch

import attnkernels as ak
from oracle import kvcache as ora
from oracle.reference import make_paged_cache
from test_kvcache import check_decode4, check_evict

pytestmark = pytest.mark.gpu

SKEWED = [90, 17, 0, 33000, 100] + [(i * 41) % 101 for i in range(40)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("weights", [False, True])
def test_decode4_a_long_sequence_among_short_ones(d, weights):
    check_decode4(SKEWED, 8, 2, d, 16, weights=weights)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [(2, 2), (8, 2)])
def test_decode_weights_a_long_sequence_among_short_ones(d, heads):
    torch.manual_seed(d)
    kc, vc, bt, lens = make_paged_cache(SKEWED, heads[1], d, block_size=16, extra_blocks=3)
    q = torch.randn(len(SKEWED), heads[0], d).half()
    w = torch.zeros(kc.shape[:3], device="cuda")
    args = (q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), lens.cuda(), max(SKEWED))
    out = ak.paged_decode_weights(*args, w).cpu().double()
    w = w.cpu().double()
    g = heads[0] // heads[1]
    for b, n in enumerate(SKEWED):
        for h in range(heads[1]):
            qd = q[b, h * g:(h + 1) * g].double()
            k, v = (ora.rows_of(c, bt[b], n, h).double() for c in (kc, vc))
            o, p = ora.attend(qd, k, v)
            if n == 0:
                assert (out[b, h * g:(h + 1) * g] == 0).all()
                continue
            s = ora.slots_of(bt[b], n, 16)
            delta = ((d + 32) * 2.0 ** -24 * d ** -0.5 * (qd.abs() @ k.abs().T) +
                     2.0 ** -22 * (qd @ k.T * d ** -0.5).abs()).amax(-1, keepdim=True)
            tol = ((2 * delta + 2.0 ** -21) * 1.1 * p).sum(0) + 2.0 ** -23 * p.sum(0)
            assert ((w[s // 16, h, s % 16] - p.sum(0)).abs() <= tol).all()
            # P (of one head alone in fp32, else in fp16, below its range by 2^-25 of a sum of at
            # least 1), weights moved as above, fp32 sums, and the output's rounding.
            mass = p @ v.abs()
            tol = (2.0 ** -11 + 2 * (2 * delta + 2.0 ** -21) + (n / 8 + 8) * 2.0 ** -23) * mass
            big_l = torch.exp((qd @ k.T) * d ** -0.5)
            big_l = (big_l / big_l.amax(-1, keepdim=True)).sum(-1, keepdim=True)
            tol = 1.1 * (tol + 2.0 ** -25 * v.abs().sum(0) / big_l) + 2.0 ** -11 * o.abs() + 2.0 ** -25
            assert ((out[b, h * g:(h + 1) * g] - o).abs() <= tol).all()
    ak.check_device_status()


@pytest.mark.parametrize("row", [40, 80])
def test_evict_4bit_rows_of_a_serving_batch(row):
    """Scattered 40- and 80-byte rows of K and V; lengths from nothing to 4096."""
    lens = [4096, 0, 1, 511, 512, 513] + [(i * 40503) % 4097 for i in range(18)]
    check_evict(lens, 4, 16, 512, 64, 4, rows=((row,), (row,)), dtypes=(torch.uint8, torch.uint8))
