"""The 4-bit paged cache and eviction on the GPU against oracle/kvcache.py (64 bits).

Tolerances of the decode tests are bounds, computed per output from the exact
values. With u = 2^-11 (half an fp16 step, relative), p a token's weight and
mid = low + 8 scale:

    P * scale is rounded to fp16, and so is mid:  u sum p scale |code - 8| + u sum p |mid|
    P (two fp16 terms, at most 4, l >= 1), its second term times scale, and P * scale,
    each below fp16's normal range:               N 2^-25 (15 scale + |mid| + 16) / (4 L)
    fp32 sums over the N tokens, two products of 16 at a time:
                                                  (N / 8 + 8) 2^-23 sum p (15 scale + |low|)
    the score's fp32 sum of D products, in units of the exponent:
        d = (D + 32) 2^-24 scale_qk sum |q| (15 scale + |low|) + 2^-22 |s|
      moves p by 2 d + 2^-21 relative (exponential and normaliser)
    the output's own rounding:                    finfo(dtype).eps / 2 |o| + 2^-25

(L = sum 2^(s - max s); terms that multiply each other are covered by a factor 1.1.)
A total of weights moves by (2 d + 2^-21) p, the sum over the group and the add.
"""
import pytest
import torch

import attnkernels as ak
from oracle import kvcache as ora
from oracle.reference import make_paged_cache

pytestmark = pytest.mark.gpu


def tables_for(lens, bs, extra=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-c // bs) for c in lens]
    order = torch.randperm(sum(counts) + extra, generator=g).to(torch.int32)
    bt = torch.zeros(len(lens), max(max(counts), 1), dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        bt[b, :n] = order[at:at + n]
        at += n
    return bt, sum(counts) + extra


def cache4(lens, hkv, d, bs, seed=0, spread=1.0):
    """4-bit caches on the CPU (packed by the oracle), tables; unused rows hold NaN groups."""
    torch.manual_seed(seed)
    bt, blocks = tables_for(lens, bs, seed=seed)
    caches = []
    for value in (False, True):
        x = torch.randn(blocks, hkv, bs, d) * spread
        x[..., ::17] *= 4
        rows = ora.pack(x.half(), value)
        junk = ora.pack(torch.full((blocks, hkv, bs, d), float("nan")).half(), value)
        keep = torch.zeros(blocks, bs, dtype=torch.bool)
        for b, n in enumerate(lens):
            s = ora.slots_of(bt[b], n, bs)
            keep[s // bs, s % bs] = True
        caches.append(torch.where(keep[:, None, :, None], rows, junk))
    return caches[0], caches[1], bt


def check_decode4(lens, hq, hkv, d, bs, dtype=torch.float16, seed=0, spread=1.0,
                  weights=True, max_ctx=None, scale=None):
    kc, vc, bt = cache4(lens, hkv, d, bs, seed, spread)
    g = hq // hkv
    q = torch.randn(len(lens), hq, d).to(dtype)
    init = torch.rand(kc.shape[:3])
    w = init.clone().cuda() if weights else None
    lens_t = torch.tensor(lens, dtype=torch.int32)
    out = ak.paged_decode_kv4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), lens_t.cuda(),
                              max(lens) if max_ctx is None else max_ctx, scale=scale,
                              weights=w)
    assert out.shape == q.shape and out.dtype == dtype
    out = out.cpu().double()
    sc = scale if scale is not None else d ** -0.5
    want_w, tol_w = init.double(), torch.full(init.shape, 0.0).double()
    u = 2.0 ** -11
    for b, n in enumerate(lens):
        for h in range(hkv):
            heads = slice(h * g, (h + 1) * g)
            if n == 0:
                assert (out[b, heads] == 0).all()
                continue
            qd = q[b, heads].double()
            kcode, kscale, klow = ora.parts(ora.rows_of(kc, bt[b], n, h), False)
            vcode, vscale, vlow = ora.parts(ora.rows_of(vc, bt[b], n, h), True)
            k, v = klow + kscale * kcode, vlow + vscale * vcode
            s = qd @ k.T * sc
            o, p = ora.attend(qd, k, v, sc)
            delta = ((d + 32) * 2.0 ** -24 * sc * (qd.abs() @ (15 * kscale + klow.abs()).T)
                     + 2.0 ** -22 * s.abs()).amax(-1, keepdim=True)
            big_l = torch.exp(s - s.amax(-1, keepdim=True)).sum(-1, keepdim=True)
            mid = vlow + 8 * vscale
            mass = p @ (15 * vscale + vlow.abs())
            tol = u * (p @ (vscale * (vcode - 8).abs())) + u * (p @ mid.abs())
            tol += n * 2.0 ** -25 * (15 * vscale.max() + mid.abs().max() + 16) / (4 * big_l)
            tol += (n / 8 + 8) * 2.0 ** -23 * mass + (2 * delta + 2.0 ** -21) * 2 * mass
            tol = 1.1 * tol + torch.finfo(dtype).eps / 2 * o.abs() + 2.0 ** -25
            bad = (out[b, heads] - o).abs() > tol
            assert not bad.any(), (b, h, (out[b, heads] - o).abs().max(), tol.min())
            slots = ora.slots_of(bt[b], n, bs)
            want_w[slots // bs, h, slots % bs] += p.sum(0)
            tol_w[slots // bs, h, slots % bs] += ((2 * delta + 2.0 ** -21) * 1.1 * p).sum(0) + \
                2.0 ** -23 * (p.sum(0) + init[slots // bs, h, slots % bs])
    if weights:
        bad = (w.cpu().double() - want_w).abs() > tol_w
        assert not bad.any(), (w.cpu().double() - want_w).abs().max()
    ak.check_device_status()


# ------------------------------------------------------------------ append, read

def check_append(k, v, bs, slots, blocks, weights=True):
    t, hkv, d = k.shape
    fill = torch.randint(0, 256, (blocks, hkv, bs, ak.kv4_row_bytes(d)), dtype=torch.uint8)
    kc, vc = fill.cuda(), fill.flip(0).contiguous().cuda()
    w0 = torch.rand(blocks, hkv, bs)
    w = w0.cuda() if weights else None
    want_k, want_v, want_w = fill.clone(), fill.flip(0).contiguous(), w0.clone()
    ak.paged_append_kv4(k.cuda(), v.cuda(), kc, vc, slots.cuda(), weights=w)
    rows = ora.pack(k, False), ora.pack(v, True)
    # NaN has many bit patterns: a poisoned group is compared by what it reads as.
    nan_k, nan_v = (~(x.double().unflatten(-1, (-1, 32)).abs() <= 65504).all(-1) for x in (k, v))
    for i, s in enumerate(slots.tolist()):
        if s < 0:
            continue
        for want, row in ((want_k, rows[0]), (want_v, rows[1])):
            want[s // bs, :, s % bs] = row[i]
        want_w[s // bs, :, s % bs] = 0
    for got, want, nan in ((kc, want_k, nan_k), (vc, want_v, nan_v)):
        if not nan.any():
            assert torch.equal(got.cpu(), want)
    if weights:
        assert torch.equal(w.cpu(), want_w)
    for dtype in (torch.float16, torch.bfloat16):
        rk, rv = ak.paged_read_kv4(kc, vc, slots.cuda(), dtype=dtype)
        for got, row, value in ((rk, rows[0], False), (rv, rows[1], True)):
            exact = ora.unpack(row, value)
            exact[slots < 0] = 0
            # One rounding, and that of the fp32 sum before it.
            tol = (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * exact.abs() + 2.0 ** -25
            got = got.cpu().double()
            assert torch.equal(got.isnan(), exact.isnan())
            assert ((got - exact).abs() <= tol)[~exact.isnan()].all()
    ak.check_device_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t,hkv,bs", [(1, 1, 1), (3, 5, 8), (65, 8, 16), (130, 3, 24)])
def test_append(d, dtype, t, hkv, bs):
    blocks = -(-t // bs) + 2
    slots = torch.randperm(blocks * bs)[:t]
    slots[t // 2 + 1::7] = -1
    check_append(torch.randn(t, hkv, d).to(dtype), torch.randn(t, hkv, d).to(dtype) * 3, bs, slots,
                 blocks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_ties_constants_and_extremes(dtype):
    """Quotients exactly between two codes, constant groups (scale 0), groups near fp16's ends,
    subnormal scales."""
    k = torch.zeros(8, 1, 128)
    k[0, 0] = torch.arange(128).remainder(31) * 0.5          # scale 1, every half a tie
    k[1, 0] = 2.5
    k[2, 0] = torch.linspace(-65000, 65000, 128)
    k[3, 0] = torch.arange(128).remainder(16) * 2.0 ** -24   # steps of fp16's smallest number
    k[4, 0] = torch.arange(128).remainder(9) * 2.0 ** -23
    k[5, 0] = torch.tensor([-1.0, 2.0 ** -14] * 64)
    k[6, 0] = torch.randn(128) * 1e-3 + 100
    k[7, 0] = torch.randn(128)
    k = k.to(dtype)
    check_append(k, k.flip(0).contiguous(), 8, torch.arange(8) + 3, 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_non_finite(dtype):
    k = torch.randn(6, 2, 64)
    k[0, 0, 5] = float("inf")
    k[1, 1, 40] = float("nan")
    k[2, 0, 63] = -float("inf")
    if dtype == torch.bfloat16:
        k[3, 1, 0] = 1e6  # finite, beyond fp16
    k = k.to(dtype)
    check_append(k, k.flip(0).contiguous(), 4, torch.arange(6), 2)


def test_append_many_near_borders():
    """Half a million values on a coarse grid, where many quotients are ties or next to one."""
    g = torch.Generator().manual_seed(3)
    k = (torch.randint(-300, 300, (512, 8, 128), generator=g).float() / 64).half()
    k[..., 1::2] += (torch.randn(512, 8, 64, generator=g) * 2.0 ** -9).half()
    check_append(k, k.flip(0).contiguous(), 16, torch.randperm(512, generator=g), 32)


@pytest.mark.parametrize("make", ["heads", "fused", "odd"])
def test_append_strided(make):
    """Slices of a fused projection, a transposed layout, and strides that need a copy."""
    if make == "heads":
        x = torch.randn(4, 33, 128).half()
        k, v = x.transpose(0, 1), x.flip(0).transpose(0, 1)
    elif make == "fused":
        x = torch.randn(33, 12, 128).half()
        k, v = x[:, 4:8], x[:, 8:]
    else:
        x = torch.randn(33, 4, 259).half()
        k, v = x[..., 1:129], x[..., 130:258]
    kc = torch.zeros(4, 4, 16, 80, dtype=torch.uint8, device="cuda")
    vc = torch.zeros_like(kc)
    slots = torch.arange(33, dtype=torch.int32) + 5
    xg = x.cuda()
    kg, vg = (torch.as_strided(xg, t.shape, t.stride(), t.storage_offset()) for t in (k, v)) \
        if make != "heads" else (xg.transpose(0, 1), xg.flip(0).transpose(0, 1))
    ak.paged_append_kv4(kg, vg, kc, vc, slots.cuda())
    rk, rv = ora.pack(k, False), ora.pack(v, True)
    s = slots.long()
    assert torch.equal(kc.cpu()[s // 16, :, s % 16], rk)
    assert torch.equal(vc.cpu()[s // 16, :, s % 16], rv)


def test_append_one_row_of_a_wider_tensor():
    """A single token and head: its strides may be anything, its address unaligned."""
    x = torch.randn(5, 4, 259).half().cuda()
    for at in (0, 1, 3):
        k = x[2:3, 1:2, at:at + 128]
        kc, vc = (torch.zeros(1, 1, 16, 80, dtype=torch.uint8, device="cuda") for _ in range(2))
        ak.paged_append_kv4(k, k, kc, vc, torch.tensor([7]).cuda())
        assert torch.equal(kc[0, 0, 7].cpu(), ora.pack(k.cpu(), False)[0, 0])
        assert torch.equal(vc[0, 0, 7].cpu(), ora.pack(k.cpu(), True)[0, 0])


def test_append_and_read_report_slots_past_the_cache():
    k = torch.randn(3, 2, 64).half().cuda()
    kc = torch.zeros(2, 2, 16, 40, dtype=torch.uint8, device="cuda")
    vc = torch.zeros_like(kc)
    slots = torch.tensor([0, 32, 1 << 40]).cuda()
    ak.paged_append_kv4(k, k, kc, vc, slots)
    assert ak.device_status()[0] == 2
    assert (kc[:, :, 1:] == 0).all() and (kc[1] == 0).all() and (kc[0, :, 0] != 0).any()
    rk, rv = ak.paged_read_kv4(kc, vc, slots)
    assert ak.device_status()[0] == 2
    assert (rk[1:] == 0).all() and (rv[1:] == 0).all() and (rk[0] != 0).any()


def test_append_and_read_nothing():
    kc = torch.zeros(2, 2, 16, 40, dtype=torch.uint8, device="cuda")
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    k = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    ak.paged_append_kv4(k, k, kc, kc.clone(), none)
    rk, rv = ak.paged_read_kv4(kc, kc, none)
    assert rk.shape == (0, 2, 64) and rv.shape == (0, 2, 64)


# ----------------------------------------------------------------- 4-bit decode

EDGES = [1, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65, 255, 256, 257]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8])
def test_decode4_lengths(d, group):
    check_decode4(EDGES, 2 * group, 2, d, 16, seed=group)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bs", [2, 6, 8, 24, 32, 64, 128])
def test_decode4_block_sizes(d, bs):
    check_decode4([300, 1, 50, 17], 8, 2, d, bs, seed=bs)


@pytest.mark.parametrize("bs", [1, 3, 5])
def test_decode4_odd_block_sizes(bs):
    check_decode4([300, 1, 50, 17], 8, 2, 128, bs, seed=bs)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1100, 257, 700, 64], [3] * 40 + [900] + [0] * 20 + [33] * 9,
                                  [31] * 700])
@pytest.mark.parametrize("weights", [False, True])
def test_decode4_runs(dtype, lens, weights):
    """Rows cut into one-stage runs, long rows among short and empty ones, and runs of several
    rows (2800 stages over the GPU's warps)."""
    check_decode4(lens, 16, 4, 128, 16, dtype=dtype, weights=weights)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("spread", [1e-4, 1e-2, 50.0, 4000.0])
def test_decode4_magnitudes(d, spread):
    """K and V far smaller and far larger than 1: scores near 0, or one token that takes all."""
    check_decode4([200, 37], 8, 2, d, 16, spread=spread)


def test_decode4_4d_query_and_scale():
    kc, vc, bt = cache4([90], 2, 64, 16)
    q = torch.randn(1, 6, 1, 64).half().cuda()
    args = (kc.cuda(), vc.cuda(), bt.cuda(), torch.tensor([90]).cuda(), 90)
    out = ak.paged_decode_kv4(q, *args, scale=0.3)
    assert out.shape == q.shape
    assert torch.equal(out[:, :, 0], ak.paged_decode_kv4(q[:, :, 0], *args, scale=0.3))
    check_decode4([90], 6, 2, 64, 16, scale=0.3)


def test_decode4_long_split():
    """A long context in many splits, few rows."""
    check_decode4([20000], 4, 1, 128, 16)


def test_decode4_many_sequences():
    """More sequences than a launch of the fp16 decode takes."""
    torch.manual_seed(1)
    n, bs = 2500, 16
    kc, vc, _ = cache4([64], 1, 64, bs)
    bt = torch.randint(0, 4, (n, 3), dtype=torch.int32)
    lens = torch.randint(0, 49, (n,), dtype=torch.int32)
    q = torch.randn(n, 2, 64).half()
    out = ak.paged_decode_kv4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), lens.cuda(), 48).cpu()
    for b in list(range(0, n, 97)) + [2047, 2048, 2049, n - 1]:
        m = int(lens[b])
        o, _ = ora.attend(q[b], ora.unpack(ora.rows_of(kc, bt[b], m, 0), False),
                          ora.unpack(ora.rows_of(vc, bt[b], m, 0), True))
        # Some of the pages are cache4's NaN ones; the others' rows: the module's bound for values
        # of a few units.
        got = out[b].double()
        assert torch.equal(got.isnan(), o.isnan()), b
        assert ((got - o).abs() < 1e-2)[~o.isnan()].all(), b


@pytest.mark.parametrize("weights", [False, True])
def test_decode4_few_sequences_behind_a_full_launch(weights):
    """2048 sequences and 52 more: the same as two calls."""
    torch.manual_seed(3)
    n, bs = 2100, 16
    kc, vc = (ora.pack(torch.randn(n, 2, bs, 64).half(), v).cuda() for v in (False, True))
    bt = torch.randperm(n).to(torch.int32).view(n, 1).cuda()
    lens = torch.randint(0, 17, (n,), dtype=torch.int32).cuda()
    q = torch.randn(n, 6, 64).half().cuda()
    w, w2 = (torch.zeros(kc.shape[:3], device="cuda") for _ in range(2))
    out = ak.paged_decode_kv4(q, kc, vc, bt, lens, 16, weights=w if weights else None)
    for part in (slice(0, 2048), slice(2048, n)):
        got = ak.paged_decode_kv4(q[part], kc, vc, bt[part], lens[part], 16,
                                  weights=w2 if weights else None)
        assert torch.equal(out[part], got)
    assert torch.equal(w, w2)  # one add per slot
    if weights:
        # Of each sequence 3 heads' weights sum to 3 per kv head.
        sums = w.sum(-1)[bt[:, 0].long()]
        assert (sums - torch.where(lens > 0, 3.0, 0.0)[:, None]).abs().max() < 1e-4


def test_weights_of_many_sequences():
    """Totals over more sequences than a launch takes, every page in one sequence."""
    torch.manual_seed(2)
    n, bs, d, hkv, g = 2300, 16, 64, 2, 2
    bt = torch.randperm(2 * n).to(torch.int32).view(n, 2)
    lens = torch.randint(0, 33, (n,), dtype=torch.int32)
    x = torch.randn(2, 2 * n, hkv, bs, d).half()
    rows = [ora.pack(x[i], i == 1) for i in range(2)]
    q = torch.randn(n, hkv * g, d).half()
    w4, w16 = (torch.zeros(2 * n, hkv, bs, device="cuda") for _ in range(2))
    args = (bt.cuda(), lens.cuda(), 32)
    ak.paged_decode_kv4(q.cuda(), rows[0].cuda(), rows[1].cuda(), *args, weights=w4)
    ak.paged_decode_weights(q.cuda(), x[0].cuda(), x[1].cuda(), *args, w16)
    for b in list(range(0, n, 57)) + [2047, 2048, n - 1]:
        m = int(lens[b])
        s = ora.slots_of(bt[b], 32, bs)
        for h in range(hkv):
            for w, k in ((w4, ora.unpack(ora.rows_of(rows[0], bt[b], m, h), False)),
                         (w16, ora.rows_of(x[0], bt[b], m, h).double())):
                got = w[s // bs, h, s % bs].cpu().double()
                _, p = ora.attend(q[b, g * h:g * h + g], k, k)
                # p moves by 2 d + 2^-21 relative, d below 1e-5 for values of a few units.
                assert ((got[:m] - p.sum(0)).abs() <= 3e-5 * p.sum(0)).all()
                assert (got[m:] == 0).all()


@pytest.mark.parametrize("d,bs", [(128, 1), (128, 3), (64, 2), (64, 6), (128, 40)])
def test_decode4_long_runs_of_small_pages(d, bs):
    """Several stages of a row per warp, each of more pages than a window of the block table
    holds in part, so that windows end inside stages."""
    torch.manual_seed(d + bs)
    n, length = 900, 397
    pool = 3 * (64 // bs + 2)
    kc, vc = (ora.pack(torch.randn(pool, 1, bs, d).half(), v) for v in (False, True))
    bt = torch.randint(0, pool, (n, -(-length // bs)), dtype=torch.int32)
    lens = torch.full((n,), length, dtype=torch.int32)
    q = torch.randn(n, 3, d).half()
    out = ak.paged_decode_kv4(q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), lens.cuda(), length).cpu()
    for b in range(0, n, 41):
        o, _ = ora.attend(q[b], ora.unpack(ora.rows_of(kc, bt[b], length, 0), False),
                          ora.unpack(ora.rows_of(vc, bt[b], length, 0), True))
        # The module's bound for values of a few units.
        assert (out[b].double() - o).abs().max() < 4e-3, b
    ak.check_device_status()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 3, 4, 8])
@pytest.mark.parametrize("weights", [False, True])
def test_decode4_short_rows_beside_a_long_one(d, group, weights):
    """The lengths of test_decode4_lengths where a row is too long for one CTA: runs over all
    warps, parts merged by the finish kernel."""
    check_decode4(EDGES + [2500], 2 * group, 2, d, 16, seed=group, weights=weights)


@pytest.mark.parametrize("d,most", [(64, 2048), (128, 1152)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("weights", [False, True])
def test_decode4_a_row_per_cta(d, most, dtype, weights):
    """Up to two stages for each warp of a CTA, 144 rows; one token more is past that."""
    lens = [most, most - 1, 0, 1, most // 2, most // 2 + 1, most // 2 - 1, 47, 48, 49, 64, 65,
            most - 48, most - 65, 700, 333, most, 2]
    check_decode4(lens, 16, 8, d, 16, dtype=dtype, weights=weights)
    check_decode4(lens[1:] + [most + 1], 16, 8, d, 32, dtype=dtype, weights=weights)


@pytest.mark.parametrize("n", [36, 37, 38])
def test_decode4_about_a_row_per_sm(n):
    """144, 148 and 152 rows."""
    check_decode4([(37 * i) % 150 for i in range(n)], 12, 4, 128, 24, seed=n)


def test_decode4_row_per_cta_at_empty_and_shared_pages():
    """No tokens at all; and pages in several sequences, whose totals get every add."""
    check_decode4([1, 0, 0], 4, 2, 64, 16, max_ctx=1)
    q = torch.randn(2, 4, 128).half().cuda()
    kc, vc, bt = cache4([200], 2, 128, 16)
    kc, vc, bt = kc.cuda(), vc.cuda(), bt.cuda()
    args = (q, kc, vc, bt.expand(2, -1).contiguous())
    w = torch.zeros(kc.shape[:3], device="cuda")
    zero = ak.paged_decode_kv4(*args, torch.tensor([0, 0]).cuda(), 200, weights=w)
    assert (zero == 0).all() and (w == 0).all()
    ak.paged_decode_kv4(*args, torch.tensor([200, 200]).cuda(), 200, weights=w)
    each = torch.zeros_like(w)
    for i in range(2):
        ak.paged_decode_kv4(q[i:i + 1], kc, vc, bt, torch.tensor([200]).cuda(), 200, weights=each)
    # Two fp32 adds to a total of at most 4, in either order: half a step of 2^-22 for each
    # of the two sides' roundings.
    assert (w - each).abs().max() <= 2.0 ** -22
    assert abs(w.sum().item() - 8) < 8 * 200 * 2.0 ** -22 + 1e-4


def test_decode4_cuts_lengths_above_max():
    kc, vc, bt = cache4([300], 2, 128, 16)
    q = torch.randn(1, 8, 128).half().cuda()
    w = torch.zeros(kc.shape[:3], device="cuda")
    args = [t.cuda() for t in (kc, vc, bt)]
    cut = ak.paged_decode_kv4(q, *args, torch.tensor([300]).cuda(), 100, weights=w)
    full = ak.paged_decode_kv4(q, *args, torch.tensor([100]).cuda(), 100)
    assert torch.equal(cut, full)
    slots = ora.slots_of(bt[0], 300, 16)
    assert (w.cpu()[slots[100:] // 16, :, slots[100:] % 16] == 0).all()
    assert (w.cpu()[slots[:100] // 16, :, slots[:100] % 16] > 0).all()


def test_decode4_nan_rows_are_the_rows_that_hold_them():
    """A NaN in one sequence's cache reaches that sequence alone; NaN rows past a sequence's end
    (cache4's unused rows) reach nothing."""
    lens = [40, 21, 48]
    kc, vc, bt = cache4(lens, 1, 64, 16)
    vc[bt[1, 0], 0, 3, 32:] = 0xFF
    q = torch.randn(3, 4, 64).half().cuda()
    out = ak.paged_decode_kv4(q, kc.cuda(), vc.cuda(), bt.cuda(), torch.tensor(lens).cuda(), 48)
    assert out[1].isnan().all() and out[[0, 2]].isfinite().all()


def test_decode4_reports_bad_blocks():
    kc, vc, bt = cache4([100], 2, 128, 16)
    bt[0, 3] = 1 << 20
    w = torch.zeros(kc.shape[:3], device="cuda")
    q = torch.randn(1, 4, 128).half().cuda()
    ak.paged_decode_kv4(q, kc.cuda(), vc.cuda(), bt.cuda(), torch.tensor([100]).cuda(), 100,
                        weights=w)
    assert ak.device_status()[0] == 2
    ak.check_device_status()


def test_decode4_infinite_query():
    """An infinite or NaN query makes its own head's row NaN (or the formula's value), no other's."""
    kc, vc, bt = cache4([40], 1, 64, 16)
    q = torch.randn(1, 4, 64).half()
    q[0, 1, 3] = float("nan")
    q[0, 2, 9] = float("inf")
    args = [t.cuda() for t in (kc, vc, bt)] + [torch.tensor([40]).cuda(), 40]
    out = ak.paged_decode_kv4(q.cuda(), *args)
    assert out[0, 1].isnan().all() and not out[0, 2].isfinite().all()
    clean = q.clone()
    clean[0, 1:3] = 0
    assert torch.equal(out[0, [0, 3]], ak.paged_decode_kv4(clean.cuda(), *args)[0, [0, 3]])


# --------------------------------------------------------- fp16 decode + weights

@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads", [(2, 2), (4, 2), (8, 2), (16, 2)])
@pytest.mark.parametrize("partition", [256, 1024])
def test_decode_weights(d, heads, partition):
    lens = EDGES + [1030]
    bs = 16
    torch.manual_seed(d)
    kc, vc, bt, lens_t = make_paged_cache(lens, heads[1], d, block_size=bs, extra_blocks=3)
    q = torch.randn(len(lens), heads[0], d).half()
    init = torch.rand(kc.shape[:3])
    w = init.cuda()
    args = (q.cuda(), kc.cuda(), vc.cuda(), bt.cuda(), lens_t.cuda(), max(lens))
    out = ak.paged_decode_weights(*args, w, partition_size=partition)
    plain = ak.paged_decode(*args, partition_size=partition)
    # The same softmax, merged from parts where paged_decode may write a row at once: one more
    # fp32 division and product before the same fp16 rounding, which may flip that rounding.
    assert ((out - plain).float().abs() <= 2.0 ** -10 * plain.float().abs() + 2.0 ** -24).all()
    g = heads[0] // heads[1]
    want, tol = init.double(), torch.zeros(init.shape).double()
    for b, n in enumerate(lens):
        for h in range(heads[1]):
            if n == 0:
                continue
            qd = q[b, h * g:(h + 1) * g].double()
            k = ora.rows_of(kc, bt[b], n, h).double()
            _, p = ora.attend(qd, k, k)
            s = ora.slots_of(bt[b], n, bs)
            delta = ((d + 32) * 2.0 ** -24 * d ** -0.5 * (qd.abs() @ k.abs().T) +
                     2.0 ** -22 * (qd @ k.T * d ** -0.5).abs()).amax(-1, keepdim=True)
            want[s // bs, h, s % bs] += p.sum(0)
            tol[s // bs, h, s % bs] += ((2 * delta + 2.0 ** -21) * 1.1 * p).sum(0) + \
                2.0 ** -23 * (p.sum(0) + init[s // bs, h, s % bs])
    assert ((w.cpu().double() - want).abs() <= tol).all()
    ak.check_device_status()


def test_decode_weights_all_nan_keys():
    """A sequence whose keys are all NaN gives NaN, in one part or several, and NaN totals; its
    neighbour is untouched."""
    kc, vc, bt, lens = make_paged_cache([600, 300], 2, 64)
    kc[bt[0].long()] = float("nan")
    for heads in (2, 8):
        for partition in (256, 1024):
            q = torch.randn(2, heads, 64).half().cuda()
            w = torch.zeros(kc.shape[:3], device="cuda")
            out = ak.paged_decode_weights(q, kc.cuda(), vc.cuda(), bt.cuda(), lens.cuda(), 600, w,
                                          partition_size=partition)
            assert out[0].isnan().all() and out[1].isfinite().all()
            s = ora.slots_of(bt[0], 600, 16)
            assert w.cpu()[s // 16, :, s % 16].isnan().all()
            s = ora.slots_of(bt[1], 300, 16)
            assert w.cpu()[s // 16, :, s % 16].isfinite().all()


def test_decode_weights_shared_pages_add_up():
    """Two sequences over the same pages: both adds land."""
    kc, vc, bt, lens = make_paged_cache([200], 2, 64)
    bt2, lens2 = bt.repeat(8, 1), lens.repeat(8)
    q = torch.randn(1, 4, 64).half().repeat(8, 1, 1)
    w1, w8 = (torch.zeros(kc.shape[:3], device="cuda") for _ in range(2))
    ak.paged_decode_weights(q[:1].cuda(), kc.cuda(), vc.cuda(), bt.cuda(), lens.cuda(), 200, w1)
    ak.paged_decode_weights(q.cuda(), kc.cuda(), vc.cuda(), bt2.cuda(), lens2.cuda(), 200, w8)
    # Eight fp32 adds of one value: each rounds by 2^-24 of a sum of at most eight of them.
    assert ((w8 - 8 * w1).abs() <= 8 * 2.0 ** -24 * 8 * w1 + 1e-12).all()


def test_decode_weights_cuts_lengths_above_max():
    kc, vc, bt, _ = make_paged_cache([300], 2, 128)
    q = torch.randn(1, 8, 128).half().cuda()
    w = torch.zeros(kc.shape[:3], device="cuda")
    args = [t.cuda() for t in (kc, vc, bt)]
    cut = ak.paged_decode_weights(q, *args, torch.tensor([300]).cuda(), 100, w)
    full = ak.paged_decode_weights(q, *args, torch.tensor([100]).cuda(), 100, torch.zeros_like(w))
    assert torch.equal(cut, full)
    s = ora.slots_of(bt[0], 300, 16)
    assert (w.cpu()[s[100:] // 16, :, s[100:] % 16] == 0).all()


# ------------------------------------------------------------------------ evict

def check_evict(lens, hkv, bs, keep, recent, sinks, rows=((128,),), dtypes=(torch.float16,),
                totals=None, seed=0, max_ctx=None, same=()):
    torch.manual_seed(seed)
    most = max(lens) if max_ctx is None else max_ctx
    cut = [min(c, keep, most) for c in lens]
    spare = sum(-(-c // bs) for c in cut)
    bt, blocks = tables_for(lens, bs, extra=3 + spare, seed=seed)
    used = {int(p) for b, c in enumerate(lens) for p in bt[b, :-(-c // bs)]}
    free = [p for p in range(blocks) if p not in used]
    new = torch.zeros(len(lens), max(1, max(-(-c // bs) for c in cut)), dtype=torch.int32)
    for b, c in enumerate(cut):
        n = -(-c // bs)
        new[b, :n] = bt[b, :n] if b in same else torch.tensor([free.pop() for _ in range(n)])
    caches = [torch.randn(blocks, hkv, bs, *r).mul(50).to(t) for r, t in zip(rows, dtypes)]
    w = torch.rand(blocks, hkv, bs) if totals is None else totals(blocks, hkv, bs)
    got = [c.cuda() for c in caches]
    got_w = w.cuda()
    new_lens, kept = ak.paged_evict(got, got_w, bt.cuda(), torch.tensor(lens).cuda(), most,
                                    new.cuda(), keep, recent=recent, sinks=sinks)
    assert new_lens.tolist() == cut and new_lens.dtype == torch.int32
    assert kept.shape == (len(lens), hkv, keep)
    want = [c.clone() for c in caches]
    want_w = w.clone()
    for b, c in enumerate(lens):
        for h in range(hkv):
            n = min(c, most)
            idx = ora.select(ora.rows_of(w, bt[b], n, h).tolist(), keep, recent, sinks)
            assert kept[b, h].tolist() == idx + [-1] * (keep - len(idx)), (b, h)
            i, j = torch.tensor(idx, dtype=torch.long), torch.arange(len(idx))
            src, dst = bt[b].long(), new[b].long()
            for a, old in zip(want + [want_w], caches + [w]):
                a[dst[j // bs], h, j % bs] = old[src[i // bs], h, i % bs]
    for a, g in zip(want + [want_w], got + [got_w]):
        # Bit for bit: rows may hold NaN.
        assert torch.equal(g.cpu().contiguous().view(torch.uint8), a.contiguous().view(torch.uint8))
    ak.check_device_status()


@pytest.mark.parametrize("keep,recent,sinks", [(1, 0, 0), (1, 1, 0), (64, 16, 4), (64, 64, 0),
                                               (64, 0, 64), (100, 7, 1), (1500, 10, 4)])
def test_evict(keep, recent, sinks):
    check_evict([1, 63, 64, 65, 0, 1000, 3000], 3, 16, keep, recent, sinks)


@pytest.mark.parametrize("bs", [1, 7, 24, 64])
def test_evict_block_sizes(bs):
    check_evict([300, 77], 2, bs, 50, 8, 2)


@pytest.mark.parametrize("rows,dtypes", [
    (((128,), (128,)), (torch.float16, torch.float16)),
    (((80,), (80,)), (torch.uint8, torch.uint8)),
    (((40,), (40,), ()), (torch.uint8, torch.uint8, torch.int32)),
    (((3,),), (torch.uint8,)),
    (((5,), (64, 2)), (torch.float16, torch.float32)),
    (((8,),) * 8, (torch.float32,) * 8),
])
def test_evict_row_types(rows, dtypes):
    check_evict([200, 90], 2, 16, 60, 8, 2, rows, dtypes)


def test_evict_ties_nan_and_signs():
    def few(blocks, hkv, bs):
        x = torch.randint(0, 3, (blocks, hkv, bs)).float()
        x[torch.rand(x.shape) < 0.1] = float("nan")
        x[torch.rand(x.shape) < 0.1] = -0.0
        x[torch.rand(x.shape) < 0.1] = -float("inf")
        x[torch.rand(x.shape) < 0.1] = float("inf")
        x[torch.rand(x.shape) < 0.1] = -1.5
        return x

    for keep in (5, 100, 290):
        check_evict([300, 290, 150], 2, 16, keep, 3, 1, totals=few)
    check_evict([300], 2, 16, 100, 3, 1, totals=lambda *s: torch.zeros(s))
    check_evict([300], 2, 16, 100, 3, 1, totals=lambda *s: torch.full(s, float("nan")))


def test_evict_uncut_sequences_may_keep_their_pages():
    check_evict([40, 200, 64], 2, 16, 64, 8, 2, same=(0, 2))


def test_evict_cuts_lengths_above_max():
    check_evict([500, 80], 2, 16, 64, 8, 2, max_ctx=300)


@pytest.mark.parametrize("n,bs", [(20000, 16), (70000, 16), (70000, 30), (420000, 16),
                                  (420000, 63)])
def test_evict_long(n, bs):
    """One sequence over a cluster of CTAs, up to more totals than their shared memory holds."""
    check_evict([n], 1, bs, n // 3, 100, 4, rows=((4,),))


def test_evict_many_sequences():
    """More (sequence, head) pairs than the GPU has SMs, lengths from nothing to a few thousand."""
    g = torch.Generator().manual_seed(5)
    check_evict(torch.randint(0, 2500, (60,), generator=g).tolist(), 4, 16, 300, 20, 3,
                rows=((8,),))


def test_evict_reports_bad_blocks():
    kc, vc, bt, lens = make_paged_cache([100], 1, 64, extra_blocks=4, device="cuda")
    w = torch.rand(kc.shape[:3], device="cuda")
    before = kc.clone()
    ak.paged_evict((kc, vc), w, bt, lens, 100, torch.full((1, 2), -3).cuda(), 32)
    assert ak.device_status()[0] == 2 and torch.equal(kc, before)
    bt[0, 2] = 1 << 24
    ak.paged_evict((kc, vc), w, bt, lens, 100, torch.tensor([[9, 10]]).cuda(), 32)
    assert ak.device_status()[0] == 2
    ak.check_device_status()


# --------------------------------------------------------------------- together

@pytest.mark.parametrize("d", [64, 128])
def test_serving_loop(d):
    """Prompt into the 4-bit cache, decode steps that append and accumulate, an eviction, more
    steps over the cut cache; every step's output against the oracle over what the cache holds."""
    torch.manual_seed(d)
    B, hkv, g, bs, prompt, keep = 3, 2, 4, 16, 90, 48
    blocks = 40
    kc, vc = (torch.zeros(blocks, hkv, bs, ak.kv4_row_bytes(d), dtype=torch.uint8, device="cuda")
              for _ in range(2))
    w = torch.rand(blocks, hkv, bs, device="cuda")
    bt = torch.arange(24, dtype=torch.int32).view(3, 8).cuda()
    lens = torch.tensor([prompt, prompt - 7, prompt - 30], dtype=torch.int32).cuda()
    for b in range(B):
        n = int(lens[b])
        x = torch.randn(2, n, hkv, d).half().cuda()
        ak.paged_append_kv4(x[0], x[1], kc, vc, ora.slots_of(bt[b].cpu(), n, bs).cuda(), weights=w)
    total = [[torch.zeros(int(lens[b]), dtype=torch.float64) for _ in range(hkv)] for b in range(B)]

    def step(table):
        at = lens.long()
        slots = table.long().gather(1, (at // bs)[:, None])[:, 0] * bs + at % bs
        x = torch.randn(2, B, hkv, d).half().cuda()
        ak.paged_append_kv4(x[0], x[1], kc, vc, slots, weights=w)
        lens.add_(1)
        q = torch.randn(B, hkv * g, d).half().cuda()
        out = ak.paged_decode_kv4(q, kc, vc, table, lens, table.shape[1] * bs, weights=w)
        out = out.cpu().double()
        for b in range(B):
            for h in range(hkv):
                rows = [ora.rows_of(c.cpu(), table[b].cpu(), int(lens[b]), h) for c in (kc, vc)]
                o, p = ora.attend(q[b, h * g:(h + 1) * g].cpu(), ora.unpack(rows[0], False),
                                  ora.unpack(rows[1], True))
                # fp16 P and output, as in the module's bound, for values below 8 in size.
                assert (out[b, h * g:(h + 1) * g] - o).abs().max() < 3 * 2 ** -11 * 8
                total[b][h] = torch.cat([total[b][h], torch.zeros(1)]) + p.sum(0)

    for _ in range(5):
        step(bt)
    new = torch.arange(24, 40, dtype=torch.int32)[:15].view(3, 5).cuda()
    old = lens.clone()
    lens, kept = ak.paged_evict((kc, vc), w, bt, lens, 128, new, keep, recent=8, sinks=2)
    for b in range(B):
        assert int(lens[b]) == min(int(old[b]), keep)
        for h in range(hkv):
            k = kept[b, h, :int(lens[b])].cpu().long()
            total[b][h] = total[b][h][k]
            got = ora.rows_of(w.cpu(), new[b].cpu(), int(lens[b]), h).double()
            assert (got - total[b][h]).abs().max() < 1e-4
            assert set(range(2)) | set(range(int(old[b]) - 8, int(old[b]))) <= set(k.tolist())
    for _ in range(3):
        step(new)
    ak.check_device_status()


def test_on_another_stream_and_in_graphs():
    """Two graphs captured of the same calls and an eager call on a third stream, replayed at the
    same time: each has scratch of its own."""
    lens = [700, 300]
    kc, vc, bt = [t.cuda() for t in cache4(lens, 2, 128, 16)]
    lt = torch.tensor(lens).cuda().int()
    f16 = torch.randn(2, kc.shape[0], 2, 16, 128, device="cuda").half()
    qs = [torch.randn(2, 8, 128).half().cuda() for _ in range(3)]
    w4 = [torch.zeros(kc.shape[:3], device="cuda") for _ in range(3)]
    w16 = [torch.zeros(kc.shape[:3], device="cuda") for _ in range(3)]

    def calls(i):
        return (ak.paged_decode_kv4(qs[i], kc, vc, bt, lt, 700, weights=w4[i]),
                ak.paged_decode_weights(qs[i], f16[0], f16[1], bt, lt, 700, w16[i],
                                        partition_size=256))

    want = [calls(i) for i in range(3)]
    want_w = [(w4[i].clone(), w16[i].clone()) for i in range(3)]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = calls(i)
        graphs.append((g, out))
    ak.release_workspaces()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for w in w4 + w16:
        w.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i][0].replay()
        with torch.cuda.stream(streams[2]):
            eager = calls(2)
    torch.cuda.synchronize()
    for i, out in enumerate([graphs[0][1], graphs[1][1], eager]):
        assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])
        for got, one in zip((w4[i], w16[i]), want_w[i]):
            # Twenty fp32 adds of one value.
            assert ((got - 20 * one).abs() <= 20 * 2.0 ** -24 * 20 * one + 1e-12).all()
    ak.check_device_status()


def test_append_and_evict_in_a_graph():
    kc, vc, bt = [t.cuda() for t in cache4([200], 2, 64, 16)]
    pad = torch.zeros(8, *kc.shape[1:], dtype=torch.uint8, device="cuda")
    kc, vc = torch.cat([kc, pad]), torch.cat([vc, pad])
    w = torch.rand(kc.shape[:3], device="cuda")
    n = kc.shape[0]
    new = torch.arange(n - 8, n, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([200], dtype=torch.int32, device="cuda")
    k = torch.randn(1, 2, 64).half().cuda()
    slot = (bt[0, 3].long() * 16 + 5).view(1)
    ak.paged_append_kv4(k, k, kc, vc, slot, weights=w)
    first = ak.paged_evict((kc, vc), w, bt, lens, 200, new, 100, recent=8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ak.paged_append_kv4(k, k, kc, vc, slot, weights=w)
        lens2, kept = ak.paged_evict((kc, vc), w, bt, lens, 200, new, 100, recent=8)
    before = [t.clone() for t in (kc, vc, w)]
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, first[1]) and torch.equal(lens2, first[0])
    for a, b in zip(before, (kc, vc, w)):
        assert torch.equal(a, b)
    k.copy_(torch.randn(1, 2, 64).half())
    w[bt[0, 7].long()] += 5
    g.replay()
    torch.cuda.synchronize()
    rk, _ = ak.paged_read_kv4(kc, vc, slot)
    assert ((rk.cpu().double() - ora.unpack(ora.pack(k.cpu(), False), False)).abs() < 4e-3).all()
    assert set(range(7 * 16, 8 * 16)) <= set(kept[0, 0].tolist())


# ----------------------------------------------------------------- hard corners

def test_negative_lengths_and_unused_table_entries():
    """A negative length is an empty sequence; table entries past a sequence's pages may hold
    anything and are not reported."""
    kc, vc, bt = cache4([100, 40], 2, 128, 16)
    bt = torch.cat([bt, torch.full((2, 40), -7, dtype=torch.int32)], 1)
    bt[1, 3:] = 1 << 30
    q = torch.randn(2, 4, 128).half().cuda()
    w = torch.rand(kc.shape[:3], device="cuda")
    args = (kc.cuda(), vc.cuda(), bt.cuda())
    lens = torch.tensor([100, 40]).cuda()
    want = ak.paged_decode_kv4(q, *args, lens, 500, weights=w)
    assert want.isfinite().all()
    out = ak.paged_decode_kv4(q, *args, torch.tensor([100, -5]).cuda(), 500)
    assert (out[1] == 0).all()
    f16 = torch.randn(2, kc.shape[0], 2, 16, 128, device="cuda").half()
    out = ak.paged_decode_weights(q, f16[0], f16[1], args[2], torch.tensor([100, -5]).cuda(), 500, w)
    assert (out[1] == 0).all() and out[0].isfinite().all()
    new = torch.zeros(2, 40, dtype=torch.int32).cuda()
    new_lens, kept = ak.paged_evict((f16[0],), w, args[2], torch.tensor([-5, 0]).cuda(), 500, new, 600)
    assert new_lens.tolist() == [0, 0] and (kept == -1).all()
    ak.check_device_status()


def test_caches_beyond_4_gib():
    """Pages whose byte offsets pass 32 bits, in every operator."""
    hkv, bs, d = 8, 16, 128
    blocks = (1 << 32) // (hkv * bs * 80) + 500
    kc, vc = (torch.empty(blocks, hkv, bs, 80, dtype=torch.uint8, device="cuda") for _ in range(2))
    assert kc.numel() > 1 << 32
    w = torch.empty(blocks, hkv, bs, device="cuda")
    pages = torch.arange(blocks - 1, blocks - 41, -1, dtype=torch.int32, device="cuda").view(2, 20)
    n = 150
    slots = (pages.long()[:, :, None] * bs + torch.arange(bs, device="cuda")).flatten(1)[:, :n]
    k, v = (torch.randn(2 * n, hkv, d).half() for _ in range(2))
    ak.paged_append_kv4(k.cuda(), v.cuda(), kc, vc, slots.flatten(), weights=w)
    assert (w.view(blocks, hkv, bs)[slots.flatten() // bs, :, slots.flatten() % bs] == 0).all()
    rk, rv = ak.paged_read_kv4(kc, vc, slots.flatten())
    for got, x, value in ((rk, k, False), (rv, v, True)):
        exact = ora.unpack(ora.pack(x, value), value)
        assert ((got.cpu().double() - exact).abs() <= 2.0 ** -10 * exact.abs() + 2.0 ** -24).all()
    q = torch.randn(2, 2 * hkv, d).half()
    lens = torch.tensor([n, n - 3], dtype=torch.int32, device="cuda")
    out = ak.paged_decode_kv4(q.cuda(), kc, vc, pages, lens, n, weights=w).cpu().double()
    kd, vd = (ora.unpack(ora.pack(x, i == 1), i == 1).view(2, n, hkv, d) for i, x in enumerate((k, v)))
    for b in range(2):
        for h in range(hkv):
            m = int(lens[b])
            o, p = ora.attend(q[b, 2 * h:2 * h + 2], kd[b, :m, h], vd[b, :m, h])
            assert (out[b, 2 * h:2 * h + 2] - o).abs().max() < 4e-3
            got = w[slots[b] // bs, h, slots[b] % bs][:m].cpu().double()
            assert (got - p.sum(0)).abs().max() < 1e-5
    new = torch.tensor([[blocks - 60], [blocks - 70]], dtype=torch.int32, device="cuda")
    src = kc[pages[0, 0].item(), 3, 2].clone()
    w[pages[0, 0].item(), 3, 2] = 9.0
    new_lens, kept = ak.paged_evict((kc, vc), w, pages, lens, n, new, 16, recent=4)
    at = kept[0, 3].tolist().index(2)
    assert torch.equal(kc[blocks - 60, 3, at], src) and w[blocks - 60, 3, at] == 9.0
    ak.check_device_status()


def test_fp16_weights_cache_beyond_4_gib():
    hkv, bs, d = 8, 16, 128
    blocks = (1 << 32) // (hkv * bs * d * 2) + 50
    kc, vc = (torch.empty(blocks, hkv, bs, d, dtype=torch.float16, device="cuda") for _ in range(2))
    pages = torch.arange(blocks - 1, blocks - 7, -1, dtype=torch.int32, device="cuda")[None]
    kc[pages[0].long()] = torch.randn(6, hkv, bs, d).half().cuda()
    vc[pages[0].long()] = torch.randn(6, hkv, bs, d).half().cuda()
    w = torch.zeros(blocks, hkv, bs, device="cuda")
    q = torch.randn(1, hkv, d).half().cuda()
    lens = torch.tensor([90], dtype=torch.int32, device="cuda")
    out = ak.paged_decode_weights(q, kc, vc, pages, lens, 90, w)
    sub = [c[pages[0].long()].contiguous() for c in (kc, vc)]
    ws = torch.zeros(6, hkv, bs, device="cuda")
    small = ak.paged_decode_weights(q, *sub, torch.arange(6, dtype=torch.int32, device="cuda")[None],
                                    lens, 90, ws)
    assert torch.equal(out, small) and torch.equal(w[pages[0].long()], ws)


def test_repeated_calls_give_the_same_bits():
    """The split goes by sizes alone, and a total with one adder has one order: bit for bit."""
    lens = [900, 33, 512]
    kc, vc, bt = [t.cuda() for t in cache4(lens, 4, 128, 16)]
    f16 = torch.randn(2, kc.shape[0], 4, 16, 128, device="cuda").half()
    q = torch.randn(3, 16, 128).half().cuda()
    lt = torch.tensor(lens).cuda()
    first = None
    for _ in range(5):
        w4, w16 = (torch.zeros(kc.shape[:3], device="cuda") for _ in range(2))
        got = (ak.paged_decode_kv4(q, kc, vc, bt, lt, 900, weights=w4), w4,
               ak.paged_decode_weights(q, f16[0], f16[1], bt, lt, 900, w16), w16)
        if first is None:
            first = got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_tensors_made_on_another_stream():
    """Inputs produced on a side stream that the call's stream has waited for."""
    side = torch.cuda.Stream()
    kc, vc, bt = cache4([200], 2, 64, 16)
    with torch.cuda.stream(side):
        q = torch.randn(1, 4, 64, device="cuda").half()
        args = [t.cuda(non_blocking=True) for t in (kc, vc, bt)] + \
            [torch.tensor([200], device="cuda"), 200]
    torch.cuda.current_stream().wait_stream(side)
    here = ak.paged_decode_kv4(q, *args)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        there = ak.paged_decode_kv4(q, *args)
    torch.cuda.synchronize()
    assert torch.equal(here, there)
