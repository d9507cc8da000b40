"""How far the 4-bit decode's outputs are from 64 bits over a long context, for values of V of
any size: the RMS error of all outputs against the RMS of the roundings that the operator
chooses. Unlike the worst case that tests/test_kvcache.py allows each output, this does not grow
with the number of tokens.

Each rounding is off by a uniform part of half a step, a third of its square on average, and the
roundings of different tokens are independent, so that their squares add up. With u = 2^-11 (half
an fp16 step, relative), p a token's weight, `code`, `scale` and `low` of its group:

    P * scale, rounded to fp16, times code less 8 or 7:    (u p scale (|code - 7.5| + 1/2))^2 / 3
    the group's middle, low + 8 (or 7) scale, in fp16:     (u p mid)^2 / 3
    the output's own rounding:                             step(o)^2 / 12

The scores' and the sums' fp32 roundings (below 2^-17 of a weight for scores of this size) are
left out, and a factor 1.5 stands for them and for the scatter of an RMS over some hundred outputs.

One set of pages stands in every sequence of a batch: with so many rows a warp has thousands of
tokens of a row after one another, all by one running maximum, where a single sequence is dealt out
to the warps a stage or two each.
"""
import pytest
import torch

import attnkernels as ak
from oracle import kvcache as ora

pytestmark = pytest.mark.gpu


def step(o, dtype):
    """Distance of neighbouring numbers of `dtype` at |o|."""
    info = torch.finfo(dtype)
    exponent = torch.frexp(o.abs())[1] - 1
    return (torch.ldexp(torch.full_like(o, info.eps), exponent)).clamp(min=info.smallest_normal *
                                                                        info.eps)


def outputs(k, v, dtype, group, bs=16, spread=2.0, batch=1, q=None):
    """k, v [n, H_kv, D] as the context of `batch` sequences: (output, exact, variance), each
    [looked at, H_kv * group, D], with scores of deviation `spread` for keys of deviation 1."""
    n, hkv, d = k.shape
    q = (torch.randn(batch, hkv * group, d) * spread).to(dtype) if q is None else q
    pad = torch.zeros(-n % bs, hkv, d).half()
    rows = [ora.pack(torch.cat([x.half(), pad]), i == 1) for i, x in enumerate((k, v))]
    kc, vc = (r.view(-1, bs, hkv, r.shape[-1]).transpose(1, 2).contiguous() for r in rows)
    pages = torch.randperm(kc.shape[0])
    tables = torch.argsort(pages).int()[None].expand(batch, -1)
    out = ak.paged_decode_kv4(q.cuda(), kc[pages].cuda(), vc[pages].cuda(), tables.cuda(),
                              torch.full((batch,), n).cuda(), n).cpu().double()
    look = sorted({0, batch // 3, 2 * batch // 3, batch - 1})
    out, q = out[look], q[look]
    exact, var = torch.empty_like(out), torch.empty_like(out)
    u2 = 2.0 ** -22 / 3
    for h in range(hkv):
        heads = slice(h * group, (h + 1) * group)
        code, scale, low = ora.parts(rows[1][:n, h], True)
        kd, vd = ora.unpack(rows[0][:n, h], False), low + scale * code
        mid = torch.maximum((low + 7 * scale).abs(), (low + 8 * scale).abs())
        chosen = u2 * ((scale * ((code - 7.5).abs() + 0.5)).square() + mid.square())
        for i in range(len(look)):
            o, p = ora.attend(q[i, heads], kd, vd)
            exact[i, heads] = o
            var[i, heads] = p.square() @ chosen + step(o, dtype).square() / 12
    ak.check_device_status()
    return out, exact, var


def check(out, exact, var):
    """Each group of 32 columns by itself."""
    err = (out - exact).square().flatten(0, -2).unflatten(-1, (-1, 32)).mean((0, 2)).sqrt()
    want = var.flatten(0, -2).unflatten(-1, (-1, 32)).mean((0, 2)).sqrt()
    assert (err <= 1.5 * want).all(), (err / want).tolist()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [30.0, 1.0, 1e-3, 1e-4])
@pytest.mark.parametrize("n,batch", [(5000, 1), (65536, 1), (32768, 512)])
def test_values_of_any_size(d, dtype, size, n, batch):
    """The weights that count are 2^-10 or so of the largest: with V of 1e-4 their products with
    the scales are below fp16's range, whose numbers end at 2^-24."""
    check(*outputs(torch.randn(n, 2, d), torch.randn(n, 2, d) * size, dtype, 8, batch=batch))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_groups_of_different_size(dtype):
    """Columns of 8, 1, 1e-2 and 1e-3 in one row: the large ones take nothing from the small."""
    size = torch.tensor([1.0, 8.0, 1e-3, 1e-2]).repeat_interleave(32)
    check(*outputs(torch.randn(20000, 2, 128), torch.randn(20000, 2, 128) * size, dtype, 8,
                   batch=512))


@pytest.mark.parametrize("large", [40.0, 400.0])
def test_a_few_large_tokens_far_apart(large):
    """V of some tokens far larger than of the others, seen first, in the middle and last, with
    weights next to nothing: their keys point away from every query."""
    n, d, batch = 20000, 128, 512
    k, v = torch.randn(n, 1, d), torch.randn(n, 1, d) * 0.05
    k[..., :32] = 0
    at = torch.tensor([0, 1, 47, 48, 9000, 9001, 17011, n - 1])
    k[at, :, 0] = -40.0
    v[at] = torch.randn(8, 1, d) * large
    q = torch.randn(batch, 4, d) * 2
    q[..., 0] = 8.0  # 8 * 40 / sqrt(128): the large tokens' scores are 28 below the others'
    check(*outputs(k, v, torch.bfloat16, 4, batch=batch, q=q.bfloat16()))


@pytest.mark.parametrize("d", [64, 128])
def test_a_group_of_nan_takes_nothing_from_the_others(d):
    """One token's group of 32 columns is NaN: those columns are NaN, the others as exact as ever."""
    n = 20000
    k, v = torch.randn(n, 1, d), torch.randn(n, 1, d) * 1e-3
    v[777, 0, 32] = float("nan")
    out, exact, var = outputs(k, v, torch.bfloat16, 8, batch=512)
    assert out[..., 32:64].isnan().all() and exact[..., 32:64].isnan().all()
    rest = torch.ones(d, dtype=torch.bool)
    rest[32:64] = False
    check(out[..., rest], exact[..., rest], var[..., rest])


@pytest.mark.parametrize("d", [64, 128])
def test_largest_values_stay_finite(d):
    """V over all of fp16's range, where a scale is 8734, next to small ones: no overflow on the
    way, and the exact value within the roundings."""
    n = 3000
    k, v = torch.randn(n, 1, d), torch.randn(n, 1, d)
    v[::7] = torch.rand(v[::7].shape) * 131008 - 65504
    v[::7, 0, 0], v[::7, 0, 1] = 65504.0, -65504.0
    out, exact, var = outputs(k, v, torch.bfloat16, 8, spread=0.5, batch=300)
    assert out.isfinite().all()
    check(out, exact, var)
