"""Attention over a cache in 8 bits whose V scales lie far apart: each query's result within a bound that knows only the keys that it
attends, weighted by their probabilities.  Other queries' keys, and large values that a query gives no probability, leave it alone."""
import math

import pytest
import torch

from pyasc_amd import kernels
from test_gpu_quantized_attention import ROUND, TINY, gather
from test_gpu_quantized_attention_kernels import operands
from test_gpu_quantized_cache import FORMATS
from test_quantized_attention_plans import LAUNCHES

pytestmark = pytest.mark.gpu


def check(got, lse, q, k, ks, v, vs, limits, scale):
    """One head, as test_gpu_quantized_attention.check, but for what is below fp16's normal range."""
    q, kk, vv = q.double(), k * ks[:, None], v * vs[:, None]
    s, size = q @ kk.T * scale, q.abs() @ kk.abs().T * scale
    seen = torch.arange(k.shape[0], device=q.device) < limits[:, None]
    s = s.masked_fill(~seen, -math.inf)
    want_lse = torch.logsumexp(s, 1)
    p = torch.exp(s - want_lse[:, None].nan_to_num(0, 0, 0))
    o, mag = p @ vv, p @ vv.abs()
    # fp32: D products per score and the FMA before exp2, a term per key in the sums, exp2 to 2^-21; the logarithm of a V scale, up to
    # 2^7, to a step of 2^-17
    largest = size.masked_fill(~seen, 0).amax(1)
    eps = (q.shape[1] + 4) * 2.0 ** -23 * largest + (k.shape[0] + 40) * 2.0 ** -22 + 2.0 ** -17
    # a row's largest probability times V scale is 2^8 at least when it is rounded to fp16, whose half step below its normal range is
    # 2^-25: 2^-33 of the largest of the attended keys, for each key.  2^-60 of it is the least that a scale counts as.
    part = (p * vs).amax(1)[:, None]
    bound = mag * (2.0 ** -11 + eps[:, None]) + (2.0 ** -33 + 2.0 ** -50) * part * (seen.double() @ v.abs())
    bound = bound + ROUND[got.dtype] * (o.abs() + bound) + TINY[got.dtype]
    off = (got.double() - o).abs()
    assert (off <= bound).all(), float((off / bound).max())
    empty = limits <= 0
    assert (lse[empty] == -math.inf).all()
    assert ((lse.double() - want_lse).abs()[~empty] <= eps[~empty] + 2.0 ** -22 * (want_lse[~empty].abs() + 1)).all()


def attend(q, cache, table, lengths, causal=True, scale=None):
    """Runs one call over a paged cache and checks each of its heads."""
    b, heads, n, d = q.shape
    k, v, ks, vs = cache
    page = k.shape[2]
    block, scale = page // ks.shape[2], d ** -0.5 if scale is None else scale
    o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device=q.device)
    kernels.quantized_cache_attention(q, *cache, torch.tensor(lengths, dtype=torch.int32, device=q.device), o, scale, block_table=table,
                                      causal=causal, lse=lse)
    for i in range(b):
        limits = torch.full((n,), lengths[i], device=q.device)
        if causal:
            limits = (torch.arange(n, device=q.device) + lengths[i] - n + 1).clamp(min=0)
        for h in range(heads):
            g = h // (heads // k.shape[1])
            kk, vv = (gather(*x, table, i, g, lengths[i], page, block) for x in ((k, ks), (v, vs)))
            check(o[i, h], lse[i, h], q[i, h], *kk, *vv, limits, scale)
    return o, lse


def at_keys(scales, table, i, keys, page):
    """The places of blocks of 16 rows of sequence i's keys."""
    keys = torch.as_tensor(keys, device=scales.device)
    return table[i].long()[keys // page], slice(None), keys % page // 16


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("far", [20, 26, 34, 60, 110])
@pytest.mark.parametrize("name", LAUNCHES)
def test_values_that_only_later_queries_attend(device, name, far, cache):
    """A last block 2^far times as large: queries before it get what they get without it."""
    q, (k, v, ks, vs), table, capacity, _ = operands(name, cache, torch.bfloat16, device, 8)
    b, _, n, _ = q.shape
    lengths = [capacity - 5 * i for i in range(b)]
    without, lse = attend(q, (k, v, ks, vs), table, lengths)
    for i in range(b):
        vs[at_keys(vs, table, i, lengths[i] - 1, k.shape[2])] *= 2.0 ** far
    got, got_lse = attend(q, (k, v, ks, vs), table, lengths)
    before = [max(0, n - 1 - (length - 1) % 16) for length in lengths]
    eps = 4 * torch.finfo(q.dtype).eps
    for i, m in enumerate(before):
        a, c = without[i, :, :m].double(), got[i, :, :m].double()
        assert ((a - c).abs() <= eps * (a.abs() + a.abs().mean(-1, keepdim=True))).all()
        assert ((lse - got_lse)[i].abs() <= 2.0 ** -14).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("far", [22, 40, 70])
@pytest.mark.parametrize("name", LAUNCHES)
def test_large_values_without_probability(device, name, far, dtype):
    """Blocks of values 2^far times the rest's, at the first, the last and a middle key, whose probabilities lie 2^(1.5 far) below."""
    q, (k, v, ks, vs), table, capacity, g = operands(name, torch.int8, dtype, device, 9)
    b, _, n, d = q.shape
    q[..., 0] = 4.0
    k[..., 0] = 0
    for i in range(b):
        for key in (0, capacity // 2, capacity - 1):
            at = at_keys(vs, table, i, key, k.shape[2])
            ks[at], vs[at] = 1.5 * far * math.log(2) * d ** 0.5 / 4 / 127, vs[at] * 2.0 ** far
            rows = slice(key // 16 * 16 % k.shape[2], key // 16 * 16 % k.shape[2] + 16)
            k[at[0], :, rows] = torch.randint(-2, 3, k[at[0], :, rows].shape, generator=g, device=device).to(torch.int8)
            k[at[0], :, rows, 0] = -127
    attend(q, (k, v, ks, vs), table, [capacity] * b, causal=False)


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("name", LAUNCHES)
def test_values_of_nothing(device, name, cache):
    """Blocks of zeros with the least scale that an append gives, most probable of all; and every other block of one."""
    q, (k, v, ks, vs), table, capacity, _ = operands(name, cache, torch.bfloat16, device, 10)
    b, _, n, _ = q.shape
    page = k.shape[2]
    for i in range(b):
        for key in (3, capacity // 2, capacity - 2):
            at = at_keys(vs, table, i, key, page)
            vs[at], ks[at] = 2.0 ** -126, ks[at] * 4
            v.view(torch.uint8)[at[0], :, key // 16 * 16 % page:key // 16 * 16 % page + 16] = 0
    attend(q, (k, v, ks, vs), table, [capacity - i for i in range(b)])
    v.view(torch.uint8).zero_()
    vs.fill_(2.0 ** -126)
    vs[1::2] = 1.0
    o, _ = attend(q, (k, v, ks, vs), table, [capacity] * b)
    assert not o.any()


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("size", [-140, -126, -100, 60, 100, 116])
@pytest.mark.parametrize("name", LAUNCHES)
def test_scales_of_any_size(device, name, size, cache):
    """V scales of 2^size and a few powers of two about it, not all of them powers."""
    q, (k, v, ks, vs), table, capacity, g = operands(name, cache, torch.bfloat16, device, 11)
    b, _, n, _ = q.shape
    vs.copy_((torch.rand(vs.shape, generator=g, device=device) + 1.0) * 2.0 ** -12)
    vs.copy_((vs.double() * 2.0 ** (12 + size)).float())
    o, _ = attend(q, (k, v, ks, vs), table, [capacity - 7 * i for i in range(b)])
    assert o.isfinite().all() and (o.any() or size < -120)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", LAUNCHES)
def test_scales_that_rise_and_fall(device, name, dtype):
    """2^-60 to 2^0 along a sequence's keys, up in one and down in the next: every query has others in reach."""
    q, (k, v, ks, vs), table, capacity, _ = operands(name, torch.int8, dtype, device, 12)
    b, _, n, _ = q.shape
    keys = torch.arange(0, capacity, 16, device=device)
    for i in range(b):
        e = -60.0 * (keys if i % 2 else capacity - keys) / capacity
        vs[at_keys(vs, table, i, keys, k.shape[2])] = torch.exp2(e.round()).float()[:, None].expand(-1, vs.shape[1])
    attend(q, (k, v, ks, vs), table, [capacity - 3 * i for i in range(b)])


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("query,key,scale", [(-118, 120, -10), (-118, -14, 127.75), (110, 0, -110), (-60, 60, -8), (-118, 0, 110)])
@pytest.mark.parametrize("name", LAUNCHES)
def test_scores_of_factors_of_any_size(device, name, query, key, scale, cache):
    """Queries, K scales and a factor of the scores near the ends of fp32, each the power of two that is named, with common scores."""
    q, (k, v, ks, vs), table, capacity, _ = operands(name, cache, torch.bfloat16, device, 13)
    b, _, n, _ = q.shape
    q.copy_((q.double() * 2.0 ** query).bfloat16())
    ks.copy_((ks.double() / 4 * (1.0 if cache is torch.int8 else 0.5) * 2.0 ** key).float())
    attend(q, (k, v, ks, vs), table, [capacity - 3 * i for i in range(b)], scale=2.0 ** scale)
