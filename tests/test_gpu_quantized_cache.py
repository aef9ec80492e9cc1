"""The append to a cache held in 8 bits and the read of its values: codes and scales are the
formulas' to the bit."""
import math

import pytest
import torch

import cache8_reference as R
from pyasc_amd import kernels

pytestmark = pytest.mark.gpu
FORMATS = [torch.int8, torch.float8_e4m3fn]


def make(pages, heads, page, d, block, dtype, g, fill=True):
    """A cache of random codes whose scales are powers of two, or of zeros."""
    if not fill:
        k, v = (torch.zeros((pages, heads, page, d), device="cuda", dtype=torch.uint8).view(dtype) for _ in range(2))
    elif dtype == torch.int8:
        k, v = (torch.randint(-127, 128, (pages, heads, page, d), generator=g, device="cuda").to(dtype) for _ in range(2))
    else:
        k, v = ((torch.randn((pages, heads, page, d), generator=g, device="cuda") * 100).clamp(-448, 448).to(dtype)
                for _ in range(2))
    ks, vs = (torch.exp2(torch.randint(-8, -3, (pages, heads, page // block), generator=g, device="cuda").float())
              for _ in range(2))
    return k, v, ks, vs


def table_of(b, width, pages, g):
    return torch.randperm(pages, generator=g, device="cuda")[:b * width].view(b, width).int()


def same(cache, codes):
    """Equal code values, NaN for NaN."""
    return torch.equal(R.values(cache.cpu()).nan_to_num(1e9), codes.nan_to_num(1e9))


def run_append(x_k, x_v, cache, lengths, news, table, page, block):
    """Appends on the device and in the reference, compares all of the cache, and reads it back."""
    k, v, ks, vs = cache
    b, h, n, d = x_k.shape
    ref = [(R.Codes(k), ks.double().cpu()), (R.Codes(v), vs.double().cpu())]
    where = R.Paged(table, page)
    cl = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    nl = None if news is None else torch.tensor(news, dtype=torch.int32, device="cuda")
    kernels.quantized_cache_append(x_k, x_v, k, v, ks, vs, cl, block_table=table, new_lengths=nl)
    torch.cuda.synchronize()
    news = [n] * b if news is None else news
    for x, (codes, scales), cache_, scales_ in zip((x_k, x_v), ref, (k, v), (ks, vs)):
        R.append(x.cpu(), codes, scales, lengths, news, where, block)
        assert same(cache_, codes.codes)
        assert torch.equal(scales_.double().cpu(), scales)
    # values of all of a sequence's keys
    total = [i + j for i, j in zip(lengths, news)]
    most = max(total)
    for dtype in (torch.float32, torch.bfloat16):
        out = [torch.full((b, h, most, d), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
        kernels.quantized_cache_read(k, v, ks, vs, torch.zeros_like(cl), *out, block_table=table,
                                     counts=torch.tensor(total, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        for o, (codes, scales) in zip(out, ref):
            o = o.cpu()
            for i in range(b):
                for key in range(total[i]):
                    pg, row = where.at(i, key)
                    want = (codes.codes[pg, :, row] * scales[pg, :, row // block, None]).float().to(dtype)
                    assert torch.equal(o[i, :, key].nan_to_num(1e9), want.nan_to_num(1e9))
                assert (o[i, :, total[i]:] == 7.0).all()


SHAPES = [(1, 1, 1, [0], None, 16, 16), (2, 3, 5, [0, 14], None, 16, 16), (3, 2, 1, [15, 16, 31], None, 48, 48),
          (2, 1, 70, [3, 50], [70, 0], 80, 16), (1, 2, 200, [7], None, 32, 32), (2, 2, 130, [100, 0], [130, 129], 256, 256),
          (1, 1, 600, [37], None, 128, 64), (2, 1, 33, [1, 255], [33, 2], 256, 128), (1, 1, 1100, [0], None, 1024, 1024),
          (1, 1, 520, [513], None, 2048, 1024)]


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("b,h,n,lengths,news,page,block", SHAPES)
def test_append(device, b, h, n, lengths, news, page, block, D, dtype, cache):
    g = torch.Generator(device=device).manual_seed(n)
    width = -(-(max(lengths) + n) // page)
    state = make(b * width + 2, h, page, D, block, cache, g)
    # larger and smaller than what is there: scales that grow and scales that stay
    x = [(torch.randn((b, n, h, D), generator=g, device=device) * s).to(dtype).transpose(1, 2) for s in (20.0, 0.02)]
    run_append(*x, state, lengths, news, table_of(b, width, b * width + 2, g), page, block)


@pytest.mark.parametrize("cache", FORMATS)
def test_append_without_pages_token_by_token(device, cache):
    """One piece per sequence; every token larger than the last one, so that its block is rescaled each time."""
    g = torch.Generator(device=device).manual_seed(5)
    state = make(2, 2, 64, 64, 32, cache, g, fill=False)
    for i in range(40):
        x = [(torch.randn((2, 2, 1, 64), generator=g, device=device) * 1.3 ** i).half() for _ in range(2)]
        run_append(*x, state, [i, i + 3], None, None, 64, 32)


@pytest.mark.parametrize("cache", FORMATS)
def test_special_values(device, cache):
    g = torch.Generator(device=device).manual_seed(6)
    state = make(4, 1, 16, 64, 16, cache, g)
    x = [(torch.randn((4, 1, 20, 64), generator=g, device=device)).bfloat16() for _ in range(2)]
    x[0][0, 0, 3, 5], x[0][0, 0, 4, 6], x[0][0, 0, 4, 7] = math.inf, -math.inf, math.nan
    x[0][1] = 0.0
    x[0][1, 0, 19] = 1e-40  # below 2^-126 * the least code
    x[0][2, 0, :, :] = torch.finfo(torch.bfloat16).max
    x[0][3, 0, :16] = math.nan
    x[1][0] = -0.0
    x[1][1, 0, 0, 0] = 127 * 2.0 ** -3  # at a scale's border, and behind it
    x[1][2, 0, 0, 0] = 448 * 2.0 ** -3
    x[1][3, 0, 0, 0] = 128 * 2.0 ** -3
    state = make(8, 1, 16, 64, 16, cache, g)
    run_append(*x, state, [0] * 4, None, table_of(4, 2, 8, g), 16, 16)
    assert state[0].float().isfinite().all() == (cache == torch.int8)


@pytest.mark.parametrize("held", [0.0, -1.0, math.inf, math.nan, 0.3, 2.0 ** -127, 2.0 ** 127])
@pytest.mark.parametrize("cache", FORMATS)
def test_held_scales(device, cache, held):
    """A scale that is no power of two divides; one that is not positive and finite counts as 0."""
    g = torch.Generator(device=device).manual_seed(7)
    state = make(2, 1, 32, 64, 32, cache, g)
    state[2][:], state[3][:] = held, held
    x = [(torch.randn((2, 1, 3, 64), generator=g, device=device) * s).half() for s in (1.0, 100.0)]
    k, v, ks, vs = state
    # the product with the held scale and the quotient are rounded to fp32, 2^-24 each, before they become a code:
    # a code of a quotient that is off by less than 2^-22
    nudges = (1 - 2.0 ** -22, 1 + 2.0 ** -22) if held == 0.3 else (1.0, 1.0)
    refs = [[(R.Codes(t), s.double().cpu()) for t, s in ((k, ks), (v, vs))] for _ in nudges]
    cl = torch.tensor([9, 12], dtype=torch.int32, device=device)
    kernels.quantized_cache_append(*x, *state, cl)
    for i, (x_, cache_, scales_) in enumerate(zip(x, (k, v), (ks, vs))):
        ends = []
        for nudge, ref in zip(nudges, refs):
            codes, scales = ref[i]
            R.append(x_.cpu(), codes, scales, [9, 12], [3, 3], R.Paged(None, 32), 32, nudge)
            assert torch.equal(scales_.double().cpu(), scales)
            ends.append(codes.codes)
        got = R.values(cache_.cpu())
        assert ((got >= torch.minimum(*ends)) & (got <= torch.maximum(*ends))).all()


@pytest.mark.parametrize("cache,held", [(torch.int8, 1.5 * 2.0 ** 121), (torch.float8_e4m3fn, 1.75 * 2.0 ** 119)] + [
    (c, x) for c in FORMATS for x in (1.5 * 2.0 ** 100, 1.5 * 2.0 ** -126, 2.0 ** -140, 1.5 * 2.0 ** -127)])
def test_codes_are_rescaled_next_to_the_ends_of_fp32(device, cache, held):
    """Earlier codes times a held scale lie outside fp32, the codes that they become do not: exact products, whose quotients by a
    power of two are rounded once."""
    g = torch.Generator(device=device).manual_seed(11)
    k, v, ks, vs = make(1, 1, 16, 64, 16, cache, g)
    ks[:], vs[:] = held, held
    # a largest value that takes a larger scale
    largest = torch.finfo(torch.bfloat16).max if held > 2.0 ** 110 else (held * 1000 if held > 1 else 2.0 ** -114)
    x = torch.rand((1, 1, 2, 64), generator=g, device=device).double() * 2 - 1
    x[0, 0, 0, 0] = 1.0
    x = (x * largest).bfloat16()
    ref = [(R.Codes(t), s.double().cpu()) for t, s in ((k, ks), (v, vs))]
    length = torch.tensor([9], dtype=torch.int32, device=device)
    kernels.quantized_cache_append(x, x, k, v, ks, vs, length)
    for (codes, scales), cache_, scales_ in zip(ref, (k, v), (ks, vs)):
        R.append(x.cpu(), codes, scales, [9], [2], R.Paged(None, 16), 16)
        assert float(scales[0, 0, 0]) > held
        assert torch.equal(scales_.double().cpu(), scales) and same(cache_, codes.codes)


def test_bad_lengths_and_pages_are_not_followed(device):
    g = torch.Generator(device=device).manual_seed(8)
    state = make(20, 1, 16, 64, 16, torch.int8, g)
    before = [t.clone() for t in state]
    x = torch.randn((6, 1, 20, 64), generator=g, device=device).half()
    table = table_of(6, 3, 20, g)
    table[4, 0], table[4, 1] = -1, 20
    lengths = torch.tensor([-1, 49, 29, 0, 0, 2 ** 31 - 1], dtype=torch.int32, device=device)
    news = torch.tensor([20, 1, 20, 21, 20, -5], dtype=torch.int32, device=device)
    kernels.quantized_cache_append(x, x, *state, lengths, block_table=table, new_lengths=news)
    assert all(torch.equal(a, b) for a, b in zip(state, before))
    out = torch.full((6, 1, 20, 64), 7.0, device=device)
    kernels.quantized_cache_read(*state, lengths, out, None, block_table=table, counts=news)
    assert out[:3].nan_to_num(9.0).eq(7.0)[1, :, 1:].all() and out[0].isnan().all() and out[1, :, :1].isnan().all()
    assert out[2].isnan().all() and out[3].isnan().all() and out[4].isnan().all() and (out[5] == 7.0).all()


def test_strides_and_layouts(device):
    """Caches as views: heads inside of rows, pages apart, scales with strides; rows out of one projection."""
    g = torch.Generator(device=device).manual_seed(9)
    base = torch.randint(-127, 128, (6, 32, 5, 80), generator=g, device=device).to(torch.int8)
    k, v = base[:, :, :2, :64].transpose(1, 2), base[:, :, 3:5, 16:].transpose(1, 2)
    scales = torch.full((6, 2, 2, 2), 0.25, device=device)
    ks, vs = scales[..., 0], scales[..., 1]
    qkv = torch.randn((2, 40, 3, 2, 64), generator=g, device=device).bfloat16()
    x = [qkv[:, :, i].transpose(1, 2) for i in (1, 2)]
    untouched = base[:, :, 2].clone(), base[:, :, :3, 64:].clone()
    run_append(*x, (k, v, ks, vs), [5, 20], [40, 31], table_of(2, 2, 6, g), 32, 16)
    assert torch.equal(base[:, :, 2], untouched[0]) and torch.equal(base[:, :, :3, 64:], untouched[1])


def test_far_rows(device):
    """Offsets beyond 32 bits: a page 5 GiB into the cache."""
    base = torch.empty((6 << 30,), dtype=torch.int8, device=device)
    cache = base.as_strided((6, 1, 16, 64), (1 << 30, 1024, 64, 1))
    cache.zero_()
    scales = torch.zeros((6, 1, 1), device=device)
    x = torch.randn((1, 1, 16, 64), device=device).half()
    table = torch.tensor([[5]], dtype=torch.int32, device=device)
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    other = torch.zeros((6, 1, 16, 64), dtype=torch.int8, device=device)
    kernels.quantized_cache_append(x, x, cache, other, scales, scales.clone(), zero, block_table=table)
    out = torch.empty_like(x)
    kernels.quantized_cache_read(cache, other, scales, scales, zero, out, None, block_table=table)
    assert (out.float() - x.float()).abs().max() <= scales[5] / 2 + 2.0 ** -10 and not cache[:5].any()


@pytest.mark.parametrize("new", [32, 5])
def test_rows_of_a_block_far_apart(device, new):
    """Rows outermost: a block that spans 5 GiB, whole, and row by row with scales that grow."""
    base = torch.zeros((6 << 30,), dtype=torch.int8, device=device)
    cache = base.as_strided((2, 1, 32, 64), (64, 128, 160 << 20, 1))
    other = torch.zeros((2, 1, 32, 64), dtype=torch.int8, device=device)
    scales, near = torch.zeros((2, 2, 1, 1), device=device)
    x = torch.randn((2, 1, new, 64), device=device).half()
    lengths = torch.zeros(2, dtype=torch.int32, device=device)
    for i in range(2 if new < 32 else 1):
        kernels.quantized_cache_append(x * 2.0 ** i, x * 2.0 ** i, cache, other, scales, near, lengths)
        lengths += new
    assert torch.equal(cache, other) and torch.equal(scales, near) and other.any()
    assert int((base != 0).sum()) == int((other != 0).sum())  # and nothing else


def test_another_stream_and_a_captured_step(device):
    g = torch.Generator(device=device).manual_seed(10)
    state, plain = (make(4, 1, 16, 64, 16, torch.int8, torch.Generator(device=device).manual_seed(1)) for _ in range(2))
    x = torch.randn((2, 1, 1, 64), generator=g, device=device).half()
    lengths = torch.zeros(2, dtype=torch.int32, device=device)
    table = table_of(2, 2, 4, g)
    out = torch.zeros((2, 1, 32, 64), device=device)
    zero = torch.zeros_like(lengths)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    kernels.quantized_cache_append(x, x, *state, lengths, block_table=table, stream=stream)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.quantized_cache_append(x, x, *state, lengths, block_table=table)
        kernels.quantized_cache_read(*state, zero, out, None, block_table=table)
    for i in range(20):
        x.copy_(torch.randn(x.shape, generator=g, device=device) * (i + 1))
        lengths.fill_(i)
        graph.replay()
        kernels.quantized_cache_append(x, x, *plain, lengths, block_table=table)
        torch.cuda.synchronize()
        want = torch.empty_like(out)
        kernels.quantized_cache_read(*plain, zero, want, None, block_table=table)
        assert torch.equal(out[:, :, :i + 1], want[:, :, :i + 1])


def test_nothing_to_do(device):
    state = make(2, 1, 16, 64, 16, torch.int8, torch.Generator(device=device).manual_seed(1))
    before = [t.clone() for t in state]
    zero = torch.zeros(2, dtype=torch.int32, device=device)
    x = torch.zeros((2, 1, 0, 64), device=device).half()
    kernels.quantized_cache_append(x, x, *state, zero)
    kernels.quantized_cache_read(*state, zero, x, x.clone())
    none = torch.zeros((0, 1, 3, 64), device=device).half()
    table = torch.zeros((0, 1), dtype=torch.int32, device=device)
    kernels.quantized_cache_append(none, none, *state, zero[:0], block_table=table)
    kernels.quantized_cache_read(*state, zero[:0], none, none.clone(), block_table=table)
    empty = torch.zeros((2, 0), dtype=torch.int32, device=device)  # tables without columns: no key fits
    x = torch.zeros((2, 1, 3, 64), device=device).half()
    kernels.quantized_cache_append(x, x, *state, zero, block_table=empty)
    out = torch.zeros_like(x)
    kernels.quantized_cache_read(*state, zero, out, None, block_table=empty)
    assert out.isnan().all() and all(torch.equal(a, b) for a, b in zip(state, before))
