"""Attention over a cache held in 8 bits against the formula in fp64 on the cache's values."""
import math

import pytest
import torch

import cache8_reference as R
from pyasc_amd import kernels
from test_gpu_quantized_cache import FORMATS, make, table_of

pytestmark = pytest.mark.gpu
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def gather(cache, scales, table, b, h, length, page, block):
    """Code values and scales [length] of a sequence's head, in fp64."""
    at = torch.arange(length, device=cache.device)
    pages = torch.full_like(at, b) if table is None else table[b].long()[at // page]
    rows = at % page if table is not None else at
    codes = cache.view(torch.uint8)[pages, h, rows].view(cache.dtype)
    return R.values(codes), scales[pages, h, rows // block].double()


def check(got, lse, q, k, ks, v, vs, limits, scale, dtype):
    """One head: q [n, d] and the keys that each of its queries attends, the first `limits` ones."""
    n, length = q.shape[0], k.shape[0]
    q, kk, vv = q.double(), k * ks[:, None], v * vs[:, None]
    s = q @ kk.T * scale
    size = q.abs() @ kk.abs().T * scale
    seen = torch.arange(length, device=q.device) < limits[:, None]
    s = s.masked_fill(~seen, -math.inf)
    want_lse = torch.logsumexp(s, 1) if length else torch.full((n,), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.exp(s - want_lse[:, None].nan_to_num(0, 0, 0))
    bad = ~vv.isfinite()
    clean = vv.nan_to_num(0, 0, 0)
    o, mag = p @ clean, p @ clean.abs()
    # a NaN reaches the queries that attend it
    o[(seen.double() @ bad.double()) > 0] = math.nan
    # fp32: D products per score and the FMA before exp2, n terms per sum, exp2 and log2 to 2^-21, the
    # V scales' logarithm to 2^-19
    largest = float(size.masked_fill(~seen, 0).nan_to_num(0).amax()) if size.numel() else 0.0
    eps = (q.shape[1] + 4) * 2.0 ** -23 * largest + (length + 40) * 2.0 ** -22 + 2.0 ** -19
    # p v rounded to fp16: 2^-11 of it, and below fp16's normal range 2^-25 where the largest probability is 2^8
    # or more and values are in units of the largest scale
    top = float(vs.max()) if length else 0.0
    bound = mag * (2.0 ** -11 + eps) + 2.0 ** -32 * top * v.nan_to_num(0).abs().sum(0)
    bound = bound + ROUND[dtype] * (o.abs() + bound) + TINY[dtype]
    nan = o.isnan()
    assert torch.equal(got.isnan(), nan)
    off = (got.double() - o).abs()
    assert (off <= bound)[~nan].all(), float((off / bound)[~nan].max())
    empty = limits <= 0
    assert not got[empty].any()
    if lse is not None:
        assert (lse[empty] == -math.inf).all()
        assert ((lse.double() - want_lse).abs()[~empty] <= eps + 2.0 ** -22 * (want_lse[~empty].abs() + 1)).all()


def attend(q, cache, lengths, table=None, news=None, causal=True, o=None, stream=None):
    """Runs and checks one call; returns o and lse."""
    b, heads, n, d = q.shape
    k, v, ks, vs = cache
    kv_heads, page = k.shape[1], k.shape[2]
    block, scale = page // ks.shape[2], d ** -0.5
    o = torch.empty_like(q) if o is None else o
    o.fill_(7.0)
    lse = torch.full((b, heads, n), 7.0, device=q.device)
    cl = torch.tensor(lengths, dtype=torch.int32, device=q.device)
    nl = None if news is None else torch.tensor(news, dtype=torch.int32, device=q.device)
    kernels.quantized_cache_attention(q, k, v, ks, vs, cl, o, scale, block_table=table, new_lengths=nl, causal=causal, lse=lse)
    torch.cuda.synchronize()
    for i in range(b):
        new = n if news is None else news[i]
        limits = torch.arange(new, device=q.device) + lengths[i] - new + 1 if causal else torch.full((new,), lengths[i], device=q.device)
        assert (o[i, :, new:] == 7.0).all() and (lse[i, :, new:] == 7.0).all()
        for h in range(heads):
            g = h // (heads // kv_heads)
            kk = gather(k, ks, table, i, g, lengths[i], page, block)
            vv = gather(v, vs, table, i, g, lengths[i], page, block)
            check(o[i, h, :new], lse[i, h, :new], q[i, h, :new], *kk, *vv, limits, scale, q.dtype)
    return o, lse


def queries(b, heads, n, d, dtype, g, scale=1.0):
    return (torch.randn((b, n, heads, d), generator=g, device="cuda") * scale).to(dtype).transpose(1, 2)


SHAPES = [(1, 1, 1, 1, [1], None, 16, 16), (2, 4, 2, 1, [16, 17], None, 16, 16), (1, 8, 1, 3, [129], None, 64, 16),
          (3, 4, 4, 1, [0, 1, 600], None, 48, 48), (2, 8, 2, 1, [3000, 64], None, 256, 128), (4, 8, 8, 2, [2000, 17, 1, 999], None, 80, 16),
          (1, 16, 1, 2, [9000], None, 128, 32), (2, 2, 1, 20, [33, 100], [20, 7], 32, 32), (1, 2, 2, 33, [40], None, 16, 16),
          (2, 4, 2, 64, [64, 500], None, 64, 64), (1, 6, 2, 100, [333], None, 48, 16), (1, 1, 1, 257, [257], None, 128, 64),
          (2, 2, 1, 300, [300, 1025], [299, 0], 16, 16), (1, 4, 4, 513, [1385], None, 96, 48), (3, 8, 2, 130, [700, 130, 90], [130, 1, 90], 256, 16)]


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("b,hq,hk,n,lengths,news,page,block", SHAPES)
def test_attention(device, b, hq, hk, n, lengths, news, page, block, D, dtype, cache):
    g = torch.Generator(device=device).manual_seed(n + page)
    width = max(1, -(-max(lengths) // page))
    state = make(b * width + 2, hk, page, D, block, cache, g)
    table = table_of(b, width, b * width + 2, g)
    q = queries(b, hq, n, D, dtype, g)
    attend(q, state, lengths, table, news)
    attend(q, state, lengths, table, news, causal=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_one_piece_and_strides(device, n, D):
    """No table: [batch, rows, heads, d] caches and results, scales with strides."""
    g = torch.Generator(device=device).manual_seed(n)
    base = torch.randint(-127, 128, (3, 320, 4, D + 16), generator=g, device=device).to(torch.int8)
    k, v = base[:, :, :2, :D].transpose(1, 2), base[:, :, 2:, 16:].transpose(1, 2)
    scales = torch.rand((3, 2, 10, 2), generator=g, device=device) / 16
    o = torch.empty((3, n, 4, D + 8), dtype=torch.bfloat16, device=device)[..., :D].transpose(1, 2)
    attend(queries(3, 4, n, D, torch.bfloat16, g), (k, v, scales[..., 0], scales[..., 1]), [320, 207, 255], o=o)


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("n,length", [(1, 1000), (5, 130), (200, 700)])
def test_behind_and_ahead_of_a_query_anything_may_lie(device, n, length, cache):
    """Rows behind a sequence and pages behind its last: NaN codes, scales of any kind, entries outside the
    cache.  A value of NaN reaches the queries that attend it, and no others."""
    g = torch.Generator(device=device).manual_seed(n)
    page, b = 32, 2
    width = length // page + 3
    state = make(b * width, 2, page, 64, 16, cache, g)
    k, v, ks, vs = state
    table = table_of(b, width, b * width, g)
    lengths = [length, length - 7]
    for i, m in enumerate(lengths):
        at = torch.arange(m, width * page, device=device)
        pages, rows = table[i].long()[at // page], at % page
        for t in (k, v):
            t.view(torch.uint8)[pages, :, rows] = 0x7f
        for s in (ks, vs):
            s[table[i, -(-m // page):].long()] = math.nan
        table[i, -(-m // page):] = torch.tensor([-1, b * width, 2 ** 31 - 1, -5], dtype=torch.int32, device=device)[:width - -(-m // page)]
    q = queries(b, 8, n, 64, torch.float16, g)
    attend(q, state, lengths, table)
    if cache is torch.float8_e4m3fn:
        last = length - 1
        v.view(torch.uint8)[int(table[0, last // page]), 1, last % page, 5] = 0xff
        if n > 1:
            last = length - n // 2
            v.view(torch.uint8)[int(table[0, last // page]), 0, last % page, 60:] = 0x7f
        o, _ = attend(q, state, lengths, table)
        assert o[0].isnan().any() and not o[1].isnan().any()


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("n", [1, 200])
def test_scales_far_apart(device, n, cache):
    """V scales that rise and fall along the keys, some of them zero; K scales that make a late block dominate."""
    g = torch.Generator(device=device).manual_seed(n)
    k, v, ks, vs = make(2, 2, 2048, 128, 16, cache, g)
    vs *= torch.exp2(torch.randint(-30, 30, vs.shape, generator=g, device=device).float())
    vs[:, :, 5:9] = 0.0
    vs[1] = torch.exp2(torch.linspace(-40, 40, 128, device=device))
    ks[:, :, 100] *= 8
    q = queries(2, 2, n, 128, torch.bfloat16, g)
    attend(q, (k, v, ks, vs), [2048, 1999])
    attend(q, (k, v, ks, torch.zeros_like(vs)), [2048, 1999])


@pytest.mark.parametrize("n", [1, 100])
@pytest.mark.parametrize("late", [3, 70, 390, 999])
def test_a_late_key_far_above_the_rest(device, late, n):
    g = torch.Generator(device=device).manual_seed(late)
    k, v, ks, vs = make(1, 2, 1024, 128, 16, torch.int8, g)
    k.clamp_(-20, 20)
    q = queries(1, 2, n, 128, torch.bfloat16, g)
    q[..., 0] = 8.0
    k[:, :, late, 0] = 127
    ks[:] = 0.05
    attend(q, (k, v, ks, vs), [1000], causal=False)
    k[:, :, :, 0] = -127  # all scores far below zero: the reference point follows them down
    attend(q, (k, v, ks, vs), [1000], causal=False)


@pytest.mark.parametrize("n", [1, 100])
@pytest.mark.parametrize("size", [1e-36, 1e-20, 1e25])
def test_queries_of_any_size(device, n, size):
    """bf16 queries beyond fp16's range, and rows of zeros, with K scales that bring the scores back."""
    g = torch.Generator(device=device).manual_seed(n)
    k, v, ks, vs = make(1, 2, 512, 64, 32, torch.int8, g)
    ks *= min(1 / size, 1e30)
    q = queries(1, 4, n, 64, torch.bfloat16, g, size)
    q[:, 1] = 0.0
    attend(q, (k, v, ks, vs), [500])


def test_bad_lengths_and_pages_are_not_followed(device):
    g = torch.Generator(device=device).manual_seed(1)
    for n in (1, 70):
        state = make(40, 1, 16, 64, 16, torch.int8, g)
        table = table_of(5, 8, 40, g)
        table[3, 2] = 40
        lengths = torch.tensor([128, 129, -1, 128, 128], dtype=torch.int32, device=device)
        news = torch.tensor([n, n, n, n, n + 1], dtype=torch.int32, device=device)
        q = queries(5, 2, n, 64, torch.float16, g)
        o, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], device=device)
        kernels.quantized_cache_attention(q, *state, lengths, o, 0.125, block_table=table, new_lengths=news, lse=lse)
        assert o[0].isfinite().all() and o[1:].isnan().all() and lse[1:].isnan().all() and lse[0].isfinite().all()
        news.fill_(-1)
        o.fill_(7.0)
        kernels.quantized_cache_attention(q, *state, lengths, o, 0.125, block_table=table, new_lengths=news)
        assert (o == 7.0).all()


@pytest.mark.parametrize("n", [1, 40])
def test_nothing_to_attend(device, n):
    state = make(2, 2, 16, 64, 16, torch.int8, torch.Generator(device=device).manual_seed(1))
    g = torch.Generator(device=device).manual_seed(2)
    q = queries(2, 4, n, 64, torch.float16, g)
    attend(q, state, [0, 0])
    attend(q, state, [min(n - 1, 16), 16], news=[n, 0])  # more queries than keys: the first have none
    none = torch.zeros((2, 0), dtype=torch.int32, device=device)
    o = torch.full_like(q, 7.0)
    kernels.quantized_cache_attention(q, *state, torch.zeros(2, dtype=torch.int32, device=device), o, 0.125, block_table=none)
    assert not o.any()
    empty = q[:, :, :0]
    kernels.quantized_cache_attention(empty, *state, torch.zeros(2, dtype=torch.int32, device=device), empty.clone(), 0.125)


def test_far_rows(device):
    """Pages and rows beyond 4 GiB."""
    g = torch.Generator(device=device).manual_seed(3)
    base = torch.empty((6 << 30,), dtype=torch.int8, device=device)
    k = base.as_strided((6, 1, 64, 64), (1 << 30, 4096, 64, 1))
    v = base.as_strided((6, 1, 64, 64), (1 << 30, 4096, 64, 1), 1 << 20)
    for t in (k, v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=g, device=device).to(torch.int8))
    scales = torch.rand((6, 1, 4), generator=g, device=device) / 16
    table = torch.tensor([[5, 0], [4, 5]], dtype=torch.int32, device=device)
    for n in (1, 60):
        attend(queries(2, 4, n, 64, torch.bfloat16, g), (k, v, scales, scales), [128, 100], table)


def test_another_stream_and_captured_calls(device):
    """Calls with and without a workspace, replayed on growing sequences beside eager ones."""
    g = torch.Generator(device=device).manual_seed(4)
    state = make(160, 2, 64, 128, 16, torch.float8_e4m3fn, g)
    table = table_of(2, 80, 160, g)
    lengths = torch.tensor([1, 1], dtype=torch.int32, device=device)
    q = [queries(2, 8, n, 128, torch.bfloat16, g) for n in (1, 300)]
    out = [torch.zeros_like(x) for x in q]

    def step(out):
        for x, y in zip(q, out):
            kernels.quantized_cache_attention(x, *state, lengths, y, 0.1, block_table=table)

    step(out)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            step(out)
    stream = torch.cuda.Stream()
    for i, m in enumerate((1, 300, 5000, 63, 4097)):
        lengths.fill_(m)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        want = [torch.zeros_like(x) for x in q]
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(want)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
