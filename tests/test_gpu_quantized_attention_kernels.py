"""Each kernel of the attention over a cache in 8 bits, with and without splits of the keys, at the launches that
test_quantized_attention_plans.py holds them to, against the formula in fp64: ragged and empty sequences, padded batches, NaN among
the values, scales far apart, a late key that outweighs the rest, pages outside the cache."""
import math

import pytest
import torch

from pyasc_amd import kernels
from test_gpu_quantized_attention import attend, queries
from test_gpu_quantized_cache import FORMATS, make, table_of
from test_quantized_attention_plans import LAUNCHES

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def operands(name, cache, dtype, device, seed=0):
    (b, hq, hk, n, width, page, d), _, _ = LAUNCHES[name]
    g = torch.Generator(device=device).manual_seed(seed + b + n + page)
    state = make(b * width + 2, hk, page, d, 16, cache, g)
    return queries(b, hq, n, d, dtype, g), state, table_of(b, width, b * width + 2, g), width * page, g


def lengths_of(b, n, capacity):
    """The first sequence fills its pages; of the others one has a single key, and one none."""
    return [capacity] + [[capacity - 17, 1, 0, capacity // 2 + 5, 65, n, 64][i % 7] for i in range(b - 1)]


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", LAUNCHES)
def test_ragged(device, name, dtype, cache):
    q, state, table, capacity, _ = operands(name, cache, dtype, device)
    b, _, n, _ = q.shape
    attend(q, state, lengths_of(b, n, capacity), table, [max(0, n - 5 * i) for i in range(b)])


@pytest.mark.parametrize("name", LAUNCHES)
def test_all_keys(device, name):
    q, state, table, capacity, _ = operands(name, torch.int8, torch.bfloat16, device, 1)
    b, _, n, _ = q.shape
    attend(q, state, lengths_of(b, n, capacity), table, causal=False)


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("name", LAUNCHES)
def test_scales_far_apart(device, name, cache):
    """V scales over 2^60, some of them zero, one of K's that makes a late block outweigh the rest."""
    q, state, table, capacity, g = operands(name, cache, torch.bfloat16, device, 2)
    k, v, ks, vs = state
    vs *= torch.exp2(torch.randint(-30, 30, vs.shape, generator=g, device=device).float())
    vs[::3, :, 0] = 0.0
    ks[int(table[0, -1]), :, -1] *= 8
    b, _, n, _ = q.shape
    attend(q, state, [capacity - i for i in range(b)], table, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", LAUNCHES)
def test_nan_of_a_value(device, name, dtype):
    """It reaches the queries that attend it, and no others: in a full tile, and within the last rows."""
    q, state, table, capacity, _ = operands(name, torch.float8_e4m3fn, dtype, device, 3)
    v, page = state[1], state[1].shape[2]
    b, _, n, _ = q.shape
    lengths = [capacity - 3 * i for i in range(b)]
    for key, column in ((lengths[0] - 1, 3), (lengths[0] - n // 2 - 1, 40)):
        v.view(torch.uint8)[int(table[0, key // page]), 0, key % page, column] = 0x7f
    if b > 2:
        v.view(torch.uint8)[int(table[2, 0]), 1, 1, 60:] = 0xff
    o, _ = attend(q, state, lengths, table)
    assert o[0].isnan().any() and not o[1].isnan().any()


@pytest.mark.parametrize("name", LAUNCHES)
def test_pages_outside_the_cache(device, name):
    """The last page's entry of one sequence, others' behind their lengths."""
    q, state, table, capacity, _ = operands(name, torch.int8, torch.float16, device, 4)
    b, _, n, _ = q.shape
    page = state[0].shape[2]
    lengths = [capacity - page] * b
    lengths[1] = capacity
    table[:, -1] = state[0].shape[0]
    o = torch.zeros_like(q)
    kernels.quantized_cache_attention(q, *state, torch.tensor(lengths, dtype=torch.int32, device=device), o, 0.125, block_table=table,
                                      causal=False)
    nan = o.isnan().flatten(1)
    assert nan[1].all() and not nan[0].any() and not nan[2:].any()


@pytest.mark.parametrize("cache", FORMATS)
@pytest.mark.parametrize("name", LAUNCHES)
def test_same_results_from_run_to_run_and_from_a_graph(device, name, cache):
    q, state, table, capacity, _ = operands(name, cache, torch.bfloat16, device, 5)
    b, _, n, _ = q.shape
    lengths = torch.tensor(lengths_of(b, n, capacity), dtype=torch.int32, device=device)
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], device=device)

    def run(o, l):
        kernels.quantized_cache_attention(q, *state, lengths, o, 0.1, block_table=table, lse=l)

    run(out, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out, lse)
    for m in (0, 1, 2):
        lengths.copy_((lengths - m * 33).clamp(min=0))
        want, want_lse = torch.full_like(q, math.nan), torch.full_like(lse, math.nan)
        run(want, want_lse)
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("name", LAUNCHES)
def test_empty_sequences_beside_full_ones(device, name):
    q, state, table, capacity, _ = operands(name, torch.int8, torch.float16, device, 6)
    b, _, n, _ = q.shape
    attend(q, state, [0] + [capacity] * (b - 1), table)
    attend(q, state, [0] * b, table, [max(0, n - i) for i in range(b)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", LAUNCHES)
def test_a_query_of_nan_or_infinity_stays_alone(device, name, dtype):
    q, state, table, capacity, _ = operands(name, torch.float8_e4m3fn, dtype, device, 7)
    b, _, n, d = q.shape
    lengths = torch.tensor(lengths_of(b, n, capacity), dtype=torch.int32, device=device)
    want, got = torch.zeros_like(q), torch.zeros_like(q)
    kernels.quantized_cache_attention(q, *state, lengths, want, 0.1, block_table=table)
    bad = q.clone()
    bad[0, 0, n // 2, 3], bad[0, -1, 0, d - 1] = math.nan, math.inf
    kernels.quantized_cache_attention(bad, *state, lengths, got, 0.1, block_table=table)
    hit = torch.zeros(q.shape[:3], dtype=torch.bool, device=device)
    hit[0, 0, n // 2], hit[0, -1, 0] = True, True
    assert got[0, 0, n // 2].isnan().all() and torch.equal(got[~hit].isnan(), want[~hit].isnan())
    # another row of a block may move its reference point: all within a few roundings of the first result
    a, c = got[~hit].double(), want[~hit].double()
    assert ((a - c).abs() <= 4 * torch.finfo(dtype).eps * (c.abs() + c.abs().mean(-1, keepdim=True)))[~c.isnan()].all()
