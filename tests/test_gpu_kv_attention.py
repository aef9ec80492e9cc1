"""Attention over other keys than the queries' own, against the formulas in fp64: cross attention
(lengths, shared heads, layouts, padded batches, sequences without keys) and draft trees over a
cache (pages of any size, masks, rows that attend nothing, bad pages and lengths)."""
import math

import pytest
import torch

from pyasc_amd import kernels

pytestmark = pytest.mark.gpu
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def attend(q, k, v, seen, scale):
    """o, the size of its terms, the sum of all values, lse and the bound of the scores' error, of one
    head in fp64."""
    q, k, v = q.double(), k.double().contiguous(), v.double().contiguous()
    s = (q @ k.T) * scale
    size = (q.abs() @ k.T.abs().contiguous()) * scale
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None].nan_to_num(0, 0, 0))
    v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
    o, mag = torch.zeros_like(q), torch.zeros_like(q)
    for bad in (False, True):  # a token that some rows do not attend may hold anything
        rows = seen[:, ~v.isfinite().all(1)].any(1) == bad
        w = v if bad else v.nan_to_num(0, 0, 0)
        o[rows], mag[rows] = p[rows] @ w, p[rows] @ w.abs()
    # fp32: D products per score and the FMA before exp2, n terms per sum, exp2 and log2 to 2^-21
    largest = size.masked_fill(~seen, 0).amax() if size.numel() else 0.0
    eps = (q.shape[1] + 4) * 2.0 ** -23 * float(largest) + (k.shape[0] + 40) * 2.0 ** -22
    return o, mag, v.nan_to_num(0, 0, 0).abs().sum(0), lse, eps


def check(got, lse_got, o, mag, total, lse, eps, dtype):
    # the probabilities and the result rounded to the type.  A probability below the type's normal
    # range is off by half its smallest value, 2^-25 for fp16 where the largest probability is at
    # least 2^8 (2^-134 and 1 for bf16), times its key's value: 2^-33 of the sum of all values.
    bound = mag * (ROUND[dtype] + eps) + 2 * TINY[dtype] + (2.0 ** -33 if dtype == torch.float16 else 0.0) * total
    bound = bound + ROUND[dtype] * (o.abs() + bound) + TINY[dtype]
    assert got.isfinite().all()
    assert ((got.double() - o).abs() <= bound).all(), float(((got.double() - o).abs() / bound).max())
    if lse_got is not None:
        empty = lse == -math.inf
        assert (lse_got[empty] == -math.inf).all() and not got[empty].any()
        assert ((lse_got.double() - lse).abs()[~empty] <= eps + 2.0 ** -22 * (lse[~empty].abs() + 1)).all()


def rows(shape, dtype, g, layout="bhsd", scale=1.0):
    b, h, s, d = shape
    if layout == "bshd":
        return (torch.randn((b, s, h, d), generator=g, device="cuda") * scale).to(dtype).transpose(1, 2)
    if layout == "padded":  # rows and heads further apart
        return (torch.randn((b, h + 1, s + 3, d + 8), generator=g, device="cuda") * scale).to(dtype)[:, :h, :s, :d]
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def cross(q, k, v, lengths=None, layout="bhsd"):
    """Runs and checks one call; returns o and lse."""
    b, h, sq, d = q.shape
    group, scale = h // k.shape[1], d ** -0.5
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o = rows(q.shape, q.dtype, None, layout)
    lse = torch.full((b, h, sq), 7.0, device="cuda")
    kernels.cross_attention_fwd(q, k, v, o, scale, kv_lengths=n, lse=lse)
    torch.cuda.synchronize()
    for i in range(b):
        for j in range(h):
            length = k.shape[2] if lengths is None else lengths[i]
            seen = torch.ones(sq, length, dtype=torch.bool, device="cuda")
            check(o[i, j], lse[i, j], *attend(q[i, j], k[i, j // group, :length], v[i, j // group, :length], seen,
                                              scale), q.dtype)
    return o, lse


SHAPES = [(1, 1, 1, 1, 1), (2, 3, 3, 1, 5), (1, 8, 2, 1, 700), (2, 4, 4, 33, 64), (1, 2, 1, 16, 65), (1, 2, 1, 17, 129),
          (2, 2, 2, 127, 63), (1, 6, 2, 100, 200), (1, 1, 1, 257, 1), (1, 2, 2, 300, 1025), (3, 2, 1, 64, 320),
          (1, 1, 1, 1, 5000), (1, 1, 1, 40, 5000), (1, 16, 16, 777, 333), (2, 8, 8, 31, 448), (1, 4, 4, 513, 385)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("b,hq,hk,sq,sk", SHAPES)
def test_cross(device, b, hq, hk, sq, sk, D, dtype):
    g = torch.Generator(device=device).manual_seed(sq + sk)
    cross(rows((b, hq, sq, D), dtype, g), rows((b, hk, sk, D), dtype, g), rows((b, hk, sk, D), dtype, g))


@pytest.mark.parametrize("layout", ["bshd", "padded"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("b,hq,hk,sq,sk", [(2, 4, 2, 5, 130), (2, 3, 3, 200, 77), (2, 8, 2, 1, 3000)])
def test_layouts(device, b, hq, hk, sq, sk, D, layout):
    g = torch.Generator(device=device).manual_seed(sk)
    dt = torch.bfloat16
    cross(rows((b, hq, sq, D), dt, g, layout), rows((b, hk, sk, D), dt, g, layout),
          rows((b, hk, sk, D), dt, g, "bhsd" if layout == "bshd" else "bshd"), layout=layout)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sq", [1, 32, 100, 300])
def test_padded_batches(device, sq, D, dtype):
    """Nothing behind a sequence's length is read: it may be infinite or NaN."""
    g = torch.Generator(device=device).manual_seed(sq)
    lengths = [500, 0, 1, 64, 63, 449, 65]
    q, k, v = rows((7, 2, sq, D), dtype, g), rows((7, 2, 500, D), dtype, g), rows((7, 2, 500, D), dtype, g)
    for i, n in enumerate(lengths):
        k[i, :, n:] = math.nan
        v[i, :, n::2] = math.inf
        v[i, :, n + 1::2] = math.nan
    o, lse = cross(q, k, v, lengths)
    assert not o[1].any() and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("sq", [1, 40])
def test_bad_lengths_are_not_followed(device, sq):
    g = torch.Generator(device=device).manual_seed(1)
    q, k, v = (rows((4, 2, s, 64), torch.bfloat16, g) for s in (sq, 300, 300))
    n = torch.tensor([300, 301, -1, 2 ** 31 - 1], dtype=torch.int32, device=device)
    o, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], device=device)
    kernels.cross_attention_fwd(q, k, v, o, 0.125, kv_lengths=n, lse=lse)
    assert o[0].isfinite().all() and o[1:].isnan().all() and lse[1:].isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sq", [1, 200])
@pytest.mark.parametrize("late", [3, 70, 200, 390, 600, 999])
def test_a_late_key_far_above_the_rest(device, late, sq, dtype):
    """The reference point moves, in one wave or split only: scores up to 2^8 apart."""
    g = torch.Generator(device=device).manual_seed(late)
    q, k, v = rows((1, 2, sq, 128), dtype, g), rows((1, 2, 1000, 128), dtype, g), rows((1, 2, 1000, 128), dtype, g)
    q[..., 0] = 8.0
    k[:, :, late, 0] = 8.0 * 128 ** 0.5 / 4
    cross(q, k, v)
    k[:, :, :, 0] = -30.0  # all scores far below zero: the reference point follows them down
    cross(q, k, v)


def test_infinite_values_that_are_attended(device):
    g = torch.Generator(device=device).manual_seed(2)
    for sq in (1, 50):
        q, k, v = rows((1, 1, sq, 64), torch.bfloat16, g), *(rows((1, 1, 70, 64), torch.bfloat16, g) for _ in range(2))
        v[0, 0, 69, 5] = math.inf
        v[0, 0, 3, 6] = math.nan
        o = torch.empty_like(q)
        kernels.cross_attention_fwd(q, k, v, o, 0.125)
        assert (o[..., 5] == math.inf).all() and o[..., 6].isnan().all()
        assert o[..., :5].isfinite().all() and o[..., 7:].isfinite().all()


def test_nothing_to_attend(device):
    q = torch.randn((2, 4, 3, 64), device=device).half()
    k = torch.empty((2, 2, 0, 64), device=device).half()
    o, lse = torch.full_like(q, 7.0), torch.full((2, 4, 3), 7.0, device=device)
    kernels.cross_attention_fwd(q, k, k, o, 0.125, lse=lse)
    assert not o.any() and (lse == -math.inf).all()
    none = q[:, :, :0]
    kernels.cross_attention_fwd(none, k, k, none.clone(), 0.125)
    kernels.cross_attention_fwd(q[:0], k[:0], k[:0], q[:0].clone(), 0.125)


# ------------------------------------------------------------------------------- draft trees

def paged(b, hk, D, lengths, page, g, dtype, extra=2):
    """A paged cache: caches, table, and each sequence's keys and values."""
    width = max(1, -(-max(lengths) // page))
    pages = b * width + extra
    kc, vc = rows((pages, hk, page, D), dtype, g), rows((pages, hk, page, D), dtype, g)
    table = torch.randperm(pages, generator=g, device="cuda")[:b * width].view(b, width).int()
    keys = []
    for i, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        p, r = table[i].long()[at // page], at % page
        keys.append((kc[p, :, r].transpose(0, 1), vc[p, :, r].transpose(0, 1)))  # [hk, n, D]
    return kc, vc, table, keys


def tree(q, keys, kd, vd, mask, lengths, drafts, call):
    """Runs `call(o, lse)` and checks every sequence against its keys."""
    b, h, n, d = q.shape
    group = h // kd.shape[1]
    o, lse = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda"), torch.full((b, h, n), 7.0, device="cuda")
    call(o, lse)
    torch.cuda.synchronize()
    for i in range(b):
        m = drafts[i] if drafts else n
        seen = mask if mask is None or mask.dim() == 2 else mask[i]
        if seen is None:
            seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        seen = torch.cat((torch.ones(m, lengths[i], dtype=torch.bool, device="cuda"), seen[:m, :m]), 1)
        for j in range(h):
            k = torch.cat((keys[i][0][j // group], kd[i, j // group, :m]))
            v = torch.cat((keys[i][1][j // group], vd[i, j // group, :m]))
            check(o[i, j, :m], lse[i, j, :m], *attend(q[i, j, :m], k, v, seen, d ** -0.5), q.dtype)
            assert (o[i, j, m:] == 7.0).all() and (lse[i, j, m:] == 7.0).all()
    return o, lse


def random_tree(b, n, g):
    mask = torch.zeros(b, n, n, dtype=torch.bool, device="cuda")
    for i in range(n):
        parent = (torch.rand(b, generator=g, device="cuda") * (i + 1)).long() - 1
        mask[:, i] = mask[torch.arange(b), parent.clamp(min=0)] & (parent >= 0)[:, None]
        mask[:, i, i] = True
    return mask


TREES = [(1, 1, 1, 1, [1], 16), (2, 4, 2, 7, [33, 100], 16), (1, 8, 1, 4, [129], 64), (3, 4, 4, 1, [0, 1, 600], 100),
         (2, 8, 2, 64, [500, 64], 48), (1, 4, 1, 65, [63], 7), (2, 2, 1, 130, [200, 3], 1), (4, 8, 8, 2, [2000, 17, 0, 999], 256),
         (1, 2, 2, 33, [0], 16), (1, 4, 1, 16, [9000], 128), (1, 16, 1, 12, [3001], 33)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("b,hq,hk,n,lengths,page", TREES)
def test_tree_over_pages(device, b, hq, hk, n, lengths, page, D, dtype):
    g = torch.Generator(device=device).manual_seed(n + page)
    kc, vc, table, keys = paged(b, hk, D, lengths, page, g, dtype)
    q, kd, vd = rows((b, hq, n, D), dtype, g), rows((b, hk, n, D), dtype, g), rows((b, hk, n, D), dtype, g)
    mask = random_tree(b, n, g)
    cl = torch.tensor(lengths, dtype=torch.int32, device=device)
    tree(q, keys, kd, vd, mask, lengths, None, lambda o, lse: kernels.tree_attention(
        q, kc, vc, cl, kd, vd, mask, o, D ** -0.5, block_table=table, lse=lse))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 6, 50])
def test_tree_over_one_piece(device, n, D):
    """A cache [batch, length, heads, head_dim], a chain, and a mask shared by the batch."""
    g = torch.Generator(device=device).manual_seed(n)
    dt = torch.bfloat16
    lengths = [300, 0, 64]
    kc, vc = rows((3, 2, 300, D), dt, g, "bshd"), rows((3, 2, 300, D), dt, g, "bshd")
    q, kd, vd = (rows((3, h, n, D), dt, g, "bshd") for h in (4, 2, 2))
    keys = [(kc[i, :, :m], vc[i, :, :m]) for i, m in enumerate(lengths)]
    cl = torch.tensor(lengths, dtype=torch.int32, device=device)
    for mask in (None, random_tree(1, n, g)[0]):
        tree(q, keys, kd, vd, mask, lengths, None, lambda o, lse: kernels.tree_attention(
            q, kc, vc, cl, kd, vd, mask, o, D ** -0.5, lse=lse))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,hq", [(5, 2), (20, 8), (70, 2)])
def test_drafts_of_ragged_numbers_and_rows_that_attend_nothing(device, n, hq, D):
    g = torch.Generator(device=device).manual_seed(n)
    dt, lengths, drafts = torch.float16, [0, 90, 0, 31], [n, n // 2, 1, 0]
    kc, vc, table, keys = paged(4, 1, D, lengths, 16, g, dt)
    q, kd, vd = rows((4, hq, n, D), dt, g), rows((4, 1, n, D), dt, g), rows((4, 1, n, D), dt, g)
    mask = torch.rand((4, n, n), generator=g, device=device) < 0.3
    mask[0, 2] = False  # without a cache, a row of nothing
    mask[0, n - 1, :n - 1] = False  # only its last key
    mask[0, n - 1, n - 1] = True
    mask[2, 0, 0] = False
    # what lies behind a sequence's drafted tokens may be anything, and a token that is not
    # attended by a row does not reach it
    for i, m in enumerate(drafts):
        kd[i, :, m:], vd[i, :, m:] = math.nan, math.inf
    cl, dl = (torch.tensor(t, dtype=torch.int32, device=device) for t in (lengths, drafts))

    def run(o, lse):
        kernels.tree_attention(q, kc, vc, cl, kd, vd, mask, o, D ** -0.5, block_table=table, draft_lengths=dl,
                               lse=lse)

    o, lse = tree(q, keys, kd, vd, mask, lengths, drafts, run)
    assert not o[0, :, 2].any() and (lse[0, :, 2] == -math.inf).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,hq", [(6, 2), (40, 8)])
def test_a_token_that_is_not_attended_may_hold_anything(device, n, hq, dtype):
    g = torch.Generator(device=device).manual_seed(n)
    kc, vc, table, keys = paged(1, 2, 128, [77], 16, g, dtype)
    q, kd, vd = rows((1, hq, n, 128), dtype, g), rows((1, 2, n, 128), dtype, g), rows((1, 2, n, 128), dtype, g)
    mask = random_tree(1, n, g)
    mask[0, :, 3] = False
    mask[0, 3, 3] = True
    vd[0, :, 3] = math.inf
    vd[0, :, 3, ::3] = math.nan
    cl = torch.tensor([77], dtype=torch.int32, device=device)
    o = torch.empty_like(q)
    lse = torch.empty(q.shape[:3], device=device)
    kernels.tree_attention(q, kc, vc, cl, kd, vd, mask, o, 128 ** -0.5, block_table=table, lse=lse)
    others = [i for i in range(n) if i != 3]
    for j in range(hq):
        h = j // (hq // 2)
        k, v = torch.cat((keys[0][0][h], kd[0, h])), torch.cat((keys[0][1][h], vd[0, h]))
        seen = torch.cat((torch.ones(n, 77, dtype=torch.bool, device=device), mask[0]), 1)
        want = attend(q[0, j, others], k, v, seen[others], 128 ** -0.5)
        check(o[0, j, others], lse[0, j, others], *want, dtype)
    assert o[0, :, 3, ::3].isnan().all() and (o[0, :, 3, 1::3] == math.inf).all()


@pytest.mark.parametrize("n", [1, 40])
def test_bad_pages_are_not_followed(device, n):
    g = torch.Generator(device=device).manual_seed(3)
    dt = torch.bfloat16
    lengths = [100, 100, 100, 100, 40]
    kc, vc, table, keys = paged(5, 2, 64, lengths, 16, g, dt)
    q, kd, vd = rows((5, 2, n, 64), dt, g), rows((5, 2, n, 64), dt, g), rows((5, 2, n, 64), dt, g)
    table[1, 6] = kc.shape[0]
    table[2, 0] = -1
    table[3, 3] = 2 ** 31 - 1
    table[4, 3:] = -7  # behind the length: not looked at
    cl = torch.tensor(lengths, dtype=torch.int32, device=device)
    o = torch.zeros_like(q)
    kernels.tree_attention(q, kc, vc, cl, kd, vd, None, o, 0.125, block_table=table)
    assert o[0].isfinite().all() and o[4].isfinite().all() and o[1:4].isnan().all()
    cl[0], cl[4] = table.shape[1] * 16 + 1, -1
    kernels.tree_attention(q, kc, vc, cl, kd, vd, None, o, 0.125, block_table=table)
    assert o.isnan().all()
    cl.fill_(20)
    table[:, :2] = 0
    dl = torch.tensor([n + 1, -1, n, 0, n], dtype=torch.int32, device=device)
    o.fill_(3.0)
    kernels.tree_attention(q, kc, vc, cl, kd, vd, None, o, 0.125, block_table=table, draft_lengths=dl)
    assert o[0].isnan().all() and (o[1] == 3.0).all() and o[2].isfinite().all() and (o[3] == 3.0).all()


def test_streams_and_graphs(device):
    """Split keys, whose workspaces belong to the stream and to each graph."""
    g = torch.Generator(device=device).manual_seed(4)
    dt = torch.bfloat16
    kc, vc, table, _ = paged(2, 2, 128, [3000, 1500], 64, g, dt)
    q, kd, vd = rows((2, 8, 9, 128), dt, g), rows((2, 2, 9, 128), dt, g), rows((2, 2, 9, 128), dt, g)
    k, v = rows((2, 2, 3000, 128), dt, g), rows((2, 2, 3000, 128), dt, g)
    cl = torch.tensor([3000, 1500], dtype=torch.int32, device=device)

    def step(outs, stream=None):
        kernels.tree_attention(q, kc, vc, cl, kd, vd, None, outs[0], 0.09, block_table=table, stream=stream)
        kernels.cross_attention_fwd(q, k, v, outs[1], 0.09, kv_lengths=cl, lse=outs[2], stream=stream)

    def outs():
        return [torch.empty_like(q), torch.empty_like(q), torch.empty(q.shape[:3], device=device)]

    want, side = outs(), outs()
    step(want)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    step(side, other)
    step(side, other)
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, side))
    captured, graphs = [outs(), outs()], []
    for c in captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(c)
        graphs.append(graph)
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=g, device=device))
        step(want)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c in captured:
            assert all(torch.equal(a, b) for a, b in zip(want, c))


def test_refusals(device):
    q, k = torch.zeros((2, 4, 3, 64), device=device).half(), torch.zeros((2, 2, 8, 64), device=device).half()
    o = torch.empty_like(q)
    n = torch.tensor([8, 8], dtype=torch.int32, device=device)

    def refused(error, match, q=q, k=k, v=k, o=o, scale=0.125, **kw):
        with pytest.raises(error, match=match):
            kernels.cross_attention_fwd(q, k, v, o, scale, **kw)

    refused(TypeError, "dtype", q=q.float())
    refused(TypeError, "'k'", k=k.bfloat16())
    refused(TypeError, "'o'", o=o.float())
    refused(ValueError, "HIP device", v=k.cpu())
    refused(ValueError, "'v'", v=k[:, :, :7])
    refused(ValueError, "does not fit", k=k[:1], v=k[:1])
    refused(ValueError, "does not fit", k=torch.zeros((2, 2, 8, 128), device=device).half())
    refused(ValueError, "head_dim", q=q[..., :32], o=o[..., :32])
    refused(ValueError, "share", k=torch.zeros((2, 3, 8, 64), device=device).half(),
            v=torch.zeros((2, 3, 8, 64), device=device).half())
    refused(ValueError, "share", k=k[:, :0], v=k[:, :0])
    refused(ValueError, "sm_scale", scale=0.0)
    refused(ValueError, "sm_scale", scale=math.nan)
    refused(ValueError, "kv_lengths", kv_lengths=n.long())
    refused(ValueError, "kv_lengths", kv_lengths=n[:1])
    refused(ValueError, "lse", lse=torch.zeros((2, 4, 4), device=device))
    refused(ValueError, "lse", lse=torch.zeros((2, 4, 3), device=device).half())
    refused(ValueError, "overlap", o=o[:1].expand(2, 4, 3, 64))
    odd = torch.zeros(2 * 2 * 8 * 64 + 1, device=device).half()
    refused(ValueError, "aligned", k=odd[1:].view(2, 2, 8, 64))
    refused(ValueError, "aligned", k=torch.zeros((2, 2, 8, 65), device=device).half()[..., :64])

    d = torch.zeros((2, 2, 3, 64), device=device).half()
    table = torch.zeros((2, 4), dtype=torch.int32, device=device)

    def tree_refused(error, match, kc=k, n=n, kd=d, mask=None, **kw):
        with pytest.raises(error, match=match):
            kernels.tree_attention(q, kc, kc, n, kd, d, mask, o, 0.125, **kw)

    tree_refused(TypeError, "cache_lengths", n=[8, 8])
    tree_refused(ValueError, "k_draft", kd=d[:, :1])
    tree_refused(ValueError, "tree_mask", mask=torch.ones((3, 3), device=device))
    tree_refused(ValueError, "tree_mask", mask=torch.ones((3, 4), device=device).bool())
    tree_refused(ValueError, "tree_mask", mask=torch.ones((3, 6), device=device).bool()[:, ::2])
    tree_refused(ValueError, "block_table", block_table=table.long())
    tree_refused(ValueError, "block_table", block_table=table[:1])
    tree_refused(ValueError, "block_table", block_table=torch.zeros((2, 8), device=device).int()[:, ::2])
    tree_refused(ValueError, "without pages", kc=k[:0], block_table=table)
    tree_refused(ValueError, "draft_lengths", draft_lengths=n[:1])


def test_refused_places_and_scales(device):
    q = torch.zeros((2, 4, 3, 64), device=device).half()
    k = torch.zeros((2, 4, 8, 64), device=device).half()
    d, n = q.clone(), torch.full((2,), 8, dtype=torch.int32, device=device)
    for kd, vd in ((d, q.clone()), (q.clone(), d)):
        with pytest.raises(ValueError, match="in place"):
            kernels.tree_attention(q, k, k, n, kd, vd, None, d, 0.125)
    with pytest.raises(ValueError, match="finite"):
        kernels.cross_attention_fwd(q, k, k, d, math.inf)
    # the smallest scale that has a gradient: all probabilities alike, as for a scale of 0
    v = torch.randn((2, 4, 8, 64), device=device).half()
    do, lse = torch.randn_like(q), torch.empty((2, 4, 3), device=device)
    kernels.cross_attention_fwd(q, k, v, d, 2.0 ** -100, lse=lse)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    kernels.cross_attention_bwd(do, q, k, v, d, lse, dq, dk, dv, 2.0 ** -100)
    assert not dq.any() and not dk.any()
    want = (do.double().sum(2, keepdim=True) / 8).expand(v.shape)
    # probabilities of 1/8 are exact; sums in fp32, then a rounding
    torch.testing.assert_close(dv.double(), want, rtol=2.0 ** -11 + 2.0 ** -20, atol=1e-6)


@pytest.mark.parametrize("seed", range(20))
def test_random_trees(device, seed):
    """Caches of any page size or in one piece, ragged lengths, sparse and dense masks, ragged drafts;
    page numbers behind a sequence's pages are garbage."""
    r = torch.Generator().manual_seed(seed)
    g = torch.Generator(device=device).manual_seed(seed)

    def pick(*values):
        return values[int(torch.randint(len(values), (1,), generator=r))]

    def size(lo, hi):
        return int(round(math.exp(float(torch.rand(1, generator=r)) * math.log(hi / lo)) * lo))

    dt, D = pick(torch.float16, torch.bfloat16), pick(64, 128)
    b, hk, group, n = size(1, 6), size(1, 4), pick(1, 2, 4, 8), size(1, 150)
    page = pick(1, 3, 16, 48, 64, 100, 128, 256)
    columns = size(1, max(1, 3000 // page))
    lengths = torch.randint(0, columns * page + 1, (b,), generator=r, dtype=torch.int32)
    lengths[0] = pick(0, 1, columns * page)
    drafts = pick(None, torch.randint(0, n + 1, (b,), generator=r, dtype=torch.int32))
    q, kd, vd = rows((b, hk * group, n, D), dt, g, "bshd"), rows((b, hk, n, D), dt, g, "bshd"), rows((b, hk, n, D), dt, g)
    kind = pick("chain", "shared", "own")
    mask = None if kind == "chain" else torch.rand((n, n) if kind == "shared" else (b, n, n), generator=g,
                                                   device=device) < pick(0.02, 0.5)
    table = None
    if pick(True, True, False):
        pages = b * columns + 3
        kc, vc = rows((pages, hk, page, D), dt, g), rows((pages, hk, page, D), dt, g, "bshd")
        table = torch.randperm(pages, generator=r)[:b * columns].view(b, columns).int()
        keys, values = (x[table.long().to(device)].permute(0, 2, 1, 3, 4).reshape(b, hk, -1, D) for x in (kc, vc))
        for i in range(b):
            table[i, -(-int(lengths[i]) // page):] = 2 ** 30
        table = table.to(device)
    else:
        kc, vc = rows((b, hk, columns * page, D), dt, g, "bshd"), rows((b, hk, columns * page, D), dt, g)
        keys, values = kc, vc
    o = torch.full_like(q, 7.0)
    lse = torch.full((b, hk * group, n), 7.0, device=device)
    kernels.tree_attention(q, kc, vc, lengths.to(device), kd, vd, mask, o, D ** -0.5, block_table=table, lse=lse,
                           draft_lengths=None if drafts is None else drafts.to(device))
    chain = torch.ones((n, n), dtype=torch.bool, device=device).tril()
    for i in range(b):
        cached, t = int(lengths[i]), n if drafts is None else int(drafts[i])
        own = (chain if mask is None else mask if mask.dim() == 2 else mask[i])[:t, :t]
        seen = torch.cat([torch.ones((t, cached), dtype=torch.bool, device=device), own], 1)
        assert (o[i, :, t:] == 7).all() and (lse[i, :, t:] == 7).all()
        for j in range(hk * group):
            k, v = (torch.cat([x[i, j // group, :cached], y[i, j // group, :t]]) for x, y in ((keys, kd), (values, vd)))
            check(o[i, j, :t], lse[i, j, :t], *attend(q[i, j, :t], k, v, seen, D ** -0.5), dt)
