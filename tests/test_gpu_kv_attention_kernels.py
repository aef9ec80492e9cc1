"""Both kernels of attention over other keys than the queries' own, with and without a split of the keys,
at the launches that test_kv_attention_plans.py holds them to, against the formulas in fp64: every
number of key tiles of a chain, odd ends, no keys, rows in the last block of few, drafted keys over
several tiles, pages that end inside a tile, rows that attend nothing."""
import math

import pytest
import torch

from pyasc_amd import kernels
from test_gpu_kv_attention import ROUND, TINY, paged, random_tree, rows
from test_kv_attention_plans import LAUNCHES, launch_of

pytestmark = pytest.mark.gpu
CROSS = [n for n in LAUNCHES if n.startswith("cross")]
TREES = [n for n in LAUNCHES if n.startswith("tree")]


def check_heads(o, lse, q, k, v, seen):
    """All heads [h, n, D] of one sequence over its keys [h_kv, m, D], of which row i attends seen[i]; with the
    bounds of test_gpu_kv_attention.check, head by head."""
    h, n, d = q.shape
    dtype, m, scale = q.dtype, k.shape[1], d ** -0.5
    q, k, v = q.double(), *(t.double().repeat_interleave(h // t.shape[0], 0) for t in (k, v))
    kt = k.transpose(1, 2).contiguous()
    s = torch.matmul(q, kt).mul_(scale).masked_fill_(~seen, -math.inf)
    size = torch.matmul(q.abs(), kt.abs()).mul_(scale).masked_fill_(~seen, 0)
    want_lse = torch.logsumexp(s, 2)
    p = torch.exp(s - want_lse[..., None].nan_to_num(0, 0, 0))
    want, mag = torch.matmul(p, v), torch.matmul(p, v.abs())
    # fp32: D products per score and the FMA before exp2, m terms per sum, exp2 and log2 to 2^-21
    largest = size.amax((1, 2), keepdim=True) if size.numel() else size.new_zeros(h, 1, 1)
    eps = (d + 4) * 2.0 ** -23 * largest + (m + 40) * 2.0 ** -22
    bound = mag * (ROUND[dtype] + eps) + 2 * TINY[dtype]
    if dtype == torch.float16:  # probabilities below the type's normal range
        bound = bound + 2.0 ** -33 * v.abs().sum(1, keepdim=True)
    bound = bound + ROUND[dtype] * (want.abs() + bound) + TINY[dtype]
    assert o.isfinite().all()
    assert ((o.double() - want).abs() <= bound).all(), float(((o.double() - want).abs() / bound).max())
    empty = want_lse == -math.inf
    assert (lse[empty] == -math.inf).all() and not o[empty].any()
    off = ((lse.double() - want_lse).abs() - eps[..., 0] - 2.0 ** -22 * (want_lse.abs() + 1))[~empty]
    assert (off <= 0).all(), float(off.max())


def cross(q, k, v, lengths):
    """Runs and checks one call; returns o and lse."""
    o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device="cuda")
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    kernels.cross_attention_fwd(q, k, v, o, q.shape[3] ** -0.5, kv_lengths=n, lse=lse)
    torch.cuda.synchronize()
    for i, m in enumerate(lengths):
        seen = torch.ones(q.shape[2], m, dtype=torch.bool, device="cuda")
        check_heads(o[i], lse[i], q[i], k[i, :, :m], v[i, :, :m], seen)
    return o, lse


def lengths_of(batch, most):
    """Of a batch's sequences: all keys, none, one, whole tiles of 64 and odd ends."""
    return ([most, 0, 65, 191, most - 64, 1, 64, 256, 129, 320, 447, 385] * 2)[:batch]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", CROSS)
def test_cross(device, name, dtype):
    b, hq, hk, n, kv_len, D, _ = LAUNCHES[name][0]
    g = torch.Generator(device=device).manual_seed(n)
    lengths = [min(m, kv_len) for m in lengths_of(b, kv_len)]
    q, k, v = rows((b, hq, n, D), dtype, g), rows((b, hk, kv_len, D), dtype, g, "bshd"), rows((b, hk, kv_len, D), dtype, g)
    for i, m in enumerate(lengths):  # what lies behind a sequence is not read
        k[i, :, m:] = math.nan
        v[i, :, m::2], v[i, :, m + 1::2] = math.inf, math.nan
    o, lse = cross(q, k, v, lengths)
    assert not o[1].any() and (lse[1] == -math.inf).all()


@pytest.mark.parametrize("name", CROSS)
def test_chains_of_tiles(device, name):
    """Sequences of 1 to 7 and of 20 tiles, the last one whole, without a key or with one: the loop over
    whole tiles starts and ends at every stage of its ring."""
    b, hq, hk, n, kv_len, D, _ = LAUNCHES[name][0]
    g = torch.Generator(device=device).manual_seed(D)
    q, k, v = (rows((b, h, s, D), torch.bfloat16, g) for h, s in ((hq, n), (hk, kv_len), (hk, kv_len)))
    k[..., 0] *= 3  # scores far enough apart for the reference point to move on the way
    chains = [t * 64 - less for t in (1, 2, 3, 4, 5, 6, 7, 20) for less in (0, 1, 63) if t * 64 <= kv_len]
    for at in range(0, len(chains), b):
        part = chains[at:at + b]
        cross(q, k, v, part + [0] * (b - len(part)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", CROSS)
def test_late_keys_far_above_the_rest(device, name, dtype):
    b, hq, hk, n, kv_len, D, _ = LAUNCHES[name][0]
    g = torch.Generator(device=device).manual_seed(7)
    q, k, v = (rows((b, h, s, D), dtype, g) for h, s in ((hq, n), (hk, kv_len), (hk, kv_len)))
    q[..., 0] = 8.0
    for i in range(b):  # another key for each sequence
        k[i, :, (kv_len - 1) * (b - i) // b, 0] = 8.0 * D ** 0.5 / 4
    cross(q, k, v, [kv_len] * b)


def tree_case(name, dtype, g, page):
    """A call of the launch `name` over a cache of `page` rows a page."""
    (b, hq, hk, n, kv_len, D, _), kernel, split = LAUNCHES[name]
    lengths = [min(m, kv_len) for m in lengths_of(b, kv_len)]
    kc, vc, table, keys = paged(b, hk, D, lengths, page, g, dtype)
    got, _, splits = launch_of(b, hq, hk, n, table.shape[1] * page, D, True)
    assert got == kernel and (splits > 1) == split
    q, kd, vd = rows((b, hq, n, D), dtype, g), rows((b, hk, n, D), dtype, g, "bshd"), rows((b, hk, n, D), dtype, g)
    for i, m in enumerate(lengths):  # the rows of a last page behind its sequence
        if m % page:
            last = int(table[i, m // page])
            kc[last, :, m % page:], vc[last, :, m % page:] = math.nan, math.inf
    return q, kc, vc, table, keys, kd, vd, lengths


def check_tree(o, lse, q, keys, kd, vd, mask, drafts):
    """Every sequence's written rows; those behind its drafted tokens hold what they held."""
    torch.cuda.synchronize()
    n = q.shape[2]
    for i, (k, v) in enumerate(keys):
        m = drafts[i] if drafts else n
        own = torch.ones(n, n, dtype=torch.bool, device="cuda").tril() if mask is None else mask[i]
        seen = torch.cat((torch.ones(m, k.shape[1], dtype=torch.bool, device="cuda"), own[:m, :m]), 1)
        check_heads(o[i, :, :m], lse[i, :, :m], q[i, :, :m], torch.cat((k, kd[i, :, :m]), 1),
                    torch.cat((v, vd[i, :, :m]), 1), seen)
        assert (o[i, :, m:] == 7.0).all() and (lse[i, :, m:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 64, 100])
@pytest.mark.parametrize("name", TREES)
def test_trees(device, name, page, dtype):
    g = torch.Generator(device=device).manual_seed(page)
    q, kc, vc, table, keys, kd, vd, lengths = tree_case(name, dtype, g, page)
    b, _, n, D = q.shape
    drafts = ([n, n // 2, n, 1, 0, n - 1] * 2 + [n])[:b]
    mask = random_tree(b, n, g)
    mask[1, 2] = False  # no cached key there: a row of nothing
    for i, m in enumerate(drafts):
        kd[i, :, m:], vd[i, :, m:] = math.nan, math.inf
    cl, dl = (torch.tensor(t, dtype=torch.int32, device=device) for t in (lengths, drafts))
    o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device=device)
    kernels.tree_attention(q, kc, vc, cl, kd, vd, mask, o, D ** -0.5, block_table=table, draft_lengths=dl, lse=lse)
    check_tree(o, lse, q, keys, kd, vd, mask, drafts)
    assert not o[1, :, 2].any() and (lse[1, :, 2] == -math.inf).all()


@pytest.mark.parametrize("name", TREES)
def test_chains_of_drafts_behind_one_piece(device, name):
    """A cache in one piece, the drafted tokens a chain."""
    b, hq, hk, n, kv_len, D, _ = LAUNCHES[name][0]
    g = torch.Generator(device=device).manual_seed(3)
    dt, lengths = torch.bfloat16, [min(m, kv_len) for m in lengths_of(b, kv_len)]
    q, kd, vd = (rows((b, h, n, D), dt, g, "bshd") for h in (hq, hk, hk))
    kc, vc = rows((b, hk, kv_len, D), dt, g, "bshd"), rows((b, hk, kv_len, D), dt, g)
    cl = torch.tensor(lengths, dtype=torch.int32, device=device)
    o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device=device)
    kernels.tree_attention(q, kc, vc, cl, kd, vd, None, o, D ** -0.5, lse=lse)
    check_tree(o, lse, q, [(kc[i, :, :m], vc[i, :, :m]) for i, m in enumerate(lengths)], kd, vd, None, None)
