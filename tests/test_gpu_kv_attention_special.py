"""Infinities and NaN among the values, and lengths and pages outside the cache, in both kernels of attention
over other keys than the queries' own, with and without a split of the keys: they reach the rows that
attend them, through the parts of the splits too, and no others."""
import math

import pytest
import torch

from pyasc_amd import kernels
from test_gpu_kv_attention import random_tree, rows
from test_gpu_kv_attention_kernels import CROSS, TREES, check_heads, lengths_of, tree_case
from test_kv_attention_plans import LAUNCHES

pytestmark = pytest.mark.gpu


def results(q):
    return torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", TREES)
def test_drafted_values(device, name, dtype):
    """Tokens that only they themselves attend, in the first and in the last tile of drafted keys, hold
    infinities and NaN: every other row is as if they held zeros."""
    g = torch.Generator(device=device).manual_seed(11)
    q, kc, vc, table, keys, kd, vd, lengths = tree_case(name, dtype, g, 64)
    b, hq, n, D = q.shape
    mask = random_tree(b, n, g)
    odd = sorted({3, n - 2})
    mask[:, :, odd] = False
    mask[:, odd, odd] = True
    clean = vd.clone()
    clean[:, :, odd] = 0
    vd[:, :, odd] = math.inf
    vd[:, :, odd, 1::3] = -math.inf
    vd[:, :, odd, 2::3] = math.nan
    cl = torch.tensor(lengths, dtype=torch.int32, device=device)
    o, lse = results(q)
    kernels.tree_attention(q, kc, vc, cl, kd, vd, mask, o, D ** -0.5, block_table=table, lse=lse)
    torch.cuda.synchronize()
    others = [i for i in range(n) if i not in odd]
    for i, (k, v) in enumerate(keys):
        k, v = torch.cat((k, kd[i]), 1), torch.cat((v, clean[i]), 1)
        seen = torch.cat((torch.ones(n, lengths[i], dtype=torch.bool, device=device), mask[i]), 1)
        check_heads(o[i][:, others], lse[i][:, others], q[i][:, others], k, v, seen[others])
    assert (o[:, :, odd, 0::3] == math.inf).all() and (o[:, :, odd, 1::3] == -math.inf).all()
    assert o[:, :, odd, 2::3].isnan().all() and lse.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", CROSS)
def test_values_that_all_rows_attend(device, name, dtype):
    b, hq, hk, n, kv_len, D, _ = LAUNCHES[name][0]
    g = torch.Generator(device=device).manual_seed(12)
    q, k, v = (rows((b, h, s, D), dtype, g) for h, s in ((hq, n), (hk, kv_len), (hk, kv_len)))
    want, _ = results(q)
    kernels.cross_attention_fwd(q, k, v, want, D ** -0.5)
    for i in range(b):  # one key each, in another place of another sequence
        v[i, :, (kv_len - 1) * i // b, 5], v[i, :, (kv_len - 1) * (b - i) // b, 6] = math.inf, math.nan
    o, lse = results(q)
    kernels.cross_attention_fwd(q, k, v, o, D ** -0.5, lse=lse)
    assert (o[..., 5] == math.inf).all() and o[..., 6].isnan().all() and lse.isfinite().all()
    rest = [c for c in range(D) if c not in (5, 6)]
    assert torch.equal(o[..., rest], want[..., rest])


@pytest.mark.parametrize("name", TREES)
def test_bad_pages(device, name):
    g = torch.Generator(device=device).manual_seed(13)
    q, kc, vc, table, keys, kd, vd, lengths = tree_case(name, torch.bfloat16, g, 64)
    b, _, n, D = q.shape
    cl = torch.tensor(lengths, dtype=torch.int32, device=device)
    for i, m in enumerate(lengths):
        table[i, -(-m // 64):] = -7  # behind the length: not looked at
    want, want_lse = results(q)
    kernels.tree_attention(q, kc, vc, cl, kd, vd, None, want, D ** -0.5, block_table=table, lse=want_lse)
    assert want.isfinite().all() and want_lse.isfinite().all()
    # one page of a sequence: the first, one in the middle or the last that its length reaches
    for place in (0.0, 0.5, 1.0):
        broken = table.clone()
        bad = [i for i in (0, 2, 4) if i < b]
        for i, page in zip(bad, (kc.shape[0], -1, 2 ** 31 - 1)):
            broken[i, int((-(-lengths[i] // 64) - 1) * place)] = page
        o, lse = results(q)
        kernels.tree_attention(q, kc, vc, cl, kd, vd, None, o, D ** -0.5, block_table=broken, lse=lse)
        assert o[bad].isnan().all() and lse[bad].isnan().all()
        good = [i for i in range(b) if i not in bad]
        assert torch.equal(o[good], want[good]) and torch.equal(lse[good], want_lse[good])


@pytest.mark.parametrize("name", CROSS + TREES)
def test_bad_lengths(device, name):
    b, hq, hk, n, kv_len, D, drafted = LAUNCHES[name][0]
    g = torch.Generator(device=device).manual_seed(14)
    q, kd, vd = (rows((b, h, n, D), torch.bfloat16, g) for h in (hq, hk, hk))
    k, v = (rows((b, hk, kv_len, D), torch.bfloat16, g) for _ in range(2))

    def run(lengths, drafts=None):
        o, lse = results(q)
        cl = torch.tensor(lengths, dtype=torch.int32, device=device)
        if drafted:
            dl = None if drafts is None else torch.tensor(drafts, dtype=torch.int32, device=device)
            kernels.tree_attention(q, k, v, cl, kd, vd, None, o, D ** -0.5, lse=lse, draft_lengths=dl)
        else:
            kernels.cross_attention_fwd(q, k, v, o, D ** -0.5, kv_lengths=cl, lse=lse)
        return o, lse

    lengths = [min(m, kv_len) for m in lengths_of(b, kv_len)]
    want, want_lse = run(lengths)
    for i, bad in ((0, kv_len + 1), (1, -1), (2, 2 ** 31 - 1), (0, -2 ** 31)):
        o, lse = run(lengths[:i] + [bad] + lengths[i + 1:])
        good = [j for j in range(b) if j != i]
        assert o[i].isnan().all() and lse[i].isnan().all()
        assert torch.equal(o[good], want[good]) and torch.equal(lse[good], want_lse[good])
    if drafted:
        o, lse = run(lengths, [n + 1] + [n] * (b - 1))
        assert o[0].isnan().all() and lse[0].isnan().all()
        assert torch.equal(o[1:], want[1:]) and torch.equal(lse[1:], want_lse[1:])
