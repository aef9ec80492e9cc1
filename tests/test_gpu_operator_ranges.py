"""Calls of the rotary and attention operators at the ends of their ranges and with operands as views: more
tokens than one launch has workgroups for, very many short sequences, hundreds of drafted tokens, tables
and masks cut out of larger ones, pages that sequences share, keys that heads and sequences share."""
import math

import pytest
import torch

from pyasc_amd import kernels
from test_gpu_kv_attention import random_tree, rows
from test_gpu_kv_attention_kernels import check_heads, check_tree
from test_gpu_rotary import U, check, norm_rows, turn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", [False, True])
def test_more_tokens_than_workgroups(device, norm):
    """2^23 workgroups of eight tokens, and as many again but for some."""
    n = (1 << 27) - 5
    g = torch.Generator(device=device).manual_seed(1)
    x = torch.randn((1, 1, n, 2), generator=g, device=device, dtype=torch.float16)
    positions = torch.arange(n, device=device, dtype=torch.int32)
    freqs = torch.full((1,), 0.1, dtype=torch.float64, device=device)
    w = torch.rand(2, generator=g, device=device) + 0.5
    out = torch.full_like(x, 7.0)
    if norm:
        kernels.qk_norm_rotary(x, None, w, None, positions, freqs, out, None, epsilon=1e-5)
    else:
        kernels.rotary(x, None, positions, freqs, out, None)
    torch.cuda.synchronize()
    for first in (0, (1 << 26) - 500, n - 1000):  # the second turn of the workgroups begins at 2^26
        part = slice(first, first + 1000)
        if norm:
            want, size, _ = norm_rows(x[:, :, part], w, positions[part], freqs, False, 1.0, 1e-5)
        else:
            want, size = turn(x[:, :, part].double(), positions[part], freqs, False, 1.0)
        # fp64 angles of 2^24 radians, each product rounded to 2^-53 of them, beside the fp32 roundings
        check(out[:, :, part], want, (30 * U + 2.0 ** -26) * size, x.dtype)
    assert not (out == 7.0).all(-1).any()


def test_many_short_sequences(device):
    """Close to 2^20 heads of one query over three keys: forward and gradients."""
    b, d, dt = (1 << 20) - 1, 64, torch.bfloat16
    g = torch.Generator(device=device).manual_seed(2)
    q, do = (torch.randn((b, 1, 1, d), generator=g, device=device, dtype=dt) for _ in range(2))
    k, v = (torch.randn((b, 1, 3, d), generator=g, device=device, dtype=dt) for _ in range(2))
    n = torch.randint(0, 4, (b,), generator=g, device=device, dtype=torch.int32)
    o, lse = torch.empty_like(q), torch.empty((b, 1, 1), device=device)
    kernels.cross_attention_fwd(q, k, v, o, 0.125, kv_lengths=n, lse=lse)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    kernels.cross_attention_bwd(do, q, k, v, o, lse, dq, dk, dv, 0.125, kv_lengths=n)
    torch.cuda.synchronize()
    r = 2.0 ** -8  # half a step of bfloat16, relative
    for part in torch.arange(b, device=device).chunk(8):
        x, y, z, w = (t[part, 0].double() for t in (q, k, v, do))
        hidden = torch.arange(3, device=device) >= n[part, None]
        s = ((x * y).sum(2) * 0.125).masked_fill(hidden, -math.inf)
        p = torch.softmax(s, 1).nan_to_num(0.0)
        dp = (w * z).sum(2)
        ds = p * (dp - (p * dp).sum(1, keepdim=True)) * 0.125
        # one rounding of a probability or a score's gradient, one of the result; the fp32 sums of 64 products
        # behind the scores and dP are off by at most 72 * 2^-23 of their terms, which ds multiplies
        f = 72 * 2.0 ** -23
        size = (x.abs() * y.abs()).sum(2) * 0.125 + 1
        dp_size = (w.abs() * z.abs()).sum(2)
        p_err = p * (r + 3 * f * size.amax(1, keepdim=True))
        ds_err = ds.abs() * (r + 3 * f * size.amax(1, keepdim=True)) + \
            0.125 * p * f * (dp_size + (p * dp_size).sum(1, keepdim=True))
        for got, want, bound in (
                (o[part, 0, 0], (p[..., None] * z).sum(1), (p_err[..., None] * z.abs()).sum(1)),
                (dq[part, 0, 0], (ds[..., None] * y).sum(1), (ds_err[..., None] * y.abs()).sum(1)),
                (dk[part, 0], ds[..., None] * x, ds_err[..., None] * x.abs()),
                (dv[part, 0], p[..., None] * w, p_err[..., None] * w.abs())):
            limit = bound + r * (want.abs() + bound) + 1e-30
            assert ((got.double() - want).abs() <= limit).all()
        assert (lse[part, 0, 0][n[part] == 0] == -math.inf).all()


@pytest.mark.parametrize("D,hq,hk", [(64, 4, 1), (128, 6, 2)])
@pytest.mark.parametrize("n", [700, 513])
def test_hundreds_of_drafted_tokens(device, n, D, hq, hk):
    """A piece of a prompt over a cache: drafted keys over many tiles, more than cached ones, in a chain and in
    a tree whose mask is cut out of a larger one."""
    g = torch.Generator(device=device).manual_seed(n)
    dt, lengths, drafts = torch.bfloat16, [200, 0, 64], [n, n - 300, 65]
    q, kd, vd = (rows((3, h, n, D), dt, g) for h in (hq, hk, hk))
    kc, vc = rows((3, hk, 200, D), dt, g), rows((3, hk, 200, D), dt, g)
    for i, m in enumerate(drafts):
        kd[i, :, m:], vd[i, :, m:] = math.nan, math.inf
    keys = [(kc[i, :, :m], vc[i, :, :m]) for i, m in enumerate(lengths)]
    cl, dl = (torch.tensor(t, dtype=torch.int32, device=device) for t in (lengths, drafts))
    larger = torch.ones((4, n + 7, n + 9), dtype=torch.bool, device=device)
    larger[1:, 3:n + 3, 5:n + 5] = random_tree(3, n, g)
    for mask in (None, larger[1:, 3:n + 3, 5:n + 5]):
        o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device=device)
        kernels.tree_attention(q, kc, vc, cl, kd, vd, mask, o, D ** -0.5, draft_lengths=dl, lse=lse)
        check_tree(o, lse, q, keys, kd, vd, mask, drafts)


@pytest.mark.parametrize("n", [1, 40])
def test_shared_pages_and_a_table_cut_out_of_a_larger_one(device, n):
    """Sequences with one prefix share its pages; a page may stand in a sequence more than once."""
    g = torch.Generator(device=device).manual_seed(n)
    dt, page, D = torch.bfloat16, 48, 64
    kc, vc = rows((9, 2, page, D), dt, g), rows((9, 2, page, D), dt, g)
    larger = torch.full((5, 12), 1 << 30, dtype=torch.int32, device=device)
    table = larger[1:4, 3:8]
    table.copy_(torch.tensor([[4, 2, 7, 0, 1], [4, 2, 8, 8, 8], [4, 4, 4, 4, 4]], device=device))
    lengths = [230, 144, 193]
    q, kd, vd = (rows((3, h, n, D), dt, g) for h in (4, 2, 2))
    keys = [tuple(c[table[i].long()].transpose(0, 1).reshape(2, 5 * page, D)[:, :m] for c in (kc, vc))
            for i, m in enumerate(lengths)]
    cl = torch.tensor(lengths, dtype=torch.int32, device=device)
    o, lse = torch.full_like(q, 7.0), torch.full(q.shape[:3], 7.0, device=device)
    kernels.tree_attention(q, kc, vc, cl, kd, vd, None, o, 0.125, block_table=table, lse=lse)
    check_tree(o, lse, q, keys, kd, vd, None, None)


def test_broadcast_operands(device):
    """One sequence's keys for all of a batch, one head's for all heads, and positions of one sequence."""
    g = torch.Generator(device=device).manual_seed(5)
    dt, D = torch.float16, 128
    q, do = rows((3, 4, 50, D), dt, g), rows((3, 4, 50, D), dt, g)
    k, v = rows((1, 1, 170, D), dt, g), rows((1, 1, 170, D), dt, g)
    wide = [t.expand(3, 2, 170, D) for t in (k, v)]
    results = []
    for keys in (wide, [t.contiguous() for t in wide]):
        o, lse = torch.empty_like(q), torch.empty((3, 4, 50), device=device)
        kernels.cross_attention_fwd(q, *keys, o, D ** -0.5, lse=lse)
        grads = [torch.empty(t.shape, dtype=dt, device=device) for t in (q, *keys)]
        kernels.cross_attention_bwd(do, q, *keys, o, lse, *grads, D ** -0.5)
        results.append([o, lse, *grads])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    o, lse = results[0][:2]
    for i in range(3):
        check_heads(o[i], lse[i], q[i], k[0].expand(4, 170, D), v[0].expand(4, 170, D),
                    torch.ones(50, 170, dtype=torch.bool, device=device))
    freqs, _ = kernels.rotary_frequencies(D)
    positions = torch.arange(50, device=device) * 3
    outs = [torch.empty_like(q) for _ in range(2)]
    kernels.rotary(q, None, positions, freqs, outs[0], None)
    kernels.rotary(q, None, positions[None].expand(3, 50), freqs, outs[1], None)
    assert torch.equal(*outs)
