"""The attention block's operators as they are used together: a training step (projection, norms and
rotation, cross attention, and every gradient back to the projected values and weights), and serving
(a prompt into a paged cache, drafted tokens over it, accepted ones into the cache), on the
framework's own products and attention; caches beyond 2^32 bytes; random shapes."""
import math

import pytest
import torch

from pyasc_amd import kernels

pytestmark = pytest.mark.gpu
DT = torch.bfloat16


def _norm_rotate(x, w, positions, freqs, eps):
    """qk_norm_rotary in fp64 with torch's gradients (half layout, whole heads)."""
    y = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    angle = positions.double()[:, None] * freqs
    c, s = torch.cos(angle), torch.sin(angle)
    a, b = y.chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


@pytest.mark.parametrize("D,hq,hk", [(64, 4, 2), (128, 4, 4)])
def test_a_training_step(device, D, hq, hk):
    B, Sq, Sk, W = 2, 75, 130, 256
    g = torch.Generator(device=device).manual_seed(D)
    x = torch.randn((B * Sq, W), generator=g, device=device).to(DT)
    wq = (torch.randn((W, hq * D), generator=g, device=device) * W ** -0.5).to(DT)
    k, v = (torch.randn((B, hk, Sk, D), generator=g, device=device).to(DT) for _ in range(2))
    qw, kw = (1 + 0.2 * torch.randn(D, generator=g, device=device) for _ in range(2))
    do = torch.randn((B, hq, Sq, D), generator=g, device=device).to(DT)
    lengths = torch.tensor([Sk, 77], dtype=torch.int32, device=device)
    freqs, _ = kernels.rotary_frequencies(D)
    positions, kpos = torch.arange(Sq, device=device) + 3, torch.arange(Sk, device=device)
    scale, eps = D ** -0.5, 1e-6

    proj = torch.empty((B * Sq, hq * D), dtype=DT, device=device)
    kernels.matmul(x, wq, proj)
    q = proj.view(B, Sq, hq, D).transpose(1, 2)
    qr = torch.empty((B, hq, Sq, D), dtype=DT, device=device)
    kr, o = torch.empty_like(k), torch.empty_like(qr)
    lse = torch.empty((B, hq, Sq), device=device)
    kernels.qk_norm_rotary(q, None, qw, None, positions, freqs, qr, None, epsilon=eps)
    kernels.qk_norm_rotary(k, None, kw, None, kpos, freqs, kr, None, epsilon=eps)
    kernels.cross_attention_fwd(qr, kr, v, o, scale, kv_lengths=lengths, lse=lse)
    dqr, dkr, dv = torch.empty_like(qr), torch.empty_like(kr), torch.empty_like(v)
    kernels.cross_attention_bwd(do, qr, kr, v, o, lse, dqr, dkr, dv, scale, kv_lengths=lengths)
    dq, dk, dqw, dkw = torch.empty_like(q), torch.empty_like(k), torch.empty_like(qw), torch.empty_like(kw)
    kernels.qk_norm_rotary_bwd(dqr, None, q, None, qw, None, positions, freqs, dq, None, dqw, None, eps)
    kernels.qk_norm_rotary_bwd(dkr, None, k, None, kw, None, kpos, freqs, dk, None, dkw, None, eps)

    # the same in fp64 by torch's autograd, from the projected values
    ins = [t.double().detach().requires_grad_() for t in (q, k, v, qw, kw)]
    a, b = _norm_rotate(ins[0], ins[3], positions, freqs, eps), _norm_rotate(ins[1], ins[4], kpos, freqs, eps)
    rep = hq // hk
    s = torch.matmul(a, b.repeat_interleave(rep, 1).transpose(2, 3).contiguous()) * scale
    s = s.masked_fill((torch.arange(Sk, device=device) >= lengths[:, None])[:, None, None], -math.inf)
    want = torch.matmul(torch.softmax(s, 3), ins[2].repeat_interleave(rep, 1))
    want.backward(do.double())
    # Each result passes through at most six roundings to bf16 one after the other (the rotated
    # values, probabilities, o, the scores' gradients, their sums, the result), each 2^-9 of its
    # value on average and independent: all elements together stay within 6 * 2^-8 of the norm.
    for name, got, ref in [("o", o, want), ("dq", dq, ins[0].grad), ("dk", dk, ins[1].grad), ("dv", dv, ins[2].grad),
                           ("dqw", dqw, ins[3].grad), ("dkw", dkw, ins[4].grad)]:
        err = float((got.double() - ref.detach()).norm() / ref.detach().norm())
        assert err <= 6 * 2.0 ** -8, (name, err)
    assert not dk[1, :, 77:].any() and not dv[1, :, 77:].any()


@pytest.mark.parametrize("D,page", [(64, 16), (128, 48)])
def test_drafting_and_accepting(device, D, page):
    """A prompt of P tokens lies in a paged cache; n drafted tokens, a chain, are attended over it and
    then join the cache; the same tokens' rows of causal attention over the whole sequence."""
    B, h, P, n, steps = 2, 4, 200, 6, 3
    S = P + n * steps
    g = torch.Generator(device=device).manual_seed(page)
    q, k, v = (torch.randn((B, h, S, D), generator=g, device=device).to(DT) for _ in range(3))
    w = 1 + 0.1 * torch.randn(D, generator=g, device=device)
    freqs, m = kernels.rotary_frequencies(D, scaling="yarn", factor=4.0, original_length=64)
    positions = torch.arange(S, device=device)
    qr, kr = torch.empty_like(q), torch.empty_like(k)
    kernels.qk_norm_rotary(q, k, w, w, positions, freqs, qr, kr, epsilon=1e-6, magnitude=m)
    whole = torch.empty_like(q)
    kernels.flash_attention_fwd(qr, kr, v, whole, D ** -0.5, True)

    width = -(-S // page)
    kc, vc = (torch.full((B * width, h, page, D), math.nan, dtype=DT, device=device) for _ in range(2))
    table = torch.randperm(B * width, generator=g, device=device).view(B, width).int()

    def put(first, last, keys, values):
        for b in range(B):
            at = torch.arange(first, last, device=device)
            pg, row = table[b].long()[at // page], at % page
            kc[pg, :, row], vc[pg, :, row] = keys[b].transpose(0, 1), values[b].transpose(0, 1)

    put(0, P, kr[:, :, :P], v[:, :, :P])
    for step in range(steps):
        at = P + n * step
        part = slice(at, at + n)
        # the drafted tokens' queries and keys alone, at their positions
        qd, kd = torch.empty((B, h, n, D), dtype=DT, device=device), torch.empty((B, h, n, D), dtype=DT, device=device)
        kernels.qk_norm_rotary(q[:, :, part], k[:, :, part], w, w, positions[part], freqs, qd, kd, epsilon=1e-6,
                               magnitude=m)
        assert torch.equal(qd, qr[:, :, part]) and torch.equal(kd, kr[:, :, part])
        o = torch.empty_like(qd)
        vd = v[:, :, part]
        kernels.tree_attention(qd, kc, vc, torch.full((B,), at, dtype=torch.int32, device=device), kd, vd, None, o,
                               D ** -0.5, block_table=table)
        # both round their probabilities and results to bf16: 2 * (2^-8 + 2^-8) of the values' size
        limit = 4 * 2.0 ** -8 * float(v.abs().max())
        assert float((o.double() - whole[:, :, part].double()).abs().max()) <= limit
        put(at, at + n, kd, vd)
    torch.cuda.synchronize()


def test_a_cache_beyond_32_bits(device):
    """Pages at both ends of a cache of 6 GiB, and a sequence whose rows lie 40 MB apart."""
    g = torch.Generator(device=device).manual_seed(1)
    pages, page = 1 << 17, 200
    kc, vc = (torch.empty((pages, 1, page, 128), dtype=DT, device=device) for _ in range(2))
    used = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32, device=device)
    for p in used[0].tolist():
        kc[p], vc[p] = (torch.randn((1, page, 128), generator=g, device=device).to(DT) for _ in range(2))
    for n in (1, 40):
        q, kd, vd = (torch.randn((1, 1, n, 128), generator=g, device=device).to(DT) for _ in range(3))
        o, dense = torch.empty_like(q), torch.empty_like(q)
        cl = torch.tensor([550], dtype=torch.int32, device=device)
        kernels.tree_attention(q, kc, vc, cl, kd, vd, None, o, 0.09, block_table=used)
        k1, v1 = (c[used[0].long()].transpose(0, 1).reshape(1, 1, 3 * page, 128) for c in (kc, vc))
        kernels.tree_attention(q, k1, v1, cl, kd, vd, None, dense, 0.09)
        assert torch.equal(o, dense)
    far = kc.view(-1)[:90 * (20 << 20)].view(1, 1, 90, 20 << 20)[..., :128]
    far.copy_(torch.randn((1, 1, 90, 128), generator=g, device=device))
    near = far.contiguous()
    q, do = (torch.randn((1, 1, 70, 128), generator=g, device=device).to(DT) for _ in range(2))
    outs = []
    for kv in (far, near):
        o, lse = torch.empty_like(q), torch.empty((1, 1, 70), device=device)
        kernels.cross_attention_fwd(q, kv, kv, o, 0.09, lse=lse)
        grads = [torch.empty_like(q), torch.empty_like(near), torch.empty_like(near)]
        kernels.cross_attention_bwd(do, q, kv, kv, o, lse, *grads, 0.09)
        x = torch.empty_like(near)
        kernels.rotary(kv, None, torch.arange(90, device=device), kernels.rotary_frequencies(128)[0], x, None)
        outs.append([o, lse, *grads, x])
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("seed", range(24))
def test_random_shapes(device, seed):
    """Whole calls against fp64 by the norm of the error: two roundings to the type, as above."""
    r = torch.Generator().manual_seed(seed)

    def pick(*values):
        return values[int(torch.randint(len(values), (1,), generator=r))]

    def size(lo, hi):
        return int(round(math.exp(float(torch.rand(1, generator=r)) * math.log(hi / lo)) * lo))

    g = torch.Generator(device=device).manual_seed(seed)
    dt, D = pick(torch.float16, DT), pick(64, 128)
    b, hk, group = size(1, 6), size(1, 6), pick(1, 2, 4, 8)
    sq, sk = size(1, 700), size(1, 3000)
    q, do = (torch.randn((b, hk * group, sq, D), generator=g, device=device).to(dt) for _ in range(2))
    k, v = (torch.randn((b, sk, hk, D), generator=g, device=device).to(dt).transpose(1, 2) for _ in range(2))
    n = torch.randint(0, sk + 1, (b,), generator=g, device=device, dtype=torch.int32)
    o, lse = torch.empty_like(q), torch.empty(q.shape[:3], device=device)
    kernels.cross_attention_fwd(q, k, v, o, D ** -0.5, kv_lengths=n, lse=lse)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    kernels.cross_attention_bwd(do, q, k, v, o, lse, *grads, D ** -0.5, kv_lengths=n)
    wants = [torch.zeros(t.shape, dtype=torch.float64, device=device) for t in (q, q, k, v)]
    for i in range(b):
        m = int(n[i])
        if m == 0:
            continue
        ins = [t.double().detach().requires_grad_() for t in (q[i], k[i, :, :m], v[i, :, :m])]
        kx, vx = (t.repeat_interleave(group, 0) for t in ins[1:])
        s = torch.matmul(ins[0], kx.transpose(1, 2).contiguous()) * D ** -0.5
        out = torch.matmul(torch.softmax(s, 2), vx)
        out.backward(do[i].double())
        wants[0][i], wants[1][i] = out.detach(), ins[0].grad
        wants[2][i, :, :m], wants[3][i, :, :m] = ins[1].grad, ins[2].grad
    for name, got, want in zip(("o", "dq", "dk", "dv"), [o, *grads], wants):
        size_of = float(want.norm())
        # one key's probability is 1 whatever its score: nothing is left of dq and dk but roundings
        floor = 1e-3 * float(do.double().norm())
        err = float((got.double() - want).norm())
        assert err <= 4 * torch.finfo(dt).eps / 2 * size_of + floor * torch.finfo(dt).eps, (name, err, size_of)
