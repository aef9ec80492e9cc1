"""Where results may lie: views of one buffer that share no element are taken (a projection's queries and keys
rotated in place, gradients side by side in one buffer), whatever shares one is refused."""
import pytest
import torch

from pyasc_amd import kernels

pytestmark = pytest.mark.gpu


def fused(g, b, s, heads, d):
    """[b, s, sum(heads), d] of bfloat16 and its [b, heads, s, d] views."""
    x = torch.randn((b, s, sum(heads), d), generator=g, device="cuda").bfloat16()
    views, at = [], 0
    for h in heads:
        views.append(x[:, :, at:at + h].transpose(1, 2))
        at += h
    return x, views


@pytest.mark.parametrize("b,s,hq,hk", [(1, 1, 1, 1), (2, 1, 4, 2), (3, 7, 8, 2), (2, 33, 1, 4), (1, 100, 3, 3)])
def test_a_projection_in_place(device, b, s, hq, hk):
    g = torch.Generator(device=device).manual_seed(s)
    freqs, _ = kernels.rotary_frequencies(64)
    w = torch.rand(64, generator=g, device=device)
    positions = torch.arange(s, device=device)
    x, (q, k, v) = fused(g, b, s, (hq, hk, hk), 64)
    before = x.clone()
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    kernels.qk_norm_rotary(q, k, w, w, positions, freqs, q_out, k_out, epsilon=1e-6)
    kernels.qk_norm_rotary(q, k, w, w, positions, freqs, q, k, epsilon=1e-6)
    assert torch.equal(q, q_out) and torch.equal(k, k_out) and torch.equal(v, before[:, :, hq + hk:].transpose(1, 2))
    x.copy_(before)
    kernels.rotary(q, k, positions, freqs, q_out, k_out)
    kernels.rotary(q, k, positions, freqs, q, k)
    assert torch.equal(q, q_out) and torch.equal(k, k_out) and torch.equal(v, before[:, :, hq + hk:].transpose(1, 2))
    # gradients into one buffer, in place of the results' gradients
    dx, (dq, dk, _) = fused(g, b, s, (hq, hk, hk), 64)
    dws = [torch.empty_like(w) for _ in range(4)]
    x.copy_(before)
    kernels.qk_norm_rotary_bwd(dq, dk, q, k, w, w, positions, freqs, q_out, k_out, *dws[:2], 1e-6)
    kernels.qk_norm_rotary_bwd(dq, dk, q, k, w, w, positions, freqs, dq, dk, *dws[2:], 1e-6)
    assert torch.equal(dq, q_out) and torch.equal(dk, k_out)
    assert torch.equal(dws[0], dws[2]) and torch.equal(dws[1], dws[3])


def test_weights_gradients_in_place_of_the_weights(device):
    g = torch.Generator(device=device).manual_seed(1)
    _, (q, k) = fused(g, 3, 300, (4, 2), 64)
    _, (dq, dk) = fused(g, 3, 300, (4, 2), 64)
    freqs, _ = kernels.rotary_frequencies(64)
    positions = torch.arange(300, device=device)
    w = [torch.rand(64, generator=g, device=device) for _ in range(2)]
    outs = [torch.empty_like(t) for t in (q, k, *w, q, k)]
    kernels.qk_norm_rotary_bwd(dq, dk, q, k, *w, positions, freqs, *outs[:4], 1e-6)
    kernels.qk_norm_rotary_bwd(dq, dk, q, k, *w, positions, freqs, *outs[4:], *w, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(outs[:4], outs[4:] + w))


def test_the_two_halves_of_a_head(device):
    """Rows of 64 of every 128 values: the result in the other half of the same rows."""
    g = torch.Generator(device=device).manual_seed(2)
    x = torch.randn((2, 3, 9, 128), generator=g, device=device).bfloat16()
    freqs, _ = kernels.rotary_frequencies(64)
    positions = torch.arange(9, device=device)
    want = torch.empty((2, 3, 9, 64), dtype=x.dtype, device=device)
    kernels.rotary(x[..., :64], None, positions, freqs, want, None)
    kernels.rotary(x[..., :64], None, positions, freqs, x[..., 64:], None)
    assert torch.equal(x[..., 64:], want)
    with pytest.raises(ValueError, match="overlaps"):
        kernels.rotary(x[..., :64], None, positions, freqs, x[..., 32:96], None)


def test_attention_gradients_side_by_side(device):
    g = torch.Generator(device=device).manual_seed(3)
    b, s, hq, hk, d = 2, 70, 4, 2, 64
    _, (q, k, v) = fused(g, b, s, (hq, hk, hk), d)
    do = torch.randn((b, hq, s, d), generator=g, device=device).bfloat16()
    o, lse = torch.empty_like(do), torch.empty((b, hq, s), device=device)
    kernels.cross_attention_fwd(q, k, v, o, 0.125, lse=lse)
    want = [torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v)]
    kernels.cross_attention_bwd(do, q, k, v, o, lse, *want, 0.125)
    _, grads = fused(g, b, s, (hq, hk, hk), d)
    kernels.cross_attention_bwd(do, q, k, v, o, lse, *grads, 0.125)
    assert all(torch.equal(a, c) for a, c in zip(grads, want))
    # a result next to the queries in their buffer
    x, (q2, room) = fused(g, b, s, (hq, hq), d)
    q2.copy_(q)
    kernels.cross_attention_fwd(q2, k, v, room, 0.125)
    assert torch.equal(room, o)


def test_refused(device):
    freqs, _ = kernels.rotary_frequencies(64)
    positions, w = torch.arange(9, device=device), torch.ones(64, device=device)
    x = torch.zeros(4 * 2 * 2 * 9 * 64, device=device).bfloat16()
    n = 2 * 2 * 9 * 64

    def rows(at):
        return x[at:at + n].view(2, 2, 9, 64)

    apart = torch.zeros_like(rows(0))
    for at in (1, 64, n - 1):
        with pytest.raises(ValueError, match="'q_out' overlaps 'q'"):
            kernels.rotary(rows(0), None, positions, freqs, rows(at), None)
        with pytest.raises(ValueError, match="'k_out' overlaps 'k'"):
            kernels.qk_norm_rotary(apart, rows(at), w, w, positions, freqs, apart, rows(0), epsilon=1e-6)
        with pytest.raises(ValueError, match="'q_out' overlaps 'k_out'"):
            kernels.rotary(apart, apart, positions, freqs, rows(0), rows(at))
    kernels.rotary(rows(0), None, positions, freqs, rows(n), None)  # next to each other
    dw = torch.zeros(127, device=device)
    for first, second in ((w, w), (dw[:64], dw[63:])):
        with pytest.raises(ValueError, match="'dq_weight' overlaps 'dk_weight'"):
            kernels.qk_norm_rotary_bwd(apart, apart.clone(), rows(0), rows(n), w, w, positions, freqs, rows(2 * n),
                                       rows(3 * n), first, second, 1e-6)

    q, k, v, do = (torch.zeros((2, 2, 9, 64), device=device).bfloat16() for _ in range(4))
    lse, lengths = torch.zeros((2, 2, 9), device=device), torch.full((2,), 9, dtype=torch.int32, device=device)
    with pytest.raises(ValueError, match="'o' overlaps 'k'"):
        kernels.cross_attention_fwd(q, rows(64), v, rows(0), 0.125)
    with pytest.raises(ValueError, match="'lse' overlaps 'q'"):
        kernels.cross_attention_fwd(q, k, v, rows(0), 0.125, lse=q.view(-1)[:72].view(torch.float32).view(2, 2, 9))
    with pytest.raises(ValueError, match="'o' overlaps 'v_draft'"):
        kernels.tree_attention(q, k, v, lengths, do, rows(n - 64), None, rows(0), 0.125)
    with pytest.raises(ValueError, match="'dv' overlaps 'dk'"):
        kernels.cross_attention_bwd(do, q, k, v, q, lse, rows(2 * n), rows(0), rows(n - 8), 0.125)
    with pytest.raises(ValueError, match="'dq' overlaps 'o'"):
        kernels.cross_attention_bwd(do, q, k, v, rows(8), lse, rows(0), rows(2 * n), rows(3 * n), 0.125)
