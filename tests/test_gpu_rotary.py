"""Rotary positions and the norms of queries and keys with them, against the formulas in fp64:
types, layouts of pairs, part of a head, odd sizes, strides and alignments, far positions, results
in place, the gradients (also against differences), no rows at all, streams, graphs, refusals."""
import math

import pytest
import torch

from pyasc_amd import kernels

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of fp32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def pairs_of(freqs, interleaved):
    i = torch.arange(freqs.numel(), device=freqs.device)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + freqs.numel())


def turn(x, positions, freqs, interleaved, magnitude, sign=1.0):
    """float64 x [b, h, s, d] turned, and the same with every term's size."""
    first, second = pairs_of(freqs, interleaved)
    angle = (positions.double()[..., None] * freqs)
    angle = angle[None, None] if angle.dim() == 2 else angle[:, None]
    c, s = torch.cos(angle) * magnitude, sign * torch.sin(angle) * magnitude
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), x.abs()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = abs(magnitude) * (a.abs() + b.abs())
    return y, size


def check(got, want, bound, dtype):
    """Within the bound of the fp32 computation and one rounding to dtype."""
    limit = bound + HALF_STEP[dtype] * (want.abs() + bound) + TINY[dtype]
    bad = ~((got.double() - want).abs() <= limit)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, largest excess " \
                          f"{float(((got.double() - want).abs() / limit).nan_to_num(float('inf')).max())}"


def heads(shape, dtype, g, layout):
    """[b, h, s, d] values: contiguous, a view of a projection's [b, s, h + 3, d], or at an odd
    offset of their storage with rows an odd number of elements apart."""
    b, h, s, d = shape
    if layout == "contiguous":
        return torch.randn(shape, generator=g, device="cuda").to(dtype)
    if layout == "fused":
        return torch.randn((b, s, h + 3, d), generator=g, device="cuda").to(dtype)[:, :, 1:h + 1].transpose(1, 2)
    flat = torch.randn(b * h * s * (d + 1) + 1, generator=g, device="cuda").to(dtype)
    return flat[1:].view(b, h, s, d + 1)[..., :d]


SHAPES = [(1, 1, 1, 1, 128, 128), (2, 3, 2, 5, 128, 64), (1, 8, 1, 33, 64, 64), (3, 5, 5, 4, 80, 20),
          (2, 2, 1, 7, 96, 96), (1, 2, 2, 3, 2, 2), (2, 3, 1, 2, 512, 512), (1, 1, 1, 9, 20, 4), (1, 4, 2, 600, 256, 128),
          (70, 2, 1, 11, 64, 32), (1, 2, 1, 6, 128, 0)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["contiguous", "fused", "odd"])
@pytest.mark.parametrize("b,hq,hk,s,d,rot", SHAPES)
def test_rotary(device, b, hq, hk, s, d, rot, layout, interleaved, dtype):
    g = torch.Generator(device=device).manual_seed(d + s)
    q, k = heads((b, hq, s, d), dtype, g, layout), heads((b, hk, s, d), dtype, g, layout)
    freqs = kernels.rotary_frequencies(rot)[0] if rot else torch.empty(0, dtype=torch.float64, device=device)
    positions = torch.randint(0, 200000, (b, s), generator=g, device=device)
    for backward in (False, True):
        qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
        kernels.rotary(q, k, positions, freqs, qo, ko, interleaved=interleaved, magnitude=1.25, backward=backward)
        for x, y in ((q, qo), (k, ko)):
            want, size = turn(x.double(), positions, freqs, interleaved, 1.25, -1.0 if backward else 1.0)
            # the angle to 2^-27, cos and sin to two ulp, the magnitude, a product and a sum
            check(y, want, 9 * U * size, dtype)
            if rot < d:
                assert torch.equal(y[..., rot:], x[..., rot:])


def test_far_positions_and_int32(device):
    x = torch.randn((1, 2, 4, 128), device=device)
    freqs, _ = kernels.rotary_frequencies(128)
    positions = torch.tensor([2 ** 31 - 1, 2 ** 31 - 2, -5, 123456789], device=device)
    out, out32 = torch.empty_like(x), torch.empty_like(x)
    kernels.rotary(x, None, positions, freqs, out, None)
    kernels.rotary(x, None, positions.int(), freqs, out32, None)
    want, size = turn(x.double(), positions, freqs, False, 1.0)
    # fp64 angles of 2^31 radians: both products round to 2^-53 of them
    check(out, want, (9 * U + 2.0 ** -20) * size, torch.float32)
    assert torch.equal(out, out32)


def test_values_behind_the_rotated_ones_may_be_anything(device):
    x = torch.randn((1, 1, 3, 64), device=device)
    x[..., 40] = math.inf
    x[..., 50] = math.nan
    freqs, _ = kernels.rotary_frequencies(32)
    out = torch.empty_like(x)
    kernels.rotary(x, None, torch.arange(3, device=device), freqs, out, None)
    assert torch.equal(out[..., 32:].nan_to_num(3.0), x[..., 32:].nan_to_num(3.0))
    assert out[..., :32].isfinite().all()


def norm_rows(x, w, positions, freqs, interleaved, magnitude, eps):
    r = 1 / torch.sqrt(x.double().pow(2).mean(-1, keepdim=True) + eps)
    return turn(x.double() * r * w.double(), positions, freqs, interleaved, magnitude) + (r,)


def norm_grad(dy, x, w, positions, freqs, interleaved, magnitude, eps):
    """dx, dw in fp64 and the sizes of the terms in them."""
    x, w = x.double(), w.double()
    r = 1 / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    g, size = turn(dy.double(), positions, freqs, interleaved, magnitude, -1.0)
    xr = x * r
    dx = r * (g * w - xr * (g * w * xr).mean(-1, keepdim=True))
    # 22 additions per sum of squares (half of it after the root) and few roundings per factor
    dx_size = r * (40 * size * w.abs() + 80 * xr.abs() * (size * w.abs() * xr.abs()).mean(-1, keepdim=True))
    return dx, (g * xr).sum((0, 1, 2)), dx_size, (size * xr.abs()).sum((0, 1, 2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["contiguous", "fused", "odd"])
@pytest.mark.parametrize("b,hq,hk,s,d,rot", SHAPES)
def test_norm_and_its_gradient(device, b, hq, hk, s, d, rot, layout, interleaved, dtype):
    g = torch.Generator(device=device).manual_seed(d + s)
    x = [heads((b, h, s, d), dtype, g, layout) for h in (hq, hk)]
    dy = [heads((b, h, s, d), dtype, g, "contiguous" if layout == "fused" else layout) for h in (hq, hk)]
    w = [1 + 0.3 * torch.randn(d, generator=g, device=device) for _ in range(2)]
    freqs = kernels.rotary_frequencies(rot)[0] if rot else torch.empty(0, dtype=torch.float64, device=device)
    positions = torch.randint(0, 5000, (s,), generator=g, device=device, dtype=torch.int32)
    out = [torch.full_like(t, 7.0) for t in x]
    kernels.qk_norm_rotary(*x, *w, positions, freqs, *out, epsilon=1e-5, interleaved=interleaved, magnitude=0.75)
    dx = [torch.full_like(t, 7.0) for t in x]
    dw = [torch.full_like(t, 7.0) for t in w]
    kernels.qk_norm_rotary_bwd(*dy, *x, *w, positions, freqs, *dx, *dw, epsilon=1e-5, interleaved=interleaved,
                               magnitude=0.75)
    for i in range(2):
        want, size, _ = norm_rows(x[i], w[i], positions, freqs, interleaved, 0.75, 1e-5)
        check(out[i], want, 30 * U * size, dtype)
        want_dx, want_dw, dx_size, dw_size = norm_grad(dy[i], x[i], w[i], positions, freqs, interleaved, 0.75, 1e-5)
        check(dx[i], want_dx, U * dx_size, dtype)
        n = x[i].numel() // d  # at most so many additions in fp32
        check(dw[i], want_dw, (n + 40) * U * dw_size, torch.float32)


def test_gradient_against_differences(device):
    g = torch.Generator(device=device).manual_seed(5)
    x = torch.randn((1, 2, 3, 16), generator=g, device=device)
    w = 1 + 0.3 * torch.randn(16, generator=g, device=device)
    up = torch.randn(x.shape, generator=g, device=device)
    positions = torch.arange(3, device=device) * 7
    freqs, m = kernels.rotary_frequencies(8, scaling="yarn", factor=8.0, original_length=64)

    def loss(x, w):
        return (norm_rows(x, w, positions, freqs, True, m, 1e-6)[0] * up.double()).sum()

    dx, dw = torch.empty_like(x), torch.empty_like(w)
    kernels.qk_norm_rotary_bwd(up, None, x, None, w, None, positions, freqs, dx, None, dw, None, 1e-6, True, m)
    step = 1e-5
    for t, grad in ((x, dx), (w, dw)):
        for i in range(0, t.numel(), 5):
            e = torch.zeros(t.numel(), dtype=torch.float64, device=device)
            e[i] = step
            e = e.view(t.shape)
            lo = loss(*((x.double() - e, w) if t is x else (x, w.double() - e)))
            hi = loss(*((x.double() + e, w) if t is x else (x, w.double() + e)))
            # third derivatives of order one: the difference is off by about step^2
            assert abs(float((hi - lo) / (2 * step)) - float(grad.flatten()[i])) <= 1e-5


@pytest.mark.parametrize("layout", ["contiguous", "fused"])
def test_in_place(device, layout):
    g = torch.Generator(device=device).manual_seed(1)
    q, k = heads((2, 4, 9, 64), torch.bfloat16, g, layout), heads((2, 2, 9, 64), torch.bfloat16, g, layout)
    w = torch.rand(64, generator=g, device=device)
    freqs, _ = kernels.rotary_frequencies(64)
    positions = torch.arange(9, device=device)
    out = [torch.empty_like(q), torch.empty_like(k)]
    kernels.qk_norm_rotary(q, k, w, w, positions, freqs, *out, epsilon=1e-6)
    dq, dk, dw, dw2 = torch.empty_like(q), torch.empty_like(k), torch.empty_like(w), torch.empty_like(w)
    kernels.qk_norm_rotary_bwd(out[0], out[1], q, k, w, w, positions, freqs, dq, dk, dw, dw2, 1e-6)
    dy = [out[0].clone(), out[1].clone()]
    dwa, dwb = torch.empty_like(w), torch.empty_like(w)
    kernels.qk_norm_rotary_bwd(dy[0], dy[1], q, k, w, w, positions, freqs, dy[0], dy[1], dwa, dwb, 1e-6)
    assert torch.equal(dy[0], dq) and torch.equal(dy[1], dk) and torch.equal(dwa, dw) and torch.equal(dwb, dw2)
    kernels.qk_norm_rotary(q, k, w, w, positions, freqs, q, k, epsilon=1e-6)
    assert torch.equal(q, out[0]) and torch.equal(k, out[1])


def test_rows_of_zeros_and_no_rows(device):
    freqs, _ = kernels.rotary_frequencies(64)
    w = torch.ones(64, device=device)
    x = torch.zeros((1, 2, 3, 64), device=device)
    out, dx, dw = torch.full_like(x, 7.0), torch.full_like(x, 7.0), torch.full_like(w, 7.0)
    positions = torch.arange(3, device=device)
    kernels.qk_norm_rotary(x, None, w, None, positions, freqs, out, None, epsilon=1e-6)
    kernels.qk_norm_rotary_bwd(x, None, x, None, w, None, positions, freqs, dx, None, dw, None, 1e-6)
    assert not out.any() and not dx.any() and not dw.any()
    none = x[:, :, :0]
    dw.fill_(7.0)
    kernels.rotary(none, None, positions[:0], freqs, none.clone(), None)
    kernels.qk_norm_rotary(none, None, w, None, positions[:0], freqs, none.clone(), None, epsilon=1e-6)
    kernels.qk_norm_rotary_bwd(none, None, none, None, w, None, positions[:0], freqs, none.clone(), None, dw, None,
                               1e-6)
    assert not dw.any()


def test_broadcast_inputs(device):
    q = torch.randn((1, 1, 5, 64), device=device).bfloat16()
    freqs, _ = kernels.rotary_frequencies(64)
    positions = torch.arange(5, device=device)
    wide = q.expand(3, 4, 5, 64)
    out, one = torch.empty(wide.shape, dtype=q.dtype, device=device), torch.empty_like(q)
    kernels.rotary(wide, None, positions, freqs, out, None)
    kernels.rotary(q, None, positions, freqs, one, None)
    assert torch.equal(out, one.expand(3, 4, 5, 64))
    with pytest.raises(ValueError, match="overlap"):
        kernels.rotary(out, None, positions, freqs, wide, None)


def test_two_streams_and_a_graph(device):
    g = torch.Generator(device=device).manual_seed(3)
    q, k, dq_out, dk_out = (torch.randn((2, 4, 65, 128), generator=g, device=device).bfloat16() for _ in range(4))
    w = torch.rand(128, generator=g, device=device)
    freqs, _ = kernels.rotary_frequencies(128)
    positions = torch.arange(65, device=device)

    def step(outs, stream=None):
        kernels.qk_norm_rotary(q, k, w, w, positions, freqs, outs[0], outs[1], epsilon=1e-6, stream=stream)
        kernels.qk_norm_rotary_bwd(dq_out, dk_out, q, k, w, w, positions, freqs, *outs[2:], epsilon=1e-6,
                                   stream=stream)

    def outs():
        return [torch.empty_like(t) for t in (q, k, q, k, w, w)]

    want, side = outs(), outs()
    step(want)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    step(side, other)
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, side))
    captured = outs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured)
    for seed in range(3):
        for t in (q, k, dq_out, dk_out):
            t.copy_(torch.randn(t.shape, generator=g, device=device))
        step(want)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, captured))


def test_refusals(device):
    q = torch.zeros((1, 2, 3, 64), device=device)
    freqs, _ = kernels.rotary_frequencies(64)
    p = torch.arange(3, device=device)
    w = torch.ones(64, device=device)
    out = torch.empty_like(q)

    def refused(error, match, *args, **kw):
        with pytest.raises(error, match=match):
            kernels.rotary(*args, **kw)

    refused(TypeError, "Tensor", 3, None, p, freqs, out, None)
    refused(TypeError, "dtype", q.double(), None, p, freqs, out, None)
    refused(ValueError, "HIP device", q.cpu(), None, p, freqs, out, None)
    refused(ValueError, "batch, heads", q[0], None, p, freqs, out, None)
    refused(ValueError, "last dimension", q.transpose(2, 3).contiguous().transpose(2, 3), None, p, freqs, out, None)
    refused(ValueError, "q_out", q, None, p, freqs, out[:, :1], None)
    refused(TypeError, "q_out", q, None, p, freqs, out.half(), None)
    refused(ValueError, "together", q, q, p, freqs, out, None)
    refused(ValueError, "'k'", q, q[:, :, :2], p, freqs, out, out)
    refused(ValueError, "positions", q, None, p[:2], freqs, out, None)
    refused(TypeError, "positions", q, None, p.float(), freqs, out, None)
    refused(ValueError, "freqs", q, None, p, freqs.float(), out, None)
    refused(ValueError, "freqs", q, None, p, torch.ones(33, dtype=torch.float64, device=device), out, None)
    refused(ValueError, "head_dim", q[..., :63], None, p, freqs[:2], out[..., :63], None)
    refused(ValueError, "in place", q, None, p, freqs,
            q.as_strided(q.shape, (384, 64, 128, 1)), None)
    big = torch.zeros((1, 1, 1, 514), device=device)
    refused(ValueError, "head_dim", big, None, p[:1], freqs, big.clone(), None)
    with pytest.raises(ValueError, match="q_weight"):
        kernels.qk_norm_rotary(q, None, w[:32], None, p, freqs, out, None, epsilon=1e-6)
    with pytest.raises(ValueError, match="epsilon"):
        kernels.qk_norm_rotary(q, None, w, None, p, freqs, out, None, epsilon=-1.0)
    with pytest.raises(ValueError, match="dk_out"):
        kernels.qk_norm_rotary_bwd(q, None, q, q, w, w, p, freqs, out, out.clone(), w, w, 1e-6)


def test_refused_places(device):
    q, k = torch.zeros((1, 2, 3, 64), device=device), torch.zeros((1, 2, 3, 64), device=device)
    p, (freqs, _) = torch.arange(3, device=device), kernels.rotary_frequencies(64)
    w = torch.ones(64, device=device)
    other = q.clone()
    for outs in ((k, other), (other, q), (other, other)):
        with pytest.raises(ValueError, match="in place of k's"):
            kernels.rotary(q, k, p, freqs, *outs)
    dq, dk = q.clone(), k.clone()
    for outs in ((dk, other), (other, dq)):
        with pytest.raises(ValueError, match="in place of k's"):
            kernels.qk_norm_rotary_bwd(dq, dk, q, k, w, w, p, freqs, *outs, w.clone(), w.clone(), 1e-6)
    none = torch.zeros((1, 0, 3, 64), device=device)  # nothing to write: nothing to refuse
    kernels.rotary(none, none, p, freqs, none, none)
    kernels.rotary(none, k, p, freqs, none, k)


@pytest.mark.parametrize("dtype,layout", [(torch.float32, "contiguous"), (torch.bfloat16, "odd"),
                                          (torch.float16, "fused")])
@pytest.mark.parametrize("b,hq,hk,s,d,rot", [(3, 1, 2, 1301, 512, 512), (9, 2, 2, 901, 128, 32), (2, 5, 1, 2500, 64, 64),
                                             (1100, 1, 1, 3, 130, 2), (1, 33, 3, 1027, 48, 16)])
def test_many_tokens_of_few_heads(device, b, hq, hk, s, d, rot, dtype, layout):
    # several tokens per workgroup, of fewer or more heads than its pass has rows, the last ones odd
    test_rotary(device, b, hq, hk, s, d, rot, layout, False, dtype)
    test_norm_and_its_gradient(device, b, hq, hk, s, d, rot, layout, True, dtype)
