"""The gradients of cross attention in float16 where the probabilities or the scores' gradients lie outside
the type's normal range (2^-14 to 65504): many keys, small and large gradients, rows and keys whose
gradients are far apart.  Against fp64 and, in bfloat16, the same calls."""
import math

import pytest
import torch

from pyasc_amd import kernels
from test_gpu_kv_attention_bwd import ROUND, SMALL, rows

pytestmark = pytest.mark.gpu


def bounds(do, q, k, v, o, lse, scale, dtype):
    """dq, dk, dv of one head in fp64 from the forward pass's o and lse, and bounds before the results are
    rounded.  Probabilities and scores' gradients are rounded to the type's precision, not to its range: a
    probability to 2^-39 at least (float16: half of 2^-24, at 2^14 times its value), a score's gradient to
    2^-32 of the largest of the row (of dq) or key (of dk) that it is summed for (half of 2^-24 where that
    one is at least 2^7)."""
    do, q, k, v, o, lse = (t.double().contiguous() for t in (do, q, k, v, o, lse))
    T = lambda t: t.T.contiguous()  # noqa: E731
    kt, vt = T(k), T(v)
    s = (q @ kt) * scale
    p = torch.exp(s - lse[:, None])
    d, r = q.shape[1], ROUND[dtype]
    # fp32: D products per score with the largest initial value, exp2 and its argument
    rel = (d + 8) * 2.0 ** -23 * (float((q.abs() @ kt.abs()).amax()) * scale + float(lse.abs().amax()) + 1)
    dp = do @ vt
    delta = (p * dp).sum(1, keepdim=True)
    ds = p * (dp - delta)
    # delta may come from o, which was rounded to the type after its probabilities were
    dp_err = (d + 8) * 2.0 ** -23 * (do.abs() @ vt.abs() + (do * o).abs().sum(1, keepdim=True))
    dp_err = dp_err + (r * (do * o).abs() + (r + rel) * (do.abs() * (p @ v.abs()))).sum(1, keepdim=True)
    p_err = p * (rel + r * (1 + rel)) + 2.0 ** -39
    ds_err = (ds.abs() * rel + p * (1 + rel) * dp_err) * (1 + r) + ds.abs() * r
    largest = ds.abs() + ds_err
    q_err = ds_err + 2.0 ** -32 * largest.amax(1, keepdim=True)
    k_err = ds_err + 2.0 ** -32 * largest.amax(0, keepdim=True)
    add = lambda terms: (terms + 64) * 2.0 ** -23  # noqa: E731  terms added in fp32
    n, m = k.shape[0], q.shape[0]
    dq = ds @ k * scale, (q_err @ k.abs() + add(n) * ((ds.abs() + q_err) @ k.abs())) * scale
    dk = T(ds) @ q * scale, (T(k_err) @ q.abs() + add(m) * (T(ds.abs() + k_err) @ q.abs())) * scale
    dv = T(p) @ do, T(p_err) @ do.abs() + add(m) * (T(p + p_err) @ do.abs())
    return dq, dk, dv


def check_run(q, k, v, do):
    b, h, sq, d = q.shape
    hk, dt = k.shape[1], q.dtype
    o, lse = torch.empty_like(q), torch.empty((b, h, sq), device="cuda")
    kernels.cross_attention_fwd(q, k, v, o, d ** -0.5, lse=lse)
    dq, dk, dv = (torch.full_like(t, 7.0) for t in (q, k, v))
    kernels.cross_attention_bwd(do, q, k, v, o, lse, dq, dk, dv, d ** -0.5)
    torch.cuda.synchronize()

    def check(name, got, want, bound):
        limit = bound + ROUND[dt] * (want.abs() + bound) + SMALL[dt]
        # from half a step above the type's largest value on, infinity is the rounded result
        top = torch.finfo(dt).max * (1 + ROUND[dt] / 2)
        near = (got.double() - want).abs() <= limit
        beyond = (got.double() == want.sign() * math.inf) & (want.abs() + bound >= top)
        assert (near | beyond).all(), (name, int((~(near | beyond)).sum()))

    for i in range(b):
        for j in range(hk):
            sums = [0.0] * 4
            for g in range(j * h // hk, (j + 1) * h // hk):
                a = bounds(do[i, g], q[i, g], k[i, j], v[i, j], o[i, g], lse[i, g], d ** -0.5, dt)
                check("dq", dq[i, g], *a[0])
                sums = [s + t for s, t in zip(sums, (*a[1], *a[2]))]
            check("dk", dk[i, j], *sums[:2])
            check("dv", dv[i, j], *sums[2:])
    return o, lse, dq, dk, dv


HALVES = [torch.float16, torch.bfloat16]
# few rows (keys or rows split over workgroups, several heads' queries in a tile) and many
SHAPES = [(1, 1, 1, 64, 8192), (2, 4, 2, 5, 4000), (1, 2, 1, 700, 333), (1, 8, 1, 3, 150), (8, 16, 8, 260, 700)]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("b,hq,hk,sq,sk", SHAPES)
def test_small_gradients(device, b, hq, hk, sq, sk, D, dtype):
    """Gradients of 2^-10, the size of an unscaled mean's: their shares of many keys lie below 2^-14."""
    g = torch.Generator(device=device).manual_seed(sk)
    q, k, v, do = (rows((b, h, s, D), dtype, g, scale=c) for h, s, c in
                   ((hq, sq, 1.0), (hk, sk, 1.0), (hk, sk, 64.0), (hq, sq, 2.0 ** -10)))
    check_run(q, k, v, do)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("name,b,hq,hk,sq,sk", [("dq", *s) for s in SHAPES] + [("dk", *s) for s in SHAPES] +
                         [("dv", 1, 1, 1, 256, 1 << 18)])
def test_small_shares_by_the_norm(device, name, b, hq, hk, sq, sk, D, dtype):
    """Probabilities, or scores' gradients, far below 2^-14 in sums that are not: a result passes through at
    most four roundings (the forward pass's probabilities and o, the operand of its sum, itself), each
    half a step of its value at most and independent, and what lies below 2^-14 of the result itself."""
    g = torch.Generator(device=device).manual_seed(sk)
    size = {"dq": (2.0 ** -6, 64.0, 2.0 ** -12), "dk": (64.0, 2.0 ** -6, 2.0 ** -12), "dv": (1.0, 1.0, 1.0)}[name]
    q, k, v, do = (rows((b, h, s, D), dtype, g, scale=c) for h, s, c in
                   ((hq, sq, size[0]), (hk, sk, size[1]), (hk, sk, 1.0), (hq, sq, size[2])))
    o, lse = torch.empty_like(q), torch.empty((b, hq, sq), device=device)
    kernels.cross_attention_fwd(q, k, v, o, D ** -0.5, lse=lse)
    grads = dict(zip(("dq", "dk", "dv"), [torch.empty_like(t) for t in (q, k, v)]))
    kernels.cross_attention_bwd(do, q, k, v, o, lse, *grads.values(), D ** -0.5)
    x, y, z, w = q.double(), *(t.double().repeat_interleave(hq // hk, 1) for t in (k, v)), do.double()
    s = torch.matmul(x, y.transpose(2, 3).contiguous()) * D ** -0.5
    p = torch.softmax(s, 3)
    dp = torch.matmul(w, z.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(3, keepdim=True)) * D ** -0.5
    if name == "dq":
        want = torch.matmul(ds, y)
    else:
        a, c = (ds, x) if name == "dk" else (p, w)
        want = torch.matmul(a.transpose(2, 3).contiguous(), c).view(b, hk, hq // hk, sk, D).sum(2)
    err = float((grads[name].double() - want).norm())
    assert err <= 4 * ROUND[dtype] * float(want.norm()) + SMALL[dtype] * want.numel() ** 0.5, err / float(want.norm())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("b,hq,hk,sq,sk", SHAPES)
def test_large_scores_gradients(device, b, hq, hk, sq, sk, D, dtype):
    """Scores' gradients beyond 65504, most of whose sums are not."""
    g = torch.Generator(device=device).manual_seed(sk)
    q, k, v, do = (rows((b, h, s, D), dtype, g, scale=c) for h, s, c in
                   ((hq, sq, 2.0 ** -7), (hk, sk, 2.0 ** -7), (hk, sk, 256.0), (hq, sq, 256.0)))
    q[..., 0], k[:, :, ::64, 0] = 8.0, 8.0  # few keys have most of the probability
    o, _, dq, dk, dv = check_run(q, k, v, do)
    assert all(t.isfinite().all() for t in (o, dq[..., 1:], dk[..., 1:], dv))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_gradients_far_apart(device, order, D, dtype):
    """The rows' gradients, and the keys' values, differ by up to 2^16 from tile to tile, so that the powers
    of two that they are held at move while the sums grow."""
    g = torch.Generator(device=device).manual_seed(3)
    sq, sk = 300, 450
    q, k, v, do = (rows((2, h, s, D), dtype, g) for h, s in ((4, sq), (2, sk), (2, sk), (4, sq)))
    for t, n in ((do, sq), (v, sk)):
        steps = torch.linspace(-8, 8, n, device=device).round()
        if order == "down":
            steps = steps.flip(0)
        if order == "mixed":
            steps = steps[torch.randperm(n, generator=g, device=device)]
        t.mul_(torch.exp2(steps)[:, None].to(dtype))
    check_run(q, k, v, do)


def test_rows_of_zeros_and_infinite_gradients(device):
    """A gradient of zeros gives zeros, an infinite one reaches its row of dq and every dk and dv."""
    g = torch.Generator(device=device).manual_seed(4)
    q, k, v, do = (rows((1, 1, s, 64), torch.float16, g) for s in (100, 200, 200, 100))
    do[0, 0, :40] = 0
    _, _, dq, dk, dv = check_run(q, k, v, do)
    assert not dq[0, 0, :40].any()
    do[0, 0, 50, 7] = math.inf
    o, lse = torch.empty_like(q), torch.empty((1, 1, 100), device=device)
    kernels.cross_attention_fwd(q, k, v, o, 0.125, lse=lse)
    more = [torch.empty_like(t) for t in (q, k, v)]
    kernels.cross_attention_bwd(do, q, k, v, o, lse, *more, 0.125)
    assert not more[0][0, 0, 50].isfinite().any() and not more[1].isfinite().any()
    others = [i for i in range(100) if i != 50]
    assert torch.equal(more[0][0, 0, others], dq[0, 0, others])
    assert (more[2][0, 0, :, 7] == math.inf).all() and more[2][0, 0, :, :7].isfinite().all()
