"""The gradients of cross attention against the formulas in fp64 and against differences: lengths,
shared heads, layouts, padded batches, sequences without keys, few rows or keys (split sums),
streams, graphs, refusals."""
import math

import pytest
import torch

from pyasc_amd import kernels

pytestmark = pytest.mark.gpu
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
SMALL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half the smallest value


def reference(do, q, k, v, o, lse, scale, dtype):
    """dq, dk, dv of one query head in fp64, from the forward pass's lse, each with its bound before it
    is rounded to the type."""
    do, q, k, v, o, lse = (t.double().contiguous() for t in (do, q, k, v, o, lse))
    kt, vt = k.T.contiguous(), v.T.contiguous()
    p = torch.exp((q @ kt) * scale - lse[:, None])
    # fp32: D products per score with the largest initial value, exp2 and its argument
    rel = (q.shape[1] + 8) * 2.0 ** -23 * (float((q.abs() @ kt.abs()).amax()) * scale + float(lse.abs().amax()) + 1)
    dp = do @ vt
    delta = (p * dp).sum(1, keepdim=True)
    ds = p * (dp - delta)
    # delta may come from o, which was rounded to the type after its probabilities were
    r, small = ROUND[dtype], SMALL[dtype]
    dp_err = (q.shape[1] + 8) * 2.0 ** -23 * (do.abs() @ vt.abs() + (do * o).abs().sum(1, keepdim=True))
    dp_err = dp_err + (r * (do * o).abs() + (r + rel) * (do.abs() * (p @ v.abs()))).sum(1, keepdim=True)
    p_err = p * (rel + r * (1 + rel)) + small
    ds_err = (ds.abs() * rel + p * (1 + rel) * dp_err) * (1 + r) + ds.abs() * r + small
    n, m = k.shape[0], q.shape[0]
    add = lambda terms: (terms + 64) * 2.0 ** -23  # noqa: E731  terms added in fp32
    T = lambda t: t.T.contiguous()  # noqa: E731
    dq = ds @ k * scale, (ds_err @ k.abs() + add(n) * ((ds.abs() + ds_err) @ k.abs())) * scale
    dk = T(ds) @ q * scale, (T(ds_err) @ q.abs() + add(m) * (T(ds.abs() + ds_err) @ q.abs())) * scale
    dv = T(p) @ do, T(p_err) @ do.abs() + add(m) * (T(p + p_err) @ do.abs())
    return dq, dk, dv


def check(name, got, want, bound, dtype):
    limit = bound + ROUND[dtype] * (want.abs() + bound) + SMALL[dtype]
    assert ((got.double() - want).abs() <= limit).all(), (name, float(((got.double() - want).abs() / limit).max()))


def rows(shape, dtype, g, layout="bhsd", scale=1.0):
    b, h, s, d = shape
    if layout == "bshd":
        return (torch.randn((b, s, h, d), generator=g, device="cuda") * scale).to(dtype).transpose(1, 2)
    if layout == "padded":
        return (torch.randn((b, h + 1, s + 3, d + 8), generator=g, device="cuda") * scale).to(dtype)[:, :h, :s, :d]
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def run(q, k, v, do, lengths=None, layout="bhsd", stream=None):
    b, h, sq, d = q.shape
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    o, lse = torch.empty_like(q), torch.empty((b, h, sq), device="cuda")
    kernels.cross_attention_fwd(q, k, v, o, d ** -0.5, kv_lengths=n, lse=lse, stream=stream)
    grads = [rows(t.shape, q.dtype, None, layout) for t in (q, k, v)]
    kernels.cross_attention_bwd(do, q, k, v, o, lse, *grads, d ** -0.5, kv_lengths=n, stream=stream)
    return o, lse, grads


def check_run(q, k, v, do, lengths=None, layout="bhsd"):
    o, lse, (dq, dk, dv) = run(q, k, v, do, lengths, layout)
    torch.cuda.synchronize()
    b, h, sq, d = q.shape
    hk, dt = k.shape[1], q.dtype
    for i in range(b):
        length = k.shape[2] if lengths is None else lengths[i]
        assert not dk[i, :, length:].any() and not dv[i, :, length:].any()
        if length == 0:
            assert not dq[i].any()
            continue
        for j in range(hk):
            sums = [0.0, 0.0, 0.0, 0.0]
            for g in range(j * h // hk, (j + 1) * h // hk):
                a = reference(do[i, g], q[i, g], k[i, j, :length], v[i, j, :length], o[i, g], lse[i, g], d ** -0.5, dt)
                check("dq", dq[i, g], *a[0], dt)
                sums = [s + t for s, t in zip(sums, (*a[1], *a[2]))]
            check("dk", dk[i, j, :length], sums[0], sums[1], dt)
            check("dv", dv[i, j, :length], sums[2], sums[3], dt)


SHAPES = [(1, 1, 1, 1, 1), (2, 3, 3, 1, 5), (1, 4, 2, 1, 700), (2, 4, 1, 33, 64), (1, 2, 1, 16, 65), (1, 1, 1, 31, 129),
          (2, 2, 2, 127, 63), (1, 6, 2, 100, 200), (1, 1, 1, 300, 1), (1, 2, 2, 300, 517), (1, 1, 1, 5, 3000),
          (1, 1, 1, 3000, 5), (1, 8, 4, 777, 333), (3, 2, 1, 257, 256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("b,hq,hk,sq,sk", SHAPES)
def test_gradients(device, b, hq, hk, sq, sk, D, dtype):
    g = torch.Generator(device=device).manual_seed(sq + sk)
    check_run(rows((b, hq, sq, D), dtype, g), rows((b, hk, sk, D), dtype, g), rows((b, hk, sk, D), dtype, g),
              rows((b, hq, sq, D), dtype, g))


@pytest.mark.parametrize("layout", ["bshd", "padded"])
@pytest.mark.parametrize("D", [64, 128])
def test_layouts(device, D, layout):
    g = torch.Generator(device=device).manual_seed(D)
    dt = torch.bfloat16
    check_run(rows((2, 4, 70, D), dt, g, layout), rows((2, 2, 150, D), dt, g, layout), rows((2, 2, 150, D), dt, g),
              rows((2, 4, 70, D), dt, g, "bhsd" if layout == "bshd" else "bshd"), layout=layout)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sq", [1, 40, 300])
def test_padded_batches(device, sq, D, dtype):
    g = torch.Generator(device=device).manual_seed(sq)
    lengths = [260, 0, 1, 64, 63, 129]
    q, do = rows((6, 2, sq, D), dtype, g), rows((6, 2, sq, D), dtype, g)
    k, v = rows((6, 1, 260, D), dtype, g), rows((6, 1, 260, D), dtype, g)
    for i, n in enumerate(lengths):
        k[i, :, n:] = math.nan
        v[i, :, n:] = math.inf
    check_run(q, k, v, do, lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[108, 193], [70, 2000], [256, 257], [1, 0]])
def test_few_keys_where_many_could_be(device, lengths, D, dtype):
    """The keys are split for the longest sequence there could be, and a short one's are not."""
    g = torch.Generator(device=device).manual_seed(lengths[0])
    q, do = rows((2, 2, 1, D), dtype, g), rows((2, 2, 1, D), dtype, g)
    check_run(q, rows((2, 1, 2000, D), dtype, g), rows((2, 1, 2000, D), dtype, g), do, lengths)


@pytest.mark.parametrize("D", [64, 128])
def test_scores_far_below_zero(device, D):
    """exp of a padding row's score against such an lse overflows: it must not reach the sums."""
    g = torch.Generator(device=device).manual_seed(D)
    q, k, v, do = (rows((1, 1, s, D), torch.bfloat16, g) for s in (33, 45, 45, 33))
    q[..., 0], k[..., 0] = 40.0, -40.0
    check_run(q, k, v, do)


def test_broadcast_gradient(device):
    """The gradient of a sum: one value, expanded."""
    g = torch.Generator(device=device).manual_seed(8)
    q, k, v = (rows((2, 2, s, 64), torch.bfloat16, g) for s in (40, 70, 70))
    one = torch.ones((1, 1, 1, 64), dtype=torch.bfloat16, device=device).expand(2, 2, 40, 64)
    a, b = run(q, k, v, one)[2], run(q, k, v, one.contiguous())[2]
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_against_differences(device):
    """Directional differences of the loss sum(o * do) in fp64, along random directions."""
    g = torch.Generator(device=device).manual_seed(6)
    dt = torch.float16
    q, k, v, do = (rows((1, h, s, 64), dt, g) for h, s in ((4, 50), (2, 90), (2, 90), (4, 50)))
    _, _, grads = run(q, k, v, do)

    def loss(q, k, v):
        kx, vx = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        s = torch.matmul(q, kx.transpose(2, 3).contiguous()) / 8
        return (torch.matmul(torch.softmax(s, 3), vx) * do.double()).sum()

    ins = [t.double() for t in (q, k, v)]
    step = 1e-5
    for i in range(3):
        for _ in range(3):
            e = torch.randn(ins[i].shape, generator=g, device=device, dtype=torch.float64)
            hi, lo = ([t + (step * e * sign if j == i else 0) for j, t in enumerate(ins)] for sign in (1, -1))
            want = float((loss(*hi) - loss(*lo)) / (2 * step))
            got = float((grads[i].double() * e).sum())
            # every element of a gradient within 2^-9 of the largest: the sum within its norm's share
            assert abs(got - want) <= 2.0 ** -9 * float(grads[i].abs().max()) * e.numel() ** 0.5 * 4


@pytest.mark.parametrize("sq", [3, 200])
def test_bad_lengths_are_not_followed(device, sq):
    g = torch.Generator(device=device).manual_seed(1)
    q, k, v, do = (rows((3, 2, s, 64), torch.bfloat16, g) for s in (sq, 300, 300, sq))
    _, _, grads = run(q, k, v, do, [300, 301, -1])
    for t in grads:
        assert t[0].isfinite().all() and t[1:].isnan().all()


def test_no_queries_and_no_keys(device):
    q, k = torch.randn((2, 4, 3, 64), device=device).half(), torch.randn((2, 2, 9, 64), device=device).half()
    o, lse, grads = run(q, k[:, :, :0], k[:, :, :0], q)
    assert not grads[0].any()
    none = q[:, :, :0]
    _, _, grads = run(none, k, k, none)
    assert not grads[1].any() and not grads[2].any()
    run(q[:0], k[:0], k[:0], q[:0])


def test_streams_and_graphs(device):
    g = torch.Generator(device=device).manual_seed(4)
    dt = torch.bfloat16
    q, k, v, do = (rows((2, h, s, 128), dt, g) for h, s in ((4, 300), (2, 500), (2, 500), (4, 300)))
    n = torch.tensor([500, 77], dtype=torch.int32, device=device)

    def outs():
        return [torch.empty_like(t) for t in (q, k, v, q)] + [torch.empty(q.shape[:3], device=device)]

    def step(x, stream=None):
        kernels.cross_attention_fwd(q, k, v, x[3], 0.09, kv_lengths=n, lse=x[4], stream=stream)
        kernels.cross_attention_bwd(do, q, k, v, x[3], x[4], *x[:3], 0.09, kv_lengths=n, stream=stream)

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
        for t in (q, do):
            t.copy_(torch.randn(t.shape, generator=g, device=device))
        step(want)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c in captured:
            assert all(torch.equal(a, b) for a, b in zip(want, c))


def test_refusals(device):
    q, k = torch.zeros((1, 2, 3, 64), device=device).half(), torch.zeros((1, 2, 8, 64), device=device).half()
    lse = torch.zeros((1, 2, 3), device=device)

    def refused(error, match, do=q.clone(), lse=lse, dq=q.clone(), dk=k.clone(), dv=k.clone()):
        with pytest.raises(error, match=match):
            kernels.cross_attention_bwd(do, q, k, k, q, lse, dq, dk, dv, 0.125)

    refused(TypeError, "lse", lse=None)
    refused(ValueError, "lse", lse=lse[:, :1])
    refused(ValueError, "'do'", do=q[:, :1])
    refused(TypeError, "'do'", do=q.float())
    refused(TypeError, "'dq'", dq=q.float())
    refused(ValueError, "'dk'", dk=k[:, :1])
    refused(ValueError, "overlap", dv=k[:, :1].expand(1, 2, 8, 64))
    refused(ValueError, "in place", dq=q)
    refused(ValueError, "in place", dv=k)
    same = k.clone()
    refused(ValueError, "in place", dk=same, dv=same)
