"""Penalties, biases and masks on logits against the formula in fp64."""
import math

import pytest
import torch

from pyasc_amd import kernels

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def reference(x, history, lengths, prompts, repetition, frequency, presence, bias, mask):
    """The result in fp64, and the sum of its terms' sizes."""
    out, size = x.double().cpu(), x.double().abs().cpu()
    rows, vocab = out.shape
    for i in range(rows):
        n = int(lengths[i])
        prompt = 0 if prompts is None else max(0, min(n, int(prompts[i])))
        tokens = history[i].cpu().long()
        ok = (tokens >= 0) & (tokens < vocab)
        seen = tokens[:n][ok[:n]].unique()
        r = 1.0 if repetition is None else float(repetition[i])
        y = out[i, seen]
        out[i, seen] = torch.where(y > 0, y / r, y * r)
        size[i, seen] = torch.maximum(size[i, seen], out[i, seen].abs())
        t, c = tokens[prompt:n][ok[prompt:n]].unique(return_counts=True)
        f = 0.0 if frequency is None else float(frequency[i])
        p = 0.0 if presence is None else float(presence[i])
        out[i, t] -= f * c + p
        size[i, t] += abs(f) * c + abs(p)
    if bias is not None:
        out, size = out + bias.double().cpu(), size + bias.double().abs().cpu()
    if mask is not None:
        bits = (mask.cpu()[:, :, None] >> torch.arange(32)) & 1
        out[bits.flatten(1)[:, :vocab] == 0] = -math.inf
    return out, size


def check(got, out, size):
    """Five fp32 operations and one rounding to the type: half a step each, of at most the terms' sizes."""
    eps = torch.finfo(got.dtype).eps / 2
    got = got.double().cpu()
    fine = out.isfinite()
    assert torch.equal(got.isfinite(), fine) and torch.equal(got[~fine].nan_to_num(5.0), out[~fine].nan_to_num(5.0))
    least = 2.0 ** -24 if eps == 2.0 ** -11 else 0.0  # half a step below fp16's normal range
    bound = 5 * 2.0 ** -24 * size * (1 + 2.0 ** -20)
    bound = bound + eps * (out.abs() + bound) * (eps > 2.0 ** -24) + least
    assert ((got - out).abs() <= bound)[fine].all()


def inputs(rows, vocab, width, dtype, g, wide):
    x = (torch.randn((rows, vocab), generator=g, device="cuda") * 4).to(dtype)
    history = torch.randint(-3, vocab + 3, (rows, width), generator=g, device="cuda")
    if width:
        history[:, ::3] = torch.randint(0, min(vocab, 7), history[:, ::3].shape, generator=g, device="cuda")
    lengths = torch.randint(0, width + 1, (rows,), generator=g, device="cuda").int()
    return x, history if wide else history.int(), lengths


def knobs(rows, g):
    return [torch.rand((rows,), generator=g, device="cuda") + s for s in (0.9, -0.2, 0.0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("rows,vocab,width", [(1, 1, 0), (1, 33, 1), (2, 500, 40), (3, 8191, 1000), (2, 8192, 9), (1, 8193, 100),
                                              (5, 20000, 3000), (2, 50001, 700), (130, 1000, 50), (1, 262147, 20000)])
def test_everything(device, rows, vocab, width, wide, dtype):
    g = torch.Generator(device=device).manual_seed(rows + vocab)
    x, history, lengths = inputs(rows, vocab, width, dtype, g, wide)
    prompts = torch.randint(-1, width + 2, (rows,), generator=g, device=device).int()
    r, f, p = knobs(rows, g)
    bias = torch.randn((rows, vocab), generator=g, device=device)
    bias[:, ::5] = -math.inf
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g, device=device).int()
    mask[-1] = 0 if rows > 1 else mask[-1]  # nothing is left of this row
    out = torch.empty_like(x)
    kernels.process_logits(x, out, history, lengths, prompts, r, f, p, bias, mask)
    want, size = reference(x, history, lengths, prompts, r, f, p, bias, mask)
    check(out, want, size)
    kernels.process_logits(x, x, history, lengths, prompts, r, f, p, bias, mask)
    assert torch.equal(x, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", range(6))
def test_each_alone(device, which, dtype):
    g = torch.Generator(device=device).manual_seed(which)
    rows, vocab, width = 3, 9001, 300
    x, history, lengths = inputs(rows, vocab, width, dtype, g, False)
    r, f, p = knobs(rows, g)
    args = [None] * 6
    choices = (lengths // 2, r, f, p, torch.randn((vocab,), generator=g, device=device),
               torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g, device=device).int())
    args[which] = choices[which]
    out = torch.empty_like(x)
    kernels.process_logits(x, out, history, lengths, *args)
    check(out, *reference(x, history, lengths, *args))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_any_offset(device, dtype):
    """Rows that begin nowhere near 16 bytes, logits and results alike or not."""
    g = torch.Generator(device=device).manual_seed(3)
    rows, vocab, width = 4, 8203, 500
    _, history, lengths = inputs(rows, vocab, width, dtype, g, False)
    r, f, p = knobs(rows, g)
    for at, step, to, to_step in ((1, 9001, 1, 9001), (3, 9001, 5, 9001), (0, 8208, 0, 9008), (7, 8203, 0, 8208)):
        base, out = (torch.full((rows * 9008 + 16,), 7.0, device=device).to(dtype) for _ in range(2))
        x = base.as_strided((rows, vocab), (step, 1), at)
        x.copy_((torch.randn((rows, vocab), generator=g, device=device) * 4).to(dtype))
        y = out.as_strided((rows, vocab), (to_step, 1), to)
        before = base.clone()
        bias = torch.randn((rows, vocab + 1), generator=g, device=device)[:, 1:]
        mask = torch.randint(-2 ** 31, 2 ** 31, (rows, 300), generator=g, device=device).int()[:, 5:5 + -(-vocab // 32)]
        kernels.process_logits(x, y, history, lengths, None, r, f, p, bias, mask)
        check(y, *reference(x, history, lengths, None, r, f, p, bias, mask))
        inside = torch.zeros(out.shape, dtype=torch.bool, device=device)
        inside.as_strided((rows, vocab), (to_step, 1), to).fill_(True)
        assert (out[~inside] == 7.0).all() and torch.equal(base, before)


def test_special_values(device):
    g = torch.Generator(device=device).manual_seed(4)
    x, history, _ = inputs(4, 300, 50, torch.float32, g, False)
    lengths = torch.tensor([50, -1, 51, 0], dtype=torch.int32, device=device)
    x[0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 0.0])
    mask = torch.full((4, 10), -1, dtype=torch.int32, device=device)
    mask[0, 0] = ~0b100  # the NaN
    mask[2] = 0
    out = torch.empty_like(x)
    kernels.process_logits(x, out, history, lengths, repetition=torch.full((4,), 2.0, device=device), mask=mask)
    assert out[0, 0] == math.inf and out[0, 1] == -math.inf and out[0, 2] == -math.inf and out[0, 3] == 0
    assert out[1].isnan().all() and (out[2] == -math.inf).all() and torch.equal(out[3], x[3])
    # one token in all of a long history: its count is exact
    history = torch.full((1, 300000), 5, dtype=torch.int32, device=device)
    x = torch.zeros((1, 8), device=device)
    out = torch.empty_like(x)
    kernels.process_logits(x, out, history, torch.tensor([300000], dtype=torch.int32, device=device),
                           frequency=torch.full((1,), 0.5, device=device))
    assert out[0, 5] == -150000.0 and not out[0, :5].any()


def test_another_stream_and_a_captured_step(device):
    g = torch.Generator(device=device).manual_seed(5)
    x, history, lengths = inputs(3, 1000, 64, torch.float32, g, True)
    f = torch.full((3,), 0.5, device=device)
    out, want = torch.empty_like(x), torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.process_logits(x, out, history, lengths, frequency=f)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=g, device=device))
        lengths.fill_(i * 16)
        graph.replay()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        kernels.process_logits(x, want, history, lengths, frequency=f, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    kernels.process_logits(x[:0], out[:0], history[:0], lengths[:0])
