"""The calls of a server's steps together, as they are used: prompts of several lengths into a paged cache of 8 bits, then steps of
append, attention, logits and a fork of the sequences, with a compaction on the way.  Held against the same steps in 64 bits on
caches of each sequence's own, which know no pages."""
import pytest
import torch

import cache8_reference as R
import test_gpu_logits as logits_test
from pyasc_amd import kernels
from test_gpu_quantized_attention import check

pytestmark = pytest.mark.gpu
CAPACITY = 160


class Server:
    """A paged cache and its books; pages are given to sequences here, as they grow."""

    def __init__(self, batch, hk, d, page, block, pages, dtype, device):
        self.page, self.pages, self.device = page, pages, device
        width = CAPACITY // page
        self.k = torch.zeros((pages, page, hk, d), dtype=dtype, device=device).transpose(1, 2)
        self.v = torch.zeros((pages, hk, page, d), dtype=dtype, device=device)
        self.ks, self.vs = torch.ones((2, pages, hk, page // block), device=device)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.refcounts = torch.zeros(pages, dtype=torch.int32, device=device)

    def caches(self):
        return [self.k, self.v, self.ks, self.vs]

    def grow(self, news):
        table, counts, lengths = self.table.cpu(), self.refcounts.cpu(), self.lengths.tolist()
        free = (counts == 0).nonzero().flatten().tolist()
        for b, (length, new) in enumerate(zip(lengths, news)):
            for column in range(-(-length // self.page), -(-(length + new) // self.page)):
                table[b, column] = free.pop(len(free) // 2)
                counts[table[b, column]] = 1
        self.table.copy_(table)
        self.refcounts.copy_(counts)

    def append(self, k, v, news):
        self.grow(news)
        new = torch.tensor(news, dtype=torch.int32, device=self.device)
        kernels.quantized_cache_append(k, v, *self.caches(), self.lengths, block_table=self.table, new_lengths=new)
        self.lengths += new
        return new

    def fork(self, parents):
        new = len(parents)
        table = torch.empty((new, self.table.shape[1]), dtype=torch.int32, device=self.device)
        lengths = torch.empty(new, dtype=torch.int32, device=self.device)
        kernels.cache_fork(self.caches(), self.table, self.lengths, torch.tensor(parents, dtype=torch.int32, device=self.device),
                           self.refcounts, self.page, table, lengths, self.refcounts)
        self.table, self.lengths = table, lengths

    def compact(self):
        page_map = torch.empty(self.pages, dtype=torch.int32, device=self.device)
        kernels.cache_compact(self.caches(), self.table, self.lengths, self.refcounts, self.page, self.table, self.refcounts, page_map)

    def read(self, shape):
        k, v = torch.zeros(shape, device=self.device), torch.zeros(shape, device=self.device)
        kernels.quantized_cache_read(*self.caches(), torch.zeros_like(self.lengths), k, v, block_table=self.table, counts=self.lengths)
        return k, v


class Plain:
    """The same in 64 bits: codes and scales of each sequence, one behind the other."""

    def __init__(self, batch, hk, d, block, dtype):
        self.block, self.lengths = block, [0] * batch
        empty = torch.zeros((batch, hk, CAPACITY, d)).to(dtype)
        self.parts = [(R.Codes(empty), torch.ones((batch, hk, CAPACITY // block), dtype=torch.float64)) for _ in range(2)]

    def append(self, k, v, news):
        for x, (codes, scales) in zip((k, v), self.parts):
            R.append(x.cpu(), codes, scales, self.lengths, news, R.Paged(None, CAPACITY), self.block)
        self.lengths = [a + b for a, b in zip(self.lengths, news)]

    def fork(self, parents):
        for i, (codes, scales) in enumerate(self.parts):
            codes.codes = codes.codes[parents].clone()
            self.parts[i] = (codes, scales[parents].clone())
        self.lengths = [self.lengths[p] for p in parents]

    def rows(self, i, b, h):
        codes, scales = self.parts[i]
        n = self.lengths[b]
        return codes.codes[b, h, :n], scales[b, h].repeat_interleave(self.block)[:n]


def check_cache(server, plain, hk, d):
    batch = len(plain.lengths)
    assert server.lengths.tolist() == plain.lengths
    for i, got in enumerate(server.read((batch, hk, CAPACITY, d))):
        for b in range(batch):
            for h in range(hk):
                codes, scales = plain.rows(i, b, h)
                assert torch.equal(got[b, h, :plain.lengths[b]].double().cpu(), codes * scales[:, None])
            assert not got[b, :, plain.lengths[b]:].any()


def check_books(server):
    held = torch.zeros(server.pages, dtype=torch.int32)
    for row, n in zip(server.table.tolist(), server.lengths.tolist()):
        for page in row[:-(-n // server.page)]:
            held[page] += 1
    assert torch.equal(held, server.refcounts.cpu())


@pytest.mark.parametrize("cache", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("d,page,block,dtype", [(64, 32, 16, torch.bfloat16), (128, 16, 16, torch.float16), (64, 80, 16, torch.float16)])
def test_prompts_steps_forks_and_a_compaction(device, d, page, block, dtype, cache):
    hq, hk, vocab, batch, steps = 4, 2, 333, 3, 9
    g = torch.Generator(device=device).manual_seed(d + page)
    server = Server(batch, hk, d, page, block, 70, cache, device)
    plain = Plain(batch, hk, d, block, cache)
    prompts, parents_of = [70, 1, 33], [[2, 0, 0, 1, 0], [4, 4, 2, 1], [3, 3], [0, 1, 1, 0, 0, 1]]
    news = prompts
    project = torch.randn((hq * d, vocab), generator=g, device=device) / d ** 0.5
    history = torch.randint(0, vocab, (batch, CAPACITY), generator=g, device=device)
    prompt_lengths = torch.tensor(prompts, dtype=torch.int32, device=device)
    for step in range(steps):
        batch, n = len(news), max(news)
        size = 2.0 ** (step % 4 - 2)  # later tokens need other scales
        k = (torch.randn((batch, n, hk, d), generator=g, device=device) * size).to(dtype).transpose(1, 2)
        v = (torch.randn((batch, n, hk, d), generator=g, device=device) / size).to(dtype).transpose(1, 2)
        q = torch.randn((batch, n, hq, d), generator=g, device=device).to(dtype).transpose(1, 2)
        new = server.append(k, v, news)
        plain.append(k, v, news)
        o, lse = torch.zeros_like(q), torch.zeros((batch, hq, n), device=device)
        kernels.quantized_cache_attention(q, *server.caches(), server.lengths, o, d ** -0.5, block_table=server.table, new_lengths=new,
                                          lse=lse)
        for b in range(batch):
            for h in range(hq):
                kk, vv = ([x.to(device) for x in plain.rows(i, b, h // (hq // hk))] for i in range(2))
                limits = torch.arange(news[b], device=device) + plain.lengths[b] - news[b] + 1
                check(o[b, h, :news[b]], lse[b, h, :news[b]], q[b, h, :news[b]], *kk, *vv, limits, d ** -0.5, dtype)
        # a token of each sequence's last row
        last = o.transpose(1, 2)[torch.arange(batch, device=device), new.long() - 1].reshape(batch, -1)
        x = (last.float() @ project).to(dtype)
        repetition = torch.rand(batch, generator=g, device=device) + 0.7
        frequency = torch.rand(batch, generator=g, device=device)
        mask = torch.randint(-2 ** 31, 2 ** 31, (batch, -(-vocab // 32)), generator=g, device=device).int()
        y = torch.zeros_like(x)
        kernels.process_logits(x, y, history, server.lengths, prompt_lengths, repetition, frequency, mask=mask)
        logits_test.check(y, *logits_test.reference(x, history, server.lengths, prompt_lengths, repetition, frequency, None, None, mask))
        tokens = y.argmax(1)
        check_cache(server, plain, hk, d)
        check_books(server)
        if step % 2 == 0 and parents_of:
            parents = parents_of.pop(0)
            server.fork(parents)
            plain.fork(parents)
            chosen = torch.tensor(parents, device=device)
            history, tokens, prompt_lengths = history[chosen], tokens[chosen], prompt_lengths[chosen]
            check_cache(server, plain, hk, d)
            check_books(server)
        if step % 4 == 3:
            server.compact()
            used = int((server.refcounts > 0).sum())
            assert (server.refcounts[:used] > 0).all() and not server.refcounts[used:].any()
            check_cache(server, plain, hk, d)
            check_books(server)
        history[torch.arange(len(tokens), device=device), server.lengths.long()] = tokens
        news = [1] * len(tokens) if step % 3 else [1 + (i + step) % 3 for i in range(len(tokens))]


def test_a_captured_step_goes_on_as_an_eager_one(device):
    """Append, attention and logits in a graph whose lengths grow in it, with pages that the sequences have already, beside an
    eager server's; eager calls of other shapes between the replays."""
    hq, hk, d, page, vocab, batch = 8, 2, 128, 32, 1000, 4
    g = torch.Generator(device=device).manual_seed(3)
    servers = [Server(batch, hk, d, page, 16, 30, torch.float8_e4m3fn, device) for _ in range(2)]
    history = torch.randint(0, vocab, (batch, CAPACITY), generator=g, device=device).int()
    frequency = torch.rand(batch, generator=g, device=device)
    inputs = [torch.zeros((batch, h, 1, d), dtype=torch.bfloat16, device=device) for h in (hk, hk, hq)]
    x = torch.zeros((batch, vocab), dtype=torch.bfloat16, device=device)

    def step(s, o, y):
        k, v, q = inputs
        kernels.quantized_cache_append(k, v, *s.caches(), s.lengths, block_table=s.table)
        s.lengths.add_(1)
        kernels.quantized_cache_attention(q, *s.caches(), s.lengths, o, 0.1, block_table=s.table)
        kernels.process_logits(x, y, history, s.lengths, frequency=frequency)

    for s in servers:
        s.grow([CAPACITY - 32] * batch)
    outs = [(torch.zeros_like(inputs[2]), torch.zeros_like(x)) for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(servers[0], *outs[0])
    for i in range(40):
        for t in inputs + [x]:
            t.copy_(torch.randn(t.shape, generator=g, device=device) * 2.0 ** (i % 5))
        graph.replay()
        step(servers[1], *outs[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        assert torch.equal(servers[0].lengths, servers[1].lengths)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(servers[0].caches()[1:2], servers[1].caches()[1:2]))
    assert torch.equal(servers[0].ks, servers[1].ks) and torch.equal(servers[0].vs, servers[1].vs)
