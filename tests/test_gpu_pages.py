"""Copies, forks and compactions of a cache's pages against the same steps in Python: every page, table and count."""
import pytest
import torch

from pyasc_amd import kernels

pytestmark = pytest.mark.gpu


def caches_of(pages, heads, page, d, block, g):
    """Keys in bf16, values as codes of 8 bits with heads inside of rows, scales of blocks."""
    k = torch.randn((pages, heads, page, d), generator=g, device="cuda").bfloat16()
    v = torch.randint(-127, 128, (pages, page, heads, d), generator=g, device="cuda").to(torch.int8).transpose(1, 2)
    s = torch.rand((pages, heads, page // block), generator=g, device="cuda")
    return [k, v, s]


def clones(tensors):
    return [torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=t.device).copy_(t) for t in tensors]


def equal(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("pages,heads,page,d,block,pairs", [(1, 1, 16, 64, 16, 1), (9, 2, 16, 64, 16, 5), (40, 3, 48, 128, 16, 40),
                                                           (300, 8, 16, 128, 16, 299), (5, 1, 256, 128, 64, 0)])
def test_copy(device, pages, heads, page, d, block, pairs):
    g = torch.Generator(device=device).manual_seed(pages)
    source, result = caches_of(pages, heads, page, d, block, g), caches_of(pages + 3, heads, page, d, block, g)
    source.append(torch.randint(0, 99, (pages, 7), generator=g, device=device).to(torch.int16))  # odd sizes of two bytes
    result.append(torch.zeros((pages + 3, 7), dtype=torch.int16, device=device))
    source.append(torch.randint(0, 99, (pages, 3, 5), generator=g, device=device).to(torch.uint8))
    result.append(torch.zeros((pages + 3, 3, 5), dtype=torch.uint8, device=device))
    want = clones(result)
    a = torch.randperm(pages, generator=g, device=device)[:pairs].int()
    b = torch.randperm(pages + 3, generator=g, device=device)[:pairs].int()
    if pairs > 4:  # pages outside the caches: left out
        a[1], a[2], b[3], b[4] = -1, pages, pages + 3, -7
    for x, y in zip(source, want):
        for i, j in zip(a.tolist(), b.tolist()):
            if 0 <= i < pages and 0 <= j < pages + 3:
                y[j] = x[i]
    before = clones(source)
    kernels.cache_copy_pages(source, result, a, b)
    assert equal(result, want) and equal(source, before)


def test_copy_within_a_cache_and_repeated_sources(device):
    g = torch.Generator(device=device).manual_seed(1)
    cache = caches_of(30, 2, 16, 64, 16, g)
    want = clones(cache)
    a = torch.tensor([3, 3, 7, 3], dtype=torch.int32, device=device)
    b = torch.tensor([20, 21, 22, 29], dtype=torch.int32, device=device)
    for t in want:
        t[[20, 21, 22, 29]] = t[[3, 3, 7, 3]]
    kernels.cache_copy_pages(cache, cache, a, b)
    assert equal(cache, want)
    kernels.cache_copy_pages(cache[0], cache[0], a[:1], b[:1])
    kernels.cache_copy_pages([], [], a, b)
    assert equal(cache, want)


def fork(table, lengths, parents, refs, page, pages):
    """Python's fork: rows, lengths, counts, and (child's new page, parent's page, rows)."""
    table, lengths, refs, width = table.tolist(), lengths.tolist(), refs.tolist(), table.shape[1]
    held = [-(-n // page) if 0 <= n <= width * page else 0 for n in lengths]
    for row, n in zip(table, held):
        for j in range(n):
            if 0 <= row[j] < pages:
                refs[row[j]] -= 1
    rows, news, wants, taken = [], [], [], set()
    for p in parents.tolist():
        ok = 0 <= p < len(table)
        n = held[p] if ok else 0
        row = table[p][:n] if ok else []
        news.append(lengths[p] if ok else 0)
        if n and lengths[p] % page and p in taken:
            wants.append((len(rows), row[-1], lengths[p] % page))
        taken |= {p}
        rows.append(row + [-1] * (width - n))
    for i, row in enumerate(rows):
        for j, x in enumerate(row):
            if 0 <= x < pages and not any(w[0] == i and row[j + 1:j + 2] in ([], [-1]) for w in wants):
                refs[x] += 1
    copies, free = [], [i for i in range(pages) if refs[i] == 0]
    for i, source, used in wants:
        last = max(j for j, x in enumerate(rows[i]) if x != -1)
        rows[i][last] = free.pop(0) if free else -1
        if rows[i][last] >= 0:
            refs[rows[i][last]] = 1
            if 0 <= source < pages:  # nothing is read from a page outside
                copies.append((rows[i][last], source, used))
    return rows, news, refs, copies


def sequences(b, width, page, pages, g, spare, shared=0):
    """Tables of sequences whose first `shared` pages are one's, lengths and counts."""
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    common = [order.pop() for _ in range(shared)]
    lengths = torch.randint(shared * page, width * page + 1, (b,), generator=g, device="cuda").int()
    table = torch.full((b, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    for i, n in enumerate(lengths.tolist()):
        row = common + [order.pop() for _ in range(-(-n // page) - shared)]
        table[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
        refs[row] += 1
    assert len(order) >= spare
    return table.cuda(), lengths, refs.cuda()


def run_fork(caches, table, lengths, parents, refs, page, in_place=False):
    pages, new, width = refs.numel(), parents.numel(), table.shape[1]
    rows, news, want_refs, copies = fork(table, lengths, parents, refs, page, pages)
    want = clones(caches)
    for t in want:
        for to, source, used in copies:
            n = -(-used * t.shape[2] // page)
            t[to][:, :n] = t[source][:, :n]
    out = torch.full((new, width), 77, dtype=torch.int32, device="cuda")
    out_lengths = torch.full((new,), 77, dtype=torch.int32, device="cuda")
    out_refs = refs if in_place else torch.full_like(refs, 77)
    kernels.cache_fork(caches, table, lengths, parents, refs, page, out, out_lengths, out_refs)
    torch.cuda.synchronize()
    assert out.tolist() == rows and out_lengths.tolist() == news and out_refs.tolist() == want_refs
    assert equal(caches, want)
    return out, out_lengths, out_refs


@pytest.mark.parametrize("b,new,width,page,block,shared", [(1, 1, 1, 16, 16, 0), (1, 5, 3, 16, 16, 0), (4, 4, 5, 48, 16, 2),
                                                          (8, 3, 4, 64, 32, 1), (3, 8, 7, 16, 16, 3), (60, 90, 9, 32, 16, 4)])
def test_fork(device, b, new, width, page, block, shared):
    g = torch.Generator(device=device).manual_seed(b + new)
    pages = b * width + new + 3
    caches = caches_of(pages, 2, page, 64, block, g)
    table, lengths, refs = sequences(b, width, page, pages, g, new, shared)
    if b > 2:
        lengths[1] = lengths[1] // page * page  # no page is partly filled
        n = int(lengths[1]) // page
        gone = table[1, n:]
        refs[gone[gone >= 0].long()] -= 1
        table[1, n:] = -1
    for step in range(3):
        parents = torch.randint(-1, table.shape[0] + 1, (new,), generator=g, device=device).int()
        table, lengths, refs = run_fork(caches, table, lengths, parents, refs, page, in_place=step == 1)


def test_fork_without_pages_left(device):
    g = torch.Generator(device=device).manual_seed(3)
    caches = caches_of(4, 1, 16, 64, 16, g)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=device)
    lengths = torch.tensor([20], dtype=torch.int32, device=device)
    refs = torch.tensor([1, 0, 1, 0], dtype=torch.int32, device=device)
    out, _, _ = run_fork(caches, table, lengths, torch.zeros(5, dtype=torch.int32, device=device), refs, 16)
    assert out.tolist() == [[2, 0], [2, 1], [2, 3], [2, -1], [2, -1]]


def test_fork_leaves_others_pages(device):
    """Pages that holders outside the batch have stay theirs; bad lengths and pages are not followed."""
    g = torch.Generator(device=device).manual_seed(4)
    caches = caches_of(12, 1, 16, 64, 16, g)
    table = torch.tensor([[5, 6], [7, 99], [8, 9]], dtype=torch.int32, device=device)
    lengths = torch.tensor([32, 17, 33], dtype=torch.int32, device=device)  # the last: longer than its table
    refs = torch.tensor([1, 0, 0, 2, 0, 2, 1, 1, 1, 1, 0, 0], dtype=torch.int32, device=device)
    parents = torch.tensor([-1, 1, 1, 2, 0, 2 ** 31 - 1], dtype=torch.int32, device=device)
    out, lens, counts = run_fork(caches, table, lengths, parents, refs, 16)
    assert lens.tolist() == [0, 17, 17, 33, 32, 0] and out[3].tolist() == [-1, -1] and counts[8:10].tolist() == [1, 1]


def test_fork_of_many_pages(device):
    """More pages than are counted at a time, and most of the sequences that fit."""
    g = torch.Generator(device=device).manual_seed(5)
    pages, b = 40000, 1500
    caches = [torch.randint(0, 99, (pages, 1, 16), generator=g, device=device).to(torch.int16)]
    table = torch.randperm(pages, generator=g, device=device)[:b * 20].view(b, 20).int()
    lengths = torch.randint(0, 321, (b,), generator=g, device=device).int()
    held = torch.arange(20, device=device) * 16 < lengths[:, None]
    refs = torch.bincount(table[held].long(), minlength=pages).int()
    parents = torch.randint(0, b, (4096,), generator=g, device=device).int()
    want = caches[0].clone()
    out, news, counts = torch.empty((4096, 20), dtype=torch.int32, device=device), torch.empty_like(parents), refs.clone()
    kernels.cache_fork(caches, table, lengths, parents, counts, 16, out, news, counts)
    assert torch.equal(news, lengths[parents.long()])
    p = parents.long()
    parent = p.tolist()
    copies = (news % 16 != 0) & torch.tensor([parent.index(x) != i for i, x in enumerate(parent)], device=device)
    inside = torch.arange(20, device=device) * 16 < news[:, None]
    last = inside & (torch.arange(20, device=device) == (news // 16)[:, None]) & copies[:, None]
    assert torch.equal(torch.where(last, 0, out), torch.where(last, 0, torch.where(inside, table[p], -1)))
    kept = torch.bincount(out[inside & ~last].long(), minlength=pages)
    free = torch.nonzero(kept == 0).flatten()[:int(copies.sum())]
    assert torch.equal(out[last].long(), free)  # in the children's order
    kept[free] += 1
    assert torch.equal(counts.long(), kept)
    for page, source, n in zip(out[last].tolist(), table[p][last].tolist(), (news % 16)[copies].tolist()):
        want[page, :, :n] = want[source, :, :n]
    assert torch.equal(caches[0], want)


@pytest.mark.parametrize("pages,used", [(1, 1), (1, 0), (10, 4), (10, 10), (300, 100), (9000, 8000), (20000, 3000)])
def test_compact(device, pages, used):
    g = torch.Generator(device=device).manual_seed(pages)
    caches = caches_of(pages, 1, 16, 64, 16, g) if pages < 1000 else \
        [torch.randint(0, 99, (pages, 1, 3), generator=g, device=device).to(torch.int16)]
    order = torch.randperm(pages, generator=g, device=device)[:used]
    width = 7
    b = max(2, -(-used // width) + 1)
    table = torch.full((b, width), -1, dtype=torch.int32, device=device)
    table.view(-1)[:used] = order.int()
    lengths = torch.full((b,), width * 16 - 3, dtype=torch.int32, device=device)
    lengths[-1], lengths[-2] = 0, (used - (b - 2) * width) * 16
    refs = torch.zeros(pages, dtype=torch.int32, device=device)
    refs[order] = torch.randint(1, 5, (used,), generator=g, device=device).int()
    in_use = (refs > 0).cpu()
    place = torch.where(in_use, torch.arange(pages), -1)
    movers = [i for i in range(used, pages) if in_use[i]]
    holes = [i for i in range(used) if not in_use[i]]
    want, counts = clones(caches), refs.clone().cpu()
    for i, j in zip(movers, holes):
        place[i], counts[j], counts[i] = j, refs[i], 0
    for t in want:
        t[holes] = t[movers]
    column = torch.arange(width, device=device) * 16 < lengths[:, None]
    rows = torch.where(column & (table >= 0), place.cuda()[table.long().clamp(min=0)], -1).int()
    for in_place in (False, True):
        mine, got = clones(caches), torch.full((pages,), 77, dtype=torch.int32, device=device)
        t, r = table.clone(), refs.clone()
        out, out_refs = (t, r) if in_place else (torch.full_like(t, 77), torch.full_like(r, 77))
        kernels.cache_compact(mine, t, lengths, r, 16, out, out_refs, got)
        assert torch.equal(got.cpu(), place.int()) and torch.equal(out_refs.cpu(), counts) and torch.equal(out, rows)
        assert equal(mine, want)


def test_captured_steps(device):
    """Fork and compact replayed on changing sequences, beside eager calls on copies."""
    g = torch.Generator(device=device).manual_seed(6)
    b, width, page, pages = 6, 4, 16, 60
    caches = caches_of(pages, 1, page, 64, 16, g)
    plain = clones(caches)
    table, lengths, refs = sequences(b, width, page, pages, g, b)
    parents = torch.zeros(b, dtype=torch.int32, device=device)
    out, news, counts = torch.empty_like(table), torch.empty_like(lengths), torch.empty_like(refs)
    after, after_counts, place = torch.empty_like(table), torch.empty_like(refs), torch.empty_like(refs)

    def step(caches, out, news, counts, after, after_counts, place):
        kernels.cache_fork(caches, table, lengths, parents, refs, page, out, news, counts)
        kernels.cache_compact(caches, out, news, counts, page, after, after_counts, place)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches, out, news, counts, after, after_counts, place)
    for _ in range(4):
        parents.copy_(torch.randint(-1, b, (b,), generator=g, device=device))
        graph.replay()
        mine = [torch.empty_like(t) for t in (out, news, counts, after, after_counts, place)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(plain, *mine)
        torch.cuda.synchronize()
        assert equal((out, news, counts, after, after_counts, place), mine) and equal(caches, plain)
        table.copy_(after), lengths.copy_(news), refs.copy_(after_counts)


def test_nothing_to_do(device):
    none = torch.zeros(0, dtype=torch.int32, device=device)
    table = torch.zeros((0, 3), dtype=torch.int32, device=device)
    kernels.cache_fork([], table, none, none, none, 16, table.clone(), none.clone(), none.clone())
    kernels.cache_compact([], table, none, none, 16, table.clone(), none.clone(), none.clone())
    refs = torch.tensor([0, 2, 0], dtype=torch.int32, device=device)
    out, place = torch.empty_like(refs), torch.empty_like(refs)
    kernels.cache_compact([], table, none, refs, 16, table.clone(), out, place)
    assert out.tolist() == [2, 0, 0] and place.tolist() == [-1, 0, -1]
    gone = torch.zeros((2, 3), dtype=torch.int32, device=device)
    lengths = torch.tensor([16, 5], dtype=torch.int32, device=device)
    gone[1, 0] = 1
    refs = torch.tensor([1, 1, 0], dtype=torch.int32, device=device)
    kernels.cache_fork([], gone, lengths, none, refs, 16, table.clone(), none.clone(), refs)  # all of them end
    assert not refs.any()
