"""Operands that the calls around a cache of 8 bits, its pages and the logits refuse before a launch, on the host's tensors: what is
not refused comes to a launch, which fails for want of a device.  test_gpu_serving_refusals.py has the same on a device's."""
import pytest
import torch

from pyasc_amd import kernels


def cache_operands(device):
    """Two sequences of up to four pages of 32 rows, two heads, blocks of 16."""
    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device=device)

    return {"k": torch.ones((2, 2, 3, 64), dtype=torch.float16, device=device), "v": torch.ones((2, 2, 3, 64), dtype=torch.float16, device=device),
            "k_cache": torch.zeros((8, 2, 32, 64), dtype=torch.int8, device=device),
            "v_cache": torch.zeros((8, 2, 32, 64), dtype=torch.int8, device=device), "k_scales": torch.ones((8, 2, 2), device=device),
            "v_scales": torch.ones((8, 2, 2), device=device), "cache_lengths": i32([5, 6]),
            "block_table": torch.arange(8, dtype=torch.int32, device=device).reshape(2, 4), "new_lengths": i32([3, 1]),
            "q": torch.ones((2, 4, 3, 64), dtype=torch.float16, device=device), "o": torch.zeros((2, 4, 3, 64), dtype=torch.float16, device=device),
            "lse": torch.zeros((2, 4, 3), device=device), "k_out": torch.zeros((2, 2, 3, 64), device=device),
            "v_out": torch.zeros((2, 2, 3, 64), device=device)}


def append(x):
    kernels.quantized_cache_append(*(x[n] for n in ("k", "v", "k_cache", "v_cache", "k_scales", "v_scales", "cache_lengths")),
                                   block_table=x["block_table"], new_lengths=x["new_lengths"])


def read(x):
    kernels.quantized_cache_read(*(x[n] for n in ("k_cache", "v_cache", "k_scales", "v_scales", "cache_lengths", "k_out", "v_out")),
                                 block_table=x["block_table"], counts=x["new_lengths"])


def attention(x, scale=0.125):
    kernels.quantized_cache_attention(*(x[n] for n in ("q", "k_cache", "v_cache", "k_scales", "v_scales", "cache_lengths", "o")),
                                      x.get("scale", scale), block_table=x["block_table"], new_lengths=x["new_lengths"], lse=x["lse"])


CALLS = {"append": append, "read": read, "attention": attention}
EVERY = tuple(CALLS)


def odd(t):
    """The same shape, 8 bytes beside 16-byte alignment."""
    flat = torch.zeros(t.numel() + 16, dtype=t.dtype, device=t.device)
    return flat[8 // t.element_size():][:t.numel()].view(t.shape)


# what is changed of the operands, the calls that refuse it, and the error
WRONG = {
    "cache type": (lambda x: {"k_cache": x["k_cache"].float()}, EVERY, TypeError),
    "other cache type": (lambda x: {"v_cache": x["v_cache"].view(torch.uint8)}, EVERY, TypeError),
    "cache of three dimensions": (lambda x: {"k_cache": x["k_cache"][0], "v_cache": x["v_cache"][0]}, EVERY, ValueError),
    "cache shapes": (lambda x: {"v_cache": x["v_cache"][:7]}, EVERY, ValueError),
    "rows that are not contiguous": (lambda x: {"k_cache": x["k_cache"].transpose(2, 3)[:, :, :64].expand(8, 2, 64, 32)}, EVERY, ValueError),
    "cache alignment": (lambda x: {"k_cache": odd(x["k_cache"])}, EVERY, ValueError),
    "head_dim": (lambda x: {"k_cache": x["k_cache"][..., :32], "v_cache": x["v_cache"][..., :32]}, EVERY, ValueError),
    "scale type": (lambda x: {"k_scales": x["k_scales"].half()}, EVERY, TypeError),
    "scale shape": (lambda x: {"k_scales": x["k_scales"][:, :1]}, EVERY, ValueError),
    "blocks of 8 rows": (lambda x: {n: torch.ones((8, 2, 4), device=x["k"].device) for n in ("k_scales", "v_scales")}, EVERY, ValueError),
    "blocks that differ": (lambda x: {"v_scales": x["v_scales"][:, :, :1]}, EVERY, ValueError),
    "lengths type": (lambda x: {"cache_lengths": x["cache_lengths"].long()}, EVERY, ValueError),
    "lengths shape": (lambda x: {"cache_lengths": x["cache_lengths"][:1]}, EVERY, ValueError),
    "new lengths shape": (lambda x: {"new_lengths": x["block_table"][:, 0]}, EVERY, ValueError),
    "table type": (lambda x: {"block_table": x["block_table"].long()}, EVERY, ValueError),
    "table rows": (lambda x: {"block_table": x["block_table"][:1]}, EVERY, ValueError),
    "no table for other pages than sequences": (lambda x: {"block_table": None}, EVERY, ValueError),
    "no tensor": (lambda x: {"cache_lengths": [5, 6]}, EVERY, TypeError),
    "type of k": (lambda x: {"k": x["k"].float(), "v": x["v"].float()}, ("append",), TypeError),
    "types of k and v": (lambda x: {"v": x["v"].bfloat16()}, ("append",), TypeError),
    "shape of v": (lambda x: {"v": x["v"][:, :, :2]}, ("append",), ValueError),
    "heads of k": (lambda x: {"k": x["k"][:, :1], "v": x["v"][:, :1]}, ("append",), ValueError),
    "alignment of k": (lambda x: {"k": odd(x["k"])}, ("append",), ValueError),
    "rows written twice": (lambda x: {"k_cache": x["k_cache"][:1].expand(8, 2, 32, 64)}, ("append",), ValueError),
    "scales written twice": (lambda x: {"v_scales": x["v_scales"][..., :1].expand(8, 2, 2)}, ("append",), ValueError),
    "one cache for both": (lambda x: {"v_cache": x["k_cache"]}, ("append",), ValueError),
    "new rows in the cache": (lambda x: {"k": x["k_cache"].view(torch.float16)[:2, :, :3].reshape(2, 2, 3, 32)}, ("append",), ValueError),
    "type of results": (lambda x: {"k_out": x["k_out"].int(), "v_out": x["v_out"].int()}, ("read",), TypeError),
    "types of results": (lambda x: {"v_out": x["v_out"].half()}, ("read",), TypeError),
    "shapes of results": (lambda x: {"v_out": x["v_out"][:, :, :2]}, ("read",), ValueError),
    "no result": (lambda x: {"k_out": None, "v_out": None}, ("read",), TypeError),
    "one result for both": (lambda x: {"v_out": x["k_out"]}, ("read",), ValueError),
    "alignment of results": (lambda x: {"v_out": odd(x["v_out"])}, ("read",), ValueError),
    "type of q": (lambda x: {"q": x["q"].float(), "o": x["o"].float()}, ("attention",), TypeError),
    "type of o": (lambda x: {"o": x["o"].bfloat16()}, ("attention",), TypeError),
    "shape of o": (lambda x: {"o": x["o"][:, :, :2]}, ("attention",), ValueError),
    "heads of q": (lambda x: {"q": x["q"][:, :3], "o": x["o"][:, :3], "lse": None}, ("attention",), ValueError),
    "head_dim of q": (lambda x: {"q": x["q"].repeat(1, 1, 1, 2), "o": x["o"].repeat(1, 1, 1, 2)}, ("attention",), ValueError),
    "alignment of q": (lambda x: {"q": odd(x["q"])}, ("attention",), ValueError),
    "shape of lse": (lambda x: {"lse": x["lse"][:, :, :2]}, ("attention",), ValueError),
    "type of lse": (lambda x: {"lse": x["lse"].half()}, ("attention",), ValueError),
    "rows of o written twice": (lambda x: {"o": x["o"][:1].expand(2, 4, 3, 64)}, ("attention",), ValueError),
    "o and q": (lambda x: {"o": x["q"]}, ("attention",), ValueError),
    "scale of zero": (lambda x: {"scale": 0.0}, ("attention",), ValueError),
    "negative scale": (lambda x: {"scale": -1.0}, ("attention",), ValueError),
    "scale of NaN": (lambda x: {"scale": float("nan")}, ("attention",), ValueError),
}


def page_operands(device):
    cache = [torch.zeros((8, 2, 32, 64), dtype=torch.int8, device=device), torch.ones((8, 2, 2), device=device)]
    table = torch.full((2, 4), -1, dtype=torch.int32, device=device)
    table[0, 0], table[1, 0] = 0, 1
    counts = torch.tensor([1, 1] + [0] * 6, dtype=torch.int32, device=device)
    pair = torch.tensor([0, 1], dtype=torch.int32, device=device)
    return {"caches": cache, "results": [t.clone() for t in cache], "from": pair, "to": pair + 4, "table": table,
            "lengths": torch.tensor([5, 6], dtype=torch.int32, device=device), "parents": torch.zeros(2, dtype=torch.int32, device=device),
            "counts": counts, "page": 32, "table_out": table.clone(), "lengths_out": torch.zeros(2, dtype=torch.int32, device=device),
            "counts_out": counts.clone(), "map": torch.zeros(8, dtype=torch.int32, device=device)}


def copy(x):
    kernels.cache_copy_pages(x["caches"], x["results"], x["from"], x["to"])


def fork(x):
    kernels.cache_fork(*(x[n] for n in ("caches", "table", "lengths", "parents", "counts", "page", "table_out", "lengths_out", "counts_out")))


def compact(x):
    kernels.cache_compact(*(x[n] for n in ("caches", "table", "lengths", "counts", "page", "table_out", "counts_out", "map")))


PAGES = {"copy": copy, "fork": fork, "compact": compact}
BOOKS = ("fork", "compact")
WRONG_PAGES = {
    "pages that differ": (lambda x: {"caches": [x["caches"][0], x["caches"][1][:7]], "results": [x["results"][0], x["results"][1][:7]]},
                          ("copy", *BOOKS), ValueError),
    "a vector for a cache": (lambda x: {"caches": [x["lengths"]], "results": [x["lengths_out"]]}, ("copy", *BOOKS), ValueError),
    "nine caches": (lambda x: {"caches": [x["caches"][0]] * 9, "results": [x["results"][0]] * 9}, ("copy", *BOOKS), ValueError),
    "a cache twice": (lambda x: {"caches": [x["caches"][0]] * 2, "results": [x["results"][0]] * 2}, ("copy", *BOOKS), ValueError),
    "pages that overlap": (lambda x: {"caches": [x["caches"][0][:1].expand(8, 2, 32, 64)]}, BOOKS, ValueError),
    "results of another type": (lambda x: {"results": [t.double() for t in x["results"]]}, ("copy",), ValueError),
    "results of another shape": (lambda x: {"results": [x["results"][0][:, :1], x["results"][1]]}, ("copy",), ValueError),
    "fewer results": (lambda x: {"results": x["results"][:1]}, ("copy",), ValueError),
    "pairs of two lengths": (lambda x: {"to": x["to"][:1]}, ("copy",), ValueError),
    "type of pairs": (lambda x: {"from": x["from"].long()}, ("copy",), ValueError),
    "pairs in the result": (lambda x: {"to": x["results"][0].view(-1)[:8].view(torch.int32)}, ("copy",), ValueError),
    "type of a table": (lambda x: {"table": x["table"].long()}, BOOKS, ValueError),
    "shape of a table": (lambda x: {"table_out": x["table_out"][:, :3]}, BOOKS, ValueError),
    "lengths of another batch": (lambda x: {"lengths": x["lengths"][:1]}, BOOKS, ValueError),
    "counts of other pages": (lambda x: {"counts": x["counts"][:7]}, BOOKS, ValueError),
    "counts out of other pages": (lambda x: {"counts_out": x["counts_out"][:7]}, BOOKS, ValueError),
    "no page size": (lambda x: {"page": 0}, BOOKS, ValueError),
    "page size that is not the rows'": (lambda x: {"page": 48}, ("fork",), ValueError),
    "type of parents": (lambda x: {"parents": x["parents"].long()}, ("fork",), ValueError),
    "lengths out of another batch": (lambda x: {"lengths_out": x["lengths_out"][:1]}, ("fork",), ValueError),
    "table out over the table": (lambda x: {"table_out": x["table"]}, ("fork",), ValueError),
    "type of the map": (lambda x: {"map": x["map"].long()}, ("compact",), ValueError),
    "map of other pages": (lambda x: {"map": x["map"][:7]}, ("compact",), ValueError),
}


def logits_operands(device):
    return {"logits": torch.zeros((2, 100), device=device), "out": torch.zeros((2, 100), device=device),
            "history": torch.zeros((2, 5), dtype=torch.int32, device=device), "lengths": torch.full((2,), 5, dtype=torch.int32, device=device),
            "prompt": torch.zeros(2, dtype=torch.int32, device=device), "repetition": torch.ones(2, device=device),
            "frequency": torch.ones(2, device=device), "presence": torch.ones(2, device=device), "bias": torch.zeros((2, 100), device=device),
            "mask": torch.full((2, 4), -1, dtype=torch.int32, device=device)}


def process(x):
    kernels.process_logits(*(x[n] for n in ("logits", "out", "history", "lengths", "prompt", "repetition", "frequency", "presence", "bias",
                                            "mask")))


WRONG_LOGITS = {
    "type": (lambda x: {"logits": x["logits"].double()}, TypeError),
    "one dimension": (lambda x: {"logits": x["logits"][0]}, ValueError),
    "type of out": (lambda x: {"out": x["out"].half()}, TypeError),
    "shape of out": (lambda x: {"out": x["out"][:, :99]}, ValueError),
    "out written twice": (lambda x: {"out": x["out"][:1].expand(2, 100)}, ValueError),
    "out over a part of the logits": (lambda x: {"out": torch.as_strided(x["logits"], (2, 100), (50, 1))}, ValueError),
    "columns apart": (lambda x: {"logits": torch.zeros((100, 2), device=x["out"].device).T}, ValueError),
    "type of history": (lambda x: {"history": x["history"].float()}, TypeError),
    "rows of history": (lambda x: {"history": x["history"][:1]}, ValueError),
    "type of lengths": (lambda x: {"lengths": x["lengths"].long()}, ValueError),
    "type of prompt lengths": (lambda x: {"prompt": x["prompt"].float()}, ValueError),
    "type of a penalty": (lambda x: {"frequency": x["frequency"].half()}, ValueError),
    "shape of a penalty": (lambda x: {"repetition": x["repetition"][:1]}, ValueError),
    "type of bias": (lambda x: {"bias": x["bias"].half()}, TypeError),
    "shape of bias": (lambda x: {"bias": x["bias"][:, :99]}, ValueError),
    "type of mask": (lambda x: {"mask": x["mask"].long()}, TypeError),
    "width of mask": (lambda x: {"mask": x["mask"][:, :3]}, ValueError),
}


@pytest.fixture
def host(monkeypatch):
    """The host's tensors taken for the current device's."""
    if torch.cuda.is_available():
        pytest.skip("a launch would follow the host's addresses")
    monkeypatch.setattr(kernels, "_current_device", lambda: -1)
    monkeypatch.setattr(kernels, "_stream", lambda stream: 0)
    monkeypatch.setattr(kernels._native, "current_stream_handle", lambda device: 0)
    return "cpu"


def refused(call, good, bad, error):
    with pytest.raises(RuntimeError, match="launch|device|HIP|hip"):
        call(good)
    with pytest.raises(error):
        call(bad)


@pytest.mark.parametrize("call,what", [(c, w) for w, (_, calls, _) in WRONG.items() for c in calls])
def test_cache_operands(host, call, what):
    change, _, error = WRONG[what]
    x = cache_operands(host)
    refused(CALLS[call], x, {**x, **change(x)}, error)


@pytest.mark.parametrize("call,what", [(c, w) for w, (_, calls, _) in WRONG_PAGES.items() for c in calls])
def test_page_operands(host, call, what):
    change, _, error = WRONG_PAGES[what]
    x = page_operands(host)
    refused(PAGES[call], x, {**x, **change(x)}, error)


@pytest.mark.parametrize("what", WRONG_LOGITS)
def test_logits_operands(host, what):
    change, error = WRONG_LOGITS[what]
    x = logits_operands(host)
    refused(process, x, {**x, **change(x)}, error)
