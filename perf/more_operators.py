"""What a serving step does around the model's products, as measurable cases.

Four operators: attention over a cache held in 8 bits, the append that quantises new keys and
values into such a cache (with the read that gives them back), the copying, forking and compacting
of a cache's pages, and the processing of logits before a token is chosen.  Each has a plain form in
elementary torch operations (``own`` false) and the calls a user makes of ``pyasc_amd.kernels``
(``own`` true).  ``listed()`` names the cases, ``draw()`` gives more of the same ranges, ``exact()``
is the definition in 64 bits."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8,
          "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
LARGEST = {"int8": 127.0, "e4m3": 448.0}
LEAST_EXPONENT = -126   # of a block's scale
MAX_FLOPS = 5e11        # of a drawn attention call
MAX_SCORES = 1 << 30    # elements of its whole score array
MAX_CACHE = 1 << 29     # elements of a drawn cache's keys and values
MAX_LOGITS = 1 << 25    # elements of a drawn call's logits


def listed():
    return [
        # one token of a short sequence, small pages: the smallest call, where latency counts
        {"name": "attend_token_500", "op": "attend", "dtype": "f16", "cache": "int8", "b": 1, "hq": 16, "hk": 4,
         "n": 1, "len": 500, "page": 16, "block": 16, "d": 64, "ragged": False},
        # decode far into long contexts, large pages of several blocks
        {"name": "attend_token_32768", "op": "attend", "dtype": "bf16", "cache": "e4m3", "b": 8, "hq": 32, "hk": 8,
         "n": 1, "len": 32768, "page": 256, "block": 64, "d": 128, "ragged": True},
        # decode of a full batch, a scale for each small block
        {"name": "attend_batch_4096", "op": "attend", "dtype": "bf16", "cache": "int8", "b": 64, "hq": 32, "hk": 8,
         "n": 1, "len": 4096, "page": 64, "block": 16, "d": 128, "ragged": True},
        # a chunk of a long prompt, behind what is in the cache already
        {"name": "attend_chunk_2048", "op": "attend", "dtype": "bf16", "cache": "e4m3", "b": 2, "hq": 32, "hk": 8,
         "n": 2048, "len": 8192, "page": 64, "block": 64, "d": 128, "ragged": False},
        # a decode step's tokens into blocks that hold rows already
        {"name": "append_token", "op": "append", "dtype": "bf16", "cache": "e4m3", "b": 64, "hk": 8, "n": 1,
         "len": 2000, "page": 64, "block": 16, "d": 128, "ragged": True},
        # ragged prompts behind a few cached tokens, pages of an uneven size
        {"name": "append_1999", "op": "append", "dtype": "f16", "cache": "int8", "b": 8, "hk": 8, "n": 1999,
         "len": 13, "page": 48, "block": 48, "d": 128, "ragged": True},
        # pages of one cache taken over into another
        {"name": "copy_2048", "op": "pages", "do": "copy", "dtype": "bf16", "hk": 8, "page": 16, "d": 128,
         "pages": 4096, "moved": 2048},
        # a beam step of few sequences
        {"name": "fork_8x4", "op": "pages", "do": "fork", "dtype": "f16", "hk": 4, "page": 16, "d": 64, "b": 8,
         "beams": 4, "len": 777, "dropped": 0.0},
        # a beam step of a full batch of long sequences, some of which have ended
        {"name": "fork_64x4", "op": "pages", "do": "fork", "dtype": "bf16", "hk": 8, "page": 64, "d": 128, "b": 64,
         "beams": 4, "len": 4096, "dropped": 0.1},
        # a cache that is two fifths full, scattered, brought to its front
        {"name": "compact_8192", "op": "pages", "do": "compact", "dtype": "bf16", "hk": 8, "page": 16, "d": 128,
         "pages": 8192, "b": 32, "full": 0.4},
        # one sequence's next token
        {"name": "logits_1", "op": "logits", "dtype": "f16", "rows": 1, "vocab": 32000, "history": 700, "bias": "none",
         "mask": False, "prompt": True, "wide": True},
        # a full batch with a grammar's masks, long histories
        {"name": "logits_64", "op": "logits", "dtype": "f32", "rows": 64, "vocab": 131072, "history": 8000,
         "bias": "shared", "mask": True, "prompt": True, "wide": False},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "pages", "pages", "logits"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    page = rng.choice([16, 16, 32, 48, 64, 80, 128, 256])
    d, hk = rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8, 8])
    if op in ("attend", "append"):
        blocks = [x for x in (16, 32, 48, 64, 128, 256) if page % x == 0] + [page]
        case = {"op": op, "dtype": dtype, "cache": rng.choice(["int8", "e4m3"]), "hk": hk, "page": page,
                "block": rng.choice(blocks), "d": d, "ragged": rng.random() < 0.6}
        if op == "append":
            while True:
                case["b"], case["len"] = _log_int(rng, 1, 64), rng.choice([0, _log_int(rng, 1, 16384)])
                case["n"] = 1 if rng.random() < 0.3 else _log_int(rng, 1, 8192)
                if 2 * case["b"] * hk * (case["len"] + case["n"]) * d <= MAX_CACHE and \
                        2 * case["b"] * hk * case["n"] * d <= 1 << 26:
                    return case
        while True:
            case["hq"] = hk * rng.choice([1, 2, 4, 4, 8, 16])
            case["b"], case["len"] = _log_int(rng, 1, 64), _log_int(rng, 1, 65536)
            case["n"] = 1 if rng.random() < 0.5 else min(case["len"], _log_int(rng, 1, 4096))
            if case["hq"] <= 64 and 2 * case["b"] * hk * case["len"] * d <= MAX_CACHE and \
                    work(case)["flops"] <= MAX_FLOPS and \
                    case["b"] * case["hq"] * case["n"] * case["len"] <= MAX_SCORES:
                return case
    if op == "logits":
        while True:
            case = {"op": op, "dtype": rng.choice(["f32", "f32", "f16", "bf16"]), "rows": _log_int(rng, 1, 256),
                    "vocab": _log_int(rng, 500, 262144), "history": _log_int(rng, 1, 32768),
                    "bias": rng.choice(["none", "shared", "rows"]), "mask": rng.random() < 0.6,
                    "prompt": rng.random() < 0.7, "wide": rng.random() < 0.5}
            if case["rows"] * case["vocab"] <= MAX_LOGITS:
                return case
    do = rng.choice(["copy", "fork", "fork", "compact"])
    case = {"op": op, "do": do, "dtype": dtype, "hk": hk, "page": page, "d": d}
    while True:
        if do == "fork":
            case["b"], case["beams"] = _log_int(rng, 1, 64), rng.choice([1, 2, 3, 4, 8])
            case["len"], case["dropped"] = _log_int(rng, 1, 16384), rng.choice([0.0, 0.1, 0.5])
        else:
            case["pages"] = _log_int(rng, 2, 16384)
            if do == "copy":
                case["moved"] = _log_int(rng, 1, case["pages"])
            else:
                case["b"], case["full"] = _log_int(rng, 1, 64), rng.choice([0.1, 0.4, 0.7, 0.95])
        pages = case["pages"] if do != "fork" else _pages_of_fork(case)
        if 2 * pages * hk * page * d <= MAX_CACHE // 2:
            return case


# ---------------------------------------------------------------------------- sizes of a case

def _lengths(case):
    """Each sequence's length: all of it, or (ragged) from the longest down to a quarter of it."""
    b, s = case["b"], case["len"]
    if not case["ragged"] or b == 1:
        return [s] * b
    return [max(min(1, s), s - (s - s // 4) * i // (b - 1)) for i in range(b)]


def _new(case):
    """New tokens of each sequence (ragged: from n down to none, where there are several)."""
    b, n = case["b"], case["n"]
    if not case["ragged"] or b == 1 or n == 1:
        news = [n] * b
    else:
        news = [n - n * i // (b - 1) for i in range(b)]
    return [min(x, y) for x, y in zip(news, _lengths(case))] if case["op"] == "attend" else news


def _width(case):
    """Pages of a sequence's table."""
    most = case["len"] + (case["n"] if case["op"] == "append" else 0)
    return max(1, -(-most // case["page"]))


def _fork_lengths(case):
    """Lengths of the sequences, beams of one group alike."""
    s, b = case["len"], case["b"]
    return [max(1, s - (s // 2) * i // b - i % 3) for i in range(b) for _ in range(case["beams"])]


def _pages_of_fork(case):
    """Pages that hold the sequences, whose beams share the full ones of their first half, and free
    ones for the copies."""
    page, total = case["page"], 0
    for n in _fork_lengths(case)[::case["beams"]]:
        held, shared = -(-n // page), n // 2 // page
        total += shared + case["beams"] * (held - shared)
    return total + case["b"] * case["beams"] + 5


def work(case):
    op = case["op"]
    if op == "logits":
        n, rows = case["rows"] * case["vocab"], case["rows"]
        size = 2 * n * BYTES[case["dtype"]] + rows * case["history"] * (8 if case["wide"] else 4)
        size += 4 * (n if case["bias"] == "rows" else case["vocab"] if case["bias"] == "shared" else 0)
        return {"bytes": size + (n // 8 if case["mask"] else 0), "flops": 4 * n}
    row = 2 * case["hk"] * case["d"] * BYTES.get(case["dtype"], 1)  # of keys and values, 16 bits
    if op == "pages":
        if case["do"] == "copy":
            return {"bytes": 2 * case["moved"] * case["page"] * row + 8 * case["moved"], "flops": 0}
        if case["do"] == "compact":
            used = _used_pages(case)
            moved = int(used * (case["pages"] - used) / case["pages"])
            return {"bytes": 2 * moved * case["page"] * row + 12 * case["pages"] + 8 * used, "flops": 0}
        rows = sum(n % case["page"] for n in _fork_lengths(case)) * (1 - case["dropped"]) / 3
        held = sum(-(-n // case["page"]) for n in _fork_lengths(case))
        return {"bytes": int(2 * rows * row) + 8 * held + 8 * _pages_of_fork(case), "flops": 0}
    news, lens, d, hk = _new(case), _lengths(case), case["d"], case["hk"]
    if op == "append":
        total = sum(news)
        return {"bytes": total * (2 * row + row) + 8 * hk * sum(-(-x // case["block"]) for x in news),
                "flops": 4 * total * 2 * hk * d}
    pairs = sum(x * (s - x) + x * (x + 1) // 2 for x, s in zip(news, lens))
    blocks = sum(-(-s // case["block"]) for s in lens)
    size = 2 * sum(lens) * hk * d + 8 * hk * blocks + 4 * sum(-(-s // case["page"]) for s in lens)
    return {"bytes": size + sum(news) * case["hq"] * (2 * d * 2 + 4), "flops": 4 * case["hq"] * pairs * d}


def _used_pages(case):
    return max(1, min(case["pages"], int(case["pages"] * case["full"])))


# ------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _codes(shape, g, kind):
    """Codes as an append leaves them: the largest of a block near the format's largest."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    if kind == "int8":
        return (x * 32).round().clamp(-127, 127).to(torch.int8)
    return (x * 110).clamp(-448, 448).to(torch.float8_e4m3fn)


def _inputs(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "logits":
        return _logits_inputs(case, g)
    dtype, hk, page, d = DTYPES[case["dtype"]], case["hk"], case["page"], case["d"]
    if op == "pages":
        return _pages_inputs(case, seed, g)
    b, width = case["b"], _width(case)
    pages, blocks = b * width + 3, page // case["block"]
    host = torch.Generator().manual_seed(int(seed))
    table = torch.randperm(pages, generator=host)[:b * width].view(b, width)
    ins = {"table": table.to(torch.int32).cuda(), "lengths": _ints(_lengths(case)), "new": _ints(_new(case))}
    for name in ("k", "v"):
        ins[name + "_cache"] = _codes((pages, hk, page, d), g, case["cache"])
        # values of about unit size, blocks up to four times apart
        scale = torch.exp2(torch.randint(-6, -3, (pages, hk, blocks), generator=g, device="cuda").float())
        ins[name + "_scales"] = scale * (1.0 if case["cache"] == "int8" else 0.25)
    if op == "attend":
        ins["q"] = _randn((b, case["hq"], case["n"], d), g, dtype)
    else:  # a projection's results, [batch, tokens, heads, head_dim], a few channels larger than the rest
        channels = 1 + 7 * (torch.rand((d,), generator=g, device="cuda") < 0.05).float()
        for name in ("k", "v"):
            x = torch.randn((b, case["n"], hk, d), generator=g, device="cuda", dtype=torch.float32)
            ins[name] = (x * channels).to(dtype).transpose(1, 2)
    return ins


def _logits_inputs(case, g):
    rows, vocab, width = case["rows"], case["vocab"], case["history"]
    u = torch.rand((rows, width), generator=g, device="cuda")
    ins = {"logits": _randn((rows, vocab), g, DTYPES[case["dtype"]], 4.0),
           # frequent tokens come often
           "history": (u ** 4 * vocab).long().clamp(max=vocab - 1).to(torch.int64 if case["wide"] else torch.int32),
           "lengths": _ints([width - width * i // (2 * rows) for i in range(rows)]), "prompts": None, "bias": None,
           "mask": None}
    if case["prompt"]:
        ins["prompts"] = ins["lengths"] // 3
    ins["repetition"] = 1 + 0.3 * torch.rand((rows,), generator=g, device="cuda")
    ins["frequency"] = 0.5 * torch.rand((rows,), generator=g, device="cuda")
    ins["presence"] = 0.5 * torch.rand((rows,), generator=g, device="cuda")
    if case["bias"] != "none":
        shape = (vocab,) if case["bias"] == "shared" else (rows, vocab)
        ins["bias"] = _randn(shape, g, torch.float32, 0.5)
        ins["bias"][..., :: 97] = -math.inf  # tokens that may not come
    if case["mask"]:
        words = -(-vocab // 32)
        two = torch.randint(-2 ** 31, 2 ** 31, (2, rows, words), generator=g, device="cuda")
        ins["mask"] = (two[0] & two[1]).to(torch.int32)  # a quarter of the tokens is allowed
        if rows >= 4:
            ins["mask"][-1] = 0
    return ins


def _pages_inputs(case, seed, g):
    """Tables, reference counts and the caches' pages."""
    dtype, hk, page, d = DTYPES[case["dtype"]], case["hk"], case["page"], case["d"]
    host, do = torch.Generator().manual_seed(int(seed)), case["do"]
    ins = {}
    if do == "copy":
        pages = case["pages"]
        ins["from"] = torch.randperm(pages, generator=host)[:case["moved"]].to(torch.int32).cuda()
        ins["to"] = torch.randperm(pages, generator=host)[:case["moved"]].to(torch.int32).cuda()
        ins["results"] = [_randn((pages, hk, page, d), g, dtype) for _ in range(2)]
    else:
        if do == "fork":
            pages, lens = _pages_of_fork(case), _fork_lengths(case)
            order, beams = torch.randperm(pages, generator=host).tolist(), case["beams"]
            rows = []
            for i in range(0, len(lens), beams):
                held, shared = -(-lens[i] // page), lens[i] // 2 // page
                common = [order.pop() for _ in range(shared)]
                rows += [common + [order.pop() for _ in range(held - shared)] for _ in range(beams)]
            # each beam goes on from one of its group's, some more than once; a few groups have ended
            group = torch.arange(len(lens)) // beams
            parents = group * beams + torch.randint(0, beams, (len(lens),), generator=host)
            ended = torch.rand(case["b"], generator=host)[group] < case["dropped"]
            ins["parents"] = parents.masked_fill(ended, -1).to(torch.int32).cuda()
        else:
            pages, used, b = case["pages"], _used_pages(case), case["b"]
            order = torch.randperm(pages, generator=host).tolist()
            held = [used // b + (i < used % b) for i in range(b)]
            rows = [[order.pop() for _ in range(n)] for n in held]
            lens = [max(0, n * page - (i % page)) for i, n in enumerate(held)]
        width = max(1, max(len(r) for r in rows))
        table = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32)
        flat = table[table >= 0].long()
        ins["table"], ins["lengths"] = table.cuda(), _ints(lens)
        ins["refcounts"] = torch.bincount(flat, minlength=pages).to(torch.int32).cuda()
    ins["caches"] = [_randn((pages, hk, page, d), g, dtype) for _ in range(2)]
    return ins


def prepare(case, seed):
    ins = _inputs(case, seed)
    state, op = {"case": case, "in": ins}, case["op"]
    if op == "attend":
        state["o"] = torch.zeros_like(ins["q"])
        state["lse"] = torch.zeros(ins["q"].shape[:3], dtype=torch.float32, device="cuda")
    elif op == "append":  # the blocks that the new tokens reach, read back from their first row on
        block = case["block"]
        state["starts"] = ins["lengths"] // block * block
        state["counts"] = ins["lengths"] - state["starts"] + ins["new"]
        shape = (case["b"], case["hk"], case["n"] + block - 1, case["d"])
        state["out"] = [torch.zeros(shape, dtype=DTYPES[case["dtype"]], device="cuda") for _ in range(2)]
    elif op == "logits":
        state["out"] = torch.empty_like(ins["logits"])
    elif case["do"] != "copy":
        state["table"] = torch.empty_like(ins["table"])
        state["refcounts"] = torch.empty_like(ins["refcounts"])
        state["other"] = torch.empty_like(ins["lengths"] if case["do"] == "fork" else ins["refcounts"])
    return state


# --------------------------------------------------------------------------------- plain forms

def _plain_attend(state):
    case, ins = state["case"], state["in"]
    b, hq, hk, n, d = (case[x] for x in ("b", "hq", "hk", "n", "d"))
    group, table = hq // hk, ins["table"].long()

    def rows(name):  # [b, hk, all keys, d] in 32 bits
        scales = ins[name + "_scales"][table].repeat_interleave(case["block"], dim=3)
        x = ins[name + "_cache"][table].float() * scales[..., None]
        return x.transpose(1, 2).reshape(b, hk, -1, d)

    k = rows("k")
    q = ins["q"].float().reshape(b, hk, group * n, d)
    scores = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    query = torch.arange(n, device="cuda")
    limit = ins["lengths"][:, None] - ins["new"][:, None] + query + 1  # keys that a query attends
    hidden = torch.arange(k.shape[2], device="cuda") >= limit[..., None]
    scores = scores.view(b, hk, group, n, -1).masked_fill_(hidden[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul((p / total).view(b, hk, group * n, -1), rows("v")).view(b, hk, group, n, d)
    behind = query >= ins["new"][:, None]
    o = o.masked_fill(behind[:, None, None, :, None], 0.0).reshape(b, hq, n, d)
    lse = (top + torch.log(total)).squeeze(-1).masked_fill(behind[:, None, None], 0.0).reshape(b, hq, n)
    return [o.to(ins["q"].dtype), lse]


def _round_codes(x, kind):
    if kind == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _plain_append(state):
    case, ins, block = state["case"], state["in"], state["case"]["block"]
    b, hk, n, d, page = (case[x] for x in ("b", "hk", "n", "d", "page"))
    blocks = -(-(n + block - 1) // block)
    at = state["starts"][:, None].long() + torch.arange(blocks * block, device="cuda")  # [b, tokens]
    old, end = ins["lengths"][:, None], (ins["lengths"] + ins["new"])[:, None]
    is_old, is_new = at < old, (at >= old) & (at < end)
    sequence = torch.arange(b, device="cuda")[:, None]
    pages = ins["table"].long()[sequence, (at // page).clamp(max=ins["table"].shape[1] - 1)]
    row, source = at % page, (at - old).clamp(0, n - 1)
    first = slice(None, None, block)
    out = []
    for name in ("k", "v"):
        cache, scales = ins[name + "_cache"], ins[name + "_scales"]
        new = ins[name].transpose(1, 2)[sequence, source].float()  # [b, tokens, hk, d]
        new = new.masked_fill(~is_new[..., None, None], 0.0).view(b, blocks, block, hk, d)
        fraction, exponent = torch.frexp(new.abs().amax((2, 4)))  # [b, blocks, hk]
        top = LARGEST[case["cache"]]
        most = math.frexp(top)
        exponent = exponent - most[1] + (fraction > most[0]).int()
        needed = torch.exp2(exponent.clamp(min=LEAST_EXPONENT).float())
        needed = torch.where(fraction == 0, 2.0 ** LEAST_EXPONENT, needed)
        held = scales[pages[:, first], :, (row // block)[:, first]]  # [b, blocks, hk]
        scale = torch.where(is_old[:, first, None], torch.maximum(held, needed), needed)
        codes = cache.view(torch.uint8)[pages, :, row].view(cache.dtype).float().view(b, blocks, block, hk, d)
        old_value = codes * held[:, :, None, :, None]
        value = torch.where(is_new.view(b, blocks, block, 1, 1), new, old_value)
        codes = _round_codes(value / scale[:, :, None, :, None], case["cache"]).view(b, -1, hk, d)
        here = is_old | is_new
        cache.view(torch.uint8)[pages[here], :, row[here]] = codes.view(torch.uint8)[here]
        touched = is_new.view(b, blocks, block).any(2)
        scales[pages[:, first][touched], :, (row // block)[:, first][touched]] = scale[touched]
        values = codes.float() * scale.repeat_interleave(block, dim=1)[..., None]
        values = values.masked_fill(~(here & (at < end))[..., None, None], 0.0)
        out.append(values[:, :n + block - 1].transpose(1, 2).to(DTYPES[case["dtype"]]))
    return out + [ins["k_scales"], ins["v_scales"]]


def _plain_logits(state):
    case, ins = state["case"], state["in"]
    rows, vocab = ins["logits"].shape
    at = torch.arange(case["history"], device="cuda")
    there = at < ins["lengths"][:, None]
    answer = there if ins["prompts"] is None else there & (at >= ins["prompts"][:, None])
    history = ins["history"].long()
    zeros = torch.zeros((rows, vocab), dtype=torch.int32, device="cuda")
    seen = zeros.scatter_add(1, history, there.int()) > 0
    count = zeros.scatter_add(1, history, answer.int()).float()
    x, r = ins["logits"].float(), ins["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - ins["frequency"][:, None] * count - ins["presence"][:, None] * (count > 0)
    if ins["bias"] is not None:
        x = x + ins["bias"]
    if ins["mask"] is not None:
        token = torch.arange(vocab, device="cuda")
        allowed = (ins["mask"][:, token >> 5] >> (token & 31)) & 1
        x = x.masked_fill(allowed == 0, float("-inf"))
    return [x.to(ins["logits"].dtype)]


def _plain_copy(state):
    ins = state["in"]
    for cache, result in zip(ins["caches"], ins["results"]):
        result[ins["to"].long()] = cache[ins["from"].long()]
    return ins["results"]


def _held(ins, page):
    """Which entries of the table hold a page."""
    return torch.arange(ins["table"].shape[1], device="cuda") * page < ins["lengths"][:, None]


def _plain_fork(state):
    case, ins, page = state["case"], state["in"], state["case"]["page"]
    held, table, pages = _held(ins, page), ins["table"].long(), ins["refcounts"].numel()
    spare = pages  # counts of no page
    refs = torch.cat((ins["refcounts"].long(), torch.zeros(1, dtype=torch.long, device="cuda")))
    refs = refs.scatter_add(0, torch.where(held, table, spare).flatten(), -torch.ones_like(table).flatten())
    parents = ins["parents"].long()
    goes_on, parent = parents >= 0, parents.clamp(min=0)
    lengths = torch.where(goes_on, ins["lengths"][parent], 0)
    index = torch.arange(parents.numel(), device="cuda")
    first = torch.full_like(index, index.numel()).scatter_reduce(0, torch.where(goes_on, parent, 0),
                                                                torch.where(goes_on, index, index.numel()), "amin")
    column = torch.arange(table.shape[1], device="cuda")
    result = torch.where(held[parent] & goes_on[:, None], table[parent], -1)
    copies = goes_on & (lengths % page > 0) & (first[parent] != index)  # in need of a page of its own
    last = (column == (lengths // page)[:, None]) & copies[:, None]
    kept = torch.where((result >= 0) & ~last, result, spare)
    refs = refs.scatter_add(0, kept.flatten(), torch.ones_like(kept).flatten())
    free = torch.nonzero(refs[:pages] == 0).flatten()
    child = torch.nonzero(copies).flatten()
    fresh, column = free[:child.numel()], (lengths // page)[child].long()
    source = result[child, column]
    result[child, column] = fresh
    refs[fresh] = 1
    used = torch.arange(page, device="cuda") < (lengths % page)[child][:, None]  # [copies, rows]
    for cache in ins["caches"]:
        cache[fresh] = torch.where(used[:, None, :, None], cache[source], cache[fresh])
    return [result.int(), lengths, refs[:pages].int()] + ins["caches"]


def _plain_compact(state):
    ins, page = state["in"], state["case"]["page"]
    refs = ins["refcounts"]
    used, index = refs > 0, torch.arange(refs.numel(), device="cuda")
    front = index < used.sum()
    source, target = index[used & ~front], index[~used & front]
    place = torch.where(used, index, -1)
    place[source] = target
    counts = refs.clone()
    counts[target] = refs[source]
    counts[source] = 0
    table = torch.where(_held(ins, page), place[ins["table"].long().clamp(min=0)], -1)
    for cache in ins["caches"]:
        cache[target] = cache[source]
    return [table.int(), counts, place.int()] + ins["caches"]


# ------------------------------------------------------------------------------------- passes

def _own(state):
    from pyasc_amd import kernels
    case, ins, op = state["case"], state["in"], state["case"]["op"]
    if op == "logits":
        kernels.process_logits(ins["logits"], state["out"], ins["history"], ins["lengths"],
                               prompt_lengths=ins["prompts"], repetition=ins["repetition"],
                               frequency=ins["frequency"], presence=ins["presence"], bias=ins["bias"],
                               mask=ins["mask"])
        return [state["out"]]
    if op == "pages":
        if case["do"] == "copy":
            kernels.cache_copy_pages(ins["caches"], ins["results"], ins["from"], ins["to"])
            return ins["results"]
        books = (ins["table"], ins["lengths"])
        if case["do"] == "fork":
            kernels.cache_fork(ins["caches"], *books, ins["parents"], ins["refcounts"], case["page"], state["table"],
                               state["other"], state["refcounts"])
            return [state["table"], state["other"], state["refcounts"]] + ins["caches"]
        kernels.cache_compact(ins["caches"], *books, ins["refcounts"], case["page"], state["table"],
                              state["refcounts"], state["other"])
        return [state["table"], state["refcounts"], state["other"]] + ins["caches"]
    cache = (ins["k_cache"], ins["v_cache"], ins["k_scales"], ins["v_scales"])
    if op == "append":
        kernels.quantized_cache_append(ins["k"], ins["v"], *cache, ins["lengths"], block_table=ins["table"],
                                       new_lengths=ins["new"])
        kernels.quantized_cache_read(*cache, state["starts"], *state["out"], block_table=ins["table"],
                                     counts=state["counts"])
        return state["out"] + [ins["k_scales"], ins["v_scales"]]
    kernels.quantized_cache_attention(ins["q"], *cache, ins["lengths"], state["o"], case["d"] ** -0.5,
                                      block_table=ins["table"], new_lengths=ins["new"], lse=state["lse"])
    return [state["o"], state["lse"]]


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["op"] == "pages":
        return {"copy": _plain_copy, "fork": _plain_fork, "compact": _plain_compact}[case["do"]](state)
    return {"attend": _plain_attend, "append": _plain_append, "logits": _plain_logits}[case["op"]](state)


# --------------------------------------------------------------------------- the definitions

def _places(case, ins, i, first, end):
    """Page and row of the tokens first .. end - 1 of sequence i."""
    at = torch.arange(first, end, device="cuda")
    return ins["table"][i].long()[at // case["page"]], at % case["page"]


def _values(case, ins, name, i, head, end):
    page, row = _places(case, ins, i, 0, end)
    codes = ins[name + "_cache"][page, head, row] if case["cache"] == "int8" else \
        ins[name + "_cache"].view(torch.uint8)[page, head, row].view(torch.float8_e4m3fn)
    return codes.float().double() * ins[name + "_scales"][page, head, row // case["block"]].double()[:, None]


def _exact_attend(case, ins):
    group, n = case["hq"] // case["hk"], case["n"]
    o = torch.zeros(ins["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(ins["q"].shape[:3], dtype=torch.float64, device="cuda")
    for i, (length, new) in enumerate(zip(_lengths(case), _new(case))):
        if new == 0:
            continue
        seen = torch.ones(new, length, dtype=torch.bool, device="cuda").tril(length - new)
        for h in range(case["hk"]):
            k, v = (_values(case, ins, name, i, h, length) for name in ("k", "v"))
            for j in range(h * group, (h + 1) * group):
                s = (ins["q"][i, j, :new].double() @ k.T / math.sqrt(case["d"])).masked_fill(~seen, -math.inf)
                lse[i, j, :new] = torch.logsumexp(s, 1)
                o[i, j, :new] = torch.softmax(s, 1) @ v
    return [o, lse]


def _to_format(x, kind):
    """float64 x rounded to the format's values, ties to the even code."""
    if kind == "int8":
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (x / step).round() * step


def _exact_append(case, ins):
    block, n, top = case["block"], case["n"], LARGEST[case["cache"]]
    result = []
    for name in ("k", "v"):
        out = torch.zeros((case["b"], case["hk"], n + block - 1, case["d"]), dtype=torch.float64, device="cuda")
        scales = ins[name + "_scales"].double()
        for i, (length, new) in enumerate(zip(_lengths(case), _new(case))):
            if new == 0:  # what is there stays, and is read back
                first = length // block * block
                for h in range(case["hk"]):
                    out[i, h, :length - first] = _values(case, ins, name, i, h, length)[first:]
                continue
            first, end = length // block * block, length + new
            fill = (first - end) % block
            x = ins[name][i, :, :new].double()  # [hk, new, d]
            before = torch.zeros((case["hk"], 0, case["d"]), dtype=torch.float64, device="cuda")
            if length > first:
                before = torch.stack([_values(case, ins, name, i, h, length)[first:] for h in range(case["hk"])])
            needs = torch.nn.functional.pad(x, (0, 0, length - first, fill)).abs()
            needs = needs.view(case["hk"], -1, block * case["d"]).amax(2)  # [hk, blocks]
            scale = torch.exp2(torch.ceil(torch.log2(needs / top)).clamp(min=LEAST_EXPONENT))
            page, row = _places(case, ins, i, first, end)
            page, row = page[::block], row[::block] // block
            if length > first:
                scale[:, 0] = torch.maximum(scale[:, 0], scales[page[0], :, row[0]])
            scales[page, :, row] = scale.T
            each = scale.repeat_interleave(block, dim=1)[:, :end - first, None]
            out[i, :, :end - first] = _to_format(torch.cat((before, x), 1) / each, case["cache"]) * each
        result.append((out, scales))
    return [result[0][0], result[1][0], result[0][1], result[1][1]]


def _exact_logits(case, ins):
    out = ins["logits"].double()
    for i, n in enumerate(ins["lengths"].tolist()):
        prompt = 0 if ins["prompts"] is None else int(ins["prompts"][i])
        tokens, count = ins["history"][i, prompt:n].unique(return_counts=True)
        seen = ins["history"][i, :n].unique()
        x, r = out[i, seen], ins["repetition"][i].double()
        out[i, seen] = torch.maximum(x, x * 0) / r + torch.minimum(x, x * 0) * r
        out[i, tokens] -= ins["frequency"][i].double() * count + ins["presence"][i].double()
    if ins["bias"] is not None:
        out = out + ins["bias"].double()
    if ins["mask"] is not None:
        bits = (ins["mask"][:, :, None] >> torch.arange(32, device="cuda")) & 1
        out[bits.flatten(1)[:, :case["vocab"]] == 0] = -math.inf
    return [out]


def exact(case, seed):
    if case["op"] == "pages":  # nothing is computed but whole numbers, and pages move as they are
        return None
    return {"attend": _exact_attend, "append": _exact_append, "logits": _exact_logits}[case["op"]](
        case, _inputs(case, seed))
