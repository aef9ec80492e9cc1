"""The attention block's operators around the framework's attention, as measurable cases.

Four operators: rotary positions, norms of queries and keys with the rotation in the same pass,
cross attention to states of another length, and attention of drafted tokens over a cache.  Each
has a plain form in elementary torch operations (``own`` false) and the calls a user makes of
``pyasc_amd.kernels`` (``own`` true).  ``listed()`` names the cases, ``draw()`` gives more of the
same ranges, ``exact()`` is the definition in 64 bits."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPSILON = 1e-6
BASE = 10000.0
TRAINED_LENGTH = 4096  # the context that scaled frequencies start from
MAX_FLOPS = 5.5e11     # of a drawn attention call
MAX_ELEMENTS = 1 << 26  # of a drawn rotation's queries and keys
MAX_CACHE = 1 << 29    # elements of a drawn call's keys and values


def listed():
    return [
        # one new token for each of eight sequences, far into a long context: the smallest call
        {"name": "rotary_token", "op": "rotary", "dtype": "bf16", "b": 8, "hq": 32, "hk": 8, "s": 1, "d": 128,
         "rot": 128, "interleaved": False, "scaling": "yarn", "factor": 32.0, "first": 100000, "backward": False,
         "fused": True},
        # a ragged prompt, half of each head rotated in interleaved pairs, positions scaled
        {"name": "rotary_part_1999", "op": "rotary", "dtype": "f16", "b": 4, "hq": 32, "hk": 32, "s": 1999, "d": 128,
         "rot": 64, "interleaved": True, "scaling": "linear", "factor": 4.0, "first": 0, "backward": False,
         "fused": False},
        # decode: queries and keys of one token per sequence, out of one projection's result
        {"name": "qk_norm_token", "op": "qk", "dtype": "bf16", "b": 16, "hq": 32, "hk": 8, "s": 1, "d": 128,
         "rot": 128, "interleaved": False, "scaling": "none", "factor": 1.0, "first": 2000, "train": False,
         "fused": True},
        # a full batch of prompts
        {"name": "qk_norm_4096", "op": "qk", "dtype": "bf16", "b": 4, "hq": 32, "hk": 8, "s": 4096, "d": 128,
         "rot": 128, "interleaved": False, "scaling": "none", "factor": 1.0, "first": 0, "train": False,
         "fused": True},
        # a training step of odd length: forward, and the gradients of inputs and weights
        {"name": "qk_norm_train_2047", "op": "qk", "dtype": "bf16", "b": 4, "hq": 32, "hk": 32, "s": 2047, "d": 64,
         "rot": 64, "interleaved": False, "scaling": "ntk", "factor": 4.0, "first": 0, "train": True, "fused": False},
        # a decoder's full context against long encoder states
        {"name": "cross_4096x2048", "op": "cross", "dtype": "bf16", "b": 4, "hq": 32, "hk": 32, "sq": 4096,
         "sk": 2048, "d": 128, "ragged": False, "train": False},
        # a padded batch of odd lengths whose last encoder sequence is empty
        {"name": "cross_ragged_777", "op": "cross", "dtype": "f16", "b": 4, "hq": 16, "hk": 16, "sq": 333,
         "sk": 777, "d": 64, "ragged": True, "train": False},
        # a training step with shared key / value heads: forward and every gradient
        {"name": "cross_train_2048x1024", "op": "cross", "dtype": "bf16", "b": 4, "hq": 32, "hk": 8, "sq": 2048,
         "sk": 1024, "d": 128, "ragged": False, "train": True},
        # decode: one token per sequence against its encoder states
        {"name": "cross_token_4096", "op": "cross", "dtype": "bf16", "b": 16, "hq": 32, "hk": 8, "sq": 1,
         "sk": 4096, "d": 128, "ragged": True, "train": False},
        # a small draft tree behind a short prompt, small pages
        {"name": "tree_16_500", "op": "tree", "dtype": "f16", "b": 1, "hq": 16, "hk": 4, "n": 16, "cache": 500,
         "page": 16, "d": 64, "ragged": False},
        # a wide draft tree for each sequence of a batch, ragged lengths
        {"name": "tree_64_4096", "op": "tree", "dtype": "bf16", "b": 8, "hq": 32, "hk": 8, "n": 64, "cache": 4096,
         "page": 64, "d": 128, "ragged": True},
        # plain decode: one token per sequence over long paged caches
        {"name": "tree_1_32768", "op": "tree", "dtype": "bf16", "b": 8, "hq": 32, "hk": 8, "n": 1, "cache": 32768,
         "page": 256, "d": 128, "ragged": True},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "qk", "qk", "cross", "cross", "cross", "tree", "tree", "tree"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op in ("rotary", "qk"):
        dtype = rng.choice(["bf16", "f16", "f32"])
        while True:
            hk, group = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 4, 8])
            case = {"op": op, "dtype": dtype, "b": _log_int(rng, 1, 32), "hq": hk * group, "hk": hk,
                    "s": _log_int(rng, 1, 8192), "d": rng.choice([64, 80, 96, 128, 128, 256])}
            if case["hq"] <= 64 and case["b"] * case["s"] * (hk * group + hk) * case["d"] <= MAX_ELEMENTS:
                break
        d = case["d"]
        case["rot"] = rng.choice([d, d, d // 2, d // 4])
        case["interleaved"] = rng.random() < 0.4
        case["scaling"] = rng.choice(["none", "linear", "ntk", "yarn"])
        case["factor"] = 1.0 if case["scaling"] == "none" else float(rng.choice([2, 4, 8, 32]))
        case["first"] = rng.choice([0, 0, _log_int(rng, 1, 120000)])
        case["fused"] = rng.random() < 0.5
        case["backward" if op == "rotary" else "train"] = rng.random() < 0.4
        return case
    if op == "cross":
        while True:
            hk, group = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 4, 8])
            case = {"op": op, "dtype": dtype, "b": _log_int(rng, 1, 16), "hq": hk * group, "hk": hk,
                    "sq": 1 if rng.random() < 0.25 else _log_int(rng, 1, 4096), "sk": _log_int(rng, 1, 8192),
                    "d": rng.choice([64, 128]), "ragged": rng.random() < 0.5, "train": rng.random() < 0.4}
            if case["hq"] <= 64 and work(case)["flops"] <= MAX_FLOPS and _scores(case) <= 1 << 30:
                return case
    while True:
        hk, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 4, 4, 8])
        case = {"op": op, "dtype": dtype, "b": _log_int(rng, 1, 32), "hq": hk * group, "hk": hk,
                "n": 1 if rng.random() < 0.25 else _log_int(rng, 1, 64), "cache": _log_int(rng, 1, 65536),
                "page": rng.choice([16, 16, 48, 64, 100, 128, 256]), "d": rng.choice([64, 128]),
                "ragged": rng.random() < 0.6}
        size = 2 * case["b"] * hk * case["cache"] * case["d"]
        if size <= MAX_CACHE and work(case)["flops"] <= MAX_FLOPS and _scores(case) <= 1 << 30:
            return case


def _scores(case):
    """Elements of the whole score array."""
    if case["op"] == "tree":
        return case["b"] * case["hq"] * case["n"] * (case["cache"] + case["n"])
    return case["b"] * case["hq"] * case["sq"] * case["sk"]


def _lengths(case):
    """Each sequence's length: all of it, or (ragged) from the longest down to a quarter of it,
    and in a batch of four or more the last one empty."""
    b, s = case["b"], case["sk"] if case["op"] == "cross" else case["cache"]
    if not case["ragged"] or b == 1:
        return [s] * b
    out = [max(1, s - (s - s // 4) * i // (b - 1)) for i in range(b)]
    if b >= 4 and case["op"] == "cross":
        out[-1] = 0
    return out


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("rotary", "qk"):
        n = case["b"] * case["s"] * (case["hq"] + case["hk"]) * case["d"]
        table = 8 * case["s"] + 4 * case["rot"] + (8 * case["d"] if case["op"] == "qk" else 0)
        if case["op"] == "rotary":
            return {"bytes": 2 * n * e + table, "flops": 3 * n * case["rot"] // case["d"]}
        if not case["train"]:
            return {"bytes": 2 * n * e + table, "flops": 7 * n}
        # inputs and the result's gradients in, results and the inputs' gradients out
        return {"bytes": 4 * n * e + 2 * table, "flops": 24 * n}
    d, hq, hk, b = case["d"], case["hq"], case["hk"], case["b"]
    total = sum(_lengths(case))
    if case["op"] == "cross":
        sq = case["sq"]
        q, kv = b * hq * sq * d * e, 2 * total * hk * d * e
        rows = 4 * b * hq * sq
        pairs = hq * sq * total
        if not case["train"]:
            return {"bytes": 2 * q + kv + rows, "flops": 4 * pairs * d}
        # q, k, v and do in; o, lse, dq, dk and dv out (two products forward, five backward)
        return {"bytes": 4 * q + 2 * kv + rows, "flops": 14 * pairs * d}
    n = case["n"]
    q, kv = b * hq * n * d * e, 2 * (total + b * n) * hk * d * e
    table = 4 * sum(-(-x // case["page"]) for x in _lengths(case)) + b * n * n
    return {"bytes": 2 * q + kv + table, "flops": 4 * hq * n * (total + b * (n + 1) // 2) * d}


# ------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(shape, g, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _heads(g, case, dtype, scale):
    """Queries and keys as [batch, heads, seq, head_dim]: views of one projection's result (values
    behind them, as in a model), or tensors of their own."""
    b, hq, hk, s, d = case["b"], case["hq"], case["hk"], case["s"], case["d"]
    if case["fused"]:
        x = _randn((b, s, hq + 2 * hk, d), g, dtype, scale)
        return x[:, :, :hq].transpose(1, 2), x[:, :, hq:hq + hk].transpose(1, 2)
    return _randn((b, hq, s, d), g, dtype, scale), _randn((b, hk, s, d), g, dtype, scale)


def _inputs(case, seed):
    g, dtype, op = _gen(seed), DTYPES[case["dtype"]], case["op"]
    b, d = case["b"], case["d"]
    if op in ("rotary", "qk"):
        # activations of a few times unit size; a prompt's positions are consecutive, and each
        # sequence starts somewhere else where it goes on from a cache
        q, k = _heads(g, case, dtype, 1.5)
        first = torch.full((b, 1), case["first"], device="cuda", dtype=torch.int64)
        if case["first"]:
            first = first + torch.randint(0, 1000, (b, 1), generator=g, device="cuda")
        ins = {"q": q, "k": k, "positions": first + torch.arange(case["s"], device="cuda")}
        if op == "qk":
            ins["q_weight"] = 1 + _randn((d,), g, torch.float32, 0.2)
            ins["k_weight"] = 1 + _randn((d,), g, torch.float32, 0.2)
            if case["train"]:
                ins["dq_out"] = _randn((b, case["hq"], case["s"], d), g, dtype)
                ins["dk_out"] = _randn((b, case["hk"], case["s"], d), g, dtype)
        return ins
    if op == "cross":
        shape, kv = (b, case["hq"], case["sq"], d), (b, case["sk"], case["hk"], d)
        # keys and values are a projection of the encoder's states: [batch, seq, heads, head_dim]
        ins = {"q": _randn(shape, g, dtype), "k": _randn(kv, g, dtype).transpose(1, 2),
               "v": _randn(kv, g, dtype).transpose(1, 2), "kv_lengths": None}
        if case["ragged"]:
            ins["kv_lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        if case["train"]:
            ins["do"] = _randn(shape, g, dtype)
        return ins
    n, hk, page = case["n"], case["hk"], case["page"]
    per_seq = -(-case["cache"] // page)
    pages = b * per_seq + 3
    kv = (pages, hk, page, d)
    host = torch.Generator().manual_seed(int(seed))
    parents = [(torch.rand(b, generator=host) * (i + 1)).long() - 1 for i in range(n)]  # -1: a root
    mask = torch.zeros(b, n, n, dtype=torch.bool)
    rows = torch.arange(b)
    for i, p in enumerate(parents):  # a token attends its ancestors and itself
        mask[:, i] = mask[rows, p.clamp(min=0)] & (p >= 0)[:, None]
        mask[:, i, i] = True
    table = torch.randperm(pages, generator=host)[:b * per_seq].view(b, per_seq)
    return {"q": _randn((b, case["hq"], n, d), g, dtype), "k_cache": _randn(kv, g, dtype),
            "v_cache": _randn(kv, g, dtype), "k_draft": _randn((b, hk, n, d), g, dtype),
            "v_draft": _randn((b, hk, n, d), g, dtype), "tree_mask": mask.cuda(),
            "block_table": table.to(torch.int32).cuda(),
            "cache_lengths": torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")}


def _frequencies(case):
    """The angle per position of each pair, and the factor on the rotated values."""
    rot, scaling, factor = case["rot"], case["scaling"], case["factor"]
    base = BASE * factor ** (rot / (rot - 2)) if scaling == "ntk" else BASE
    freqs = torch.tensor([base ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64)
    if scaling == "linear":
        freqs = freqs / factor
    if scaling == "yarn":  # pairs that turn often in the trained context keep their frequency
        turns = TRAINED_LENGTH * freqs / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        freqs = freqs * (keep + (1 - keep) / factor)
    return freqs.cuda(), 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0


def prepare(case, seed):
    state = {"case": case, "in": _inputs(case, seed)}
    ins, op = state["in"], case["op"]
    if op in ("rotary", "qk"):
        if own:
            from pyasc_amd import kernels
            state["freqs"], state["magnitude"] = kernels.rotary_frequencies(
                case["rot"], BASE, None if case["scaling"] == "none" else case["scaling"], case["factor"],
                TRAINED_LENGTH)
        else:
            state["freqs"], state["magnitude"] = _frequencies(case)
        names = ["q", "k"]
    elif op == "cross":
        names = ["q"]
        state["lse"] = torch.empty(ins["q"].shape[:3], dtype=torch.float32, device="cuda")
    else:
        names = ["q"]
    # results, contiguous: attention reads them, and a step writes the same ones every time
    state["out"] = [torch.empty(ins[n].shape, dtype=ins[n].dtype, device="cuda") for n in names]
    if case.get("train"):
        grads = ["q", "k"] if op == "qk" else ["q", "k", "v"]
        state["grads"] = [torch.empty_like(ins[n]) for n in grads]
        if op == "qk":
            state["grads"] += [torch.empty_like(ins[n]) for n in ("q_weight", "k_weight")]
    return state


# --------------------------------------------------------------------------------- plain forms

def _angles(state):
    """cos and sin [batch, 1, seq, pairs]: angles in 64 bits, where far positions keep their
    fraction of a turn."""
    angle = state["in"]["positions"].double()[:, None, :, None] * state["freqs"]
    return (torch.cos(angle) * state["magnitude"]).float(), (torch.sin(angle) * state["magnitude"]).float()


def _rotate(x, cos, sin, interleaved, backward=False):
    """float32 x with its first 2 * pairs columns rotated."""
    pairs = cos.shape[-1]
    if backward:
        sin = -sin
    part = x[..., :2 * pairs]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
    else:
        a, b = part[..., :pairs], part[..., pairs:]
    ra, rb = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((ra, rb), dim=-1).flatten(-2) if interleaved else torch.cat((ra, rb), dim=-1)
    return torch.cat((turned, x[..., 2 * pairs:]), dim=-1)


def _plain_qk(state):
    case, ins = state["case"], state["in"]
    cos, sin = _angles(state)
    outs, grads, weight_grads = [], [], []
    for n in ("q", "k"):
        x, w = ins[n].float(), ins[n + "_weight"]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON)
        outs.append(_rotate(x * r * w, cos, sin, case["interleaved"]).to(ins[n].dtype))
        if case["train"]:
            dy = _rotate(ins["d" + n + "_out"].float(), cos, sin, case["interleaved"], backward=True)
            xhat = x * r
            g = dy * w
            grads.append((r * (g - xhat * (g * xhat).mean(-1, keepdim=True))).to(ins[n].dtype))
            weight_grads.append((dy * xhat).double().sum((0, 1, 2)).float())
    return outs + grads + weight_grads


def _softmax(scores):
    """Probabilities (zeros in a row of no keys) and the logarithm of the sum of exponentials."""
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    return p / total.clamp(min=torch.finfo(torch.float32).tiny), lse


def _plain_cross(state):
    case, ins = state["case"], state["in"]
    b, hq, hk, sq, sk, d = (case[n] for n in ("b", "hq", "hk", "sq", "sk", "d"))
    scale = d ** -0.5
    q = ins["q"].float().reshape(b, hk, hq // hk * sq, d)
    k, v = ins["k"].float().contiguous(), ins["v"].float().contiguous()
    scores = torch.matmul(q, k.transpose(-1, -2)) * scale
    if case["ragged"]:
        behind = torch.arange(sk, device="cuda") >= ins["kv_lengths"][:, None]
        scores = scores.masked_fill(behind[:, None, None], float("-inf"))
    p, lse = _softmax(scores)
    o = torch.matmul(p, v)
    outs = [o.reshape(b, hq, sq, d).to(ins["q"].dtype), lse.reshape(b, hq, sq)]
    if case["train"]:
        do = ins["do"].float().reshape(b, hk, hq // hk * sq, d)
        dv = torch.matmul(p.transpose(-1, -2), do)
        dp = torch.matmul(do, v.transpose(-1, -2))
        ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
        dq = torch.matmul(ds, k).reshape(b, hq, sq, d)
        dk = torch.matmul(ds.transpose(-1, -2), q)
        outs += [x.to(ins["q"].dtype) for x in (dq, dk, dv)]
    return outs


def _plain_tree(state):
    case, ins = state["case"], state["in"]
    b, hq, hk, n, page, d = (case[x] for x in ("b", "hq", "hk", "n", "page", "d"))
    group = hq // hk
    q = ins["q"].float().reshape(b, hk, group * n, d)
    table = ins["block_table"].long()

    def rows(cache, draft):  # [b, hk, cached + n, d] in 32 bits
        cached = cache[table].transpose(1, 2).reshape(b, hk, -1, d)
        return torch.cat((cached, draft), dim=2).float()

    k, v = rows(ins["k_cache"], ins["k_draft"]), rows(ins["v_cache"], ins["v_draft"])
    width = table.shape[1] * page
    seen = torch.arange(width, device="cuda") < ins["cache_lengths"][:, None]
    seen = torch.cat((seen[:, None].expand(b, n, width), ins["tree_mask"]), dim=2)  # [b, n, cached + n]
    scores = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    scores = scores.view(b, hk, group, n, -1).masked_fill(~seen[:, None, None], float("-inf"))
    p, _ = _softmax(scores.view(b, hk, group * n, -1))
    return [torch.matmul(p, v).reshape(b, hq, n, d).to(ins["q"].dtype)]


# ------------------------------------------------------------------------------------- passes

def _own(state):
    from pyasc_amd import kernels
    case, ins, out, op = state["case"], state["in"], state["out"], state["case"]["op"]
    if op == "rotary":
        kernels.rotary(ins["q"], ins["k"], ins["positions"], state["freqs"], out[0], out[1],
                       interleaved=case["interleaved"], magnitude=state["magnitude"], backward=case["backward"])
        return out
    if op == "qk":
        weights = (ins["q_weight"], ins["k_weight"], ins["positions"], state["freqs"])
        options = {"epsilon": EPSILON, "interleaved": case["interleaved"], "magnitude": state["magnitude"]}
        kernels.qk_norm_rotary(ins["q"], ins["k"], *weights, *out, **options)
        if not case["train"]:
            return out
        kernels.qk_norm_rotary_bwd(ins["dq_out"], ins["dk_out"], ins["q"], ins["k"], *weights, *state["grads"],
                                   **options)
        return out + state["grads"]
    scale = case["d"] ** -0.5
    if op == "cross":
        args = (ins["q"], ins["k"], ins["v"], out[0])
        kernels.cross_attention_fwd(*args, scale, kv_lengths=ins["kv_lengths"], lse=state["lse"])
        if not case["train"]:
            return out + [state["lse"]]
        kernels.cross_attention_bwd(ins["do"], *args, state["lse"], *state["grads"], scale,
                                    kv_lengths=ins["kv_lengths"])
        return out + [state["lse"]] + state["grads"]
    kernels.tree_attention(ins["q"], ins["k_cache"], ins["v_cache"], ins["cache_lengths"], ins["k_draft"],
                           ins["v_draft"], ins["tree_mask"], out[0], scale, block_table=ins["block_table"])
    return out


def run(state):
    if own:
        return _own(state)
    case, op = state["case"], state["case"]["op"]
    if op == "rotary":
        cos, sin = _angles(state)
        return [_rotate(state["in"][n].float(), cos, sin, case["interleaved"], case["backward"])
                .to(DTYPES[case["dtype"]]) for n in ("q", "k")]
    return {"qk": _plain_qk, "cross": _plain_cross, "tree": _plain_tree}[op](state)


# --------------------------------------------------------------------------- the definitions

def _exact_turn(x, positions, case, sign):
    """float64 x [batch, heads, seq, head_dim] as complex pairs times magnitude * e^(i angle)."""
    freqs, magnitude = _frequencies(case)
    pairs = case["rot"] // 2
    index = torch.arange(pairs, device="cuda")
    first, second = (2 * index, 2 * index + 1) if case["interleaved"] else (index, index + pairs)
    turn = torch.polar(torch.full((), magnitude, dtype=torch.float64, device="cuda"),
                       sign * positions.double().unsqueeze(-1) * freqs)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_qk(case, ins):
    result, grads, weight_grads = [], [], []
    for n in ("q", "k"):
        x, w = ins[n].double(), ins[n + "_weight"].double()
        norm = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["d"] + EPSILON)
        result.append(_exact_turn(x / norm * w, ins["positions"], case, 1.0))
        if case["train"]:
            dy = _exact_turn(ins["d" + n + "_out"].double(), ins["positions"], case, -1.0)
            along = (dy * w * x).sum(-1, keepdim=True) / (case["d"] * norm.pow(3))
            grads.append(dy * w / norm - along * x)
            weight_grads.append((dy * x / norm).flatten(0, 2).sum(0))
    return result + grads + weight_grads


def _exact_cross(case, ins):
    b, hq, group = case["b"], case["hq"], case["hq"] // case["hk"]
    scale = case["d"] ** -0.5
    o = torch.zeros(ins["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(ins["q"].shape[:3], float("-inf"), dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(o)
    dk, dv = (torch.zeros(ins["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for i, length in enumerate(_lengths(case)):
        for h in range(hq if length else 0):
            q = ins["q"][i, h].double()
            k, v = (ins[n][i, h // group, :length].double().contiguous() for n in ("k", "v"))
            s = q @ k.T * scale
            lse[i, h] = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[i, h][:, None])
            o[i, h] = p @ v
            if case["train"]:
                do = ins["do"][i, h].double()
                dp = do @ v.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                dq[i, h] = ds @ k
                dk[i, h // group, :length] += ds.T @ q
                dv[i, h // group, :length] += p.T @ do
    return [o, lse, dq, dk, dv] if case["train"] else [o, lse]


def _exact_tree(case, ins):
    group = case["hq"] // case["hk"]
    o = torch.zeros(ins["q"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(_lengths(case)):
        at = torch.arange(length, device="cuda")
        page, row = ins["block_table"][i].long()[at // case["page"]], at % case["page"]
        hidden = torch.cat((torch.zeros(case["n"], length, dtype=torch.bool, device="cuda"), ~ins["tree_mask"][i]), 1)
        for h in range(case["hk"]):
            k = torch.cat((ins["k_cache"][page, h, row], ins["k_draft"][i, h])).double()
            v = torch.cat((ins["v_cache"][page, h, row], ins["v_draft"][i, h])).double()
            for g in range(h * group, (h + 1) * group):
                s = (ins["q"][i, g].double() @ k.T) / math.sqrt(case["d"])
                o[i, g] = torch.softmax(s.masked_fill(hidden, float("-inf")), 1) @ v
    return [o]


def exact(case, seed):
    ins, op = _inputs(case, seed), case["op"]
    if op == "rotary":
        return [_exact_turn(ins[n].double(), ins["positions"], case, -1.0 if case["backward"] else 1.0)
                for n in ("q", "k")]
    return {"qk": _exact_qk, "cross": _exact_cross, "tree": _exact_tree}[op](case, ins)
