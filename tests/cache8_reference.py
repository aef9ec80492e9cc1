"""A cache of 8 bits in 64-bit arithmetic, for the tests of the calls around it."""
import math

import torch

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def to_codes(x, dtype):
    """The values of the codes of float64 x within the format's range, ties to even."""
    x = x.clamp(-MOST[dtype], MOST[dtype])
    if dtype == torch.int8:
        return x.nan_to_num(0.0).round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return (x / step).round() * step


def scale_for(amax, dtype):
    """The least power of two, at least 2^-126, that holds amax (a float)."""
    if amax == 0:
        return 2.0 ** -126
    e = math.ceil(math.log2(amax / MOST[dtype]))
    while amax > MOST[dtype] * 2.0 ** e:
        e += 1
    while e > -126 and amax <= MOST[dtype] * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** max(e, -126)


def values(cache):
    """The codes' own values in fp64."""
    return cache.float().double()


class Paged:
    """Where the rows of sequences lie: pages of a table, or (table None) a page per sequence."""

    def __init__(self, table, page):
        self.table, self.page = None if table is None else table.tolist(), page

    def at(self, b, key):
        return (b, key) if self.table is None else (self.table[b][key // self.page], key % self.page)


def append(x, cache, scales, lengths, news, where, block, nudge=1.0):
    """x [b, h, n, d] behind the rows of a cache (float64 code values [pages, h, rows, d]) and its scales (float64), in
    place; `lengths` and `news` are lists.  Quotients are taken times `nudge` before they are rounded."""
    raw = cache.dtype_of
    codes, s = cache.codes, scales
    for b, (length, new) in enumerate(zip(lengths, news)):
        for start in range(length // block * block, length + new, block):
            end, old = min(start + block, length + new), max(length - start, 0)
            if end <= max(start, length):
                continue
            page, row = where.at(b, start)
            for h in range(x.shape[1]):
                rows = x[b, h, start + old - length:end - length].double()
                finite = rows[rows.isfinite()]
                need = scale_for(float(finite.abs().max()) if finite.numel() else 0.0, raw)
                held = float(s[page, h, row // block]) if old else 0.0
                held = held if 0 < held < math.inf else 0.0
                scale = max(held, need)
                if scale > held and old:
                    earlier = codes[page, h, row:row + old] * held / scale * nudge
                    codes[page, h, row:row + old] = to_codes(earlier, raw)
                codes[page, h, row + old:row + end - start] = to_codes(rows / scale * nudge, raw)
                s[page, h, row // block] = scale


class Codes:
    """A cache's codes as float64 values, with their type."""

    def __init__(self, cache):
        self.codes, self.dtype_of = values(cache.cpu()), cache.dtype
