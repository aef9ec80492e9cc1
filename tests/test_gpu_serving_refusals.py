"""Operands that the calls around a cache of 8 bits, its pages and the logits refuse before a launch (test_serving_refusals.py has
the tables)."""
import pytest
import torch

from test_serving_refusals import (CALLS, PAGES, WRONG, WRONG_LOGITS, WRONG_PAGES, cache_operands, logits_operands, page_operands,
                                   process)

pytestmark = pytest.mark.gpu
HOST = ("k_cache", "v_scales", "cache_lengths", "block_table")


@pytest.mark.parametrize("call,what", [(c, w) for w, (_, calls, _) in WRONG.items() for c in calls])
def test_cache_operands(device, call, what):
    change, _, error = WRONG[what]
    x = cache_operands(device)
    CALLS[call](x)
    with pytest.raises(error):
        CALLS[call]({**x, **change(x)})


@pytest.mark.parametrize("call,what", [(c, w) for w, (_, calls, _) in WRONG_PAGES.items() for c in calls])
def test_page_operands(device, call, what):
    change, _, error = WRONG_PAGES[what]
    x = page_operands(device)
    with pytest.raises(error):
        PAGES[call]({**x, **change(x)})
    before = x["counts"].clone()
    PAGES[call](x)
    assert torch.equal(x["counts"], before)


@pytest.mark.parametrize("what", WRONG_LOGITS)
def test_logits_operands(device, what):
    change, error = WRONG_LOGITS[what]
    x = logits_operands(device)
    process(x)
    with pytest.raises(error):
        process({**x, **change(x)})


@pytest.mark.parametrize("what", HOST)
@pytest.mark.parametrize("call", CALLS)
def test_operands_on_the_host(device, call, what):
    x = cache_operands(device)
    with pytest.raises(ValueError):
        CALLS[call]({**x, what: x[what].cpu()})
    y = page_operands(device)
    with pytest.raises(ValueError):
        PAGES["copy"]({**y, "caches": [t.cpu() for t in y["caches"]]})
    z = logits_operands(device)
    with pytest.raises(ValueError):
        process({**z, "presence": z["presence"].cpu()})
