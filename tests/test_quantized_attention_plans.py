"""Which kernel the attention over a cache in 8 bits launches, and whether its keys are split, without a GPU.  LAUNCHES names
shapes of every kind; the GPU tests run these very shapes, so that a new rule of choice cannot leave one of them untested."""
import ctypes

import pytest

from pyasc_amd import _native

AT, FAR = 1 << 20, 1 << 36  # addresses that are never followed


def launch_of(batch, q_heads, kv_heads, n, width, page, head_dim, cache_dtype=_native.DT_INT8, dtype=_native.DT_BFLOAT16):
    """The kernel, the blocks of rows of a key / value head, and the splits of the keys, for tables of `width` pages."""
    a = _native.Cache8Args()
    a.dtype, a.cache_dtype, a.head_dim, a.page_size, a.scale_block = dtype, cache_dtype, head_dim, page, 16
    a.causal, a.sm_scale = 1, 0.125
    a.batch, a.q_heads, a.kv_heads, a.n, a.kv_len, a.num_pages = batch, q_heads, kv_heads, n, width * page, 100
    row = _native.Rows(AT, kv_heads * page * head_dim, page * head_dim, head_dim)
    scale = _native.Rows(AT, kv_heads * page // 16, page // 16, 1)
    a.k, a.v, a.k_scales, a.v_scales = row, row, scale, scale
    a.q = _native.Rows(AT, q_heads * n * head_dim, n * head_dim, head_dim)
    a.o = _native.Rows(AT + FAR, q_heads * n * head_dim, n * head_dim, head_dim)
    a.lengths, a.block_table, a.table_stride = AT, AT, width
    plan = _native.AttentionPlan()
    code = _native.load_library().asc_quantized_cache_attention_plan(ctypes.byref(a), ctypes.byref(plan))
    assert code == 0, _native.last_error()
    return plan.kernel.decode(), plan.row_blocks, plan.splits


# name: (batch, query heads, key / value heads, queries, pages of a sequence, rows of a page, head_dim), the kernel, and
# whether the keys are split
LAUNCHES = {
    "token_64": ((3, 6, 3, 1, 5, 64, 64), "cache8_narrow", False),
    "token_128": ((3, 6, 3, 1, 5, 64, 128), "cache8_narrow", False),
    "token_split_64": ((3, 4, 2, 1, 63, 48, 64), "cache8_narrow", True),
    "token_split_128": ((3, 4, 2, 1, 63, 48, 128), "cache8_narrow", True),
    "rows_64": ((7, 6, 3, 40, 10, 48, 64), "cache8_narrow", False),
    "rows_128": ((7, 6, 3, 40, 10, 48, 128), "cache8_narrow", False),
    "rows_split_64": ((3, 4, 2, 29, 50, 64, 64), "cache8_narrow", True),
    "rows_split_128": ((3, 4, 2, 29, 50, 64, 128), "cache8_narrow", True),
    "wide_64": ((12, 16, 8, 260, 28, 48, 64), "cache8_wide", False),
    "wide_128": ((12, 14, 7, 260, 28, 48, 128), "cache8_wide", False),
    "wide_split_64": ((2, 4, 2, 523, 150, 64, 64), "cache8_wide", True),
    "wide_split_128": ((2, 4, 2, 523, 150, 64, 128), "cache8_wide", True),
}


@pytest.mark.parametrize("cache_dtype", [_native.DT_INT8, _native.DT_FLOAT8_E4M3])
@pytest.mark.parametrize("dtype", [_native.DT_BFLOAT16, _native.DT_FLOAT16])
@pytest.mark.parametrize("name", LAUNCHES)
def test_launches(name, dtype, cache_dtype):
    shape, kernel, split = LAUNCHES[name]
    got, row_blocks, splits = launch_of(*shape, cache_dtype, dtype)
    rows = shape[1] // shape[2] * shape[3]
    per_block = 32 if kernel == "cache8_narrow" else 2 * shape[6]
    assert got == kernel and row_blocks == -(-rows // per_block) and (splits > 1) == split


def test_splits_have_work_and_an_end():
    """No split without two tiles of its own, and none more where heads and rows fill the card."""
    for width in (1, 2, 3, 4, 7, 1000, 1 << 15):
        for batch in (1, 5, 64, 1000):
            for n in (1, 33, 700):
                kernel, row_blocks, splits = launch_of(batch, 32, 8, n, width, 64, 128)
                assert 1 <= splits <= max(1, min(64, width // 2))
                if batch * 8 * row_blocks >= 8 * 256:
                    assert splits == 1
