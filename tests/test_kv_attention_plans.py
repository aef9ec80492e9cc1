"""Which kernel the attention over other keys than the queries' own launches, and whether its keys are
split, without a GPU.  LAUNCHES names shapes of every kind; the GPU tests of the two kernels run these
very shapes, so that a new rule of choice cannot leave one of them untested."""
import ctypes

import pytest

from pyasc_amd import _native

AT = 1 << 20  # an address that is never followed


def launch_of(batch, q_heads, kv_heads, n, kv_len, head_dim, tree, dtype=_native.DT_BFLOAT16):
    """The kernel, the blocks of rows of a key / value head, and the splits of the keys."""
    a = _native.AttentionArgs()
    a.dtype, a.head_dim, a.sm_scale = dtype, head_dim, 0.125
    a.batch, a.q_heads, a.kv_heads, a.q_len, a.kv_len = batch, q_heads, kv_heads, n, kv_len

    def rows(heads, length):
        return _native.Rows(AT, heads * length * head_dim, length * head_dim, head_dim)

    a.q = a.o = rows(q_heads, n)
    a.k = a.v = rows(kv_heads, kv_len)
    a.k_draft = a.v_draft = rows(kv_heads, n)
    plan = _native.AttentionPlan()
    code = _native.load_library().asc_attention_plan(ctypes.byref(a), tree, ctypes.byref(plan))
    assert code == 0, _native.last_error()
    return plan.kernel.decode(), plan.row_blocks, plan.splits


# name: (batch, query heads, key / value heads, queries, keys of a sequence at most, head_dim, drafted),
# the kernel, and whether the keys are split
LAUNCHES = {
    "cross_wide_64": ((12, 16, 8, 260, 1340, 64, False), "kv_wide", False),
    "cross_wide_128": ((12, 14, 7, 260, 1340, 128, False), "kv_wide", False),
    "cross_wide_split_64": ((6, 8, 4, 277, 1340, 64, False), "kv_wide", True),
    "cross_wide_split_128": ((6, 8, 4, 277, 1340, 128, False), "kv_wide", True),
    "cross_narrow_64": ((7, 6, 3, 40, 500, 64, False), "kv_narrow", False),
    "cross_narrow_128": ((7, 6, 3, 40, 500, 128, False), "kv_narrow", False),
    "cross_narrow_split_64": ((3, 4, 2, 9, 3000, 64, False), "kv_narrow", True),
    "cross_narrow_split_128": ((3, 4, 2, 9, 3000, 128, False), "kv_narrow", True),
    "tree_wide_64": ((12, 32, 8, 130, 1340, 64, True), "kv_wide", False),
    "tree_wide_128": ((12, 28, 7, 130, 1340, 128, True), "kv_wide", False),
    "tree_wide_split_64": ((6, 8, 2, 139, 1340, 64, True), "kv_wide", True),
    "tree_wide_split_128": ((6, 8, 2, 139, 1340, 128, True), "kv_wide", True),
    "tree_narrow_64": ((7, 6, 3, 20, 400, 64, True), "kv_narrow", False),
    "tree_narrow_128": ((7, 6, 3, 20, 400, 128, True), "kv_narrow", False),
    "tree_narrow_split_64": ((3, 4, 2, 9, 3000, 64, True), "kv_narrow", True),
    "tree_narrow_split_128": ((3, 4, 2, 9, 3000, 128, True), "kv_narrow", True),
}


@pytest.mark.parametrize("dtype", [_native.DT_BFLOAT16, _native.DT_FLOAT16])
@pytest.mark.parametrize("name", LAUNCHES)
def test_launches(name, dtype):
    shape, kernel, split = LAUNCHES[name]
    got, row_blocks, splits = launch_of(*shape, dtype)
    rows = shape[1] // shape[2] * shape[3]
    per_block = 32 if kernel == "kv_narrow" else 2 * shape[5]
    assert got == kernel and row_blocks == -(-rows // per_block) and (splits > 1) == split


def test_workspace_belongs_to_the_splits():
    for shape, _, split in LAUNCHES.values():
        batch, hq, hk, n, kv_len, d, tree = shape
        a = _native.AttentionArgs()
        a.dtype, a.head_dim, a.sm_scale = _native.DT_BFLOAT16, d, 0.125
        a.batch, a.q_heads, a.kv_heads, a.q_len, a.kv_len = batch, hq, hk, n, kv_len
        a.q = a.o = a.k = a.v = a.k_draft = a.v_draft = _native.Rows(AT, 8, 8, 8)
        name = "asc_tree_attention_workspace" if tree else "asc_cross_attention_fwd_workspace"
        need = getattr(_native.load_library(), name)(ctypes.byref(a))
        units = batch * hk * launch_of(*shape)[2]
        assert need == (units * (hq // hk * n * (d + 2) + 1) * 4 if split else 0)


def test_nothing_to_launch_and_errors():
    assert launch_of(0, 4, 2, 5, 100, 64, False) == ("", 0, 0)
    assert launch_of(2, 4, 2, 0, 100, 64, True) == ("", 0, 0)
    lib, plan = _native.load_library(), _native.AttentionPlan()
    a = _native.AttentionArgs()
    assert lib.asc_attention_plan(ctypes.byref(a), 0, ctypes.byref(plan)) == _native.ERR_UNSUPPORTED
    assert "asc_attention_plan" in _native.last_error()
    assert lib.asc_attention_plan(ctypes.byref(a), 0, None) == _native.ERR_INVALID_ARG
    assert lib.asc_attention_plan(None, 0, ctypes.byref(plan)) == _native.ERR_INVALID_ARG
