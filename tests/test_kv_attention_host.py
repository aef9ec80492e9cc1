"""Attention over other keys than the queries' own without a GPU: what the C entries refuse before a
launch, their workspaces, and the structs that the typed calls pack."""
import ctypes

import pytest

from pyasc_amd import _native, kernels

ENTRIES = ("asc_cross_attention_fwd", "asc_cross_attention_bwd", "asc_tree_attention")
AT = 1 << 20  # an address that is never followed


def test_packed_structs_have_the_declared_layout():
    assert kernels._ATTENTION.size == ctypes.sizeof(_native.AttentionArgs)
    assert kernels._ROTARY.size == ctypes.sizeof(_native.RotaryArgs)
    a = _native.AttentionArgs.from_buffer_copy(kernels._ATTENTION.pack(
        1, 64, 0.5, 16, *range(1, 7), *(v for i in range(6) for v in (i, 10 * i, 100 * i, 1000 * i)), 11, 12, 13, 14,
        15, 16, 17, 18, *(v for i in range(6, 10) for v in (i, 10 * i, 100 * i, 1000 * i))))
    assert (a.dtype, a.head_dim, a.sm_scale, a.page_size) == (1, 64, 0.5, 16)
    assert (a.batch, a.q_heads, a.kv_heads, a.q_len, a.kv_len, a.num_pages) == (1, 2, 3, 4, 5, 6)
    for i, name in enumerate(("q", "o", "k", "v", "k_draft", "v_draft", "d_o", "dq", "dk", "dv")):
        r = getattr(a, name)
        assert (r.data or 0, r.batch_stride, r.head_stride, r.seq_stride) == (i, 10 * i, 100 * i, 1000 * i), name
    assert (a.lse, a.kv_lengths, a.draft_lengths, a.block_table, a.table_stride) == (11, 12, 13, 14, 15)
    assert (a.tree_mask, a.mask_batch_stride, a.mask_row_stride) == (16, 17, 18)


def _args(**kw):
    """Two sequences, eight heads on two, five queries, 300 keys."""
    a = _native.AttentionArgs()
    a.dtype, a.head_dim, a.sm_scale, a.page_size = _native.DT_BFLOAT16, 64, 0.125, 16
    a.batch, a.q_heads, a.kv_heads, a.q_len, a.kv_len, a.num_pages = 2, 8, 2, 5, 300, 40
    q, k = _native.Rows(AT, 2560, 320, 64), _native.Rows(AT, 38400, 19200, 64)
    a.q = a.o = a.d_o = a.dq = a.k_draft = a.v_draft = q
    a.k = a.v = a.dk = a.dv = k
    a.lse = AT
    for name, value in kw.items():
        setattr(a, name, value)
    return a


INVALID, UNSUPPORTED, ALIGNMENT = _native.ERR_INVALID_ARG, _native.ERR_UNSUPPORTED, _native.ERR_ALIGNMENT
COMMON = [({"dtype": 0}, UNSUPPORTED), ({"head_dim": 96}, UNSUPPORTED), ({"batch": -1}, INVALID),
          ({"q_len": -1}, INVALID), ({"kv_len": -1}, INVALID), ({"q_heads": 9}, INVALID), ({"kv_heads": 0}, INVALID),
          ({"sm_scale": 0.0}, INVALID), ({"sm_scale": float("nan")}, INVALID), ({"q": _native.Rows()}, INVALID),
          ({"o": _native.Rows()}, INVALID), ({"k": _native.Rows()}, INVALID), ({"v": _native.Rows()}, INVALID),
          ({"q": _native.Rows(AT + 8, 2560, 320, 64)}, ALIGNMENT), ({"o": _native.Rows(AT, 2560, 320, 65)}, ALIGNMENT),
          ({"k": _native.Rows(AT, 38401, 19200, 64)}, ALIGNMENT), ({"v": _native.Rows(AT + 2, 0, 0, 64)}, ALIGNMENT),
          ({"k": _native.Rows(AT, -8, 19200, 64)}, INVALID), ({"kv_len": 1 << 30}, UNSUPPORTED),
          ({"q_len": 1 << 30}, UNSUPPORTED), ({"batch": 1 << 20}, UNSUPPORTED), ({"q_len": 1 << 28}, UNSUPPORTED),
          ({"v": _native.Rows(AT, 1 << 40, 64, 64)}, UNSUPPORTED),  # more than 64 GiB
          ({"k": _native.Rows(AT, 64, 64, 1 << 62)}, UNSUPPORTED)]


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("kw,code", COMMON)
def test_refusals(entry, kw, code):
    lib = _native.load_library()
    a = _args(**kw)
    assert getattr(lib, entry)(ctypes.byref(a), AT, 1 << 40, None) == code
    assert entry in _native.last_error()
    assert getattr(lib, entry + "_workspace")(ctypes.byref(a)) == 0


@pytest.mark.parametrize("entry,kw,code", [
    ("asc_cross_attention_bwd", {"lse": None}, INVALID), ("asc_cross_attention_bwd", {"d_o": _native.Rows()}, INVALID),
    ("asc_cross_attention_bwd", {"dq": _native.Rows()}, INVALID),
    ("asc_cross_attention_bwd", {"dk": _native.Rows(AT + 4, 0, 0, 64)}, ALIGNMENT),
    ("asc_tree_attention", {"k_draft": _native.Rows()}, INVALID),
    ("asc_tree_attention", {"v_draft": _native.Rows(AT, 2560, 320, 68)}, ALIGNMENT),
    ("asc_tree_attention", {"block_table": AT, "page_size": 0}, INVALID),
    ("asc_tree_attention", {"block_table": AT, "num_pages": 0}, INVALID),
    ("asc_tree_attention", {"block_table": AT, "num_pages": 1 << 31}, INVALID),
    ("asc_tree_attention", {"block_table": AT, "table_stride": -1}, INVALID),
    ("asc_tree_attention", {"block_table": AT, "num_pages": 1 << 30}, UNSUPPORTED)])
def test_refusals_of_one_entry(entry, kw, code):
    a = _args(**kw)
    assert getattr(_native.load_library(), entry)(ctypes.byref(a), AT, 1 << 40, None) == code
    assert entry in _native.last_error()


@pytest.mark.parametrize("entry", ENTRIES)
def test_workspaces(entry):
    lib = _native.load_library()
    # few rows over many keys: they are split, and the parts need a workspace
    a = _args(kv_len=5000, k=_native.Rows(AT, 640000, 320000, 64), v=_native.Rows(AT, 640000, 320000, 64))
    need = getattr(lib, entry + "_workspace")(ctypes.byref(a))
    assert need > 0
    for ws, nbytes in ((None, need), (AT, need - 1), (AT + 4, need)):
        assert getattr(lib, entry)(ctypes.byref(a), ws, nbytes, None) == INVALID
        assert "workspace" in _native.last_error()
    assert getattr(lib, entry)(None, None, 0, None) == INVALID


def test_nothing_to_do():
    lib = _native.load_library()
    for entry in ENTRIES:
        for kw in ({"batch": 0}, {"q_len": 0, "kv_len": 0}, {"q_heads": 0, "kv_heads": 0}):
            a = _args(**kw)
            assert getattr(lib, entry + "_workspace")(ctypes.byref(a)) == 0
            assert getattr(lib, entry)(ctypes.byref(a), None, 0, None) == 0


@pytest.mark.parametrize("entry", ENTRIES)
def test_scales(entry):
    a = _args(sm_scale=float("inf"))
    assert getattr(_native.load_library(), entry)(ctypes.byref(a), AT, 1 << 40, None) == INVALID
    assert "finite" in _native.last_error()
    if entry == "asc_cross_attention_bwd":  # lse / sm_scale would not be finite
        a = _args(sm_scale=2.0 ** -101)
        assert getattr(_native.load_library(), entry)(ctypes.byref(a), AT, 1 << 40, None) == UNSUPPORTED
        assert "2^-100" in _native.last_error()
