"""The serving calls without a GPU: what the C entries refuse before a launch, their workspaces, and the structs that
the typed calls pack."""
import ctypes

import pytest

from pyasc_amd import _native, kernels

AT = 1 << 20  # addresses that are never followed, 16 MiB apart
FAR = 1 << 24
INVALID, UNSUPPORTED, ALIGNMENT = _native.ERR_INVALID_ARG, _native.ERR_UNSUPPORTED, _native.ERR_ALIGNMENT
Rows = _native.Rows


def test_packed_structs_have_the_declared_layout():
    assert kernels._CACHE8.size == ctypes.sizeof(_native.Cache8Args)
    assert kernels._LOGITS.size == ctypes.sizeof(_native.LogitsArgs)
    assert kernels._PAGE_TENSOR.size == ctypes.sizeof(_native.PageTensor)
    assert kernels._PAGES_HEAD.size == _native.PagesArgs.tensors.offset
    assert kernels._PAGES_HEAD.size + len(kernels._NO_PAGES) == ctypes.sizeof(_native.PagesArgs)
    for packer, struct, size in ((kernels._CACHE8, _native.Cache8Args, 50), (kernels._LOGITS, _native.LogitsArgs, 20),
                                 (kernels._PAGES_HEAD, _native.PagesArgs, 20), (kernels._PAGE_TENSOR, _native.PageTensor, 9)):
        flat = []

        def walk(s):
            for name, kind in s._fields_:
                value = getattr(s, name)
                if isinstance(value, ctypes.Structure):
                    walk(value)
                elif not isinstance(value, ctypes.Array):
                    flat.append(value)

        walk(struct.from_buffer_copy(packer.pack(*range(1, size + 1)).ljust(ctypes.sizeof(struct), b"\0")))
        assert flat == list(range(1, size + 1)), struct


def cache8(**kw):
    """Two sequences of two heads in pages of 32 rows, blocks of 16."""
    a = _native.Cache8Args()
    a.dtype, a.cache_dtype, a.head_dim, a.page_size, a.scale_block = _native.DT_BFLOAT16, _native.DT_INT8, 64, 32, 16
    a.causal, a.sm_scale = 1, 0.125
    a.batch, a.q_heads, a.kv_heads, a.n, a.kv_len, a.num_pages = 2, 8, 2, 5, 320, 40
    a.k, a.v = Rows(AT, 4096, 2048, 64), Rows(AT + FAR, 4096, 2048, 64)
    a.k_scales, a.v_scales = Rows(AT + 2 * FAR, 4, 2, 1), Rows(AT + 3 * FAR, 4, 2, 1)
    a.q, a.o = Rows(AT + 4 * FAR, 2560, 320, 64), Rows(AT + 5 * FAR, 2560, 320, 64)
    a.k_new, a.v_new = Rows(AT + 6 * FAR, 640, 320, 64), Rows(AT + 7 * FAR, 640, 320, 64)
    a.lse, a.lengths, a.new_lengths = AT + 8 * FAR, AT + 9 * FAR, AT + 10 * FAR
    a.block_table, a.table_stride = AT + 11 * FAR, 10
    for name, value in kw.items():
        setattr(a, name, value)
    return a


CACHE = [({"cache_dtype": 0}, UNSUPPORTED), ({"dtype": 3}, UNSUPPORTED), ({"head_dim": 96}, UNSUPPORTED), ({"batch": -1}, INVALID),
         ({"n": -1}, INVALID), ({"kv_len": -1}, INVALID), ({"kv_heads": -1}, INVALID), ({"scale_block": 8}, INVALID),
         ({"scale_block": 24}, INVALID), ({"scale_block": 48}, INVALID), ({"page_size": 40}, INVALID), ({"page_size": 0}, INVALID),
         ({"num_pages": -1}, INVALID), ({"num_pages": 1 << 31}, INVALID), ({"table_stride": -1}, INVALID), ({"lengths": None}, INVALID),
         ({"k": Rows()}, INVALID), ({"v_scales": Rows()}, INVALID), ({"k": Rows(AT + 8, 4096, 2048, 64)}, ALIGNMENT),
         ({"v": Rows(AT, 4096, 2048, 72)}, ALIGNMENT), ({"k": Rows(AT, -16, 2048, 64)}, INVALID),
         ({"k_scales": Rows(AT, -1, 2, 1)}, INVALID), ({"v": Rows(AT, 1 << 38, 2048, 64)}, UNSUPPORTED),
         ({"k": Rows(AT, 64, 64, 1 << 62)}, UNSUPPORTED), ({"k_scales": Rows(AT, 1 << 32, 2, 1)}, UNSUPPORTED),
         ({"kv_len": 1 << 30}, UNSUPPORTED), ({"n": 1 << 30}, UNSUPPORTED), ({"batch": 1 << 20}, UNSUPPORTED),
         ({"block_table": None, "kv_len": 40}, INVALID)]


@pytest.mark.parametrize("entry", ["asc_quantized_cache_append", "asc_quantized_cache_read"])
@pytest.mark.parametrize("kw,code", CACHE + [({"k_new": Rows(AT + 6 * FAR + 8, 640, 320, 64)}, ALIGNMENT),
                                             ({"v_new": Rows(AT + 7 * FAR, 640, 320, 65)}, ALIGNMENT)])
def test_cache_refusals(entry, kw, code):
    a = cache8(**kw)
    assert getattr(_native.load_library(), entry)(ctypes.byref(a), None) == code
    assert entry in _native.last_error()


def test_cache_refusals_of_one_entry():
    lib = _native.load_library()
    assert lib.asc_quantized_cache_append(ctypes.byref(cache8(k_new=Rows())), None) == INVALID
    assert lib.asc_quantized_cache_append(ctypes.byref(cache8(dtype=0)), None) == UNSUPPORTED
    assert lib.asc_quantized_cache_read(ctypes.byref(cache8(k_new=Rows(), v_new=Rows())), None) == INVALID
    assert lib.asc_quantized_cache_append(ctypes.byref(cache8(n=1 << 27)), None) == UNSUPPORTED  # workgroups
    for entry in (lib.asc_quantized_cache_append, lib.asc_quantized_cache_read):
        assert entry(None, None) == INVALID
        for kw in ({"batch": 0}, {"n": 0}, {"kv_heads": 0}):
            assert entry(ctypes.byref(cache8(**kw)), None) == 0


@pytest.mark.parametrize("head_dim,most", [(64, 1 << 27), (128, 1 << 26)])
def test_blocks_whose_vectors_do_not_fit_32_bits(head_dim, most):
    """An append numbers a block's vectors of eight values: 2^28 rows of 128 codes are -2^31 of them."""
    bad = Rows(AT + 8, 640, 320, 64)
    for rows in (1 << 28, most, most - 16):
        row, scale = Rows(1 << 40, rows * head_dim, rows * head_dim, head_dim), Rows(AT, 1, 1, 1)
        a = cache8(head_dim=head_dim, block_table=None, batch=1, kv_heads=1, kv_len=rows, scale_block=rows, k=row, v=row, k_scales=scale,
                   v_scales=scale, k_new=bad, v_new=bad)  # refused all the same
        code = _native.load_library().asc_quantized_cache_append(ctypes.byref(a), None)
        assert code == (UNSUPPORTED if rows >= most else ALIGNMENT)
        assert ("scale_block" in _native.last_error()) == (rows >= most)


@pytest.mark.parametrize("entry,kw,names", [
    ("asc_quantized_cache_append", {"k_new": Rows(AT + 64, 640, 320, 64)}, "'k_new' overlaps 'k'"),
    ("asc_quantized_cache_append", {"v_new": Rows(AT + 2 * FAR, 640, 320, 64)}, "'v_new' overlaps 'k_scales'"),
    ("asc_quantized_cache_append", {"v": Rows(AT, 4096, 2048, 64)}, "'k' overlaps 'v'"),
    ("asc_quantized_cache_append", {"v_scales": Rows(AT + 2 * FAR + 8, 4, 2, 1)}, "'k_scales' overlaps 'v_scales'"),
    ("asc_quantized_cache_append", {"lengths": AT + 3 * FAR}, "'v_scales' overlaps 'lengths'"),
    ("asc_quantized_cache_append", {"block_table": AT + FAR + 4}, "'v' overlaps 'block_table'"),
    ("asc_quantized_cache_read", {"k_new": Rows(AT + 64, 640, 320, 64)}, "'k_new' overlaps 'k'"),
    ("asc_quantized_cache_read", {"v_new": Rows(AT + 6 * FAR + 128, 640, 320, 64)}, "'k_new' overlaps 'v_new'"),
    ("asc_quantized_cache_read", {"new_lengths": AT + 7 * FAR}, "'v_new' overlaps 'new_lengths'")])
def test_cache_places(entry, kw, names):
    assert getattr(_native.load_library(), entry)(ctypes.byref(cache8(**kw)), None) == INVALID
    assert names in _native.last_error()


def pages(**kw):
    a = _native.PagesArgs()
    a.n_tensors, a.page_size, a.num_pages, a.to_num_pages, a.pairs, a.batch, a.new_batch, a.width = 2, 16, 40, 40, 3, 4, 6, 5
    a.from_pages, a.to_pages, a.block_table, a.table_stride = AT, AT + FAR, AT + 2 * FAR, 5
    a.lengths, a.parents, a.refcounts, a.table_out, a.table_out_stride = AT + 3 * FAR, AT + 4 * FAR, AT + 5 * FAR, AT + 6 * FAR, 5
    a.lengths_out, a.refcounts_out, a.page_map = AT + 7 * FAR, AT + 8 * FAR, AT + 9 * FAR
    for i in range(2):
        a.tensors[i] = tensor(AT + (10 + i) * FAR)
    for name, value in kw.items():
        if name == "tensor":
            a.tensors[1] = value
        else:
            setattr(a, name, value)
    return a


def tensor(at, to=None, **kw):
    t = _native.PageTensor(at, at if to is None else to, 8192, 8192, 4, 16, 128, 2048, 128)
    for name, value in kw.items():
        setattr(t, name, value)
    return t


ENTRIES = ("asc_cache_copy_pages", "asc_cache_fork", "asc_cache_compact")


def call(entry, a, ws=AT + 20 * FAR, nbytes=1 << 30):
    lib = _native.load_library()
    args = (ctypes.byref(a) if a is not None else None,) + (() if entry == ENTRIES[0] else (ws, nbytes)) + (None,)
    return getattr(lib, entry)(*args)


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("kw,code", [({"n_tensors": 9}, INVALID), ({"n_tensors": -1}, INVALID), ({"num_pages": -1}, INVALID),
                                     ({"tensor": tensor(0)}, INVALID), ({"tensor": tensor(AT + 12 * FAR, heads=0)}, INVALID),
                                     ({"tensor": tensor(AT + 12 * FAR, row_bytes=0)}, INVALID),
                                     ({"tensor": tensor(AT + 12 * FAR, row_stride=-128)}, INVALID),
                                     ({"tensor": tensor(AT + 10 * FAR + 4096)}, INVALID)])
def test_pages_refusals(entry, kw, code):
    assert call(entry, pages(**kw)) == code and entry in _native.last_error()
    assert call(entry, None) == INVALID


@pytest.mark.parametrize("entry", ENTRIES[1:])
@pytest.mark.parametrize("kw,code", [({"page_size": 0}, INVALID), ({"num_pages": 1 << 30}, INVALID), ({"batch": -1}, INVALID),
                                     ({"width": -1}, INVALID), ({"table_stride": -1}, INVALID), ({"block_table": None}, INVALID),
                                     ({"lengths": None}, INVALID), ({"refcounts": None}, INVALID), ({"refcounts_out": None}, INVALID),
                                     ({"table_out": None}, INVALID), ({"batch": 1 << 20}, UNSUPPORTED),
                                     ({"page_size": 1 << 29, "width": 1 << 20}, UNSUPPORTED),
                                     ({"tensor": tensor(AT + 12 * FAR, AT + 13 * FAR)}, INVALID),
                                     ({"refcounts_out": AT + 5 * FAR + 4}, INVALID), ({"refcounts_out": AT + 3 * FAR}, INVALID),
                                     ({"table_out": AT + 2 * FAR + 8}, INVALID), ({"table_out": AT + 8 * FAR}, INVALID),
                                     ({"table_out": AT + 10 * FAR}, INVALID), ({"lengths": AT + 11 * FAR}, INVALID)])
def test_fork_and_compact_refusals(entry, kw, code):
    a = pages(**kw)
    assert call(entry, a) == code and entry in _native.last_error()
    assert getattr(_native.load_library(), entry + "_workspace")(ctypes.byref(a)) == 0


def test_pages_whose_heads_are_too_large():
    """A head of a page that is copied by one workgroup, of 2 GiB."""
    far = dict(heads=2, rows=1 << 16, row_bytes=1 << 15, head_stride=1 << 32, row_stride=1 << 15)
    t = _native.PageTensor(1 << 44, 1 << 45, 1 << 34, 1 << 34, 1, 1, 1, 1, 1)
    for name, value in far.items():
        setattr(t, name, value)
    assert call("asc_cache_copy_pages", pages(tensor=t)) == UNSUPPORTED and "too large" in _native.last_error()


def test_pages_whose_heads_end_next_to_2_gib():
    """A workgroup's numbers of a head's bytes and a step behind them fit 31 bits: 512 bytes less than 2^31 do, rows of odd ones."""
    for rows, row_bytes, refused in ((4, (1 << 29) - 1, True), (3, 715827713, True), (3, 715827711, False)):
        t = _native.PageTensor(1 << 44, 1 << 45, 1 << 34, 1 << 34, 2, rows, row_bytes, 1 << 33, row_bytes)
        code = call("asc_cache_copy_pages", pages(tensor=t, from_pages=None))  # refused all the same
        assert code == (UNSUPPORTED if refused else INVALID)
        assert ("too large" in _native.last_error()) == refused


def test_pages_refusals_of_one_entry():
    assert call("asc_cache_fork", pages(parents=None)) == INVALID
    assert call("asc_cache_fork", pages(lengths_out=None)) == INVALID
    assert call("asc_cache_fork", pages(batch=4097)) == UNSUPPORTED
    assert call("asc_cache_fork", pages(new_batch=4097)) == UNSUPPORTED
    assert call("asc_cache_fork", pages(lengths_out=AT + 4 * FAR)) == INVALID and "'parents'" in _native.last_error()
    assert call("asc_cache_fork", pages(table_out=AT + 2 * FAR)) == INVALID  # the rows are another order
    assert call("asc_cache_fork", pages(page_size=24)) == INVALID  # 16 rows of a page of 24
    assert call("asc_cache_compact", pages(page_map=None)) == INVALID
    assert call("asc_cache_compact", pages(page_map=AT + 5 * FAR)) == INVALID
    assert call("asc_cache_copy_pages", pages(from_pages=None)) == INVALID
    assert call("asc_cache_copy_pages", pages(pairs=-1)) == INVALID
    assert call("asc_cache_copy_pages", pages(to_pages=AT + 10 * FAR)) == INVALID
    assert call("asc_cache_copy_pages", pages(tensor=tensor(AT + 12 * FAR, AT + 10 * FAR))) == INVALID
    assert call("asc_cache_copy_pages", pages(pairs=0)) == 0 and call("asc_cache_copy_pages", pages(n_tensors=0)) == 0


@pytest.mark.parametrize("entry", ENTRIES[1:])
def test_pages_workspaces(entry):
    a = pages()
    need = getattr(_native.load_library(), entry + "_workspace")(ctypes.byref(a))
    assert need > 0
    for ws, nbytes in ((None, need), (AT, need - 1), (AT + 4, need)):
        assert call(entry, a, ws, nbytes) == INVALID and "workspace" in _native.last_error()


def logits(**kw):
    a = _native.LogitsArgs()
    a.dtype, a.history_int64, a.rows, a.vocab, a.history_width = 0, 0, 3, 1000, 50
    a.logits, a.logits_stride, a.out, a.out_stride = AT, 1000, AT + FAR, 1000
    a.history, a.history_stride, a.history_lengths, a.prompt_lengths = AT + 2 * FAR, 50, AT + 3 * FAR, AT + 4 * FAR
    a.repetition, a.frequency, a.presence = AT + 5 * FAR, AT + 6 * FAR, AT + 7 * FAR
    a.bias, a.bias_stride, a.mask, a.mask_stride = AT + 8 * FAR, 0, AT + 9 * FAR, 32
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw,code", [({"dtype": 4}, UNSUPPORTED), ({"rows": -1}, INVALID), ({"vocab": -1}, INVALID),
                                     ({"history_width": -1}, INVALID), ({"vocab": 1 << 30}, UNSUPPORTED),
                                     ({"history_width": 1 << 30}, UNSUPPORTED), ({"logits": None}, INVALID), ({"out": None}, INVALID),
                                     ({"history": None}, INVALID), ({"history_lengths": None}, INVALID),
                                     ({"logits": AT + 2}, ALIGNMENT), ({"rows": 1 << 24, "logits": 1 << 51, "out": 1 << 52}, UNSUPPORTED),
                                     ({"out": AT + 4}, INVALID), ({"out": AT, "out_stride": 1001}, INVALID),
                                     ({"out": AT + 2 * FAR}, INVALID), ({"out": AT + 3 * FAR}, INVALID),
                                     ({"out": AT + 8 * FAR + 64}, INVALID), ({"out": AT + 9 * FAR}, INVALID)])
def test_logits_refusals(kw, code):
    lib = _native.load_library()
    assert lib.asc_process_logits(ctypes.byref(logits(**kw)), None) == code
    assert "asc_process_logits" in _native.last_error()
    assert lib.asc_process_logits(None, None) == INVALID
    assert lib.asc_process_logits(ctypes.byref(logits(rows=0)), None) == 0
    assert lib.asc_process_logits(ctypes.byref(logits(vocab=0)), None) == 0


ATTENTION = "asc_quantized_cache_attention"


def attention(a, ws=AT + 20 * FAR, nbytes=1 << 40):
    return _native.load_library().asc_quantized_cache_attention(ctypes.byref(a), ws, nbytes, None)


@pytest.mark.parametrize("kw,code", CACHE + [({"q_heads": 9}, INVALID), ({"q_heads": -1}, INVALID), ({"kv_heads": 0}, INVALID),
                                             ({"sm_scale": 0.0}, INVALID), ({"sm_scale": float("inf")}, INVALID),
                                             ({"dtype": 0}, UNSUPPORTED), ({"q": Rows()}, INVALID), ({"o": Rows()}, INVALID),
                                             ({"q": Rows(AT + 4 * FAR + 8, 2560, 320, 64)}, ALIGNMENT),
                                             ({"o": Rows(AT + 5 * FAR, 2560, 320, 65)}, ALIGNMENT),
                                             ({"k": Rows(AT, 1 << 27, 1 << 27, 1 << 26)}, UNSUPPORTED),
                                             ({"n": 1 << 28}, UNSUPPORTED)])
def test_attention_refusals(kw, code):
    a = cache8(**kw)
    assert attention(a) == code and ATTENTION in _native.last_error()
    assert _native.load_library().asc_quantized_cache_attention_workspace(ctypes.byref(a)) == 0


@pytest.mark.parametrize("kw,names", [({"o": Rows(AT + 4 * FAR, 2560, 320, 64)}, "'o' overlaps 'q'"),
                                      ({"o": Rows(AT + FAR, 2560, 320, 64)}, "'o' overlaps 'v'"),
                                      ({"lse": AT + 2 * FAR}, "'lse' overlaps 'k_scales'"),
                                      ({"lse": AT + 5 * FAR}, "'o' overlaps 'lse'"),
                                      ({"block_table": AT + 8 * FAR}, "'lse' overlaps 'block_table'")])
def test_attention_places(kw, names):
    assert attention(cache8(**kw)) == INVALID and names in _native.last_error()


def test_attention_plans_and_workspaces():
    lib = _native.load_library()
    plan = _native.AttentionPlan()
    seen = set()
    for kv_len, n in ((64, 1), (64000, 1), (6400, 5000), (64000, 300), (640, 40000)):
        a = cache8(kv_len=kv_len, n=n, q=Rows(AT + 4 * FAR, 8 * n * 64, n * 64, 64), o=Rows(AT + 16 * FAR, 8 * n * 64, n * 64, 64),
                   num_pages=3000, lse=None, k=Rows(AT + 24 * FAR, 4096, 2048, 64), v=Rows(AT + 32 * FAR, 4096, 2048, 64),
                   k_scales=Rows(AT + 40 * FAR, 4, 2, 1), v_scales=Rows(AT + 41 * FAR, 4, 2, 1))
        assert lib.asc_quantized_cache_attention_plan(ctypes.byref(a), ctypes.byref(plan)) == 0
        seen.add((plan.kernel, plan.splits > 1))
        need = lib.asc_quantized_cache_attention_workspace(ctypes.byref(a))
        assert (need > 0) == (plan.splits > 1)
        if need:
            for ws, nbytes in ((None, need), (AT, need - 1), (AT + 4, need)):
                assert attention(a, ws, nbytes) == INVALID and "workspace" in _native.last_error()
    assert {x for x, _ in seen} == {b"cache8_narrow", b"cache8_wide"} and {x for _, x in seen} == {False, True}
    assert lib.asc_quantized_cache_attention(None, None, 0, None) == INVALID
    assert lib.asc_quantized_cache_attention_plan(ctypes.byref(cache8()), None) == INVALID
    for kw in ({"batch": 0}, {"n": 0}, {"q_heads": 0}):
        assert attention(cache8(**kw), None, 0) == 0
