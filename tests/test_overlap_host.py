"""Results that share bytes with an operand or another result, without a GPU: the C entries of the rotary calls
and of attention over other keys refuse them before a launch."""
import ctypes

import pytest

from pyasc_amd import _native
from pyasc_amd._native import Rows

FAR = 1 << 30  # addresses that are never followed, far apart


def place(i):
    return (1 + i) * FAR


def refused(entry, args, first, second, *more):
    code = getattr(_native.load_library(), entry)(ctypes.byref(args), *more, None)
    assert code == _native.ERR_INVALID_ARG
    error = _native.last_error()
    assert entry in error and "overlaps" in error and f"'{first}'" in error and f"'{second}'" in error, error


def rotary_args():
    """Two sequences of five tokens, four query and two key heads of 64 bfloat16 values."""
    a = _native.RotaryArgs()
    a.dtype, a.head_dim, a.rotary_dim, a.magnitude = _native.DT_BFLOAT16, 64, 64, 1.0
    a.batch, a.q_heads, a.k_heads, a.seq = 2, 4, 2, 5
    for i, name in enumerate(("q", "q_out", "dq_out")):
        setattr(a, name, Rows(place(i), 1280, 320, 64))
    for i, name in enumerate(("k", "k_out", "dk_out")):
        setattr(a, name, Rows(place(3 + i), 640, 320, 64))
    for i, name in enumerate(("positions", "freqs", "q_weight", "k_weight", "dq_weight", "dk_weight")):
        setattr(a, name, place(6 + i))
    return a


Q_BYTES, K_BYTES = 2 * 4 * 5 * 64 * 2, 2 * 2 * 5 * 64 * 2
ROTARY = [("asc_rotary", ()), ("asc_qk_norm_rotary", ()), ("asc_qk_norm_rotary_bwd", (place(20), 1 << 24))]


@pytest.mark.parametrize("entry,more", ROTARY)
def test_rotary_results(entry, more):
    grad = entry.endswith("bwd")
    names = ("dq", "dk") if grad else ("q_out", "k_out")
    # one row into its own input, from before it and from behind it
    for shift in (128, -128, Q_BYTES - 128, 128 - Q_BYTES):
        a = rotary_args()
        a.q_out.data = place(0) + shift
        refused(entry, a, names[0], "q", *more)
    a = rotary_args()  # in place, but in another order
    a.q_out = Rows(place(0), 1280, 64, 256)
    refused(entry, a, names[0], "q", *more)
    a = rotary_args()  # over another operand, in place or not
    a.q_out.data = place(3) + K_BYTES - 2
    refused(entry, a, names[0], "k", *more)
    a = rotary_args()
    a.k_out.data = place(0)
    refused(entry, a, names[1], "q", *more)
    a = rotary_args()
    a.k_out.data = place(1) + 256
    refused(entry, a, names[0], names[1], *more)
    for name, last in (("positions", 2 * 5 * 4 - 2), ("freqs", 32 * 8 - 2)):
        a = rotary_args()
        a.position_batch_stride, a.position_seq_stride = 5, 1
        a.k_out.data = getattr(a, name) + last
        refused(entry, a, names[1], name, *more)
    if entry != "asc_rotary":
        for t, name in enumerate(("q_weight", "k_weight")):
            a = rotary_args()
            (a.k_out if t else a.q_out).data = getattr(a, name) - K_BYTES + 2 if t else getattr(a, name) + 254
            refused(entry, a, names[t], name, *more)


def test_rotary_gradients():
    entry, more = ROTARY[2]
    a = rotary_args()
    a.q_out.data = a.dq_out.data + 64
    refused(entry, a, "dq", "dq_out", *more)
    a = rotary_args()
    a.k_out.data = a.dq_out.data + Q_BYTES - 2
    refused(entry, a, "dk", "dq_out", *more)
    for shift in (0, 4, -252):  # the weights' gradients, of one norm for queries and keys or next to each other
        a = rotary_args()
        a.dk_weight = a.dq_weight + shift
        refused(entry, a, "dq_weight", "dk_weight", *more)
    a = rotary_args()
    a.dq_weight = a.k_out.data + K_BYTES - 4
    refused(entry, a, "dk", "dq_weight", *more)
    a = rotary_args()  # no rows: the weights' gradients are still written
    a.seq, a.dk_weight = 0, a.dq_weight
    refused(entry, a, "dq_weight", "dk_weight", *more)


def attention_args():
    """Two sequences, eight heads on two, five queries, 300 keys in one piece, all contiguous."""
    a = _native.AttentionArgs()
    a.dtype, a.head_dim, a.sm_scale = _native.DT_BFLOAT16, 64, 0.125
    a.batch, a.q_heads, a.kv_heads, a.q_len, a.kv_len = 2, 8, 2, 5, 300
    for i, name in enumerate(("q", "o", "d_o", "dq")):
        setattr(a, name, Rows(place(i), 2560, 320, 64))
    for i, name in enumerate(("k", "v", "dk", "dv")):
        setattr(a, name, Rows(place(4 + i), 38400, 19200, 64))
    for i, name in enumerate(("k_draft", "v_draft")):
        setattr(a, name, Rows(place(8 + i), 640, 320, 64))
    for i, name in enumerate(("lse", "kv_lengths", "draft_lengths", "tree_mask")):
        setattr(a, name, place(10 + i))
    a.mask_batch_stride, a.mask_row_stride = 25, 5
    return a


WORKSPACE = (place(20), 1 << 28)


@pytest.mark.parametrize("entry", ["asc_cross_attention_fwd", "asc_tree_attention"])
def test_attention_results(entry):
    q_bytes, kv_bytes, draft_bytes = 2 * 8 * 5 * 64 * 2, 2 * 2 * 300 * 64 * 2, 2 * 2 * 5 * 64 * 2
    sizes = {"q": q_bytes, "k": kv_bytes, "v": kv_bytes, "kv_lengths": 8}
    if entry == "asc_tree_attention":
        sizes.update(k_draft=draft_bytes, v_draft=draft_bytes, draft_lengths=8, tree_mask=50)
    for name, nbytes in sizes.items():
        at = getattr(attention_args(), name)
        at = at if isinstance(at, int) else at.data
        for first in (at + (nbytes - 1) // 16 * 16, at - q_bytes + 16):
            a = attention_args()
            a.o.data = first
            refused(entry, a, "o", name, *WORKSPACE)
        a = attention_args()
        a.lse = at + nbytes - 2
        refused(entry, a, "lse", name, *WORKSPACE)
    a = attention_args()
    a.lse = a.o.data + 4
    refused(entry, a, "lse", "o", *WORKSPACE)


def test_pages_and_their_table():
    a = attention_args()
    a.page_size, a.num_pages, a.block_table, a.table_stride, a.kv_len = 16, 40, place(14), 19, 304
    a.k = a.v = Rows(place(4), 2048, 1024, 64)
    a.o.data = place(4) + 40 * 4096 - 16
    refused("asc_tree_attention", a, "o", "k", *WORKSPACE)
    a.o.data = place(14) + (2 * 19 * 4 - 1) // 16 * 16
    refused("asc_tree_attention", a, "o", "block_table", *WORKSPACE)


def test_attention_gradients():
    entry = "asc_cross_attention_bwd"
    for result, like in (("dq", "q"), ("dk", "k"), ("dv", "v")):
        for name in ("do", "q", "k", "v", "o", "lse", "kv_lengths"):
            a = attention_args()
            at = getattr(a, "d_o" if name == "do" else name)
            getattr(a, result).data = at if isinstance(at, int) else at.data + 128
            refused(entry, a, result, name, *WORKSPACE)
        for other in ("dq", "dk", "dv"):
            if other == result:
                continue
            a = attention_args()
            getattr(a, result).data = getattr(a, other).data + 128
            refused(entry, a, *sorted((result, other)), *WORKSPACE)
