"""Rotary positions without a GPU: the frequencies, and what the C entries refuse before a launch."""
import ctypes
import math

import pytest
import torch

from pyasc_amd import _native, kernels


def test_frequencies():
    f, m = kernels.rotary_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0
    for i in range(32):
        assert math.isclose(float(f[i]), 10000.0 ** (-i / 32), rel_tol=1e-14)
    linear, m = kernels.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(linear, f / 4) and m == 1.0
    ntk, _ = kernels.rotary_frequencies(64, scaling="ntk", factor=4.0, device="cpu")
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-13)
    yarn, m = kernels.rotary_frequencies(64, scaling="yarn", factor=4.0, original_length=2048, device="cpu")
    assert m == 0.1 * math.log(4.0) + 1.0
    for i in range(32):
        turns = 2048 * float(f[i]) / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1) / 31))
        assert math.isclose(float(yarn[i]), float(f[i]) * (keep + (1 - keep) / 4), rel_tol=1e-12)
    same, m = kernels.rotary_frequencies(64, scaling="yarn", factor=1.0, original_length=2048, device="cpu")
    assert torch.allclose(same, f, rtol=1e-14) and m == 1.0


@pytest.mark.parametrize("args,kw", [((0,), {}), ((3,), {}), ((-2,), {}), ((64, -1.0), {}),
                                     ((64,), {"scaling": "other"}), ((64,), {"factor": 0.0}),
                                     ((2,), {"scaling": "ntk"}), ((64,), {"scaling": "yarn", "factor": 2.0})])
def test_frequencies_refused(args, kw):
    with pytest.raises(ValueError):
        kernels.rotary_frequencies(*args, device="cpu", **kw)


def _args(**kw):
    a = _native.RotaryArgs()
    a.head_dim, a.rotary_dim, a.batch, a.q_heads, a.seq, a.magnitude = 64, 64, 1, 2, 3, 1.0
    rows = _native.Rows(1024, 384, 192, 64)
    a.q, a.q_out, a.dq_out = rows, rows, rows
    a.positions = a.freqs = a.q_weight = a.dq_weight = 1024
    for name, value in kw.items():
        setattr(a, name, value)
    return a


CASES = [({"dtype": 3}, _native.ERR_UNSUPPORTED), ({"batch": -1}, _native.ERR_INVALID_ARG),
         ({"seq": -1}, _native.ERR_INVALID_ARG), ({"head_dim": 63}, _native.ERR_UNSUPPORTED),
         ({"head_dim": 514}, _native.ERR_UNSUPPORTED), ({"rotary_dim": 66}, _native.ERR_INVALID_ARG),
         ({"rotary_dim": 3}, _native.ERR_INVALID_ARG), ({"positions": None}, _native.ERR_INVALID_ARG),
         ({"freqs": None}, _native.ERR_INVALID_ARG), ({"q": _native.Rows()}, _native.ERR_INVALID_ARG),
         ({"q_out": _native.Rows()}, _native.ERR_INVALID_ARG), ({"k_heads": 1}, _native.ERR_INVALID_ARG),
         ({"seq": 1 << 31}, _native.ERR_UNSUPPORTED), ({"batch": 1 << 30, "seq": 64}, _native.ERR_UNSUPPORTED),
         ({"q_heads": 1 << 21}, _native.ERR_UNSUPPORTED)]


@pytest.mark.parametrize("fn", ["asc_rotary", "asc_qk_norm_rotary", "asc_qk_norm_rotary_bwd"])
@pytest.mark.parametrize("kw,code", CASES + [({"epsilon": -1.0}, None), ({"q_weight": None}, None),
                                             ({"dq_weight": None}, None), ({"dq_out": _native.Rows()}, None)])
def test_refusals(fn, kw, code):
    lib = _native.load_library()
    if code is None:  # an argument of the norm or of its gradient
        if fn == "asc_rotary" or (fn == "asc_qk_norm_rotary" and "dq" in next(iter(kw))):
            pytest.skip("not an argument of this entry")
        code = _native.ERR_INVALID_ARG
    a = _args(**kw)
    args = (1024, 1 << 30) if fn.endswith("bwd") else ()
    assert getattr(lib, fn)(ctypes.byref(a), *args, None) == code
    assert fn in _native.last_error()


def test_null_arguments_and_small_workspaces():
    lib = _native.load_library()
    assert lib.asc_rotary(None, None) == _native.ERR_INVALID_ARG
    a = _args()
    need = lib.asc_qk_norm_rotary_bwd_workspace(ctypes.byref(a))
    assert need == 3 * 2 * 64 * 4  # the sums of a workgroup for every token
    assert lib.asc_qk_norm_rotary_bwd(ctypes.byref(a), 1024, need - 1, None) == _native.ERR_INVALID_ARG
    assert lib.asc_qk_norm_rotary_bwd(ctypes.byref(a), None, need, None) == _native.ERR_INVALID_ARG


def test_nothing_to_do():
    lib = _native.load_library()
    for kw in ({"seq": 0}, {"batch": 0}, {"q_heads": 0}):
        a = _args(**kw)
        assert lib.asc_rotary(ctypes.byref(a), None) == 0
        assert lib.asc_qk_norm_rotary(ctypes.byref(a), None) == 0
        assert lib.asc_qk_norm_rotary_bwd_workspace(ctypes.byref(a)) == 0
