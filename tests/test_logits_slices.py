"""The slices of process_logits' rows, on the host: they cover a row, and a count lies inside of its slice, whatever the rows' length and
the place of their first byte."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "pyasc_amd" / "csrc"
SOURCE = """
#include "logits_slices.h"
extern "C" int64_t slices_of(int64_t vocab, int size, int element, int aligned) { return asc::slices_of(vocab, size, element, aligned); }
extern "C" int slice_first(int slice, int size, int lead) { return asc::slice_first(slice, size, lead); }
extern "C" uint32_t slice_places(int first, int size, int vocab) { return asc::slice_places(first, size, vocab); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no C++ compiler")
    folder = tmp_path_factory.mktemp("slices")
    (folder / "s.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}", str(folder / "s.cpp"), "-o", str(folder / "s.so")], check=True)
    lib = ctypes.CDLL(str(folder / "s.so"))
    lib.slices_of.restype, lib.slices_of.argtypes = ctypes.c_int64, [ctypes.c_int64] + [ctypes.c_int] * 3
    lib.slice_places.restype = ctypes.c_uint32
    return lib


@pytest.mark.parametrize("element", [4, 2])
@pytest.mark.parametrize("size", [2048, 16384])
def test_slices(lib, size, element):
    vector = 16 // element
    vocabs = sorted({1, 2, 7, 50001} | {size * k + d for k in (1, 2, 8) for d in range(-vector - 1, vector + 2)})
    for vocab in vocabs:
        for aligned in (True, False):
            slices = lib.slices_of(vocab, size, element, aligned)
            for lead in range(1 if aligned else vector):
                end = 0
                for i in range(slices):
                    first, places = lib.slice_first(i, size, lead), lib.slice_places(lib.slice_first(i, size, lead), size, vocab)
                    assert max(first, 0) == end or places == 0, (vocab, lead, i)
                    assert 0 <= places <= size, (vocab, lead, i, places)
                    end = first + places if places else end
                    # what the kernel tells inside from outside by: token - first, in 32 bits without a sign
                    for token in (0, first - 1, first, vocab - 1):
                        if 0 <= token < vocab and (token - first) % 2 ** 32 < places:
                            assert first <= token < first + size
                assert end == vocab, (vocab, lead)
