"""What a forward of ``adsp_attn_cross_fwd`` keeps for its backward lies as the sizes of the call and ADSP_SPARSE say.  A backward that is handed a buffer of another layout
refuses it in front of any launch."""

import ctypes
import os

import pytest

from adasplash_amd import _lib

CASES = [
    (4, 32, 8, 1024, 5000, 128, "bf16"),  # on the supports; with ADSP_SPARSE=0 lists of the forward on 32 rows
    (2, 8, 8, 448, 1500, 64, "f32"),      # lists
    (2, 4, 2, 100, 2500, 128, "f16"),     # lists
]
DTYPES = {"f32": _lib.ADSP_F32, "bf16": _lib.ADSP_BF16, "f16": _lib.ADSP_F16}
ERR_WORKSPACE = 6


def backward(lib, case, supports_bytes):
    """The call on addresses that no launch may see: a status, or the test does not get this far."""
    B, Hq, Hkv, Nq, Nk, D, dtype = case
    at = ctypes.c_void_p(1 << 20)
    ws = lib.adsp_attn_cross_bwd_workspace_bytes(B, Hq, Hkv, Nq, Nk, D, DTYPES[dtype], 1.5, 1)
    return lib.adsp_attn_cross_bwd(at, at, at, at, at, None, 0, None, 0, at, at, at, at, at, B, Hq, Hkv, Nq, Nk, D, DTYPES[dtype], 1.5, at, ws, at, supports_bytes, None)


@pytest.mark.parametrize("case", CASES)
def test_a_buffer_of_another_layout_is_refused(case, monkeypatch):
    lib = _lib.load()
    size = lambda: lib.adsp_attn_cross_supports_bytes(*case[:6], DTYPES[case[6]], 1.5)  # noqa: E731
    monkeypatch.delenv("ADSP_SPARSE", raising=False)
    here = size()
    assert here > 0
    for other in (here - 16, here + 16, 2 * here):
        assert backward(lib, case, other) == ERR_WORKSPACE
    monkeypatch.setenv("ADSP_SPARSE", "0")
    there = size()
    if there != here:
        assert backward(lib, case, here) == ERR_WORKSPACE
        monkeypatch.delenv("ADSP_SPARSE")
        assert backward(lib, case, there) == ERR_WORKSPACE
    assert (there != here) == (case[6] == "bf16")
    assert "ADSP_SPARSE" not in os.environ or os.environ["ADSP_SPARSE"] == "0"
