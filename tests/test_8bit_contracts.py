"""CPU: contracts of the 8-bit operators that need no launch: scratch and launches of the integer projection, sizes that
32-bit indices cannot hold, calls without rows, and when the C++ binding is compiled again."""

from __future__ import annotations

import importlib
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

ARG, UNSUPPORTED = -1, -4
A = 1 << 20  # an aligned address that is never read: every call here is refused first
ROOT = Path(__file__).resolve().parents[1]


def _lib():
    return importlib.import_module("nari-qwen3-tts_b200._lib").lib()


def test_linear_launches():
    """One launch for up to 8 tokens whose codes, in 1, 2, 4 or 8 rows of k rounded up to 16, fit 96 KB."""

    f = _lib().nqt_linear_int8_launches
    for m in range(1, 20):
        slots = next((s for s in (1, 2, 4, 8) if s >= m), None)
        for k in (1, 16, 2048, 12288, 12289, 24576, 24577, 49152, 49153, 98304, 98305, 131072):
            one = slots is not None and slots * math.ceil(k / 16) * 16 <= 96 * 1024
            assert f(m, k) == (1 if one else 2)
    assert f(0, 64) == 0


@pytest.mark.parametrize(("m", "k"), [(9, 64), (64, 2048), (8, 12304), (3, 24592), (1, 98320)])
def test_linear_refuses_missing_scratch_where_it_is_used(m, k):
    def call(xq, ldxq, xscale):
        return _lib().nqt_linear_int8(A, k, xq, ldxq, xscale, A, k, A, None, A, 4, m, 4, 4, k, 0, A, None)

    for args in ((None, k, A), (A, k, None), (A + 8, k, A), (A, k - 16, A), (A, k + 8, A)):
        assert call(*args) == ARG


@pytest.mark.parametrize(("m", "n"), [(2**31 - 1, 4), (2**31 - 127, 4), (4, 2**31 - 1), (4, 2**31 - 255)])
def test_sizes_behind_32_bit_indices_are_refused(m, n):
    """Rows and columns are rounded up to whole tiles in 32 bits.  In a process of its own: a product that went on with
    them would not come back."""

    code = f"""
import importlib
lib = importlib.import_module("nari-qwen3-tts_b200._lib").lib()
print(lib.nqt_gemm_int8({A}, 16, {A}, {A}, 16, {A}, None, {A}, {n}, {m}, {n}, {n}, 16, 0, {A}, None))
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and int(r.stdout) == UNSUPPORTED


def test_rows_behind_32_bit_indices_are_refused(nqt):
    """The same limits at the functions, which would cut the counts to 32 bits."""

    weight = nqt.kernels.Int8Weight.__new__(nqt.kernels.Int8Weight)
    weight._lay_out(torch.zeros(6, 16, dtype=torch.int8), torch.ones(6), False)
    row = torch.zeros(1, 16, dtype=torch.bfloat16)
    for rows in (2**31 - 127, 2**32 + 5):
        with pytest.raises(ValueError, match="rows"):
            nqt.kernels.linear_int8(row.expand(rows, 16), weight)
    for shape in ((1, 2**31 - 7), (1, 2**32 + 5), (2**32 + 5, 1)):
        with pytest.raises(ValueError, match="rows"):
            nqt.kernels.int8_quantize_rows(torch.empty(shape, dtype=torch.bfloat16, device="meta"))
    assert _lib().nqt_int8_quantize_rows(A, 2**31, 1, 2**31 - 7, A, 2**31, A, None) == UNSUPPORTED
    for rows in (2**31 - 254, 2**32 + 2):
        for gate_up in (False, True):
            with pytest.raises(ValueError, match="rows"):
                weight._lay_out(torch.zeros(1, 16, dtype=torch.int8).expand(rows, 16), torch.ones(1).expand(rows), gate_up)


def test_quantize_no_rows():
    assert _lib().nqt_int8_quantize_rows(None, 8, 0, 8, None, 16, None, None) == 0
    assert _lib().nqt_int8_quantize_rows(None, 8, -1, 8, None, 16, None, None) == ARG
    assert _lib().nqt_int8_quantize_rows(None, 8, 0, 0, None, 16, None, None) == ARG


def test_one_row_of_codes_with_any_pitch(nqt):
    """Only the missing GPU stops a single row of codes whose stride is odd."""

    weight = nqt.kernels.Int8Weight.__new__(nqt.kernels.Int8Weight)
    weight._lay_out(torch.zeros(6, 33, dtype=torch.int8), torch.ones(6), False)
    base = torch.zeros(4, 101, dtype=torch.int8)
    with pytest.raises(ValueError, match="CUDA"):
        nqt.kernels.linear_int8(base[:1, :33], weight, xscale=torch.ones(1))
    with pytest.raises(ValueError, match="16-byte"):
        nqt.kernels.linear_int8(base[:2, :33], weight, xscale=torch.ones(2))
    with pytest.raises(ValueError, match="16-byte"):
        nqt.kernels.linear_int8(base[1:2, :33], weight, xscale=torch.ones(1))


@pytest.mark.parametrize("theta", [math.inf, 1e300, 1e-60, -1.0])
def test_rope_theta_has_to_be_a_positive_float32(nqt, theta):
    q, k = torch.zeros(2, 16, 128, dtype=torch.bfloat16), torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    w, i = torch.ones(128, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.long)
    cache, scales = torch.zeros(4, 2, 16, 8, 128, dtype=torch.int8), torch.ones(4, 2, 1, 8)
    with pytest.raises(ValueError, match="rope_theta"):
        nqt.paired_qk_norm_rope_paged_cache8(q, k, k, w, w, i, 1e-6, theta, cache, scales, i, i)
    if abs(theta) < 1e30 or theta == math.inf:
        args = [A, 4096, 128, A, 4096, 128, A, 4096, 128, A, A, A, A, A, A, 2048, 128, A, A, 64, 16, 3, 16, 8, 128, 1e-6,
                theta, 3, A, None]
        assert _lib().nqt_qk_norm_rope_paged_cache8(*args) == ARG


def test_binding_is_compiled_again_for_another_torch(monkeypatch, tmp_path):
    """The binding belongs to the torch and the Python that it was compiled against, whatever its age."""

    build = importlib.import_module("nari-qwen3-tts_b200.build")
    for path in ("BUILD_DIR", "BIND_PATH"):
        monkeypatch.setattr(build, path, tmp_path / path)
    build.BUILD_DIR.mkdir()
    build.BIND_PATH.write_bytes(b"")
    assert not build._bind_up_to_date()  # nothing says what it was compiled against
    build._mark_bind()
    assert build._bind_up_to_date()
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert not build._bind_up_to_date()
