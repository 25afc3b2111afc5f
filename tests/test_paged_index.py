"""The paged cache's index arithmetic, walked on the host (no GPU), and the
refusals that need no device."""

from __future__ import annotations

import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_index_arithmetic_stays_in_bounds(tmp_path):
    exe = tmp_path / "paged_index"
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-fsanitize=address,undefined",
                    str(ROOT / "tests" / "paged_index.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout.strip() == "ok", res.stdout + res.stderr


class _Ctx:  # the checks below come before any call of the library
    _h = None
    handle = None


def _array(shape, dtype=np.float32):
    from franken_ocr_amd.device import DeviceArray

    return DeviceArray.borrow(_Ctx(), 256, shape, dtype)


def _cache(**kw):
    from franken_ocr_amd.engine import PagedCache

    c = PagedCache.__new__(PagedCache)
    c.ctx, c._h = _Ctx(), None
    c.n_pages, c.page_size, c.n_kv_heads, c.head_dim, c.dtype = 8, 16, 2, 64, "f32"
    return c


@pytest.mark.parametrize("change,text", [
    ({"lens": (3,)}, "3 lengths for 4 rows"),
    ({"q": (3, 256)}, "q of shape"),
    ({"out": (4, 128)}, "out of shape"),
    ({"k": (4, 64)}, "k_steps of shape"),
    ({"prefix": (2,)}, "prefix of shape"),
    ({"weights": (4, 3, 64)}, "weights of shape"),
    ({"weights": (4, 128)}, "weights of shape"),
])
def test_step_refuses_arrays_that_do_not_fit(change, text):
    from franken_ocr_amd import _abi

    sh = {"q": (4, 256), "k": (4, 128), "v": (4, 128), "out": (4, 256), "tables": (4, 2), "lens": (4,)}
    sh.update(change)
    a = {n: _array(s, np.uint32 if n in ("tables", "lens", "prefix") else np.float32) for n, s in sh.items()}
    with pytest.raises(_abi.ContractViolation, match=text):
        _cache().step(a["q"], a["k"], a["v"], a["tables"], a["lens"], a["out"], prefix=a.get("prefix"),
                      weights=a.get("weights"), n_heads=4)


@pytest.mark.parametrize("shapes,n_heads,want", [
    # q, k, v, out of four rows; what the call passes on: heads, ldq, ldkv, ldo
    (((4, 256), (4, 128), (4, 128), (4, 256)), None, (4, 256, 128, 256)),
    (((4, 512), (4, 200), (4, 200), (4, 300)), 4, (4, 512, 200, 300)),      # wider rows: the arrays' widths
    (((4, 4, 64), (4, 2, 64), (4, 2, 64), (4, 4, 64)), None, (4, 256, 128, 256)),
    (((6, 260), (9, 128), (5, 128), (4, 256)), 4, (4, 260, 128, 256)),      # more rows than are read
    (((1024,), (8, 64), (512,), (2, 512)), 4, (4, 256, 128, 256)),          # flat, or in rows of their own
])
def test_row_strides_are_the_arrays_widths(monkeypatch, shapes, n_heads, want):
    from franken_ocr_amd import _abi

    seen = {}
    monkeypatch.setattr(_abi, "call", lambda name, *a: seen.update({name: a}))
    q, k, v, out = (_array(s) for s in shapes)
    tables, lens = _array((4, 2), np.uint32), _array((4,), np.uint32)
    _cache().step(q, k, v, tables, lens, out, n_heads=n_heads)
    a = seen["focr_hip_paged_step"]
    assert (a[4], a[3], a[7], a[17]) == want
    _cache().attention(q, tables, lens, out, n_heads=n_heads)
    a = seen["focr_hip_paged_attention"]
    assert (a[4], a[3], a[14]) == (want[0], want[1], want[3])
    _cache().write(k, v, lens, tables)
    assert seen["focr_hip_paged_write"][4] == want[2]
    _cache().step(q, k, v, tables, lens, out, n_heads=2, ldq=129, ldkv=128, ldo=130)  # given ones come first
    a = seen["focr_hip_paged_step"]
    assert (a[4], a[3], a[7], a[17]) == (2, 129, 128, 130)


@pytest.mark.parametrize("shapes,text", [
    (((4, 250), (4, 128), (4, 128), (4, 256)), "no whole heads"),
    (((4, 256), (4, 128), (4, 130), (4, 256)), "k rows of 128 and v rows of 130"),
])
def test_step_refuses_rows_of_no_one_width(shapes, text):
    from franken_ocr_amd import _abi

    q, k, v, out = (_array(s) for s in shapes)
    with pytest.raises(_abi.ContractViolation, match=text):
        _cache().step(q, k, v, _array((4, 2), np.uint32), _array((4,), np.uint32), out)


def test_beam_calls_refuse_rows_that_are_no_groups():
    from franken_ocr_amd import _abi, engine

    u = lambda *s: _array(s, np.uint32)  # noqa: E731
    with pytest.raises(_abi.ContractViolation, match="no groups of 4"):
        engine.beam_select(_array((6, 100)), _array((6,)), 4, u(6), u(6), _array((6,)))
    with pytest.raises(_abi.ContractViolation, match="tokens of shape"):
        engine.beam_select(_array((8, 100)), _array((8,)), 4, u(8), u(6), _array((8,)))
    with pytest.raises(_abi.ContractViolation, match="no groups of 0"):
        engine.beam_reorder(u(6), 0)
    with pytest.raises(_abi.ContractViolation, match="history_len of shape"):
        engine.beam_reorder(u(8), 4, history=u(8, 10), history_len=u(7))


@pytest.mark.parametrize("owner", [None, np.zeros(1), np.zeros(3), [], 0])
def test_borrowed_memory_is_not_freed(monkeypatch, owner):
    """Whatever owns it: an empty or zero owner, one without a truth value."""
    from franken_ocr_amd import _abi
    from franken_ocr_amd.device import DeviceArray

    class Lib:
        def focr_hip_dfree(self, *a):
            raise AssertionError("borrowed memory freed")

    monkeypatch.setattr(_abi, "lib", Lib)
    a = DeviceArray.borrow(_Ctx(), 256, (4, 2), np.float32, owner=owner)
    assert a.ptr == 256 and a.nbytes == 32
    v = a.view_rows(1, 3)
    v.free()
    a.free()
    assert a.ptr == 0


def test_unknown_dtype_is_refused():
    from franken_ocr_amd.engine import PagedCache

    with pytest.raises(ValueError, match="dtype"):
        PagedCache(8, 16, 2, 64, "f8", ctx=_Ctx())


def test_null_handles_are_bad_handles():
    from franken_ocr_amd import _abi

    lib = _abi.lib()
    assert lib.focr_hip_paged_create(None, 1, 16, 1, 64, 0, None, None, None) == _abi.E_BAD_HANDLE
    assert lib.focr_hip_paged_regions(None, None, None) == _abi.E_BAD_HANDLE
    assert lib.focr_hip_paged_free(None) == _abi.OK
    assert lib.focr_hip_beam_reorder(None, 1, 1, None, None, None, 0, None, 0, None, 0, None, 0, None, None, 0,
                                     0) == _abi.E_BAD_HANDLE
