"""The 4-bit paged key/value cache without a GPU: its layout and arithmetic on lengths (csrc/cache_dev.h) in a host
program, and the calls that its entry points refuse before any device work. No counterpart in the reference."""
import ctypes as C
import os
import subprocess

import pytest

from jepa_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_layout_and_lengths(tmp_path):
    exe = str(tmp_path / "host_cache")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-I" + os.path.join(ROOT, "jepa.cpp_amd", "csrc"),
                    os.path.join(ROOT, "tests", "host_cache.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr


SHAPE = dict(n_head=8, n_kv_head=2, head_dim=64, page_size=16, n_pages=10)
P = 0x10000      # a non-null, 16-byte aligned address that no refused call reads


def _shape(**kw):
    return C.byref(_lib.CacheShape(*{**SHAPE, **kw}.values()))


def test_page_bytes():
    L = _lib.lib()
    for ps in (16, 32, 64, 128, 256):
        for hd in (32, 64, 96, 128):
            assert L.jepa_amd_cache_page_bytes(_shape(page_size=ps, head_dim=hd)) == 2 * ps * 2 * (hd // 2 + hd // 16)      # 4.5 bits a value
    assert L.jepa_amd_cache_work_bytes(_shape(), 0, 0, 1) >= 0


@pytest.mark.parametrize("kw", [dict(head_dim=80), dict(head_dim=0), dict(head_dim=256), dict(page_size=24), dict(page_size=8), dict(page_size=0),
                                dict(page_size=512), dict(n_kv_head=3), dict(n_kv_head=0), dict(n_head=0), dict(n_head=-8), dict(n_head=8192),
                                dict(n_pages=0), dict(n_pages=-1), dict(n_pages=1 << 31)])
def test_shapes_refused(kw):
    L = _lib.lib()
    s = _shape(**kw)
    L.jepa_error_reset()
    assert L.jepa_amd_cache_page_bytes(s) == -1 and "not supported" in _lib.error_text()
    assert L.jepa_amd_cache_work_bytes(s, 1, 1, 1) == -1
    assert L.jepa_amd_cache_plan(0, s, 1, 1, P, P, P, 1, P, P, P, P, P, P, P, None) == -1
    assert L.jepa_amd_cache_store(0, s, P, 0, P, 512, P, 512, 1, P, None) == -1
    assert L.jepa_amd_cache_read(0, s, P, P, 1, 0, P, 512, P, 512, None) == -1
    assert L.jepa_amd_cache_attention(0, s, P, 0, P, 4096, 1, 1, P, P, P, 1, 1.0, 1, P, 4096, P, 1 << 40, None) == -1


def test_null_shape():
    assert _lib.lib().jepa_amd_cache_page_bytes(None) == -1
    assert _lib.lib().jepa_amd_cache_plan(0, None, 1, 1, P, P, P, 1, P, P, P, P, P, P, P, None) == -1


def _plan(**kw):
    a = dict(n_seq=1, n_rows=1, len=P, n_new=P, table=P, width=1, ring=P, free_in=P, free_out=P, kv_len=P, row_start=P, slot=P, refused=P)
    a.update(kw)
    return _lib.lib().jepa_amd_cache_plan(0, _shape(), a["n_seq"], a["n_rows"], a["len"], a["n_new"], a["table"], a["width"], a["ring"], a["free_in"],
                                          a["free_out"], a["kv_len"], a["row_start"], a["slot"], a["refused"], None)


@pytest.mark.parametrize("kw", [dict(n_seq=-1), dict(n_seq=4097), dict(n_rows=-1), dict(n_rows=1 << 31), dict(width=0), dict(width=1 << 27)] +
                         [{k: None} for k in ("len", "n_new", "table", "ring", "free_in", "free_out", "kv_len", "row_start", "slot", "refused")])
def test_plan_refuses(kw):
    _lib.lib().jepa_error_reset()
    assert _plan(**kw) == -1
    assert "jepa_amd_cache_plan" in _lib.error_text()


def _rows(fn, **kw):
    a = dict(cache=P, type=0, k=P, ldk=128, v=P, ldv=128, n_rows=3, slot=P)
    a.update(kw)
    if fn == "jepa_amd_cache_store":
        return _lib.lib().jepa_amd_cache_store(0, _shape(), a["cache"], a["type"], a["k"], a["ldk"], a["v"], a["ldv"], a["n_rows"], a["slot"], None)
    return _lib.lib().jepa_amd_cache_read(0, _shape(), a["cache"], a["slot"], a["n_rows"], a["type"], a["k"], a["ldk"], a["v"], a["ldv"], None)


BAD_ROWS = [dict(type=2), dict(type=8), dict(type=-1), dict(k=None), dict(v=None), dict(slot=None), dict(cache=None), dict(cache=P + 8), dict(k=P + 4),
            dict(v=P + 8), dict(ldk=127), dict(ldv=64), dict(ldk=130), dict(type=1, ldk=132), dict(type=30, ldv=132), dict(n_rows=-1),
            dict(n_rows=1 << 31), dict(ldk=1 << 50)]


@pytest.mark.parametrize("kw", BAD_ROWS)
@pytest.mark.parametrize("fn", ["jepa_amd_cache_store", "jepa_amd_cache_read"])
def test_rows_refused(fn, kw):
    _lib.lib().jepa_error_reset()
    assert _rows(fn, **kw) == -1
    assert fn in _lib.error_text()


@pytest.mark.parametrize("kw", [dict(type=2), dict(q=None), dict(out=None), dict(q=P + 8), dict(ldq=508), dict(ldo=511), dict(type=1, ldq=516), dict(n_seq=4097),
                                dict(n_rows=-1), dict(row_start=None), dict(kv_len=None), dict(table=None), dict(width=0), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(block=-1), dict(work=None), dict(work=P + 4), dict(work_bytes=0), dict(cache=None)])
def test_attention_refuses(kw):
    a = dict(cache=P, type=0, q=P, ldq=512, n_seq=2, n_rows=3, row_start=P, kv_len=P, table=P, width=4, scale=0.125, block=1, out=P, ldo=512, work=P,
             work_bytes=1 << 40)
    a.update(kw)
    L = _lib.lib()
    L.jepa_error_reset()
    assert L.jepa_amd_cache_attention(0, _shape(), a["cache"], a["type"], a["q"], a["ldq"], a["n_seq"], a["n_rows"], a["row_start"], a["kv_len"], a["table"],
                                      a["width"], a["scale"], a["block"], a["out"], a["ldo"], a["work"], a["work_bytes"], None) == -1
    assert "jepa_amd_cache_attention" in _lib.error_text()


def test_work_space_too_small_is_named():
    L = _lib.lib()
    need = L.jepa_amd_cache_work_bytes(_shape(), 2, 3, 4)
    L.jepa_error_reset()
    assert L.jepa_amd_cache_attention(0, _shape(), P, 0, P, 512, 2, 3, P, P, P, 4, 0.125, 1, P, 512, P, need - 1, None) == -1
    assert str(need) in _lib.error_text()


@pytest.mark.parametrize("heads,kvh,hd,page", [(1, 1, 128, 64), (32, 8, 128, 64), (40, 8, 96, 32), (16, 16, 64, 16), (64, 1, 32, 256)])
def test_work_space_for_the_largest_step_does_for_smaller_ones(heads, kvh, hd, page):
    """The bytes never fall where one of the sizes grows: a program asks once."""
    s = _shape(n_head=heads, n_kv_head=kvh, head_dim=hd, page_size=page)
    need = lambda *a: _lib.lib().jepa_amd_cache_work_bytes(s, *a)  # noqa: E731
    for n_seq in (1, 2, 7, 64, 300):
        for width in (1, 4, 16, 100, 2000):
            rows = sorted({1, 2, 5, 24, 25, 63, 64, 65, 100, 192, 193, 256, 257, 500, 768, 769, 800, 1000, 1001, 2000, 4000, 20000, 32001, 100000})
            got = [need(n_seq, r, width) for r in rows]
            assert got == sorted(got), (n_seq, width, list(zip(rows, got)))
            for r, b in zip(rows, got):
                assert b >= need(max(1, n_seq // 2), r, width) and b >= need(n_seq, r, max(1, width // 2)), (n_seq, r, width)
