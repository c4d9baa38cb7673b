"""Rotary positions of several axes and the calls that select the 4-bit cache's pages, without a GPU: what their entry points refuse before any device
work, and the sizes of their work spaces. No counterpart in the reference."""
import ctypes as C

import pytest

from jepa_amd import _lib

P = 0x10000      # a non-null, 16-byte aligned address that no refused call reads
SHAPE = dict(n_head=8, n_kv_head=2, head_dim=64, page_size=16, n_pages=10)
AXES = dict(head_dim=64, form=1, dims=(20, 20, 20), theta=1e4, scale=None)


def shape(**kw):
    return C.byref(_lib.CacheShape(*{**SHAPE, **kw}.values()))


def axes(**kw):
    return C.byref(_lib.RopeAxes.of(**{**AXES, **kw}))


def rope(**kw):
    a = dict(rope=axes(), type=0, x=P, ldx=512, n_rows=3, n_head=8, pos=P, out=P, ldo=512)
    a.update(kw)
    return _lib.lib().jepa_amd_rope_rows(0, a["rope"], a["type"], a["x"], a["ldx"], a["n_rows"], a["n_head"], a["pos"], 0, a["out"], a["ldo"], None)


def append(**kw):
    a = dict(shape=shape(), rope=axes(), cache=P, type=0, q=P, ldq=512, k=P, ldk=128, v=P, ldv=128, n_rows=3, pos=P, slot=P, q_out=P, ldo=512)
    a.update(kw)
    return _lib.lib().jepa_amd_cache_append(0, a["shape"], a["rope"], a["cache"], a["type"], a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"], a["n_rows"],
                                            a["pos"], a["slot"], a["q_out"], a["ldo"], None)


def digest(**kw):
    a = dict(shape=shape(), cache=P, n_seq=2, n_rows=3, row_start=P, kv_len=P, table=P, width=4, digest=P)
    a.update(kw)
    return _lib.lib().jepa_amd_cache_digest(0, a["shape"], a["cache"], a["n_seq"], a["n_rows"], a["row_start"], a["kv_len"], a["table"], a["width"], a["digest"], None)


def digest_read(**kw):
    a = dict(shape=shape(), digest=P, page=P, n=3, bounds=P)
    a.update(kw)
    return _lib.lib().jepa_amd_cache_digest_read(0, a["shape"], a["digest"], a["page"], a["n"], a["bounds"], None)


def select(**kw):
    a = dict(shape=shape(), digest=P, type=0, q=P, ldq=512, n_seq=2, n_rows=3, row_start=P, kv_len=P, table=P, width=4, block=1, first=1, last=2, take=8, selected=P,
             work=P, work_bytes=1 << 40)
    a.update(kw)
    return _lib.lib().jepa_amd_cache_select(0, a["shape"], a["digest"], a["type"], a["q"], a["ldq"], a["n_seq"], a["n_rows"], a["row_start"], a["kv_len"], a["table"],
                                            a["width"], a["block"], a["first"], a["last"], a["take"], a["selected"], a["work"], a["work_bytes"], None)


def attend(**kw):
    a = dict(shape=shape(), cache=P, type=0, q=P, ldq=512, n_seq=2, n_rows=3, row_start=P, kv_len=P, table=P, width=4, selected=P, take=200, scale=0.125, block=1, out=P,
             ldo=512, work=P, work_bytes=1 << 40)
    a.update(kw)
    return _lib.lib().jepa_amd_cache_attention_selected(0, a["shape"], a["cache"], a["type"], a["q"], a["ldq"], a["n_seq"], a["n_rows"], a["row_start"], a["kv_len"],
                                                        a["table"], a["width"], a["selected"], a["take"], a["scale"], a["block"], a["out"], a["ldo"], a["work"],
                                                        a["work_bytes"], None)


def refused(call, name, **kw):
    _lib.lib().jepa_error_reset()
    assert call(**kw) == -1
    assert name in _lib.error_text(), _lib.error_text()


BAD_AXES = [dict(head_dim=0, dims=(2,)), dict(head_dim=20, dims=(2,)), dict(head_dim=264, dims=(2,)), dict(form=-1), dict(form=4), dict(dims=(21, 20, 20)), dict(dims=(0, 20)),
            dict(dims=(-2, 20)), dict(dims=(20, 20, 26)), dict(form=2), dict(form=2, dims=(16, 24)), dict(form=3), dict(form=3, dims=(10, 4)), dict(theta=0.0),
            dict(theta=-1e4), dict(theta=float("nan")), dict(theta=float("inf")), dict(scale=(1.0, float("nan"), 1.0)), dict(scale=(float("inf"), 1.0, 1.0))]


@pytest.mark.parametrize("kw", BAD_AXES)
def test_rotations_refused(kw):
    refused(rope, "jepa_amd_rope_rows", rope=axes(**kw))
    refused(append, "jepa_amd_cache_append", rope=axes(**kw))


@pytest.mark.parametrize("form, dims", [(0, (20, 20, 20)), (1, (20, 20, 20)), (2, (16, 16)), (3, (20, 20, 24))])
def test_angles_past_64_bits_refused(form, dims):
    # theta^(-2 f / w) of 1e-320 passes 1e288 = 2^957 in the higher of these widths, the scale takes it past 2^990
    refused(rope, "jepa_amd_rope_rows", rope=axes(form=form, dims=dims, theta=1e-320, scale=(1e40,) * len(dims)))
    refused(append, "jepa_amd_cache_append", rope=axes(form=form, dims=dims, theta=5e-324, scale=(1e200,) * len(dims)))
    refused(rope, "jepa_amd_rope_rows", rope=axes(form=form, dims=dims, scale=(1e299,) * len(dims)))


@pytest.mark.parametrize("n", [-1, 0, 5])
def test_number_of_axes_refused(n):
    r = _lib.RopeAxes.of(64, 1, (20, 20, 20))
    r.n_axes = n
    refused(rope, "jepa_amd_rope_rows", rope=C.byref(r))


def test_binding_refuses_axes():
    for dims, scale in (((), None), ((2,) * 5, None), ((2, 2), (1.0,))):
        with pytest.raises(ValueError):
            _lib.RopeAxes.of(64, 1, dims, scale=scale)


@pytest.mark.parametrize("kw", [dict(rope=None), dict(type=2), dict(x=None), dict(out=None), dict(pos=None), dict(x=P + 8), dict(out=P + 4), dict(ldx=511), dict(ldo=508),
                                dict(ldx=514), dict(type=1, ldx=516), dict(n_rows=-1), dict(n_rows=1 << 40), dict(n_rows=1 << 23), dict(n_head=0), dict(n_head=4097, ldx=1 << 20, ldo=1 << 20),
                                dict(ldx=1 << 50), dict(ldx=516)])
def test_rope_refuses(kw):
    refused(rope, "jepa_amd_rope_rows", **kw)


@pytest.mark.parametrize("kw", [dict(shape=None), dict(rope=None), dict(shape=shape(head_dim=128), ldq=1024, ldk=256, ldv=256, ldo=1024), dict(cache=None), dict(cache=P + 8),
                                dict(type=8), dict(k=None), dict(v=None), dict(q_out=None), dict(pos=None), dict(slot=None), dict(q=P + 4), dict(ldq=508), dict(ldk=64),
                                dict(ldv=64), dict(ldo=256), dict(n_rows=-1), dict(n_rows=1 << 31), dict(n_rows=1 << 23), dict(ldq=516)])
def test_append_refuses(kw):
    refused(append, "jepa_amd_cache_append", **kw)


TABLES = [dict(shape=None), dict(shape=shape(head_dim=80)), dict(n_seq=-1), dict(n_seq=4097), dict(n_rows=-1), dict(n_rows=1 << 31), dict(row_start=None), dict(kv_len=None),
          dict(table=None), dict(width=0), dict(width=1 << 27)]


@pytest.mark.parametrize("kw", TABLES + [dict(cache=None), dict(cache=P + 8), dict(digest=None), dict(digest=P + 4),
                                         dict(shape=shape(n_head=4096, n_kv_head=4096), n_seq=4096, n_rows=1 << 24)])
def test_digest_refuses(kw):
    refused(digest, "jepa_amd_cache_digest", **kw)


@pytest.mark.parametrize("kw", [dict(shape=None), dict(digest=None), dict(digest=P + 4), dict(page=None), dict(bounds=None), dict(bounds=P + 4), dict(n=-1), dict(n=1 << 24),
                                dict(n=1 << 40)])
def test_digest_read_refuses(kw):
    refused(digest_read, "jepa_amd_cache_digest_read", **kw)


TAKES = [dict(take=0), dict(take=-1), dict(take=257)]


@pytest.mark.parametrize("kw", TABLES + TAKES + [dict(first=-1), dict(first=7, last=2), dict(last=0), dict(last=-1), dict(last=9), dict(first=1 << 40), dict(type=2), dict(q=None),
                                                 dict(q=P + 8), dict(ldq=508), dict(block=-1), dict(selected=None), dict(digest=None), dict(digest=P + 8),
                                                 dict(width=5000, work=None), dict(width=5000, work=P + 8), dict(width=5000, work_bytes=0),
                                                 dict(shape=shape(n_head=4096, n_kv_head=4096), ldq=1 << 18, n_seq=4096, n_rows=16383)])
def test_select_refuses(kw):
    refused(select, "jepa_amd_cache_select", **kw)


@pytest.mark.parametrize("kw", TABLES + TAKES + [dict(type=2), dict(q=None), dict(out=None), dict(q=P + 8), dict(ldq=508), dict(ldo=511), dict(scale=float("nan")),
                                                 dict(scale=float("inf")), dict(block=-1), dict(selected=None), dict(cache=None), dict(cache=P + 8), dict(work=None),
                                                 dict(work=P + 8), dict(work_bytes=0), dict(shape=shape(n_head=4096, n_kv_head=4096), ldq=1 << 18, ldo=1 << 18, n_rows=32767)])
def test_attention_refuses(kw):
    refused(attend, "jepa_amd_cache_attention_selected", **kw)


def test_digest_bytes():
    L = _lib.lib()
    for hd in (32, 64, 96, 128):
        assert L.jepa_amd_cache_digest_bytes(shape(head_dim=hd)) == 2 * (2 * hd + 16)
    assert L.jepa_amd_cache_digest_bytes(shape(head_dim=80)) == -1
    assert L.jepa_amd_cache_digest_bytes(None) == -1


@pytest.mark.parametrize("heads,kvh,hd,page", [(1, 1, 128, 64), (32, 8, 128, 64), (40, 8, 96, 32), (16, 16, 64, 16), (64, 1, 32, 256), (4096, 4096, 32, 16)])
def test_work_space_for_the_largest_step_does_for_smaller_ones(heads, kvh, hd, page):
    """The bytes never fall where one of the sizes grows: a program asks once."""
    L, s = _lib.lib(), shape(n_head=heads, n_kv_head=kvh, head_dim=hd, page_size=page)
    rows, widths, takes = [0, 1, 2, 3, 7, 8, 64, 100, 511, 513, 4095, 5000, 1 << 20], [1, 5, 1023, 1024, 1025, 2048, 70000, 1 << 22], [1, 2, 16, 17, 64, 255, 256]
    for ws in (lambda r, w, t: L.jepa_amd_cache_select_work_bytes(s, 3, r, w, t), lambda r, w, t: L.jepa_amd_cache_selected_work_bytes(s, r, t)):
        for w in widths:
            for t in takes:
                sizes = [ws(r, w, t) for r in rows]
                assert sizes[0] >= 0 and sizes == sorted(sizes)
        for r in rows:
            assert [ws(r, w, 16) for w in widths] == sorted(ws(r, w, 16) for w in widths)
            assert [ws(r, 70000, t) for t in takes] == sorted(ws(r, 70000, t) for t in takes)
            assert ws(r, 1 << 22, 256) <= 64 << 20


def test_work_space_too_small_is_named():
    L = _lib.lib()
    need = L.jepa_amd_cache_select_work_bytes(shape(), 2, 3, 5000, 8)
    assert need > 0
    refused(select, str(need), width=5000, work_bytes=need - 1)
    need = L.jepa_amd_cache_selected_work_bytes(shape(), 3, 200)
    assert need > 0
    refused(attend, str(need), work_bytes=need - 1)


def test_work_space_sizes_are_refused():
    L = _lib.lib()
    for take in (0, 257, -1):
        assert L.jepa_amd_cache_select_work_bytes(shape(), 1, 1, 1, take) == -1
        assert L.jepa_amd_cache_selected_work_bytes(shape(), 1, take) == -1
    assert L.jepa_amd_cache_select_work_bytes(shape(), 1, -1, 1, 4) == -1
    assert L.jepa_amd_cache_select_work_bytes(None, 1, 1, 1, 4) == -1
    assert L.jepa_amd_cache_selected_work_bytes(None, 1, 4) == -1


@pytest.mark.parametrize("call", [rope, append, digest, select, attend])
def test_no_rows_get_as_far_as_the_device(call):
    """A call without rows has nothing to launch and refuses nothing by its pointers."""
    _lib.lib().jepa_error_reset()
    rc = call(n_rows=0)
    assert rc == 0 or "jepa_amd" not in _lib.error_text(), _lib.error_text()
