"""Paged key-value cache entry points on the CPU: refusals, workspace sizes, rotation table."""

import ctypes

import numpy as np
import pytest

import rpgbarenginecuda_b200 as rpg
from rpgbarenginecuda_b200 import EngineError, _lib

FAKE = 1 << 20  # a 16-byte aligned address that no refused call may touch


def cache(kind=rpg.KV_Q8, **kw):
    a = dict(kv_type=kind, head_dim=128, n_kv=8, page_size=16, n_pages=4, k_ptr=FAKE, v_ptr=FAKE, k_scale_ptr=FAKE,
             v_scale_ptr=FAKE)
    a.update(kw)
    return rpg.PagedKv(**a)


def attend(kv, table=None, **kw):
    a = dict(table=table or rpg.PageTable(FAKE, 2, 4), dtype=rpg.F32, q_ptr=FAKE, n_heads=16, lens_ptr=FAKE, scale=0.1,
             out_ptr=FAKE, workspace_ptr=FAKE, workspace_bytes=1 << 30)
    a.update(kw)
    kv.attend(**a)


def append(kv, table=None, **kw):
    a = dict(table=table or rpg.PageTable(FAKE, 2, 4), rotary=None, dtype=rpg.F32, qkv_ptr=FAKE, n_heads=16,
             pos_ptr=FAKE, n_tok=2, q_out_ptr=FAKE)
    a.update(kw)
    kv.append(**a)


def gather(kv, table=None, **kw):
    a = dict(table=table or rpg.PageTable(FAKE, 2, 4), dtype=rpg.F32, pos_ptr=FAKE, n_tok=2, k_out_ptr=FAKE,
             v_out_ptr=FAKE)
    a.update(kw)
    kv.gather(**a)


@pytest.mark.parametrize("call", [attend, append, gather])
@pytest.mark.parametrize("bad,why", [
    (dict(kind=7), "type"), (dict(head_dim=96), "head_dim"), (dict(n_kv=0), "KV head"), (dict(n_pages=0), "page count"),
    (dict(page_size=8), "page size"), (dict(page_size=48), "page size"), (dict(page_size=8192), "page size"),
    (dict(k_ptr=0), "NULL"), (dict(v_ptr=FAKE + 8), "aligned"), (dict(k_scale_ptr=0), "scale"),
    (dict(v_scale_ptr=FAKE + 2), "aligned"), (dict(pos_stride=64), "stride"), (dict(pos_stride=136), "stride"),
    (dict(head_stride=-2048), "stride"), (dict(scale_head_stride=16), "scale stride"),
])
def test_bad_caches_are_refused(call, bad, why):
    with pytest.raises(EngineError, match=why):
        call(cache(**bad))


@pytest.mark.parametrize("call", [attend, append, gather])
def test_bad_tables_and_types_are_refused(call):
    for t in (rpg.PageTable(0, 2, 4), rpg.PageTable(FAKE + 2, 2, 4), rpg.PageTable(FAKE, -1, 4),
              rpg.PageTable(FAKE, 2, 0), rpg.PageTable(FAKE, 2, 4, 3), rpg.PageTable(FAKE, 2, 1 << 27), rpg.PageTable(FAKE, (1 << 20) + 1, 4)):
        with pytest.raises(EngineError):
            call(cache(), table=t)
    with pytest.raises(EngineError, match="element type"):
        call(cache(), dtype=3)


@pytest.mark.parametrize("bad", [
    dict(q_ptr=0), dict(out_ptr=0), dict(q_ptr=FAKE + 4), dict(q_stride=2047), dict(q_stride=1024), dict(out_stride=2050),
    dict(n_heads=12), dict(n_heads=0), dict(lens_ptr=0), dict(workspace_ptr=0), dict(workspace_bytes=1000),
    dict(workspace_ptr=FAKE + 16), dict(scale=float("nan")), dict(scale=float("inf")),
])
def test_bad_attend_arguments_are_refused(bad):
    with pytest.raises(EngineError):
        attend(cache(), **bad)


@pytest.mark.parametrize("bad", [
    dict(qkv_ptr=0), dict(qkv_ptr=FAKE + 8), dict(qkv_stride=4095), dict(n_heads=-1), dict(pos_ptr=0), dict(n_tok=-1),
    dict(n_tok=3), dict(q_out_ptr=FAKE + 4), dict(n_heads=0, q_out_ptr=FAKE),
    dict(rotary=rpg.Rotary(FAKE, 0)), dict(rotary=rpg.Rotary(FAKE + 4, 16)), dict(rotary=rpg.Rotary(q_norm_ptr=FAKE + 4)),
    dict(rotary=rpg.Rotary(k_norm_ptr=FAKE, eps=-1.0)), dict(rotary=rpg.Rotary(k_norm_ptr=FAKE, eps=float("nan"))),
])
def test_bad_append_arguments_are_refused(bad):
    with pytest.raises(EngineError):
        append(cache(), **bad)


@pytest.mark.parametrize("bad", [dict(k_out_ptr=0, v_out_ptr=0), dict(k_out_ptr=FAKE + 4), dict(out_stride=1000),
                                 dict(pos_ptr=0), dict(n_tok=-1), dict(n_tok=3), dict(n_tok=1 << 40, seq_ptr=FAKE)])
def test_bad_gather_arguments_are_refused(bad):
    with pytest.raises(EngineError):
        gather(cache(), **bad)


def test_null_descriptors_are_refused():
    lib = _lib.load_engine()
    kv, t = cache(), rpg.PageTable(FAKE, 2, 4)
    assert lib.rpgb_kv_gather(None, t._ref, 0, None, FAKE, 2, FAKE, FAKE, 1024, None) < 0
    assert b"NULL" in lib.rpgb_last_error()
    assert lib.rpgb_kv_gather(kv._ref, None, 0, None, FAKE, 2, FAKE, FAKE, 1024, None) < 0
    assert b"NULL" in lib.rpgb_last_error()


def test_nothing_to_do_is_no_error():
    append(cache(), n_tok=0)
    gather(cache(), n_tok=0)
    attend(cache(), table=rpg.PageTable(0, 0, 4))


def test_workspace_size():
    n = rpg.attend_workspace(16, 8, 128)
    assert 0 < n <= 16 << 20
    assert rpg.attend_workspace(64, 8, 128) > n > rpg.attend_workspace(16, 8, 64)
    for bad in ((0, 8, 128), (12, 8, 128), (16, 0, 128), (16, 8, 80)):
        with pytest.raises(EngineError):
            rpg.attend_workspace(*bad)


def test_rope_table():
    t = rpg.rope_table(100, 128, 1e6)
    assert t.shape == (100, 128) and t.dtype == np.float32
    ang = 57 * 1e6 ** (-2 * 11 / 128)
    assert abs(t[57, 11] - np.cos(ang)) < 1e-7 and abs(t[57, 64 + 11] - np.sin(ang)) < 1e-7


def test_descriptors_match_the_header():
    """Sizes of the C structs on a 64-bit host: six int32, four pointers, five int64; and so on."""
    assert ctypes.sizeof(_lib.KvPagesDesc) == 24 + 32 + 40
    assert ctypes.sizeof(_lib.KvTableDesc) == 24
    assert ctypes.sizeof(_lib.KvRotaryDesc) == 32
