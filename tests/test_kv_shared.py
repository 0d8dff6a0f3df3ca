"""Attention of several rows, over shared beginnings, and sampling of a batch on the CPU: refusals, workspace sizes."""

import pytest

import rpgbarenginecuda_b200 as rpg
from rpgbarenginecuda_b200 import EngineError
from test_kv_paged import FAKE, cache


def rows(kv, table=None, **kw):
    a = dict(table=table or rpg.PageTable(FAKE, 2, 4), dtype=rpg.F32, q_ptr=FAKE, n_heads=16, rows_ptr=FAKE, n_rows=5,
             ends_ptr=FAKE, scale=0.1, out_ptr=FAKE, workspace_ptr=FAKE, workspace_bytes=1 << 31)
    a.update(kw)
    kv.attend_rows(**a)


def shared(kv, table=None, **kw):
    a = dict(table=table or rpg.PageTable(FAKE, 2, 4), dtype=rpg.F32, q_ptr=FAKE, n_heads=16, lens_ptr=FAKE,
             groups_ptr=FAKE, n_groups=1, prefix_ptr=FAKE, scale=0.1, out_ptr=FAKE, workspace_ptr=FAKE,
             workspace_bytes=1 << 31)
    a.update(kw)
    kv.attend_shared(**a)


@pytest.mark.parametrize("call", [rows, shared])
@pytest.mark.parametrize("bad,why", [
    (dict(kind=7), "type"), (dict(head_dim=96), "head_dim"), (dict(n_kv=0), "KV head"), (dict(page_size=48), "page size"),
    (dict(k_ptr=0), "NULL"), (dict(v_ptr=FAKE + 8), "aligned"), (dict(k_scale_ptr=0), "scale"), (dict(pos_stride=64), "stride"),
])
def test_bad_caches_are_refused(call, bad, why):
    with pytest.raises(EngineError, match=why):
        call(cache(**bad))


@pytest.mark.parametrize("call", [rows, shared])
@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(q_ptr=0), dict(out_ptr=0), dict(q_ptr=FAKE + 4), dict(q_stride=2047), dict(out_stride=2050),
    dict(n_heads=12), dict(n_heads=0), dict(workspace_ptr=0), dict(workspace_bytes=1000), dict(workspace_ptr=FAKE + 16),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(starts_ptr=FAKE + 2), dict(table=rpg.PageTable(0, 2, 4)),
])
def test_bad_arguments_are_refused(call, bad):
    with pytest.raises(EngineError):
        call(cache(), **bad)


@pytest.mark.parametrize("bad", [
    dict(rows_ptr=0), dict(rows_ptr=FAKE + 2), dict(ends_ptr=0), dict(ends_ptr=FAKE + 1), dict(n_rows=-1),
    dict(n_rows=(1 << 24) + 1), dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(slopes_ptr=FAKE),
    dict(slopes_ptr=FAKE + 2, pos_ptr=FAKE), dict(slopes_ptr=FAKE, pos_ptr=FAKE + 2),
])
def test_bad_rows_are_refused(bad):
    with pytest.raises(EngineError):
        rows(cache(), **bad)


@pytest.mark.parametrize("bad", [
    dict(lens_ptr=0), dict(lens_ptr=FAKE + 2), dict(groups_ptr=0), dict(groups_ptr=FAKE + 2), dict(prefix_ptr=0),
    dict(prefix_ptr=FAKE + 2), dict(n_groups=-1), dict(n_groups=(1 << 20) + 1),
])
def test_bad_groups_are_refused(bad):
    with pytest.raises(EngineError):
        shared(cache(), **bad)


def test_nothing_to_do():
    rows(cache(), n_rows=0, q_ptr=0, out_ptr=0, rows_ptr=0, ends_ptr=0, workspace_ptr=0)
    rows(cache(), table=rpg.PageTable(0, 0, 4), q_ptr=0, out_ptr=0)
    shared(cache(), n_groups=0, q_ptr=0, out_ptr=0, groups_ptr=0)
    shared(cache(), table=rpg.PageTable(0, 0, 4), q_ptr=0, out_ptr=0)
    rpg.sample_rows(0, rpg.F32, 0, 100, 0, u_ptr=FAKE)


def test_workspace_sizes():
    assert rpg.attend_rows_workspace(16, 8, 128) >= rpg.attend_rows_workspace(16, 8, 64) > 0
    n = rpg.attend_shared_workspace(16, 8, 128, 64)
    assert n > rpg.attend_shared_workspace(16, 8, 128, 1) > rpg.attend_workspace(16, 8, 128)
    for bad in ((12, 8, 128), (16, 0, 128), (16, 8, 96)):
        with pytest.raises(EngineError):
            rpg.attend_rows_workspace(*bad)
        with pytest.raises(EngineError):
            rpg.attend_shared_workspace(*bad, 4)
    for bad in (-1, (1 << 20) + 1):
        with pytest.raises(EngineError):
            rpg.attend_shared_workspace(16, 8, 128, bad)


@pytest.mark.parametrize("bad,why", [
    (dict(dtype=5), "type"), (dict(n_rows=-1), "row count"), (dict(n_rows=(1 << 24) + 1), "row count"), (dict(vocab=0), "vocabulary"), (dict(vocab=262145), "vocabulary"),
    (dict(stride=99), "stride"), (dict(u_ptr=0), "random"), (dict(u_ptr=FAKE + 2), "aligned"),
    (dict(top_k_ptr=FAKE + 1), "aligned"), (dict(logits_ptr=0), "NULL"), (dict(logits_ptr=FAKE + 2), "aligned"),
    (dict(tok_ptr=0), "NULL"), (dict(prob_ptr=FAKE + 2), "aligned"),
])
def test_bad_sampling_arguments_are_refused(bad, why):
    a = dict(logits_ptr=FAKE, dtype=rpg.F32, n_rows=2, vocab=100, tok_ptr=FAKE, u_ptr=FAKE)
    a.update(bad)
    with pytest.raises(EngineError, match=why):
        rpg.sample_rows(**a)
