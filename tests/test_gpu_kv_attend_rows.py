"""Attention of several rows over pages, and over shared beginnings, against the formulas in 64 bits.

Tolerances.  f32: the scores are sums of D products of q in two 11-bit terms
(2^-22 of the head's largest value) in f32, which the tensor cores add with
truncation: as for one row a conversation, 4e-5 of max |v|.  The running sum of
n positions is added to n / 16 times per term with a truncation of at most
2^-23 of it, so at most 2 n / 16 * 2^-23 (n = 1500: 2.3e-5) of max |v| more:
6e-5 in all.  16-bit q and weights: q is exact (f16) or held exactly as f16
times a power of two (bf16); a weight rounds by at most 2^-11 of itself, which
moves a weighted mean of v by at most that share of max |v| (and the sum under
it is of weights before they round): 2^-11 of max |v|.  All round once to their
type at the end: half a step of the result.
"""

import math
import os
import sys

import pytest

import rpgbarenginecuda_b200 as rpg

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from test_gpu_kv import ACT, Pool, i32  # noqa: E402

TOL = {"f32": 6e-5, "f16": 6e-5 + 2.0 ** -11, "bf16": 6e-5 + 2.0 ** -11}


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def row_bounds(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def attend_rows(pool, q, counts, ends, starts=None, scale=None, act="f32", cap=0.0, slopes=None, pos=None, ws=None,
                out=None, stream=0):
    code, dt, _ = ACT[act]
    n_heads = q.shape[1] // pool.dim
    if ws is None:
        ws = torch.full((rpg.attend_rows_workspace(n_heads, pool.n_kv, pool.dim),), 255, dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
    a = [i32(row_bounds(counts)), i32(ends)] + [None if x is None else i32(x) for x in (starts, pos)]
    sl = None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    pool.kv.attend_rows(pool.pt, code, q.data_ptr(), n_heads, a[0].data_ptr(), q.shape[0], a[1].data_ptr(),
                        pool.dim ** -0.5 if scale is None else scale, out.data_ptr(), ws.data_ptr(), ws.numel(),
                        starts_ptr=a[2].data_ptr() if a[2] is not None else 0, cap=cap,
                        slopes_ptr=sl.data_ptr() if sl is not None else 0, pos_ptr=a[3].data_ptr() if a[3] is not None else 0,
                        q_stride=q.stride(0), out_stride=out.stride(0), stream=stream)
    torch.cuda.synchronize()
    return out


def formula(pool, q, counts, ends, starts=None, scale=None, cap=0.0, slopes=None, pos=None):
    """[row][q head][dim] in 64 bits."""
    n_heads, dim = q.shape[1] // pool.dim, pool.dim
    group = n_heads // pool.n_kv
    scale = dim ** -0.5 if scale is None else scale
    b = row_bounds(counts)
    outs = []
    for s, n in enumerate(counts):
        if n == 0:
            continue
        at = slice(b[s], b[s + 1])
        k, v = (pool.value[x][s].cuda().repeat_interleave(group, 0) for x in ("k", "v"))
        x = torch.einsum("rhd,hnd->hrn", q[at].double().view(n, n_heads, dim), k) * scale
        if cap:
            x = cap * torch.tanh(x / cap)
        p = torch.arange(k.shape[1], device="cuda")
        if slopes is not None:
            own = torch.tensor(pos[at], device="cuda")[:, None]
            x = x - torch.tensor(slopes, device="cuda").double()[:, None, None] * (own - p).abs()
        lo = torch.tensor(starts[at] if starts is not None else [0] * n, device="cuda")[:, None]
        hi = torch.tensor(ends[at], device="cuda")[:, None]
        x = x.masked_fill(~((p >= lo) & (p < hi)), -math.inf)
        w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        w = torch.where((hi > lo), w, 0.0)
        outs.append(torch.einsum("hrn,hnd->rhd", w, v).reshape(n, -1))
    return torch.cat(outs)


def close(out, want, pool, act, tol=None):
    largest = max(float(x.abs().max()) for x in pool.value["v"] if x.numel())
    out, half = out.double(), ACT[act][2]
    assert bool(torch.isfinite(out).all())
    off = (out - want).abs() - half * want.abs()
    assert float(off.max()) <= (tol or TOL[act]) * largest, (float(off.max()), largest)


def masks(kind, at, count, total, span):
    pos = [at + i for i in range(count)]
    start, end = [0] * count, [p + 1 for p in pos]
    if kind == "window":
        start = [max(0, e - span) for e in end]
    elif kind == "documents":
        start = [p // span * span for p in pos]
    elif kind == "prefix":
        end = [max(e, min(span, total)) for e in end]
    return pos, start, end


def problem(kind, heads, n_kv, dim, act, page, counts, ats, mask="causal", span=0, order="page-head-pos", seed=0):
    lens = [a + c for a, c in zip(ats, counts)]
    pool = Pool(kind, lens, page, n_kv, dim, seed=seed, order=order)
    pos, starts, ends = [], [], []
    for a, c, n in zip(ats, counts, lens):
        x = masks(mask, a, c, n, span)
        pos += x[0]
        starts += x[1]
        ends += x[2]
    q = (2.0 * randn(sum(counts), heads * dim, seed=seed + 1)).to(ACT[act][1]).cuda()
    return pool, q, pos, (starts if mask in ("window", "documents") else None), ends


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,dim", [(2, 2, 128), (8, 2, 128), (12, 2, 64)])
def test_prompts(kind, act, heads, n_kv, dim):
    counts, ats = [300, 1, 17, 0, 64, 129], [0, 0, 5, 9, 200, 77]
    pool, q, _, starts, ends = problem(kind, heads, n_kv, dim, act, 16, counts, ats)
    out = attend_rows(pool, q, counts, ends, starts, act=act)
    close(out, formula(pool, q, counts, ends, starts), pool, act)


@pytest.mark.parametrize("mask,span", [("window", 1), ("window", 50), ("window", 1000), ("documents", 1), ("documents", 37),
                                       ("documents", 128), ("prefix", 40), ("prefix", 3000)])
@pytest.mark.parametrize("kind,act", [("f16", "f16"), ("f16", "f32"), ("q8", "bf16"), ("q4", "f32")])
def test_masks(mask, span, kind, act):
    counts, ats = [260, 33, 200], [0, 90, 1]
    pool, q, _, starts, ends = problem(kind, 4, 2, 128, act, 32, counts, ats, mask, span)
    out = attend_rows(pool, q, counts, ends, starts, act=act)
    close(out, formula(pool, q, counts, ends, starts), pool, act)


@pytest.mark.parametrize("kind,act", [("f16", "f16"), ("f16", "f32"), ("q8", "f32"), ("q4", "bf16")])
@pytest.mark.parametrize("cap,bias,dim", [(5.0, False, 128), (0.0, True, 128), (20.0, True, 128), (20.0, True, 64)])
def test_capped_and_biased_scores(kind, act, cap, bias, dim):
    counts, ats = [190, 40], [30, 300]
    pool, q, pos, starts, ends = problem(kind, 6, 2, dim, act, 16, counts, ats, "window", 150)
    slopes = [2.0 ** -(i + 1) for i in range(6)] if bias else None
    kw = dict(cap=cap, slopes=slopes, pos=pos if bias else None)
    out = attend_rows(pool, q, counts, ends, starts, act=act, **kw)
    close(out, formula(pool, q, counts, ends, starts, **kw), pool, act)


@pytest.mark.parametrize("page,order", [(16, "padded"), (16, "page-pos-head"), (128, "padded"), (4096, "page-head-pos")])
@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
def test_pages_and_strides(page, order, kind):
    counts, ats = [140, 70], [13, 200]
    pool, q, _, starts, ends = problem(kind, 4, 2, 128, "f16", page, counts, ats, order=order)
    wide = torch.zeros(q.shape[0], q.shape[1] + 24, dtype=q.dtype, device="cuda")
    wide[:, :q.shape[1]] = q
    out = torch.full((q.shape[0], q.shape[1] + 8), 7.0, dtype=q.dtype, device="cuda")
    attend_rows(pool, wide[:, :q.shape[1]], counts, ends, starts, act="f16", out=out[:, :q.shape[1]])
    close(out[:, :q.shape[1]], formula(pool, q, counts, ends), pool, "f16")
    assert bool((out[:, q.shape[1]:] == 7.0).all())


@pytest.mark.parametrize("page", [32, 64, 256])
@pytest.mark.parametrize("mask,span", [("causal", 0), ("window", 100), ("documents", 90), ("prefix", 700)])
@pytest.mark.parametrize("heads,dim,act", [(4, 128, "f16"), (8, 64, "bf16"), (4, 128, "f32"), (2, 64, "f32")])
def test_pages_that_hold_a_whole_step(page, mask, span, heads, dim, act):
    # one tile of rows and two, in turn; ranges that begin and end inside a step
    counts, ats = [70, 300, 1, 129, 64, 5], [500, 0, 640, 63, 64, 129]
    pool, q, _, starts, ends = problem("f16", heads, 2, dim, act, page, counts, ats, mask, span)
    out = attend_rows(pool, q, counts, ends, starts, act=act)
    close(out, formula(pool, q, counts, ends, starts), pool, act)


@pytest.mark.parametrize("kind,act", [("f16", "f32"), ("f16", "f16"), ("q8", "f32"), ("q8", "bf16"), ("q4", "f16")])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_rise_step_after_step(kind, act, dim):
    # by 32 to 128 over 64 positions, so that the largest one so far is left behind at every step
    counts, ats = [200, 33], [400, 900]
    pool, q, pos, starts, ends = problem(kind, 4, 2, dim, act, 64, counts, ats)
    kw = dict(slopes=[0.5, 1.0, 2.0, 0.7], pos=pos)
    out = attend_rows(pool, q, counts, ends, starts, act=act, **kw)
    close(out, formula(pool, q, counts, ends, starts, **kw), pool, act)


@pytest.mark.parametrize("heads,n_kv", [(1, 1), (5, 1), (40, 1), (96, 3), (300, 1)])
@pytest.mark.parametrize("act", ["f16", "f32"])
def test_many_queries_of_a_kv_head(heads, n_kv, act):
    counts, ats = [30, 3], [50, 0]
    pool, q, _, starts, ends = problem("f16", heads, n_kv, 64, act, 16, counts, ats)
    out = attend_rows(pool, q, counts, ends, starts, act=act)
    close(out, formula(pool, q, counts, ends, starts), pool, act)


@pytest.mark.parametrize("kind,act", [("f16", "f32"), ("f16", "f16"), ("q8", "f32"), ("q4", "f16")])
@pytest.mark.parametrize("count,at", [(1, 5000), (3, 3333), (64, 1500), (700, 800)])
def test_lengths_split_over_the_gpu(kind, act, count, at):
    pool, q, _, starts, ends = problem(kind, 4, 2, 128, act, 64, [count], [at])
    out = attend_rows(pool, q, [count], ends, starts, act=act)
    # (n = 5001: 2 n / 16 * 2^-23 = 7.5e-5 where one block has it all)
    close(out, formula(pool, q, [count], ends, starts), pool, act, tol=TOL[act] + 7e-5)


def test_many_conversations_of_few_rows():
    n = 700
    counts = [(i * 7) % 4 for i in range(n)]
    ats = [(i * 13) % 60 for i in range(n)]
    pool, q, _, starts, ends = problem("f16", 4, 2, 64, "f16", 16, counts, [a + (c == 0) for a, c in zip(ats, counts)])
    out = attend_rows(pool, q, counts, ends, starts, act="f16")
    close(out, formula(pool, q, counts, ends, starts), pool, "f16")


def test_rows_that_see_nothing_and_rows_of_no_conversation():
    pool = Pool("f16", [50, 20], 16, 2, 128)
    q = randn(12, 4 * 128).half().cuda()
    ends, starts = [0, 0, 3, 50, 50, 0, 20, 20, 20, 0, 0, 0], [0, 0, 3, 10, 50, 0, 0, 19, 20, 0, 0, 0]
    ends_call = [0, 0, 3, 50, 50] + [0, 20, 20, 20] + [9, 9, 9]  # rows 9 .. 11 belong to nobody
    out = attend_rows(pool, q, [5, 4], ends_call, starts, act="f16")
    want = formula(pool, q[:9], [5, 4], ends[:9], starts[:9])
    close(out[:9], want, pool, "f16")
    for r in (0, 1, 2, 4, 5, 8):
        assert bool((out[r] == 0).all())
    assert bool((out[9:] == 7.0).all())


def test_bad_pages_positions_past_the_table_and_bounds_that_decrease_give_nan():
    counts, ats = [40, 40], [0, 60]
    pool, q, _, _, ends = problem("f16", 4, 2, 128, "f16", 16, counts, ats)
    want = formula(pool, q, counts, ends)
    pool.dev_table[0, 1] = -1  # positions 16 .. 31 of the first conversation
    pool.dev_table[1, 3] = pool.n_pages
    out = attend_rows(pool, q, counts, ends, act="f16")
    bad = torch.tensor([e > 16 for e in ends[:40]] + [True] * 40, device="cuda")
    assert bool(out[bad].isnan().all())
    close(out[~bad], want[~bad], pool, "f16")
    starts = [0] * 40 + [64] * 40  # behind the bad page of the second
    out = attend_rows(pool, q, counts, ends, starts, act="f16")
    close(out[40:], formula(pool, q, counts, ends, starts)[40:], pool, "f16")
    pool.dev_table.copy_(pool.table)
    far = list(ends)
    far[-1] = pool.width * 16 + 1
    out = attend_rows(pool, q, counts, far, act="f16")
    assert bool(out[-1].isnan().all())
    close(out[:-1], want[:-1], pool, "f16")


def test_bounds_that_decrease_give_nan_and_lists_without_rows_nothing():
    counts, ats = [50, 30], [10, 0]
    pool, q, _, _, ends = problem("f16", 4, 2, 128, "f16", 16, counts, ats)
    want = formula(pool, q, counts, ends)
    odd = list(ends)
    odd[49] = 30  # the last of the first conversation sees less than the others before it
    out = attend_rows(pool, q, counts, odd, act="f16")
    bad = torch.tensor([e > 30 for e in odd[:50]] + [False] * 30, device="cuda")
    assert bool(out[bad].isnan().all())
    good = ~bad
    good[49] = False  # (it sees something else now)
    close(out[good], want[good], pool, "f16")
    out = attend_rows(pool, q, [0, 0], ends, act="f16")
    assert bool((out == 7.0).all())


def test_on_another_stream_behind_what_fills_its_inputs():
    counts, ats = [90, 40], [10, 0]
    pool, q, _, _, ends = problem("q8", 4, 2, 128, "f16", 16, counts, ats)
    want = formula(pool, q, counts, ends)
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    out = torch.full_like(q, 7.0)
    ws = torch.empty(rpg.attend_rows_workspace(4, 2, 128), dtype=torch.uint8, device="cuda")
    rows, e = i32(row_bounds(counts)), i32(ends)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big * 1e-3
        late.copy_(q)
        pool.kv.attend_rows(pool.pt, rpg.F16, late.data_ptr(), 4, rows.data_ptr(), q.shape[0], e.data_ptr(), 128 ** -0.5,
                            out.data_ptr(), ws.data_ptr(), ws.numel(), stream=side.cuda_stream)
        late.zero_()
    torch.cuda.synchronize()
    close(out, want, pool, "f16")


def test_two_calls_at_once():
    # each with a workspace of its own, on streams of their own
    problems = [problem(kind, 8, 2, 128, act, 16, [300, 70], [400, 5], seed=i)
                for i, (kind, act) in enumerate((("f16", "f16"), ("q8", "f32"), ("f16", "f32")))]
    alone = [attend_rows(pool, q, [300, 70], ends, act="f32" if q.dtype == torch.float32 else "f16")
             for pool, q, _, _, ends in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    outs = [torch.empty_like(q) for _, q, *_ in problems]
    ws = [torch.empty(rpg.attend_rows_workspace(8, 2, 128), dtype=torch.uint8, device="cuda") for _ in problems]
    args = [(i32([0, 300, 370]), i32(ends)) for *_, ends in problems]
    torch.cuda.synchronize()
    for _ in range(20):
        for (pool, q, *_), s, o, w, (r, e) in zip(problems, streams, outs, ws, args):
            pool.kv.attend_rows(pool.pt, rpg.F32 if q.dtype == torch.float32 else rpg.F16, q.data_ptr(), 8, r.data_ptr(),
                                370, e.data_ptr(), 128 ** -0.5, o.data_ptr(), w.data_ptr(), w.numel(), stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for a, o in zip(alone, outs))


def nonfinite(pool, name, s, h, pos, dim, value):
    page, at = int(pool.table[s, pos // pool.page]), pos % pool.page
    pool.mem[name][page, h, at, dim] = value
    pool.value[name][s][h, pos, dim] = value


@pytest.mark.parametrize("act", ["f32", "f16"])
def test_infinities_and_nan_in_the_cache(act):
    counts, ats = [150, 70], [10, 0]
    pool, q, _, _, ends = problem("f16", 4, 2, 128, act, 16, counts, ats)
    base = formula(pool, q, counts, ends)
    nonfinite(pool, "v", 0, 0, 100, 5, math.inf)   # rows that see position 100: dimension 5 infinite
    nonfinite(pool, "v", 1, 1, 30, 7, math.nan)
    nonfinite(pool, "k", 1, 0, 40, 3, math.inf)    # scores of plus or minus infinity
    out = attend_rows(pool, q, counts, ends, act=act)
    want = base.view(-1, 4, 128).clone()
    sees = torch.tensor(ends, device="cuda")
    first = torch.arange(len(ends), device="cuda") < counts[0]
    want[first & (sees > 100), :2, 5] = math.inf
    want[~first & (sees > 30), 2:, 7] = math.nan
    late = ~first & (sees > 40)
    qv = q.view(-1, 4, 128)
    plus = late[:, None] & (qv[:, :2, 3] > 0)
    pool.value["k"][1][0, 40] = 0
    minus = late[:, None] & (qv[:, :2, 3] < 0)
    # minus infinity drops the position
    k, v = pool.value["k"][1][0].cuda(), pool.value["v"][1][0].cuda()
    for r in torch.nonzero(late)[:, 0].tolist():
        for h in range(2):
            n = ends[r]
            keep = [i for i in range(n) if i != 40]
            w = torch.softmax((k[keep] @ qv[r, h].double()) * 128 ** -0.5, 0)
            want[r, h] = w @ v[keep]
    mask = torch.zeros(len(ends), 4, dtype=torch.bool, device="cuda")
    mask[:, :2] = plus
    assert bool((minus | ~late[:, None] | plus).all())
    got = out.double().view(-1, 4, 128)
    assert bool(got[mask].isnan().all())
    want, got = want[~mask], got[~mask]
    assert bool((want.isnan() == got.isnan()).all()) and bool((want.isinf() == got.isinf()).all())
    fine = want.isfinite()
    assert float(((got - want).abs() - ACT[act][2] * want.abs())[fine].max()) <= TOL[act] * 6


def test_queries_that_are_not_finite():
    counts, ats = [90], [10]
    pool, q, _, _, ends = problem("f16", 4, 2, 128, "f32", 16, counts, ats)
    want = formula(pool, q, counts, ends).view(-1, 4, 128)
    q.view(-1, 4, 128)[5, 1, 3] = math.nan
    q.view(-1, 4, 128)[80, 2, 120] = -math.inf
    out = attend_rows(pool, q, counts, ends).view(-1, 4, 128)
    bad = torch.zeros(90, 4, dtype=torch.bool, device="cuda")
    bad[5, 1] = bad[80, 2] = True
    assert bool(out[bad].isnan().all())
    close(out[~bad], want[~bad], pool, "f32")


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_large_and_small_queries_and_scales(kind):
    counts, ats = [100], [30]
    for factor, scale in ((1e-30, 1e29), (1e30, 1e-31), (1.0, 0.0), (1.0, -0.1), (2.0, 3.0)):
        pool, q, _, _, ends = problem(kind, 4, 2, 128, "f32", 16, counts, ats)
        q = q * factor
        out = attend_rows(pool, q, counts, ends, scale=scale)
        # scores of up to 2 * 2 * 128 * 3 in size err by that times 2^-22
        close(out, formula(pool, q, counts, ends, scale=scale), pool, "f32", tol=1.5e-3 if scale == 3.0 else 4e-4)


def test_far_offsets_in_a_large_pool():
    # pages behind 2^32 bytes of a pool
    n_kv, dim, page = 2, 128, 16
    n_pages = (5 << 30) // (n_kv * page * dim * 2)
    k = torch.zeros(n_pages, n_kv, page, dim, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    ids = [n_pages - 1, 3, n_pages - 7, n_pages // 2]
    for name, m in (("k", k), ("v", v)):
        m[ids] = randn(4, n_kv, page, dim, seed=len(name) + (name == "v")).half().cuda()
    table = i32(ids)
    kv = rpg.PagedKv(rpg.KV_F16, dim, n_kv, page, n_pages, k.data_ptr(), v.data_ptr())
    q = randn(60, 4 * dim, seed=3).half().cuda()
    out, ends, rows = torch.empty_like(q), i32(range(1, 61)), i32([0, 60])
    ws = torch.empty(rpg.attend_rows_workspace(4, n_kv, dim), dtype=torch.uint8, device="cuda")
    kv.attend_rows(rpg.PageTable(table.data_ptr(), 1, 4), rpg.F16, q.data_ptr(), 4, rows.data_ptr(), 60, ends.data_ptr(),
                   dim ** -0.5, out.data_ptr(), ws.data_ptr(), ws.numel())
    kk, vv = (m[ids].double().transpose(0, 1).reshape(n_kv, 64, dim).repeat_interleave(2, 0)[:, :60] for m in (k, v))
    x = torch.einsum("rhd,hnd->hrn", q.double().view(60, 4, dim), kk) * dim ** -0.5
    x = x.masked_fill(torch.ones(60, 60, device="cuda").triu(1).bool(), -math.inf)
    want = torch.einsum("hrn,hnd->rhd", torch.softmax(x, -1), vv).reshape(60, -1)
    assert float((out.double() - want).abs().max()) <= TOL["f16"] * 6


def test_repeats_bit_for_bit_on_any_workspace_and_in_graphs():
    counts, ats = [500, 9, 130], [700, 2000, 0]
    pool, q, _, _, ends = problem("f16", 8, 2, 128, "f32", 16, counts, ats)
    first = attend_rows(pool, q, counts, ends)
    ws = torch.randint(0, 255, (rpg.attend_rows_workspace(8, 2, 128),), dtype=torch.uint8, device="cuda")
    assert torch.equal(first, attend_rows(pool, q, counts, ends, ws=ws))
    rows, e = i32(row_bounds(counts)), i32(ends)
    out, other = torch.zeros_like(q), torch.zeros_like(q)
    small = q[:3].clone()
    few, few_ends = i32([0, 1, 2, 3]), i32([5, 6, 7])
    stream = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):  # two graphs on one workspace, one after the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            s = torch.cuda.current_stream().cuda_stream
            pool.kv.attend_rows(pool.pt, rpg.F32, small.data_ptr(), 8, few.data_ptr(), 3, few_ends.data_ptr(), 0.1,
                                other.data_ptr(), ws.data_ptr(), ws.numel(), stream=s)
            pool.kv.attend_rows(pool.pt, rpg.F32, q.data_ptr(), 8, rows.data_ptr(), q.shape[0], e.data_ptr(),
                                128 ** -0.5, out.data_ptr(), ws.data_ptr(), ws.numel(), stream=s)
        graphs.append(g)
    for g in graphs * 2:
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    q.copy_(q * 0.5)  # new queries, fewer rows: a replay follows the device's arrays
    rows.copy_(i32([0, 100, 100, 200]))
    e.copy_(i32([700 + i for i in range(1, 101)] + list(range(1, 101)) + [0] * (len(ends) - 200)))
    out.fill_(7.0)
    graphs[0].replay()
    torch.cuda.synchronize()
    want = formula(pool, q[:200], [100, 0, 100], e.tolist()[:200])
    close(out[:200], want, pool, "f32")
    assert bool((out[200:] == 7.0).all())


# ---------------------------------------------------------------- shared beginnings


def share(pool, groups, prefix):
    """Makes the conversations of each group begin alike: the same pages, and a copy where a page is shared in part."""
    for (a, b), n in zip(groups, prefix):
        whole, rest = n // pool.page, n % pool.page
        for c in range(a + 1, b):
            pool.table[c, :whole] = pool.table[a, :whole]
            if rest:
                src, dst = int(pool.table[a, whole]), int(pool.table[c, whole])
                for mem in (pool.mem, pool.scale):
                    for name in mem:
                        mem[name][dst, :, :rest] = mem[name][src, :, :rest]
            for name in ("k", "v"):
                pool.value[name][c][:, :n] = pool.value[name][a][:, :n]
    pool.dev_table.copy_(pool.table)


def attend_shared(pool, q, groups, prefix, lens, starts=None, act="f32", ws=None, out=None, bounds=None):
    code, dt, _ = ACT[act]
    n_heads = q.shape[1] // pool.dim
    if ws is None:
        ws = torch.zeros(rpg.attend_shared_workspace(n_heads, pool.n_kv, pool.dim, q.shape[0]), dtype=torch.uint8,
                         device="cuda")
    if out is None:
        out = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
    per = [0] * q.shape[0]
    for (a, b), n in zip(groups, prefix):
        per[a:b] = [n] * (b - a)
    x = [i32(lens), i32(bounds or [g[0] for g in groups] + [groups[-1][1]]), i32(per), None if starts is None else i32(starts)]
    torch.cuda.synchronize()
    pool.kv.attend_shared(pool.pt, code, q.data_ptr(), n_heads, x[0].data_ptr(), x[1].data_ptr(), len(groups),
                          x[2].data_ptr(), pool.dim ** -0.5, out.data_ptr(), ws.data_ptr(), ws.numel(),
                          starts_ptr=x[3].data_ptr() if x[3] is not None else 0, q_stride=q.stride(0),
                          out_stride=out.stride(0))
    torch.cuda.synchronize()
    return out


def shared_problem(kind, heads, n_kv, dim, act, page, sizes, prefix, tails, seed=0):
    groups, a = [], 0
    for n in sizes:
        groups.append((a, a + n))
        a += n
    lens = []
    for (b, e), n in zip(groups, prefix):
        lens += [n + tails[i % len(tails)] for i in range(b, e)]
    pool = Pool(kind, lens, page, n_kv, dim, seed=seed)
    share(pool, groups, prefix)
    q = (2.0 * randn(a, heads * dim, seed=seed + 1)).to(ACT[act][1]).cuda()
    return pool, q, groups, lens


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,n_kv,dim", [(2, 2, 128), (8, 2, 128), (12, 2, 64), (10, 1, 128)])
def test_shared(kind, act, heads, n_kv, dim):
    sizes, prefix = [7, 1, 40, 2, 3], [300, 64, 130, 0, 5]
    pool, q, groups, lens = shared_problem(kind, heads, n_kv, dim, act, 16, sizes, prefix, [1, 0, 40, 7, 100])
    out = attend_shared(pool, q, groups, prefix, lens, act=act)
    close(out, formula(pool, q, [1] * len(lens), lens), pool, act)


@pytest.mark.parametrize("size,prefix", [(1, 4000), (3, 3000), (128, 1000), (129, 200), (300, 77)])
@pytest.mark.parametrize("kind,act", [("f16", "f32"), ("f16", "bf16"), ("q8", "f16")])
def test_shared_sizes(size, prefix, kind, act):
    pool, q, groups, lens = shared_problem(kind, 4, 2, 128, act, 32, [size], [prefix], [3, 20])
    out = attend_shared(pool, q, groups, [prefix], lens, act=act)
    # (n = 4000: 2 n / 16 * 2^-23 = 6e-5)
    close(out, formula(pool, q, [1] * len(lens), lens), pool, act, tol=TOL[act] + 6e-5)


def test_shared_windows_short_conversations_and_strangers():
    sizes, prefix = [6, 6], [200, 100]
    pool, q, groups, lens = shared_problem("f16", 4, 2, 128, "f16", 16, sizes, prefix, [30])
    full = list(lens)
    lens = [230, 150, 200, 0, 1, 230, 130, 130, 130, 100, 50, 130]  # some end inside the common positions
    starts = [0, 20, 199, 0, 0, 229, 99, 100, 129, 0, 50, 7]
    out = attend_shared(pool, q, groups, prefix, lens, starts, act="f16")
    close(out, formula(pool, q, [1] * 12, lens, starts), pool, "f16")
    assert bool((out[3] == 0).all()) and bool((out[10] == 0).all())
    # conversations before the first group and behind the last are left as they are
    out = attend_shared(pool, q, groups[:1], prefix[:1], full, act="f16", bounds=[1, 5])
    close(out[1:5], formula(pool, q, [1] * 12, full)[1:5], pool, "f16")
    assert bool((out[0] == 7.0).all()) and bool((out[5:] == 7.0).all())


def test_shared_bad_pages_lengths_and_prefixes_give_nan():
    sizes, prefix = [5, 4], [100, 60]
    pool, q, groups, lens = shared_problem("f16", 4, 2, 128, "f16", 16, sizes, prefix, [40])
    want = formula(pool, q, [1] * 9, lens)
    pool.dev_table[2, 8] = -1                # a page of its own (positions 128 ..)
    pool.dev_table[5, 1] = pool.n_pages + 5  # of the first of the second group: all of the group sees it
    out = attend_shared(pool, q, groups, prefix, lens, act="f16")
    bad = [2, 5, 6, 7, 8]
    assert bool(out[bad].isnan().all())
    close(out[[0, 1, 3, 4]], want[[0, 1, 3, 4]], pool, "f16")
    pool.dev_table.copy_(pool.table)
    lens[1] = pool.width * 16 + 1
    out = attend_shared(pool, q, groups, prefix, lens, act="f16")
    assert bool(out[1].isnan().all())
    close(out[2:], want[2:], pool, "f16")


def test_shared_prefixes_that_differ():
    # shorter than the group's first: the rest is the conversation's own; longer: NaN
    pool, q, groups, lens = shared_problem("f16", 4, 2, 128, "f16", 16, [4], [100], [40])
    want = formula(pool, q, [1] * 4, lens)
    lens_dev, g, per = i32(lens), i32([0, 4]), i32([100, 60, 0, 101])
    ws = torch.zeros(rpg.attend_shared_workspace(4, 2, 128, 4), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    pool.kv.attend_shared(pool.pt, rpg.F16, q.data_ptr(), 4, lens_dev.data_ptr(), g.data_ptr(), 1, per.data_ptr(), 128 ** -0.5,
                          out.data_ptr(), ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    close(out[:3], want[:3], pool, "f16")
    assert bool(out[3].isnan().all())


def test_shared_in_a_graph_with_lengths_that_grow():
    pool, q, groups, lens = shared_problem("q8", 8, 2, 128, "f32", 16, [20, 11], [150, 70], [30])
    short = [n - 10 for n in lens]
    n, g, per = i32(short), i32([0, 20, 31]), i32([150] * 20 + [70] * 11)
    ws = torch.zeros(rpg.attend_shared_workspace(8, 2, 128, 31), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pool.kv.attend_shared(pool.pt, rpg.F32, q.data_ptr(), 8, n.data_ptr(), g.data_ptr(), 2, per.data_ptr(), 128 ** -0.5,
                              out.data_ptr(), ws.data_ptr(), ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    for k in (0, 3, 10):
        n.copy_(i32([x + k for x in short]))
        graph.replay()
        torch.cuda.synchronize()
        close(out, formula(pool, q, [1] * 31, [x + k for x in short]), pool, "f32")


def test_shared_infinities():
    pool, q, groups, lens = shared_problem("f16", 4, 2, 128, "f32", 16, [6], [100], [20])
    want = formula(pool, q, [1] * 6, lens).view(6, 4, 128)
    page = int(pool.table[0, 3])
    pool.mem["v"][page, 0, 4, 9] = math.inf       # seen by all
    pool.mem["v"][int(pool.table[2, 7]), 1, 0, 2] = -math.inf  # position 112 of conversation 2
    out = attend_shared(pool, q, groups, [100], lens).view(6, 4, 128)
    want[:, :2, 9] = math.inf
    want[2, 2:, 2] = -math.inf
    fine = want.isfinite()
    assert torch.equal(out.double()[~fine], want[~fine])
    assert float((out.double() - want)[fine].abs().max()) <= TOL["f32"] * 5


def test_shared_is_attend_on_one_workspace_for_all_batches():
    ws = torch.zeros(rpg.attend_shared_workspace(8, 2, 128, 64), dtype=torch.uint8, device="cuda")
    for sizes, prefix in (([40, 24], [500, 33]), ([3], [2000]), ([64], [16]), ([1, 1, 1], [7, 0, 300])):
        pool, q, groups, lens = shared_problem("q8", 8, 2, 128, "f16", 16, sizes, prefix, [5, 60], seed=len(sizes))
        a = attend_shared(pool, q, groups, prefix, lens, act="f16", ws=ws)
        b = attend_shared(pool, q, groups, prefix, lens, act="f16", ws=ws)
        assert torch.equal(a, b)
        out = torch.empty_like(q)
        w = torch.zeros(rpg.attend_workspace(8, 2, 128), dtype=torch.uint8, device="cuda")
        n = i32(lens)
        pool.kv.attend(pool.pt, rpg.F16, q.data_ptr(), 8, n.data_ptr(), 128 ** -0.5, out.data_ptr(), w.data_ptr(), w.numel())
        close(a, out.double(), pool, "f16", tol=2 * TOL["f16"])
