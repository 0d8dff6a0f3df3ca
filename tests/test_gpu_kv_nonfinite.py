"""Infinities and NaN in the cache and in q: attend gives what the formula in f32 gives.

A score of minus infinity drops its position, one of plus infinity or NaN makes the head's row NaN, an infinite value
makes its dimension infinite (NaN where infinities of both signs meet, or where its weight is zero).  A conversation
whose scores are all minus infinity has no weights: zeros, as an empty range.  Finite results are held to the bound of
tests/test_gpu_kv.py: 4e-5 of the largest |v| (f32 sums of at most 16 terms that may truncate, |score| up to 40) and
half a unit of the output type.
"""

import pytest

import rpgbarenginecuda_b200 as rpg

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv import ACT, Pool, attend, queries  # noqa: E402

INF, NAN = float("inf"), float("nan")


def put(pool, name, i, pos, head, dim, x):
    """One value of conversation i, on the device and in the 64-bit copy."""
    pool.mem[name][int(pool.table[i, pos // pool.page]), head, pos % pool.page, dim] = x
    pool.value[name][i][head, pos, dim] = x


def formula(pool, q, i, head_of, scale):
    """Row i in 64 bits, position by position where that matters: infinities and NaN go through."""
    out = []
    for h in range(q.shape[1] // pool.dim):
        k, v = pool.value["k"][i][head_of(h)], pool.value["v"][i][head_of(h)]
        s = (q[i].double().cpu().view(-1, pool.dim)[h] * k).sum(-1) * scale
        top = s.amax()
        w = torch.exp(s - (0.0 if top == -INF else top))
        total = w.sum()
        out.append((w[:, None] * v).sum(0) / (1.0 if total == 0 else total))
    return torch.cat(out)


def same(got, want, top, unit):
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    big = torch.isinf(want)
    assert torch.equal(got[big], want[big])
    fine = torch.isfinite(want)
    assert ((got - want).abs()[fine] <= 4e-5 * top + unit * want.abs()[fine]).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [2, 4, 7])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [40, 1500])
def test_infinities_of_an_f16_cache(dim, group, act, n):
    pool = Pool("f16", [n] * 10, 16, n_kv=2, dim=dim, seed=group)
    q = queries(10, 2 * group, dim, act)
    q[5] = q[5].abs() + 1.0
    q[8] = q[8].abs() + 1.0
    if act != "f16":
        q[7, 1::2] *= 1e-6  # far under the row's largest value, not zero
    assert (q != 0).all()
    at = n // 2 + 3
    put(pool, "k", 0, at, 0, 5, -INF)  # minus infinity in some heads, plus in others, by q's sign
    put(pool, "k", 1, at, 1, 6, INF)
    put(pool, "v", 2, at, 0, 9, INF)
    put(pool, "v", 2, 1, 1, 10, -INF)
    put(pool, "v", 3, at, 0, 9, INF)  # both signs in one dimension
    put(pool, "v", 3, 2, 0, 9, -INF)
    put(pool, "k", 4, at, 0, 5, -INF)  # a dropped position with a finite value, and one with an infinite value
    put(pool, "v", 4, at + 1, 0, 3, INF)
    pool.mem["k"][pool.table[5].long(), :, :, 3] = -INF  # every score minus infinity
    pool.value["k"][5][:, :, 3] = -INF
    put(pool, "k", 6, 0, 0, 0, NAN)
    put(pool, "v", 6, n - 1, 1, 127 % dim, NAN)
    put(pool, "k", 7, at, 0, 1, -INF)  # against a q value that is lost beside the row's largest
    pool.mem["k"][pool.table[8].long(), 1, ::3, 2] = -INF  # many positions dropped
    pool.value["k"][8][1, torch.arange(n) % 16 % 3 == 0, 2] = -INF
    got = attend(pool, q, act=act)
    top = max(float(v[torch.isfinite(v)].abs().max()) for v in pool.value["v"])
    for i in range(10):
        same(got[i], formula(pool, q, i, lambda h: h // group, dim ** -0.5), top, ACT[act][2])
    assert (got[5] == 0).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [3, 8])
@pytest.mark.parametrize("act", ["f32", "f16"])
def test_infinities_among_many_conversations(dim, group, act):
    """900 short conversations and one that is split over many blocks, windows on some, infinities in a few: those are
    the formula's, the others the same bits as without."""
    lens = [1 + (i * 29) % 41 for i in range(900)]
    lens[411] = 6000
    starts = [3 if i % 5 == 0 else 0 for i in range(900)]
    pool = Pool("f16", lens, 16, n_kv=2, dim=dim, seed=group)
    q = queries(900, 2 * group, dim, act)
    assert (q != 0).all()
    before = attend(pool, q, starts=starts, act=act).clone()
    put(pool, "v", 411, 5999, 0, 7, INF)
    put(pool, "v", 411, 20, 1, 9, -INF)
    put(pool, "k", 411, 3333, 0, 1, -INF)
    marked = {411}
    for j, i in enumerate(range(3, 900, 37)):
        if lens[i] > 4:
            marked.add(i)
            put(pool, "kv"[j % 2], i, lens[i] - 1, j % 2, j % dim, (INF, -INF)[j // 2 % 2])
    put(pool, "v", 10, 1, 0, 0, INF)  # before the window: not looked at
    got = attend(pool, q, starts=starts, act=act)
    rest = torch.ones(900, dtype=torch.bool, device="cuda")
    rest[sorted(marked)] = False
    assert torch.equal(got[rest], before[rest])
    top = max(float(v[torch.isfinite(v)].abs().max()) for v in pool.value["v"])
    for i in marked:
        for name in ("k", "v"):
            pool.value[name][i] = pool.value[name][i][:, starts[i]:]
        same(got[i], formula(pool, q, i, lambda h: h // group, dim ** -0.5), top, ACT[act][2])


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("group", [3, 8])
def test_queries_that_are_not_finite(kind, group):
    """An infinite q value makes scores infinite (NaN rows, unless every score is minus infinity), a NaN makes its head
    NaN; the other heads and conversations are untouched."""
    pool = Pool(kind, [90, 90, 90, 0], 16, n_kv=2, dim=128, seed=1)
    q = queries(4, 2 * group, 128, "f32")
    q[0, 5] = NAN
    q[1, 128 + 7] = INF
    q[3, 9] = NAN
    got = attend(pool, q).cpu()
    head = got.view(4, -1, 128)
    assert torch.isnan(head[0, 0]).all() and torch.isnan(head[1, 1]).all()
    assert (head[3] == 0).all()
    rest = torch.ones(4, 2 * group, dtype=torch.bool)
    rest[0, 0] = rest[1, 1] = False
    assert torch.isfinite(head[rest]).all()
    top = max(float(v.abs().max()) for v in pool.value["v"][:3])
    for i in range(3):
        want = formula(pool, q, i, lambda h: h // group, 128 ** -0.5).view(-1, 128)
        err = (head[i].double() - want).abs()[rest[i]]
        assert float(err.max()) <= 4e-5 * top


@pytest.mark.parametrize("kind", ["q8", "q4"])
@pytest.mark.parametrize("group", [2, 8])
def test_nan_scales_of_a_quantised_cache(kind, group):
    """append marks a group that held a NaN by a NaN scale: a NaN key makes the rows of its KV head NaN, a NaN value its
    64 dimensions."""
    pool = Pool(kind, [700, 700, 700], 16, n_kv=2, dim=128, seed=1)
    pool.scale["k"][int(pool.table[0, 20]), 1, 3, 0] = NAN
    pool.scale["v"][int(pool.table[1, 43]), 0, 11, 1] = NAN
    q = queries(3, 2 * group, 128, "f32")
    got = attend(pool, q).cpu().view(3, 2, group, 128)
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[1, 0, :, 64:]).all()
    top = max(float(v.abs().max()) for v in pool.value["v"])
    for i in range(3):
        want = formula(pool, q, i, lambda h: h // group, 128 ** -0.5).view(2, group, 128)
        fine = torch.isfinite(got[i])
        assert int(fine.sum()) == group * (128, 192, 256)[i]
        assert float((got[i].double() - want).abs()[fine].max()) <= 4e-5 * top


def test_append_of_values_past_f16():
    """The f16 cache rounds as f16 does: past 65504 to infinity; the quantised ones saturate."""
    for kind, most in (("f16", INF), ("q8", 127 * 65504.0), ("q4", 7 * 65504.0)):
        pool = Pool(kind, [16], 16, n_kv=1, dim=64, seed=1)
        x = torch.ones(1, 128, device="cuda")
        x[0, 3], x[0, 70], x[0, 71] = 1e9, -1e9, 65504.0
        pos = torch.tensor([4], dtype=torch.int32, device="cuda")
        pool.kv.append(pool.pt, None, rpg.F32, x.data_ptr(), 0, pos.data_ptr(), 1)
        k, v = (torch.empty(1, 64, device="cuda") for _ in range(2))
        pool.kv.gather(pool.pt, rpg.F32, pos.data_ptr(), 1, k.data_ptr(), v.data_ptr())
        torch.cuda.synchronize()
        assert float(k[0, 3]) == most and float(v[0, 6]) == -most
        if kind == "f16":
            assert float(v[0, 7]) == 65504.0
