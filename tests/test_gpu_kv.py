"""Paged key-value cache on the GPU against the formulas in 64 bits.

Tolerances.  attend: the scores are sums of D products in f32.  With |q| about
2 and |k| about 1 per value, sum |q_i k_i| scale is at most about 40 here, and
an f32 sum of it in 8 to 16 steps that may truncate is off by at most
16 * 2^-23 * 40 = 8e-5; the same relative error in every weight moves the
output by at most that share of the largest |v|; in practice errors do not all
align, so 4e-5 of max |v| is the bound, plus half a unit of the output type.
append: norm and rotation are a dozen f32 operations, 1e-6 of the row's
largest value, plus half a unit of the stored type (half a code step where the
cache is quantised).  gather: a code times an f16 scale is exact in f32, so
the result has to be equal.
"""

import numpy as np
import pytest

import rpgbarenginecuda_b200 as rpg

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ACT = {"f32": (rpg.F32, torch.float32, 0.0), "f16": (rpg.F16, torch.float16, 2.0 ** -11),
       "bf16": (rpg.BF16, torch.bfloat16, 2.0 ** -8)}
KIND = {"f16": rpg.KV_F16, "q8": rpg.KV_Q8, "q4": rpg.KV_Q4}
MOST = {"q8": 127, "q4": 7}
EPS = 1e-6


class Pool:
    """Pages with random content (poison where no conversation owns a position) and a page table.

    Values are held in 64 bits in `value[name][seq][head][pos][dim]`."""

    def __init__(self, kind, lens, page, n_kv=2, dim=128, seed=0, order="page-head-pos", extra=3, width=None):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.page, self.n_kv, self.dim, self.lens = kind, page, n_kv, dim, lens
        counts = [-(-n // page) for n in lens]
        self.n_pages = sum(counts) + extra
        self.width = width or max(max(counts), 1)
        ids = torch.randperm(self.n_pages, generator=g)[:sum(counts)].tolist()
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        shape = (self.n_pages, n_kv, page, dim)
        self.value = {"k": [], "v": []}
        code, scale = {}, {}
        for name in ("k", "v"):
            if kind == "f16":
                code[name] = torch.full(shape, float("nan"), dtype=torch.float16)
            else:
                code[name] = torch.randint(-MOST[kind], MOST[kind] + 1, shape, generator=g)
                scale[name] = torch.full(shape[:3] + (dim // 64,), float("nan"), dtype=torch.float16)
        at = 0
        for i, n in enumerate(lens):
            mine = ids[at:at + counts[i]]
            at += counts[i]
            self.table[i, :counts[i]] = torch.tensor(mine, dtype=torch.int32)
            for name in ("k", "v"):
                out = torch.zeros(n_kv, n, dim, dtype=torch.float64)
                for j, pg in enumerate(mine):
                    m = min(page, n - j * page)
                    if kind == "f16":
                        x = torch.randn(n_kv, m, dim, generator=g).half()
                        code[name][pg, :, :m] = x
                        out[:, j * page:j * page + m] = x.double()
                    else:
                        d = ((torch.rand(n_kv, m, dim // 64, generator=g) + 0.3) * 2.0 / MOST[kind]).half()
                        scale[name][pg, :, :m] = d
                        c = code[name][pg, :, :m]
                        out[:, j * page:j * page + m] = c.double() * d.double().repeat_interleave(64, -1)
                self.value[name].append(out)
        self.mem, self.scale = {}, {}
        for name in ("k", "v"):
            c = code[name]
            if kind == "q8":
                c = c.to(torch.int8)
            elif kind == "q4":
                c = ((c[..., 0::2] + 8) | ((c[..., 1::2] + 8) << 4)).to(torch.uint8)
            if order == "page-pos-head":
                c = c.transpose(1, 2).contiguous().cuda().transpose(1, 2)
            elif order == "padded":
                big = torch.zeros(self.n_pages + 1, n_kv + 1, page + 2, c.shape[-1] + 32, dtype=c.dtype, device="cuda")
                big[:self.n_pages, :n_kv, :page, :c.shape[-1]] = c.cuda()
                c = big[:self.n_pages, :n_kv, :page, :c.shape[-1]]
            else:
                c = c.cuda()
            self.mem[name] = c
            if kind != "f16":
                s = torch.zeros(self.n_pages, n_kv + 1, page, dim // 64, dtype=torch.float16, device="cuda")
                s[:, :n_kv] = scale[name].cuda()
                self.scale[name] = s
        self.dev_table = self.table.cuda()
        k = self.mem["k"]
        b = k.element_size()
        st = dict(page_stride=k.stride(0) * b, head_stride=k.stride(1) * b, pos_stride=k.stride(2) * b)
        sp = [0, 0]
        if kind != "f16":
            s = self.scale["k"]
            sp = [self.scale["k"].data_ptr(), self.scale["v"].data_ptr()]
            st.update(scale_page_stride=s.stride(0) * 2, scale_head_stride=s.stride(1) * 2)
        self.kv = rpg.PagedKv(KIND[kind], dim, n_kv, page, self.n_pages, k.data_ptr(), self.mem["v"].data_ptr(), *sp, **st)
        self.pt = rpg.PageTable(self.dev_table.data_ptr(), len(lens), self.width)


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def attend(pool, q, lens=None, starts=None, scale=None, act="f32", stream=0, ws=None, out=None):
    code, dt, _ = ACT[act]
    rows, width = q.shape
    lens = i32(pool.lens if lens is None else lens)
    st = i32(starts) if starts is not None else None
    n_heads = width // pool.dim
    if ws is None:
        ws = torch.zeros(rpg.attend_workspace(n_heads, pool.n_kv, pool.dim), dtype=torch.uint8, device="cuda")
    if out is None:
        out = torch.full((rows, width), 7.0, dtype=dt, device="cuda")
    torch.cuda.synchronize()
    pool.kv.attend(pool.pt, code, q.data_ptr(), n_heads, lens.data_ptr(), pool.dim ** -0.5 if scale is None else scale, out.data_ptr(),
                   ws.data_ptr(), ws.numel(), starts_ptr=st.data_ptr() if st is not None else 0, stream=stream,
                   q_stride=q.stride(0), out_stride=out.stride(0))
    torch.cuda.synchronize()
    return out


def expected(pool, q, lens=None, starts=None, scale=None):
    q = q.double().cpu()
    rows, width = q.shape
    out = torch.zeros(rows, width, dtype=torch.float64)
    for i in range(rows):
        n = (pool.lens if lens is None else lens)[i]
        s0 = max(0, starts[i]) if starts is not None else 0
        if n <= s0:
            continue
        qi = q[i].view(pool.n_kv, -1, pool.dim)
        k, v = pool.value["k"][i][:, s0:n], pool.value["v"][i][:, s0:n]
        w = torch.softmax(qi @ k.transpose(1, 2) * (pool.dim ** -0.5 if scale is None else scale), -1)
        out[i] = (w @ v).reshape(-1)
    return out


def check(got, want, pool, act):
    unit = ACT[act][2]
    top = max([float(v.abs().max()) for v in pool.value["v"] if v.numel()] or [0.0])
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    bound = 4e-5 * top + unit * want.abs() + 1e-30
    assert (err <= bound).all(), float((err / bound).max())


def queries(rows, heads, dim, act, seed=5):
    g = torch.Generator().manual_seed(seed)
    return (2.0 * torch.randn(rows, heads * dim, generator=g)).to(ACT[act][1]).cuda()


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 300]


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 12, 16])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_attend_heads_and_types(kind, dim, group, act):
    pool = Pool(kind, LENS, 16, n_kv=2, dim=dim, seed=group)
    q = queries(len(LENS), 2 * group, dim, act)
    check(attend(pool, q, act=act), expected(pool, q), pool, act)


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_attend_page_sizes(kind, page):
    lens = [5, 1000, 0, 47, 2049]
    pool = Pool(kind, lens, page, seed=page)
    q = queries(len(lens), 4, 128, "f32")
    check(attend(pool, q), expected(pool, q), pool, "f32")


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
def test_attend_one_long_conversation(kind):
    """Split over the length and joined: 20011 positions of one conversation."""
    pool = Pool(kind, [20011], 64, n_kv=1, seed=3)
    for heads in (1, 7):
        q = queries(1, heads, 128, "f32")
        check(attend(pool, q), expected(pool, q), pool, "f32")


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_attend_many_conversations(kind):
    lens = [(i * 53) % 131 for i in range(700)]
    pool = Pool(kind, lens, 16, n_kv=3, seed=3)
    q = queries(len(lens), 6, 128, "f16")
    check(attend(pool, q, act="f16"), expected(pool, q), pool, "f16")


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_attend_many_short_and_one_long(kind, dim, group):
    """900 conversations of two KV heads, nearly all a page or two long, one of 30000 positions, windows on some."""
    lens = [(i * 29) % 41 for i in range(900)]
    lens[411] = 30000
    starts = [3 if i % 5 == 0 else (29990 if i == 411 and group == 3 else 0) for i in range(900)]
    pool = Pool(kind, lens, 16, n_kv=2, dim=dim, seed=group)
    q = queries(900, 2 * group, dim, "f32")
    check(attend(pool, q, starts=starts), expected(pool, q, starts=starts), pool, "f32")


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
def test_attend_windows(kind):
    """Starts inside a page and a tile, on their edges, at and past the length, negative; pages before them may be gone."""
    lens = [300, 300, 300, 300, 300, 300, 300, 40, 300]
    starts = [0, 1, 16, 100, 128, 299, 300, 400, -5]
    pool = Pool(kind, lens, 16, seed=9)
    for i, s in enumerate(starts):
        pool.dev_table[i, :max(0, s) // 16] = -1
    for n, s, name in ((i, s, name) for i, s in enumerate(starts) for name in ("k", "v")):
        for pos in range(min(max(0, s), lens[n])):  # what is before the start is poison
            if kind == "f16":
                pool.mem[name][int(pool.table[n, pos // 16]), :, pos % 16] = float("nan")
            else:
                pool.scale[name][int(pool.table[n, pos // 16]), :, pos % 16] = float("nan")
    q = queries(len(lens), 4, 128, "f32")
    got = attend(pool, q, starts=starts)
    check(got, expected(pool, q, starts=starts), pool, "f32")
    assert (got[6] == 0).all() and (got[7] == 0).all()


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("order", ["page-pos-head", "padded"])
def test_attend_strides(kind, order):
    lens = [100, 33, 257]
    pool = Pool(kind, lens, 32, n_kv=4, seed=4, order=order)
    wide = torch.zeros(3, 8 * 128 + 64, dtype=torch.float32, device="cuda")
    wide[:, :1024] = queries(3, 8, 128, "f32")
    out = torch.full((3, 8 * 128 + 32), 7.0, device="cuda")
    q = wide[:, :1024]
    attend(pool, q, out=out[:, :1024])
    check(out[:, :1024], expected(pool, q), pool, "f32")
    assert (out[:, 1024:] == 7.0).all()


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
def test_attend_bad_pages_give_nan(kind):
    lens = [100, 100, 100, 100, 20]
    pool = Pool(kind, lens, 16, seed=6, width=8)
    pool.dev_table[1, 3] = -1
    pool.dev_table[2, 6] = pool.n_pages
    q = queries(5, 4, 128, "f32")
    got = attend(pool, q, lens=[100, 100, 100, 129, 20])  # row 3: past the table's 8 pages
    assert torch.isnan(got[1:4]).all()
    check(got[[0, 4]], expected(pool, q)[[0, 4]], pool, "f32")


def test_attend_extreme_scores():
    """Very large scores of both signs, a score range that leaves one position, queries tiny and large."""
    pool = Pool("f16", [200, 200, 200, 200], 16, seed=8)
    q = queries(4, 4, 128, "f32")
    q[0] *= 1000.0
    q[1] *= -300.0
    q[2] *= 1e-20
    q[3] = 0.0
    got, want = attend(pool, q), expected(pool, q)
    top = max(float(v.abs().max()) for v in pool.value["v"])
    # scores of rows 0 and 1 are 1000 and 300 times the others', and so is their error
    for i, f in enumerate((1000.0, 300.0, 1.0, 1.0)):
        assert float((got[i].double().cpu() - want[i]).abs().max()) <= 4e-5 * f * top


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("heads", [4, 14])
def test_attend_softmax_scales(kind, heads):
    """Zero (the mean of the values), negative, and a hundredth of the usual one."""
    lens = [0, 1, 90, 200]
    pool = Pool(kind, lens, 16, seed=8)
    q = queries(4, heads, 128, "f32")
    for scale in (0.0, -(128 ** -0.5), 1e-2 * 128 ** -0.5):
        check(attend(pool, q, scale=scale), expected(pool, q, scale=scale), pool, "f32")


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_attend_many_queries_to_one_head(kind):
    """37 query heads over one KV head: five passes of at most eight."""
    pool = Pool(kind, [333, 20], 16, n_kv=1, seed=8)
    q = queries(2, 37, 128, "f16")
    check(attend(pool, q, act="f16"), expected(pool, q), pool, "f16")


def test_attend_very_many_conversations():
    """70000 conversations of 64 heads, most of them empty: more than 2^21 tiles of work."""
    n, heads = 70000, 64
    lens = [0] * n
    for i in range(0, n, 7001):
        lens[i] = 1 + i % 40
    pool = Pool("f16", lens, 16, n_kv=heads, dim=64, seed=3)
    q = torch.zeros(n, heads * 64, dtype=torch.float16, device="cuda")
    some = [i for i in range(n) if lens[i]]
    q[some] = queries(len(some), heads, 64, "f16")
    got = attend(pool, q, act="f16")
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[some] = False
    assert int((got[rest] != 0).sum()) == 0
    few = Pool.__new__(Pool)
    few.__dict__.update(pool.__dict__)
    few.value = {k: [pool.value[k][i] for i in some] for k in pool.value}
    few.lens = [lens[i] for i in some]
    check(got[some], expected(few, q[some]), few, "f16")


@pytest.mark.parametrize("kind", ["q8", "q4"])
def test_attend_scales_of_all_sizes(kind):
    """Value scales that span f16's range inside one conversation: zero, subnormal, and growing along it."""
    pool = Pool(kind, [400], 16, n_kv=1, seed=2)
    order = pool.table[0].long()
    for pos in range(400):
        d = 2.0 ** (-24 + pos // 12) if pos % 7 else 0.0
        pool.scale["v"][order[pos // 16], 0, pos % 16] = d
        old = pool.value["v"][0][:, pos]
        code = pool.mem["v"][order[pos // 16], 0, pos % 16].cpu()
        if kind == "q4":
            code = torch.stack([code & 15, code >> 4], -1).flatten().double() - 8
        pool.value["v"][0][:, pos] = code.double().view_as(old[0]) * float(torch.tensor(d).half())
    q = queries(1, 2, 128, "f32")
    for n in (30, 100, 399):
        got, want = attend(pool, q, lens=[n]), expected(pool, q, lens=[n])
        top = float(pool.value["v"][0][:, :n].abs().max())
        assert float((got.double().cpu() - want).abs().max()) <= 4e-5 * top, n


def test_attend_nan_and_infinity_go_through():
    """A NaN key and an infinite value inside the range show, in their row and value alone."""
    pool = Pool("f16", [50, 50, 50], 16, seed=1)
    pool.mem["k"][int(pool.table[0, 1]), :, 3, 5] = float("nan")
    pool.mem["v"][int(pool.table[1, 2]), :, 1, 9] = float("inf")
    q = queries(3, 4, 128, "f32")
    got = attend(pool, q).cpu()
    assert torch.isnan(got[0]).all()
    assert not torch.isfinite(got[1].view(4, 128)[:, 9]).any()
    rest = [d for d in range(128) if d != 9]
    want = expected(pool, q)
    assert float((got[1].view(4, 128)[:, rest].double() - want[1].view(4, 128)[:, rest]).abs().max()) < 1e-3
    assert float((got[2].double() - want[2]).abs().max()) < 1e-3


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
def test_attend_repeats_and_leaves_the_workspace_ready(kind):
    """The same bits call after call with one workspace, whatever ran between, also from a CUDA graph."""
    a, b = Pool(kind, [5000, 3, 700], 16, seed=1), Pool(kind, [9, 2222], 32, n_kv=1, seed=2)
    qa, qb = queries(3, 8, 128, "f32"), queries(2, 5, 128, "f32")
    ws = torch.zeros(16 << 20, dtype=torch.uint8, device="cuda")
    first, other = attend(a, qa, ws=ws).clone(), attend(b, qb, ws=ws).clone()
    for _ in range(3):
        assert torch.equal(attend(a, qa, ws=ws), first)
        assert torch.equal(attend(b, qb, ws=ws), other)
    lens, out = i32(a.lens), torch.zeros_like(first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.kv.attend(a.pt, rpg.F32, qa.data_ptr(), 8, lens.data_ptr(), 128 ** -0.5, out.data_ptr(), ws.data_ptr(),
                    ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)


def test_attend_one_workspace_for_batches_of_all_sizes():
    """Batches that grow and shrink, of other head layouts, one after another on one workspace."""
    ws = torch.zeros(rpg.attend_workspace(24, 3, 128), dtype=torch.uint8, device="cuda")
    for rows, longest, n_kv, group, dim, kind in ((1, 4000, 1, 2, 128, "f16"), (400, 50, 5, 4, 64, "q8"),
                                                  (3, 3000, 3, 8, 128, "q4"), (900, 20, 8, 1, 64, "f16"),
                                                  (17, 700, 8, 3, 128, "q8"), (1, 9000, 2, 8, 64, "q4"),
                                                  (150, 60, 3, 7, 128, "f16")):
        lens = [1 + (i * 31) % longest for i in range(rows - 1)] + [longest]
        pool = Pool(kind, lens, 16, n_kv=n_kv, dim=dim, seed=rows)
        q = queries(rows, n_kv * group, dim, "f32")
        check(attend(pool, q, ws=ws), expected(pool, q), pool, "f32")


def test_attend_on_another_stream():
    pool = Pool("q8", [3000, 50], 16, seed=1)
    q = queries(2, 4, 128, "f32")
    want = attend(pool, q).clone()
    side = torch.cuda.Stream()
    assert torch.equal(attend(pool, q, stream=side.cuda_stream), want)


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_offsets_past_32_bits(kind):
    """Pages 300 MB apart: byte offsets up to 4.8e9 in append, attend and gather."""
    stride, n_pages, page = 300 << 20, 17, 16
    pool = Pool(kind, [60], page, n_kv=2, seed=1)
    row = 256 if kind == "f16" else 128
    mem = {n: torch.zeros(stride * (n_pages - 1) + 2 * page * row, dtype=torch.uint8, device="cuda") for n in ("k", "v")}
    sc = {n: torch.zeros(n_pages, 2, page, 2, dtype=torch.float16, device="cuda") for n in ("k", "v")}
    ids = [16, 3, 15, 9]
    table = i32(ids)
    kv = rpg.PagedKv(KIND[kind], 128, 2, page, n_pages, mem["k"].data_ptr(), mem["v"].data_ptr(),
                     sc["k"].data_ptr() if kind != "f16" else 0, sc["v"].data_ptr() if kind != "f16" else 0,
                     page_stride=stride)
    pt = rpg.PageTable(table.data_ptr(), 1, 4)
    x = torch.randn(60, 6 * 128, generator=torch.Generator().manual_seed(1)).cuda()
    pos = torch.arange(60, dtype=torch.int32, device="cuda")
    seq = torch.zeros(60, dtype=torch.int32, device="cuda")
    kv.append(pt, None, rpg.F32, x.data_ptr(), 2, pos.data_ptr(), 60, 0, seq_ptr=seq.data_ptr())
    ko, vo = torch.empty(60, 256, device="cuda"), torch.empty(60, 256, device="cuda")
    kv.gather(pt, rpg.F32, pos.data_ptr(), 60, ko.data_ptr(), vo.data_ptr(), seq_ptr=seq.data_ptr())
    torch.cuda.synchronize()
    step = 2.0 ** -11 if kind == "f16" else 1.01 / 254
    assert float((ko - x[:, 256:512]).abs().max()) <= step * float(x.abs().max())
    assert float((vo - x[:, 512:]).abs().max()) <= step * float(x.abs().max())
    pool.kv, pool.pt, pool.lens = kv, pt, [60]
    pool.value = {"k": [ko.double().cpu().view(60, 2, 128).transpose(0, 1)],
                  "v": [vo.double().cpu().view(60, 2, 128).transpose(0, 1)]}
    q = queries(1, 4, 128, "f32")
    check(attend(pool, q), expected(pool, q), pool, "f32")


# ---------------------------------------------------------------- append and gather


def norm_rope(x, w, table, pos):
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    if table is None:
        return x
    h = x.shape[-1] // 2
    c, s = (t[:, None] for t in (table[pos][:, :h].double(), table[pos][:, h:].double()))
    return torch.cat([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)


def rows_of(pool, act, n_heads, n_tok, seed, pad=0):
    cols = (n_heads + 2 * pool.n_kv) * pool.dim
    x = torch.randn(n_tok, cols + pad, generator=torch.Generator().manual_seed(seed)).to(ACT[act][1])
    return x.cuda()[:, :cols], x[:, :cols].double()


def read(pool, seq, pos, dtype=rpg.F32, tdt=torch.float32):
    n = len(pos)
    k = torch.empty(n, pool.n_kv * pool.dim, dtype=tdt, device="cuda")
    v = torch.empty_like(k)
    s, p = i32(seq), i32(pos)
    pool.kv.gather(pool.pt, dtype, p.data_ptr(), n, k.data_ptr(), v.data_ptr(), seq_ptr=s.data_ptr())
    torch.cuda.synchronize()
    return k.cpu(), v.cpu()


def close_to_stored(got, want, kind):
    """Stored values against the values that were to be stored, [row][head][dim] in 64 bits."""
    got = got.double().view_as(want)
    top = want.abs().amax(-1, keepdim=True)
    if kind == "f16":
        bound = want.abs() * 2.0 ** -11 + 1e-6 * top + 2.0 ** -25
    else:
        group = want.unflatten(-1, (-1, 64)).abs().amax(-1).repeat_interleave(64, -1)
        # half a step of the scale f16(max / most), which may itself be rounded by 2^-11, and round-off of the values
        bound = (0.5 + 1e-3) * group / MOST[kind] * (1 + 2.0 ** -11) + 2e-6 * top
        bound = torch.maximum(bound, group * 2.0 ** -11 + 2e-6 * top)  # the clamp at the largest code
    err = (got - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads", [(2, 2), (7, 1), (16, 8), (5, 5)])
def test_append_writes_and_gather_reads(kind, dim, act, heads):
    n_heads, n_kv = heads
    lens = [37, 1, 100]
    pool = Pool(kind, lens, 16, n_kv=n_kv, dim=dim, seed=2)
    seq = [i for i, n in enumerate(lens) for _ in range(n)][::-1]
    pos = [p for n in lens for p in range(n)][::-1]
    x, x64 = rows_of(pool, act, n_heads, len(pos), 3, pad=8)
    table = torch.from_numpy(rpg.rope_table(100, dim, 1e6))
    w = [1 + 0.2 * torch.randn(dim, generator=torch.Generator().manual_seed(s)) for s in (1, 2)]
    dev = [t.cuda() for t in (table, *w)]
    rot = rpg.Rotary(dev[0].data_ptr(), 100, dev[1].data_ptr(), dev[2].data_ptr(), EPS)
    q = torch.full((len(pos), n_heads * dim + 8), 7.0, dtype=ACT[act][1], device="cuda")
    s, p = i32(seq), i32(pos)
    pool.kv.append(pool.pt, rot, ACT[act][0], x.data_ptr(), n_heads, p.data_ptr(), len(pos), q.data_ptr(),
                   seq_ptr=s.data_ptr(), qkv_stride=x.stride(0), q_stride=q.stride(0))
    torch.cuda.synchronize()
    parts = x64.reshape(len(pos), -1, dim).split([n_heads, n_kv, n_kv], 1)
    want_q, want_k = norm_rope(parts[0], w[0], table, pos), norm_rope(parts[1], w[1], table, pos)
    err = (q[:, :n_heads * dim].double().cpu().view_as(want_q) - want_q).abs()
    assert (err <= 1e-6 * want_q.abs().amax(-1, keepdim=True) + ACT[act][2] * want_q.abs()).all()
    assert (q[:, n_heads * dim:] == 7.0).all()
    k, v = read(pool, seq, pos)
    close_to_stored(k, want_k, kind)
    close_to_stored(v, parts[2], kind)


@pytest.mark.parametrize("kind", ["q8", "q4"])
def test_append_codes_are_exact_without_norm_and_rotation(kind):
    """rotary None: scales and codes are single IEEE operations on the inputs, so they are equal to numpy's."""
    pool = Pool(kind, [64], 16, n_kv=2, seed=2)
    x, x64 = rows_of(pool, "f32", 2, 64, 3)
    x[3, 256:320] = 0.0            # an all-zero group
    x[4, 256:320] *= 1e-9          # a scale that underflows to zero
    x[5, 256:320] *= 3e-6          # a subnormal scale, far from the exact one
    x[6, 256] = 1e9                # past f16's range times the largest code
    x[7, 256] = float("inf")
    x[7, 300] = -float("inf")
    x[8, 270] = float("nan")
    pos = torch.arange(64, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    pool.kv.append(pool.pt, None, rpg.F32, x.data_ptr(), 2, pos.data_ptr(), 64, 0, seq_ptr=seq.data_ptr())
    torch.cuda.synchronize()
    page, at = pool.table[0].long()[torch.arange(64) // 16], torch.arange(64) % 16
    most = np.float32(MOST[kind])
    for name, lo in (("k", 256), ("v", 512)):
        rows = x[:, lo:lo + 256].cpu().numpy().reshape(64, 2, 2, 64)
        m = np.abs(rows).max(-1)  # NaN where there is one
        with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
            d16 = np.where(np.isnan(m), m, np.minimum(m * (np.float32(1) / most), np.float32(65504))).astype(np.float16)
            d = d16.astype(np.float32)[..., None]
            c = np.where(d > 0, np.clip(np.rint(rows / np.where(d > 0, d, 1)), -most, most), 0)
        got_d = pool.scale[name][page, :2][torch.arange(64), :, at].cpu().numpy()
        assert np.array_equal(got_d, d16, equal_nan=True)
        got = pool.mem[name].cpu()[page][torch.arange(64), :, at]
        if kind == "q4":
            got = torch.stack([got & 15, got >> 4], -1).flatten(-2).int() - 8
        got = got.numpy().reshape(64, 2, 2, 64)
        fine = ~np.isnan(rows) & ~np.isnan(m)[..., None]
        assert np.array_equal(got[fine], c[fine].astype(got.dtype))
    k, _ = read(pool, [0], [8])
    assert torch.isnan(k[0, :64]).all() and torch.isfinite(k[0, 64:]).all()


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("order", ["page-head-pos", "page-pos-head", "padded"])
def test_gather_is_exact(kind, act, order):
    lens = [70, 1, 33]
    pool = Pool(kind, lens, 32, n_kv=3, seed=5, order=order)
    seq = [0, 2, 1, 0, 2, 0, 0]
    pos = [69, 32, 0, 0, 31, 31, 32]
    k, v = read(pool, seq, pos, ACT[act][0], ACT[act][1])
    for got, name in ((k, "k"), (v, "v")):
        want = torch.stack([pool.value[name][s][:, p] for s, p in zip(seq, pos)]).reshape(len(pos), -1)
        assert torch.equal(got, want.float().to(ACT[act][1]))


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
def test_rows_without_a_place(kind):
    """Padding rows, conversations and positions outside the table, missing pages, rotation rows that do not exist."""
    pool = Pool(kind, [40, 40], 16, n_kv=2, seed=5, width=4)
    seq = [0, 0, -1, 2, 0, 1, 1, 0]
    pos = [3, -1, 3, 3, 64, 50, 45, 39]  # row 5: table entry -1; row 6: past the rotation table
    pool.dev_table[1, 2] = 0
    x, x64 = rows_of(pool, "f32", 2, 8, 3)
    table = torch.from_numpy(rpg.rope_table(45, 128)).cuda()
    rot = rpg.Rotary(table.data_ptr(), 45)
    before = {n: (pool.mem[n].clone(), pool.scale[n].clone() if kind != "f16" else None) for n in ("k", "v")}
    q = torch.full((8, 256), 7.0, device="cuda")
    s, p = i32(seq), i32(pos)
    pool.kv.append(pool.pt, rot, rpg.F32, x.data_ptr(), 2, p.data_ptr(), 8, q.data_ptr(), seq_ptr=s.data_ptr())
    torch.cuda.synchronize()
    assert (q[1] == 0).all()
    assert torch.isnan(q[[2, 3, 4, 5, 6]]).all()
    assert torch.isfinite(q[[0, 7]]).all()
    touched = torch.zeros(pool.n_pages, 16, dtype=torch.bool)
    touched[int(pool.table[0, 0]), 3] = touched[int(pool.table[0, 2]), 39 % 16] = True
    for n in ("k", "v"):
        for now, old in ((pool.mem[n], before[n][0]), (pool.scale.get(n), before[n][1])):
            if now is not None:
                same = (now.contiguous().view(torch.uint8) == old.contiguous().view(torch.uint8)).all(-1).all(1)
                same = same.cpu() if same.shape[1] == 16 else same.cpu()[:, :16]
                assert same[~touched].all()
    k, v = read(pool, [0, 0, -1, 2, 0, 1], [3, -1, 3, 3, 64, 50])
    assert (k[1] == 0).all() and (v[1] == 0).all()
    assert torch.isnan(k[[2, 3, 4, 5]]).all() and torch.isnan(v[[2, 3, 4, 5]]).all()
    assert torch.isfinite(k[0]).all()


def test_append_in_place_and_without_q():
    pool = Pool("f16", [16], 16, n_kv=2, seed=5)
    x, x64 = rows_of(pool, "f32", 3, 1, 3)
    table = torch.from_numpy(rpg.rope_table(16, 128))
    dev = table.cuda()
    rot = rpg.Rotary(dev.data_ptr(), 16)
    pos = i32([7])
    want = norm_rope(x64.reshape(1, -1, 128), None, table, [7])
    pool.kv.append(pool.pt, rot, rpg.F32, x.data_ptr(), 3, pos.data_ptr(), 1, x.data_ptr(), q_stride=x.stride(0))
    torch.cuda.synchronize()
    assert float((x[:, :384].double().cpu().view(1, 3, 128) - want[:, :3]).abs().max()) < 1e-5
    assert torch.equal(x[:, 384:].double().cpu(), x64[:, 384:])
    k, _ = read(pool, [0], [7])
    close_to_stored(k, want[:, 3:5], "f16")
    # rows of k and v alone, q not wanted
    y = x64[:, 384:].float().cuda()
    pos = i32([9])
    pool.kv.append(pool.pt, None, rpg.F32, y.data_ptr(), 0, pos.data_ptr(), 1)
    k, v = read(pool, [0], [9])
    assert torch.equal(k, y[:, :256].half().float().cpu()) and torch.equal(v, y[:, 256:].half().float().cpu())


def test_gather_one_side():
    pool = Pool("q8", [20], 16, n_kv=2, seed=5)
    both = read(pool, [0] * 3, [0, 5, 19])
    s, p = i32([0] * 3), i32([0, 5, 19])
    out = torch.empty(3, 256, device="cuda")
    for i, kw in enumerate((dict(k_out_ptr=out.data_ptr()), dict(v_out_ptr=out.data_ptr()))):
        pool.kv.gather(pool.pt, rpg.F32, p.data_ptr(), 3, seq_ptr=s.data_ptr(), **kw)
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), both[i])


@pytest.mark.parametrize("kind,tol", [("f16", 2e-3), ("q8", 2e-2), ("q4", 0.3)])
def test_a_conversation_step_by_step(kind, tol):
    """Tokens appended one by one and attended to give the causal attention of the whole conversation; a quantised
    cache moves the result by about its step (1/254 and 1/14 of a group's largest value)."""
    n, n_heads, n_kv, dim = 50, 4, 2, 128
    pool = Pool(kind, [64, 64], 16, n_kv=n_kv, seed=5)
    x, x64 = rows_of(pool, "f32", n_heads, 2 * n, 3)
    table = torch.from_numpy(rpg.rope_table(n, dim))
    dev = table.cuda()
    rot = rpg.Rotary(dev.data_ptr(), n)
    x, x64 = x.view(n, 2, -1), x64.view(n, 2, -1, dim)
    ws = torch.zeros(rpg.attend_workspace(n_heads, n_kv, dim), dtype=torch.uint8, device="cuda")
    out = torch.empty(n, 2, n_heads * dim, device="cuda")
    q = torch.empty(2, n_heads * dim, device="cuda")
    for t in range(n):
        pos, lens = i32([t, t]), i32([t + 1, t + 1])
        pool.kv.append(pool.pt, rot, rpg.F32, x[t].data_ptr(), n_heads, pos.data_ptr(), 2, q.data_ptr())
        pool.kv.attend(pool.pt, rpg.F32, q.data_ptr(), n_heads, lens.data_ptr(), dim ** -0.5, out[t].data_ptr(),
                       ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    for s in range(2):
        qkv = x64[:, s]
        q64 = norm_rope(qkv[:, :n_heads], None, table, range(n)).view(n, n_kv, 2, dim)
        k64 = norm_rope(qkv[:, n_heads:n_heads + n_kv], None, table, range(n))
        scores = torch.einsum("thgd,nhd->hgtn", q64, k64) * dim ** -0.5
        scores = scores.masked_fill(~torch.tril(torch.ones(n, n, dtype=torch.bool)), float("-inf"))
        want = torch.einsum("hgtn,nhd->thgd", torch.softmax(scores, -1), qkv[:, n_heads + n_kv:]).reshape(n, -1)
        assert float((out[:, s].double().cpu() - want).abs().max()) <= tol * 3.5


@pytest.mark.parametrize("kind", ["f16", "q8"])
def test_buffers_updated_in_place_between_calls(kind):
    """200 steps on the same buffers, lengths, positions and rows updated by other kernels in between and nothing
    waited for: each step sees what was written before it."""
    n_seq, n_heads, n_kv, dim, steps = 40, 8, 2, 128, 200
    pool = Pool(kind, [208] * n_seq, 16, n_kv=n_kv, dim=dim, seed=5)
    cols = (n_heads + 2 * n_kv) * dim
    x = torch.randn(steps, n_seq, cols, generator=torch.Generator().manual_seed(4)).cuda()
    row = torch.empty(n_seq, cols, device="cuda")
    pos, lens = i32([-1] * n_seq), i32([0] * n_seq)
    ws = torch.zeros(rpg.attend_workspace(n_heads, n_kv, dim), dtype=torch.uint8, device="cuda")
    out = torch.empty(n_seq, n_heads * dim, device="cuda")
    kept = torch.empty(steps, n_seq, n_heads * dim, device="cuda")
    for t in range(steps):
        row.copy_(x[t])
        pos += 1
        lens += 1
        pool.kv.append(pool.pt, None, rpg.F32, row.data_ptr(), n_heads, pos.data_ptr(), n_seq, row.data_ptr(),
                       q_stride=cols)
        pool.kv.attend(pool.pt, rpg.F32, row.data_ptr(), n_heads, lens.data_ptr(), dim ** -0.5, out.data_ptr(),
                       ws.data_ptr(), ws.numel(), q_stride=cols)
        kept[t].copy_(out)
    torch.cuda.synchronize()
    seq = [s for s in range(n_seq) for _ in range(steps)]
    k, v = read(pool, seq, list(range(steps)) * n_seq)
    k, v = (y.double().view(n_seq, steps, n_kv, dim).transpose(1, 2) for y in (k, v))
    top = float(v.abs().max())
    q = x[:, :, :n_heads * dim].double().cpu().view(steps, n_seq, n_kv, -1, dim)
    for t in (0, 1, 15, 16, 63, 64, 127, 128, steps - 1):
        w = torch.softmax(torch.einsum("shgd,shnd->shgn", q[t], k[:, :, :t + 1]) * dim ** -0.5, -1)
        want = torch.einsum("shgn,shnd->shgd", w, v[:, :, :t + 1]).reshape(n_seq, -1)
        assert float((kept[t].double().cpu() - want).abs().max()) <= 4e-5 * top, t
