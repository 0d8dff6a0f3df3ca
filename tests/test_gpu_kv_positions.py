"""Every position of a range counts once: planted values that a lost, doubled or foreign position would change.

With q = 0 all weights are equal, so a row of the output is the mean of the range's values.  The values are random
bits.  Weights are powers of two and counts of bits at most 65521, so the f32 sums are exact; what rounds is 1 / n and
the product with it, so n times an output is a whole number to 2^-22 of itself: 0.01 at most.  A position lost or read
twice moves n times the output by about a half in every value, one read from elsewhere by one in half of them.  The
bound is 0.05.
"""

import pytest

import rpgbarenginecuda_b200 as rpg

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv import KIND, Pool, attend, expected, queries  # noqa: E402


class Bits:
    """A pool whose values are random bits and whose keys are random; what no conversation owns is poison."""

    def __init__(self, kind, lens, page, n_kv=2, dim=128, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.n_kv, self.dim = lens, n_kv, dim
        counts = [-(-n // page) for n in lens]
        pool, self.width = sum(counts) + 2, max(max(counts), 1)
        ids = torch.randperm(pool, generator=g, device="cuda")[:sum(counts)]
        bits = torch.randint(0, 2, (pool, n_kv, page, dim), generator=g, device="cuda", dtype=torch.uint8)
        owned = torch.zeros(pool, page, dtype=torch.bool, device="cuda")
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        self.bits, at = [], 0
        for i, n in enumerate(lens):
            mine = ids[at:at + counts[i]]
            at += counts[i]
            self.table[i, :counts[i]] = mine.int().cpu()
            here = torch.arange(counts[i] * page, device="cuda").view(-1, page) < n
            owned[mine] = here
            self.bits.append(bits[mine].transpose(1, 2).reshape(-1, n_kv, dim)[:n])
        self.mem, self.scale = {}, {}
        for name in ("k", "v"):
            if kind == "f16":
                x = bits.half() if name == "v" else torch.randn(bits.shape, generator=g, device="cuda").half()
                x[~owned[:, None].expand(-1, n_kv, -1)] = float("nan")
            else:
                x = bits if name == "v" else torch.randint(0, 7, bits.shape, generator=g, device="cuda", dtype=torch.uint8)
                d = torch.ones(pool, n_kv, page, dim // 64, dtype=torch.float16, device="cuda")
                d[~owned[:, None].expand(-1, n_kv, -1)] = float("nan")
                self.scale[name] = d
                x = x.to(torch.int8) if kind == "q8" else (x[..., 0::2] + 8) | ((x[..., 1::2] + 8) << 4)
            self.mem[name] = x.contiguous()
        self.dev_table = self.table.cuda()
        scales = [self.scale[n].data_ptr() for n in ("k", "v")] if kind != "f16" else []
        self.kv = rpg.PagedKv(KIND[kind], dim, n_kv, page, pool, self.mem["k"].data_ptr(), self.mem["v"].data_ptr(), *scales)
        self.pt = rpg.PageTable(self.dev_table.data_ptr(), len(lens), self.width)

    def counts(self, i, first, last):
        return self.bits[i][first:last].sum(0, dtype=torch.int64)


def every_position_once(pool, group, starts=None, lens=None):
    lens = lens or pool.lens
    q = torch.zeros(len(lens), pool.n_kv * group * pool.dim, device="cuda")
    out = attend(pool, q, lens=lens, starts=starts).double().view(len(lens), pool.n_kv, group, pool.dim)
    for i, n in enumerate(lens):
        first = max(0, starts[i]) if starts is not None else 0
        n = max(0, n - first)
        want = pool.counts(i, first, first + n)[:, None].expand(-1, group, -1) if n else 0.0
        off = float((out[i] * max(n, 1) - want).abs().max())
        assert off <= 0.05, (i, first, n, off)


FORMS = [(1, 128), (4, 128), (5, 128), (8, 128), (2, 64), (8, 64)]


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("group,dim", FORMS)
@pytest.mark.parametrize("n", [20011, 30000, 65521])
def test_one_long_conversation(kind, group, dim, n):
    """Split over its length: many shares, records and joins."""
    every_position_once(Bits(kind, [n], 64, n_kv=1, dim=dim, seed=n), group)


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("group,dim", FORMS)
def test_lengths_around_every_border(kind, group, dim):
    """Every length to 300, and around the multiples of 128 and 512 to 4700, in few and in many conversations."""
    short = list(range(301))
    long = [m + d for m in (384, 512, 640, 1024, 1536, 2048, 4096, 4608) for d in (-17, -16, -1, 0, 1, 15, 16, 17)]
    for lens in (short + long, long, short[:40], [4607], [4608, 1]):
        every_position_once(Bits(kind, lens, 16, dim=dim, seed=len(lens)), group)


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("group,dim", FORMS)
def test_windows_around_every_border(kind, group, dim):
    """One conversation's pages seen through windows that begin and end at every place."""
    pool = Bits(kind, [3000], 32, dim=dim, seed=3)
    for step in (1, 7, 131):
        starts = [(i * step) % 2990 for i in range(260)]
        lens = [min(3000, s + 1 + (i * 37) % 1300) for i, s in enumerate(starts)]
        many = Bits.__new__(Bits)
        many.__dict__.update(pool.__dict__)
        many.dev_table = pool.dev_table.expand(260, -1).contiguous()
        many.pt = rpg.PageTable(many.dev_table.data_ptr(), 260, pool.width)
        many.lens, many.bits = lens, pool.bits * 260
        every_position_once(many, group, starts=starts, lens=lens)


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("group", [2, 7])
def test_shares_of_ragged_batches(kind, group):
    """Batches whose shares begin and end at all places of items: a few lengths times a growing number of conversations."""
    for rows in (2, 3, 5, 9, 17, 33, 57, 101, 190):
        lens = [1 + (i * 1009 + rows * 97) % (40000 // rows) for i in range(rows)]
        every_position_once(Bits(kind, lens, 16, n_kv=3, seed=rows), group)


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("heads", [4, 14])
def test_extreme_scores(kind, heads):
    """Queries from 1e-20 to a thousand times the usual, of both signs, zero, and with one value far over the others.

    A score is an f32 sum of D products in at most 16 steps that may truncate, of partial sums under a quarter of the
    sum of the magnitudes: off by 8 * 2^-24 of that, and by 2^-24 of the row's largest |q| times the sum of |k|: q is
    held to 2^-23, and these errors do not all align.  An error e of the scores moves the output by at most 2 e max |v|; 4e-5 of max |v| is the rest."""
    pool = Pool(kind, [200] * 7, 16, n_kv=2, seed=8)
    q = queries(7, heads, 128, "f32")
    for i, f in enumerate((1000.0, -300.0, 30.0, 1e-20, 0.0, 1e-3)):
        q[i] *= f
    q[6, ::128] = 3000.0
    got, want = attend(pool, q), expected(pool, q)
    top = max(float(v.abs().max()) for v in pool.value["v"])
    x = q.double().cpu().view(7, 2, -1, 128)
    for i in range(7):
        k = pool.value["k"][i].abs()
        each = (x[i].abs() @ k.transpose(1, 2)).amax(-1)  # [kv head][query]
        largest = x[i].abs().amax(-1) * k.sum(-1).amax(-1)[:, None]
        e = 128 ** -0.5 * 2.0 ** -24 * (8 * each + largest)
        bound = (4e-5 + 2 * e) * top
        err = (got[i].double().cpu() - want[i]).abs().view(2, -1, 128).amax(-1)
        assert (err <= bound).all(), (i, float((err / bound).max()))
