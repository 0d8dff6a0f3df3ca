"""Sampling of a batch against the definition in 64 bits.

Tokens have to be equal: the reference's sums are in 64 bits and the kernel's in
integers of 2^-44, so a random number decides differently only within about
2^18 * 2^-45 / total of a border, which the fixed seeds here do not meet; rows
whose random number lies within 1e-9 of a border are not asked (there are none
in most batches).  Probabilities are f32: half a step of 2^-24, and the error of
the sums, under 2^-27: 1.3e-7 relative in all.
"""

import math

import numpy as np
import pytest

import rpgbarenginecuda_b200 as rpg

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": (rpg.F32, torch.float32), "f16": (rpg.F16, torch.float16), "bf16": (rpg.BF16, torch.bfloat16)}


def call(x, u=None, temperature=None, top_k=None, top_p=None, min_p=None, probs=True, stride=None, out=None, stream=0):
    n, vocab = x.shape
    kind = {v[1]: v[0] for v in TYPES.values()}[x.dtype]
    put = lambda v, t: None if v is None else torch.as_tensor(v, dtype=t, device="cuda").expand(n).contiguous()  # noqa: E731
    a = dict(u_ptr=put(u, torch.float32), temperature_ptr=put(temperature, torch.float32), top_k_ptr=put(top_k, torch.int32),
             top_p_ptr=put(top_p, torch.float32), min_p_ptr=put(min_p, torch.float32))
    tok, prob = out or (torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.full((n,), -7.0, device="cuda"))
    torch.cuda.synchronize()
    rpg.sample_rows(x.data_ptr(), kind, n, vocab, tok.data_ptr(), prob_ptr=prob.data_ptr() if probs else 0,
                    stride=x.stride(0), stream=stream, **{k: v.data_ptr() if v is not None else 0 for k, v in a.items()})
    torch.cuda.synchronize()
    return tok.cpu().numpy(), prob.cpu().numpy()


def one(x, u, t, k, p, m):
    """(token, probability, distance of u to the next border) of one row, in 64 bits on the CPU."""
    x = x.astype(np.float64)
    live = x > -math.inf  # (NaN is not)
    if not live.any():
        return -1, math.nan, 1.0
    top = x[live].max()
    if not t > 0:
        return int(np.flatnonzero(x == top)[0]), 1.0, 1.0
    if top == math.inf:
        w = (x == top).astype(np.float64)
    else:
        w = np.where(live, np.exp((np.where(live, x, 0) - top) / np.float64(np.float32(t))), 0.0)
    keep = live.copy()
    if 1 < k < len(x) and live.sum() > k:
        keep &= x >= np.sort(x[live])[-k]
    if 0 < p < 1:
        left = np.where(keep, w, 0.0)
        level, inverse = np.unique(np.where(live, x, -math.inf), return_inverse=True)
        mass = np.bincount(inverse, left, len(level))
        above = mass[::-1].cumsum()[::-1] - mass
        keep &= (above < np.float64(np.float32(p)) * left.sum() * (1 - 1e-13))[inverse]
    if 0 < m <= 1:
        keep &= w >= np.float64(np.float32(m))
    w = np.where(keep, w, 0.0)
    c = w.cumsum()
    u = np.float64(np.float32(u)) * c[-1]
    i = min(int(np.searchsorted(c, u, "right")), int(np.flatnonzero(w)[-1]))
    return i, w[i] / c[-1], float(np.abs(c - u).min() / c[-1])


def check(x, u, t=1.0, k=0, p=1.0, m=0.0, asked=0.9):
    n = x.shape[0]
    full = lambda v: np.broadcast_to(np.asarray(v), (n,))  # noqa: E731
    tok, prob = call(x, u, t, k, p, m)
    host, seen = x.float().cpu().numpy(), 0
    for r in range(n):
        i, q, gap = one(host[r], full(u)[r], full(t)[r], full(k)[r], full(p)[r], full(m)[r])
        if gap < 1e-9:
            continue
        seen += 1
        assert tok[r] == i, (r, tok[r], i, gap)
        if math.isnan(q):
            assert math.isnan(prob[r])
        else:
            assert abs(prob[r] - q) <= 1.3e-7 * q
    assert seen >= asked * n
    return tok, prob


def logits(n, vocab, act="f32", seed=0, peak=True, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = spread * torch.randn(n, vocab, generator=g, device="cuda")
    if peak:
        at = torch.randint(0, vocab, (n, 40), generator=g, device="cuda")
        x.scatter_add_(1, at, 4.0 + 3.0 * torch.randn(n, 40, generator=g, device="cuda"))
    return x.to(TYPES[act][1]), torch.rand(n, generator=g, device="cuda").cpu().numpy()


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 1000, 4097, 32001, 151936, 262144])
def test_whole_distribution(act, vocab):
    x, u = logits(9, vocab, act, seed=vocab)
    check(x, u, t=[0.7, 1.0, 1.3] * 3)


@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 32001, 151936])
@pytest.mark.parametrize("peak", [True, False])
def test_filters(act, vocab, peak):
    n = 60
    x, u = logits(n, vocab, act, seed=vocab + peak, peak=peak)
    i = np.arange(n)
    k = np.array([0, 1, 2, 20, 64, 100, 1000, 5000, vocab - 1, vocab, -3])[i % 11]
    p = np.array([1.0, 0.8, 0.95, 0.999, 0.1, 0.0, 1.5])[i % 7].astype(np.float32)
    m = np.array([0.0, 0.05, 0.5, 0.0, 1.0, 0.001])[i % 6].astype(np.float32)
    t = np.array([0.7, 1.0, 0.0, 1.5, 0.85])[i % 5].astype(np.float32)
    check(x, u, t, k, p, m)


@pytest.mark.parametrize("k,p", [(20, 0.8), (50, 1.0), (0, 0.9), (0, 0.5), (1000, 0.99)])
def test_filters_as_rpgb_sample(k, p):
    # the same tokens as one-row sampling with the same random number, but for rows within f32 rounding of a border
    x, _ = logits(24, 151936, seed=k)
    u = [rpg.counter_uniform(11, r) for r in range(24)]
    tok, prob = call(x, u, 0.7, k, p)
    out = torch.empty(24, dtype=torch.int32, device="cuda")
    for r in range(24):
        rpg.sample(x[r].data_ptr(), 151936, rpg.SampleOptions(0.7, k, p), 11, r, out[r:].data_ptr())
    torch.cuda.synchronize()
    host = x.cpu().numpy()
    for r in np.flatnonzero(out.cpu().numpy() != tok):
        assert one(host[r], u[r], 0.7, k, p, 0.0)[2] < 1e-5


def test_equal_values():
    # many ties: at the k-th value all stay, the share is cut between values
    x = torch.zeros(8, 5000, device="cuda")
    x[:, 100:160] = 3.0
    x[:, 3000] = 3.5
    u = np.linspace(0.01, 0.99, 8)
    check(x, u, t=1.0, k=10)
    check(x, u, t=1.0, p=0.3)
    check(x, u, t=1.0, k=61, p=0.5, m=0.2)
    check(torch.full((4, 151936), -2.5, device="cuda"), [0.0, 0.3, 0.7, 0.999], k=50, p=0.9)
    check(torch.full((4, 7000), 1.0, device="cuda").bfloat16(), [0.0, 0.3, 0.7, 0.999])


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [9, 5000])
def test_zeros_of_both_signs_are_equal(act, vocab):
    x = torch.full((12, vocab), -1.0, device="cuda")
    x[:, 2], x[:, 4], x[:, vocab - 2] = -0.0, 0.0, -0.0
    u = np.linspace(0.02, 0.98, 12)
    for rows in (x, x - 1.0 * (torch.arange(vocab, device="cuda") == 4), x.index_fill(1, torch.tensor([6], device="cuda"), 1.5)):
        rows = rows.to(TYPES[act][1])
        check(rows, u, t=0.0)
        check(rows, u, t=1.0)
        check(rows, u, t=1.0, k=2)
        check(rows, u, t=1.0, k=3)
        check(rows, u, t=1.0, p=0.0005)
        check(rows, u, t=0.2, p=0.5, k=4)
        check(rows, u, t=1.0, m=1.0)


def test_extremes_of_the_random_number():
    x, _ = logits(4, 3000, seed=5)
    check(x, [0.0, 2.0 ** -30, 1.0 - 2.0 ** -24, 0.5], t=1.0)
    tok, _ = call(x, [1.0, 2.0, -1.0, math.nan], 1.0)  # held to [0, 1)
    assert tok[0] == tok[1] == 2999 and tok[2] == tok[3] == 0


def test_not_finite():
    x, u = logits(9, 4000, seed=8)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 17:] = -math.inf
    x[3, ::2] = math.nan
    x[4, 100] = x[4, 3500] = math.inf
    x[5] = torch.finfo(torch.float32).min
    x[6, 5] = math.nan
    x[7] = -math.inf
    x[7, 1234] = -1e38
    for t in (1.0, 0.0, math.nan):
        for kw in (dict(), dict(k=20, p=0.9), dict(p=0.5, m=0.1)):
            check(x, u, t=t, **kw)
    tok, prob = call(x, u, 1.0)
    assert tok[0] == tok[1] == -1 and np.isnan(prob[:2]).all()
    assert tok[4] in (100, 3500) and prob[4] == 0.5 and tok[7] == 1234


@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_fewer_values_than_are_wanted(act):
    # a mask that leaves a few values, scattered or side by side, under a larger k and a share
    x, u = logits(8, 40000, act, seed=9)
    for r in range(8):
        keep = torch.arange(40000, device="cuda") % (5000 + r) == r if r % 2 else torch.arange(40000, device="cuda") < 3 * r + 1
        x[r, ~keep] = -math.inf if r < 4 else math.nan
    for kw in (dict(k=100), dict(k=600), dict(k=2000, p=0.9), dict(p=0.7), dict(k=30, m=0.2)):
        check(x, u, t=1.2, **kw)


def test_values_in_order():
    # the largest values side by side, in one block's part
    x = torch.linspace(-20, 20, 100000, device="cuda").flip(0).expand(6, -1).contiguous()
    x[3:] = x[3:].flip(1)
    u = [0.1, 0.5, 0.9] * 2
    for kw in (dict(k=50), dict(k=700), dict(p=0.9), dict(k=1200, p=0.5), dict(k=5000), dict()):
        check(x, u, t=1.0, **kw)


def test_temperatures_near_zero_and_huge():
    x, u = logits(6, 9000, seed=2)
    check(x, u, t=[1e-30, 1e-3, 1e-2, 100.0, 1e6, 1e30])
    check(x, u, t=[1e-30, 1e-3, 1e-2, 100.0, 1e6, 1e30], k=30, p=0.7)


def test_strides_alignments_and_rows_behind_the_last():
    g = torch.Generator(device="cuda").manual_seed(3)
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        wide = torch.randn(7, 5003, generator=g, device="cuda").to(dt)
        for first in (0, 1, 3):
            x = wide[:, first:first + 4321]
            u = np.linspace(0.05, 0.95, 7)
            check(x, u, t=0.9, k=500)
    x, u = logits(3, 999)
    out = torch.full((5,), -7, dtype=torch.int32, device="cuda"), torch.full((5,), -7.0, device="cuda")
    call(x, u, 1.0, out=out)
    assert out[0][3:].tolist() == [-7, -7] and out[1][3:].tolist() == [-7.0, -7.0]


def test_options_left_out_and_a_row_alone():
    x, u = logits(50, 20000, "f16", seed=4)
    t = np.where(np.arange(50) % 3 == 0, 0.0, 0.8).astype(np.float32)
    all_at_once, probs = call(x, u, t, 40, 0.9, 0.02)
    for r in (0, 1, 7, 49):
        tok, prob = call(x[r:r + 1], u[r], t[r], 40, 0.9, 0.02)
        assert tok[0] == all_at_once[r] and prob[0] == probs[r]
    a, _ = call(x, u)
    b, _ = call(x, u, 1.0, 0, 1.0, 0.0)
    assert (a == b).all()
    c, _ = call(x, None, np.zeros(50), probs=False)
    assert (c == x.float().argmax(-1).cpu().numpy()).all()


def test_in_a_graph():
    x, u = logits(30, 50000, seed=6)
    dev = torch.tensor(u, device="cuda")
    t, k, p = torch.full((30,), 0.8, device="cuda"), torch.full((30,), 30, dtype=torch.int32, device="cuda"), torch.full(
        (30,), 0.9, device="cuda")
    tok = torch.zeros(30, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        rpg.sample_rows(x.data_ptr(), rpg.F32, 30, 50000, tok.data_ptr(), dev.data_ptr(), t.data_ptr(), k.data_ptr(),
                        p.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    for seed in (1, 2):
        y, u = logits(30, 50000, seed=seed)
        x.copy_(y)
        dev.copy_(torch.tensor(u))
        g.replay()
        torch.cuda.synchronize()
        assert (tok.cpu().numpy() == call(y, u, 0.8, 30, 0.9)[0]).all()


def test_frequencies():
    # 20000 draws of one row: counts within 5 standard deviations of their means
    base = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5, -math.inf], device="cuda")
    n = 20000
    tok, _ = call(base.expand(n, 6).contiguous(), (np.arange(n) + 0.5) / n, 1.0)
    want = torch.softmax(base, 0).cpu().numpy() * n
    assert (np.abs(np.bincount(tok, minlength=6) - want) <= 1.5).all()  # (evenly spaced random numbers)
