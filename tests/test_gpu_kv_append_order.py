"""append's norm and rotation round every product and sum on its own, in the order that include/rpg_b200.h gives; so
scales, codes and q equal, bit for bit, that order evaluated operation by operation in f32.  (The reciprocal root is
CUDA's, here and there.)"""

import pytest

import rpgbarenginecuda_b200 as rpg

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv import ACT, KIND, MOST  # noqa: E402

EPS = 1e-6


def sum_of_squares(x):
    """[..., D] f32 -> [..., 1]: the order of the additions is the operator's definition."""
    x = x * x
    if x.shape[-1] == 128:  # runs of four from the left; then runs 64, 32, 16, 8 and 4 values apart
        x = x.unflatten(-1, (32, 4))
        run = x[..., 0]
        for e in (1, 2, 3):
            run = run + x[..., e]
    else:  # values 32, 16, 8, 4, 2 and 1 apart
        run = x
    while run.shape[-1] > 1:
        half = run.shape[-1] // 2
        run = run[..., :half] + run[..., half:]
    return run


def norm_and_turn(x, w, rope, pos):
    r = torch.rsqrt(sum_of_squares(x) * (1.0 / x.shape[-1]) + torch.tensor(EPS, device=x.device))
    x = (x * r) * w
    a, b = x.chunk(2, -1)
    c, s = rope[pos.long()][:, None].chunk(2, -1)
    ac, bs = a * c, b * s
    bc, as_ = b * c, a * s
    return torch.cat([ac - bs, bc + as_], -1)


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("act", ["f32", "bf16"])
@pytest.mark.parametrize("n", [3, 4001])
def test_codes_are_those_of_the_order(kind, dim, act, n):
    n_heads, n_kv, page = 5, 3, 16
    g = torch.Generator(device="cuda").manual_seed(n)
    code, dt, _ = ACT[act]
    x = torch.randn(n, n_heads + 2 * n_kv, dim, generator=g, device="cuda")
    x = (x * torch.exp(torch.randn(n, n_heads + 2 * n_kv, 1, generator=g, device="cuda"))).to(dt)
    wq, wk = (1 + 0.2 * torch.randn(dim, generator=g, device="cuda") for _ in range(2))
    rope = torch.from_numpy(rpg.rope_table(n, dim)).cuda()
    pages = -(-n // page)
    row = {"f16": 2 * dim, "q8": dim, "q4": dim // 2}[kind]
    mem = [torch.zeros(pages, n_kv, page, row, dtype=torch.uint8, device="cuda") for _ in range(2)]
    sc = [torch.zeros(pages, n_kv, page, dim // 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    kv = rpg.PagedKv(KIND[kind], dim, n_kv, page, pages, *(t.data_ptr() for t in mem + sc))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    q = torch.empty(n, n_heads, dim, dtype=dt, device="cuda")
    rot = rpg.Rotary(rope.data_ptr(), n, wq.data_ptr(), wk.data_ptr(), EPS)
    kv.append(rpg.PageTable(table.data_ptr(), 1, pages), rot, code, x.data_ptr(), n_heads, pos.data_ptr(), n, q.data_ptr(),
              seq_ptr=seq.data_ptr())
    torch.cuda.synchronize()
    y = x.float()
    assert torch.equal(q, norm_and_turn(y[:, :n_heads], wq, rope, pos).to(dt))
    k, v = norm_and_turn(y[:, n_heads:n_heads + n_kv], wk, rope, pos), y[:, n_heads + n_kv:]
    for want, got, scale in ((k, mem[0], sc[0]), (v, mem[1], sc[1])):
        got = got.transpose(1, 2).reshape(-1, n_kv, row)[:n]
        if kind == "f16":
            assert torch.equal(got.contiguous().view(torch.float16), want.half())
            continue
        groups = want.unflatten(-1, (-1, 64))
        most = torch.tensor(1.0 / MOST[kind], dtype=torch.float32, device="cuda")
        d16 = (groups.abs().amax(-1) * most).clamp(max=65504.0).half()
        assert torch.equal(scale.transpose(1, 2).reshape(-1, n_kv, dim // 64)[:n], d16)
        d = d16.float()[..., None].expand_as(groups)
        c = torch.round(groups / d).clamp(-MOST[kind], MOST[kind]).flatten(-2).to(torch.int8)
        if kind == "q8":
            assert torch.equal(got.view(torch.int8), c)
        else:
            c = (c + 8).to(torch.uint8)
            assert torch.equal(got, c[..., 0::2] | (c[..., 1::2] << 4))
