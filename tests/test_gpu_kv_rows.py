"""Numbers of rows on both sides of the borders where append and gather lay their launches out anew: the same bits."""

import pytest

import rpgbarenginecuda_b200 as rpg

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_kv import ACT, KIND  # noqa: E402


@pytest.mark.parametrize("kind", ["f16", "q8", "q4"])
@pytest.mark.parametrize("heads", [(3, 1, 128), (2, 2, 128), (32, 8, 128), (6, 3, 64), (8, 1, 64)])
@pytest.mark.parametrize("act", ["f32", "f16"])
@pytest.mark.parametrize("n", [789, 790, 7104, 7107, 9601])
def test_rows_together_and_in_small_batches(kind, heads, act, n):
    n_heads, n_kv, dim = heads
    page, step = 64, 97
    code, dt, _ = ACT[act]
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, (n_heads + 2 * n_kv) * dim, generator=g, device="cuda").to(dt)
    w = 1 + 0.2 * torch.randn(dim, generator=g, device="cuda")
    rope = torch.from_numpy(rpg.rope_table(n, dim)).cuda()
    rot = rpg.Rotary(rope.data_ptr(), n, w.data_ptr(), w.data_ptr())
    pages = -(-n // page)
    table = torch.randperm(pages, generator=g, device="cuda").int()
    pt = rpg.PageTable(table.data_ptr(), 1, pages)
    pos, seq = torch.arange(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    row = {"f16": 2 * dim, "q8": dim, "q4": dim // 2}[kind]
    got = []
    for batch in (n, step):
        mem = [torch.zeros(pages, n_kv, page, row, dtype=torch.uint8, device="cuda") for _ in range(2)]
        sc = [torch.zeros(pages, n_kv, page, dim // 64, dtype=torch.float16, device="cuda") for _ in range(2)]
        kv = rpg.PagedKv(KIND[kind], dim, n_kv, page, pages, *(t.data_ptr() for t in mem + sc))
        q = torch.empty(n, n_heads * dim, dtype=dt, device="cuda")
        k, v = (torch.empty(n, n_kv * dim, dtype=dt, device="cuda") for _ in range(2))
        for i in range(0, n, batch):
            m = min(batch, n - i)
            kv.append(pt, rot, code, x[i].data_ptr(), n_heads, pos[i:].data_ptr(), m, q[i].data_ptr(), seq_ptr=seq.data_ptr())
        for i in range(0, n, batch):
            m = min(batch, n - i)
            kv.gather(pt, code, pos[i:].data_ptr(), m, k[i].data_ptr(), v[i].data_ptr(), seq_ptr=seq.data_ptr())
        torch.cuda.synchronize()
        got.append([*mem, *sc, q, k, v])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert torch.isfinite(got[0][4].float()).all()
    v = x[:, (n_heads + n_kv) * dim:].float()
    step = {"f16": 2.0 ** -11, "q8": 1.01 / 254, "q4": 1.01 / 14}[kind]  # half a code step of the largest value
    assert float((got[0][6].float() - v).abs().max()) <= (step + ACT[act][2]) * float(v.abs().max())
