"""State of the paged batch example: what a call that raises leaves behind, its limits, and its stream."""

import numpy as np
import pytest

from rpgbarenginecuda_b200 import EngineError

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_paged_example import example  # noqa: E402


def model(path, **kw):
    return example().PagedModel(path, "f16", **{"n_pages": 5, "max_conversations": 2, "max_positions": 256, **kw})


def rows(c, n, seed):
    return [(c, int(t)) for t in np.random.default_rng(seed).integers(0, 200, n)]


def state(m):
    return dict(m.lengths), list(m.free), m.table.tolist()


def test_a_batch_that_does_not_fit_changes_nothing(tiny_model):
    """Two conversations in five pages; a batch of both that needs two more pages than there are."""
    m, calm = model(tiny_model), model(tiny_model)
    for x in (m, calm):
        a, b = x.open(), x.open()
        x.forward(rows(a, 40, 1))
        x.forward(rows(b, 14, 2))
    before = state(m)
    with pytest.raises(RuntimeError, match="no page"):
        m.forward(rows(a, 3, 3) + rows(b, 30, 4))
    assert state(m) == before
    batch = rows(a, 2, 5) + rows(b, 4, 6)
    assert torch.equal(m.forward(batch), calm.forward(batch))
    assert state(m) == state(calm)


def test_a_bad_token_changes_nothing(tiny_model):
    m, calm = model(tiny_model), model(tiny_model)
    for x in (m, calm):
        x.forward(rows(x.open(), 20, 1))
    before = state(m)
    with pytest.raises(EngineError):
        m.forward(rows(0, 15, 2) + [(0, m.embd.rows)])
    assert state(m) == before
    assert torch.equal(m.forward(rows(0, 3, 3)), calm.forward(rows(0, 3, 3)))


def test_the_last_position(tiny_model):
    """max_positions that is no multiple of the page: all of them work, the next one raises."""
    m = model(tiny_model, n_pages=10, max_positions=50)
    a = m.open()
    logits = m.forward(rows(a, 49, 1))
    assert torch.isfinite(logits).all()
    assert torch.isfinite(m.forward(rows(a, 1, 2))).all()
    before = state(m)
    with pytest.raises(RuntimeError, match="full"):
        m.forward(rows(a, 1, 3))
    assert state(m) == before


def test_all_conversations_open(tiny_model):
    m = model(tiny_model)
    m.open(), m.open()
    with pytest.raises(RuntimeError, match="open"):
        m.open()
    m.close(1)
    assert m.open() == 1


def test_on_another_stream(tiny_model):
    m, calm = model(tiny_model), model(tiny_model)
    a = (m.open(), calm.open())[0]
    side = torch.cuda.Stream()
    for n in (30, 1, 1, 9):
        want = calm.forward(rows(a, n, n))
        with torch.cuda.stream(side):
            got = m.forward(rows(a, n, n))
        side.synchronize()
        assert torch.equal(got, want)
