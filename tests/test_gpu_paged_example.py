"""The paged batch example against the engine's own sessions."""

import importlib.util
import os

import numpy as np
import pytest

from rpgbarenginecuda_b200 import Model, Session

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("paged_batch", os.path.join(ROOT, "examples", "paged_batch.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("model", ["tiny_model", "tiny_g4_model"])
def test_logits_match_the_session(model, request):
    """Prompts of several conversations, then steps of all of them together: each row's logits are those of the
    conversation alone in a session, within the engine's own bound of 1e-3 of full scale (fp16 cache)."""
    path = request.getfixturevalue(model)
    m = example().PagedModel(path, "f16", n_pages=64, max_conversations=4, max_positions=512)
    eng = Model(path, 0, 512)
    rng = np.random.default_rng(3)
    rows = {}
    for n in (21, 1, 40):
        c = m.open()
        rows[c] = (rng.integers(0, eng.vocab, n).tolist(), Session(eng, 256))

    def near(got, want):
        assert float(np.abs(got.cpu().numpy() - want).max()) <= 1e-3 * float(np.abs(want).max())

    nexts = {}
    for c, (prompt, s) in rows.items():
        want = s.prefill(prompt)
        near(m.forward([(c, t) for t in prompt])[-1], want)
        nexts[c] = int(want.argmax())
    for _ in range(20):  # teacher-forced with the session's tokens
        logits = m.forward([(c, nexts[c]) for c in rows])
        for i, (c, (_, s)) in enumerate(rows.items()):
            want = s.prefill([nexts[c]])
            near(logits[i], want)
            nexts[c] = int(want.argmax())
    taken = len(m.free)
    for c in list(rows):
        m.close(c)
    assert len(m.free) == 64 and taken < 64


@pytest.mark.parametrize("cache", ["f16", "q8", "q4"])
def test_main_runs(cache, model_cache, capsys):
    out = example().main(["--cache", cache, "--conversations", "3", "--steps", "4"])
    assert sorted(out) == [0, 1, 2] and all(len(v) == 5 for v in out.values())
    assert "tokens/s" in capsys.readouterr().out
