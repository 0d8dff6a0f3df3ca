"""The paged batch example with conversations that branch off others, prompts in one call, and drawn tokens."""

import numpy as np
import pytest

from rpgbarenginecuda_b200 import Model, Session

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_paged_example import example  # noqa: E402


def near(got, want):
    assert float(np.abs(got.cpu().numpy() - want).max()) <= 1e-3 * float(np.abs(want).max())


@pytest.mark.parametrize("common", [16, 37, 100])
def test_branches_match_sessions(tiny_g4_model, common):
    """Conversations that begin alike, at a page's end and inside one: each row's logits are those of the whole
    conversation in a session of its own, within the engine's bound of 1e-3 of full scale."""
    path = tiny_g4_model
    m = example().PagedModel(path, "f16", n_pages=64, max_conversations=6, max_positions=512)
    eng = Model(path, 0, 512)
    rng = np.random.default_rng(common)
    start = rng.integers(0, eng.vocab, common + 5).tolist()
    root = m.open()
    m.forward([(root, t) for t in start])
    pages = len(m.free)
    ids = [m.branch(root, common) for _ in range(3)]
    assert pages - len(m.free) == 3 * (common % m.page > 0)  # whole pages are shared
    ids.append(root)
    alone = m.open()
    text = {c: start[:common] for c in ids[:3]} | {root: start, alone: []}
    sessions = {}
    prompts = {c: rng.integers(0, eng.vocab, 3 + 4 * i).tolist() for i, c in enumerate([*ids, alone])}
    # all prompts in one call, the conversations' tokens in turns
    rows = [(c, prompts[c][i]) for i in range(20) for c in prompts if i < len(prompts[c])]
    logits = m.forward(rows)
    nexts = {}
    for c in prompts:
        sessions[c] = Session(eng, 256)
        want = sessions[c].prefill(text[c] + prompts[c])
        near(logits[max(i for i, r in enumerate(rows) if r[0] == c)], want)
        nexts[c] = int(want.argmax())
    for step in range(8):
        if step == 4:  # the others live on
            m.close(root)
            del nexts[root]
        order = list(nexts)[::1 if step % 2 else -1]
        logits = m.forward([(c, nexts[c]) for c in order])
        for i, c in enumerate(order):
            want = sessions[c].prefill([nexts[c]])
            near(logits[i], want)
            nexts[c] = int(want.argmax())
    for c in list(nexts):
        m.close(c)
    assert len(m.free) == 64 and not m.used.any()


def test_branches_of_branches_and_refusals(tiny_model):
    m = example().PagedModel(tiny_model, "q8", n_pages=8, max_conversations=4, max_positions=64)
    a = m.open()
    m.forward([(a, t) for t in range(40)])
    b = m.branch(a)
    c = m.branch(b, 20)
    assert m.alike[a][0] == m.alike[b][0] == m.alike[c][0] and m.lengths[c] == 20
    with pytest.raises(ValueError):
        m.branch(c, 21)
    m.forward([(x, 7) for x in (a, b, c)])
    d = m.branch(c)  # shares more with c than c does with the others
    assert m.alike[c] == m.alike[d] and m.alike[c][0] != m.alike[a][0]
    before = list(m.free)
    with pytest.raises(RuntimeError, match="open"):
        m.branch(a, 32)
    assert m.free == before
    for x in (a, b, c, d):
        m.close(x)
    assert sorted(m.free) == list(range(8))


@pytest.mark.parametrize("args", [["--instructions", "50"], ["--instructions", "33", "--cache", "q4", "--temperature", "0.8",
                                                             "--top-k", "20", "--top-p", "0.9", "--min-p", "0.02"]])
def test_main_with_a_common_beginning(args, model_cache, capsys):
    out = example().main([*args, "--conversations", "3", "--steps", "4"])
    assert len(out) == 3 and all(len(v) == 5 and min(v) >= 0 for v in out.values())
    assert example().main([*args, "--conversations", "3", "--steps", "4"]) == out
    assert "tokens/s" in capsys.readouterr().out
