"""Host logic of TreeSpecDecoder on the CPU: a toy engine, the operators by
their definitions."""
import pytest

torch = pytest.importorskip("torch")

import tree_stub as stub
from arc_chain_b200.runtime import tree_spec as ts

PROMPTS = [[5, 3, 9], [2, 2, 7, 11, 4, 1]]


@pytest.fixture
def toy_ops(monkeypatch):
    monkeypatch.setattr(ts.ops, "draw_tokens", stub.draw_tokens)
    monkeypatch.setattr(ts.ops, "verify_tree", stub.verify_tree)


def decoder(branches=(2, 2), temperature=0.0, draft_seed=0, lanes=2, **kw):
    draft = stub.ToyEngine(draft_seed) if branches else None
    return ts.TreeSpecDecoder(stub.ToyEngine(), draft, branches, lanes, temperature, use_graph=False, **kw)


@pytest.mark.parametrize("branches,draft_seed", [((2, 2), 0), ((3, 1, 1), 4), ((), 0)])
def test_greedy_rounds(toy_ops, branches, draft_seed):
    sd = decoder(branches, draft_seed=draft_seed)
    assert [t for t, _ in sd.generate(PROMPTS, 20)] == [stub.plain(p, 20) for p in PROMPTS]
    assert all(e.kv.pool.used <= 1 for e in (sd.t, sd.d) if e)  # the scratch page


@pytest.mark.parametrize("where", ["target", "draft", "second level"])
def test_an_error_word_ends_the_call(toy_ops, where):
    """A kernel that could not do its work says so in its buffers' error word:
    such a round's tokens are not returned."""
    sd = decoder((2, 2))
    bb = {"target": sd.tb, "draft": sd.db[0], "second level": sd.db[1]}[where]
    eng = sd.t if where == "target" else sd.d
    forward, calls = eng.forward, []

    def failing(b, B, with_logits=True):
        forward(b, B, with_logits)
        if b is bb:
            calls.append(0)
            if len(calls) == 2:
                bb.err.fill_(8)

    eng.forward = failing
    with pytest.raises(RuntimeError, match="0x8"):
        sd.generate(PROMPTS, 20)
    assert len(calls) == 2
    assert sd.t.kv.pool.used <= 1 and sd.d.kv.pool.used <= 1
    eng.forward = forward
    assert eng.check_errors() == 8  # stays readable
    # the next call starts from clear words, and leaves what it found
    assert [t for t, _ in sd.generate(PROMPTS, 20)] == [stub.plain(p, 20) for p in PROMPTS]
    assert eng.check_errors() == 8


def test_an_error_word_of_the_prompt_ends_the_call(toy_ops):
    sd = decoder((2,))
    sd.t._bufs["prompt"] = bb = type("B", (), {"err": torch.zeros(1, dtype=torch.int32)})()
    prefill = sd.t.prefill
    sd.t.prefill = lambda *a, **kw: (prefill(*a, **kw), bb.err.fill_(32))
    with pytest.raises(RuntimeError, match="0x20"):
        sd.generate(PROMPTS, 20)
    assert sd.rounds == 0 and sd.t.kv.pool.used <= 1
