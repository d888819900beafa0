"""What tree speculation checks and refuses, on the GPU."""
import pytest

torch = pytest.importorskip("torch")

from arc_chain_b200.formats import gen
from arc_chain_b200.models.config import preset
from arc_chain_b200.oracle import arcref

pytestmark = pytest.mark.gpu


def engine(host):
    from arc_chain_b200.models import dense
    from arc_chain_b200.runtime.engine import Engine

    return Engine(dense.from_host(host, "cuda"))


@pytest.mark.parametrize("where", ["target", "draft", "prompt"])
@pytest.mark.parametrize("use_graph", [False, True])
def test_an_error_word_ends_the_call(where, use_graph):
    """The word is set from the host, between a round and its reading."""
    from arc_chain_b200.runtime.tree_spec import TreeSpecDecoder

    host = gen.random_model(preset("micro_gqa"), 0)
    target, draft = engine(host), engine(host)
    prompt = gen.seeded_prompt(12, preset("micro_gqa").vocab, 21)
    want = arcref.Model(host).generate(prompt, 20)
    sd = TreeSpecDecoder(target, draft, (2, 1), draft_temperature=0.0, use_graph=use_graph)
    assert sd.generate([prompt], 20) == [want]
    run, rounds, at = sd._run, [], 0 if where == "prompt" else 2
    word = {"target": sd.tb, "draft": sd.db[0], "prompt": target.buffers(16)}[where].err

    def failing():
        run()
        rounds.append(0)
        if len(rounds) == 2:
            word.fill_(32)

    if where == "prompt":
        prefill = target.prefill
        target.prefill = lambda *a, **kw: (prefill(*a, **kw), word.fill_(32))
    sd._run = failing
    with pytest.raises(RuntimeError, match="0x20"):
        sd.generate([prompt], 20)
    assert len(rounds) == at
    assert (draft if where == "draft" else target).check_errors() == 32
    assert target.kv.pool.used <= 1 and draft.kv.pool.used <= 1
    sd._run = run
    if where == "prompt":
        target.prefill = prefill
    assert sd.generate([prompt], 20) == [want]
