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


@pytest.mark.parametrize("nq,heads,kv,dh,lanes,few", [(1, 64, 64, 128, 4000, True), (20, 64, 64, 16, 3200, False)])
def test_attn_tree_batches_of_short_lanes(nq, heads, kv, dh, lanes, few):
    """Lanes of few keys whose digits and sums fill a launch's workspace: the
    result is that of calls of fewer lanes, and a lane's is the definition's."""
    import numpy as np

    from arc_chain_b200 import spec
    from arc_chain_b200.ops import tree_ops as ops
    from arc_chain_b200.ops._lib import lib

    t_lim = 100 if few else 600
    # all of the lanes in one launch would pass 6 GB: they go in several
    per = (lib().arcb_attn_tree_ws(2, nq, heads, kv, dh, t_lim) - lib().arcb_attn_tree_ws(1, nq, heads, kv, dh, t_lim))
    assert lanes * per > 6 << 30
    g = torch.Generator("cuda").manual_seed(nq)
    I32, I64 = torch.int32, torch.int64
    i = lambda lo, hi, s, t=I64: torch.randint(lo, hi, s, generator=g, device="cuda", dtype=t)
    q = i(-1 << 18, 1 << 18, (lanes * nq, heads * dh))
    pages = 500
    K, V = (i(-1 << 18, 1 << 18, (pages, kv, 16, dh)) for _ in range(2))
    pt = i(0, pages, (lanes, t_lim // 16 + 1), I32)
    base, n_tree = i(0, t_lim - nq - 1, (lanes,), I32), i(0, nq + 1, (lanes,), I32)
    mask = i(0, 1 << 62, (lanes * nq,)) | 1
    err = torch.zeros(1, dtype=I32, device="cuda")

    def run(a, b):
        out = torch.full(((b - a) * nq, heads * dh), 77, dtype=I64, device="cuda")
        ops.attn_tree(q[a * nq:b * nq], K, V, pt[a:b], base[a:b], n_tree[a:b], mask[a * nq:b * nq], heads, kv, dh,
                      9000, b - a, nq, None, None, t_lim, err, o_out=out)
        return out

    got = run(0, lanes)
    assert torch.equal(got, torch.cat([run(a, min(lanes, a + 500)) for a in range(0, lanes, 500)]))
    assert int(err.item()) == 0
    for b in (0, lanes // 2, lanes - 1):
        t = int(base[b] + n_tree[b])
        rows = pt[b, :(t + 15) // 16].long()
        for h in (0, heads - 1):
            k, v = (c[rows, h * kv // heads].reshape(-1, dh)[:t].cpu().numpy() for c in (K, V))
            for j in (0, nq - 1):
                s = b * nq + j
                want = spec.tree_attention(q[s, h * dh:(h + 1) * dh].cpu().numpy(), k, v, int(base[b]), int(n_tree[b]),
                                           int(mask[s]), 9000)
                np.testing.assert_array_equal(got[s, h * dh:(h + 1) * dh].cpu().numpy(), want)


@pytest.mark.parametrize("kind", ["tree", "chain", "plain"])
def test_a_graph_left_in_a_cycle_does_not_end_a_capture(kind):
    """A decoder that an exception's traceback held is freed by Python's
    collector, at any allocation: not while another one is captured."""
    import gc

    from arc_chain_b200.runtime.spec_decode import SpecDecoder
    from arc_chain_b200.runtime.tree_spec import TreeSpecDecoder

    class Holder:
        pass

    host = gen.random_model(preset("micro_gqa"), 0)
    target, draft = engine(host), engine(host)
    prompt = gen.seeded_prompt(12, preset("micro_gqa").vocab, 21)
    old, x = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    x.add_(1)
    torch.cuda.synchronize()
    with torch.cuda.graph(old):
        x.add_(1)
    box, forward = [old], target.forward
    del old

    def littering(*a, **kw):
        if box and torch.cuda.is_current_stream_capturing():
            h = Holder()
            h.self, h.graph = h, box.pop()
            del h
            [[] for _ in range(20000)]  # the collector's allocation count passes its limit
        return forward(*a, **kw)

    target.forward = littering
    if kind == "tree":
        got = TreeSpecDecoder(target, draft, (2, 1), draft_temperature=0.0).generate([prompt], 20)[0]
    elif kind == "chain":
        got = SpecDecoder(target, draft, k=2).generate([prompt], 20)[0]
    else:
        got = target.generate(prompt, 20)
    assert not box and gc.isenabled()
    assert got == arcref.Model(host).generate(prompt, 20)
