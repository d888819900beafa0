"""Tree speculation end to end: greedy output equals the CPU oracle's, sampled
output equals a host simulation of the same rounds (oracle logits, integer
definitions of ``arc_chain_b200.spec``, the same random streams), and neither
the batch nor CUDA graphs change it."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from arc_chain_b200 import spec
from arc_chain_b200.formats import gen
from arc_chain_b200.models.config import preset
from arc_chain_b200.oracle import arcref

pytestmark = pytest.mark.gpu


def engine(host):
    from arc_chain_b200.models import dense
    from arc_chain_b200.runtime.engine import Engine

    return Engine(dense.from_host(host, "cuda"))


def simulate(tm, dm, prompt, max_tokens, branches, temp, dtemp, seed, request, eos=()):
    """The decoder's rounds on the host, node by node."""
    from arc_chain_b200.runtime import tree_spec as ts

    par, n = ts.tree_parents(branches), ts.tree_levels(branches)[-1][1]
    inv, dinv = ts.inverse_temperature(temp), ts.inverse_temperature(dtemp)
    caches = [m.new_cache() for m in (tm, dm) if m is not None]
    confirmed = [1] + list(prompt)
    for c in caches:
        for t in confirmed:
            c.forward(t)
    out, last, used = [], prompt[-1], 0

    def at(c, tokens, node):
        path = []
        while node >= 0:
            path.insert(0, node)
            node = par[node]
        c.truncate(len(confirmed))
        for j in path:
            lg = c.forward(max(0, int(tokens[j])))
        return lg

    while True:
        u = (gen.rng_u64(seed, ts.STREAM + request, 3 * n - 1, start=used) >> np.uint64(33)).astype(np.int64)
        used += 3 * n - 1
        ring = np.zeros(64, np.int64)
        for k in range(max(0, len(out) - 64), len(out)):
            ring[k & 63] = out[k]
        tokens, dl = np.full(n, last), [None] * n
        for i in range(n):
            kids = [c for c in range(n) if par[c] == i]
            if kids:
                dl[i] = at(caches[1], tokens, i)
                ids = spec.tree_history(tokens, par, ring, len(out), i)
                tokens[kids] = spec.draw_tokens(dl[i], ids, dinv, [u[c - 1] for c in kids])
        tl = [at(caches[0], tokens, i) for i in range(n)]
        path, nxt = spec.tree_verify(tl, dl, tokens, par, n, inv, dinv, u[n - 1:].reshape(n, 2), ring, len(out))
        new = [int(tokens[j]) for j in path[1:]] + [nxt]
        for c in caches:
            c.truncate(len(confirmed))
            for j in path:
                c.forward(int(tokens[j]))
        confirmed += [int(tokens[j]) for j in path]
        for t in new:
            out.append(t)
            if t in eos or len(out) >= max_tokens:
                return out
        last = new[-1]


@pytest.mark.parametrize("branches,same", [((3, 2, 1), False), ((1, 1, 1, 1), True), ((2, 2, 2, 2, 2), True),
                                           ((5,), False), ((), False)])
def test_greedy_equals_the_oracle(branches, same):
    from arc_chain_b200.runtime.tree_spec import TreeSpecDecoder

    cfg = preset("micro_gqa")
    host = gen.random_model(cfg, 0)
    target = engine(host)
    draft = engine(host if same else gen.random_model(cfg, 9)) if branches else None
    om = arcref.Model(host)
    prompts = [gen.seeded_prompt(12, cfg.vocab, 21), gen.seeded_prompt(37, cfg.vocab, 22)]
    for dt in (0.0, 1.0):
        sd = TreeSpecDecoder(target, draft, branches, lanes=2, draft_temperature=dt, seed=3)
        out = sd.generate(prompts, 30)
        for p, (toks, h) in zip(prompts, out):
            assert (toks, h) == om.generate(p, 30)
        if same and dt == 0.0:
            assert sd.acceptance == 1.0
        eos = out[0][0][7]
        again = TreeSpecDecoder(target, draft, branches, lanes=2, draft_temperature=dt, seed=8, use_graph=False)
        for p, (toks, h) in zip(prompts, again.generate(prompts, 25, eos=[eos])):
            assert (toks, h) == om.generate(p, 25, eos=[eos])
    assert target.check_errors() == 0 and (draft is None or draft.check_errors() == 0)
    assert target.kv.pool.used <= 1  # the scratch page


@pytest.mark.parametrize("branches,temp,dtemp", [((3, 2), 1.0, 1.0), ((2, 2, 1), 0.6, 1.2), ((1, 1, 1), 1.5, 0.0), ((), 0.9, 1.0)])
def test_sampled_equals_the_simulation(branches, temp, dtemp):
    from arc_chain_b200.runtime.tree_spec import TreeSpecDecoder

    cfg = preset("micro_gqa")
    ht, hd = gen.random_model(cfg, 0), gen.random_model(cfg, 0)
    hd.layers = hd.layers[:1] + hd.layers[:1]  # a draft that agrees now and then
    target, draft = engine(ht), engine(hd) if branches else None
    tm, dm = arcref.Model(ht), arcref.Model(hd) if branches else None
    prompts = [gen.seeded_prompt(9, cfg.vocab, 31), gen.seeded_prompt(20, cfg.vocab, 32), gen.seeded_prompt(1, cfg.vocab, 33)]
    sd = TreeSpecDecoder(target, draft, branches, 3, temp, dtemp, seed=5)
    out = sd.generate(prompts, 24)
    for i, (p, (toks, _)) in enumerate(zip(prompts, out)):
        assert toks == simulate(tm, dm, p, 24, branches, temp, dtemp, 5, i), i
    assert sd.generate(prompts, 24) == out                       # the same seed, the same tokens
    solo = TreeSpecDecoder(target, draft, branches, 1, temp, dtemp, seed=5, use_graph=False)
    assert solo.generate(prompts[:1], 24) == out[:1]
    other = TreeSpecDecoder(target, draft, branches, 3, temp, dtemp, seed=6)
    assert other.generate(prompts, 24) != out
    assert target.check_errors() == 0 and (draft is None or draft.check_errors() == 0)
    assert target.kv.pool.used <= 1


def test_the_longest_request_and_one_beyond():
    """The last positions of max_seq, which is no multiple of a page here."""
    from arc_chain_b200.models import dense
    from arc_chain_b200.runtime.engine import Engine
    from arc_chain_b200.runtime.tree_spec import TreeSpecDecoder

    cfg = preset("micro_gqa")
    host = gen.random_model(cfg, 0)
    target, draft = (Engine(dense.from_host(host, "cuda"), max_seq=m) for m in (77, 73))
    p = gen.seeded_prompt(40, cfg.vocab, 5)
    sd = TreeSpecDecoder(target, draft, (2, 2), 1, draft_temperature=0.0)
    toks, _ = sd.generate([p], 73 - 41 - 7)[0]
    assert toks == arcref.Model(host).generate(p, 73 - 41 - 7)[0]
    with pytest.raises(ValueError, match="max_seq 73"):
        sd.generate([p], 73 - 41 - 6)
    assert target.check_errors() == 0 and draft.check_errors() == 0 and target.kv.pool.used <= 1


def test_command_line_samples(capsys):
    import json

    from arc_chain_b200 import cli

    def run(*extra):
        argv = ["generate", "--prompt-ids", "5,9,17", "--max-tokens", "12", "--set", "model=micro_gqa"]
        for x in extra:
            argv += ["--set", x]
        assert cli.main(argv) == 0
        return json.loads(capsys.readouterr().out.strip().splitlines()[-1])

    greedy = run()
    tree = run("draft=micro_gqa", "spec_tree=2,2", "draft_temperature=0")
    assert tree["output_hash_blake3"] == greedy["output_hash_blake3"]
    a, b = run("temperature=0.8", "sample_seed=3"), run("temperature=0.8", "sample_seed=3")
    assert a["output_hash_blake3"] == b["output_hash_blake3"] != greedy["output_hash_blake3"]
