"""Host logic of TreeSpecDecoder on the CPU: a toy engine, the operators by
their definitions, tensor parallelism as gloo ranks."""
import datetime
import os
import socket
import time

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


# ------------------------------------------------------------ ranks
def _fail(*a, **kw):
    raise MemoryError("planted")


def _call(comm, fault):
    """A call on this rank, with a fault planted in it: its tokens or its
    error, and whether the pages are free again."""
    leads, verify = comm.rank == 0, stub.verify_tree
    target, draft = stub.ToyEngine(0, comm=comm), stub.ToyEngine(3, max_seq=48 if fault == "limit" else 128)
    if fault == "request" and leads:
        draft.new_request = _fail
    if fault == "prompt" and leads:
        draft.prefill = _fail
    if fault == "level" and leads:
        draft.forward = _fail
    if fault == "kept rows" and leads:
        draft.kv.keep_path = _fail
    if fault == "pages" and not leads:
        target.kv.pool.free = target.kv.pool.free[:2]
    ts.ops.draw_tokens, ts.ops.verify_tree = stub.draw_tokens, _fail if fault == "decision" and leads else verify
    used = target.kv.pool.used
    try:
        sd = ts.TreeSpecDecoder(target, draft if leads and fault != "no draft" else None, (2, 2), 2, 0.9, seed=4)
        if fault == "word" and not leads:
            forward = target.forward
            target.forward = lambda *a: (forward(*a), sd.tb.err.fill_(8))
        out = [t for t, _ in sd.generate(PROMPTS, 20 if fault != "limit" else 40)]
    except (ValueError, MemoryError, RuntimeError) as e:
        out = f"{type(e).__name__}: {e}"
    return out, target.kv.pool.used <= used + 1 and draft.kv.pool.used <= 1


def _worker(rank, world, port, group_ranks, faults, q):
    import torch.distributed as dist

    from arc_chain_b200.parallel.tp import NcclComm

    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=15))
    try:
        group = dist.new_group(group_ranks) if group_ranks else None
        if group_ranks and rank not in group_ranks:
            q.put((rank, None))
            return
        comm = NcclComm(group)
        q.put((rank, {f: _call(comm, f) for f in faults}))  # each on the same group: in step all along
    finally:
        dist.destroy_process_group()


def _ranks(faults, group_ranks=()):
    import multiprocessing as mp

    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    ctx, world = mp.get_context("spawn"), 3 if group_ranks else 2
    q = ctx.Queue()
    ps = [ctx.Process(target=_worker, args=(r, world, port, list(group_ranks), faults, q)) for r in range(world)]
    for p in ps:
        p.start()
    res, t0 = {}, time.time()
    while len(res) < world and time.time() - t0 < 120:
        try:
            r, v = q.get(timeout=1)
            res[r] = v
        except Exception:
            pass
    for p in ps:
        p.join(timeout=30)
        if p.is_alive():
            p.kill()
    assert [p.exitcode for p in ps] == [0] * world and len(res) == world
    return [res[r] for r in range(world)]


FAULTS = {
    "limit": ("ValueError: a prompt of 3 tokens, 40 new ones and a tree of 7 nodes exceed max_seq 48",) * 2,
    "no draft": ("ValueError: a tree of drafted tokens needs a draft engine", "RuntimeError: tree spec"),
    "request": ("MemoryError: planted", "RuntimeError: tree spec"),
    "prompt": ("MemoryError: planted", "RuntimeError: tree spec"),
    "level": ("MemoryError: planted", "RuntimeError: tree spec"),
    "decision": ("MemoryError: planted", "RuntimeError: tree spec"),
    "kept rows": ("MemoryError: planted", "RuntimeError: tree spec"),
    "pages": ("RuntimeError: tree spec", "MemoryError: KV cache out of pages"),
    "word": ("RuntimeError: tree spec", "RuntimeError: a kernel reported an error (error bits 0x8)"),
}


@pytest.fixture(scope="module")
def two_ranks():
    return _ranks([*FAULTS, "none"])


def test_ranks_equal_one_process(toy_ops, two_ranks):
    """Also behind failed calls, and over a communicator of some of the ranks,
    whose first is not the world's."""
    want = [t for t, _ in decoder((2, 2), 0.9, 3, seed=4).generate(PROMPTS, 20)]
    assert [r["none"] for r in two_ranks] == [(want, True)] * 2
    some = _ranks(["none"], (1, 2))
    assert some == [None, {"none": (want, True)}, {"none": (want, True)}]


@pytest.mark.parametrize("fault", FAULTS)
def test_ranks_fail_together(two_ranks, fault):
    """What one rank refuses or fails at ends the call on both."""
    for r, want in zip(two_ranks, FAULTS[fault]):
        out, released = r[fault]
        assert isinstance(out, str) and out.startswith(want) and released


def test_a_rank_that_cannot_ask_the_others_raises_its_own_error(toy_ops):
    sd = decoder((2,))

    def lost(*a):
        raise RuntimeError("connection closed")

    sd._agree = lost
    with pytest.raises(RuntimeError, match="connection closed"):
        with sd._together():
            pass
    with pytest.raises(MemoryError, match="planted"):
        with sd._together():
            _fail()


# ------------------------------------------------------------ refusals
def test_latent_attention_engines_are_refused(toy_ops):
    """They share the dense engine's class, but neither its cache rows nor its buffers."""
    from arc_chain_b200.models.mla_moe_engine import MlaMoeEngine

    mla = object.__new__(MlaMoeEngine)
    mla.m = stub.ToyEngine().m
    mla.comm, mla.max_pages, mla._bufs = stub.Comm(), 8, {}
    for target, draft in ((mla, None), (stub.ToyEngine(), mla)):
        with pytest.raises(TypeError, match="MlaMoeEngine"):
            ts.TreeSpecDecoder(target, draft, (2, 2) if draft else (), 1)
    with pytest.raises(TypeError, match="MlaMoeEngine"):
        mla.tree_buffers(1, 4)


@pytest.mark.parametrize("t", [1e-9, 1e-310, 0.01, 0.0624, 65537.0, 1e9, float("inf"), float("nan"), -1.0])
def test_temperatures_that_would_be_another(toy_ops, t):
    """Inverse temperatures are Q16 up to 16: 0.01 would be sampled as 1/16, 1e9 as 65536."""
    from arc_chain_b200.config import RunConfig

    for kw in (dict(temperature=t), dict(draft_temperature=t)):
        with pytest.raises(ValueError, match="temperature"):
            decoder((2, 2), **kw)
        with pytest.raises(ValueError, match="temperature"):
            RunConfig(**kw)


@pytest.mark.parametrize("t", [0.0, 1 / 16, 0.7, 1, 65536.0])
def test_temperatures_that_are_taken(toy_ops, t):
    from arc_chain_b200.config import RunConfig

    sd = decoder((2,), temperature=t, draft_temperature=t)
    assert sd.inv.tolist() == sd.dinv.tolist() == [0 if t == 0 else round(65536 / t)] * 2
    assert RunConfig(temperature=t, draft_temperature=t).temperature == t


def test_engines_on_two_devices_are_refused(toy_ops):
    target, draft = stub.ToyEngine(), stub.ToyEngine()
    draft.m.emb = torch.zeros(1, device="meta")
    with pytest.raises(ValueError, match="device"):
        ts.TreeSpecDecoder(target, draft, (2,), 1)
