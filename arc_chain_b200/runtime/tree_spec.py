"""Speculative decoding with a tree of drafted tokens, greedy or sampled.

The reference decodes greedily only; with temperature 0 the output equals its
greedy step's (crates/arc-inference/src/cached_integer_model.rs:1518-1557) token
for token, like ``runtime.spec_decode``.  With a temperature the tokens follow
the target's own distribution (softmax of its penalised logits over the
temperature, in the exact integers of csrc/kernels/draw_ops.cu), whatever the
draft proposes, to within the 2^-31 that probabilities and random numbers are
held to.  Random numbers come from the seeded SplitMix64 streams of
``formats.gen``, one stream per request, so a run is a function of the
model, the prompts and the seed (its low 32 bits): neither the other requests
of the batch nor CUDA graphs change it.

A round, per lane (request), with branches (b_1, ..., b_L):

1. the draft runs the root (the last confirmed token) and draws b_1 children
   from its distribution without replacement, then b_2 for each of those, and
   so on: a level is one forward of the draft over its nodes, whose K/V rows
   follow the confirmed prefix in the order of the nodes;
2. the target runs all nodes in one forward (RoPE positions by depth, attention
   over the prefix and each node's own path);
3. the accepted path and the token behind it are decided on the device;
4. the path's K/V rows move to their positions in both caches.

With branches () there is no draft: plain sampled decoding.  The draft never
runs the deepest level; where the path ends there, it is fed that token before
the next round.  With tensor parallelism the draft, the drawing and the
decision run on rank 0 of the target's communicator and are broadcast over its
group; every rank runs the target's forward.  Every rank builds the decoder and
calls generate with the same arguments (only rank 0 needs the draft); where one
rank refuses or fails outside the target's forward, all of them raise before the
next collective.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass, field
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from arc_chain_b200.formats import gen
from arc_chain_b200.ops import tree_ops as ops
from arc_chain_b200.runtime.engine import Engine, I32, I64, capturing
from arc_chain_b200.spec import check_temperature
from arc_chain_b200.utils.hashing import blake3

ONE = 1 << 16
STREAM = 0x54524545  # random streams of the requests: STREAM + request


def tree_levels(branches: Sequence[int]) -> List[Tuple[int, int]]:
    """[first, last) node of each level of a tree that is numbered level by
    level, children of one node next to each other."""
    levels = [(0, 1)]
    for b in branches:
        if b < 1:
            raise ValueError(f"every level has at least one child per node, got {tuple(branches)}")
        a, e = levels[-1]
        levels.append((e, e + (e - a) * b))
    if levels[-1][1] > ops.MAX_NODES:
        raise ValueError(f"branches {tuple(branches)} make {levels[-1][1]} nodes; a tree has at most {ops.MAX_NODES}")
    return levels


def tree_parents(branches: Sequence[int]) -> List[int]:
    par = [-1]
    for (a, _), (s, e), b in zip(tree_levels(branches), tree_levels(branches)[1:], branches):
        par += [a + i // b for i in range(e - s)]
    return par


def inverse_temperature(t: float) -> int:
    """Q16 inverse temperature, the nearest that the operators use; 0 is greedy."""
    if not t >= 0:
        raise ValueError(f"a temperature is at least 0, got {t}")
    return 0 if t == 0 else max(1, round(min(ops.MAX_INV_TEMP, ONE / t)))


@dataclass
class _Lane:
    rid_t: int
    rid_d: int
    max_tokens: int
    stream: int
    prompt: List[int]                                 # with BOS
    gen: List[int] = field(default_factory=list)
    last: int = 0
    pos: int = 0
    drawn: int = 0                                    # random numbers used
    pending: List[int] = field(default_factory=list)  # tokens the draft has not consumed
    done: bool = False


class TreeSpecDecoder:
    def __init__(self, target: Engine, draft: Optional[Engine] = None, branches: Sequence[int] = (3, 2, 1),
                 lanes: int = 1, temperature: float = 0.0, draft_temperature: float = 1.0, seed: int = 0,
                 use_graph: bool = True):
        self._dense(target)
        self.cm = target.comm
        self.leads, self.group = self.cm.rank == 0, getattr(self.cm, "group", None)
        self.dev = target.m.emb.device
        with self._together():
            self._build(target, draft, branches, lanes, temperature, draft_temperature, seed, use_graph)

    @staticmethod
    def _dense(e) -> None:
        if not getattr(e, "runs_trees", False):
            raise TypeError(f"tree speculation runs dense engines, got {type(e).__name__}")

    def _build(self, target, draft, branches, lanes, temperature, draft_temperature, seed, use_graph) -> None:
        if draft is not None:
            self._dense(draft)
        check_temperature(temperature)
        check_temperature(draft_temperature)
        if lanes < 1:
            raise ValueError(f"lanes must be at least 1, got {lanes}")
        self.branches = tuple(int(b) for b in branches)
        self.t, self.n_lanes, self.seed, self.use_graph = target, lanes, seed, use_graph
        if self.branches and self.leads and draft is None:
            raise ValueError("a tree of drafted tokens needs a draft engine")
        if draft is not None and draft.m.cfg.vocab != target.m.cfg.vocab:
            raise ValueError("target and draft must share a vocabulary")
        self.d = draft if self.branches and self.leads else None
        if self.d is not None and self.d.m.emb.device != self.dev:
            raise ValueError(f"target and draft share a device, got {self.dev} and {self.d.m.emb.device}")
        if self.d is not None and self.d.comm.size > 1:
            raise ValueError("the draft runs on one rank: its engine takes no communicator")
        self.levels = tree_levels(self.branches)
        self.n = n = self.levels[-1][1]
        dev = self.dev
        par = tree_parents(self.branches)
        depth, mask = [], []
        for i, p in enumerate(par):
            depth.append(0 if p < 0 else depth[p] + 1)
            mask.append((0 if p < 0 else mask[p]) | 1 << i)
        signed = [m - (1 << 64) if m >> 63 else m for m in mask]
        self.parent = torch.tensor([par] * lanes, dtype=I32, device=dev)
        self.depth = torch.tensor(depth, dtype=I32, device=dev)
        self.node = torch.arange(n, dtype=I32, device=dev)
        self.mask = torch.tensor(signed, dtype=I64, device=dev)
        V = target.m.cfg.vocab
        self.tb = target.tree_buffers(lanes, n)
        self.db = [self.d.tree_buffers(lanes, b - a) for a, b in self.levels[:-1]] if self.d is not None else []
        z = lambda *s, dt=I32: torch.zeros(*s, dtype=dt, device=dev)
        self.pos, self.live, self.root = z(lanes), z(lanes), z(lanes)
        self.tokens = z(lanes, n)
        self.hist, self.count = z(lanes, 64), z(lanes)
        self.inv = torch.full((lanes,), inverse_temperature(temperature), dtype=I64, device=dev)
        self.dinv = torch.full((lanes,), inverse_temperature(draft_temperature), dtype=I64, device=dev)
        self.dlogits = z(lanes * n, V, dt=I64) if self.branches and self.leads else None
        # random numbers of a round: one per drafted node (its drawing), then two per node (its verification)
        self.u_draw = [z(lanes * (b - a), k) for (a, b), k in zip(self.levels, self.branches)]
        self.u_ver = z(lanes, n, 2)
        self.path, self.n_path, self.nxt = z(lanes, n), z(lanes), z(lanes)
        self._graph = None
        self.rounds = self.proposed = self.accepted = 0

    # ------------------------------------------------------------ ranks
    def _agree(self, x: int, least: bool) -> int:
        """The least or the largest of the ranks' numbers."""
        if self.cm.size == 1:
            return x
        import torch.distributed as dist

        t = torch.tensor([x], dtype=I64, device=self.dev)
        dist.all_reduce(t, dist.ReduceOp.MIN if least else dist.ReduceOp.MAX, group=self.group)
        return int(t.item())

    @contextmanager
    def _together(self):
        """A part that every rank enters and that holds no collective: where it
        raises on one rank, it raises on all."""
        err: Optional[Exception] = None
        try:
            yield
        except Exception as e:
            err = e
        try:
            if self._agree(int(err is not None), False) and err is None:
                err = RuntimeError("tree speculation failed on another rank")
        except Exception as e:
            raise e if err is None else err
        if err is not None:
            raise err

    def _broadcast(self, *tensors: torch.Tensor) -> None:
        if self.cm.size > 1:
            import torch.distributed as dist

            for x in tensors:
                dist.broadcast(x, group=self.group, group_src=0)

    # ------------------------------------------------------------ device side
    def _set(self, bb, a: int, b: int) -> None:
        """Node range [a, b) of every lane into a forward's buffers."""
        L, w = self.n_lanes, b - a
        live = self.live[:, None]
        bb.tokens.view(L, w).copy_(self.tokens[:, a:b].clamp(min=0))  # -1: nothing was left to draw
        bb.pos.view(L, w).copy_(live * (self.pos[:, None] + self.depth[a:b]))
        bb.kv_pos.view(L, w).copy_(live * (self.pos[:, None] + self.node[a:b]))
        bb.tree.base.copy_(self.pos * self.live)
        bb.tree.n_tree.copy_(self.live * b)
        bb.tree.mask.view(L, w).copy_(self.mask[a:b].expand(L, w))

    def _draft(self) -> None:
        L, n, V = self.n_lanes, self.n, self.t.m.cfg.vocab
        for (a, b), (s, e), k, bb, u in zip(self.levels, self.levels[1:], self.branches, self.db, self.u_draw):
            self._set(bb, a, b)
            self.d.forward(bb, bb.B, True)
            self.dlogits.view(L, n, V)[:, a:b].copy_(bb.logits.view(L, b - a, V))
            out = torch.empty(L * (b - a), k, dtype=I32, device=u.device)
            ops.draw_tokens(bb.logits, V, L, b - a, a, k, self.dinv, u, self.hist, self.count, self.tokens,
                            self.parent, out)
            self.tokens[:, s:e].copy_(out.view(L, e - s))

    def _decide(self) -> None:
        d = self.dlogits if self.dlogits is not None else self.tb.logits
        ops.verify_tree(self.tb.logits, d, self.t.m.cfg.vocab, self.n_lanes, self.n, self.tokens, self.parent,
                        self.tb.tree.n_tree, self.inv, self.dinv, self.u_ver, self.hist, self.count, self.path,
                        self.n_path, self.nxt)

    def _keep(self, eng: Engine, bb) -> None:
        eng.kv.keep_path(bb.pt[::bb.tree.nq], bb.tree.base, self.path, self.n_path, self.n_lanes, self.n, bb.err)

    def _propose(self) -> None:
        self.tokens[:, 0].copy_(self.root)
        if self.db:
            self._draft()

    def _verify(self) -> None:
        self._broadcast(self.tokens)
        self._set(self.tb, 0, self.n)
        self.t.forward(self.tb, self.tb.B, True)
        with self._together():
            if self.leads:
                self._decide()
        self._broadcast(self.path, self.n_path, self.nxt)

    def _settle(self) -> None:
        if self.branches:
            self._keep(self.t, self.tb)
            if self.db:
                self._keep(self.d, self.db[0])

    def _round(self) -> None:
        self._propose()
        self._verify()
        self._settle()

    def _run(self) -> None:
        if not self.use_graph:
            self._round()
            return
        if self._graph is None:
            # a first round with every lane idle: it sets the kernels'
            # attributes and writes no request's rows
            live = self.live.clone()
            saved = [bb.pt.clone() for bb in (self.tb, *self.db)]
            self.live.zero_()
            for bb, e in ((self.tb, self.t), *((x, self.d) for x in self.db)):
                bb.pt.copy_(torch.tensor(e.kv.table_row(e.scratch_rid), dtype=I32).expand_as(bb.pt))
            self._round()
            torch.cuda.synchronize()
            for bb, s in zip((self.tb, *self.db), saved):
                bb.pt.copy_(s)
            self.live.copy_(live)
            g = torch.cuda.CUDAGraph()
            with capturing(g):
                self._round()
            self._graph = g
        self._graph.replay()

    # ------------------------------------------------------------ host side
    def _error_words(self) -> List[torch.Tensor]:
        """The error words of every buffer of the engines: a round's, and the prompts'."""
        engines = [self.t] if self.d is None or self.d is self.t else [self.t, self.d]
        return [bb.err for e in engines for bb in e._bufs.values()]

    def _read(self, *tensors: torch.Tensor) -> List[np.ndarray]:
        """Copies of int32 tensors on the host, in one transfer with the error words.  Raises
        where a kernel reported that it could not do its work (a page or a length out of
        range, a wait that ran out): the tokens behind that are not the model's."""
        parts = [t.reshape(-1) for t in (*tensors, *self._error_words())]
        flat = torch.cat(parts).cpu().numpy()
        ends = np.cumsum([len(p) for p in parts[:len(tensors)]], dtype=np.int64)
        bits = int(np.bitwise_or.reduce(flat[ends[-1] if len(ends) else 0:]))
        if bits:
            raise RuntimeError(f"a kernel reported an error (error bits {bits:#x})")
        return [x.reshape(t.shape) for x, t in zip(np.split(flat, ends), tensors)]

    def _numbers(self, ln: _Lane, k: int) -> np.ndarray:
        r = gen.rng_u64(self.seed, ln.stream, k, start=ln.drawn)
        ln.drawn += k
        return (r >> np.uint64(33)).astype(np.int32)

    def _upload(self, lanes: List[_Lane]) -> None:
        L, n = self.n_lanes, self.n
        I = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32))
        self.pos.copy_(I([0 if ln.done else ln.pos for ln in lanes]))
        self.live.copy_(I([0 if ln.done else 1 for ln in lanes]))
        self.root.copy_(I([0 if ln.done else ln.last for ln in lanes]))
        ring = np.zeros((L, 64), np.int32)
        for i, ln in enumerate(lanes):
            for k in range(max(0, len(ln.gen) - 64), len(ln.gen)):
                ring[i, k & 63] = ln.gen[k]
        self.hist.copy_(I(ring))
        self.count.copy_(I([len(ln.gen) for ln in lanes]))
        draws, ver = [[] for _ in self.u_draw], np.zeros((L, n, 2), np.int32)
        for i, ln in enumerate(lanes):
            u = np.zeros(3 * n - 1, np.int32) if ln.done else self._numbers(ln, 3 * n - 1)
            for k, (s, e) in enumerate(self.levels[1:]):
                draws[k].append(u[s - 1:e - 1])
            ver[i] = u[n - 1:].reshape(n, 2)
        for t, u in zip(self.u_draw, draws):
            t.copy_(I(np.concatenate(u).reshape(t.shape)))
        self.u_ver.copy_(torch.from_numpy(ver))
        for bb, e, rid in ((self.tb, self.t, "rid_t"), *((x, self.d, "rid_d") for x in self.db)):
            idle = e.kv.table_row(e.scratch_rid)
            rows = [idle if ln.done else e.kv.table_row(getattr(ln, rid)) for ln in lanes]
            bb.pt.copy_(I(np.repeat(rows, bb.tree.nq, 0)))

    def _step(self, lanes: List[_Lane], eos: set) -> None:
        one = self.cm.size == 1
        with self._together():
            if self.db:
                for ln in lanes:
                    if not ln.done and ln.pending:
                        self.d.prefill(ln.rid_d, ln.pending, start_pos=ln.pos - len(ln.pending))
                        ln.pending = []
            self._upload(lanes)
            if one:
                self._run()
            else:
                self._propose()
        if not one:
            self._verify()
        with self._together():
            if not one:
                self._settle()
            path, n_path, nxt, tokens = self._read(self.path, self.n_path, self.nxt, self.tokens)
        self.rounds += 1
        for i, ln in enumerate(lanes):
            if ln.done:
                continue
            k = int(n_path[i])
            new = [int(tokens[i, j]) for j in path[i, 1:k]] + [int(nxt[i])]
            self.proposed += len(self.branches)
            self.accepted += k - 1
            for tok in new:
                ln.gen.append(tok)
                if tok in eos or len(ln.gen) >= ln.max_tokens:
                    ln.done = True
                    break
            if not ln.done:
                # the draft has run every level but the deepest
                ln.pending = [new[-2]] if self.branches and k == len(self.levels) else []
                ln.last = new[-1]
                ln.pos += k

    def generate(self, prompts: Sequence[Sequence[int]], max_tokens: int, eos: Sequence[int] = ()) \
            -> List[Tuple[List[int], bytes]]:
        """Tokens and output hash of each prompt.  Request i of a call uses
        random stream i of the decoder's seed.  A request takes positions for
        its prompt, max_tokens and one tree, up to the engines' max_seq.
        Raises RuntimeError, with no tokens of any prompt, where a kernel
        reports an error."""
        most = self._agree(min(e.max_seq for e in (self.t, self.d) if e is not None), True)
        lanes: List[_Lane] = []
        before: List[Tuple[torch.Tensor, torch.Tensor]] = []
        try:
            with self._together():
                if len(prompts) != self.n_lanes:
                    raise ValueError(f"one prompt per lane: {self.n_lanes} lanes, {len(prompts)} prompts")
                for p in prompts:
                    if 1 + len(p) + max_tokens + self.n > most:
                        raise ValueError(f"a prompt of {len(p)} tokens, {max_tokens} new ones and a tree of {self.n} "
                                         f"nodes exceed max_seq {most}")
                ends = set(int(e) for e in eos)
                before = [(w, w.clone()) for w in self._error_words()]  # other calls' errors stay readable
                for w, _ in before:
                    w.zero_()
                for i, p in enumerate(prompts):
                    p = [int(x) for x in p]
                    need = 1 + len(p) + max_tokens + self.n
                    ln = _Lane(self.t.new_request(need), -1, max_tokens, STREAM + i, [1] + p, last=p[-1] if p else 0,
                               pos=len(p) + 1, done=max_tokens <= 0)
                    lanes.append(ln)
                    if self.db:
                        ln.rid_d = self.d.new_request(need)
                        self.d.prefill(ln.rid_d, ln.prompt)
            for ln in lanes:
                self.t.prefill(ln.rid_t, ln.prompt)
            with self._together():
                self._read()
            while not all(ln.done for ln in lanes):
                self._step(lanes, ends)
        finally:
            for ln in lanes:
                self.t.kv.release(ln.rid_t)
                if ln.rid_d >= 0:
                    self.d.kv.release(ln.rid_d)
            for w, b in before:
                w.bitwise_or_(b)
        return [(ln.gen, blake3(np.asarray(ln.gen, dtype="<u4").tobytes())) for ln in lanes]

    @property
    def acceptance(self) -> float:
        """Accepted drafted tokens over the tree's depth, mean of the rounds."""
        return self.accepted / max(1, self.proposed)
