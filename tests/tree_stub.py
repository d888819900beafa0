"""A dense engine's stand-in on the CPU for the tests of TreeSpecDecoder's host
logic: a model whose logits are a function of the tokens that a node attends
(read from the paged cache through its mask, so a row that is out of place
shows), and the operators by their definitions in ``arc_chain_b200.spec``."""
from types import SimpleNamespace

import numpy as np
import torch

from arc_chain_b200 import spec
from arc_chain_b200.formats import gen
from arc_chain_b200.runtime.engine import Comm, TreeStep
from arc_chain_b200.runtime.kv_paged import PAGE, PagedKV

VOCAB = 13


def toy_logits(tokens, seed: int) -> np.ndarray:
    """Q16 logits behind a sequence of tokens."""
    h = seed
    for t in tokens:
        h = (h * 31 + int(t) + 7) % (1 << 20)
    return (gen.rng_u64(seed, 900 + h, VOCAB) % np.uint64(4 << 16)).astype(np.int64)


class ToyEngine:
    runs_trees = True

    def __init__(self, seed: int = 0, max_seq: int = 128, comm=None, n_pages: int = 64):
        self.m = SimpleNamespace(emb=torch.zeros(1), cfg=SimpleNamespace(vocab=VOCAB))
        self.seed, self.max_seq, self.comm = seed, max_seq, comm or Comm()
        self.max_pages = (max_seq + PAGE - 1) // PAGE
        self.kv = PagedKV(1, n_pages, 1, 2, "cpu", self.max_pages)
        self.kv.keep_path = self._keep_path
        self._bufs, self._rid, self._scratch = {}, 0, None

    def tree_buffers(self, lanes, nq):
        if (lanes, nq) not in self._bufs:
            B, z = lanes * nq, lambda *s: torch.zeros(*s, dtype=torch.int32)
            self._bufs[lanes, nq] = SimpleNamespace(
                B=B, tokens=z(B), pos=z(B), kv_pos=z(B), pt=z(B, self.max_pages), err=z(1),
                logits=torch.zeros(B, VOCAB, dtype=torch.int64), tree=TreeStep(lanes, nq, "cpu"))
        return self._bufs[lanes, nq]

    def check_errors(self):
        return int(sum(bb.err.item() for bb in self._bufs.values()))

    def new_request(self, n):
        self._rid += 1
        self.kv.reserve(self._rid, n)
        return self._rid

    @property
    def scratch_rid(self):
        if self._scratch is None:
            self._scratch = self.new_request(1)
        return self._scratch

    def _row(self, table, at):
        return self.kv.K[0][int(table[at // PAGE]), 0, at % PAGE]

    def prefill(self, rid, tokens, start_pos=0):
        for i, t in enumerate(tokens):
            self._row(self.kv.table_row(rid), start_pos + i)[0] = t

    def forward(self, bb, B, with_logits=True):
        for s in range(B):
            self._row(bb.pt[s], int(bb.kv_pos[s]))[0] = bb.tokens[s]
        for s in range(B):
            lane = s // bb.tree.nq
            base, nodes, mask = int(bb.tree.base[lane]), int(bb.tree.n_tree[lane]), int(bb.tree.mask[s])
            seen = list(range(base)) + [base + j for j in range(nodes) if mask >> j & 1]
            assert not seen or int(bb.pos[s]) == len(seen) - 1  # RoPE position: the node's depth
            bb.logits[s] = torch.from_numpy(toy_logits([self._row(bb.pt[s], j)[0] for j in seen], self.seed))

    def _keep_path(self, pt, base, path, n_path, lanes, n, err):
        for b in range(lanes):
            rows = [self._row(pt[b], int(base[b]) + int(p)).clone() for p in path[b, :n_path[b]]]
            for i, r in enumerate(rows):
                self._row(pt[b], int(base[b]) + i).copy_(r)


def draw_tokens(logits, V, lanes, nr, node0, m, inv, u, hist, count, tokens, parent, out):
    for r in range(lanes * nr):
        b = r // nr
        ids = spec.tree_history(tokens[b], parent[b], hist[b], count[b], node0 + r % nr)
        out[r] = torch.tensor(spec.draw_tokens(logits[r].numpy(), ids, int(inv[b]), u[r].tolist()))


def verify_tree(logits, dlogits, V, lanes, n, tokens, parent, n_tree, inv, dinv, u, hist, count, path, n_path, nxt):
    path.fill_(-1)
    for b in range(lanes):
        at = slice(b * n, (b + 1) * n)
        p, t = spec.tree_verify(logits[at].numpy(), dlogits[at].numpy(), tokens[b], parent[b], int(n_tree[b]),
                                int(inv[b]), int(dinv[b]), u[b].numpy(), hist[b], int(count[b]))
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        n_path[b], nxt[b] = len(p), t


def plain(prompt, max_tokens, seed=0, eos=()):
    """Greedy decoding of the toy model."""
    seq, out, last = [1] + list(prompt), [], prompt[-1]
    while len(out) < max_tokens:
        seq.append(last)
        x = toy_logits(seq, seed)
        for t in out[:-65:-1]:
            x[t] = spec.penalize(int(x[t]))
        last = spec.argmax(x)
        out.append(last)
        if last in eos:
            break
    return out

