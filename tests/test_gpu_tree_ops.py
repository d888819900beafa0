"""Tree-speculation kernels against their 64-bit integer definitions in
``arc_chain_b200.spec``.  Everything is an exact integer: no tolerance."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from arc_chain_b200 import spec

pytestmark = pytest.mark.gpu
PAGE, I32, I64 = 16, torch.int32, torch.int64
ERR_BOUNDS, ERR_SEQ = 8, 32


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda")


def masks(parents):
    m = []
    for i, p in enumerate(parents):
        m.append((m[p] if p >= 0 else 0) | 1 << i)
    return np.array([x - (1 << 64) if x >> 63 else x for x in m], dtype=np.int64)


def heap(n, fan):
    return [-1] + [(i - 1) // fan for i in range(1, n)]


class Attn:
    """Random inputs of attn_tree; lens and nodes per lane, queries = the last nq nodes of an n-node tree."""

    def __init__(self, dh, heads, kv, lens, nodes, nq, fan, kmag, vmag, seed=0):
        rng = np.random.default_rng([seed, dh, heads, nq, len(lens)])
        self.dh, self.heads, self.kv, self.nq, self.lanes = dh, heads, kv, nq, len(lens)
        self.base, self.nodes = np.array(lens, np.int32), np.array(nodes, np.int32)
        self.t_lim = int((self.base + self.nodes).max()) or 1
        self.width = (self.t_lim + PAGE - 1) // PAGE + 1
        pages = self.lanes * self.width + 2
        self.K = rng.integers(-kmag, kmag, (pages, kv, PAGE, dh))
        self.V = rng.integers(-vmag, vmag, (pages, kv, PAGE, dh))
        self.q = rng.integers(-kmag, kmag, (self.lanes * nq, heads * dh))
        self.pt = rng.permutation(pages)[:self.lanes * self.width].reshape(self.lanes, self.width).astype(np.int32)
        self.mask = np.zeros((self.lanes, nq), np.int64)
        for b, n in enumerate(nodes):
            m = masks(heap(n, fan)) if n else np.zeros(0, np.int64)
            k = min(n, nq)
            if k:
                self.mask[b, :k] = m[n - k:]
        self.mask = self.mask.reshape(-1)
        self.scale = {64: 8192, 128: 5793}.get(dh, 9000)

    def want(self):
        out = np.zeros((self.lanes * self.nq, self.heads * self.dh), np.int64)
        g = self.heads // self.kv
        with np.errstate(over="ignore"):
            for b in range(self.lanes):
                t = int(self.base[b] + self.nodes[b])
                if t == 0:
                    continue
                pages = self.pt[b, :(t + PAGE - 1) // PAGE]
                for h in range(self.heads):
                    K = self.K[pages, h // g].reshape(-1, self.dh)[:t]
                    V = self.V[pages, h // g].reshape(-1, self.dh)[:t]
                    for i in range(self.nq):
                        s, at = b * self.nq + i, slice(h * self.dh, (h + 1) * self.dh)
                        out[s, at] = spec.tree_attention(self.q[s, at], K, V, int(self.base[b]), int(self.nodes[b]),
                                                         int(self.mask[s]), self.scale)
        return out

    def tensors(self):
        return [dev(a) for a in (self.q, self.K, self.V, self.pt, self.base, self.nodes, self.mask)]

    def run(self, ts=None, X=None, lmax=None, o=True, err=None, t_lim=None):
        from arc_chain_b200.ops import tree_ops as ops

        err = torch.zeros(1, dtype=I32, device="cuda") if err is None else err
        out = torch.full((self.lanes * self.nq, self.heads * self.dh), 77, dtype=I64, device="cuda") if o else None
        ops.attn_tree(*(ts or self.tensors()), self.heads, self.kv, self.dh, self.scale, self.lanes, self.nq, X, lmax,
                      t_lim or self.t_lim, err, o_out=out)
        torch.cuda.synchronize()
        return out, int(err.item())


M18, M40 = 1 << 18, 1 << 40
SHAPES = [
    # dh, heads, kv, lens, nodes, nq, fan, K/q magnitude, V magnitude
    (64, 4, 2, [37], [5], 5, 1, M18, M18),
    (64, 4, 4, [0], [1], 1, 1, M18, M18),          # one key: the root alone
    (64, 2, 1, [1], [0], 3, 1, M18, M18),          # no tree, one cached key
    (128, 4, 4, [386], [16], 16, 2, M18, M18),
    (128, 8, 2, [1, 17, 130, 255], [31, 7, 1, 64], 31, 3, M18, M18),  # ragged trees, padded queries
    (128, 16, 2, [0, 15, 16, 127, 128, 129], [64, 64, 64, 1, 2, 63], 64, 4, M18, M18),  # page and tile edges
    (128, 8, 1, [1000], [64], 40, 5, 1 << 20, 1 << 20),
    (128, 2, 2, [300, 40], [9, 9], 9, 2, M40, M40),           # wrapping dots, wide values
    (128, 4, 2, [200], [12], 12, 2, 1 << 30, M18),            # 5 digits of K and q
    (128, 4, 2, [200], [12], 12, 2, 1 << 22, (1 << 23) + 5),  # values beyond 24 bits
    (64, 4, 2, [77], [12], 12, 2, M18, 1 << 62),              # values near the type's end
    (64, 4, 2, [77], [12], 12, 2, (1 << 63) - 1, M18),        # K and q over the whole type
    (8, 3, 1, [20], [4], 4, 1, M18, M18),
    (72, 6, 2, [150], [10], 10, 3, M18, M18),
    (96, 5, 5, [140], [33], 33, 2, M18, M18),
    (128, 64, 8, [513], [33], 7, 2, M18, M18),
    (128, 14, 2, [259], [20], 20, 2, 1 << 15, M18),           # 7 query heads per KV head, flat scores
    (128, 2, 2, [4097, 5], [13, 13], 13, 3, M18, M18),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(str(x).replace(" ", "") for x in s))
def test_attn_tree(shape):
    from arc_chain_b200.ops import int_ops

    a = Attn(*shape)
    B, d = a.lanes * a.nq, a.heads * a.dh
    want = a.want()
    X = torch.full((int_ops.limb_rows(B), d), 3, dtype=torch.int8, device="cuda")
    lmax = torch.zeros(1, dtype=I32, device="cuda")
    got, err = a.run(X=X, lmax=lmax)
    assert err == 0
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    planes, need = int_ops.limb_planes(want, int_ops.limb_rows(B))
    used = 8 * int_ops.n_tiles(B) * int_ops.limb_slots(B)
    rows = [int_ops.limb_row(l, b, B) for b in range(B) for l in range(8)]
    np.testing.assert_array_equal(X.cpu().numpy()[rows], planes[rows])
    if X.shape[0] > used:
        assert bool((X[used:] == 3).all())  # rows behind the last slot stay as they were
    assert int(lmax.item()) == (need if want.any() else 0)
    X.fill_(3)
    a.run(X=X, o=False)
    np.testing.assert_array_equal(X.cpu().numpy()[rows], planes[rows])


def test_attn_tree_idle_lanes_and_empty_rows():
    a = Attn(64, 4, 2, [0, 40, 0], [0, 5, 6], 4, 1, M18, M18)
    a.mask[:] = 0
    a.mask[9] = 1 << 3            # lane 2 has no prefix: only query 1 sees a key
    a.mask[10] = 1 << 40          # a bit behind the tree's nodes
    want = a.want()
    assert not want[:4].any() and want[4:8].any() and not want[8].any() and want[9].any() and not want[10].any()
    got, err = a.run()
    assert err == 0
    np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_attn_tree_equal_and_lopsided_scores():
    """Equal scores (all weights equal), one key far above the rest (its weight
    is ONE), and two keys 8.0 apart (the lower weight is 0)."""
    for seed, kind in enumerate(("equal", "one", "edge")):
        a = Attn(64, 2, 1, [50], [3], 3, 1, M18, M18, seed=seed)
        a.q[:] = 0
        a.q[:, ::64] = 1 << 16
        a.K[:] = 0
        if kind != "equal":
            row = (a.pt[0, 20 // PAGE], 0, 20 % PAGE, 0)
            a.K[row] = (1 << 16) * (9 if kind == "one" else 8) * 8  # scale 1/8
        want = a.want()
        got, err = a.run()
        assert err == 0
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_attn_tree_bad_lanes_give_zeros_and_an_error():
    for what, bit in (("page", ERR_BOUNDS), ("low page", ERR_BOUNDS), ("base", ERR_SEQ), ("nodes", ERR_SEQ),
                      ("too many", ERR_SEQ), ("long", ERR_SEQ)):
        a = Attn(64, 4, 2, [40, 50], [5, 6], 5, 2, M18, M18)
        want = a.want()
        want[:5] = 0
        if what == "page":
            a.pt[0, 1] = a.K.shape[0]
        elif what == "low page":
            a.pt[0, 2] = -1
        elif what == "base":
            a.base[0] = -1
        elif what == "nodes":
            a.nodes[0] = -3
        elif what == "too many":
            a.nodes[0] = 65
        else:
            a.base[0] = 52  # 57 keys: beyond t_lim, inside the table
        got, err = a.run(t_lim=56)
        assert err == bit, what
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_attn_tree_strided_table_other_stream_and_graph():
    """A page table of every nq-th row of a per-slot table, a launch on a side
    stream, and one captured call replayed on changed inputs."""
    from arc_chain_b200.ops import tree_ops as ops

    a, b = (Attn(128, 4, 2, [100, 300], [9, 13], 9, 2, M18, M18, seed=s) for s in (1, 2))
    ts = a.tensors()
    ts[3] = ts[3].repeat_interleave(9, 0)[::9]
    assert not ts[3].is_contiguous()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, err = a.run(ts)
    assert err == 0
    np.testing.assert_array_equal(got.cpu().numpy(), a.want())
    out, e = torch.zeros_like(got), torch.zeros(1, dtype=I32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.attn_tree(*ts, a.heads, a.kv, a.dh, a.scale, a.lanes, a.nq, None, None, a.t_lim, e, o_out=out)
    for x in (a, b, a):
        for t, v in zip(ts, x.tensors()):
            t.copy_(v)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert int(e.item()) == 0
        np.testing.assert_array_equal(out.cpu().numpy(), x.want())


def test_attn_tree_calls_on_two_streams_at_once():
    xs = [Attn(128, 8, 2, [400 + 100 * s, 90], [13, 31], 13, 3, M18, M18, seed=s) for s in range(2)]
    from arc_chain_b200.ops import tree_ops as ops

    streams, ins = [torch.cuda.Stream() for _ in xs], [x.tensors() for x in xs]
    outs = [torch.zeros(x.lanes * x.nq, x.heads * x.dh, dtype=I64, device="cuda") for x in xs]
    e = torch.zeros(1, dtype=I32, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        for x, s, t, o in zip(xs, streams, ins, outs):
            with torch.cuda.stream(s):
                ops.attn_tree(*t, x.heads, x.kv, x.dh, x.scale, x.lanes, x.nq, None, None, x.t_lim, e, o_out=o)
    torch.cuda.synchronize()
    assert int(e.item()) == 0
    for x, o in zip(xs, outs):
        np.testing.assert_array_equal(o.cpu().numpy(), x.want())


@pytest.mark.parametrize("dh,heads,kv,lens,nodes,nq", [
    (64, 2, 1, [40], [4], 4),            # 8 rows
    (128, 8, 1, [250], [4], 4),          # 32 rows of 254 keys: 8128, the most that two kernels take
    (128, 8, 1, [252], [5], 4),          # 32 rows of 257 keys
    (128, 11, 1, [40], [3], 3),          # 33 rows
    (128, 8, 2, [60, 3], [8, 8], 8),     # 32 rows, two lanes
    (128, 5, 1, [300], [13], 13),        # 65 rows: value CTAs of five warps
    (128, 8, 1, [300], [10], 10),        # 80 rows
    (64, 8, 1, [90, 500, 1], [9, 9, 9], 9),
    (128, 3, 1, [131], [27], 27),        # 81 rows
    (128, 8, 1, [131], [17], 17),        # 136 rows: two groups
], ids=str)
def test_attn_tree_row_counts(dh, heads, kv, lens, nodes, nq):
    """Row counts around the variants' borders; the keys' limit decides one of
    them and must not change a result."""
    a = Attn(dh, heads, kv, lens, nodes, nq, 2, M18, M18)
    want = a.want()
    a.pt = np.concatenate([a.pt, np.full((a.lanes, 700), -1, np.int32)], 1)  # pages behind the last key are not read
    for t_lim in (a.t_lim, 2100, 9000):
        got, err = a.run(t_lim=t_lim)
        assert err == 0
        np.testing.assert_array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("kind", ["wide values", "wide keys", "empty", "bad"])
def test_attn_tree_few_keys(kind):
    """Two lanes of few rows and keys: the other kinds of values, keys and lanes."""
    a = Attn(64, 4, 2, [100, 17], [9, 5], 5, 2, (1 << 63) - 1 if kind == "wide keys" else M18,
             1 << 62 if kind == "wide values" else M18, seed=3)
    if kind == "empty":
        a.base[1] = a.nodes[1] = 0
        a.mask[2] = 0
        a.base[0] = 0
    want = a.want()
    if kind == "bad":
        a.pt[1, 0] = -2
        want[5:] = 0
    for _ in range(2):
        got, err = a.run()
        assert err == (ERR_BOUNDS if kind == "bad" else 0)
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_attn_tree_sums_beyond_32_bits():
    """Equal scores: every exp is ONE, and from 2^14 keys a row's sum passes
    2^30, from 2^16 keys 2^32; the weights of the longer one are all 0."""
    for n, vmag in ((16500, M18), (40000, 1 << 30), (65600, M18)):
        a = Attn(64, 3, 1, [n], [3], 3, 2, M18, vmag)
        a.q[:] = 0
        want = a.want()
        got, err = a.run()
        assert err == 0 and (n > 65536) == (not want.any())
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_attn_tree_lanes_in_several_launches():
    """Scores of more keys and rows than one launch's workspace holds: the
    lanes go in batches."""
    a = Attn(8, 64, 8, [50, 0, 17, 130, 16, 3, 64], [64, 2, 64, 40, 1, 64, 0], 64, 3, M18, M18)
    want = a.want()
    a.pt = np.concatenate([a.pt, np.zeros((a.lanes, 1300), np.int32)], 1)
    got, err = a.run(t_lim=20000)
    assert err == 0
    np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_attn_tree_many_lanes():
    """More lanes than the GPU has value CTAs, idle ones among them."""
    rng = np.random.default_rng(12)
    lens, nodes = rng.integers(0, 40, 2500).tolist(), rng.integers(0, 3, 2500).tolist()
    a = Attn(8, 2, 1, lens, nodes, 1, 1, M18, M18)
    want = a.want()
    a.pt[7, 0] = -1
    want[7] = 0
    for t_lim in (a.t_lim, 1000):
        got, err = a.run(t_lim=t_lim)
        assert err == (ERR_BOUNDS if lens[7] + nodes[7] else 0)
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_attn_tree_key_limit_beyond_the_table():
    """t_lim bounds lengths only as far as the table's pages reach."""
    a = Attn(64, 4, 2, [40, 70], [5, 6], 5, 2, M18, M18)
    want = a.want()
    for t_lim in (a.width * PAGE + 1, 1 << 30, 1 << 40):
        got, err = a.run(t_lim=t_lim)
        assert err == 0
        np.testing.assert_array_equal(got.cpu().numpy(), want)
    a.base[0] = a.width * PAGE - 4  # 5 nodes: one beyond the table
    want[:5] = 0
    got, err = a.run(t_lim=1 << 30)
    assert err == ERR_SEQ
    np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_attn_tree_equals_decode_attention():
    """Chain queries equal the decode kernel at consecutive positions."""
    from arc_chain_b200.ops import int_ops

    a = Attn(128, 8, 2, [75], [6], 6, 1, M18, M18)
    got, err = a.run()
    ts = a.tensors()
    pos = torch.arange(75, 81, dtype=I32, device="cuda")
    out = torch.zeros_like(got)
    e = torch.zeros(1, dtype=I32, device="cuda")
    int_ops.attn(ts[0], ts[1], ts[2], ts[3].expand(6, -1).contiguous(), pos, 8, 2, 128, a.scale, 6, None, None,
                 a.width * PAGE, e, o_out=out)
    torch.cuda.synchronize()
    assert err == 0 and int(e.item()) == 0
    assert torch.equal(got, out)


# ------------------------------------------------------------ drawing and verifying
class Rows:
    def __init__(self, lanes, n, V, fan=2, seed=0, inv=(65536,), dinv=(65536,), near=0.5, parent=None, tie=False):
        rng = np.random.default_rng([seed, lanes, n, V])
        self.lanes, self.n, self.V = lanes, n, V
        self.logits = (rng.normal(size=(lanes * n, V)) * 2.5 * 65536).astype(np.int64)
        if tie:
            self.logits = self.logits >> 15 << 15
        self.dlogits = self.logits + (rng.normal(size=(lanes * n, V)) * near * 65536).astype(np.int64)
        self.parent = np.array([parent or heap(n, fan)] * lanes, np.int32)
        self.hist = rng.integers(0, V, (lanes, 64)).astype(np.int32)
        self.count = np.array([(0, 3, 64, 1000, -5)[b % 5] for b in range(lanes)], np.int32)
        self.inv = np.array([inv[b % len(inv)] for b in range(lanes)], np.int64)
        self.dinv = np.array([dinv[b % len(dinv)] for b in range(lanes)], np.int64)
        self.u = rng.integers(0, 1 << 31, (lanes, n, 2)).astype(np.int32)
        self.n_tree = np.full(lanes, n, np.int32)
        self.tokens = np.zeros((lanes, n), np.int32)
        for b in range(lanes):
            self.tokens[b, 0] = rng.integers(V)
            for i in range(n):
                kids = [c for c in range(n) if self.parent[b, c] == i]
                if kids:
                    ids = spec.tree_history(self.tokens[b], self.parent[b], self.hist[b], max(self.count[b], 0), i)
                    got = spec.draw_tokens(self.dlogits[b * n + i], ids, int(self.dinv[b]),
                                           rng.integers(0, 1 << 31, len(kids)))
                    self.tokens[b, kids] = got

    def verify(self):
        from arc_chain_b200.ops import tree_ops as ops

        z = lambda *s: torch.full(s, 9, dtype=I32, device="cuda")
        path, n_path, nxt = z(self.lanes, self.n), z(self.lanes), z(self.lanes)
        ops.verify_tree(dev(self.logits), dev(self.dlogits), self.V, self.lanes, self.n, dev(self.tokens),
                        dev(self.parent), dev(self.n_tree), dev(self.inv), dev(self.dinv), dev(self.u),
                        dev(self.hist), dev(self.count), path, n_path, nxt)
        torch.cuda.synchronize()
        return path.cpu().numpy(), n_path.cpu().numpy(), nxt.cpu().numpy()

    def check(self):
        path, n_path, nxt = self.verify()
        n = self.n
        for b in range(self.lanes):
            p, t = spec.tree_verify(self.logits[b * n:][:n], self.dlogits[b * n:][:n], self.tokens[b], self.parent[b],
                                    min(int(self.n_tree[b]), n), int(self.inv[b]), int(self.dinv[b]), self.u[b],
                                    self.hist[b], max(int(self.count[b]), 0))
            assert list(path[b]) == p + [-1] * (n - len(p)) and int(n_path[b]) == len(p) and int(nxt[b]) == t, b
        return n_path


@pytest.mark.parametrize("lanes,n,V,kw", [
    (1, 5, 32000, dict(fan=1)),
    (5, 13, 1000, dict(fan=3)),
    (3, 31, 4099, dict(fan=2, near=1.5)),
    (2, 64, 777, dict(fan=4, near=1.0)),
    (1, 64, 300, dict(fan=1, near=0.05)),                                  # a deep accepted chain
    (4, 7, 512, dict(fan=2, inv=(0, 65536, 1 << 30, -7), dinv=(0, 0, 65536, 65536))),  # greedy, clamped
    (4, 7, 200, dict(fan=2, inv=(0, 65536), dinv=(0, 65536), tie=True)),   # ties: the first maximum
    (2, 1, 33, dict()),                                                    # a root alone: a plain draw
    (3, 9, 1, dict(fan=8)),                                                # one token: drafts run out
    (3, 9, 2, dict(fan=8)),
    (12, 40, 300, dict(fan=3, near=0.4)),                                  # more nodes than the GPU decides at once
    (10, 64, 65, dict(fan=2, near=0.2, inv=(40000, 65536))),
    (9, 31, 2001, dict(fan=2, near=0.5)),
    (1, 3, 102400, dict(fan=2)),
    (1, 2, 152064, dict(fan=1)),                                           # 16 CTAs per row
    (1, 2, 272896, dict(fan=1)),                                           # more shared memory per CTA
])
def test_verify_tree(lanes, n, V, kw):
    for seed in range(3 if V < 50000 else 1):
        Rows(lanes, n, V, seed=seed, **kw).check()


def test_verify_tree_ragged_strange_and_masked():
    r = Rows(6, 9, 700, fan=2, near=0.3, seed=4)
    r.n_tree[:] = [0, 1, 4, 9, 12, -2]
    r.parent[2] = [-1, 0, 5, -4, 2, 4, 6, 7, 2 ** 31 - 1]  # orphans and loops: nodes without a parent
    r.tokens[3, 2] = -1
    r.tokens[3, 1] = 700
    r.tokens[4, 1:3] = r.tokens[4, 1]       # the same token twice under one node
    lo = np.iinfo(np.int64).min
    r.logits[:, ::3] = lo                    # masked vocabulary
    r.dlogits[:, 1::3] = lo
    r.logits[9 * 3] = lo                     # a row whose mask leaves nothing
    r.logits[9 * 4, 5] = np.iinfo(np.int64).max
    r.hist[:, :10] = 3
    r.hist[:, 10:14] = [-1, 700, 2 ** 31 - 1, 0]
    r.count[:] = [64, 64, 14, 64, 64, 64]
    n_path = r.check()
    assert n_path[0] == 0 and n_path[5] == 0


def test_largest_vocabulary():
    from arc_chain_b200.ops import tree_ops as ops

    V = ops.lib_max_vocab()
    r = Rows(1, 3, V, fan=2, seed=8)
    r.tokens[0, 1] = V - 1
    r.check()
    out = torch.full((3, 2), 9, dtype=I32, device="cuda")
    u = np.array([[0, 1 << 30], [(1 << 31) - 1, 5], [77, 1 << 29]], np.int32)
    ops.draw_tokens(dev(r.logits), V, 1, 3, 0, 2, dev(r.inv), dev(u), dev(r.hist), dev(r.count), dev(r.tokens),
                    dev(r.parent), out)
    for i in range(3):
        ids = spec.tree_history(r.tokens[0], r.parent[0], r.hist[0], max(int(r.count[0]), 0), i)
        assert out[i].tolist() == spec.draw_tokens(r.logits[i], ids, int(r.inv[0]), u[i]), i


def test_verify_tree_one_lane_equals_its_place_in_a_batch():
    """A small call gives every node its cluster, a larger one every lane: the
    same drafts are kept either way."""
    from arc_chain_b200.ops import tree_ops as ops

    for V, near, inv in ((901, 0.4, 65536), (5000, 1.0, 90000), (64, 0.5, 0)):
        r = Rows(45, 13, V, fan=3, seed=11, near=near, inv=(inv,), dinv=(inv,))
        r.n_tree[:8] = [13, 12, 1, 2, 13, 0, 40, 13]
        r.parent[4] = [-1, 0, 0, 7, 1, 4, 4, 3, 0, 8, 8, -2, 13]
        r.logits[13 * 7:13 * 20, 1::2] = np.iinfo(np.int64).min
        assert r.check().max() > 2
        path, n_path, nxt = r.verify()
        for b in range(45):
            z = lambda *s: torch.full(s, 9, dtype=I32, device="cuda")
            p, k, t = z(1, 13), z(1), z(1)
            ops.verify_tree(dev(r.logits[13 * b:][:13]), dev(r.dlogits[13 * b:][:13]), V, 1, 13, dev(r.tokens[b:b + 1]),
                            dev(r.parent[b:b + 1]), dev(r.n_tree[b:b + 1]), dev(r.inv[b:b + 1]), dev(r.dinv[b:b + 1]),
                            dev(r.u[b:b + 1]), dev(r.hist[b:b + 1]), dev(r.count[b:b + 1]), p, k, t)
            assert p[0].tolist() == list(path[b]) and int(k) == n_path[b] and int(t) == nxt[b], (V, b)


def test_verify_and_draw_in_a_graph_and_on_two_streams():
    from arc_chain_b200.ops import tree_ops as ops

    rs = [Rows(1, 5, 2000, fan=2, seed=s) for s in range(2)] + [Rows(6, 9, 700, fan=2, seed=9)]
    want = [r.verify() for r in rs]
    ins = [[dev(x) for x in (r.logits, r.dlogits, r.tokens, r.parent, r.n_tree, r.inv, r.dinv, r.u, r.hist, r.count)]
           for r in rs]
    outs = [[torch.zeros(s, dtype=I32, device="cuda") for s in ((r.lanes, r.n), (r.lanes,), (r.lanes,))] for r in rs]

    def call(r, i, o):
        ops.verify_tree(i[0], i[1], r.V, r.lanes, r.n, *i[2:], *o)

    streams = [torch.cuda.Stream() for _ in rs]
    torch.cuda.synchronize()
    for _ in range(10):
        for r, i, o, s in zip(rs, ins, outs, streams):
            with torch.cuda.stream(s):
                call(r, i, o)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for x, y in zip(w, o):
            np.testing.assert_array_equal(x, y.cpu().numpy())
    for o in outs:
        for y in o:
            y.fill_(-9)
    g = torch.cuda.CUDAGraph()
    draws = torch.zeros(2, 3, dtype=I32, device="cuda")
    u = torch.randint(0, (1 << 31) - 1, (2, 3), dtype=I32, device="cuda")
    row = ins[0][0][:2].contiguous()
    args = (row, 2000, 1, 2, 0, 3, ins[0][5], u, ins[0][8], ins[0][9], ins[0][2], ins[0][3])
    ops.draw_tokens(*args, draws)
    plain = draws.clone()
    with torch.cuda.graph(g):
        for r, i, o in zip(rs, ins, outs):
            call(r, i, o)
        ops.draw_tokens(*args, draws)
    draws.zero_()
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for x, y in zip(w, o):
            np.testing.assert_array_equal(x, y.cpu().numpy())
    assert torch.equal(draws, plain)


def test_verify_tree_strided_rows():
    from arc_chain_b200.ops import tree_ops as ops

    r = Rows(2, 5, 501, fan=2, seed=6)
    big = torch.full((10, 600), 1 << 50, dtype=I64, device="cuda")
    big[:, :501] = dev(r.logits)
    want = r.verify()
    z = lambda *s: torch.zeros(s, dtype=I32, device="cuda")
    path, n_path, nxt = z(2, 5), z(2), z(2)
    ops.verify_tree(big[:, :501], dev(r.dlogits), 501, 2, 5, dev(r.tokens), dev(r.parent), dev(r.n_tree), dev(r.inv),
                    dev(r.dinv), dev(r.u), dev(r.hist), dev(r.count), path, n_path, nxt)
    for a, b in zip(want, (path, n_path, nxt)):
        np.testing.assert_array_equal(a, b.cpu().numpy())
    np.testing.assert_array_equal(big[:, :501].cpu().numpy(), r.logits)  # the logits stay as they were


@pytest.mark.parametrize("lanes,n,nr,V,m,kw", [
    (1, 1, 1, 32000, 1, dict()), (3, 13, 9, 1031, 3, dict(fan=3)), (2, 4, 4, 5, 7, dict()),
    (4, 3, 2, 300, 2, dict(inv=(0, 65536, 1 << 40, -1))), (2, 3, 3, 128, 40, dict(tie=True)),
    (1, 64, 2, 900, 2, dict(fan=1)), (1, 1, 1, 102400, 4, dict()), (1, 1, 1, 272896, 2, dict(inv=(6000,))),
    (2, 2, 1, 1, 2, dict())])
def test_draw_tokens(lanes, n, nr, V, m, kw):
    from arc_chain_b200.ops import tree_ops as ops

    r = Rows(lanes, n, V, seed=1, **kw)
    node0 = n - nr
    rng = np.random.default_rng(V)
    u = rng.integers(0, 1 << 31, (lanes * nr, m)).astype(np.int32)
    u.flat[0], u.flat[-1] = 0, 2 ** 31 - 1
    rows = r.logits.reshape(lanes, n, V)[:, node0:].reshape(lanes * nr, V).copy()
    out = torch.full((lanes * nr, m), 9, dtype=I32, device="cuda")
    ops.draw_tokens(dev(rows), V, lanes, nr, node0, m, dev(r.inv), dev(u), dev(r.hist), dev(r.count), dev(r.tokens),
                    dev(r.parent), out)
    for i in range(lanes * nr):
        b, node = i // nr, node0 + i % nr
        ids = spec.tree_history(r.tokens[b], r.parent[b], r.hist[b], max(int(r.count[b]), 0), node)
        assert out[i].tolist() == spec.draw_tokens(rows[i], ids, int(r.inv[b]), u[i]), i


# ------------------------------------------------------------ keeping the path
def keep_want(caches, pt, base, path, n_path):
    for c in caches:
        for b in range(len(base)):
            at = [(pt[b, (base[b] + j) // PAGE], (base[b] + j) % PAGE) for j in path[b, :n_path[b]]]
            rows = [c[p, :, o].copy() for p, o in at]
            for i, row in enumerate(rows):
                c[pt[b, (base[b] + i) // PAGE], :, (base[b] + i) % PAGE] = row


@pytest.mark.parametrize("layers,kv,dh,alias", [(1, 1, 8, False), (3, 2, 64, False), (2, 8, 128, False), (2, 1, 576, True)])
def test_kv_keep_path(layers, kv, dh, alias):
    from arc_chain_b200.ops import tree_ops as ops

    rng = np.random.default_rng(dh)
    lanes, n, width = 5, 40, 8
    pages = lanes * width + 1
    Ks = [rng.integers(-1 << 40, 1 << 40, (pages, kv, PAGE, dh)) for _ in range(layers)]
    Vs = Ks if alias else [rng.integers(-1 << 40, 1 << 40, (pages, kv, PAGE, dh)) for _ in range(layers)]
    pt = rng.permutation(pages)[:lanes * width].reshape(lanes, width).astype(np.int32)
    base = np.array([0, 13, 63, 88, 20], np.int32)
    path = np.full((lanes, n), -1, np.int32)
    n_path = np.array([0, 1, 5, 40, 9], np.int32)
    for b, k in enumerate(n_path):
        if k:
            path[b, 0] = 0
            path[b, 1:k] = np.sort(rng.permutation(n - 1)[:k - 1]) + 1
    path[4, :9] = range(9)  # nothing moves
    tK = [dev(c) for c in Ks]
    tV = tK if alias else [dev(c) for c in Vs]
    planes = ops.KvPlanes(tK, tV)
    assert len(planes.tensors) == layers * (1 if alias else 2)
    err = torch.zeros(1, dtype=I32, device="cuda")
    ops.kv_keep_path(planes, dev(pt), dev(base), dev(path), dev(n_path), lanes, n, err)
    keep_want(Ks if alias else Ks + Vs, pt, base, path, n_path)
    assert int(err.item()) == 0
    for t, c in zip(tK + tV, Ks + Vs):
        np.testing.assert_array_equal(t.cpu().numpy(), c)


def test_kv_keep_path_leaves_bad_lanes_alone():
    from arc_chain_b200.ops import tree_ops as ops

    rng = np.random.default_rng(0)
    K = rng.integers(-9, 9, (30, 2, PAGE, 8))
    pt = rng.permutation(30)[:28].reshape(7, 4).astype(np.int32)
    base = np.array([10, 10, 10, 60, -1, 10, 10], np.int32)
    path = np.array([[0, 2, 5, -1], [1, 2, 5, -1], [0, 5, 2, -1], [0, 2, 5, -1], [0, 2, 5, -1], [0, 2, 8, -1],
                     [0, 2, 5, -1]], np.int32)
    n_path = np.array([3, 3, 3, 3, 3, 3, 9], np.int32)
    pt[0, 0] = 30
    for lanes in (1, 7):
        t = dev(K)
        err = torch.zeros(1, dtype=I32, device="cuda")
        p4 = np.concatenate([path[:lanes], np.full((lanes, 4), -1, np.int32)], 1)  # 8-node trees
        ops.kv_keep_path(ops.KvPlanes([t], [t]), dev(pt[:lanes]), dev(base[:lanes]), dev(p4), dev(n_path[:lanes]),
                         lanes, 8, err)
        assert int(err.item()) == ERR_BOUNDS
        np.testing.assert_array_equal(t.cpu().numpy(), K)
