"""Tree-speculation operators without a GPU: the bounds rules that the kernels
share with the host library, what the entry points refuse, and properties of
the integer definitions (a tree node attends as a plain step along its path;
verified drafts follow the target's distribution)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from arc_chain_b200 import spec
from arc_chain_b200.oracle import arcref
from arc_chain_b200.ops import tree_ops as ops

I32, I64 = torch.int32, torch.int64


# ------------------------------------------------------------ bounds rules
@pytest.mark.parametrize("base,n,t_lim,width,keys", [
    (0, 0, 1, 1, 0), (0, 1, 1, 1, 1), (5, 3, 8, 1, 8), (5, 3, 7, 1, -1), (14, 3, 100, 1, -1), (13, 3, 100, 1, 16),
    (-1, 3, 100, 9, -1), (0, -1, 100, 9, -1), (0, 64, 64, 4, 64), (0, 65, 100, 9, -1),
    (2 ** 31 - 1, 64, 2 ** 31 - 1, 2 ** 27, -1), (2 ** 31 - 65, 64, 2 ** 31 - 1, 2 ** 27, 2 ** 31 - 1)])
def test_lane_keys(base, n, t_lim, width, keys):
    assert arcref.lib().arcref_tree_lane_keys(base, n, t_lim, width) == keys


def test_pages_and_visibility():
    L = arcref.lib()
    assert [L.arcref_tree_page_ok(p, 4) for p in (-2 ** 31, -1, 0, 3, 4, 2 ** 31 - 1)] == [0, 0, 1, 1, 0, 0]
    mask = 1 | 1 << 3 | 1 << 63
    seen = [j for j in range(-2, 80) if L.arcref_tree_visible(j, 5, 64, mask)]
    assert seen == [0, 1, 2, 3, 4, 5, 8, 68]
    assert [j for j in range(80) if L.arcref_tree_visible(j, 5, 3, mask)] == [0, 1, 2, 3, 4, 5]
    assert [j for j in range(80) if L.arcref_tree_visible(j, 0, 64, 0)] == []


def test_parents_and_paths():
    L = arcref.lib()
    par = np.array([-1, 0, 7, 1, 3, 5, -9, 2 ** 31 - 1], dtype=np.int32)
    assert [L.arcref_tree_parent_of(par.ctypes.data, i) for i in range(8)] == [-1, 0, -1, 1, 3, -1, -1, -1]

    def ok(path, n, base=3, width=2):
        a = np.array(path, dtype=np.int32)
        return [L.arcref_tree_path_ok(a.ctypes.data, i, n, base, width) for i in range(len(path))]

    assert ok([0, 2, 5], 6) == [1, 1, 1]
    assert ok([1, 2, 5], 6) == [0, 1, 1]
    assert ok([0, 2, 2, 1, -1], 6) == [1, 1, 0, 0, 0]
    assert ok([0, 2, 6], 6) == [1, 1, 0]
    assert ok([0, 28, 29], 64) == [1, 1, 0]  # 32 rows: positions 3 + 28 in, 3 + 29 out
    assert ok([0, 1], 6, base=-1) == [0, 0]
    assert ok([0, 1], 6, base=2 ** 31 - 1, width=2 ** 27) == [1, 0]


# ------------------------------------------------------------ refusals
def _attn_args(**kw):
    lanes, nq, heads, kv, dh = 2, 3, 4, 2, 64
    z = dict(q=torch.zeros(lanes * nq, heads * dh, dtype=I64), Kc=torch.zeros(5, kv, 16, dh, dtype=I64),
             Vc=torch.zeros(5, kv, 16, dh, dtype=I64), pt=torch.zeros(lanes, 2, dtype=I32),
             base=torch.zeros(lanes, dtype=I32), n_tree=torch.zeros(lanes, dtype=I32),
             mask=torch.zeros(lanes * nq, dtype=I64), n_heads=heads, n_kv=kv, dh=dh, attn_scale=8192, lanes=lanes,
             nq=nq, X=None, lmax=None, t_lim=32, err=torch.zeros(1, dtype=I32),
             o_out=torch.zeros(lanes * nq, heads * dh, dtype=I64))
    return {**z, **kw}


@pytest.mark.parametrize("bad,exc", [
    (dict(lanes=0), ValueError), (dict(nq=0), ValueError), (dict(n_heads=5), ValueError), (dict(n_kv=0), ValueError),
    (dict(dh=60), ValueError), (dict(dh=136), ValueError), (dict(dh=0), ValueError), (dict(t_lim=0), ValueError),
    (dict(lanes=4), ValueError), (dict(q=torch.zeros(6, 256)), TypeError), (dict(q=None), TypeError),
    (dict(q=torch.zeros(256, 6, dtype=I64).t()), ValueError), (dict(Vc=torch.zeros(4, 2, 16, 64, dtype=I64)), ValueError),
    (dict(Kc=torch.zeros(5, 2, 8, 64, dtype=I64)), ValueError), (dict(pt=torch.zeros(2, 2, dtype=I64)), TypeError),
    (dict(pt=torch.zeros(1, 2, dtype=I32)), ValueError), (dict(pt=torch.zeros(2, 0, dtype=I32)), ValueError),
    (dict(pt=torch.zeros(1, 2, dtype=I32).expand(2, 2)), ValueError),
    (dict(mask=torch.zeros(2, dtype=I64)), ValueError), (dict(base=torch.zeros(2, dtype=I64)), TypeError),
    (dict(o_out=None), ValueError), (dict(o_out=None, X=torch.zeros(47, 256, dtype=torch.int8)), ValueError),
    (dict(lmax=torch.zeros(2, dtype=I32)), ValueError), (dict(err=torch.zeros(0, dtype=I32)), ValueError),
    ({}, ValueError)])  # the last: tensors on the CPU
def test_attn_tree_refuses(bad, exc):
    with pytest.raises(exc):
        ops.attn_tree(**_attn_args(**bad))


def test_attn_tree_refuses_unaligned_tensors_and_wide_scales():
    from arc_chain_b200.ops import tree_ops as ops

    good = _attn_args()
    for name in ("q", "Kc", "Vc", "o_out"):
        t = good[name]
        moved = torch.zeros(t.numel() + 1, dtype=t.dtype)[1:].view(t.shape)
        with pytest.raises(ValueError, match="16-byte"):
            ops.attn_tree(**{**good, name: moved})
    for scale in (1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="64-bit"):
            ops.attn_tree(**{**good, "attn_scale": scale})


def _verify_args(**kw):
    lanes, n, V = 2, 4, 10
    z = dict(logits=torch.zeros(lanes * n, V, dtype=I64), dlogits=torch.zeros(lanes * n, V, dtype=I64), V=V,
             lanes=lanes, n=n, tokens=torch.zeros(lanes, n, dtype=I32), parent=torch.zeros(lanes, n, dtype=I32),
             n_tree=torch.zeros(lanes, dtype=I32), inv_temp=torch.zeros(lanes, dtype=I64),
             d_inv_temp=torch.zeros(lanes, dtype=I64), u=torch.zeros(lanes, n, 2, dtype=I32),
             hist=torch.zeros(lanes, 64, dtype=I32), count=torch.zeros(lanes, dtype=I32),
             path=torch.zeros(lanes, n, dtype=I32), n_path=torch.zeros(lanes, dtype=I32),
             nxt=torch.zeros(lanes, dtype=I32))
    return {**z, **kw}


@pytest.mark.parametrize("bad,exc", [
    (dict(V=0), ValueError), (dict(V=11), ValueError), (dict(V=1 << 30), ValueError), (dict(lanes=0), ValueError),
    (dict(n=0), ValueError), (dict(n=65), ValueError), (dict(logits=torch.zeros(8, 10)), TypeError),
    (dict(logits=torch.zeros(7, 10, dtype=I64)), ValueError), (dict(dlogits=torch.zeros(8, 9, dtype=I64)), ValueError),
    (dict(logits=torch.zeros(1, 10, dtype=I64).expand(8, 10)), ValueError),
    (dict(logits=torch.zeros(10, 8, dtype=I64).t()), ValueError),
    (dict(u=torch.zeros(2, 4, dtype=I32)), ValueError), (dict(u=torch.zeros(2, 4, 2)), TypeError),
    (dict(hist=torch.zeros(2, 63, dtype=I32)), ValueError), (dict(inv_temp=torch.zeros(2)), TypeError),
    (dict(path=torch.zeros(2, 5, dtype=I32)), ValueError), ({}, ValueError)])
def test_verify_tree_refuses(bad, exc):
    with pytest.raises(exc):
        ops.verify_tree(**_verify_args(**bad))


@pytest.mark.parametrize("bad,exc", [
    (dict(nr=0), ValueError), (dict(node0=-1), ValueError), (dict(nr=4), ValueError), (dict(m=0), ValueError),
    (dict(tokens=None), ValueError), (dict(tokens=torch.zeros(2, 65, dtype=I32)), ValueError),
    (dict(u=torch.zeros(6, 1, dtype=I32)), ValueError), (dict(out=torch.zeros(6, 2, dtype=I64)), TypeError),
    (dict(V=11), ValueError), ({}, ValueError)])
def test_draw_tokens_refuses(bad, exc):
    a = dict(logits=torch.zeros(6, 10, dtype=I64), V=10, lanes=2, nr=3, node0=1, m=2,
             inv_temp=torch.zeros(2, dtype=I64), u=torch.zeros(6, 2, dtype=I32), hist=torch.zeros(2, 64, dtype=I32),
             count=torch.zeros(2, dtype=I32), tokens=torch.zeros(2, 4, dtype=I32),
             parent=torch.zeros(2, 4, dtype=I32), out=torch.zeros(6, 2, dtype=I32))
    with pytest.raises(exc):
        ops.draw_tokens(**{**a, **bad})


def test_kv_planes_refuse():
    t = torch.zeros(3, 2, 16, 64, dtype=I64)
    for bad, exc in (([], ValueError), ([t, t[:2]], ValueError), ([t.int()], TypeError), ([t[:, :, :8]], ValueError),
                     ([t[..., :63]], ValueError), ([t[..., ::2]], ValueError), ([t], ValueError)):
        with pytest.raises(exc):
            ops.KvPlanes(bad, [])
    with pytest.raises(TypeError):
        ops.kv_keep_path([t], t, t, t, t, 1, 4, t)


# ------------------------------------------------------------ definitions
def test_tree_attention_is_a_plain_step_along_the_path():
    rng = np.random.default_rng(3)
    base, n, dh = 21, 9, 32
    par = [-1, 0, 0, 1, 1, 2, 4, 4, 5]
    K, V = (rng.integers(-1 << 18, 1 << 18, (base + n, dh)) for _ in range(2))
    q = rng.integers(-1 << 18, 1 << 18, (n, dh))
    for i in range(n):
        path, j = [], i
        while j >= 0:
            path.insert(0, j)
            j = par[j]
        rows = list(range(base)) + [base + j for j in path]
        dots = (K[rows] * q[i]).sum(1)
        w = spec.softmax(((dots >> 16) * 11585) >> 16)
        want = ((w[:, None] * V[rows]) >> 16).sum(0)
        got = spec.tree_attention(q[i], K, V, base, n, sum(1 << j for j in path), 11585)
        np.testing.assert_array_equal(got, want)
    assert not spec.tree_attention(q[0], K, V, 0, n, 0, 11585).any()


@pytest.mark.parametrize("inv_t,inv_q,kids", [(65536, 65536, 2), (98304, 40000, 3), (65536, 0, 1), (0, 65536, 2)])
def test_verified_drafts_follow_the_target(inv_t, inv_q, kids):
    """First emitted token over many random numbers: its frequencies against
    the target's weights.  With N samples a frequency is off by more than
    5 sqrt(p (1 - p) / N) with a probability below 6e-7 for each of the 8 tokens;
    the 31-bit roundings add at most 8 * 2^-31."""
    V, N = 8, 4000
    rng = np.random.default_rng(kids)
    t, d = (rng.integers(-2 << 16, 2 << 16, V) for _ in range(2))
    hist = np.zeros(64, np.int32)
    parent = np.array([-1] + [0] * kids)
    got = np.zeros(V)
    for _ in range(N):
        u = rng.integers(0, 1 << 31, (kids + 1, 2))
        c = spec.draw_tokens(d, [], inv_q, rng.integers(0, 1 << 31, kids))
        tok = np.array([0] + c)
        path, nxt = spec.tree_verify(np.stack([t] * (kids + 1)), np.stack([d] * (kids + 1)), tok, parent, kids + 1,
                                     inv_t, inv_q, u, hist, 0)
        got[tok[path[1]] if len(path) > 1 else nxt] += 1
    e = spec.draw_weights(t, [], inv_t)
    p = e / e.sum()
    # children are drawn with an empty history but verified as the definition does: the root has no path ids
    assert np.all(np.abs(got / N - p) <= 5 * np.sqrt(p * (1 - p) / N) + 1e-8)


def test_masked_and_extreme_logits():
    lo = np.iinfo(np.int64).min
    x = np.array([lo, 70000, lo, 65536, lo], dtype=np.int64)
    e = spec.draw_weights(x, [0, 0, 1], 65536)
    assert e[0] == e[2] == e[4] == 0 and e[1] > 0 and e[3] > 0
    assert list(spec.draw_weights(np.full(3, lo), [], 65536)) == [65536] * 3
    assert spec.draw_index(np.zeros(4, np.int64), 5) == -1
    assert spec.draw_tokens(x, [], 0, [7, 7]) == [1, -1]


# ------------------------------------------------------------ topology and configuration
def test_tree_topology():
    from arc_chain_b200.runtime import tree_spec as ts

    assert ts.tree_levels((3, 2, 1)) == [(0, 1), (1, 4), (4, 10), (10, 16)]
    assert ts.tree_parents((3, 2)) == [-1, 0, 0, 0, 1, 1, 2, 2, 3, 3]
    assert ts.tree_levels(()) == [(0, 1)] and ts.tree_parents(()) == [-1]
    assert ts.tree_levels((63,))[-1][1] == 64
    for bad in ((64,), (2, 0), (4, 4, 4), (-1,)):
        with pytest.raises(ValueError):
            ts.tree_levels(bad)
    assert [ts.inverse_temperature(t) for t in (0, 1, 0.5, 1e-9, 1e9)] == [0, 65536, 131072, 1 << 20, 1]
    for bad in (-0.1, float("nan")):
        with pytest.raises(ValueError):
            ts.inverse_temperature(bad)


def test_run_config_of_sampled_trees():
    from arc_chain_b200.config import RunConfig

    c = RunConfig().with_overrides(["draft=draft1b", "spec_tree=3,2,1", "temperature=0.7", "sample_seed=4"])
    assert (c.spec_tree, c.temperature, c.sample_seed, c.draft_temperature) == ([3, 2, 1], 0.7, 4, 1.0)
    assert RunConfig.from_dict(__import__("json").loads(c.to_json())) == c
    for bad in (["spec_tree=3,2"], ["temperature=-1"], ["draft=tiny", "spec_tree=9,9"], ["draft_temperature=nan"]):
        with pytest.raises(ValueError):
            RunConfig().with_overrides(bad)


def test_oracle_refuses_sampling():
    from arc_chain_b200 import cli

    with pytest.raises(SystemExit):
        cli.main(["generate", "--prompt-ids", "5", "--oracle", "--set", "model=micro", "--set", "temperature=1"])


def test_decoder_refuses():
    from arc_chain_b200.runtime.tree_spec import TreeSpecDecoder

    with pytest.raises(TypeError):
        TreeSpecDecoder(object())
