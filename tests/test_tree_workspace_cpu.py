"""The workspace that attn_tree documents: 6 GB at most, or what one lane needs."""
import pytest

pytest.importorskip("torch")

from arc_chain_b200.ops._lib import lib

MOST = 6 << 30


@pytest.mark.parametrize("nq,heads,kv,dh,t_lim", [
    (64, 64, 8, 128, 128), (64, 64, 64, 128, 100), (1, 64, 8, 128, 64), (4, 32, 32, 128, 254), (64, 64, 8, 128, 2048),
    (31, 32, 32, 128, 528), (9, 64, 8, 128, 30024), (64, 4, 4, 64, 1 << 20), (16, 128, 128, 8, 16),
    (1, 32, 32, 128, 128), (64, 128, 128, 128, 100)])
@pytest.mark.parametrize("lanes", [1, 8, 256, 1000, 8000])
def test_workspace_stays_within_its_bound(lanes, nq, heads, kv, dh, t_lim):
    lanes = min(lanes, 65535 // nq)
    ws = lib().arcb_attn_tree_ws(lanes, nq, heads, kv, dh, t_lim)
    assert 0 < ws <= max(MOST, lib().arcb_attn_tree_ws(1, nq, heads, kv, dh, t_lim))


def test_scores_alone_fill_a_batch():
    """Two lanes of 64 nodes and 32 thousand keys, whose scores are 1 GB, go together."""
    ws = [lib().arcb_attn_tree_ws(n, 64, 64, 8, 128, 1 << 15) for n in (1, 2, 3)]
    assert ws[0] < 600e6 < 1 << 30 < ws[1] == ws[2]


@pytest.mark.parametrize("bad", [dict(kv=0), dict(kv=-1), dict(t_lim=0), dict(t_lim=-5), dict(lanes=0), dict(nq=0),
                                 dict(heads=0), dict(dh=0), dict(heads=7), dict(dh=136), dict(dh=12), dict(t_lim=(1 << 31) - 1),
                                 dict(lanes=1 << 20), dict(nq=1 << 30)], ids=str)
def test_sizes_that_no_call_takes(bad):
    """Asked in a process of its own: a division by zero would end it."""
    import subprocess
    import sys

    a = {**dict(lanes=2, nq=4, heads=8, kv=2, dh=64, t_lim=100), **bad}
    code = (f"from arc_chain_b200.ops._lib import lib; print(lib().arcb_attn_tree_ws({a['lanes']}, {a['nq']}, "
            f"{a['heads']}, {a['kv']}, {a['dh']}, {a['t_lim']}))")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and int(r.stdout.strip()) < 0, (r.returncode, r.stdout, r.stderr)
