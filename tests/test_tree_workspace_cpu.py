"""The workspace that attn_tree documents: about 1 GB, or what one lane needs."""
import pytest

pytest.importorskip("torch")

from arc_chain_b200.ops._lib import lib

GB = 1 << 30


@pytest.mark.parametrize("nq,heads,kv,dh,t_lim", [
    (64, 64, 8, 128, 128), (64, 64, 64, 128, 100), (1, 64, 8, 128, 64), (4, 32, 32, 128, 254), (64, 64, 8, 128, 2048),
    (31, 32, 32, 128, 528), (9, 64, 8, 128, 30024), (64, 4, 4, 64, 1 << 20), (16, 128, 128, 8, 16)])
@pytest.mark.parametrize("lanes", [1, 8, 256, 1000])
def test_workspace_stays_within_its_bound(lanes, nq, heads, kv, dh, t_lim):
    ws = lib().arcb_attn_tree_ws(lanes, nq, heads, kv, dh, t_lim)
    assert 0 < ws <= max(GB, lib().arcb_attn_tree_ws(1, nq, heads, kv, dh, t_lim))


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
