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
