"""KvPlanes: a cache tensor given twice is moved once, overlapping ones are refused."""
import pytest

torch = pytest.importorskip("torch")

from arc_chain_b200.ops import tree_ops as ops


def test_views_of_one_tensor_are_one_plane():
    """Two planes of one tensor would move its rows twice at once."""
    k, other = (torch.zeros(3, 2, 16, 64, dtype=torch.int64) for _ in range(2))
    got = ops.KvPlanes.distinct([k, other, k, k.view_as(k), k[:], other.detach()])
    assert len(got) == 2 and got[0] is k and got[1] is other


def test_overlapping_tensors_are_refused():
    pool = torch.zeros(5, 2, 16, 64, dtype=torch.int64)
    with pytest.raises(ValueError, match="overlap"):
        ops.KvPlanes([pool[:3]], [pool[2:]])
    with pytest.raises(ValueError, match="CUDA"):  # next to each other: refused for the CPU only
        ops.KvPlanes([pool[:2]], [pool[2:4]])
