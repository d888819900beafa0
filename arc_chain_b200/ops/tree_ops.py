"""torch-facing wrappers of the tree-speculation kernels: attention of drafted
nodes, drawing tokens, verifying drafts, keeping the accepted path.

One round of speculative decoding with a tree of drafted tokens uses them in
this order: the draft model attends its frontier nodes (:func:`attn_tree`) and
draws their children (:func:`draw_tokens`) level by level; the target model
scores every node in one forward (:func:`attn_tree`); :func:`verify_tree` picks
the accepted path and the token behind it; :func:`kv_keep_path` moves the
path's K/V rows to their positions in the sequence.
``arc_chain_b200.runtime.tree_spec`` runs such rounds.

A lane is one request.  Its tree has at most 64 nodes, node 0 the last
confirmed token, every other node behind its parent (``parent[i] < i``).  All
tensors are contiguous and on one CUDA device; launches go to that device's
current stream.  Wrong shapes, types or devices raise before anything is
launched; what only the device knows (lengths, page ids, paths) is checked by
the kernels, which skip the lane and set a bit of ``err``.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from arc_chain_b200.ops import int_ops
from arc_chain_b200.ops._lib import check, lib

MAX_NODES = 64
HIST = 64
MAX_INV_TEMP = 1 << 20  # Q16: inverse temperatures are used up to 16
PAGE = 16
I32, I64, I8 = torch.int32, torch.int64, torch.int8


def _need(what: str, t, dtype, shape) -> None:
    """t is a contiguous tensor of the given type and shape (None: any size)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    s = t.shape
    if len(s) != len(shape) or any(w is not None and g != w for g, w in zip(s, shape)):
        raise ValueError(f"{what} must have shape {tuple('any' if w is None else w for w in shape)}, got {tuple(s)}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")


def _rows(what: str, t, dtype, rows: int, cols: int) -> int:
    """t is [>= rows, >= cols] with contiguous rows; returns the row stride."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.dim() != 2 or t.shape[0] < rows or t.shape[1] < cols:
        raise ValueError(f"{what} must be at least [{rows}, {cols}], got {tuple(t.shape)}")
    if t.stride(1) != 1 or (rows > 1 and t.stride(0) < cols):
        raise ValueError(f"{what} must have contiguous rows that do not overlap")
    return t.stride(0)


def _place(*ts) -> torch.device:
    dev = ts[0].device
    for t in ts:
        if t is not None and t.device != dev:
            raise ValueError(f"all tensors must be on one device, got {dev} and {t.device}")
    if dev.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, got {dev}")
    return dev


def _call(dev: torch.device, f, what: str, *args) -> None:
    if dev.index == torch.cuda.current_device():
        rc = f(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = f(*args, torch.cuda.current_stream().cuda_stream)
    int_ops._count()
    check(rc, what)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def attn_tree(q, Kc, Vc, pt, base, n_tree, mask, n_heads: int, n_kv: int, dh: int, attn_scale: int, lanes: int,
              nq: int, X, lmax, t_lim: int, err, o_out=None) -> None:
    """Attention of nq tree nodes of each lane over its paged cache.

    q [lanes * nq, n_heads * dh] int64 (slot = lane * nq + i); Kc, Vc [pages,
    n_kv, 16, dh]; pt [lanes, pages per lane] int32 (rows may be strided);
    base [lanes] cached tokens; n_tree [lanes] drafted nodes, whose K/V rows
    are at positions base + i; mask [lanes * nq] int64: bit j set lets the
    query see node j.  Every query sees all keys below base.  t_lim bounds
    base + n_tree.  base = n_tree = 0 is an idle lane (zero outputs).

    Outputs: the limb planes X of the W_o operand with their count lmax
    (int_ops.limb_row layout of lanes * nq slots), and / or o_out [lanes * nq,
    n_heads * dh] int64.  A lane whose lengths or pages are out of range gets
    zeros and sets a bit of err."""
    if lanes < 1 or nq < 1 or lanes * nq > 65535:
        raise ValueError(f"lanes and nq must be at least 1 and lanes * nq at most 65535, got {lanes} and {nq}")
    if n_kv < 1 or n_heads < 1 or n_heads % n_kv:
        raise ValueError(f"n_heads must be a multiple of n_kv, got {n_heads} and {n_kv}")
    if dh < 8 or dh > 128 or dh % 8:
        raise ValueError(f"dh must be a multiple of 8 up to 128, got {dh}")
    if t_lim < 1:
        raise ValueError(f"t_lim must be at least 1, got {t_lim}")
    B, d = lanes * nq, n_heads * dh
    _need("q", q, I64, (B, d))
    _need("Kc", Kc, I64, (None, n_kv, PAGE, dh))
    _need("Vc", Vc, I64, tuple(Kc.shape))
    ps = _rows("pt", pt, I32, lanes, 1)
    _need("base", base, I32, (lanes,))
    _need("n_tree", n_tree, I32, (lanes,))
    _need("mask", mask, I64, (B,))
    _need("err", err, I32, (1,))
    if X is None and o_out is None:
        raise ValueError("one of X and o_out must be given")
    if X is not None:
        _need("X", X, I8, (None, d))
        if X.shape[0] < 8 * int_ops.n_tiles(B) * int_ops.limb_slots(B):
            raise ValueError(f"X has {X.shape[0]} rows, too few for {B} slots")
    if lmax is not None:
        _need("lmax", lmax, I32, (1,))
    if o_out is not None:
        _need("o_out", o_out, I64, (B, d))
    dev = _place(q, Kc, Vc, pt, base, n_tree, mask, err, X, lmax, o_out)
    if any(t is not None and t.data_ptr() % 16 for t in (q, Kc, Vc, X, o_out)):
        raise ValueError("q, Kc, Vc, X and o_out must start on a 16-byte boundary")
    L = lib()
    ws = torch.empty(L.arcb_attn_tree_ws(lanes, nq, n_heads, n_kv, dh, t_lim), dtype=torch.uint8, device=dev)
    _call(dev, L.arcb_attn_tree, "attn_tree", _p(q), _p(Kc), _p(Vc), Kc.shape[0], _p(pt), ps, pt.shape[1], _p(base),
          _p(n_tree), _p(mask), nq, n_heads, n_kv, dh, int(attn_scale), t_lim, lanes, _p(ws), _p(X), _p(lmax),
          _p(o_out), _p(err))


def _vocab(V: int, lanes: int) -> None:
    if V < 1 or V > lib_max_vocab():
        raise ValueError(f"vocabulary must have 1 to {lib_max_vocab()} tokens, got {V}")
    if lanes < 1 or lanes > 65535:
        raise ValueError(f"lanes must be 1 to 65535, got {lanes}")


def lib_max_vocab() -> int:
    """Largest vocabulary of draw_tokens and verify_tree."""
    return lib().arcb_draw_max_vocab()


def draw_tokens(logits, V: int, lanes: int, nr: int, node0: int, m: int, inv_temp, u, hist, count, tokens, parent,
                out) -> None:
    """m tokens drawn from each logits row without replacement, into out
    [lanes * nr, m] int32 (-1 where nothing is left to draw).

    Row lane * nr + i of logits (int64 Q16, at least V columns) is node node0 +
    i of the lane's tree tokens / parent [lanes, n] int32.  Its newest 64 ids
    (the tokens on its path, then the lane's ring hist [lanes, 64] of count
    [lanes] tokens) are penalised as the greedy step does.  inv_temp [lanes]
    int64 is the Q16 inverse temperature, used up to 16; 0 or less draws the
    first maximum.  u [lanes * nr, m] int32 are the random numbers, uniform in
    [0, 2^31).  A plain sampled step is nr = 1, node0 = 0, m = 1 with one-node
    trees."""
    _vocab(V, lanes)
    if not isinstance(tokens, torch.Tensor) or tokens.dim() != 2:
        raise ValueError("tokens must be a tensor [lanes, nodes]")
    n = tokens.shape[1]
    if n < 1 or n > MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {n}")
    if nr < 1 or node0 < 0 or node0 + nr > n:
        raise ValueError(f"rows stand for nodes {node0} to {node0 + nr - 1} of a {n}-node tree")
    if m < 1:
        raise ValueError(f"m must be at least 1, got {m}")
    ldl = _rows("logits", logits, I64, lanes * nr, V)
    _need("inv_temp", inv_temp, I64, (lanes,))
    _need("u", u, I32, (lanes * nr, m))
    _need("hist", hist, I32, (lanes, HIST))
    _need("count", count, I32, (lanes,))
    _need("tokens", tokens, I32, (lanes, n))
    _need("parent", parent, I32, (lanes, n))
    _need("out", out, I32, (lanes * nr, m))
    dev = _place(logits, inv_temp, u, hist, count, tokens, parent, out)
    _call(dev, lib().arcb_draw_tokens, "draw_tokens", _p(logits), ldl, V, lanes, nr, n, node0, m, _p(inv_temp), _p(u),
          _p(hist), _p(count), _p(tokens), _p(parent), _p(out))


def verify_tree(logits, dlogits, V: int, lanes: int, n: int, tokens, parent, n_tree, inv_temp, d_inv_temp, u, hist,
                count, path, n_path, nxt) -> None:
    """The accepted path of each lane's tree and the token behind it, so that
    the tokens are distributed as the target's own (speculative sampling with
    several children per node, drawn without replacement).

    Row lane * n + i of logits and of dlogits are the target's and the draft's
    Q16 logits at node i (the draft's are read for nodes that have children).
    tokens, parent [lanes, n] int32; n_tree [lanes] live nodes; inv_temp,
    d_inv_temp [lanes] as in draw_tokens, each as its model was drawn from; u
    [lanes, n, 2] int32 in [0, 2^31): u[..., 0] decides node i, u[..., 1]
    draws the token behind node i.  Children of a node are asked in node order.
    With inv_temp 0 the accepted path is the greedy one.

    path [lanes, n] int32 gets the accepted nodes from the root on, then -1;
    n_path [lanes] their number; nxt [lanes] the next token (-1 and 0 nodes for
    n_tree = 0)."""
    _vocab(V, lanes)
    if n < 1 or n > MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {n}")
    ldl = _rows("logits", logits, I64, lanes * n, V)
    ldd = _rows("dlogits", dlogits, I64, lanes * n, V)
    _need("tokens", tokens, I32, (lanes, n))
    _need("parent", parent, I32, (lanes, n))
    _need("n_tree", n_tree, I32, (lanes,))
    _need("inv_temp", inv_temp, I64, (lanes,))
    _need("d_inv_temp", d_inv_temp, I64, (lanes,))
    _need("u", u, I32, (lanes, n, 2))
    _need("hist", hist, I32, (lanes, HIST))
    _need("count", count, I32, (lanes,))
    _need("path", path, I32, (lanes, n))
    _need("n_path", n_path, I32, (lanes,))
    _need("nxt", nxt, I32, (lanes,))
    dev = _place(logits, dlogits, tokens, parent, n_tree, inv_temp, d_inv_temp, u, hist, count, path, n_path, nxt)
    scratch = torch.empty(2 * lanes * n, dtype=I32, device=dev)
    _call(dev, lib().arcb_verify_tree, "verify_tree", _p(logits), ldl, _p(dlogits), ldd, V, lanes, n, _p(tokens),
          _p(parent), _p(n_tree), _p(inv_temp), _p(d_inv_temp), _p(u), _p(hist), _p(count), _p(scratch), _p(path),
          _p(n_path), _p(nxt))
    int_ops._count()  # two kernels


class KvPlanes:
    """The K and V tensors of a paged cache's layers as a device table of
    their addresses, for kernels that touch every layer in one launch."""

    def __init__(self, Ks: Sequence[torch.Tensor], Vs: Sequence[torch.Tensor]):
        ts = {id(t): t for t in [*Ks, *Vs]}  # a latent cache's V is its K
        self.tensors = list(ts.values())
        if not self.tensors:
            raise ValueError("a cache has at least one layer")
        first = self.tensors[0]
        if not isinstance(first, torch.Tensor) or first.dim() != 4 or first.shape[2] != PAGE or first.shape[3] % 2:
            raise ValueError("cache tensors are [pages, n_kv, 16, d_head] with an even d_head")
        for t in self.tensors:
            _need("cache tensor", t, I64, tuple(first.shape))
        self.n_pages, self.n_kv, _, self.dh = first.shape
        self.device = _place(*self.tensors)
        self.table = torch.tensor([t.data_ptr() for t in self.tensors], dtype=I64, device=self.device)


def kv_keep_path(planes: KvPlanes, pt, base, path, n_path, lanes: int, n: int, err) -> None:
    """Moves, in every layer's K and V, the rows of an accepted path to
    consecutive positions: row base + path[i] to base + i for i < n_path.

    pt [lanes, pages per lane] int32 (rows may be strided), base [lanes], path
    [lanes, n] and n_path [lanes] int32 as verify_tree leaves them.  A lane
    whose path is not increasing from 0, or leaves the table or the cache, is
    left as it is and sets a bit of err.  Lanes share no page."""
    if lanes < 1 or lanes > 65535:
        raise ValueError(f"lanes must be 1 to 65535, got {lanes}")
    if n < 1 or n > MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {n}")
    if not isinstance(planes, KvPlanes):
        raise TypeError(f"planes must be KvPlanes, got {type(planes).__name__}")
    ps = _rows("pt", pt, I32, lanes, 1)
    _need("base", base, I32, (lanes,))
    _need("path", path, I32, (lanes, n))
    _need("n_path", n_path, I32, (lanes,))
    _need("err", err, I32, (1,))
    dev = _place(planes.table, pt, base, path, n_path, err)
    _call(dev, lib().arcb_kv_keep_path, "kv_keep_path", _p(planes.table), len(planes.tensors), planes.n_pages,
          planes.n_kv, planes.dh, _p(pt), ps, pt.shape[1], _p(base), _p(path), _p(n_path), lanes, n, _p(err))
