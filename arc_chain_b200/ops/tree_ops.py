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

import functools
from typing import Optional, Sequence

import torch

from arc_chain_b200.ops import int_ops
from arc_chain_b200.ops._lib import check, lib

MAX_NODES = 64
HIST = 64
MAX_INV_TEMP = 1 << 20  # Q16: inverse temperatures are used up to 16
PAGE = 16
I32, I64, I8 = torch.int32, torch.int64, torch.int8


def _refuse(what: str, t, dtype, shape, dev) -> None:
    """Raises what is wrong with a tensor that _check did not pass."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    raise ValueError(f"{what} is on {t.device}, other tensors on {dev}")


def _check(dev, *specs) -> None:
    """Every (name, tensor, type, shape) is a contiguous tensor on dev.  On the
    path of calls of some 10 us: only what costs least is asked of a good one."""
    at = -1 if dev.index is None else dev.index
    try:
        for what, t, dtype, shape in specs:
            if t.dtype is not dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != at:
                _refuse(what, t, dtype, shape, dev)
    except AttributeError:
        _refuse(what, t, dtype, shape, dev)
        raise


def _rows(dev, what: str, t, dtype, rows: int, cols: int) -> int:
    """t is [>= rows, >= cols] on dev with contiguous rows; returns the row stride."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.dim() != 2 or t.shape[0] < rows or t.shape[1] < cols:
        raise ValueError(f"{what} must be at least [{rows}, {cols}], got {tuple(t.shape)}")
    step, one = t.stride()
    if one != 1 or (rows > 1 and step < cols):
        raise ValueError(f"{what} must have contiguous rows that do not overlap")
    if t.device != dev:
        raise ValueError(f"{what} is on {t.device}, other tensors on {dev}")
    return step


def _device(what: str, t, dims: int) -> torch.device:
    """The device that the first tensor of a call is on."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor, got {type(t).__name__}")
    if t.dim() != dims:
        raise ValueError(f"{what} must have {dims} dimensions, got {tuple(t.shape)}")
    return t.device


def _call(dev: torch.device, f, what: str, *args) -> None:
    """Launches on dev's current stream."""
    if dev.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, got {dev}")
    if dev.index == torch._C._cuda_getDevice():  # tensors on the device: CUDA is initialised
        rc = f(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = f(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    int_ops._count()
    check(rc, what)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=256)
def _attn_ws(lanes: int, nq: int, n_heads: int, n_kv: int, dh: int, t_lim: int) -> int:
    """Bytes of attn_tree's workspace."""
    return lib().arcb_attn_tree_ws(lanes, nq, n_heads, n_kv, dh, t_lim)


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
    zeros and sets a bit of err.

    A call takes a workspace of some 4 bytes for each key up to t_lim, and 2 to
    4 KB, for every query and query head (those of a KV head counted as 8, or
    as a multiple of 16): of as many lanes as 1 GB of scores and 6 GB in all
    hold (one at least); the others follow in further launches."""
    if lanes < 1 or nq < 1 or lanes * nq > 65535:
        raise ValueError(f"lanes and nq must be at least 1 and lanes * nq at most 65535, got {lanes} and {nq}")
    if n_kv < 1 or n_heads < 1 or n_heads % n_kv:
        raise ValueError(f"n_heads must be a multiple of n_kv, got {n_heads} and {n_kv}")
    if dh < 8 or dh > 128 or dh % 8:
        raise ValueError(f"dh must be a multiple of 8 up to 128, got {dh}")
    if t_lim < 1:
        raise ValueError(f"t_lim must be at least 1, got {t_lim}")
    if not -1 << 63 <= attn_scale < 1 << 63:
        raise ValueError(f"attn_scale must be a 64-bit integer, got {attn_scale}")
    B, d = lanes * nq, n_heads * dh
    dev = _device("Kc", Kc, 4)
    pages = Kc.shape[0]
    cache = (pages, n_kv, PAGE, dh)
    _check(dev, ("q", q, I64, (B, d)), ("Kc", Kc, I64, cache), ("Vc", Vc, I64, cache), ("base", base, I32, (lanes,)),
           ("n_tree", n_tree, I32, (lanes,)), ("mask", mask, I64, (B,)), ("err", err, I32, (1,)))
    ps = _rows(dev, "pt", pt, I32, lanes, 1)
    t_lim = min(t_lim, pt.shape[1] * PAGE)  # no lane has more keys than its pages hold
    at = q.data_ptr() | Kc.data_ptr() | Vc.data_ptr()
    if X is None and o_out is None:
        raise ValueError("one of X and o_out must be given")
    if X is not None:
        if _rows(dev, "X", X, I8, 8 * int_ops.n_tiles(B) * int_ops.limb_slots(B), d) != d or X.shape[1] != d:
            raise ValueError(f"X must have {d} columns, got {tuple(X.shape)}")
        at |= X.data_ptr()
    if lmax is not None:
        _check(dev, ("lmax", lmax, I32, (1,)))
    if o_out is not None:
        _check(dev, ("o_out", o_out, I64, (B, d)))
        at |= o_out.data_ptr()
    if at % 16:
        raise ValueError("q, Kc, Vc, X and o_out must start on a 16-byte boundary")
    size = _attn_ws(lanes, nq, n_heads, n_kv, dh, t_lim)
    if size < 0:
        raise ValueError(f"attn_tree takes up to {65535 * 32 // n_kv} queries times query heads per KV head and "
                         f"{65535 * 16 * 128} keys a lane, got {nq * (n_heads // n_kv)} and {t_lim}")
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _call(dev, lib().arcb_attn_tree, "attn_tree", q.data_ptr(), Kc.data_ptr(), Vc.data_ptr(), pages, pt.data_ptr(), ps,
          pt.shape[1], base.data_ptr(), n_tree.data_ptr(), mask.data_ptr(), nq, n_heads, n_kv, dh, int(attn_scale),
          t_lim, lanes, ws.data_ptr(), _p(X), _p(lmax), _p(o_out), err.data_ptr())


def _vocab(V: int, lanes: int) -> None:
    if V < 1 or V > lib_max_vocab():
        raise ValueError(f"vocabulary must have 1 to {lib_max_vocab()} tokens, got {V}")
    if lanes < 1 or lanes > 65535:
        raise ValueError(f"lanes must be 1 to 65535, got {lanes}")


@functools.lru_cache(maxsize=None)
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
    dev = _device("logits", logits, 2)
    ldl = _rows(dev, "logits", logits, I64, lanes * nr, V)
    _check(dev, ("inv_temp", inv_temp, I64, (lanes,)), ("u", u, I32, (lanes * nr, m)),
           ("hist", hist, I32, (lanes, HIST)), ("count", count, I32, (lanes,)), ("tokens", tokens, I32, (lanes, n)),
           ("parent", parent, I32, (lanes, n)), ("out", out, I32, (lanes * nr, m)))
    _call(dev, lib().arcb_draw_tokens, "draw_tokens", logits.data_ptr(), ldl, V, lanes, nr, n, node0, m,
          inv_temp.data_ptr(), u.data_ptr(), hist.data_ptr(), count.data_ptr(), tokens.data_ptr(), parent.data_ptr(),
          out.data_ptr())


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
    dev = _device("logits", logits, 2)
    ldl = _rows(dev, "logits", logits, I64, lanes * n, V)
    ldd = _rows(dev, "dlogits", dlogits, I64, lanes * n, V)
    one, per = (lanes,), (lanes, n)
    _check(dev, ("tokens", tokens, I32, per), ("parent", parent, I32, per), ("n_tree", n_tree, I32, one),
           ("inv_temp", inv_temp, I64, one), ("d_inv_temp", d_inv_temp, I64, one), ("u", u, I32, (lanes, n, 2)),
           ("hist", hist, I32, (lanes, HIST)), ("count", count, I32, one), ("path", path, I32, per),
           ("n_path", n_path, I32, one), ("nxt", nxt, I32, one))
    _call(dev, lib().arcb_verify_tree, "verify_tree", logits.data_ptr(), ldl, dlogits.data_ptr(), ldd, V, lanes, n,
          tokens.data_ptr(), parent.data_ptr(), n_tree.data_ptr(), inv_temp.data_ptr(), d_inv_temp.data_ptr(),
          u.data_ptr(), hist.data_ptr(), count.data_ptr(), path.data_ptr(), n_path.data_ptr(), nxt.data_ptr())


class KvPlanes:
    """The K and V tensors of a paged cache's layers as a device table of
    their addresses, for kernels that touch every layer in one launch."""

    def __init__(self, Ks: Sequence[torch.Tensor], Vs: Sequence[torch.Tensor]):
        ts = [*Ks, *Vs]
        if not ts:
            raise ValueError("a cache has at least one layer")
        first = ts[0]
        if not isinstance(first, torch.Tensor) or first.dim() != 4 or first.shape[2] != PAGE or first.shape[3] % 2:
            raise ValueError("cache tensors are [pages, n_kv, 16, d_head] with an even d_head")
        self.device = first.device
        _check(self.device, *(("cache tensor", t, I64, first.shape) for t in ts))
        self.tensors = self.distinct(ts)
        if self.device.type != "cuda":
            raise ValueError(f"tensors must be on a CUDA device, got {self.device}")
        if any(t.data_ptr() % 16 for t in self.tensors):
            raise ValueError("cache tensors must start on a 16-byte boundary")
        self.n_pages, self.n_kv, _, self.dh = first.shape
        self.table = torch.tensor([t.data_ptr() for t in self.tensors], dtype=I64, device=self.device)

    @staticmethod
    def distinct(ts: Sequence[torch.Tensor]) -> list:
        """Tensors of one shape, each piece of memory once (a latent cache's V
        is its K): every plane's rows are moved at the same time."""
        at = {}
        for t in ts:
            at.setdefault(t.data_ptr(), t)
        starts = sorted(at)
        if any(b - a < t.numel() * t.element_size() for a, b in zip(starts, starts[1:])):
            raise ValueError("cache tensors overlap")
        return list(at.values())


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
    dev = planes.device
    ps = _rows(dev, "pt", pt, I32, lanes, 1)
    _check(dev, ("base", base, I32, (lanes,)), ("path", path, I32, (lanes, n)), ("n_path", n_path, I32, (lanes,)),
           ("err", err, I32, (1,)))
    _call(dev, lib().arcb_kv_keep_path, "kv_keep_path", planes.table.data_ptr(), len(planes.tensors), planes.n_pages,
          planes.n_kv, planes.dh, pt.data_ptr(), ps, pt.shape[1], base.data_ptr(), path.data_ptr(), n_path.data_ptr(),
          lanes, n, err.data_ptr())
