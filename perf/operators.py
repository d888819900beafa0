"""Cases of the tree-speculation operators: what is measured, their plain forms and their 64-bit definitions.

Four operators make one round of speculative decoding with a tree of drafted tokens over the paged Q16 cache:

* ``attn_tree``: attention of tree nodes over the cached prefix and over their own ancestors in the tree;
* ``draw_tokens``: tokens drawn from logits with given random numbers, several per row without replacement;
* ``verify_tree``: the accepted path of drafted tokens and the token that follows it, from given random numbers;
* ``kv_keep_path``: the accepted path's K/V rows moved to the positions that they have in the sequence.

Everything is an integer: Q16 values are int64, probabilities are multiples of 2^-31, random numbers are 31-bit
integers.  Outputs are equal or wrong.
"""
import math

import numpy as np
import torch

own = False

ONE = 1 << 16
PAGE = 16
CLAMP = 1 << 40      # logits are used within +-2^40
MAX_INV_T = 1 << 20  # inverse temperatures (Q16) are used up to 16
HIST = 64            # ids that the repetition penalty looks back over

# heads, KV heads, head dim of the framework's model presets
SHAPES = {"micro_gqa": (4, 2, 64), "tiny": (4, 4, 64), "draft1b": (16, 16, 128), "llama7b": (32, 32, 128),
          "llama70b": (64, 8, 128)}


# ------------------------------------------------------------------ cases
def _attn(shape, lanes, nq, n_tree, fan, lo, hi):
    return {"op": "attn_tree", "shape": shape, "lanes": lanes, "nq": nq, "n_tree": n_tree, "fan": fan, "lo": lo,
            "hi": hi}


def _verify(lanes, n, fan, vocab, temp, near):
    return {"op": "verify_tree", "lanes": lanes, "n": n, "fan": fan, "vocab": vocab, "temp": temp, "near": near}


def _draw(lanes, n, nr, fan, m, vocab, temp):
    return {"op": "draw_tokens", "lanes": lanes, "n": n, "nr": nr, "fan": fan, "m": m, "vocab": vocab, "temp": temp}


def _keep(shape, layers, lanes, n, moved, lo, hi):
    return {"op": "kv_keep_path", "shape": shape, "layers": layers, "lanes": lanes, "n": n, "moved": moved, "lo": lo,
            "hi": hi}


def listed():
    cases = {
        # a chain of 4 drafts after a short prompt on the smallest grouped-query model: latency counts
        "attn_micro_chain": _attn("micro_gqa", 1, 5, 5, 1, 37, 37),
        # one user's request on the 7B shape, 256 tokens after a 128-token prompt, a 16-node tree
        "attn_7b_one": _attn("llama7b", 1, 16, 16, 2, 386, 386),
        # a served batch of 8 with 31-node trees, ragged lengths up to the speculative preset's
        "attn_7b_batch": _attn("llama7b", 8, 31, 31, 3, 129, 497),
        # grouped-query heads, the widest trees, lengths of the continuous-batching preset
        "attn_70b_wide": _attn("llama70b", 4, 64, 64, 4, 700, 1488),
        # one long document and the 9 newest nodes of a 13-node tree: the cache's bytes count
        "attn_70b_long": _attn("llama70b", 1, 9, 13, 3, 30011, 30011),
        # the chain of 4 drafts that the speculative decoder takes by default, one request
        "verify_chain_one": _verify(1, 5, 1, 32000, 1.0, 0.5),
        # the served batch's 31-node trees
        "verify_tree_batch": _verify(8, 31, 3, 32000, 0.7, 0.5),
        # the widest trees over the largest vocabulary with a poor draft: many residual steps
        "verify_wide_vocab": _verify(4, 64, 4, 102400, 1.0, 1.5),
        # one sampled decode step of one request
        "draw_one": _draw(1, 1, 1, 1, 1, 32000, 0.8),
        # a draft level of a served batch: 3 children of each of 9 frontier nodes
        "draw_level": _draw(8, 13, 9, 3, 3, 102400, 1.0),
        # the accepted paths of the served 7B batch, 32 layers
        "keep_7b_batch": _keep("llama7b", 32, 8, 31, 3, 129, 497),
        # one request of the grouped-query model, 80 layers, a deep path
        "keep_70b_one": _keep("llama70b", 80, 1, 64, 7, 700, 700),
    }
    return [{"name": k, **v} for k, v in cases.items()]


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 2


def _held(case):
    """Bytes of the layers' caches that a case keeps on the GPU."""
    if case["op"] != "kv_keep_path":
        return 0
    _, kv, dh = SHAPES[case["shape"]]
    return case["layers"] * case["lanes"] * (case["hi"] + case["n"] + PAGE) * kv * dh * 16


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))

    op = rng.choice(["attn_tree", "attn_tree", "verify_tree", "draw_tokens", "kv_keep_path"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        lanes, n, fan = log(1, 16), log(1, 64), rng.randint(1, 5)
        if op == "attn_tree":
            lo = log(1, 30000)
            case = _attn(rng.choice(sorted(SHAPES)), lanes, rng.randint(max(1, n // 2), n), n, fan, lo,
                         min(30011, lo + log(1, 1000)))
        elif op == "verify_tree":
            case = _verify(min(lanes, 8), n, fan, log(500, 102400), rng.choice([0.0, 0.5, 0.7, 1.0, 1.3]),
                           rng.uniform(0.0, 2.0))
        elif op == "draw_tokens":
            case = _draw(lanes, n, rng.randint(max(1, n // 2), n), fan, rng.randint(1, 8), log(500, 102400),
                         rng.choice([0.0, 0.5, 0.7, 1.0, 1.3]))
        else:
            lo = log(1, 1500)
            case = _keep(rng.choice(sorted(SHAPES)), log(2, 80), lanes, max(n, 4), rng.randint(1, max(n, 4) // 2 - 1),
                         lo, lo + log(1, 500))
        if _cost(case) <= most and _held(case) <= 10 << 30:
            return case


def _lens(case):
    """The lanes' prefix lengths, spread evenly over [lo, hi]."""
    k = case["lanes"]
    return [case["lo"] + (case["hi"] - case["lo"]) * i // max(1, k - 1) for i in range(k)]


def _parents(n, fan):
    """Level by level, `fan` children of every node (fan 1: a chain)."""
    return [-1] + [(i - 1) // fan for i in range(1, n)]


def _depths(n, fan):
    d = [0]
    for p in _parents(n, fan)[1:]:
        d.append(d[p] + 1)
    return d


def work(case):
    if case["op"] == "attn_tree":
        heads, kv, dh = SHAPES[case["shape"]]
        nq, n, lens = case["nq"], case["n_tree"], _lens(case)
        dep = _depths(n, case["fan"])[n - nq:]
        # K and V rows, queries, masks, tables and outputs once; a product and a sum for q.k and for w.v of each
        # visible (query, key) pair
        b = sum((t + n) * kv * dh * 16 + nq * (heads * dh * 16 + 8) + (t + n + 15) // 16 * 4 + 8 for t in lens)
        return {"bytes": b, "flops": 4 * heads * dh * sum(t + d + 1 for t in lens for d in dep)}
    if case["op"] == "verify_tree":
        n, v, lanes = case["n"], case["vocab"], case["lanes"]
        inner = len(set(_parents(n, case["fan"])[1:]))
        # every node's target logits, the draft's logits of the nodes that have children
        rows = lanes * (n + inner)
        return {"bytes": rows * v * 8 + lanes * (n * 20 + HIST * 4 + 28), "flops": 4 * rows * v}
    if case["op"] == "draw_tokens":
        rows = case["lanes"] * case["nr"]
        return {"bytes": rows * (case["vocab"] * 8 + case["m"] * 8) + case["lanes"] * (HIST * 4 + 12 + 8 * case["n"]),
                "flops": 4 * rows * case["vocab"]}
    _, kv, dh = SHAPES[case["shape"]]
    moved = sum(_n_moved(case, i) for i in range(case["lanes"]))
    # each moved row of K and of V read and written once in every layer
    return {"bytes": moved * case["layers"] * kv * dh * 32 + case["lanes"] * (case["n"] * 4 + 8), "flops": 0}


def _n_moved(case, lane):
    return max(1, case["moved"] - lane % 2)


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    i32 = torch.int32

    def normal(shape, std):
        return (torch.randn(shape, generator=g, device=dev) * (std * ONE)).to(torch.int64)

    def ints(lo, hi, shape, dtype=i32):
        return torch.randint(lo, hi, shape, generator=g, device=dev, dtype=dtype)

    lanes = case["lanes"]
    if case["op"] in ("attn_tree", "kv_keep_path"):
        heads, kv, dh = SHAPES[case["shape"]]
        n = case["n_tree"] if case["op"] == "attn_tree" else case["n"]
        lens = _lens(case)
        width = (max(lens) + n + PAGE - 1) // PAGE
        pages = lanes * width + 3
        pt = torch.randperm(pages, generator=g, device=dev)[:lanes * width].to(i32).view(lanes, width)
        base = torch.tensor(lens, dtype=i32, device=dev)
    if case["op"] == "attn_tree":
        nq = case["nq"]
        mask, par = [], _parents(n, case["fan"])
        for i in range(n):
            mask.append((mask[par[i]] if i else 0) | 1 << i)
        mask = [m - (1 << 64) if m >> 63 else m for m in mask[n - nq:]]
        return {"q": normal((lanes * nq, heads * dh), 2.0), "K": normal((pages, kv, PAGE, dh), 1.0),
                "V": normal((pages, kv, PAGE, dh), 1.0), "pt": pt, "base": base,
                "n_tree": torch.full((lanes,), n, dtype=i32, device=dev),
                "mask": torch.tensor(mask * lanes, dtype=torch.int64, device=dev), "heads": heads, "kv": kv, "dh": dh,
                "lanes": lanes, "nq": nq, "scale": {64: 8192, 128: 5793}[dh], "t_lim": max(lens) + n}
    if case["op"] == "kv_keep_path":
        paths = torch.full((lanes, n), -1, dtype=i32, device=dev)
        counts = [_n_moved(case, i) + 1 for i in range(lanes)]
        for i, c in enumerate(counts):
            # accepted nodes of a tree laid out level by level lie behind the path's own length
            paths[i, 1:c] = (torch.randperm(n - c, generator=g, device=dev)[:c - 1].sort().values + c).to(i32)
            paths[i, 0] = 0
        shape = (case["layers"], pages, kv, PAGE, dh)
        return {"K": normal(shape, 1.0), "V": normal(shape, 1.0), "pt": pt, "base": base, "path": paths,
                "n_path": torch.tensor(counts, dtype=i32, device=dev), "lanes": lanes, "n": n}
    n, fan, vocab = case["n"], case["fan"], case["vocab"]
    inv = 0 if case["temp"] == 0 else round(ONE / case["temp"])
    s = {"parent": torch.tensor([_parents(n, fan)] * lanes, dtype=i32, device=dev),
         "hist": ints(0, vocab, (lanes, HIST)), "count": ints(0, 300, (lanes,)),
         "inv_temp": torch.full((lanes,), inv, dtype=torch.int64, device=dev), "lanes": lanes, "n": n, "vocab": vocab,
         "depth": max(_depths(n, fan))}
    if case["op"] == "draw_tokens":
        nr, m = case["nr"], case["m"]
        return {**s, "logits": normal((lanes * nr, vocab), 2.5), "u": ints(0, 2 ** 31 - 1, (lanes * nr, m)),
                "tokens": ints(0, vocab, (lanes, n)), "nr": nr, "node0": n - nr, "m": m}
    logits = normal((lanes * n, vocab), 2.5)
    dlogits = logits + normal((lanes * n, vocab), case["near"])
    # the draft draws every node's children at temperature 1, without replacement
    kids = torch.multinomial(torch.softmax(dlogits.double() / ONE, -1).float(), fan, generator=g).view(lanes, n, fan)
    tokens = ints(0, vocab, (lanes, n))
    at = torch.arange(1, n, device=dev) - 1
    tokens[:, 1:] = kids[:, at // fan, at % fan].to(i32)
    return {**s, "logits": logits, "dlogits": dlogits, "tokens": tokens,
            "n_tree": torch.full((lanes,), n, dtype=i32, device=dev),
            "d_inv_temp": torch.full((lanes,), ONE, dtype=torch.int64, device=dev),
            "u": ints(0, 2 ** 31 - 1, (lanes, n, 2)), "fan": fan}


def prepare(case, seed):
    s = {"op": case["op"], **_inputs(case, seed)}
    if s["op"] == "attn_tree":
        s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if own and s["op"] == "kv_keep_path":
        from arc_chain_b200.ops import tree_ops as ops

        s["planes"] = ops.KvPlanes(list(s["K"]), list(s["V"]))
        s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _table(dev):
    t = [ONE]  # exp(0), then a step of 1/32 down at a time
    for _ in range(256):
        t.append((t[-1] * 63521) >> 16)
    return torch.tensor(t[::-1], dtype=torch.int64, device=dev)


def _exp(x):
    """The Q16 exponential of x <= 0: 0 from -8 down, linear between the table's steps of 1/32."""
    t = _table(x.device)
    off = (x + 8 * ONE).clamp(0, 8 * ONE)
    at = (off >> 11).clamp(max=255)
    e = t[at] + ((t[at + 1] - t[at]) * (off - (at << 11)) >> 11)
    return torch.where(x <= -8 * ONE, 0, e)


def _attn_plain(s):
    lanes, kv, nq, dh = s["lanes"], s["kv"], s["nq"], s["dh"]
    group = s["heads"] // kv
    width = (s["t_lim"] + PAGE - 1) // PAGE
    pages = s["pt"][:, :width].long()

    def rows(c):  # [lanes, kv, keys, dh]
        return c[pages].permute(0, 2, 1, 3, 4).reshape(lanes, kv, width * PAGE, dh)

    q = s["q"].view(lanes, nq, kv, group, dh).permute(0, 2, 1, 3, 4).reshape(lanes, kv, nq * group, dh)
    # products below 2^53: the 64-bit floating sum is the integer
    dots = torch.matmul(q.double(), rows(s["K"]).double().transpose(-1, -2)).to(torch.int64)
    scores = ((dots >> 16) * s["scale"]) >> 16
    j = torch.arange(width * PAGE, device=q.device) - s["base"][:, None]
    bit = (s["mask"].view(lanes, nq, 1) >> j.clamp(0, 63)[:, None]) & 1
    inside = ((j >= 0) & (j < s["n_tree"][:, None]))[:, None]
    seen = (j < 0)[:, None] | (inside & (bit == 1))
    seen = seen[:, None, :, None].expand(lanes, kv, nq, group, -1).reshape(lanes, kv, nq * group, -1)
    scores = torch.where(seen, scores, -(1 << 62))
    e = torch.where(seen, _exp(scores - scores.amax(-1, keepdim=True)), 0)
    w = e * ONE // e.sum(-1, keepdim=True).clamp(min=1)
    v = rows(s["V"])
    out = torch.zeros_like(q)
    step = max(1, (1 << 26) // out.numel())
    for a in range(0, width * PAGE, step):  # keys a few at a time: each term is rounded down by itself
        out += ((w[..., a:a + step, None] * v[:, :, None, a:a + step]) >> 16).sum(-2)
    return out.view(lanes, kv, nq, group, dh).permute(0, 2, 1, 3, 4).reshape(lanes * nq, -1)


def _weights(s, logits, inv_temp, node0, nr):
    """Unnormalised Q16 probabilities [lanes * nr, vocab] of rows that stand for nodes node0 .. node0 + nr - 1."""
    lanes, n, vocab = s["lanes"], s["n"], s["vocab"]
    dev = logits.device
    node = torch.arange(node0, node0 + nr, device=dev).expand(lanes, nr)
    # the ids behind each node, newest first: its own path up to the root, then the lane's history
    path, length = [], torch.zeros(lanes, nr, dtype=torch.int64, device=dev)
    parent, tokens = s["parent"].long(), s["tokens"].long()
    for _ in range(s["depth"]):
        live = node > 0
        path.append(torch.where(live, tokens.gather(1, node), -1))
        length += live
        node = torch.where(live, parent.gather(1, node), 0)
    path = torch.stack(path + [torch.full_like(node, -1)] * (HIST - len(path)), -1)
    at = torch.arange(HIST, device=dev) - length[..., None]
    count = s["count"].long()[:, None, None]
    old = s["hist"].long()[:, None].expand(lanes, nr, HIST).gather(2, (count - 1 - at) % HIST)
    ids = torch.where(at < 0, path, torch.where(at < count, old, vocab)).view(lanes * nr, HIST)
    # an id met several times is penalised as often; a column behind the vocabulary takes the ids that are none
    x = torch.cat([logits.clamp(-CLAMP, CLAMP), torch.zeros_like(logits[:, :1])], 1)
    met = (ids[:, :, None] == ids[:, None]).sum(-1)
    g = x.gather(1, ids)
    top, low = torch.where(g > 0, 5, 6), torch.where(g > 0, 6, 5)  # no step changes a sign
    for k in range(HIST):
        p = torch.div(g * top, low, rounding_mode="trunc").clamp(-CLAMP, CLAMP)
        g = torch.where(met > k, p, g)
    x = x.scatter_(1, ids, g)[:, :vocab]
    inv = inv_temp.clamp(0, MAX_INV_T).repeat_interleave(nr)[:, None]
    z = (x * inv) >> 16
    first = ((x == x.amax(-1, keepdim=True)).cumsum(-1) == 0).sum(-1, keepdim=True)
    hot = torch.zeros_like(x).scatter_(1, first, ONE)
    return torch.where(inv > 0, _exp(z - z.amax(-1, keepdim=True)), hot)


def _pick(w, t):
    """The first index whose running sum of w is above t."""
    return (w.cumsum(-1) <= t).sum(-1, keepdim=True)


def _draw_plain(s):
    e = _weights(s, s["logits"], s["inv_temp"], s["node0"], s["nr"])
    out = []
    for k in range(s["m"]):
        total = e.sum(-1, keepdim=True)
        u = s["u"][:, k:k + 1].long()
        t = ((u >> 16) * total + (((u & 0xFFFF) * total) >> 16)) >> 15  # u * total / 2^31 without its 64th bit
        v = _pick(e, t).clamp(max=s["vocab"] - 1)
        out.append(torch.where(total > 0, v, -1))
        e.scatter_(1, v, 0)
    return torch.cat(out, 1).to(torch.int32)


def _verify_plain(s):
    lanes, n, vocab, fan = s["lanes"], s["n"], s["vocab"], s["fan"]
    rows = lanes * n
    e = _weights(s, s["logits"], s["inv_temp"], 0, n)
    p = (e << 31) // e.sum(-1, keepdim=True)
    del e
    eq = _weights(s, s["dlogits"], s["d_inv_temp"], 0, n)
    tokens = s["tokens"].long()
    u = s["u"].long()
    node = torch.arange(n, device=p.device)
    choice = torch.full((rows, 1), -1, dtype=torch.int64, device=p.device)
    for k in range(fan):  # every node's k-th child
        child = node * fan + 1 + k
        c = child.clamp(max=n - 1).expand(lanes, n)
        d = tokens.gather(1, c).view(rows, 1)
        sq = eq.sum(-1, keepdim=True)
        asked = ((child < n).expand(lanes, n).reshape(rows, 1)) & (choice < 0) & (sq > 0) & (d >= 0) & (d < vocab)
        d = d.clamp(0, vocab - 1)
        q = (eq << 31) // sq.clamp(min=1)
        pd, qd = p.gather(1, d), q.gather(1, d)
        yes = asked & ((u[..., 0].gather(1, c).view(rows, 1) * qd >> 31) < pd)
        choice = torch.where(yes, c.reshape(rows, 1), choice)
        rest = (p - q).clamp(min=0)
        left = rest.sum(-1, keepdim=True)
        no = asked & ~yes
        p = torch.where(no & (left > 0), (rest << 31) // left.clamp(min=1), p)
        eq.scatter_(1, d, torch.where(no, 0, eq.gather(1, d)))
    drawn = _pick(p, u[..., 1].reshape(rows, 1) * p.sum(-1, keepdim=True) >> 31).view(lanes, n)
    choice = choice.view(lanes, n)
    path = torch.full((lanes, n), -1, dtype=torch.int64, device=p.device)
    path[:, 0] = 0
    last = torch.zeros(lanes, 1, dtype=torch.int64, device=p.device)
    for k in range(1, s["depth"] + 1):
        nxt = choice.gather(1, last)
        go = (nxt >= 0) & (path[:, k - 1:k] >= 0)
        path[:, k:k + 1] = torch.where(go, nxt, -1)
        last = torch.where(go, nxt, last)
    i32 = torch.int32
    return {"path": path.to(i32), "n_path": (path >= 0).sum(-1).to(i32), "next": drawn.gather(1, last)[:, 0].to(i32)}


def _keep_plain(s):
    node = torch.arange(s["n"], device=s["path"].device)
    live = node < s["n_path"][:, None]
    src = s["base"][:, None].long() + torch.where(live, s["path"].long(), 0)
    dst = s["base"][:, None].long() + torch.where(live, node, 0)
    pt = s["pt"].long()
    a, b = pt.gather(1, src // PAGE), pt.gather(1, dst // PAGE)
    k, v = s["K"][:, a, :, src % PAGE], s["V"][:, a, :, src % PAGE]
    s["K"][:, b, :, dst % PAGE] = k
    s["V"][:, b, :, dst % PAGE] = v
    return {"K": s["K"], "V": s["V"]}


# ------------------------------------------------------------------ the framework's calls
def _run_own(s):
    from arc_chain_b200.ops import tree_ops as ops

    dev = s["pt"].device if "pt" in s else s["logits"].device
    lanes = s["lanes"]
    if s["op"] == "attn_tree":
        out = torch.empty_like(s["q"])
        ops.attn_tree(s["q"], s["K"], s["V"], s["pt"], s["base"], s["n_tree"], s["mask"], s["heads"], s["kv"],
                      s["dh"], s["scale"], lanes, s["nq"], None, None, s["t_lim"], s["err"], o_out=out)
        return out
    if s["op"] == "draw_tokens":
        out = torch.empty(lanes * s["nr"], s["m"], dtype=torch.int32, device=dev)
        ops.draw_tokens(s["logits"], s["vocab"], lanes, s["nr"], s["node0"], s["m"], s["inv_temp"], s["u"], s["hist"],
                        s["count"], s["tokens"], s["parent"], out)
        return out
    if s["op"] == "verify_tree":
        path = torch.empty(lanes, s["n"], dtype=torch.int32, device=dev)
        n_path, nxt = (torch.empty(lanes, dtype=torch.int32, device=dev) for _ in range(2))
        ops.verify_tree(s["logits"], s["dlogits"], s["vocab"], lanes, s["n"], s["tokens"], s["parent"], s["n_tree"],
                        s["inv_temp"], s["d_inv_temp"], s["u"], s["hist"], s["count"], path, n_path, nxt)
        return {"path": path, "n_path": n_path, "next": nxt}
    ops.kv_keep_path(s["planes"], s["pt"], s["base"], s["path"], s["n_path"], lanes, s["n"], s["err"])
    return {"K": s["K"], "V": s["V"]}


def run(state):
    if own:
        return _run_own(state)
    plain = {"attn_tree": _attn_plain, "draw_tokens": _draw_plain, "verify_tree": _verify_plain,
             "kv_keep_path": _keep_plain}
    return plain[state["op"]](state)


# ------------------------------------------------------------------ the definitions, in 64 bits
def _steps():
    t = np.zeros(257, np.int64)
    t[256] = ONE
    for i in range(255, -1, -1):
        t[i] = int(t[i + 1]) * 63521 // ONE
    return t


def _soft(z):
    """Q16 weights e of one row of Q16 values: interpolated table of exp at multiples of 1/32."""
    t = _steps()
    x = z - z.max()
    near = x > -8 * ONE
    at, part = np.divmod(np.where(near, x, 0) + 8 * ONE, 2048)
    up = np.minimum(at + 1, 256)
    return np.where(near, t[at] + (t[up] - t[at]) * part // 2048, 0)


def _row(logits, ids, inv):
    x = np.clip(logits, -CLAMP, CLAMP)
    for i in ids:
        if 0 <= i < len(x):
            v = int(x[i])
            x[i] = max(-CLAMP, min(CLAMP, v * 5 // 6 if v > 0 else -((-v * 6) // 5)))
    if inv <= 0:
        e = np.zeros_like(x)
        e[int(np.argmax(x))] = ONE
        return e
    return _soft((x * min(inv, MAX_INV_T)) >> 16)


def _behind(h, lane, node):
    """The newest 64 ids behind a node."""
    ids = []
    while node > 0:
        ids.append(int(h["tokens"][lane, node]))
        node = int(h["parent"][lane, node])
    c = int(h["count"][lane])
    ids += [int(h["hist"][lane, (c - 1 - k) % HIST]) for k in range(min(c, HIST))]
    return ids[:HIST]


def exact(case, seed):
    if _held(case) > 2 << 30 or (case["op"] == "attn_tree" and work(case)["flops"] > 1.5e9):
        return None
    s = _inputs(case, seed)
    h = {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in s.items() if k not in ("K", "V")}
    lanes = case["lanes"]
    if case["op"] == "attn_tree":
        out = np.zeros(h["q"].shape, np.int64)
        dh, group = h["dh"], h["heads"] // h["kv"]
        for b in range(lanes):
            t = int(h["base"][b])
            total = t + int(h["n_tree"][b])
            table = s["pt"][b, :(total + PAGE - 1) // PAGE].long()
            k, v = (c[table].transpose(0, 1).reshape(h["kv"], -1, dh)[:, :total].cpu().numpy()
                    for c in (s["K"], s["V"]))
            for i in range(h["nq"]):
                bits = int(h["mask"][b * h["nq"] + i])
                keys = list(range(t)) + [t + j for j in range(total - t) if bits >> j & 1]
                for head in range(h["heads"]):
                    at = slice(head * dh, (head + 1) * dh)
                    kk, vv = k[head // group][keys], v[head // group][keys]
                    dots = (kk * h["q"][b * h["nq"] + i, at]).sum(1)
                    e = _soft(((dots >> 16) * h["scale"]) >> 16)
                    w = e * ONE // e.sum()
                    out[b * h["nq"] + i, at] = ((w[:, None] * vv) >> 16).sum(0)
        return out
    if case["op"] == "draw_tokens":
        out = np.zeros((lanes * h["nr"], h["m"]), np.int32)
        for r in range(lanes * h["nr"]):
            b, node = r // h["nr"], h["node0"] + r % h["nr"]
            e = _row(h["logits"][r], _behind(h, b, node), int(h["inv_temp"][b]))
            for k in range(h["m"]):
                total = int(e.sum())
                out[r, k] = -1
                if total > 0:
                    out[r, k] = np.searchsorted(np.cumsum(e), int(h["u"][r, k]) * total >> 31, side="right")
                    e[out[r, k]] = 0
        return out
    if case["op"] == "verify_tree":
        path = np.full((lanes, h["n"]), -1, np.int32)
        n_path, nxt = np.zeros(lanes, np.int32), np.zeros(lanes, np.int32)
        for b in range(lanes):
            node, length = 0, 0
            while True:
                path[b, length] = node
                length += 1
                r, ids = b * h["n"] + node, _behind(h, b, node)
                e = _row(h["logits"][r], ids, int(h["inv_temp"][b]))
                p = (e << 31) // int(e.sum())
                eq = _row(h["dlogits"][r], ids, int(h["d_inv_temp"][b]))
                taken = -1
                for c in np.flatnonzero(h["parent"][b] == node):
                    d, sq = int(h["tokens"][b, c]), int(eq.sum())
                    if sq == 0 or not 0 <= d < len(p):
                        continue
                    q = (eq << 31) // sq
                    if int(h["u"][b, c, 0]) * int(q[d]) >> 31 < int(p[d]):
                        taken = int(c)
                        break
                    rest = np.maximum(p - q, 0)
                    if rest.any():
                        p = (rest << 31) // int(rest.sum())
                    eq[d] = 0
                if taken < 0:
                    break
                node = taken
            n_path[b] = length
            nxt[b] = np.searchsorted(np.cumsum(p), int(h["u"][b, node, 1]) * int(p.sum()) >> 31, side="right")
        return {"path": path, "n_path": n_path, "next": nxt}
    out = {}
    for name in ("K", "V"):
        c = s[name].cpu().numpy()
        for b in range(lanes):
            where = [(int(h["pt"][b, r // PAGE]), r % PAGE) for r in range(int(h["base"][b]), int(h["base"][b]) + h["n"])]
            rows = [c[:, where[int(i)][0], :, where[int(i)][1]].copy() for i in h["path"][b, :h["n_path"][b]]]
            for i, row in enumerate(rows):
                c[:, where[i][0], :, where[i][1]] = row
        out[name] = c
    return out
