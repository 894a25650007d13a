"""Operators for drafted trees: what a guard beside a speculating language model calls, one operator at a time.

The model drafts a tree of continuations of a live session; the guard scores every node of it against the session's state
without moving that state, and moves it along the nodes that were accepted (a row's first ``commits`` nodes, a chain).
A row is one session's tree: nodes in an order in which every parent comes first, ``parents`` row-local (-1: the child of
the session's last token), all rows packed one after another.

* ``maps``: offsets, positions and ancestor sets of the packed rows from their lengths and parents, on the GPU.
* ``conv``: the gated-delta layer's causal depthwise convolution (4 taps) + SiLU along each node's own path, over the
  slot's history where the path ends.
* ``gdn``: the gated-delta rule along each node's path from the slot's recurrent state, with the layer's gated RMSNorm.
* ``attention``: window attention of each node over the slot's ring of 512 keys and the node's own ancestors.

Where ``own`` is false ``run`` computes the formulas in plain torch operations in 32 bits; where it is true it calls
``hs_guard.engine.kernels``.
"""
import math
import os
import random
import sys

import torch

own = False

BF16, F32, F64, I64 = torch.bfloat16, torch.float32, torch.float64, torch.long
DEV = "cuda"
H, KD = 16, 128                # gated-delta key heads; key and value width
HD, W = 256, 512               # attention head width and window
TAPS = 4
MOST = 64                      # nodes of a row
EPS = 1e-6


def listed():
    return [
        # maps: a handful of sessions' drafts (a launch's latency), and every session of a large engine
        {"name": "maps_4x24", "op": "maps", "rows": 4, "nodes": 24, "commits": False},
        {"name": "maps_512x64", "op": "maps", "rows": 512, "nodes": 64, "commits": True},
        # conv: one session's draft; a full engine's drafts with the accepted nodes committed to the histories
        {"name": "conv_1x12", "op": "conv", "rows": 1, "nodes": 12, "commits": False, "value_heads": 16},
        {"name": "conv_352x21", "op": "conv", "rows": 352, "nodes": 21, "commits": True, "value_heads": 16},
        # gdn: one session's draft (latency)
        {"name": "gdn_1x12", "op": "gdn", "rows": 1, "nodes": 12, "commits": False, "value_heads": 16, "state": "float32"},
        # one candidate token for each session of a full engine, before it is sent: bound by reading the states
        {"name": "gdn_352x1", "op": "gdn", "rows": 352, "nodes": 1, "commits": False, "value_heads": 16,
         "state": "float32"},
        # ordinary trees with commits, states in 16 bits, two value heads to a key head
        {"name": "gdn_96x33", "op": "gdn", "rows": 96, "nodes": 33, "commits": True, "value_heads": 32,
         "state": "float16"},
        # the largest trees of many sessions, with commits
        {"name": "gdn_128x64", "op": "gdn", "rows": 128, "nodes": 64, "commits": True, "value_heads": 16,
         "state": "float32"},
        # attention: one session's draft (latency)
        {"name": "attention_1x12", "op": "attention", "rows": 1, "nodes": 12, "commits": False, "q_heads": 16},
        # one candidate token for each session of a full engine: bound by reading the rings
        {"name": "attention_352x1", "op": "attention", "rows": 352, "nodes": 1, "commits": False, "q_heads": 16},
        # ordinary trees with commits at the released head counts
        {"name": "attention_96x33", "op": "attention", "rows": 96, "nodes": 33, "commits": True, "q_heads": 8},
        # the largest trees of many sessions
        {"name": "attention_128x64", "op": "attention", "rows": 128, "nodes": 64, "commits": True, "q_heads": 16},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["maps", "conv", "gdn", "attention", "gdn", "attention"])
    nodes = rng.choice([1, rng.randint(2, 8), spread(2, MOST), rng.randint(9, MOST)])
    case = {"op": op, "rows": spread(1, 512 if op == "maps" else min(352, 128 * MOST // nodes)), "nodes": nodes,
            "commits": rng.random() < 0.5}
    if op in ("conv", "gdn"):
        case["value_heads"] = rng.choice([16, 16, 32])
    if op == "gdn":
        case["state"] = rng.choice(["float32", "float16"])
        if case["value_heads"] == 32:
            case["rows"] = max(1, case["rows"] // 2)
    if op == "attention":
        case["q_heads"] = rng.choice([16, 8])
    return case


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------
def _rows(case, seed):
    """The rows' trees: (parents, nodes to commit) of each. The sizes are one multiset a case, so that every seed is the
    same work; their order and the trees come from the seed."""
    sizes = random.Random("%d %d" % (case["rows"], case["nodes"]))
    lens = [case["nodes"] if n == 0 else sizes.randint(max(1, case["nodes"] // 3), case["nodes"])
            for n in range(case["rows"])]
    rng = random.Random(int(seed))
    rng.shuffle(lens)
    rows = []
    for size in lens:
        # a chain; a few continuations of the recent nodes (a beam); any tree
        style = rng.random()
        chain = rng.randint(0, size) if case["commits"] else 0
        parents = []
        for i in range(size):
            if i < chain or style < 0.2 or rng.random() < 0.35:
                parents.append(i - 1)
            elif style < 0.7:
                parents.append(rng.randint(max(-1, i - 6), i - 1))
            else:
                parents.append(rng.randint(-1, i - 1))
        rows.append((parents, chain))
    return rows


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=I64).to(DEV)


def _trees(s, case, seed, g):
    """A batch of trees: what the maps are made of, and the maps."""
    rows = _rows(case, seed)
    n = case["rows"]
    # one session in four is in its first window, the others past it
    starts = torch.randint(1, 8000, (n,), generator=g, device=DEV)
    s["starts"] = torch.where(torch.rand(n, generator=g, device=DEV) < 0.25, starts % W, starts + W)
    s["parents"] = _ints([p for parents, _ in rows for p in parents])
    s["lens"] = _ints([len(parents) for parents, _ in rows])
    s["commits"] = _ints([c for _, c in rows]) if case["commits"] else None
    s["slots"] = torch.randperm(n, generator=g, device=DEV)
    if case["op"] != "maps":
        s["trees"] = _plain_maps(s["parents"], s["lens"], s["starts"], s["commits"], case["nodes"])
    return int(s["parents"].numel())


def _decay(g, heads):
    """A_log and dt_bias as gated-delta layers are initialised: A in [1, 16], time steps in [1e-3, 1e-1]."""
    a_log = torch.log(torch.rand(heads, generator=g, device=DEV) * 15 + 1)
    dt = torch.exp(torch.rand(heads, generator=g, device=DEV) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    return a_log.to(BF16), torch.log(torch.expm1(dt)).to(BF16)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    total, n, op = _trees(s, case, seed, g), case["rows"], case["op"]
    if op == "conv":
        c = (2 * H + case["value_heads"]) * KD
        s.update(x=_randn(g, total, c), pool=_randn(g, n + 1, TAPS - 1, c), weight=_randn(g, c, 1, TAPS, scale=0.5))
    elif op == "gdn":
        hv = case["value_heads"]
        dtype = F32 if case["state"] == "float32" else torch.float16
        # the layer's convolution ends in SiLU: q, k, v are SiLU outputs
        s["packed"] = torch.nn.functional.silu(_randn(g, total, (2 * H + hv) * KD, dtype=F32)).to(BF16)
        s["A_log"], s["dt_bias"] = _decay(g, hv)
        s.update(a=_randn(g, total, hv), b=_randn(g, total, hv), z=_randn(g, total, hv * KD),
                 norm=(1 + _randn(g, KD, scale=0.1, dtype=F32)).to(BF16),
                 state=_randn(g, n + 1, hv, KD, KD, scale=0.1, dtype=dtype))
    elif op == "attention":
        hq, hkv = case["q_heads"], case["q_heads"] // 4
        columns = torch.arange(W, device=DEV)[None]
        start = s["starts"][:, None]
        last = start - W + torch.remainder(columns - start, W)      # the last position before the start in each column
        ring_pos = torch.full((n + 1, W + 1), -1, dtype=I64, device=DEV)
        ring_pos[s["slots"], :W] = torch.where(last >= 0, last, -1)
        s.update(ring_pos=ring_pos, q=_randn(g, total, hq, HD), new_k=_randn(g, total, hkv, HD),
                 value=_randn(g, total, hkv, HD), gate=_randn(g, total, hq * 2 * HD),
                 ring_k=_randn(g, n + 1, hkv, W + 1, HD), ring_v=_randn(g, n + 1, hkv, W + 1, HD))
    return s


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------
def _kernels():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hs-guard_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from hs_guard.engine import kernels
    return kernels


@torch.no_grad()
def run(s):
    case = s["case"]
    op, nodes = case["op"], case["nodes"]
    if op == "maps":
        if own:
            maps = _kernels().draft_tree_maps(s["parents"], s["lens"], s["starts"], s["commits"], max_nodes=nodes)[:5]
        else:
            maps = _plain_maps(s["parents"], s["lens"], s["starts"], s["commits"], nodes)
        return dict(zip(("offsets", "lens", "commits", "pos", "masks"), maps))
    if own:
        trees = _kernels().DraftTrees(*s["trees"], max_nodes=nodes)
    if op == "conv":
        if own:
            out = _kernels().tree_conv_silu(s["x"], s["pool"], s["weight"], s["slots"], trees)
        else:
            out = _plain_conv(s["x"], s["pool"], s["weight"], s["slots"], s["trees"], nodes)
        return {"out": out, "pool": s["pool"]} if case["commits"] else out
    if op == "gdn":
        hv = case["value_heads"]
        if own:
            out = _kernels().gdn_tree_step(s["packed"], H * KD, H, KD, hv, KD, s["a"], s["b"], s["A_log"], s["dt_bias"],
                                           s["state"], s["slots"], trees, z=s["z"], norm_weight=s["norm"], eps=EPS)
        else:
            out = _plain_gdn(s, hv, nodes)
        return {"out": out, "state": s["state"]} if case["commits"] else out
    if own:
        out = _kernels().tree_ring_attention(s["q"], s["ring_k"], s["ring_v"], s["new_k"], s["value"], s["gate"],
                                             s["ring_pos"], s["slots"], s["starts"], trees, HD ** -0.5, W)
    else:
        out = _plain_attention(s, nodes)
    return {"out": out, "ring_k": s["ring_k"], "ring_v": s["ring_v"]} if case["commits"] else out


def _plain_maps(parents, lens, starts, commits, nodes):
    """(offsets, lens, commits, pos, masks): bit j of a node's mask is set for j itself and its ancestors. A row that is no
    tree (a parent that does not come first, more than ``nodes`` of them, commits that are no chain) has no nodes."""
    total, index = parents.numel(), torch.arange(nodes, device=parents.device)
    size = lens.clamp(0, total + 1)
    offsets = torch.cumsum(size, 0) - size
    done = torch.zeros_like(lens) if commits is None else commits
    inside = index < size[:, None]
    at = (offsets[:, None] + index).clamp(max=total - 1)
    p = torch.where(inside, parents[at], index - 1)
    good = (p >= -1) & (p < index) & ((p == index - 1) | (index >= done[:, None]))
    good = good.all(1) & (lens >= 0) & (size <= nodes) & (offsets + size <= total) & (starts >= 0)
    good = good & (done >= 0) & (done <= size)
    # ancestors: the transitive closure of "is or has as parent", by doubling
    reach = ((index == p[:, :, None]) | (index == index[:, None])).float()
    for _ in range(6):
        reach = (torch.matmul(reach, reach) > 0).float()
    reach = reach > 0
    live = inside & good[:, None]
    where = at[live]
    pos = torch.zeros_like(parents)
    masks = torch.zeros_like(parents)
    pos[where] = (starts[:, None] + reach.sum(-1) - 1)[live]
    masks[where] = torch.where(reach, torch.ones_like(p)[..., None] << index, 0).sum(-1)[live]
    return offsets, torch.where(good, size, 0), None if commits is None else torch.where(good, done, 0), pos, masks


def _padded(trees, nodes):
    """Of the rows padded to ``nodes``: which places hold a node, its token, and its ancestors and itself [n, nodes, nodes]."""
    offsets, lens, _, _, masks = trees
    index = torch.arange(nodes, device=DEV)
    live = index < lens[:, None]
    at = torch.where(live, offsets[:, None] + index, 0)
    own_bits = (masks[at][..., None] >> index) & 1
    return live, at, (own_bits > 0) & live[:, :, None]


def _silu(x):
    return x / (1 + torch.exp(-x))


def _plain_conv(x, pool, weight, slots, trees, nodes):
    live, at, reach = _padded(trees, nodes)
    n, c = live.shape[0], x.shape[1]
    depth = reach.sum(-1) - 1
    # how many ancestors (or itself) come at or after column j: the nearest is 1
    nth = reach.flip(-1).long().cumsum(-1).flip(-1) * reach
    history = pool[slots].float()
    w = weight.reshape(c, TAPS).float()
    xf = x.float()
    acc = torch.zeros(n, nodes, c, dtype=F32, device=DEV)
    rows = torch.arange(n, device=DEV)[:, None]
    for t in range(TAPS):
        found = depth >= t
        near = (nth == t + 1).long().argmax(-1)
        value = torch.where(found[..., None], xf[torch.gather(at, 1, near)],
                            history[rows, (TAPS - 1 + depth - t).clamp(0, TAPS - 2)])
        acc = acc + value * w[:, TAPS - 1 - t]
    out = torch.zeros_like(x)
    out[at[live]] = _silu(acc[live]).to(BF16)
    done = trees[2]
    if done is None:
        return out
    # the committed chain moves the history: the last three values of (history, chain)
    ext = done[:, None] + torch.arange(TAPS - 1, device=DEV)
    kept = torch.gather(at, 1, (ext - TAPS + 1).clamp(0, nodes - 1))
    moved = torch.where((ext < TAPS - 1)[..., None], pool[slots][rows, ext.clamp(max=TAPS - 2)], x[kept])
    pool[slots] = torch.where((done > 0)[:, None, None], moved, pool[slots])
    return out


def _unit(x):
    return x * (x.square().sum(-1, keepdim=True) + EPS).rsqrt()


def _plain_gdn(s, hv, nodes):
    """The rule along a path, S <- e^g S + k u^T with u = beta (v - e^g S^T k), unrolled over the node's ancestors:
    u_i = beta_i (v_i - e^(G_i) S0^T k_i - sum over ancestors j of e^(G_i - G_j) (k_i . k_j) u_j),
    o_i = e^(G_i) S0^T q_i + sum over ancestors and itself of e^(G_i - G_j) (q_i . k_j) u_j, G the decays' sum down to i."""
    trees, state, slots = s["trees"], s["state"], s["slots"]
    live, at, reach = _padded(trees, nodes)
    n, per = live.shape[0], hv // H
    x = s["packed"].float()[at]                                             # [n, nodes, channels]

    def heads(y, repeat):
        return y.reshape(n, nodes, -1, KD).repeat_interleave(repeat, 2).transpose(1, 2).contiguous()

    q = _unit(heads(x[..., :H * KD], per)) * KD ** -0.5
    k = _unit(heads(x[..., H * KD:2 * H * KD], per)) * live[:, None, :, None]
    v = heads(x[..., 2 * H * KD:], 1)
    t = s["a"].float()[at] + s["dt_bias"].float()
    g = -torch.exp(s["A_log"].float()) * torch.where(t > 20, t, torch.log1p(torch.exp(t.clamp(max=20.0))))
    beta = (1 / (1 + torch.exp(-s["b"].float()[at]))).transpose(1, 2) * live[:, None]        # [n, hv, nodes]
    down = torch.matmul(reach.float(), g).transpose(1, 2)                   # [n, hv, nodes]: G
    near = reach[:, None]
    decay = torch.exp(torch.where(near, down[..., :, None] - down[..., None, :], 0.0)) * near
    s0 = state[slots].float()
    kt = k.transpose(-1, -2).contiguous()
    strict = ~torch.eye(nodes, dtype=torch.bool, device=DEV)
    mix = beta[..., None] * torch.matmul(k, kt) * decay * strict            # A, nilpotent: (I + A)^-1 = prod (I + (-A)^2^i)
    u = beta[..., None] * (v - torch.exp(down)[..., None] * torch.matmul(k, s0))
    u = u - torch.matmul(mix, u)
    for _ in range(5):
        mix = torch.matmul(mix, mix)
        u = u + torch.matmul(mix, u)
    o = torch.exp(down)[..., None] * torch.matmul(q, s0) + torch.matmul(torch.matmul(q, kt) * decay, u)
    y = o * (o.square().mean(-1, keepdim=True) + EPS).rsqrt() * s["norm"].float()
    y = y.transpose(1, 2).reshape(n, nodes, hv * KD) * _silu(s["z"].float()[at])
    out = torch.zeros(s["z"].shape, dtype=BF16, device=DEV)
    out[at[live]] = y[live].to(BF16)
    done = trees[2]
    if done is None:
        return out
    last = torch.gather(down, 2, (done - 1).clamp(min=0)[:, None, None].expand(n, hv, 1))
    chain = torch.arange(nodes, device=DEV) < done[:, None]
    left = torch.exp(torch.where(chain[:, None], last - down, 0.0)) * chain[:, None]
    s1 = torch.exp(last)[..., None] * s0 + torch.matmul((k * left[..., None]).transpose(-1, -2).contiguous(), u)
    state[slots] = torch.where((done > 0)[:, None, None, None], s1, s0).to(state.dtype)
    return out


def _plain_attention(s, nodes):
    trees, slots, starts = s["trees"], s["slots"], s["starts"]
    live, at, reach = _padded(trees, nodes)
    n = live.shape[0]
    hq, hkv = s["q"].shape[1], s["new_k"].shape[1]
    per = hq // hkv
    qpos = starts[:, None] + reach.sum(-1) - 1
    kpos = s["ring_pos"][slots][:, None, :W]
    ring = (kpos >= 0) & (kpos < starts[:, None, None]) & (kpos > qpos[..., None] - W)
    tree = reach & (qpos[:, None] > qpos[..., None] - W)
    seen = (torch.cat([ring, tree], -1) & live[..., None])[:, None, None]    # [n, 1, 1, nodes, W + nodes]

    def keys(ring_x, new_x):
        return torch.cat([ring_x[slots][:, :, :W].float(), new_x.float()[at].transpose(1, 2)], 2)

    q = s["q"].float()[at].reshape(n, nodes, hkv, per, HD).permute(0, 2, 3, 1, 4).reshape(n, hkv, per * nodes, HD)
    scores = torch.matmul(q, keys(s["ring_k"], s["new_k"]).transpose(-1, -2).contiguous()) * HD ** -0.5
    scores = scores.reshape(n, hkv, per, nodes, W + nodes)
    top = torch.where(seen, scores, -math.inf).amax(-1, keepdim=True)
    p = torch.exp(torch.where(seen, scores - top, -math.inf))
    o = torch.matmul(p.reshape(n, hkv, per * nodes, W + nodes), keys(s["ring_v"], s["value"]))
    o = o.reshape(n, hkv, per, nodes, HD) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, nodes, hq, HD)
    gate = s["gate"].float()[at].reshape(n, nodes, hq, 2, HD)[:, :, :, 1]
    out = torch.zeros(s["q"].shape[0], hq * HD, dtype=BF16, device=DEV)
    out[at[live]] = (o / (1 + torch.exp(-gate))).reshape(n, nodes, hq * HD)[live].to(BF16)
    if trees[2] is None:
        return out
    chain = torch.arange(nodes, device=DEV) < trees[2][:, None]
    row, node = torch.nonzero(chain, as_tuple=True)
    column = (starts[row] + node) % W
    s["ring_k"][slots[row], :, column] = s["new_k"][at[row, node]]
    s["ring_v"][slots[row], :, column] = s["value"][at[row, node]]
    return out


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    rows = _rows(case, 0)
    lens = [len(p) for p, _ in rows]
    n, total, op = case["rows"], sum(lens), case["op"]
    committed = sum(c > 0 for _, c in rows)
    depths = []
    for parents, _ in rows:
        d = []
        for p in parents:
            d.append(1 + (d[p] if p >= 0 else 0))
        depths.append(d)
    pairs = sum(map(sum, depths))           # (node, ancestor or itself)
    if op == "maps":
        return {"bytes": 8 * (3 * total + n * (5 + case["commits"])), "flops": pairs}
    index = 16 * n + 8 * total + 8 * n * case["commits"]       # offsets and lengths, masks, commits
    if op == "conv":
        c = (2 * H + case["value_heads"]) * KD
        return {"bytes": index + 8 * n + 2 * c * (2 * total + (TAPS - 1) * (n + committed) + TAPS),
                "flops": total * c * (2 * TAPS + 4)}
    if op == "gdn":
        hv, size = case["value_heads"], 4 if case["state"] == "float32" else 2
        return {"bytes": index + 8 * n + (n + committed) * hv * KD * KD * size
                + 2 * total * ((2 * H + hv) * KD + 2 * hv + 2 * hv * KD),
                "flops": hv * (total * 4 * KD * KD + pairs * 8 * KD + sum(c for _, c in rows) * 2 * KD * KD)}
    hq, hkv = case["q_heads"], case["q_heads"] // 4
    in_ring = n * W * 7 // 8                # one session in four has half a window on average
    return {"bytes": index + 16 * n + n * W * 8 + 2 * hkv * HD * 2 * (in_ring + total + sum(c for _, c in rows))
            + 2 * total * 3 * hq * HD,
            "flops": 4 * hq * HD * (total * W * 7 // 8 + pairs)}


# ---------------------------------------------------------------------------------------------------------------
# The same in 64 bits, by walking the trees
# ---------------------------------------------------------------------------------------------------------------
def _walk(case, seed, s):
    """Per node index i, in which every parent comes first: (i, the rows that have node i, their tokens, their parents)."""
    rows = _rows(case, seed)
    offsets = [0]
    for parents, _ in rows:
        offsets.append(offsets[-1] + len(parents))
    for i in range(case["nodes"]):
        have = [r for r, (parents, _) in enumerate(rows) if i < len(parents)]
        yield (i, _ints(have), _ints([offsets[r] + i for r in have]), _ints([rows[r][0][i] for r in have]),
               _ints([j for j, r in enumerate(have) if rows[r][1] == i + 1]))


@torch.no_grad()
def exact(case, seed):
    if case["op"] == "maps":
        return None
    s = prepare(case, seed)
    n, nodes, slots = case["rows"], case["nodes"], s["slots"]
    if case["op"] == "conv":
        x, pool, w = s["x"].double(), s["pool"].double(), s["weight"].double()[:, 0]
        out = torch.zeros_like(x)
        # the last three inputs on the way to each node; slot 0: before the first
        last = torch.zeros(nodes + 1, n, TAPS - 1, x.shape[1], dtype=F64, device=DEV)
        last[0] = pool[slots]
        for i, have, tokens, parent, ends in _walk(case, seed, s):
            span = torch.cat([last[parent + 1, have], x[tokens][:, None]], 1)
            acc = (span * w.T).sum(1)
            out[tokens] = acc * torch.sigmoid(acc)
            last[i + 1, have] = span[:, 1:]
            pool[slots[have[ends]]] = span[ends, 1:]
        return {"out": out, "pool": pool} if case["commits"] else out
    if case["op"] == "gdn":
        hv = case["value_heads"]
        per = hv // H
        x = s["packed"].double()
        q, k, v = (y.reshape(len(x), -1, KD) for y in x.split([H * KD, H * KD, hv * KD], -1))
        q = (q / (q.square().sum(-1, keepdim=True) + EPS).sqrt() * KD ** -0.5).repeat_interleave(per, 1)
        k = (k / (k.square().sum(-1, keepdim=True) + EPS).sqrt()).repeat_interleave(per, 1)
        fade = torch.exp(-s["A_log"].double().exp() * torch.nn.functional.softplus(s["a"].double() + s["dt_bias"].double()))
        beta = torch.sigmoid(s["b"].double())
        state = s["state"].double()
        at = torch.empty(nodes + 1, n, hv, KD, KD, dtype=F64, device=DEV)
        at[0] = state[slots]
        o = torch.zeros(len(x), hv, KD, dtype=F64, device=DEV)
        for i, have, tokens, parent, ends in _walk(case, seed, s):
            now = at[parent + 1, have] * fade[tokens][..., None, None]
            read = (now * k[tokens][..., None]).sum(-2)
            now += k[tokens][..., None] * (beta[tokens][..., None] * (v[tokens] - read))[..., None, :]
            o[tokens] = (now * q[tokens][..., None]).sum(-2)
            at[i + 1, have] = now
            state[slots[have[ends]]] = now[ends]
        y = o / (o.square().mean(-1, keepdim=True) + EPS).sqrt() * s["norm"].double()
        z = s["z"].double().reshape(y.shape)
        out = (y * z * torch.sigmoid(z)).reshape(len(x), -1)
        return {"out": out, "state": state} if case["commits"] else out
    hq, hkv = case["q_heads"], case["q_heads"] // 4
    per = hq // hkv
    ring_k, ring_v = s["ring_k"].double(), s["ring_v"].double()
    old_k, old_v, old_pos = ring_k[slots][:, :, :W], ring_v[slots][:, :, :W], s["ring_pos"][slots][:, :W]
    out = torch.zeros(len(s["q"]), hq, HD, dtype=F64, device=DEV)
    # a node's path as token numbers, itself last; -1: none
    path = torch.full((nodes + 1, n, nodes), -1, dtype=I64, device=DEV)
    depth = torch.zeros(nodes + 1, n, dtype=I64, device=DEV)
    for i, have, tokens, parent, _ in _walk(case, seed, s):
        mine = path[parent + 1, have]
        d = depth[parent + 1, have]
        mine[torch.arange(len(have), device=DEV), d] = tokens
        path[i + 1, have], depth[i + 1, have] = mine, d + 1
        m = int(d.max()) + 1
        mine, pos = mine[:, :m], s["starts"][have] + d
        steps = s["starts"][have][:, None] + torch.arange(m, device=DEV)
        kpos = torch.cat([old_pos[have], torch.where(mine >= 0, steps, -1)], 1)
        seen = (kpos >= 0) & (kpos > pos[:, None] - W)
        q = s["q"][tokens].double().reshape(len(have), hkv, per, HD)
        keys = torch.cat([old_k[have], s["new_k"][mine.clamp(min=0)].double().transpose(1, 2)], 2)
        values = torch.cat([old_v[have], s["value"][mine.clamp(min=0)].double().transpose(1, 2)], 2)
        score = torch.matmul(q, keys.transpose(-1, -2).contiguous()) * HD ** -0.5
        p = torch.softmax(score.masked_fill(~seen[:, None, None], -math.inf), -1)
        out[tokens] = torch.matmul(p, values).reshape(len(have), hq, HD)
    out = out * torch.sigmoid(s["gate"].double().reshape(len(out), hq, 2, HD)[:, :, 1])
    for i, have, tokens, _, _ in _walk(case, seed, s) if case["commits"] else ():
        some = torch.nonzero(s["commits"][have] > i).flatten()
        column = (s["starts"][have[some]] + i) % W
        ring_k[slots[have[some]], :, column] = s["new_k"][tokens[some]].double()
        ring_v[slots[have[some]], :, column] = s["value"][tokens[some]].double()
    out = out.reshape(len(out), -1)
    return {"out": out, "ring_k": ring_k, "ring_v": ring_v} if case["commits"] else out
