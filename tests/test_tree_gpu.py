"""Drafted-tree operators on the GPU against the float64 oracle (oracle/tree.py), which walks the trees node by node.

Tolerances. Every output is rounded once: half a step of its type (bf16 2^-8, fp16 2^-11 of the value). Before that
  conv       4 products and a SiLU (slope at most 1.1, its own error 2^-21): 2^-20 of the sum of the products' magnitudes;
  gdn        a state column's 128 products in three parts, at most 64 terms of the solve and 64 of the outputs, 512 roundings
             of 2^-24: 2^-15 of the oracle's majorant (the same sums over magnitudes);
  attention  probabilities rounded to bf16: 2^-8 of sum p |v|; scores of 256 products, off by at most 2^-16 of |q| . |k|
             scale, which moves each probability and the normaliser by as much: 2^-15 of that times sum p |v|; the fp32 sums
             of at most 576 terms 2^-14.
"""
import numpy as np
import pytest
import torch

from oracle import tree
from oracle.bf16 import sigmoid

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
KD, D = 128, 256


def _f64(t):
    return t.double().cpu().numpy()


def within(got, want, slack, step, what):
    """|got - want| <= step |want| + slack (and the least normal number of the type, below which steps do not shrink)."""
    got, want = _f64(got) if torch.is_tensor(got) else got, np.asarray(want)
    off = np.abs(got - want) - (step * (np.abs(want) + slack) + slack + 2.0 ** -120)
    assert np.isfinite(got).all(), f"{what}: not finite"
    assert (off <= 0).all(), f"{what}: {(off > 0).sum()} of {off.size} values beyond the bar, by up to {off.max():.3g}"


def random_tree(rng, n, style):
    if style == "chain":
        return list(range(-1, n - 1))
    if style == "star":
        return [-1] * n
    return [int(rng.integers(max(-1, i - 5) if style == "beam" else -1, i)) for i in range(n)]


def batch(seed, lens, commit=True, tail=0, slots=None, pool=None):
    """Rows of random trees: (rows for the oracle, device tensors). Slots in random order out of ``pool``."""
    rng = np.random.default_rng(seed)
    rows, parents, at = [], [], 0
    for n in lens:
        p = random_tree(rng, n, rng.choice(["chain", "beam", "any", "star"]))
        done = int(rng.integers(0, n + 1)) if commit and n else 0
        p[:done] = range(-1, done - 1)
        rows.append((at, p, done))
        parents += p
        at += n
    n = len(lens)
    pool = pool or n + 2
    slots = rng.permutation(pool)[:n].tolist() if slots is None else slots
    starts = [int(rng.choice([0, 1, rng.integers(1, 700), rng.integers(512, 9000)])) for _ in lens]
    dev = {"parents": torch.tensor(parents + [-1] * tail, dtype=torch.long, device="cuda"),
           "lens": torch.tensor(lens, dtype=torch.long, device="cuda"),
           "starts": torch.tensor(starts, dtype=torch.long, device="cuda"),
           "commits": torch.tensor([r[2] for r in rows], dtype=torch.long, device="cuda") if commit else None,
           "slots": torch.tensor(slots, dtype=torch.long, device="cuda")}
    return rows, slots, starts, pool, dev


def maps_of(dev, max_nodes=64):
    from hs_guard.engine.kernels import draft_tree_maps
    return draft_tree_maps(dev["parents"], dev["lens"], dev["starts"], dev["commits"], max_nodes)


def randn(seed, *shape, scale=1.0, dtype=BF16):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()


def signed(masks):
    return [m - (1 << 64) if m >> 63 else m for m in masks]


LENS = [[1], [64], [0, 0], [1, 1, 1], [12, 0, 33, 1, 16, 17, 64], [8] * 9, [15, 16, 17, 31, 32, 33]]


# ---------------------------------------------------------------------------------------------------------------
# maps
# ---------------------------------------------------------------------------------------------------------------
def check_maps(trees, want):
    for name, got, ref in zip(("offsets", "lens", "commits", "pos", "masks"), trees[:5], want):
        if got is not None:
            assert got.tolist() == (signed(ref) if name == "masks" else ref), name


@pytest.mark.parametrize("lens", LENS + [[3] * 700, [64] * 70, []])
@pytest.mark.parametrize("commit,tail", [(True, 0), (False, 5), (True, 300)])
def test_maps(lens, commit, tail):
    rows, _, starts, _, dev = batch(len(lens) + tail, lens, commit, tail)
    want = tree.tree_maps(dev["parents"].tolist(), lens, starts, [r[2] for r in rows] if commit else None, 64)
    trees = maps_of(dev)
    check_maps(trees, want)
    assert (trees.commits is None) != commit


def test_maps_reject_rows_that_are_no_trees():
    """Bad rows among good ones: they come back empty, their neighbours whole."""
    cases = [([-1, 0, 1], 0), ([0], 0), ([-1, 2, 0], 0), ([-1, 0, 0], 2), ([-1, -2], 0), ([-1, 0, 0], 3), ([-1, 0], -1),
             ([-1, 0], 4), (list(range(-1, 69)), 0), ([-1 << 40, 0], 0), ([1 << 40], 0), ([-1, 0, 1, 2], 4)]
    parents = [p for row, _ in cases for p in row]
    lens = [len(row) for row, _ in cases]
    commits = [c for _, c in cases]
    for lens2, most in ((lens, 64), (lens + [-3, 9, 1 << 62, -(1 << 62)], 64), (lens, 2)):
        done = commits + [0] * (len(lens2) - len(lens))
        starts = list(range(len(lens2)))
        starts[0] = -1 if most == 2 else 7
        dev = {k: torch.tensor(v, dtype=torch.long, device="cuda") for k, v in
               (("parents", parents), ("lens", lens2), ("starts", starts), ("commits", done))}
        check_maps(maps_of(dev, most), tree.tree_maps(parents, lens2, starts, done, most))


# ---------------------------------------------------------------------------------------------------------------
# conv
# ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("channels,commit,gap", [(8, True, 0), (1000, True, 24), (2056, False, 0)])
def test_conv(lens, channels, commit, gap):
    from hs_guard.engine.kernels import tree_conv_silu
    rows, slots, _, pool_rows, dev = batch(len(lens) + channels, lens, commit, 3)
    total = dev["parents"].numel()
    wide = randn(1, total, channels + gap)
    x = wide[:, :channels]
    pool, w = randn(2, pool_rows, 3, channels), randn(3, channels, 1, 4, scale=0.5)
    want, size, pool2 = tree.tree_conv_silu(_f64(x), _f64(pool), _f64(w), slots, rows)
    for most in sorted({max(max(lens), 1), 64}):
        got_pool = pool.clone()
        out = tree_conv_silu(x, got_pool, w, dev["slots"], maps_of(dev, most))
        live = sum(lens)
        within(out[:live], want[:live], 2.0 ** -20 * size[:live], 2.0 ** -8, "out")
        np.testing.assert_array_equal(_f64(got_pool), pool2)


@pytest.mark.parametrize("most", [1, 7, 16, 29, 32, 64])
@pytest.mark.parametrize("rows_n,channels", [(33, 520), (90, 1032)])
def test_conv_over_many_rows(most, rows_n, channels):
    """The tiles that calls of many rows take, by the bound on a row's nodes; in place, bitwise the same."""
    from hs_guard._lib import calls
    from hs_guard.engine.kernels import tree_conv_silu
    lens = np.random.default_rng(most + rows_n).integers(0, most + 1, rows_n).tolist()
    lens[5] = most
    rows, slots, _, pool_rows, dev = batch(rows_n + most, lens, True, 2)
    x, w = randn(1, dev["parents"].numel(), channels), randn(3, channels, 1, 4, scale=0.5)
    pool = randn(2, pool_rows, 3, channels)
    want, size, pool2 = tree.tree_conv_silu(_f64(x), _f64(pool), _f64(w), slots, rows)
    t, live, got_pool, same_pool = maps_of(dev, most), sum(lens), pool.clone(), pool.clone()
    out = tree_conv_silu(x, got_pool, w, dev["slots"], t)
    within(out[:live], want[:live], 2.0 ** -20 * size[:live], 2.0 ** -8, "out")
    np.testing.assert_array_equal(_f64(got_pool), pool2)
    assert calls().hsg_tree_conv_silu(x.data_ptr(), channels, same_pool.data_ptr(), pool_rows, w.data_ptr(), 4,
                                      dev["slots"].data_ptr(), t.lens.data_ptr(), t.offsets.data_ptr(),
                                      t.commits.data_ptr(), t.masks.data_ptr(), rows_n, most, channels, x.data_ptr(),
                                      channels, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(x[:live], out[:live]) and torch.equal(same_pool, got_pool)


def test_conv_leaves_the_rest_alone_and_runs_in_place():
    """Rows of an unknown slot and tokens of no row keep their outputs; out may be the input."""
    from hs_guard._lib import calls
    C, lens = 264, [5, 7, 4]
    rows, slots, _, pool_rows, dev = batch(3, lens, True, 4)
    dev["slots"][1] = pool_rows + 5
    x, pool, w = randn(1, 20, C), randn(2, pool_rows, 3, C), randn(3, C, 1, 4)
    t = maps_of(dev)
    live = [i for r in (0, 2) for i in range(rows[r][0], rows[r][0] + lens[r])]
    want, size, pool2 = tree.tree_conv_silu(_f64(x), _f64(pool), _f64(w), [slots[0], slots[2]], [rows[0], rows[2]])
    apart = torch.full_like(x, 7.0)
    for out in (apart, x):
        p2 = pool.clone()
        before = out.clone()
        assert calls().hsg_tree_conv_silu(x.data_ptr(), C, p2.data_ptr(), pool_rows, w.data_ptr(), 4,
                                          dev["slots"].data_ptr(), t.lens.data_ptr(), t.offsets.data_ptr(),
                                          t.commits.data_ptr(), t.masks.data_ptr(), 3, 64, C, out.data_ptr(), C,
                                          torch.cuda.current_stream().cuda_stream) == 0
        rest = [i for i in range(20) if i not in live]
        assert torch.equal(out[rest], before[rest])
        within(out[live], want[live], 2.0 ** -20 * size[live], 2.0 ** -8, "out")
        np.testing.assert_array_equal(_f64(p2), pool2)


# ---------------------------------------------------------------------------------------------------------------
# gdn
# ---------------------------------------------------------------------------------------------------------------
def gdn_inputs(seed, total, pool_rows, H, HV, state_dtype, a_scale=1.0):
    packed = torch.nn.functional.silu(randn(seed, total, (2 * H + HV) * KD, dtype=torch.float32)).to(BF16)
    gen = torch.Generator().manual_seed(seed + 9)
    dt = torch.exp(torch.rand(HV, generator=gen) * 4.6 - 6.9)
    return {"packed": packed, "a": randn(seed + 1, total, HV, scale=a_scale), "b": randn(seed + 2, total, HV),
            "A_log": torch.log(torch.rand(HV, generator=gen) * 15 + 1).to(BF16).cuda(),
            "dt_bias": torch.log(torch.expm1(dt)).to(BF16).cuda(),
            "state": randn(seed + 3, pool_rows, HV, KD, KD, scale=0.3, dtype=state_dtype),
            "z": randn(seed + 4, total, HV * KD), "norm_weight": (1 + randn(seed + 5, KD, scale=0.2).float()).to(BF16)}


def gdn_oracle(s, H, HV, slots, rows):
    return tree.gdn_tree_step(_f64(s["packed"]), H, HV, _f64(s["a"]), _f64(s["b"]), _f64(s["A_log"]), _f64(s["dt_bias"]),
                              _f64(s["state"]), slots, rows)


def gdn_call(s, H, HV, slots, trees, state, gate=True):
    from hs_guard.engine.kernels import gdn_tree_step
    more = {"z": s["z"], "norm_weight": s["norm_weight"], "eps": 1e-6} if gate else {}
    return gdn_tree_step(s["packed"], H * KD, H, KD, HV, KD, s["a"], s["b"], s["A_log"], s["dt_bias"], state, slots, trees,
                         **more)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("H,HV,dtype,commit", [(2, 2, torch.float32, True), (1, 3, torch.float16, True),
                                                (2, 4, torch.float32, False)])
def test_gdn(lens, H, HV, dtype, commit):
    rows, slots, _, pool_rows, dev = batch(7 * len(lens) + HV, lens, commit, 2)
    s = gdn_inputs(len(lens), dev["parents"].numel(), pool_rows, H, HV, dtype)
    o, osize, st, ssize = gdn_oracle(s, H, HV, slots, rows)
    y, ysize = tree.gated(o, osize, _f64(s["z"]).reshape(o.shape), _f64(s["norm_weight"]), 1e-6)
    live = sum(lens)
    step = 0.0 if dtype is torch.float32 else 2.0 ** -11
    for most in sorted({max(max(lens), 1), 64}):
        trees = maps_of(dev, most)
        for gate, ref, size in ((False, o, osize), (True, y, ysize)):
            state = s["state"].clone()
            out = gdn_call(s, H, HV, dev["slots"], trees, state, gate).reshape(o.shape)
            within(out[:live], ref[:live], 2.0 ** -15 * size[:live], 2.0 ** -8, f"out, gate {gate}, bound {most}")
            within(state, st, 2.0 ** -15 * ssize, step, "state")
            idle = [x for x in range(pool_rows) if x not in [a for a, r in zip(slots, rows) if r[2]]]
            assert torch.equal(state[idle], s["state"][idle])


def test_gdn_takes_columns_of_a_projection_and_steep_decays():
    """a, b and z inside one wider projection, as the layer's GEMM leaves them; decays of up to e^-600 a node, after which
    the nodes below must keep all their digits."""
    H = HV = 2
    rows, slots, _, pool_rows, dev = batch(5, [40, 9], True)
    total = 49
    s = gdn_inputs(3, total, pool_rows, H, HV, torch.float32)
    s["a"][3::11] = 40.0
    width = HV * KD + 2 * HV + 12
    proj = randn(11, total, width)
    for name, at, n in (("z", 0, HV * KD), ("b", HV * KD, HV), ("a", HV * KD + HV, HV)):
        proj[:, at:at + n] = s[name]
        s[name] = proj[:, at:at + n]
    o, osize, st, ssize = gdn_oracle(s, H, HV, slots, rows)
    y, ysize = tree.gated(o, osize, _f64(s["z"]).reshape(o.shape), _f64(s["norm_weight"]), 1e-6)
    state = s["state"].clone()
    out = gdn_call(s, H, HV, dev["slots"], maps_of(dev), state).reshape(o.shape)
    within(out, y, 2.0 ** -15 * ysize, 2.0 ** -8, "out")
    within(state, st, 2.0 ** -15 * ssize, 0.0, "state")


@pytest.mark.parametrize("what", ["k", "v", "q", "a", "b", "inf v", "inf a"])
@pytest.mark.parametrize("n", [9, 30, 64])
def test_gdn_keeps_a_bad_node_to_its_branch(what, n):
    """Two branches below a committed root; one node of the first is not finite. The other branch, and the state, do not
    see it."""
    H = HV = 2
    half = n // 2
    parents = [-1] + list(range(0, half - 1)) + [0] + list(range(half, n - 1))
    bad = half // 2 + 1
    dev = {"parents": torch.tensor(parents, device="cuda"), "lens": torch.tensor([n], device="cuda"),
           "starts": torch.tensor([5], device="cuda"), "commits": torch.tensor([1], device="cuda"),
           "slots": torch.tensor([1], device="cuda")}
    s = gdn_inputs(n, n, 3, H, HV, torch.float32)
    rows = [(0, parents, 1)]
    o, osize, st, ssize = gdn_oracle(s, H, HV, [1], rows)
    value = float("inf") if what.startswith("inf") else float("nan")
    name = what[-1]
    if name in "qkv":
        s["packed"][bad, {"q": 0, "k": H * KD, "v": 2 * H * KD}[name] + 3] = value
    else:
        s[name][bad, 0] = value
    below = [i for i in range(n) if bad in tree.path(parents, i)]
    if what == "inf a":     # the state decays to nothing there: all stays finite
        o, osize, st, ssize = gdn_oracle(s, H, HV, [1], rows)
        below = []
    rest = [i for i in range(n) if i not in below]
    y, ysize = tree.gated(o, osize, _f64(s["z"]).reshape(o.shape), _f64(s["norm_weight"]), 1e-6)
    for gate, ref, size in ((False, o, osize), (True, y, ysize)):
        state = s["state"].clone()
        out = gdn_call(s, H, HV, dev["slots"], maps_of(dev, n), state, gate).reshape(o.shape)
        within(out[rest], ref[rest], 2.0 ** -15 * size[rest], 2.0 ** -8, f"the other nodes, gate {gate}")
        within(state, st, 2.0 ** -15 * ssize, 0.0, "state")
        if below:
            seen = [bad] if name == "q" else below
            assert not torch.isfinite(out[seen, 0]).all(-1).any()
    # committed, it reaches the state of its head alone
    if name in "kv" and what != "inf v":
        dev["commits"][0] = half
        state = s["state"].clone()
        gdn_call(s, H, HV, dev["slots"], maps_of(dev, n), state)
        assert not torch.isfinite(state[1, 0]).all() and torch.isfinite(state[1, 1]).all()
        assert torch.equal(state[[0, 2]], s["state"][[0, 2]])


@pytest.mark.parametrize("n", [12, 24, 40])
def test_gdn_recomputed_rows_of_an_fp16_state(n):
    """One value of the last node of one row of three is not finite: all else, and every state, as without it."""
    H, HV = 1, 2
    parents = [-1, 0] + [0] * (n - 2)
    rows, slots, _, pool_rows, dev = batch(6, [n] * 3, True)
    rows = [(r * n, parents, 2) for r in range(3)]
    dev["parents"] = torch.tensor(parents * 3, device="cuda")
    dev["commits"] = torch.tensor([2] * 3, device="cuda")
    s = gdn_inputs(n, 3 * n, pool_rows, H, HV, torch.float16)
    o, osize, st, ssize = gdn_oracle(s, H, HV, slots, rows)
    y, ysize = tree.gated(o, osize, _f64(s["z"]).reshape(o.shape), _f64(s["norm_weight"]), 1e-6)
    s["packed"][2 * n - 1, 2 * H * KD + 7] = float("nan")
    state = s["state"].clone()
    out = gdn_call(s, H, HV, dev["slots"], maps_of(dev, n), state).reshape(o.shape)
    rest = [i for i in range(3 * n) if i != 2 * n - 1]
    within(out[rest], y[rest], 2.0 ** -15 * ysize[rest], 2.0 ** -8, "the other nodes")
    within(state, st, 2.0 ** -15 * ssize, 2.0 ** -11, "state")
    assert not torch.isfinite(out[2 * n - 1, 0]).any() and torch.isfinite(out[2 * n - 1, 1]).all()


# ---------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------
def ring_positions(slots, starts, pool_rows, W, fills=None):
    pos = torch.full((pool_rows, W + 1), -1, dtype=torch.long)
    for i, (s, start) in enumerate(zip(slots, starts)):
        for p in range(max(0, start - (W if fills is None else fills[i])), start):
            pos[s, p % W] = p
    return pos.cuda()


def attention_inputs(seed, total, pool_rows, slots, starts, hkv, G, W, scale=1.0):
    return {"q": randn(seed, total, hkv * G, D, scale=scale), "new_k": randn(seed + 1, total, hkv, D),
            "value": randn(seed + 2, total, hkv, D), "gate": randn(seed + 3, total, hkv * G * 2 * D),
            "ring_k": randn(seed + 4, pool_rows, hkv, W + 1, D), "ring_v": randn(seed + 5, pool_rows, hkv, W + 1, D),
            "ring_pos": ring_positions(slots, starts, pool_rows, W)}


def attention_oracle(s, slots, starts, rows, W, scale):
    o, size, reach, rk, rv = tree.tree_attention(*(_f64(s[k]) for k in ("q", "ring_k", "ring_v", "new_k", "value")),
                                                 s["ring_pos"].cpu().numpy(), slots, starts, rows, scale, W)
    slack = size * (2.0 ** -8 + 2.0 ** -14 + 2.0 ** -15 * reach[..., None])
    if s["gate"] is not None:
        g = sigmoid(_f64(s["gate"]).reshape(*o.shape[:2], 2, D)[:, :, 1])
        o, slack = o * g, slack * g
    return o.reshape(len(o), -1), slack.reshape(len(o), -1), rk, rv


def attention_call(s, dev, trees, W, scale, rings=None, **kw):
    from hs_guard.engine.kernels import tree_ring_attention
    rk, rv = rings or (s["ring_k"], s["ring_v"])
    return tree_ring_attention(s["q"], rk, rv, s["new_k"], s["value"], s["gate"], s["ring_pos"], dev["slots"],
                               dev["starts"], trees, scale, W, **kw)


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("hkv,G,W,commit,gated", [(2, 4, 512, True, True), (1, 1, 64, True, False), (1, 3, 32, True, True),
                                                   (1, 16, 512, False, True)])
def test_attention(lens, hkv, G, W, commit, gated):
    rows, slots, starts, pool_rows, dev = batch(11 * len(lens) + G, lens, commit, 2)
    s = attention_inputs(len(lens), dev["parents"].numel(), pool_rows, slots, starts, hkv, G, W)
    if not gated:
        s["gate"] = None
    scale = D ** -0.5
    want, slack, rk, rv = attention_oracle(s, slots, starts, rows, W, scale)
    live = sum(lens)
    for most in sorted({max(max(lens), 1), 64}):
        for kw in ({}, {"workspace": torch.empty(0, dtype=torch.uint8, device="cuda")}):
            rings = s["ring_k"].clone(), s["ring_v"].clone()
            out = attention_call(s, dev, maps_of(dev, most), W, scale, rings, **kw)
            within(out[:live], want[:live], slack[:live], 2.0 ** -8, f"out, bound {most}, {list(kw)}")
            np.testing.assert_array_equal(_f64(rings[0]), rk)
            np.testing.assert_array_equal(_f64(rings[1]), rv)


@pytest.mark.parametrize("rows_n", [1, 20, 300])
def test_attention_over_many_rows(rows_n):
    """Every way a call splits its keys (8, 4 and 1 workgroups a row), at head counts of the released model."""
    rng = np.random.default_rng(rows_n)
    lens = rng.integers(1, 9 if rows_n > 100 else 20, rows_n).tolist()
    hkv, G, W = 2, 4, 512
    rows, slots, starts, pool_rows, dev = batch(rows_n, lens, True)
    s = attention_inputs(rows_n, sum(lens), pool_rows, slots, starts, hkv, G, W)
    want, slack, rk, rv = attention_oracle(s, slots, starts, rows, W, 0.0625)
    rings = s["ring_k"].clone(), s["ring_v"].clone()
    out = attention_call(s, dev, maps_of(dev, max(lens)), W, 0.0625, rings)
    within(out, want, slack, 2.0 ** -8, "out")
    np.testing.assert_array_equal(_f64(rings[0]), rk)
    np.testing.assert_array_equal(_f64(rings[1]), rv)


def test_attention_with_far_scores_and_few_keys():
    """Scores some hundreds apart (one key takes all), empty rings, rings of one key."""
    lens = [20, 3, 1, 6]
    hkv, G, W = 2, 4, 512
    rows, slots, _, pool_rows, dev = batch(21, lens, True)
    starts = [700, 0, 0, 1]
    dev["starts"] = torch.tensor(starts, device="cuda")
    for scale in (0.0625, 2.0, -1.5, 0.0):
        s = attention_inputs(31, sum(lens), pool_rows, slots, starts, hkv, G, W)
        want, slack, _, _ = attention_oracle(s, slots, starts, rows, W, scale)
        out = attention_call(s, dev, maps_of(dev), W, scale, (s["ring_k"].clone(), s["ring_v"].clone()))
        within(out, want, slack, 2.0 ** -8, f"scale {scale}")


@pytest.mark.parametrize("n,G", [(3, 4), (8, 4), (15, 4), (40, 4), (64, 2)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_keeps_a_bad_value_to_who_sees_it(n, G, value):
    """Ring columns of no position and the row past the window hold anything; one branch's value is not finite: only its
    descendants see it. A bad query or key reaches only its own, or who sees it."""
    hkv, W = 1, 512
    half = n // 2
    parents = [-1] + list(range(0, half - 1)) + [0] + list(range(max(half, 1), n - 1)) if n > 3 else [-1, 0, 0]
    bad = half // 2 + 1 if n > 3 else 1
    dev = {"parents": torch.tensor(parents, device="cuda"), "lens": torch.tensor([n], device="cuda"),
           "starts": torch.tensor([300], device="cuda"), "commits": None, "slots": torch.tensor([1], device="cuda")}
    s = attention_inputs(n, n, 2, [1], [300], hkv, G, W)
    rows = [(0, parents, 0)]
    want, slack, _, _ = attention_oracle(s, [1], [300], rows, W, 0.0625)
    s["ring_k"][1, :, 300:] = value
    s["ring_v"][1, :, 300:] = value
    out = attention_call(s, dev, maps_of(dev, n), W, 0.0625)
    within(out, want, slack, 2.0 ** -8, "dead ring columns")
    clean = {**s, "ring_k": s["ring_k"].nan_to_num(0, 0), "ring_v": s["ring_v"].nan_to_num(0, 0)}
    assert torch.equal(out, attention_call(clean, dev, maps_of(dev, n), W, 0.0625)), "dead ring columns are not read"
    below = [i for i in range(n) if bad in tree.path(parents, i)]
    rest = [i for i in range(n) if i not in below]
    for name, seen in (("value", below), ("new_k", below), ("q", [bad])):
        t = {**s, name: s[name].clone()}
        t[name][bad, 0, 5] = value
        out = attention_call(t, dev, maps_of(dev, n), W, 0.0625)
        others = [i for i in range(n) if i not in seen]
        within(out[others], want[others], slack[others], 2.0 ** -8, name)
        if name == "value" or value != value:
            got = torch.isfinite(out[seen].reshape(len(seen), G, D)[:, 0])
            assert not got[:, 5].any()
            if name == "value":   # the other dims of the value are as they were
                keep = [d for d in range(G * D) if d % D != 5]
                within(out[below][:, keep], want[below][:, keep], slack[below][:, keep], 2.0 ** -8, "its other dims")
    assert rest


@pytest.mark.parametrize("rows_n,n,G,W", [(70, 3, 4, 512), (70, 12, 4, 64), (70, 40, 4, 64), (260, 64, 2, 32)])
def test_attention_of_many_rows_with_bad_values(rows_n, n, G, W):
    """As many rows as leave none split: one workgroup a row (which writes its committed chain itself) or several. A value of
    three rows' last node is not finite: only these nodes see it, and the rings take it where it is committed."""
    hkv, bad = 1, (0, 7, rows_n - 1)
    parents = [-1, 0] + [(i - 1) // 2 for i in range(2, n)]
    total = rows_n * n
    rng = np.random.default_rng(rows_n + n)
    slots = rng.permutation(rows_n + 1)[:rows_n].tolist()
    starts = rng.integers(0, 3 * W, rows_n).tolist()
    commits = [2 if r % 3 else 0 for r in range(rows_n)]
    dev = {"parents": torch.tensor(parents * rows_n, device="cuda"), "lens": torch.tensor([n] * rows_n, device="cuda"),
           "starts": torch.tensor(starts, device="cuda"), "commits": torch.tensor(commits, device="cuda"),
           "slots": torch.tensor(slots, device="cuda")}
    s = attention_inputs(n, total, rows_n + 1, slots, starts, hkv, G, W)
    some = sorted({*bad, 1, 2, rows_n // 2})
    rows = [(r * n, parents, commits[r]) for r in range(rows_n)]
    want, slack, _, _ = attention_oracle(s, [slots[r] for r in some], [starts[r] for r in some], [rows[r] for r in some], W,
                                         0.0625)
    rings = s["ring_k"].clone(), s["ring_v"].clone()
    clean = attention_call(s, dev, maps_of(dev, n), W, 0.0625, rings)
    last = [r * n + n - 1 for r in bad]
    s["value"][last, 0, 9] = float("nan")
    moved = s["ring_k"].clone(), s["ring_v"].clone()
    out = attention_call(s, dev, maps_of(dev, n), W, 0.0625, moved)
    nodes = [r * n + i for r in some for i in range(n)]
    within(clean[nodes], want[nodes], slack[nodes], 2.0 ** -8, "without it")
    rest = [i for i in nodes if i not in last]
    within(out[rest], want[rest], slack[rest], 2.0 ** -8, "the other nodes")
    others = [r * n + i for r in range(rows_n) if r not in bad for i in range(n)]
    assert torch.equal(out[others], clean[others])
    dims = out[last].reshape(len(bad), G, D)
    assert not torch.isfinite(dims[:, :, 9]).any()
    keep = [g * D + d for g in range(G) for d in range(D) if d != 9]
    within(out[last][:, keep], want[last][:, keep], slack[last][:, keep], 2.0 ** -8, "its other dims")
    ref = s["ring_k"].clone(), s["ring_v"].clone()
    for r in range(rows_n):
        for j in range(commits[r]):
            for x, y in zip(ref, (s["new_k"], s["value"])):
                x[slots[r], :, (starts[r] + j) % W] = y[r * n + j]
    for x, y in zip(moved, ref):
        assert torch.equal(x, y)
    for x, y in zip(rings, ref):
        assert torch.equal(x, y)


def test_attention_takes_tokens_that_lie_apart():
    """q, new_k, value and the gate as columns of one wider projection: bitwise the packed ones."""
    lens, hkv, G, W = [7, 30], 2, 3, 512
    _, slots, starts, pool_rows, dev = batch(12, lens, True)
    total, hq = sum(lens), hkv * G
    s = attention_inputs(12, total, pool_rows, slots, starts, hkv, G, W)
    before = s["ring_k"].clone(), s["ring_v"].clone()
    rings = tuple(x.clone() for x in before)
    want = attention_call(s, dev, maps_of(dev), W, 0.0625, rings)
    widths = {"q": hq * D, "new_k": hkv * D, "value": hkv * D, "gate": hq * 2 * D}
    wide = randn(3, total, sum(widths.values()) + 24)
    at, t = 8, dict(s)
    for name, w in widths.items():
        wide[:, at:at + w] = s[name].reshape(total, w)
        t[name] = wide[:, at:at + w].unflatten(1, s[name].shape[1:]) if s[name].dim() > 2 else wide[:, at:at + w]
        at += w
    assert not t["q"].is_contiguous()
    other = tuple(x.clone() for x in before)
    assert torch.equal(attention_call(t, dev, maps_of(dev), W, 0.0625, other), want)
    for x, y in zip(rings, other):
        assert torch.equal(x, y)


def test_attention_leaves_the_rest_alone():
    """Rows of an unknown slot, longer than the bound, and tokens of no row keep their outputs; a pool whose elements pass
    2^31; positions past 2^31."""
    from hs_guard._lib import calls
    hkv, G, W, lens = 1, 2, 512, [5, 7, 4, 12]
    pool_rows = (1 << 31) // (513 * 256) + 40
    rows, _, _, _, dev = batch(3, lens, True, 4, slots=[pool_rows - 1, pool_rows, 3, 4], pool=pool_rows)
    starts = [(1 << 33) + 5, 9, 800, 2]
    dev["starts"] = torch.tensor(starts, device="cuda")
    t = maps_of(dev, 64)._replace(max_nodes=8)
    total = sum(lens) + 4
    s = attention_inputs(5, total, 5, [1, 3], [100, 800], hkv, G, W)
    small = s["ring_k"], s["ring_v"], s["ring_pos"]
    big = [torch.zeros(pool_rows, hkv, W + 1, D, dtype=BF16, device="cuda") for _ in range(2)]
    big_pos = torch.full((pool_rows, W + 1), -1, dtype=torch.long, device="cuda")
    last = starts[0] - 1
    columns = torch.arange(W)
    far = last - torch.remainder(last - columns, W)
    small[2][1, :W] = far.cuda()
    for slot, at in ((pool_rows - 1, 1), (3, 3)):
        for x, y in zip(big, small[:2]):
            x[slot] = y[at]
        big_pos[slot] = small[2][at]
    live_rows, live_starts = [rows[0], rows[2]], [starts[0], starts[2]]
    want, slack, rk, rv = attention_oracle(s, [1, 3], live_starts, live_rows, W, 0.0625)
    out = torch.full((total, hkv * G * D), 7.0, dtype=BF16, device="cuda")
    rc = calls().hsg_tree_attention(
        s["q"].data_ptr(), hkv * G * D, G * D, D, big[0].data_ptr(), big[1].data_ptr(), pool_rows, W,
        s["new_k"].data_ptr(), hkv * D, D, s["value"].data_ptr(), hkv * D, D, s["gate"].data_ptr(), hkv * G * 2 * D,
        G * 2 * D, 2 * D, D, big_pos.data_ptr(), dev["slots"].data_ptr(), dev["starts"].data_ptr(), t.lens.data_ptr(),
        t.offsets.data_ptr(), t.commits.data_ptr(), t.masks.data_ptr(), 4, 8, hkv, G, D, 0.0625, out.data_ptr(),
        hkv * G * D, G * D, D, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    live = [i for r in (0, 2) for i in range(rows[r][0], rows[r][0] + lens[r])]
    rest = [i for i in range(total) if i not in live]
    assert (out[rest] == 7.0).all()
    within(out[live], want[live], slack[live], 2.0 ** -8, "out")
    for x, ref in zip(big, (rk, rv)):
        np.testing.assert_array_equal(_f64(x[pool_rows - 1]), ref[1])
        np.testing.assert_array_equal(_f64(x[3]), ref[3])
        assert not x[4].any()


def test_gdn_state_past_32_bits():
    H = HV = 1
    pool_rows = (1 << 31) // (KD * KD) + 9
    rows, slots, _, _, dev = batch(3, [6, 17], True, slots=[pool_rows - 1, 2], pool=pool_rows)
    dev["commits"][:] = 1
    rows = [(a, p, 1) for a, p, _ in rows]
    s = gdn_inputs(8, 23, 4, H, HV, torch.float32)
    o, osize, st, ssize = gdn_oracle(s, H, HV, [3, 2], rows)
    big = torch.zeros(pool_rows, HV, KD, KD, dtype=torch.float32, device="cuda")
    big[pool_rows - 1], big[2] = s["state"][3], s["state"][2]
    out = gdn_call(s, H, HV, dev["slots"], maps_of(dev), big, False).reshape(o.shape)
    within(out, o, 2.0 ** -15 * osize, 2.0 ** -8, "out")
    within(big[[pool_rows - 1, 2]], st[[3, 2]], 2.0 ** -15 * ssize[[3, 2]], 0.0, "state")
    assert not big[3].any()


# ---------------------------------------------------------------------------------------------------------------
# a run of them together
# ---------------------------------------------------------------------------------------------------------------
def layer_inputs(seed, lens, H, HV, hkv, G, W, pool_rows, slots, starts):
    total = sum(lens)
    s = gdn_inputs(seed, total, pool_rows, H, HV, torch.float32)
    s.update(attention_inputs(seed + 20, total, pool_rows, slots, starts, hkv, G, W))
    c = (2 * H + HV) * KD
    s.update(x=randn(seed + 40, total, c), pool=randn(seed + 41, pool_rows, 3, c), weight=randn(seed + 42, c, 1, 4, scale=0.5))
    return s


def layers(s, dev, H, HV, W, max_nodes):
    """The maps, a gated-delta layer's conv and step, an attention layer: outputs and moved state."""
    from hs_guard.engine.kernels import tree_conv_silu
    trees = maps_of(dev, max_nodes)
    t = {**s, "packed": tree_conv_silu(s["x"], s["pool"], s["weight"], dev["slots"], trees)}
    y = gdn_call(t, H, HV, dev["slots"], trees, s["state"])
    return trees, t["packed"], y, attention_call(s, dev, trees, W, 0.0625)


def test_run_of_all_in_a_graph():
    """Captured once, replayed with other inputs in the same buffers and eager work between: bitwise the eager run, state
    and all."""
    lens, H, HV, hkv, G, W = [9, 1, 30, 16], 2, 4, 2, 4, 512
    sets = [batch(k, lens, True, pool=7) for k in (1, 2, 3)]
    data = [layer_inputs(50 * k, lens, H, HV, hkv, G, W, 7, b[1], b[2]) for k, b in enumerate(sets)]
    moved = ("state", "pool", "ring_k", "ring_v")
    dev = {k: v.clone() for k, v in sets[0][4].items()}
    live = {k: v.clone() for k, v in data[0].items()}
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layers(live, dev, H, HV, W, 32)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layers(live, dev, H, HV, W, 32)
    for k in (0, 1, 2, 1, 0):
        for name, v in sets[k][4].items():
            dev[name].copy_(v)
        for name, v in data[k].items():
            live[name].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        fresh = {name: v.clone() for name, v in data[k].items()}
        want = layers(fresh, sets[k][4], H, HV, W, 32)
        for a, b in zip(list(got[0][:5]) + list(got[1:]), list(want[0][:5]) + list(want[1:])):
            assert torch.equal(a, b)
        for name in moved:
            assert torch.equal(live[name], fresh[name]), name


def test_run_on_another_stream_and_shared_slots():
    """On a stream of its own, bitwise the same; rows without commits may score one session several times."""
    lens, H, HV, hkv, G, W = [12, 5, 12], 2, 2, 1, 4, 512
    rows, slots, starts, _, dev = batch(4, lens, False, slots=[1, 0, 1], pool=2)
    starts[2] = starts[0]
    dev["starts"] = torch.tensor(starts, device="cuda")
    s = layer_inputs(9, lens, H, HV, hkv, G, W, 2, slots, starts)
    before = {k: s[k].clone() for k in ("state", "pool", "ring_k", "ring_v")}
    want = layers(s, dev, H, HV, W, 16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layers(s, dev, H, HV, W, 16)
    side.synchronize()
    for a, b in zip(want[1:], got[1:]):
        assert torch.equal(a, b)
    for k, v in before.items():
        assert torch.equal(s[k], v)
    # each row alone gives what it gives in the batch
    for r in range(3):
        at = slice(rows[r][0], rows[r][0] + lens[r])
        one = {k: (v[at] if k in ("x", "a", "b", "z", "q", "new_k", "value", "gate") else v) for k, v in s.items()}
        d1 = {k: None if v is None else v[r:r + 1] for k, v in dev.items() if k != "parents"}
        d1["parents"] = dev["parents"][at]
        alone = layers(one, d1, H, HV, W, 16)
        for a, b in zip(alone[1:], want[1:]):
            assert torch.equal(a, b[at])


def test_two_streams_at_once_and_a_workspace_of_two_graphs():
    """Lone rows, whose attention splits its keys over a workspace: calls of two streams that overlap, and two graphs over one
    workspace replayed in turn, give what each gives alone."""
    hkv, G, W = 2, 4, 512
    sides = []
    for k in (1, 2):
        rows, slots, starts, pool_rows, dev = batch(60 + k, [11 + k], False)
        s = attention_inputs(70 + k, 11 + k, pool_rows, slots, starts, hkv, G, W)
        trees = maps_of(dev, 16)
        sides.append((s, dev, trees, attention_call(s, dev, trees, W, 0.0625)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sides]
    got = [[], []]
    for _ in range(12):
        for k, (s, dev, trees, _) in enumerate(sides):
            with torch.cuda.stream(streams[k]):
                got[k].append(attention_call(s, dev, trees, W, 0.0625))
    torch.cuda.synchronize()
    for k, (_, _, _, want) in enumerate(sides):
        assert all(torch.equal(x, want) for x in got[k])
    from hs_guard._lib import lib
    space = torch.empty(lib().hsg_tree_attention_workspace_bytes(1, hkv, G, 16), dtype=torch.uint8, device="cuda")
    assert space.numel() > 0
    graphs = []
    for s, dev, trees, _ in sides:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attention_call(s, dev, trees, W, 0.0625, workspace=space)
        graphs.append((graph, out))
    for _ in range(3):
        for (graph, out), (_, _, _, want) in zip(graphs, sides):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)


def test_refusals():
    from hs_guard.engine import kernels as K
    _, _, _, pool_rows, dev = batch(1, [4, 3], True)
    trees = maps_of(dev)
    s = layer_inputs(1, [4, 3], 2, 2, 1, 2, 512, pool_rows, [0, 1], [4, 4])
    conv = lambda **kw: K.tree_conv_silu(**{"qkv": s["x"], "pool": s["pool"], "weight": s["weight"],   # noqa: E731
                                            "slots": dev["slots"], "trees": trees, **kw})
    for bad in ({"qkv": s["x"].float()}, {"qkv": s["x"].t().contiguous().t()}, {"pool": s["pool"][:, :2]},
                {"slots": dev["slots"].int()}, {"slots": dev["slots"][:1]}, {"trees": trees._replace(max_nodes=65)},
                {"trees": trees._replace(masks=trees.masks[:3])}, {"qkv": s["x"].cpu()}):
        with pytest.raises((AssertionError, ValueError)):
            conv(**bad)
    odd = torch.zeros(7 * 12, dtype=BF16, device="cuda")
    with pytest.raises(ValueError):       # 12 channels: no multiple of 8
        conv(qkv=odd.reshape(7, 12), pool=odd.new_zeros(2, 3, 12), weight=odd.new_zeros(12, 1, 4))
    for bad in ({"state": s["state"].to(BF16)}, {"a": s["a"][:, :1]}, {"z": None}, {"norm_weight": None},
                {"packed": s["packed"][:, :-8]}):
        with pytest.raises((AssertionError, ValueError)):
            gdn_call({**s, **bad}, 2, 2, dev["slots"], trees, bad.get("state", s["state"]))
    for bad in (float("nan"), float("inf")):
        with pytest.raises(ValueError):
            attention_call(s, dev, trees, 512, bad)
    for bad in ({"q": s["q"][:, :, :128]}, {"ring_k": s["ring_k"][:, :, :-1]}, {"ring_pos": s["ring_pos"][:, :-1]},
                {"new_k": s["new_k"].transpose(0, 1)}, {"gate": s["gate"][:, :-8]}):
        with pytest.raises((AssertionError, ValueError)):
            attention_call({**s, **bad}, dev, trees, 512, 1.0)
    with pytest.raises(AssertionError):
        K.draft_tree_maps(dev["parents"], dev["lens"], dev["starts"][:1])
    with pytest.raises(AssertionError):
        K.draft_tree_maps(dev["parents"], dev["lens"], dev["starts"], max_nodes=0)
