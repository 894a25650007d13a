"""How exact the tree gated-delta step is: the committed state and the outputs against float64, to bars that do not grow with
a path's depth (tests/tree_helpers.py; tests/test_tree_bars.py shows on the CPU what they let through and what not).

The majorant of tests/test_tree_gpu.py adds magnitudes where the rule subtracts, so it grows with every node: on a chain of
64 it is above the values themselves."""
import numpy as np
import pytest
import torch

from oracle import tree
from tree_helpers import KD, STATE_NORM, VALUE, beyond_rounding, f64, like_keys, rel_norm

pytestmark = pytest.mark.gpu


def run(s, rows, HV, most, slots, gate=False):
    """One key head: (out [T, HV, KD], state) of the rows (offset, parents, commits)."""
    from hs_guard.engine.kernels import draft_tree_maps, gdn_tree_step
    d = {k: v.cuda() for k, v in s.items()}
    ints = lambda x: torch.tensor(x, dtype=torch.long, device="cuda")   # noqa: E731
    trees = draft_tree_maps(ints([p for _, parents, _ in rows for p in parents]), ints([len(r[1]) for r in rows]),
                            ints([9] * len(rows)), ints([r[2] for r in rows]), most)
    more = {"z": d["z"], "norm_weight": d["norm_weight"]} if gate else {}
    out = gdn_tree_step(d["packed"], KD, 1, KD, HV, KD, d["a"], d["b"], d["A_log"], d["dt_bias"], d["state"], ints(slots),
                        trees, **more)
    return out.reshape(-1, HV, KD), d["state"]


def oracle(s, rows, HV, slots):
    o, _, st, _ = tree.gdn_tree_step(f64(s["packed"]), 1, HV, f64(s["a"]), f64(s["b"]), f64(s["A_log"]), f64(s["dt_bias"]),
                                     f64(s["state"]), slots, rows)
    return o, st


def check(s, rows, HV, most, slots, gate=False, skip=()):
    """skip: nodes whose outputs are not looked at."""
    dtype = s["state"].dtype
    out, state = run(s, rows, HV, most, slots, gate)
    want_o, want_s = oracle(s, rows, HV, slots)
    bar = VALUE
    if gate:   # an error of o times r w silu(z), of which the largest is at most 8 times a row's rms
        want_o = tree.gated(want_o, np.abs(want_o), f64(s["z"]).reshape(want_o.shape), f64(s["norm_weight"]), 1e-6)[0]
        bar = 8 * VALUE
    kept = [i for i in range(len(want_o)) if i not in skip]
    out, want_o = out[kept], want_o[kept]
    moved = [slot for slot, r in zip(slots, rows) if r[2]]
    if dtype is torch.float32:
        assert rel_norm(state[moved], want_s[moved]) <= STATE_NORM
    assert beyond_rounding(state[moved], want_s[moved], dtype) <= VALUE
    assert beyond_rounding(out, want_o, torch.bfloat16) <= bar
    still = [i for i in range(len(state)) if i not in moved]
    assert torch.equal(state[still].cpu(), s["state"][still])


@pytest.mark.parametrize("n", [3, 9, 16, 33, 48, 64])
@pytest.mark.parametrize("noise", [0.0, 0.05, 0.1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_chains_of_like_keys(n, noise, dtype):
    """Text that repeats itself, committed whole: what the chain's products do must not cancel."""
    s = like_keys(n, n, 2, noise, dtype)
    for most in sorted({n, 64}):
        check(s, [(0, list(range(-1, n - 1)), n)], 2, most, [1])


@pytest.mark.parametrize("n", [1, 3, 12, 17, 40, 64])
def test_an_fp16_state_takes_whole_updates(n):
    """Chains of unlike keys over an fp16 state, committed whole and in part: rounded once, from fp32's digits."""
    s = like_keys(2 + n, n, 2, 1.0, torch.float16)
    for done in sorted({1, (n + 1) // 2, n}):
        for most in sorted({n, 64}):
            check(s, [(0, list(range(-1, n - 1)), done)], 2, most, [0])


def trees_of(seed, lens):
    """Rows of random trees, of which the first nodes, a chain, are committed; every other row commits nothing."""
    rng = np.random.default_rng(seed)
    rows, at = [], 0
    for r, n in enumerate(lens):
        done = int(rng.integers(1, n + 1)) if r % 2 == 0 else 0
        near = int(rng.choice([1, 3, n]))
        parents = [i - 1 if i < done else int(rng.integers(max(-1, i - near), i)) for i in range(n)]
        rows.append((at, parents, done))
        at += n
    return rows


@pytest.mark.parametrize("lens", [[64], [1, 1, 2], [12, 5, 33, 1, 16, 17, 64], [33] * 5, [15, 16, 31, 32, 48, 49, 63]])
@pytest.mark.parametrize("noise", [0.2, 1.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("gate", [False, True])
def test_trees(lens, noise, dtype, gate):
    rows = trees_of(len(lens), lens)
    s = like_keys(sum(lens), sum(lens), 2, noise, dtype, pool_rows=len(lens) + 1)
    slots = np.random.default_rng(1).permutation(len(lens) + 1)[:len(lens)].tolist()
    for most in sorted({max(lens), 64}):
        check(s, rows, 2, most, slots, gate)


@pytest.mark.parametrize("n", [20, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_steep_decays(n, dtype):
    """Nodes that forget all but e^-20 or e^-600 of what came before them, in the middle of a chain and at its end."""
    s = like_keys(n, n, 2, 1.0, dtype)
    s["A_log"][:] = 2.7
    for at, a in ((n // 3, 8.0), (n // 2, 47.0), (n - 2, 8.0)):
        s["a"][at] = a
    check(s, [(0, list(range(-1, n - 1)), n)], 2, n, [0])
    check(s, [(0, list(range(-1, n - 1)), n // 2)], 2, n, [1])


@pytest.mark.parametrize("n", [9, 16, 30, 64])
@pytest.mark.parametrize("noise", [0.0, 1.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_computed_again(n, noise, dtype):
    """A NaN at a leaf: the row's other results come from the walk over each node's own ancestors, as exact."""
    s = like_keys(n, n, 2, noise, dtype)
    parents = list(range(-1, n - 2)) + [n // 2]
    want = [(0, parents, n - 1)]
    s["packed"][n - 1, 2 * KD:] = 0.0        # the oracle's values; its own outputs are not compared
    clean = {k: v.clone() for k, v in s.items()}
    check(clean, want, 2, n, [0], skip=[n - 1])
    s["packed"][n - 1, 2 * KD + 5] = float("nan")
    s["packed"][n - 1, 3 * KD + 9] = float("nan")
    out, state = run(s, want, 2, n, [0])
    want_o, want_s = oracle(clean, want, 2, [0])
    if dtype is torch.float32:
        assert rel_norm(state[0], want_s[0]) <= STATE_NORM
    assert beyond_rounding(state[0], want_s[0], dtype) <= VALUE
    assert beyond_rounding(out[:n - 1], want_o[:n - 1], torch.bfloat16) <= VALUE
    assert torch.isnan(out[n - 1]).any(-1).all()
