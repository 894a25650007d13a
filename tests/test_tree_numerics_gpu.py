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


def check(s, rows, HV, most, slots):
    dtype = s["state"].dtype
    out, state = run(s, rows, HV, most, slots)
    want_o, want_s = oracle(s, rows, HV, slots)
    moved = [slot for slot, r in zip(slots, rows) if r[2]]
    if dtype is torch.float32:
        assert rel_norm(state[moved], want_s[moved]) <= STATE_NORM
    assert beyond_rounding(state[moved], want_s[moved], dtype) <= VALUE
    assert beyond_rounding(out, want_o, torch.bfloat16) <= VALUE
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
