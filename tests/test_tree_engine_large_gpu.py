"""The largest trees that the public path takes (33 to 64 nodes, a window of 512), over both state types: step_tree against
step() along every root-to-leaf path and against step() of the committed tokens, at the bars of tests/test_tree_engine_gpu.py
(1e-2 on probabilities, 2e-2 relative on states), and bitwise where nothing may move."""
import numpy as np
import pytest
import torch

from test_tree_engine_gpu import POOLS, STATE_TOL, TOL, a_tree, chain_of, pools, streamed

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    from hs_guard.model import GuardConfig, GuardModel
    cfg = GuardConfig(vocab_size=1000, hidden_size=1024, num_hidden_layers=4, intermediate_size=1024,
                      linear_num_key_heads=2, linear_num_value_heads=4, num_attention_heads=8, num_key_value_heads=2,
                      window_tokens=512)
    return GuardModel.random(cfg, seed=1, device="cuda:0")


def engine(model, state_dtype, **kw):
    from hs_guard.engine.slot_engine import SlotStreamEngine
    eng = SlotStreamEngine(model, 4, state_dtype=state_dtype, **kw)
    rng = np.random.default_rng(5)
    eng.step([(s, rng.integers(0, 1000, n).tolist()) for s, n in zip(range(4), (5, 700, 490, 1))])
    return eng


@pytest.mark.parametrize("state_dtype", ["float32", "float16"])
@pytest.mark.parametrize("sizes", [(64,), (40, 64), (33, 1, 64, 49)])
@pytest.mark.parametrize("graphs", [True, False])
def test_large_trees_score_as_their_paths(model, state_dtype, sizes, graphs):
    eng = engine(model, state_dtype, use_graphs=graphs)
    rng = np.random.default_rng(len(sizes))
    trees = [(int(s),) + a_tree(rng, n) for s, n in zip(rng.permutation(4), sizes)]
    trees[0] = (trees[0][0], trees[0][1], list(range(-1, sizes[0] - 1)))         # the deepest there is
    before, length = pools(eng), eng.length.copy()
    out = eng.step_tree(trees)
    for name, t in before.items():
        now = getattr(eng, name)
        assert torch.equal(now[:4], t[:4]) if name == "ring_pos" else torch.equal(now[:, :4], t[:, :4]), name
    assert (eng.length == length).all()
    for k, (slot, ids, parents) in enumerate(trees):
        for leaf in [i for i in range(len(ids)) if i not in parents]:
            way = chain_of(parents, leaf)
            want = streamed(eng, slot, [ids[i] for i in way])
            for role in eng.roles:
                assert np.abs(out[role][k].numpy()[way] - want[role]).max() < TOL


@pytest.mark.parametrize("state_dtype", ["float32", "float16"])
def test_large_committed_chains_move_as_a_step_would(model, state_dtype):
    eng, ref = engine(model, state_dtype), engine(model, state_dtype)
    rng = np.random.default_rng(2)
    requests, accepted = [], []
    for slot, (n, c) in enumerate(((40, 33), (64, 0), (64, 64), (50, 1))):
        ids, parents = a_tree(rng, n)
        parents[:c] = range(-1, c - 1)
        requests.append((slot, ids, parents, c))
        if c:
            accepted.append((slot, ids[:c]))
    still = eng.snapshot(1)
    out = eng.step_tree(requests)
    want = ref.step(accepted)
    for role in eng.roles:
        for (slot, ids), w in zip(accepted, want[role]):
            assert np.abs(out[role][slot][:len(ids)].numpy() - w.numpy()).max() < TOL
    after = eng.snapshot(1)
    for name in POOLS:
        assert torch.equal(after[name], still[name])
    assert eng.length.tolist() == ref.length.tolist()
    assert torch.equal(eng.ring_pos[:4], ref.ring_pos[:4])
    for name in ("rec", "conv", "ring_k", "ring_v"):
        a, b = (getattr(e, name)[:, :4].double() for e in (eng, ref))
        if name.startswith("ring"):
            a, b = a[:, :, :, :512], b[:, :, :, :512]
        assert float((a - b).norm() / b.norm()) < STATE_TOL, name
    more = [(s, rng.integers(0, 1000, 3).tolist()) for s in range(4)]
    x, y = eng.step(more), ref.step(more)
    for role in eng.roles:
        for a, b in zip(x[role], y[role]):
            assert np.abs(a.numpy() - b.numpy()).max() < TOL


@pytest.mark.parametrize("state_dtype", ["float32", "float16"])
def test_a_session_with_a_nan_leaves_the_others_alone(model, state_dtype):
    """One session's recurrent state and ring hold a NaN: the other sessions' scores and states are as without it, bitwise."""
    eng, ref = engine(model, state_dtype), engine(model, state_dtype)
    rng = np.random.default_rng(8)
    trees = []
    for slot, n in enumerate((12, 40, 64, 9)):
        ids, parents = a_tree(rng, n)
        parents[:3] = range(-1, 2)
        trees.append((slot, ids, parents, 3))
    eng.rec[:, 1, :, 3, 5] = float("nan")
    eng.ring_v[:, 1, :, :, 7] = float("nan")
    x, y = eng.step_tree(trees), ref.step_tree(trees)
    for role in eng.roles:
        assert torch.isnan(x[role][1]).all()
        for slot in (0, 2, 3):
            assert torch.equal(x[role][slot], y[role][slot])
    for name in POOLS:
        a, b = getattr(eng, name), getattr(ref, name)
        for slot in (0, 2, 3):
            assert torch.equal(a[slot], b[slot]) if name == "ring_pos" else torch.equal(a[:, slot], b[:, slot]), name
