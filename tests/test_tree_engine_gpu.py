"""Drafted trees through the engine (SlotStreamEngine.step_tree): every node scores as the tokens of its own path would if they
were streamed (step on a restored session), and nothing moves but the committed chains.

The two routes round at other places (the tree's conv, norm and attention outputs once, the streaming kernels' as the reference
does) and run their products at other sizes, so they agree as the streaming path does with independently computed products:
1e-2 on probabilities (tests/test_engine_gpu.py), and states to the same end-to-end bar, 2e-2 relative. What must not move is
compared bitwise.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
POOLS = ("rec", "conv", "ring_k", "ring_v", "ring_pos")
TOL, STATE_TOL = 1e-2, 2e-2


@pytest.fixture(scope="module")
def model():
    from hs_guard.model import GuardConfig, GuardModel
    cfg = GuardConfig(vocab_size=1000, hidden_size=1024, num_hidden_layers=4, intermediate_size=1024,
                      linear_num_key_heads=2, linear_num_value_heads=4, num_attention_heads=8, num_key_value_heads=2,
                      window_tokens=32)
    return GuardModel.random(cfg, seed=0, device="cuda:0")


def engine(model, slots=4, **kw):
    from hs_guard.engine.slot_engine import SlotStreamEngine
    eng = SlotStreamEngine(model, slots, **kw)
    rng = np.random.default_rng(5)
    eng.step([(s, rng.integers(0, 1000, n).tolist()) for s, n in zip(range(slots), (5, 70, 33, 1))])
    return eng


def a_tree(rng, n):
    return rng.integers(0, 1000, n).tolist(), [int(rng.integers(max(-1, i - 4), i)) for i in range(n)]


def chain_of(parents, i):
    way = [i]
    while parents[way[-1]] >= 0:
        way.append(parents[way[-1]])
    return way[::-1]


def pools(eng):
    return {name: getattr(eng, name).clone() for name in POOLS}


def streamed(eng, slot, ids):
    """Probabilities of ids streamed onto the slot, which is then put back."""
    snap = eng.snapshot(slot)
    out = eng.step([(slot, ids)])
    eng.restore(slot, snap)
    return {r: out[r][0].numpy() for r in out}


@pytest.mark.parametrize("sizes", [(1,), (3, 1), (14, 2, 9, 31), (32, 32)])
@pytest.mark.parametrize("graphs", [True, False])
def test_nodes_score_as_their_paths_and_nothing_moves(model, sizes, graphs):
    eng = engine(model, use_graphs=graphs)
    rng = np.random.default_rng(len(sizes))
    trees = [(int(s),) + a_tree(rng, n) for s, n in zip(rng.permutation(4), sizes)]
    before, length = pools(eng), eng.length.copy()
    out = eng.step_tree(trees)
    for name, t in before.items():
        # (the scratch slot is padding rows' and holds anything)
        assert torch.equal(getattr(eng, name)[:, :4] if name != "ring_pos" else eng.ring_pos[:4],
                           t[:, :4] if name != "ring_pos" else t[:4]), name
    assert (eng.length == length).all()
    for k, (slot, ids, parents) in enumerate(trees):
        leaves = [i for i in range(len(ids)) if i not in parents]
        for leaf in leaves:
            way = chain_of(parents, leaf)
            want = streamed(eng, slot, [ids[i] for i in way])
            for role in eng.roles:
                assert np.abs(out[role][k].numpy()[way] - want[role]).max() < TOL


def test_committed_chains_move_as_a_step_would(model):
    """Rows that commit nothing, some and all of their nodes; the next step goes on from there."""
    eng, ref = engine(model), engine(model)
    rng = np.random.default_rng(2)
    requests, accepted = [], []
    for slot, (n, c) in enumerate(((9, 4), (17, 0), (6, 6), (32, 30))):
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
            a, b = a[:, :, :, :32], b[:, :, :, :32]
        assert float((a - b).norm() / b.norm()) < STATE_TOL, name
    more = [(s, rng.integers(0, 1000, 3).tolist()) for s in range(4)]
    x, y = eng.step(more), ref.step(more)
    for role in eng.roles:
        for a, b in zip(x[role], y[role]):
            assert np.abs(a.numpy() - b.numpy()).max() < TOL


def test_graph_equals_eager_and_calls_repeat(model):
    """Captured tree ticks between ordinary ones, bitwise the eager engine; the same call again gives the same."""
    a, b = engine(model, use_graphs=True), engine(model, use_graphs=False)
    rng = np.random.default_rng(9)
    for k in range(3):
        trees = []
        for slot, n in enumerate((5, 12, 1, 20)):
            ids, parents = a_tree(rng, n)
            c = int(rng.integers(0, 3)) if k else 0
            c = min(c, n)
            parents[:c] = range(-1, c - 1)
            trees.append((slot, ids, parents, c))
        free = [t[:3] for t in trees]
        for calls in (free, free, trees):
            x, y = a.step_tree(calls), b.step_tree(calls)
            for role in a.roles:
                for u, v in zip(x[role], y[role]):
                    assert torch.equal(u, v)
        ticks = [(s, rng.integers(0, 1000, 2).tolist()) for s in range(4)]
        x, y = a.step(ticks), b.step(ticks)
        for role in a.roles:
            for u, v in zip(x[role], y[role]):
                assert torch.equal(u, v)
        for name in POOLS:
            u, v = getattr(a, name), getattr(b, name)
            assert torch.equal(u[:4], v[:4]) if name == "ring_pos" else torch.equal(u[:, :4], v[:, :4])
    assert a.stats["graph_replays"] > 0 and b.stats["graph_replays"] == 0


def test_one_session_many_trees_and_more_rows_than_a_tick(model):
    eng = engine(model, session_buckets=(1, 2))
    rng = np.random.default_rng(4)
    trees = [(2,) + a_tree(rng, n) for n in (3, 8, 1)] + [(0,) + a_tree(rng, 5)]
    out = eng.step_tree(trees)
    for k, t in enumerate(trees):
        alone = eng.step_tree([t])
        for role in eng.roles:
            assert np.abs(out[role][k].numpy() - alone[role][0].numpy()).max() < TOL


def test_api_and_refusals(model):
    from hs_guard.runtime import StreamingGuard, random_metadata
    guard = StreamingGuard(model, random_metadata(window_tokens=32), max_slots=3)
    guard.step([(1, [5, 6, 7])])
    records = guard.step_tree([(1, [1, 2, 3], [-1, 0, 0]), (0, [4], [-1])], role="user")
    assert [r["slot"] for r in records] == [1, 0] and [len(r["cut_scores"]) for r in records] == [3, 1]
    assert all(0 <= x <= 1 for r in records for x in r["cut_scores"])
    eng = guard.engine
    eng.prepare_trees(2, [8], 5, commits=True)
    length = eng.length.copy()
    for bad in ([(3, [1], [-1])], [(0, [], [])], [(0, [1000], [-1])], [(0, [1, 2], [-1])], [(0, [1, 2], [-1, 1])],
                [(0, [1], [-2])], [(0, [1, 2], [-1, -1], 2)], [(0, [1], [-1], 2)], [(0, [1], [-1], -1)], [(0, [1])],
                [(0, [1] * 33, [-1] * 33)], [(0, [1], [-1], 1), (0, [2], [-1])], [(0, [1], [-1]), (0, [2], [-1], 1)],
                [(0, [1.5], [-1])], [(0, [1], [-1], 0.5)], [(0.5, [1], [-1])]):
        with pytest.raises(ValueError):
            eng.step_tree(bad)
    with pytest.raises(ValueError):
        guard.step_tree([])
    with pytest.raises(ValueError):
        guard.step_tree([(0, [1], [-1])], role="system")
    assert (eng.length == length).all()
    assert eng.step_tree([]) == {r: [] for r in eng.roles}
