"""The drafted-tree oracle against the streaming ones: on a chain each operator is the streaming one, and a branch is the
chain of its own path."""
import numpy as np
import pytest

from oracle import bf16, gdn, glue, ring, tree


def _rng(seed):
    return np.random.default_rng(seed)


def test_maps_of_a_small_tree():
    # two rows: a fork below a chain of two, and a chain; three tokens behind them
    parents = [-1, 0, 1, 1, 3, -1, -1, 0, 7, 7, 7]
    off, lens, done, pos, masks = tree.tree_maps(parents, [5, 3], [10, 0], [2, 0], 64)
    assert off == [0, 5] and lens == [5, 3] and done == [2, 0]
    assert pos == [10, 11, 12, 12, 13, 0, 0, 1, 0, 0, 0]
    assert masks == [0b1, 0b11, 0b111, 0b1011, 0b11011, 0b1, 0b10, 0b101, 0, 0, 0]


@pytest.mark.parametrize("parents,lens,starts,commits,most", [
    ([0], [1], [0], [0], 64),              # its own parent
    ([-1, 2, 0], [3], [0], [0], 64),       # a parent after its child
    ([-1, -2], [2], [0], [0], 64),         # no such parent
    ([-1, 0, 1], [3], [0], [0], 2),        # more than max_nodes
    ([-1, 0], [3], [0], [0], 64),          # more than the buffer holds
    ([-1, 0], [2], [-1], [0], 64),         # a negative start
    ([-1, -1], [2], [0], [2], 64),         # commits over a fork
    ([-1, 0], [2], [0], [3], 64),          # more commits than nodes
    ([-1, 0], [2], [0], [-1], 64),
    ([-1, 0], [-2], [0], [0], 64),
])
def test_maps_reject_what_is_no_tree(parents, lens, starts, commits, most):
    _, lens_out, done, pos, masks = tree.tree_maps(parents, lens, starts, commits, most)
    assert lens_out == [0] and done == [0] and not any(pos) and not any(masks)


def test_conv_on_a_chain_and_a_branch():
    r = _rng(0)
    C, L = 6, 7
    with bf16.exact():
        x, pool, w = r.standard_normal((L, C)), r.standard_normal((2, 3, C)), r.standard_normal((C, 4))
        want, pool2 = glue.conv_silu_update(x[None], pool, w, [1], [L])
        out, _, got = tree.tree_conv_silu(x, pool, w, [1], [(0, list(range(-1, L - 1)), L)])
        np.testing.assert_allclose(out, want[0], rtol=1e-6, atol=1e-7)   # its sums are rounded to float32
        np.testing.assert_array_equal(got, pool2)
        # node 5 hangs on node 1: its path is 0, 1, 5
        out, _, got = tree.tree_conv_silu(x, pool, w, [1], [(0, [-1, 0, 1, 2, 3, 1, 5], 0)])
        want, _ = glue.conv_silu_update(x[None][:, [0, 1, 5, 6]], pool, w, [1], [4])
        np.testing.assert_allclose(out[[0, 1, 5, 6]], want[0], rtol=1e-6, atol=1e-7)
        np.testing.assert_array_equal(got, pool)


def test_gdn_on_a_chain_and_a_branch():
    r = _rng(1)
    H, HV, K, L = 2, 4, 8, 6
    packed = r.standard_normal((L, 2 * H * K + HV * K))
    a, b = r.standard_normal((2, L, HV))
    A, dt = r.standard_normal((2, HV))
    state = r.standard_normal((2, HV, K, K))
    o, osize, st, ssize = tree.gdn_tree_step(packed, H, HV, a, b, A, dt, state, [1], [(0, list(range(-1, L - 1)), 4)])
    want, _, _ = gdn.gdn_slot_step(packed[None], H * K, H, K, HV, K, a[None], b[None], A, dt, state, [1], [L])
    np.testing.assert_allclose(o, want[0], rtol=1e-12, atol=1e-13)
    _, _, after = gdn.gdn_slot_step(packed[None, :4], H * K, H, K, HV, K, a[None, :4], b[None, :4], A, dt, state, [1], [4])
    np.testing.assert_allclose(st, after, rtol=1e-12, atol=1e-13)
    assert (osize >= np.abs(o)).all() and (ssize >= np.abs(st)).all()
    at = [0, 1, 5]
    o, _, st, _ = tree.gdn_tree_step(packed, H, HV, a, b, A, dt, state, [0], [(0, [-1, 0, 1, 2, 3, 1], 0)])
    want, _, _ = gdn.gdn_slot_step(packed[None, at], H * K, H, K, HV, K, a[None, at], b[None, at], A, dt, state, [0], [3])
    np.testing.assert_allclose(o[at], want[0], rtol=1e-12, atol=1e-13)
    np.testing.assert_array_equal(st, state)


def test_attention_on_a_chain_and_a_branch():
    r = _rng(2)
    hkv, G, D, W, L, start = 2, 2, 8, 4, 6, 9
    q, k, v = (r.standard_normal((L, h, D)) for h in (hkv * G, hkv, hkv))
    ring_k, ring_v = r.standard_normal((2, 2, hkv, W + 1, D))
    ring_pos = np.full((2, W + 1), -1)
    for p in range(start - W, start):
        ring_pos[1, p % W] = p

    def streamed(at):
        n = len(at)
        out = ring.ring_attention_reference(
            q[at].reshape(n, hkv, G, D).transpose(1, 2, 0, 3).reshape(1, hkv, G * n, D), ring_k, ring_v,
            k[at].transpose(1, 0, 2)[None], v[at].transpose(1, 0, 2)[None], ring_pos, [1], [start], [n], 0.3, W)
        return out.reshape(hkv, G, n, D).transpose(2, 0, 1, 3).reshape(n, hkv * G, D)

    o, size, _, rk, _ = tree.tree_attention(q, ring_k, ring_v, k, v, ring_pos, [1], [start],
                                            [(0, list(range(-1, L - 1)), 5)], 0.3, W)
    np.testing.assert_allclose(o, streamed(list(range(L))), rtol=1e-12, atol=1e-13)
    # a chain of 5 over a ring of 4: the last 4 stay
    for j in range(1, 5):
        np.testing.assert_array_equal(rk[1, :, (start + j) % W], k[j])
    at = [0, 1, 5]
    o, _, _, rk, _ = tree.tree_attention(q, ring_k, ring_v, k, v, ring_pos, [1], [start], [(0, [-1, 0, 1, 2, 3, 1], 0)],
                                         0.3, W)
    np.testing.assert_allclose(o[at], streamed(at), rtol=1e-12, atol=1e-13)
    np.testing.assert_array_equal(rk, ring_k)
