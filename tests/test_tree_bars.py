"""The bars of the tree gated-delta step's precision tests (tests/test_tree_numerics_gpu.py), on the CPU: the unrolled form in
fp32 as the kernel computes it passes them, and mistakes that matter do not. Every mistake is planted in the model here."""
import numpy as np
import pytest
import torch

from oracle import gdn, tree
from tree_helpers import KD, STATE_NORM, VALUE, beyond_rounding, f64, like_keys, rel_norm

F = np.float32


def unrolled(s, parents, done, head, mistake=None):
    """(I + A) U = R and the outputs and state from it, one head, in fp32 with 16 x 16 blocks inverted one by one."""
    n = len(parents)
    packed = f64(s["packed"])
    q = (gdn.l2norm(packed[:, :KD]) * KD ** -0.5).astype(F)
    k = gdn.l2norm(packed[:, KD:2 * KD]).astype(F)
    v = packed[:, (2 + head) * KD:(3 + head) * KD].astype(F)
    g, beta = (x[:, head] for x in gdn.gates(f64(s["a"]), f64(s["b"]), f64(s["A_log"]), f64(s["dt_bias"])))
    near = np.zeros((n, n), bool)
    G = np.zeros(n)
    for i, p in enumerate(parents):
        if p >= 0:
            near[i] = near[p]
            G[i] = G[p]
        near[i, i] = True
        G[i] += g[i]
    s0 = f64(s["state"])[0, head].astype(F)
    decay = np.where(near, np.exp(np.where(near, G[:, None] - G[None], 0.0)), 0.0).astype(F)
    A = beta.astype(F)[:, None] * decay * (k @ k.T) * ~np.eye(n, dtype=bool)
    P = decay * (q @ k.T)
    eG = np.exp(G).astype(F)[:, None]
    R = beta.astype(F)[:, None] * (v - eG * (k @ s0))
    if mistake == "an ancestor is lost":
        A[n - 1, n - 40] = 0
    if mistake == "a block is lost":
        A[32:48, :16] = 0
    if mistake == "an output's ancestor is lost":
        P[n - 1, n - 40] = 0
    U = np.zeros((n, KD), F)
    for b in range(0, n, 16):
        X = -A[b:b + 16, b:b + 16]
        T = np.eye(len(X), dtype=F)
        if mistake == "powers":
            T, X2 = T + X, X
            for _ in range(3):
                X2 = X2 @ X2
                T = T + T @ X2
        else:
            for m in range(len(X) - 1):
                T[m + 1:] += X[m + 1:, m:m + 1] * T[m]
        U[b:b + 16] = T @ (R[b:b + 16] - A[b:b + 16, :b] @ U[:b])
    o = eG * (q @ s0) + P @ U
    up = U[:done]
    if mistake == "16 digits of an update":
        up = (up.view(np.uint32) & 0xffff0000).view(F)
        rest = U[:done] - up
        up = up + (rest.view(np.uint32) & 0xffff0000).view(F)
    left = np.exp(G[done - 1] - G[:done]).astype(F)[:, None]
    return o, eG[done - 1] * s0 + (k[:done] * left).T @ up


def oracle(s, parents, done, HV):
    o, _, st, _ = tree.gdn_tree_step(f64(s["packed"]), 1, HV, f64(s["a"]), f64(s["b"]), f64(s["A_log"]), f64(s["dt_bias"]),
                                     f64(s["state"]), [0], [(0, parents, done)])
    return o[:, 0], st[0, 0]


def errors(s, parents, done, mistake=None):
    """(state's norm, outputs beyond a bf16 rounding, state beyond its type's rounding) of head 0."""
    want_o, want_s = oracle(s, parents, done, s["a"].shape[1])
    o, state = unrolled(s, parents, done, 0, mistake)
    dtype = s["state"].dtype
    return (rel_norm(state, want_s), beyond_rounding(torch.tensor(o).to(torch.bfloat16), want_o, torch.bfloat16),
            beyond_rounding(torch.tensor(state).to(dtype), want_s, dtype))


@pytest.mark.parametrize("n", [16, 33, 64])
@pytest.mark.parametrize("noise", [0.0, 0.05, 0.1])
def test_like_keys_by_substitution_and_by_powers(n, noise):
    chain = list(range(-1, n - 1))
    s = like_keys(n, n, 1, noise)
    norm, out, value = errors(s, chain, n)
    assert norm < STATE_NORM and out < VALUE and value < VALUE
    norm, out, _ = errors(s, chain, n, "powers")   # (33: the last block, of one node, has nothing to invert)
    assert norm > 2 * STATE_NORM or out > 2 * VALUE


@pytest.mark.parametrize("mistake", ["an ancestor is lost", "a block is lost", "an output's ancestor is lost"])
def test_mistakes_deep_in_a_tree_are_seen(mistake):
    n = 64
    rng = np.random.default_rng(3)
    for parents, done in ((list(range(-1, n - 1)), n), ([int(rng.integers(max(-1, i - 2), i)) if i > 50 else i - 1
                                                         for i in range(n - 1)] + [n - 2], 50)):
        s = like_keys(5, n, 1, 1.0)
        norm, out, value = errors(s, parents, done)
        assert norm < STATE_NORM and out < VALUE and value < VALUE
        if "output" in mistake or "block" in mistake or done == n:
            norm, out, _ = errors(s, parents, done, mistake)
            assert out > 4 * VALUE
            assert norm > 4 * STATE_NORM or "output" in mistake


@pytest.mark.parametrize("n", [20, 64])
def test_steep_decays_pass(n):
    s = like_keys(n, n, 1, 1.0)
    s["A_log"][:] = 2.7
    for at, a in ((n // 3, 8.0), (n // 2, 47.0), (n - 2, 8.0)):
        s["a"][at] = a
    for done in (n, n // 2):
        norm, out, value = errors(s, list(range(-1, n - 1)), done)
        assert norm < STATE_NORM and out < VALUE and value < VALUE


@pytest.mark.parametrize("n", [1, 3, 12, 40])
def test_an_fp16_state_tells_an_update_of_16_digits(n):
    """What fp32 leaves moves few values over a border of fp16, and these by little."""
    chain = list(range(-1, n - 1))
    s = like_keys(2, n, 1, 1.0, torch.float16)
    assert errors(s, chain, n)[2] < VALUE
    assert errors(s, chain, n, "16 digits of an update")[2] > VALUE
