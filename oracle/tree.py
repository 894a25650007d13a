"""Drafted-tree oracle (test infrastructure only; float64): the operators of ``hs_guard.engine.kernels`` over packed trees,
node by node along the parents. The reference has no counterpart; on a chain every operator is its streaming one, which is
how ``tests/test_oracle_tree.py`` pins them (``oracle.gdn``, ``oracle.glue``, ``oracle.ring``).

Every function that computes values also returns a majorant of what rounding can do to them: the same sums over magnitudes.
A sum of n products rounded to fp32 at each step is off by at most n 2^-24 of the sum of the products' magnitudes.
"""
import numpy as np

from .bf16 import sigmoid, silu
from .gdn import gates, l2norm


def tree_maps(parents, lens, starts, commits, max_nodes):
    """(offsets, lens, commits, pos, masks as Python ints): hsg_tree_maps."""
    total = len(parents)
    offsets, lens_out, commits_out = [], [], []
    pos, masks = [0] * total, [0] * total
    at = 0
    for n, size in enumerate(lens):
        size = int(size)
        done = int(commits[n]) if commits is not None else 0
        offsets.append(at)
        good = 0 <= size <= max_nodes and at + size <= total and starts[n] >= 0 and 0 <= done <= size
        row = [int(p) for p in parents[at:at + size]] if good else []
        good = good and all(-1 <= p < i and (i >= done or p == i - 1) for i, p in enumerate(row))
        lens_out.append(size if good else 0)
        commits_out.append(done if good else 0)
        for i, p in enumerate(row if good else []):
            masks[at + i] = (1 << i) | (masks[at + p] if p >= 0 else 0)
            pos[at + i] = int(starts[n]) + (pos[at + p] - int(starts[n]) + 1 if p >= 0 else 0)
        at += min(max(size, 0), total + 1)
    return offsets, lens_out, commits_out, pos, masks


def path(parents, i):
    """Node i's ancestors from the root on, itself last."""
    out = [i]
    while parents[out[-1]] >= 0:
        out.append(parents[out[-1]])
    return out[::-1]


def tree_conv_silu(x, pool, weight, slots, rows):
    """rows: (offset, parents, commits) each. Returns (out float64 [T, C], zeros where no row is; magnitudes of the sums;
    pool')."""
    x = np.asarray(x, np.float64)
    w = np.asarray(weight, np.float64).reshape(x.shape[1], -1)
    taps = w.shape[1]
    out, size = np.zeros(x.shape), np.zeros(x.shape)
    pool2 = np.array(pool, copy=True)
    for s, (off, parents, done) in zip(slots, rows):
        for i in range(len(parents)):
            ext = np.concatenate([np.asarray(pool[s], np.float64), x[[off + j for j in path(parents, i)]]])[-taps:]
            acc = (ext * w.T).sum(0)
            out[off + i] = silu(acc)
            size[off + i] = (np.abs(ext) * np.abs(w.T)).sum(0)
        if done:
            pool2[s] = np.concatenate([np.asarray(pool[s]), np.asarray(x[off:off + done], pool2.dtype)])[-(taps - 1):]
    return out, size, pool2


def gdn_tree_step(packed, heads, value_heads, a, b, A_log, dt_bias, state, slots, rows, scale=None):
    """The recurrence from each node's parent's state: (o [T, HV, V], its magnitudes, state', its magnitudes)."""
    packed = np.asarray(packed, np.float64)
    H, HV = heads, value_heads
    K, V = state.shape[2:]
    scale = K ** -0.5 if scale is None else scale
    kh = np.arange(HV) // (HV // H)
    T = len(packed)
    q = l2norm(packed[:, :H * K].reshape(T, H, K)[:, kh]) * scale
    k = l2norm(packed[:, H * K:2 * H * K].reshape(T, H, K)[:, kh])
    v = packed[:, 2 * H * K:].reshape(T, HV, V)
    g, beta = gates(a, b, A_log, dt_bias)
    o, osize = np.zeros((T, HV, V)), np.zeros((T, HV, V))
    st = np.array(state, np.float64, copy=True)
    ssize = np.abs(st)
    for s, (off, parents, done) in zip(slots, rows):
        S0 = np.asarray(state[s], np.float64)
        after = {-1: (S0, np.abs(S0))}
        for i, p in enumerate(parents):
            t = off + i
            e = np.exp(g[t])[:, None, None]
            S, M = after[p][0] * e, after[p][1] * e
            u = beta[t][:, None] * (v[t] - np.matmul(k[t][:, None], S)[:, 0])
            us = beta[t][:, None] * (np.abs(v[t]) + np.matmul(np.abs(k[t])[:, None], M)[:, 0])
            S = S + k[t][:, :, None] * u[:, None]
            M = M + np.abs(k[t])[:, :, None] * us[:, None]
            o[t] = np.matmul(q[t][:, None], S)[:, 0]
            osize[t] = np.matmul(np.abs(q[t])[:, None], M)[:, 0]
            after[i] = (S, M)
        if done:
            st[s], ssize[s] = after[done - 1]
    return o, osize, st, ssize


def gated(o, osize, z, w, eps):
    """out = w o rsqrt(mean o^2 + eps) silu(z) over the last dim, and what an error of up to 1 x osize in o does to it."""
    r = 1.0 / np.sqrt((o * o).mean(-1, keepdims=True) + eps)
    f = np.asarray(w, np.float64) * silu(z)
    norm = np.sqrt((osize * osize).mean(-1, keepdims=True))
    return o * r * f, np.abs(r * f) * osize + np.abs(o * r * f) * r * norm


def tree_attention(q, ring_k, ring_v, new_k, value, ring_pos, slots, starts, rows, scale, window):
    """q [T, Hq, D], new_k, value [T, Hkv, D]: (o [T, Hq, D], sum p |v|, the largest |q||k| scale among the seen keys
    [T, Hq], ring_k', ring_v')."""
    T, hq, D = q.shape
    hkv = new_k.shape[1]
    G = hq // hkv
    o, size, reach = np.zeros((T, hq, D)), np.zeros((T, hq, D)), np.zeros((T, hq))
    rk, rv = np.array(ring_k, copy=True), np.array(ring_v, copy=True)
    for n, (s, (off, parents, done)) in enumerate(zip(slots, rows)):
        start = int(starts[n])
        for i in range(len(parents)):
            way = path(parents, i)
            here = start + len(way) - 1
            cols = [c for c in range(window) if 0 <= ring_pos[s, c] < start and ring_pos[s, c] > here - window]
            toks = [off + j for d, j in enumerate(way) if start + d > here - window]
            for h in range(hkv):
                keys = np.concatenate([ring_k[s, h, cols], new_k[toks, h]]).astype(np.float64)
                vals = np.concatenate([ring_v[s, h, cols], value[toks, h]]).astype(np.float64)
                for j in range(h * G, h * G + G):
                    x = keys @ q[off + i, j].astype(np.float64) * scale
                    e = np.exp(x - x.max())
                    e /= e.sum()
                    o[off + i, j] = e @ vals
                    size[off + i, j] = e @ np.abs(vals)
                    reach[off + i, j] = (np.abs(keys) @ np.abs(q[off + i, j].astype(np.float64))).max() * abs(scale)
        for j in range(max(0, done - window), done):
            rk[s, :, (start + j) % window] = new_k[off + j]
            rv[s, :, (start + j) % window] = value[off + j]
    return o, size, reach, rk, rv


def gate(o, g):
    return o * sigmoid(np.asarray(g, np.float64))
