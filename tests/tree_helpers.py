"""Bars and inputs of the tree gated-delta step's precision tests.

A result that is computed in fp32 and rounded once to fewer digits is off by at most half a step of its type, and by what the
fp32 arithmetic left before it. An fp32 recurrence adds a few roundings of 2^-24 a node, which do not compound: the rule
shrinks what it has (a decay and a projection). A chain of 64 nodes all rounded to one side is off by 64 x 2^-24 = 2^-18 of
its row, as a norm; a single value, at eight times the row's rms error of up to 2^-20, by 2^-17 of the row's rms."""
import numpy as np
import torch

KD = 128
STATE_NORM = 2.0 ** -18
VALUE = 2.0 ** -17
DIGITS = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}
LOWEST = {torch.float32: -126, torch.float16: -14, torch.bfloat16: -126}


def f64(t):
    return t.double().cpu().numpy() if torch.is_tensor(t) else np.asarray(t, np.float64)


def rel_norm(got, want):
    """The largest norm of the error over the norm, over matrices (the last two dims)."""
    got, want = f64(got), f64(want)
    return float((np.linalg.norm(got - want, axis=(-2, -1)) / np.linalg.norm(want, axis=(-2, -1))).max())


def beyond_rounding(got, want, dtype):
    """The largest error beyond half a step of ``dtype``, over the rms of the value's row (the last dim)."""
    got, want = f64(got), f64(want)
    _, e = np.frexp(np.maximum(np.abs(got), np.abs(want)))           # |x| = m 2^e, m in [1/2, 1)
    half = np.ldexp(1.0, np.maximum(e - 1, LOWEST[dtype]) - DIGITS[dtype])
    rms = np.sqrt((want * want).mean(-1, keepdims=True))
    return float(((np.abs(got - want) - half) / rms).max())


def like_keys(seed, n, HV, noise, state_dtype=torch.float32, pool_rows=2):
    """A chain over repetitive text: keys that are one vector and ``noise`` times another for each node, betas of .95 to .999,
    a decay of .1 % a node. One key head."""
    gen = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    packed = randn(n, (2 + HV) * KD)
    packed[:, KD:2 * KD] = randn(KD) + noise * randn(n, KD)
    return {"packed": packed.to(torch.bfloat16), "a": torch.zeros(n, HV, dtype=torch.bfloat16),
            "b": (3 + 4 * torch.rand(n, HV, generator=gen)).to(torch.bfloat16),
            "A_log": torch.zeros(HV, dtype=torch.bfloat16), "dt_bias": torch.full((HV,), -7.0, dtype=torch.bfloat16),
            "state": (0.3 * randn(pool_rows, HV, KD, KD)).to(state_dtype),
            "z": randn(n, HV * KD).to(torch.bfloat16), "norm_weight": torch.ones(KD, dtype=torch.bfloat16)}
