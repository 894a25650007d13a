"""A session whose history holds a NaN: its own results by definition, and the time of the call, for which every other session
of the call waits.

Times. A row with a result that is not finite is computed again by one workgroup, on one compute unit, which moves 20 GB/s at
the very least: 64 nodes of 4 heads read 128 x 576 keys and values of 512 bytes each, 75 MB, twice over for the two workgroups
that a unit may hold: 8 ms. A row of the gated-delta step takes its nodes in turn: 64 KB of state each, 3 us
at that rate, and 63 ancestors of 0.6 us at most, 41 us a node and 3 ms for 64."""
import numpy as np
import pytest
import torch

from oracle import tree
from test_tree_gpu import KD, attention_call, attention_inputs, attention_oracle, batch, gdn_call, gdn_inputs, gdn_oracle
from test_tree_gpu import maps_of, within

pytestmark = pytest.mark.gpu
D = 256


def least_ms(call, times=5):
    call()
    torch.cuda.synchronize()
    got = []
    for _ in range(times):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        got.append(a.elapsed_time(b))
    return min(got)


@pytest.mark.parametrize("n,hkv,G,W", [(1, 1, 1, 32), (5, 2, 3, 64), (11, 1, 4, 512), (33, 1, 3, 512), (64, 1, 16, 512)])
@pytest.mark.parametrize("rows_n", [1, 70])
def test_attention_over_a_ring_with_a_nan(n, hkv, G, W, rows_n):
    """One dim of one key's value is a NaN in one session's ring: that dim of the queries that see it, and no other result."""
    lens = [n] + np.random.default_rng(n).integers(0, n + 1, rows_n - 1).tolist()
    rows, slots, starts, pool_rows, dev = batch(n + rows_n, lens, False)
    starts[0] = 2 * W + 7
    dev["starts"][0] = starts[0]
    s = attention_inputs(n, sum(lens), pool_rows, slots, starts, hkv, G, W)
    want, slack, _, _ = attention_oracle(s, slots, starts, rows, W, 0.0625)
    last = starts[0] - 1                     # the session's newest key: every query at a depth below W - 1 sees it
    s["ring_v"][slots[0], 0, last % W, 9] = float("nan")
    depth = maps_of(dev, 64).pos[:n].cpu().numpy() - starts[0]
    for most in sorted({n, 64}):
        for kw in ({}, {"workspace": torch.empty(0, dtype=torch.uint8, device="cuda")}):
            out = attention_call(s, dev, maps_of(dev, most), W, 0.0625, **kw)
            hit = torch.zeros(out.shape, dtype=torch.bool)
            for i in range(n):
                if depth[i] < W - 1:
                    hit[i].view(hkv * G, D)[:G, 9] = True
            hit = hit.cuda()
            assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit]).all()
            fixed = out.double().cpu().numpy()
            at = hit.cpu().numpy()
            fixed[at] = want[at]
            within(fixed, want, slack, 2.0 ** -8, f"bound {most}")


@pytest.mark.parametrize("n", [1, 16, 64])
def test_attention_takes_no_other_session_with_it(n):
    lens, hkv, G, W = [n] * 128, 4, 4, 512
    rows, slots, starts, pool_rows, dev = batch(5, lens, False)
    starts = [900] * 128
    dev["starts"].fill_(900)
    s = attention_inputs(5, n * 128, pool_rows, slots, starts, hkv, G, W)
    s["ring_v"][slots[3], :, :, 7] = float("nan")
    trees = maps_of(dev, n)
    assert least_ms(lambda: attention_call(s, dev, trees, W, 0.0625)) < 8.0


@pytest.mark.parametrize("n", [1, 2, 13, 16, 17, 40, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("commit", [False, True])
@pytest.mark.parametrize("gate", [False, True])
def test_gdn_rows_computed_again(n, dtype, commit, gate):
    """The last node's value holds a NaN, which no other node sees: the row is walked, and everything else is as without it,
    the state of a committed chain that ends before it too."""
    H, HV = 2, 4
    rows, slots, _, pool_rows, dev = batch(n, [n, n], commit)
    rows = [(at, p[:-1] + [min(0, n - 2)], min(done, n - 1)) for at, p, done in rows]   # the last hangs on the root
    dev["parents"] = torch.tensor([p for _, ps, _ in rows for p in ps], device="cuda")
    if commit:
        dev["commits"] = torch.tensor([done for _, _, done in rows], device="cuda")
    s = gdn_inputs(n, 2 * n, pool_rows, H, HV, dtype)
    o, osize, st, ssize = gdn_oracle(s, H, HV, slots, rows)
    if gate:
        o, osize = tree.gated(o, osize, s["z"].double().cpu().numpy().reshape(o.shape), s["norm_weight"].double().cpu().numpy(),
                              1e-6)
    s["packed"][n - 1, 2 * H * KD + KD + 7] = float("nan")     # value head 1
    for most in sorted({n, 64}):
        state = s["state"].clone()
        out = gdn_call(s, H, HV, dev["slots"], maps_of(dev, most), state, gate).reshape(o.shape)
        bad = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
        bad[n - 1, 1] = True if gate else torch.arange(KD, device="cuda") == 7
        assert torch.isnan(out[bad]).all()
        got = torch.where(bad, torch.tensor(o).cuda(), out.double())
        within(got, o, 2.0 ** -15 * osize, 2.0 ** -8, f"out, bound {most}")
        # (below 2^-14 fp16's values are 2^-24 apart, so that a rounding moves them by up to 2^-25, more than 2^-11 of themselves)
        least, step = (0.0, 0.0) if dtype is torch.float32 else (2.0 ** -25, 2.0 ** -11)
        within(state, st, 2.0 ** -15 * ssize + least, step, "state")
        idle = [x for x in range(pool_rows) if x not in [a for a, r in zip(slots, rows) if r[2]]]
        assert torch.equal(state[idle], s["state"][idle])


@pytest.mark.parametrize("n", [16, 64])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gdn_takes_no_other_session_with_it(n, dtype):
    H = HV = 16
    rows, slots, _, pool_rows, dev = batch(3, [n] * 16, False)
    dev["parents"] = torch.arange(-1, n - 1, device="cuda").repeat(16)
    s = gdn_inputs(3, n * 16, pool_rows, H, HV, dtype)
    s["state"][slots[2], :, 3, 5] = float("nan")
    trees = maps_of(dev, n)
    assert least_ms(lambda: gdn_call(s, H, HV, dev["slots"], trees, s["state"])) < 3.0
