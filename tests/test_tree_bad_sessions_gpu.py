"""A session whose history holds a NaN: its own results by definition, and the time of the call, for which every other session
of the call waits.

Times. A row with a result that is not finite is computed again by one workgroup, on one compute unit, which moves 20 GB/s at
the very least: 64 nodes of 4 heads read 128 x 576 keys and values of 512 bytes each, 75 MB, twice over for the two workgroups
that a unit may hold: 8 ms."""
import numpy as np
import pytest
import torch

from test_tree_gpu import attention_call, attention_inputs, attention_oracle, batch, maps_of, within

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
