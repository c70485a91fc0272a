"""GPU calls of the paged 8-bit KV cache's operators at the ends of what they
take, against oracle/kv8.py (64 bits) with the tolerances of test_gpu_kv8_more.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from megakernel_amd import kv8
from tests.test_gpu_kv8 import Case, _f64, _hint, _say

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- slopes
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,new,hint", [([100], [40], 64), ([100], [40], 1 << 20), ([100, 33], [1, 2], 64)])
def test_slopes_as_steep_as_fp32_holds(dim, lens, new, hint):
    """Slopes whose products with distances pass fp32's range: falling ones leave a
    row its own position, rising ones the farthest, position 0: a single weight that
    is not zero, so outputs are that position's values but for the weight's division
    by itself and the output's rounding.  Log-sum-exps are finite and no more is
    asked of them: a score is rounded beside the row's reference, which after a first
    step is -slope times a distance of at least 1, 2^94 and more, half a step of
    which (2^70) is beyond every score."""
    _say(f"steep slopes D={dim} {lens} hint {hint}")
    steep = [3.4028234e38, 2.4e38, 2.0 ** 94, 1e20, -3.4028234e38, -2.4e38]
    c = _hint(Case(16, 2, dim, lens, new, seed=dim), hint)
    q, n_q = c.rows(6, torch.bfloat16).cuda(), 6
    out, lse = torch.empty((c.tokens, n_q, dim), dtype=torch.bfloat16, device="cuda"), torch.empty((c.tokens, n_q), device="cuda")
    kv8.attention(c.cache, c.batch, q, out, scores=kv8.Scores(slopes=torch.tensor(steep, device="cuda")), lse=lse)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    for i in range(len(lens)):
        for t in range(c.start[i], c.start[i + 1]):
            p = lens[i] - int(c.start[i + 1]) + t
            for h in range(n_q):
                _, v = c.pool.values(*c.pool.place(c.table[i], p if steep[h] > 0 else 0))
                assert np.all(np.abs(_f64(out[t, h]) - v[h // 3]) <= 2.0 ** -7 * np.abs(v[h // 3])), (t, h)


@pytest.mark.parametrize("slope", [2.4e38, 3.4028234e38])
def test_weights_under_steep_slopes_are_finite(slope):
    """One step, whose own position is seen, so its reference is a score: with lse
    from the 64-bit definition, the row's own score, all weight is its own."""
    _say(f"weights under slopes of {slope}")
    for new in (1, 40):  # a wave for all rows, workgroups for many
        c = Case(16, 1, 64, [60], [new], seed=3)
        q = c.rows(1, torch.bfloat16)
        own = [c.pool.values(*c.pool.place(c.table[0], 60 - new + t))[0][0] @ _f64(q[t, 0]) * 0.125 for t in range(new)]
        mass = torch.zeros((1, 1, 64), device="cuda")
        kv8.weigh(c.cache, c.batch, q.cuda(), torch.tensor(own, device="cuda").float()[:, None].contiguous(), mass,
                  scores=kv8.Scores(slopes=torch.tensor([slope], device="cuda")))
        torch.cuda.synchronize()
        want = np.zeros(64)
        want[60 - new : 60] = 1.0
        # (67 + 8) u of scores and their references of at most 40
        np.testing.assert_allclose(_f64(mass[0, 0]), want, rtol=75 * 40 * 2.0 ** -24)


def test_a_slope_that_is_nan_reaches_its_own_head_alone():
    _say("NaN slope")
    c = Case(16, 2, 64, [100], [3], seed=5)
    q, out = c.rows(4, torch.bfloat16).cuda(), torch.empty((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    kv8.attention(c.cache, c.batch, q, out, scores=kv8.Scores(slopes=torch.tensor([0.5, float("nan"), 0.25, 0.0], device="cuda")))
    torch.cuda.synchronize()
    assert torch.isnan(out[:, 1]).all() and torch.isfinite(out[:, [0, 2, 3]]).all()
