"""GPU calls of the paged 8-bit KV cache's operators at the ends of what they
take, against oracle/kv8.py (64 bits) with the tolerances of test_gpu_kv8_more.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from megakernel_amd import kv8
from oracle import kv8 as okv8
from tests.test_gpu_kv8 import Case, _f64, _hint, _say

pytestmark = pytest.mark.gpu


def _one_hot(c, n_q, size):
    """Queries of one dimension each, so that a score is one product, exact in fp32."""
    q = np.zeros((c.tokens, n_q, c.dim))
    d = c.rng.integers(0, c.dim, (c.tokens, n_q, 1))
    np.put_along_axis(q, d, size * c.rng.standard_normal((c.tokens, n_q, 1)), 2)
    return torch.from_numpy(q).to(torch.bfloat16)


# ------------------------------------------------------------------- slopes
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,new,hint", [([100], [40], 64), ([100], [40], 1 << 20), ([100, 33], [1, 2], 64)])
def test_slopes_as_steep_as_fp32_holds(dim, lens, new, hint):
    """Slopes whose products with distances pass fp32's range: falling ones leave a
    row its own position, rising ones the farthest, position 0: a single weight that
    is not zero, so outputs are that position's values but for the weight's division
    by itself and the output's rounding.  Log-sum-exps of falling ones are its score, a
    sum of D products (with the scale's roundings (D + 3) u of their magnitudes), to
    base 2 and back (8 u)."""
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
                k, v = c.pool.values(*c.pool.place(c.table[i], p if steep[h] > 0 else 0))
                assert np.all(np.abs(_f64(out[t, h]) - v[h // 3]) <= 2.0 ** -7 * np.abs(v[h // 3])), (t, h)
                s, reach = (f(k[h // 3]) @ f(_f64(q[t, h])) * dim ** -0.5 for f in (np.asarray, np.abs))
                assert steep[h] < 0 or abs(float(lse[t, h]) - s) <= 2.0 ** -24 * ((dim + 3) * reach + 8 * abs(s)), (t, h)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,new,hint", [([700, 1999], [1, 3], 2000), ([700], [60], 1 << 20), ([1300], [1], 1 << 20)])
def test_biased_scores_keep_what_near_ones_are(dim, lens, new, hint):
    """Log-sum-exps of rows whose first steps lie far away.  A raw score is one product
    (13 u of it as in the test of caps), a bias and its sums 4 u of it, each position's by its weight;
    of positions with a weight above fp32's smallest, 104 / slope and less, sums (u
    each) and the logarithm (20 u), and 4 u |lse|."""
    _say(f"near scores under slopes D={dim} {lens} hint {hint}")
    slopes = [0.7, 3.0, 20.0, 0.3, 150.0, 1e4]
    c = _hint(Case(32, 2, dim, lens, new, seed=dim), hint)
    q, n_q, u = _one_hot(c, 6, 1.0), 6, 2.0 ** -24
    out, lse = torch.empty((c.tokens, n_q, dim), dtype=torch.bfloat16, device="cuda"), torch.empty((c.tokens, n_q), device="cuda")
    kv8.attention(c.cache, c.batch, q.cuda(), out, scale=1.0, scores=kv8.Scores(slopes=torch.tensor(slopes, device="cuda")), lse=lse)
    torch.cuda.synchronize()
    got = _f64(lse)
    for i, t, h, j, s, w, v, reach, bias in okv8.scored_rows(c.pool, c.table, c.start, c.lens, _f64(q), 1.0, okv8.Scores(slopes=slopes)):
        far = slopes[h] * np.abs(j - (int(c.lens[i]) - int(c.start[i + 1]) + t))
        ref = s.max() + np.log(np.exp(s - s.max()).sum())
        tol = u * (13 * (w @ np.abs(s + far)) + 4 * (w @ far) + min(len(j), 104 / slopes[h] + 2) + 20 + 4 * abs(ref))
        assert abs(got[t, h] - ref) <= tol, (i, h, got[t, h], ref, tol)


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


# ------------------------------------------------------------ after eviction
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 32)])
def test_rows_after_a_compaction_stand_behind_the_kept_ones(dim, block):
    """As the usage has it: lengths are kept_len plus the new rows.  Kept rows, their
    weights and the recent positions among them stay as compaction left them; new
    rows are attended to with them and start from no weight."""
    _say(f"rows after a compaction D={dim} block {block}")
    n_kv, n_q, keep, recent = 2, 4, 40, 8
    c = Case(block, n_kv, dim, [100, 61, 12], [100, 61, 12], seed=dim + block, extra=3 * (96 // block) + 3)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    used = {int(b) for b in c.table.ravel()}
    free = [b for b in range(c.pool.n_blocks) if b not in used]
    width = 96 // block
    new_table = i32(free[: 3 * width]).view(3, width).contiguous()
    mass, new_mass = torch.rand((3, n_kv, c.table.shape[1] * block), device="cuda"), torch.full((3, n_kv, 96), 5.0, device="cuda")
    kept, kept_len = torch.empty((3, n_kv, keep), dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    kv8.select(c.cache, c.batch, mass, kept, kept_len, recent=recent)
    kv8.compact(c.cache, c.batch, kept, kept_len, new_table, mass, new_mass)
    assert kept_len.tolist() == [40, 40, 12] and kept[0, :, -recent:].tolist() == [list(range(92, 100))] * n_kv

    def rows():  # what the cache holds of the kept rows
        start = torch.cat([i32([0]), kept_len.cumsum(0, dtype=torch.int32)])
        k, v = (torch.empty((92, n_kv, dim), device="cuda") for _ in range(2))
        kv8.read(c.cache, kv8.Batch(new_table, start, kept_len, 92), k, v)
        return torch.cat([k, v])

    before, weights = rows(), new_mass.clone()
    new = [1, 20, 0]
    q_start = i32([0, 1, 21, 21])
    kv_len = kept_len + (q_start[1:] - q_start[:-1])
    batch = kv8.Batch(new_table, q_start, kv_len, 21)
    k, v = 0.1 * c.rng.standard_normal((2, 21, n_kv, dim))  # smaller than what is there: no scale grows
    kv8.append(c.cache, batch, *(torch.from_numpy(x).to(torch.bfloat16).cuda() * 2.0 ** -8 for x in (k, v)))
    q, out = torch.from_numpy(c.rng.standard_normal((21, n_q, dim))).to(torch.bfloat16).cuda(), torch.empty((21, n_q, dim), dtype=torch.bfloat16, device="cuda")
    lse = torch.empty((21, n_q), device="cuda")
    kv8.attention(c.cache, batch, q, out, lse=lse)
    kv8.weigh(c.cache, batch, q, lse, new_mass)
    torch.cuda.synchronize()
    assert torch.equal(rows(), before)
    for i, (n, had) in enumerate(zip(new, kept_len.tolist())):
        gained = (new_mass[i, :, : had + n] - torch.nn.functional.pad(weights[i, :, :had], (0, n))).double()
        # each of a row's two heads gives 1 in all, off by 1e-5 of itself at most; new positions began at none
        assert torch.all(gained >= -1e-5) and torch.all((gained.sum(-1) - 2 * n).abs() <= 1e-3), i
        assert torch.all(new_mass[i, :, had + n :] == 5.0)


# --------------------------------------------------------------------- caps
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cap,size,of_cap", [(50.0, 0.25, 0), (1024.0, 1.0, 0), (1024.0, 0.01, 0), (2.0 ** -30, 2.0 ** -38, 0), (3.0, 3.0, 2), (40.0, 40.0, 2)])
@pytest.mark.parametrize("hint", [64, 1 << 20])
def test_capped_scores_keep_what_small_ones_are(dim, cap, size, of_cap, hint):
    """Log-sum-exps and weights of one to four positions.  A score is one product: its
    scale and quotient by the cap 3 u of it, the polynomial 8 u, the sum with the
    reference 2 u; where some score passes half the cap, 2 u of the cap besides
    (of_cap).  Sums of at most four weights and the logarithm: 20 u, and 4 u |lse|."""
    _say(f"small scores under a cap of {cap} D={dim} hint {hint}")
    rng = np.random.default_rng(int(cap) + dim)
    lens = [1, 2, 3, 4] * 8 + [int(v) for v in rng.integers(1, 5, 30)]
    c = _hint(Case(16, 2, dim, lens, [1] * len(lens), seed=dim), hint)
    c.pool.ks[:] = 2.0 ** -1
    c.upload()
    q, n_q, u = _one_hot(c, 4, size), 4, 2.0 ** -24
    x = okv8.Scores(softcap=cap)
    given, qc = kv8.Scores(softcap=cap), q.cuda()
    out, lse = torch.empty((c.tokens, n_q, dim), dtype=torch.bfloat16, device="cuda"), torch.empty((c.tokens, n_q), device="cuda")
    mass = torch.zeros((len(lens), 2, c.table.shape[1] * 16), device="cuda")
    kv8.attention(c.cache, c.batch, qc, out, scale=1.0, scores=given, lse=lse)
    for _ in range(4):  # older positions gather, the row's own starts anew
        kv8.weigh(c.cache, c.batch, qc, lse, mass, scale=1.0, scores=given)
    torch.cuda.synchronize()
    got, want_mass, tol_mass = _f64(lse), np.zeros(mass.shape), np.zeros(mass.shape)
    largest = 0.0
    for i, t, h, j, s, w, v, reach, bias in okv8.scored_rows(c.pool, c.table, c.start, c.lens, _f64(q), 1.0, x):
        largest = max(largest, np.abs(s).max() / cap)
        e = 13 * u * np.abs(s).max() + of_cap * u * cap
        ref = s.max() + np.log(np.exp(s - s.max()).sum())
        assert abs(got[t, h] - ref) <= e + 20 * u + 4 * u * abs(ref), (i, h, got[t, h], ref)
        times = np.where(j == c.lens[i] - 1, 1, 4)
        want_mass[i, h // 2, j] += times * w
        tol_mass[i, h // 2, j] += times * w * (2 * e + 40 * u + 8 * u * (np.abs(s) + abs(ref)) + 40 * u)
    assert (largest > 0.5) == (of_cap > 0)
    assert np.all(np.abs(_f64(mass) - want_mass) <= tol_mass)


def test_scores_far_beyond_a_cap():
    """Scores of up to fp32's infinity are the cap, NaN stays NaN, in one step."""
    _say("scores beyond a cap")
    c = Case(16, 1, 64, [16, 16], [1, 1], seed=2)
    c.pool.ks[:] = 2.0 ** 119
    b = [int(v) for v in c.table[:, 0]]
    c.pool.k[b[0], 0] = 0
    c.pool.k[b[0], 0, :, 0] = [0x7E, 0xFE] * 8     # +-448, the largest
    c.pool.k[b[1], 0] = c.pool.k[b[0], 0]
    c.pool.k[b[1], 0, 5, 1] = 0x7F                 # a NaN, times zero or not
    c.pool.ks[b[1]] = 2.0 ** 3
    c.upload()
    q = torch.zeros((2, 1, 64), dtype=torch.bfloat16, device="cuda")
    q[:, 0, 0] = 1e6                               # 448 * 2^119 * 1e6 is infinite
    out, lse = torch.empty_like(q), torch.empty((2, 1), device="cuda")
    for cap in (5.0, 1000.0):
        kv8.attention(c.cache, c.batch, q, out, scale=1.0, scores=kv8.Scores(softcap=cap), lse=lse)
        torch.cuda.synchronize()
        assert abs(float(lse[0, 0]) - (cap + np.log(8 + 8 * np.exp(-2 * cap)))) <= 2.0 ** -24 * (8 * cap + 40)
        want = np.mean([c.pool.values(b[0], p)[1][0] for p in range(0, 16, 2)], axis=0)
        low = np.mean([np.abs(c.pool.values(b[0], p)[1][0]) for p in range(16)], axis=0)
        assert np.all(np.abs(_f64(out[0, 0]) - want) <= 2.0 ** -6 * low + 8 * np.exp(-2 * cap) * low)
        assert torch.isnan(lse[1, 0]) and torch.isnan(out[1, 0]).all()
