"""GPU parity of rotary positions, attention with scores, gathered weights and
eviction over the paged 8-bit KV cache with oracle/kv8.py (64 bits).

Tolerances; u = 2^-24, half a step of fp32, h half a step of the output's type
(2^-8 bf16, u fp32).  What selects, moves or counts is exact.
  rotary: |y| h + 10 u A (|a| + |b|) for a pair (a, b): the angle's fraction of a
    turn and its sine (5 u), the amplitude A (1 u), the rotation (3 u), one to spare.
  a score, e in units of its own: D products with sum |q k| scale <= reach
    summed in fp32 (D u reach); the scale and its product (3 u reach); with a cap C
    10 u C: t = e^2y is off by (6 |y| + 2) u of itself, 1 / (t + 1) by t / (t + 1) of
    that and 3 u, which 2 C / (t + 1) turns into at most 9.4 u C, and the last sum
    rounds (u C); with slopes the slope to base 2, its product and the sum
    (4 u bias); the sum with the reference (3 u |s|).
  attention: |o| h + (2^-8 + 2 e + (n + 16) u) sum_j p_j |v_j| + n 2^-126 * 448 vs: weights
    rounded to bf16; e enters the weight and the sum; n positions summed in fp32;
    exponentials and divisions; weights beside the largest below 2^-126 may be zero.
  log-sum-exp: e + (n + 16) u + 4 u |lse| + n 2^-126.
  gathered weights, of each p: 2 e, the log-sum-exp's own tolerance, its product and
    the sum to the exponent (4 u (|s| + |lse|)), the exponential (4 u); of their sum
    over R rows and what was there before (R + 32) u; 2^-126 each.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from megakernel_amd import _lib, kv8
from oracle import kv8 as okv8
from tests.test_gpu_kv8 import HALF, U, Case, _f64, _hint, _say

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -126


# ------------------------------------------------------------------- rotary
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                     (torch.float32, torch.float32)])
@pytest.mark.parametrize("tokens,n_q,n_kv,dim,turned,layout", [
    (1, 16, 8, 64, 64, "packed"), (37, 5, 1, 128, 32, "packed"), (700, 4, 2, 128, 64, "in place"), (300, 3, 3, 64, 16, "heads"),
    (19, 2, 1, 80, 20, "packed"), (33, 3, 2, 96, 96, "in place"), (5, 1, 1, 2, 2, "packed"), (3, 2, 1, 1024, 1024, "packed"),
    (21, 2, 2, 6, 4, "in place"), (65, 2, 2, 64, 64, "odd"), (600, 7, 1, 256, 128, "packed"), (1, 1, 1, 1024, 2, "heads")])
def test_rotary(tokens, n_q, n_kv, dim, turned, layout, src, dst, interleaved):
    if layout == "in place":
        dst = src
    _say(f"rotary T={tokens} {n_q}/{n_kv} D={dim} turned {turned} {layout} {src} -> {dst} interleaved {interleaved}")
    g = torch.Generator().manual_seed(tokens * dim + turned)
    x = torch.randn((tokens, n_q + 2 * n_kv, dim), generator=g) * 3
    if layout == "odd":  # rows that lie on no 16 bytes
        wide = torch.zeros((tokens, n_q + 2 * n_kv, dim + 1)).to(src).cuda()
        wide[..., 1:] = x.to(src).cuda()
        x = wide[..., 1:]
    else:
        x = x.to(src).cuda()
    inv = torch.tensor([1e4 ** (-2 * i / turned) for i in range(turned // 2)], dtype=torch.float32).cuda()
    pos = torch.randint(-1000, 200000, (tokens,), generator=g, dtype=torch.int32)
    if tokens > 2:
        pos[:3] = torch.tensor([0, 2 ** 31 - 1, -2 ** 31])
    pos, amp = pos.cuda(), 1.25
    q, k = x[:, :n_q], x[:, n_q : n_q + n_kv]
    want = [okv8.rotary(_f64(r), _f64(inv), pos.cpu().numpy(), interleaved, amp) for r in (q, k)]
    raw, rest = [r.clone() for r in (q, k)], x[:, n_q + n_kv :].clone()
    if layout == "in place":
        outs = [q, k]
    elif layout == "heads":
        outs = [torch.full((h, tokens, dim), float("nan"), dtype=dst, device="cuda").transpose(0, 1) for h in (n_q, n_kv)]
    else:
        outs = [torch.full((tokens, h, dim), float("nan"), dtype=dst, device="cuda") for h in (n_q, n_kv)]
    kv8.rotary(q, k, inv, pos, *outs, interleaved=interleaved, amplitude=amp)
    torch.cuda.synchronize()
    for got, (y, size), was in zip(outs, want, raw):
        assert torch.equal(got[..., turned:], was[..., turned:].to(dst))  # what is not turned is copied
        err, tol = np.abs(_f64(got) - y)[..., :turned], (np.abs(y) * HALF[dst] + 10 * U * amp * size)[..., :turned]
        assert np.all(err <= tol), f"worst {np.max(err / np.maximum(tol, 1e-30)):.2f} of the tolerance"
    assert torch.equal(x[:, n_q + n_kv :], rest)


def test_rotary_of_whole_heads_is_the_rotation_of_qk_norm_rope():
    """Rows whose mean square is 1 and gains of 1: the norm changes them by rounding alone."""
    _say("rotary and qk_norm_rope")
    x = torch.where(torch.rand((40, 3, 128), generator=torch.Generator().manual_seed(1)) < 0.5, -1.0, 1.0).cuda()
    inv, _ = kv8.rotary_frequencies(128)
    pos, one = torch.arange(900, 940, dtype=torch.int32, device="cuda"), torch.ones(128, dtype=torch.bfloat16, device="cuda")
    a, b = (torch.empty_like(x) for _ in range(2))
    kv8.rotary(x[:, :2], x[:, 2:], inv, pos, a[:, :2], a[:, 2:])
    kv8.qk_norm_rope(x[:, :2], x[:, 2:], one, one, inv, pos, b[:, :2], b[:, 2:], eps=0.0)
    torch.cuda.synchronize()
    assert (a - b).abs().max().item() <= 2.0 ** -20


# ------------------------------------------------- attention with scores, weights
def _given(x: okv8.Scores):
    """The same as kv8.Scores."""
    up = lambda v, t: None if v is None else torch.tensor(np.asarray(v), dtype=t, device="cuda")
    return kv8.Scores(x.softcap, up(x.slopes, torch.float32), x.window, up(x.first, torch.int32), up(x.prefix, torch.int32))


def _check(c: Case, n_q, x: okv8.Scores, q=None, nan_ok=False, scale=None, tokens=None, mass=True, say=""):
    """attention() with and without a log-sum-exp, and weigh(), against the
    oracle; of `tokens` alone where given (and no weights)."""
    q = c.rows(n_q, torch.bfloat16, 1.5) if q is None else q
    sc, given = c.dim ** -0.5 if scale is None else scale, _given(x)
    out, plain = (torch.full((c.tokens, n_q, c.dim), 5.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    lse = torch.full((c.tokens, n_q), 7.0, device="cuda")
    qc = q.cuda()
    kv8.attention(c.cache, c.batch, qc, plain, scale=scale, scores=given)
    kv8.attention(c.cache, c.batch, qc, out, scale=scale, scores=given, lse=lse)
    n_seq, width = c.table.shape
    old = c.rng.random((n_seq, c.n_kv, width * c.block + 3)) * 4
    held = torch.from_numpy(old).float().cuda()
    if mass:
        kv8.weigh(c.cache, c.batch, qc, lse, held, scale=scale, scores=given)
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(out.float(), nan=9.0), torch.nan_to_num(plain.float(), nan=9.0))
    n = int(max(list(c.lens) + [1]))
    want, tol = np.full((c.tokens, n_q, c.dim), 5.0), np.zeros((c.tokens, n_q, c.dim))
    want_lse, tol_lse = np.full((c.tokens, n_q), 7.0), np.zeros((c.tokens, n_q))
    old = held_before = torch.from_numpy(old).float().double().numpy()
    want_mass, tol_mass = held_before.copy(), np.zeros_like(old)
    group = n_q // c.n_kv
    for i in range(n_seq):
        rows, length = int(c.start[i + 1] - c.start[i]), min(max(int(c.lens[i]), 0), width * c.block)
        if rows:
            want_mass[i, :, max(0, int(c.lens[i]) - rows) : length] = 0.0
            tol_mass[i, :, :length] = (rows * group + 32) * U * np.abs(want_mass[i, :, :length])
    with np.errstate(invalid="ignore"):
        for i, t, h, j, s, w, v, reach, bias in okv8.scored_rows(c.pool, c.table, c.start, c.lens, _f64(q), sc, x, tokens):
            if j is None:
                want[t, h], want_lse[t, h] = 0.0, -np.inf
                continue
            e = (c.dim + 3) * U * reach + 10 * U * x.softcap + 4 * U * bias + 3 * U * np.abs(s).max()
            want[t, h] = w @ v
            tol[t, h] = np.abs(want[t, h]) * 2.0 ** -8 + (2.0 ** -8 + 2 * e + (n + 16) * U) * (w @ np.abs(v)) + n * TINY * 448 * np.nanmax(c.pool.vs)
            ref = s.max() + np.log(np.exp(s - s.max()).sum())
            want_lse[t, h] = ref
            tol_lse[t, h] = e + (n + 16) * U + 4 * U * abs(ref) + n * TINY
            rows = int(c.start[i + 1] - c.start[i]) * group
            want_mass[i, h // group, j] += w
            tol_mass[i, h // group, j] += w * (2 * e + tol_lse[t, h] + 4 * U * (np.abs(s) + abs(ref)) + (rows + 36) * U) + TINY
    some = np.ones(c.tokens, bool) if tokens is None else np.isin(np.arange(c.tokens), list(tokens))
    checks = [("out", _f64(out)[some], want[some], tol[some]), ("lse", _f64(lse)[some], want_lse[some], tol_lse[some])]
    if mass and tokens is None:
        checks.append(("mass", _f64(held), want_mass, tol_mass))
    for name, got, ref, t in checks:
        with np.errstate(invalid="ignore"):
            bad = ~((np.abs(got - ref) <= t) | (got == ref))
        if nan_ok:
            np.testing.assert_array_equal(np.isnan(got), np.isnan(ref), err_msg=name)
            bad &= ~np.isnan(ref)
        assert not bad.any(), f"{say} {name}: {int(bad.sum())} off, first at {np.argwhere(bad)[:1]}, {got[bad][:1]} not {ref[bad][:1]} +- {t[bad][:1]}"
    return q, out, lse, held


def _scores_of(kind, c: Case, n_q):
    rng, pos = np.random.default_rng(len(kind)), np.zeros(c.tokens, np.int64)
    for i in range(len(c.lens)):
        n = int(c.start[i + 1] - c.start[i])
        pos[c.start[i] : c.start[i + 1]] = int(c.lens[i]) - n + np.arange(n)
    slopes = [2.0 ** (-8 * (h + 1) / n_q) for h in range(n_q)]
    docs = pos // 37 * 37  # documents of 37 positions
    part = [max(0, int(v)) * 2 // 3 for v in c.lens]
    return {
        "plain": okv8.Scores(),
        "cap": okv8.Scores(softcap=3.0),
        "wide cap": okv8.Scores(softcap=1000.0),
        "slopes": okv8.Scores(slopes=slopes),
        "rising": okv8.Scores(slopes=[-0.01] * n_q),
        "window 1": okv8.Scores(window=1),
        "window 20": okv8.Scores(window=20),
        "window 64": okv8.Scores(window=64),
        "window 129": okv8.Scores(window=129, softcap=20.0),
        "huge window": okv8.Scores(window=2 ** 31 - 1),
        "documents": okv8.Scores(first=docs),
        "nothing": okv8.Scores(first=np.where(rng.random(c.tokens) < 0.4, pos + 1 + rng.integers(0, 900, c.tokens), docs)),
        "any start": okv8.Scores(first=rng.choice([-5, 0, 3, 64, 2 ** 31 - 1, -2 ** 31], c.tokens)),
        "prefix": okv8.Scores(prefix=part),
        "long prefix": okv8.Scores(prefix=[2 ** 31 - 1 if i % 2 else -3 for i in range(len(c.lens))]),
        "all": okv8.Scores(softcap=15.0, slopes=slopes, window=70, first=np.where(pos > 40, 11, 0), prefix=part),
    }[kind]


KINDS = ["plain", "cap", "wide cap", "slopes", "rising", "window 1", "window 20", "window 64", "window 129", "huge window", "documents",
         "nothing", "any start", "prefix", "long prefix", "all"]
FEW = [
    # block, n_kv, group, dim, lens, new
    (16, 2, 2, 64, [1, 64, 65, 0, 200], [1, 1, 1, 0, 1]),
    (32, 1, 5, 128, [70, 129, 300], [1, 2, 9]),
    (128, 1, 20, 64, [130, 40, 400], [2, 1, 3]),
    (64, 2, 3, 128, [250, 66, 3], [33, 1, 3]),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", FEW, ids=[f"b{c[0]}h{c[1]}g{c[2]}d{c[3]}" for c in FEW])
def test_scores_of_few_rows(case, kind):
    block, n_kv, group, dim, lens, new = case
    _say(f"scores {case} {kind}")
    c = Case(block, n_kv, dim, lens, new, seed=block * dim + sum(lens), missing=0.15, gap=1)
    _check(c, n_kv * group, _scores_of(kind, c, n_kv * group))


# announced as long, contexts go to the kernel for many rows, split; with many
# rows times KV heads to the same kernel, whole
TILES = [
    (16, 2, 3, 64, [90, 40, 170], [90, 33, 150], 1 << 20),
    (64, 1, 2, 128, [350, 66, 3], [240, 1, 3], 1 << 20),
    (32, 1, 16, 128, [300, 5, 80], [70, 1, 3], 1 << 20),
    (128, 64, 2, 64, [200, 5], [140, 5], 64),
    (32, 32, 2, 128, [260], [200], 64),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", TILES, ids=[f"b{c[0]}h{c[1]}g{c[2]}d{c[3]}" for c in TILES])
def test_scores_of_many_rows(case, kind):
    block, n_kv, group, dim, lens, new, hint = case
    _say(f"scores of many rows {case} {kind}")
    c = _hint(Case(block, n_kv, dim, lens, new, seed=block * dim + sum(lens), missing=0.1, gap=1), hint)
    _check(c, n_kv * group, _scores_of(kind, c, n_kv * group))


@pytest.mark.parametrize("kind", ["plain", "documents", "all"])
@pytest.mark.parametrize("dim,group,lens,new", [(64, 1, [560], [170]), (64, 3, [640], [60]), (128, 1, [560], [170]), (128, 5, [700], [40]),
                                                (64, 2, [260, 70, 300, 0, 33], [70, 40, 41, 0, 33])])
def test_weights_of_many_steps_and_heads(dim, group, lens, new, kind):
    """Enough steps times KV heads for workgroups of 64 positions, and in the last case for a wave to each."""
    _say(f"weights of many steps D={dim} group {group} {kind}")
    c = Case(16, 64, dim, lens, new, seed=dim + group, missing=0.1, gap=1)
    _check(c, 64 * group, _scores_of(kind, c, 64 * group))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [33, 40, 70])
def test_scores_of_more_heads_than_a_tile_has_rows(dim, group):
    _say(f"scores group {group} D={dim}")
    c = Case(16, 1, dim, [90, 33], [5, 2], seed=group + dim, missing=0.1, gap=1)
    for kind in ("plain", "all"):
        _check(c, group, _scores_of(kind, c, group), say=kind)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,new,hint", [([3000], [1], 0), ([2100, 30, 900], [1, 1, 1], 4096), ([1500], [1], 1500), ([2500], [40], 1 << 20)])
def test_scores_over_split_contexts(dim, lens, new, hint):
    for kind in ("cap", "slopes", "window 129", "prefix"):
        _say(f"scores split D={dim} {lens} hint {hint} {kind}")
        c = _hint(Case(32, 1, dim, lens, new, seed=dim, missing=0.05), hint)
        _check(c, 2, _scores_of(kind, c, 2), say=kind)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hint,n_kv", [(64, 2), (1 << 20, 2), (64, 64)])
def test_scores_never_see_what_they_may_not(dim, hint, n_kv):
    """NaN before a window, before a document, behind a prefix, in a step that
    some rows see, reaches no row that does not see it and every row that does."""
    _say(f"scores NaN D={dim} hint {hint} heads {n_kv}")
    c = _hint(Case(16, n_kv, dim, [150], [100], seed=21), hint)
    b = [int(c.table[0, p // 16]) for p in range(150)]
    c.pool.v[b[70], :, 5, 70 % 16] = 0x7F
    c.pool.v[b[3], 0, 9, 3] = 0xFF
    c.pool.k[b[64], 1, 64 % 16, 7] = 0x7F
    c.upload()
    x = okv8.Scores(window=30, prefix=[60])
    _, out, _, _ = _check(c, n_kv, x, nan_ok=True)
    assert torch.isnan(out[20, 0, 5]) and torch.isnan(out[49, 0, 5]) and not torch.isnan(out[50:, 0]).any()  # 70 is seen from 70 to 99
    assert not torch.isnan(out[:14, 1, 5]).any() and torch.isnan(out[14:44, 1]).all()                       # key 64 from 64 to 93
    _check(c, n_kv, okv8.Scores(first=np.where(np.arange(50, 150) >= 80, 71, 4)), nan_ok=True)


def test_scores_of_pages_of_garbage():
    """A fresh pool holds NaN codes and NaN scales: what is missing or unseen stays out."""
    _say("scores garbage")
    for hint in (64, 1 << 20):
        c = _hint(Case(16, 2, 64, [100], [60], seed=22, fill=False), hint)
        ids = c.table[0]
        for j in range(2, 7):  # positions 32 on hold values
            c.pool.k[ids[j]], c.pool.v[ids[j]] = 0x38, 0x38
            c.pool.ks[ids[j]], c.pool.vs[ids[j]] = 0.5, 0.25
        c.table[0, 3] = -1
        c.upload()
        _check(_hint(c, hint), 4, okv8.Scores(window=8, first=np.full(60, 35)))


def test_scores_at_both_ends():
    """Scores of thousands under a cap, and without one with slopes that leave one key."""
    _say("scores extremes")
    c = Case(32, 2, 64, [150, 80], [1, 20], seed=10)
    c.pool.ks[:] = 2.0 ** 9
    c.upload()
    q = c.rows(4, torch.bfloat16, 3.0)
    _check(c, 4, okv8.Scores(softcap=50.0), q=q, scale=2.0 ** -10)
    _check(c, 4, okv8.Scores(softcap=1024.0), q=q, scale=2.0 ** -10)
    _check(c, 4, okv8.Scores(slopes=[1e4, 100.0, 3.0, 0.0]), q=q, scale=2.0 ** -10)


def test_scores_strides_side_stream_and_a_given_workspace():
    _say("scores strides")
    c = _hint(Case(16, 2, 64, [3060, 9], [5, 4], seed=11), 4096)
    x = okv8.Scores(softcap=9.0, window=2800)
    q, want, lse, mass = _check(c, 4, x)
    given = _given(x)
    wide = torch.zeros((c.tokens, 9, 96), dtype=torch.bfloat16, device="cuda")
    wide[:, 2:6, 16:80] = q.cuda()
    out, got = torch.full((4, c.tokens + 2, 64), 3.0, dtype=torch.bfloat16, device="cuda"), torch.empty_like(lse)
    need = kv8.workspace_bytes(c.cache, c.batch, 4, given, lse=True)
    assert need > kv8.workspace_bytes(c.cache, c.batch, 4, given) > 0
    work = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    # weights of sequences apart, heads before sequences
    n = c.table.shape[1] * 16
    held = torch.full((2, 5, n + 4), -1.0, device="cuda")
    view = held.transpose(0, 1)[1:3]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv8.attention(c.cache, c.batch, wide[:, 2:6, 16:80], out.transpose(0, 1)[: c.tokens], workspace=work, scores=given, lse=got)
        view.zero_()
        kv8.weigh(c.cache, c.batch, wide[:, 2:6, 16:80], got, view, scores=given)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out.transpose(0, 1)[: c.tokens], want) and torch.all(out[:, c.tokens :] == 3.0) and torch.equal(got, lse)
    assert torch.all(held[:, 0] == -1) and torch.all(held[:, 3:] == -1)
    again = torch.zeros((2, 2, n), device="cuda")
    kv8.weigh(c.cache, c.batch, q.cuda(), lse, again, scores=given)
    assert torch.equal(view[..., :n], again)  # the same sums in the same order


def test_more_rows_than_positions_with_scores():
    _say("scores negative positions")
    c = Case(16, 2, 64, [5, 40], [9, 50], seed=8)
    _, out, lse, _ = _check(c, 4, okv8.Scores(prefix=[4, 4], window=7))
    assert torch.all(out[:4] == 0) and torch.all(lse[:4] == -float("inf")) and torch.all(lse[9:19] == -float("inf"))


def test_weights_of_a_row_sum_to_one():
    """One row, fresh positions: what the positions got is that row's softmax."""
    _say("weights sum")
    c = Case(32, 2, 128, [700], [700], seed=30)
    q, out, lse, mass = _check(c, 4, okv8.Scores(), tokens={0, 1, 350, 699}, mass=False)
    held = torch.full((1, 2, c.table.shape[1] * 32), float("nan"), device="cuda")
    kv8.weigh(c.cache, c.batch, q.cuda(), lse, held)
    torch.cuda.synchronize()
    got = held[0, :, :700].double().sum(-1).cpu()
    # 700 rows of two heads, each weight off by 1e-5 of itself at most
    assert torch.all((got - 1400).abs() <= 1400 * 1e-5), got
    assert torch.isnan(held[0, :, 700:]).all()


def test_weights_of_a_hundred_and_fifty_sequences():
    _say("weights of many sequences")
    rng = np.random.default_rng(31)
    lens = [int(v) for v in rng.integers(0, 90, 150)]
    for new in ([min(1, v) for v in lens], [min(v, 40) for v in lens]):
        c = Case(16, 1, 64, lens, new, seed=31)
        _check(c, 2, okv8.Scores(window=50))


# ------------------------------------------------------------------ eviction
def _select(mass, lens, keep, recent, sinks, block=16, hint=0):
    """kept and kept_len of sequences whose table is as wide as mass."""
    n_seq, n_kv, positions = mass.shape
    cache = kv8.Cache.empty(2, n_kv, 64, block)
    table = torch.full((n_seq, positions // block), -1, dtype=torch.int32, device="cuda")
    batch = kv8.Batch(table, torch.zeros(n_seq + 1, dtype=torch.int32, device="cuda"),
                      torch.tensor(lens, dtype=torch.int32, device="cuda"), 0, hint)
    kept = torch.full((n_seq, n_kv, keep), 77, dtype=torch.int32, device="cuda")
    kept_len = torch.full((n_seq,), 77, dtype=torch.int32, device="cuda")
    kv8.select(cache, batch, mass, kept, kept_len, recent=recent, sinks=sinks)
    torch.cuda.synchronize()
    return kept.cpu().numpy(), kept_len.cpu().numpy()


def _masses(rng, kind, shape):
    if kind == "long tail":
        return np.exp(2 * rng.standard_normal(shape)) * (rng.random(shape) > 0.2)
    if kind == "ties":
        return rng.integers(0, 4, shape).astype(float)
    if kind == "equal":
        return np.full(shape, 0.25)
    if kind == "odd":
        return rng.choice([0.0, -0.0, 1.0, -1.0, np.inf, -np.inf, np.nan, 1e-40, -1e-40, 3.4e38], shape)
    return rng.integers(0, 2 ** 32, shape, dtype=np.uint32).view(np.float32)  # every bit pattern


@pytest.mark.parametrize("kind", ["long tail", "ties", "equal", "odd", "bits"])
@pytest.mark.parametrize("lens,keep,recent,sinks", [
    ([0, 1, 5, 6, 63, 64, 65], 6, 2, 1), ([300, 17, 299], 100, 0, 0), ([300, 1000, 999], 250, 128, 4), ([500], 1, 0, 0), ([500], 1, 1, 0),
    ([130, 131], 130, 65, 65), ([4100, 4096, 4097], 1000, 13, 2), ([5000], 4999, 0, 0), ([6000, 5999], 6100, 5, 5)])
def test_select(lens, keep, recent, sinks, kind):
    _say(f"select {lens} keep {keep} {recent}+{sinks} {kind}")
    rng = np.random.default_rng(sum(lens) + keep)
    positions = -(-max(lens + [1]) // 16) * 16
    m = _masses(rng, kind, (len(lens), 2, positions)).astype(np.float32)
    for hint in (0, 64):  # a hint that is far too short changes no result
        kept, kept_len = _select(torch.from_numpy(m).cuda(), lens, keep, recent, sinks, hint=hint)
        for i, n in enumerate(lens):
            assert kept_len[i] == min(n, keep)
            for h in range(2):
                want = okv8.select(m[i, h].tolist(), n, keep, recent, sinks)
                np.testing.assert_array_equal(kept[i, h], want + [-1] * (keep - len(want)))


@pytest.mark.parametrize("kind", ["long tail", "ties", "bits"])
@pytest.mark.parametrize("length", [32768, 32780, 70001])
def test_select_of_long_contexts(length, kind):
    """More candidates than stay in LDS."""
    _say(f"select {length} {kind}")
    rng = np.random.default_rng(length)
    m = _masses(rng, kind, (1, 2, -(-length // 16) * 16)).astype(np.float32)
    kept, kept_len = _select(torch.from_numpy(m).cuda(), [length], 4097, 100, 4)
    assert kept_len[0] == 4097
    for h in range(2):
        np.testing.assert_array_equal(kept[0, h], okv8.select(m[0, h].tolist(), length, 4097, 100, 4))


def test_select_lengths_past_the_table_and_negative_ones():
    _say("select garbage lengths")
    m = torch.rand((3, 1, 64), generator=torch.Generator().manual_seed(2)).cuda()
    kept, kept_len = _select(m, [2 ** 31 - 1, -5, 70], 10, 3, 1)
    assert kept_len.tolist() == [10, 0, 10]
    for i in (0, 2):
        assert kept[i, 0].tolist() == okv8.select(m[i, 0].double().tolist(), 64, 10, 3, 1)
    assert np.all(kept[1] == -1)


def _evict(c: Case, kept, kept_len, new_table, width=None):
    """compact() and the oracle's, over the same pool."""
    mass = c.rng.random((len(c.lens), c.n_kv, c.table.shape[1] * c.block)).astype(np.float32)
    room = new_table.shape[1] * c.block
    old, new = torch.from_numpy(mass).cuda(), torch.full((len(c.lens), c.n_kv, room + 2), 9.0, device="cuda")
    up = lambda v: torch.from_numpy(np.ascontiguousarray(v, np.int32)).cuda()
    kv8.compact(c.cache, c.batch, up(kept), up(kept_len), up(new_table), old, new)
    torch.cuda.synchronize()
    before = okv8.Pool(c.pool.k, c.pool.v, c.pool.ks, c.pool.vs)
    okv8.compact(c.pool, c.table, kept, kept_len, new_table)
    got = okv8.Pool(c.cache.k.cpu().numpy(), c.cache.v.cpu().numpy(), c.cache.k_scale.double().cpu().numpy(), c.cache.v_scale.double().cpu().numpy())
    np.testing.assert_array_equal(got.ks, c.pool.ks)
    np.testing.assert_array_equal(got.vs, c.pool.vs)
    for a, b in ((got.k, c.pool.k), (got.v, c.pool.v)):
        nan = (a & 0x7F) == 0x7F
        np.testing.assert_array_equal(nan, (b & 0x7F) == 0x7F)
        np.testing.assert_array_equal(a[~nan], b[~nan])
    want = np.full((len(c.lens), c.n_kv, room + 2), 9.0, np.float32)
    for i, n in enumerate(kept_len):
        for h in range(c.n_kv):
            for r in range(min(int(n), kept.shape[2], room)):
                p = int(kept[i, h, r])
                want[i, h, r] = mass[i, h, p] if 0 <= p < c.table.shape[1] * c.block else 0.0
    np.testing.assert_array_equal(new.cpu().numpy(), want)
    return before


COMPACTS = [
    # block, n_kv, dim, lens, keep
    (16, 1, 64, [1, 17], 5), (16, 5, 128, [100, 40, 0], 37), (32, 8, 64, [200, 33], 64), (32, 3, 128, [150], 150), (64, 2, 64, [400, 5], 99),
    (64, 3, 128, [300], 130), (128, 2, 64, [500, 129], 200), (128, 1, 128, [700], 300),
]


@pytest.mark.parametrize("missing", [0.0, 0.3])
@pytest.mark.parametrize("case", COMPACTS, ids=[f"b{c[0]}h{c[1]}d{c[2]}" for c in COMPACTS])
def test_compact(case, missing):
    """Codes, scales and weights bit for bit; what no row was moved to stays."""
    block, n_kv, dim, lens, keep = case
    _say(f"compact {case} missing {missing}")
    rows = [min(n, keep) for n in lens]
    need = [-(-n // block) for n in rows]
    c = Case(block, n_kv, dim, lens, lens, seed=block + dim + keep, missing=missing, extra=sum(need) + 2)
    c.pool.ks[:], c.pool.vs[:] = (2.0 ** c.rng.integers(-12, 9, c.pool.ks.shape) for _ in range(2))
    for codes in (c.pool.k, c.pool.v):  # some NaN, and blocks of small values
        codes[c.rng.random(codes.shape) < 0.002] = 0x7F
        codes[c.rng.integers(0, c.pool.n_blocks)] &= 0x87
    c.upload()
    used = {int(b) for b in c.table.ravel() if 0 <= b < c.pool.n_blocks}
    free = [b for b in range(c.pool.n_blocks) if b not in used]
    new_table, at = np.full((len(lens), max(need + [1]) + 1), -1), 0
    for i, k in enumerate(need):
        new_table[i, :k] = free[at : at + k]
        at += k
    kept = np.full((len(lens), n_kv, keep), -1)
    for i, n in enumerate(rows):
        for h in range(n_kv):
            kept[i, h, :n] = np.sort(c.rng.choice(lens[i], n, replace=False)) if n else []
    _evict(c, kept, np.array(rows), new_table)


def test_compact_of_odd_entries():
    """Kept entries outside the table, more rows than the new table holds, new
    blocks that are missing, lengths of garbage: nothing else is written."""
    _say("compact odd entries")
    c = Case(16, 2, 64, [60, 60, 60], [60, 60, 60], seed=41, extra=6)
    used = {int(b) for b in c.table.ravel()}
    free = [b for b in range(c.pool.n_blocks) if b not in used]
    kept = np.sort(c.rng.integers(0, 60, (3, 2, 40)), -1)
    kept[0, 0, 3], kept[0, 1, 5], kept[0, 0, 20] = -1, 2 ** 31 - 1, 64
    new_table = np.array([[free[0], -1], [free[1], free[2]], [2 ** 31 - 1, free[3]]])
    _evict(c, kept, np.array([40, 2 ** 31 - 1, 20]), new_table)
    c.upload()
    _evict(c, kept, np.array([-4, 0, 1]), new_table)


def test_weights_and_moves_past_four_gigabytes():
    _say("weigh and compact in a pool of 4.5 GB")
    n_blocks, n_kv, block, dim = 18500, 16, 128, 128
    cache = kv8.Cache(*(torch.zeros(s, dtype=torch.uint8, device="cuda") for s in ((n_blocks, n_kv, block, dim), (n_blocks, n_kv, dim, block))),
                      *(torch.ones((n_blocks, n_kv), device="cuda") for _ in range(2)))
    small = kv8.Cache.empty(4, n_kv, dim, block)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    start, length = i32([0, 140]), i32([140])
    far, near = kv8.Batch(i32([[n_blocks - 1, n_blocks - 2]]), start, length, 140), kv8.Batch(i32([[0, 1]]), start, length, 140)
    g = torch.Generator().manual_seed(5)
    k, v, q = (torch.randn((140, n_kv, dim), generator=g).to(torch.bfloat16).cuda() for _ in range(3))
    got = []
    for pool, batch, new in ((cache, far, [[n_blocks - 3]]), (small, near, [[2]])):
        kv8.append(pool, batch, k, v)
        out, lse, mass = torch.empty_like(q), torch.empty((140, n_kv), device="cuda"), torch.empty((1, n_kv, 256), device="cuda")
        kv8.attention(pool, batch, q, out, lse=lse)
        kv8.weigh(pool, batch, q, lse, mass)
        kept, kept_len = torch.empty((1, n_kv, 60), dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
        kv8.select(pool, batch, mass, kept, kept_len, recent=8)
        kv8.compact(pool, batch, kept, kept_len, i32(new))
        rows = [torch.empty((60, n_kv, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        kv8.read(pool, kv8.Batch(i32(new), i32([0, 60]), kept_len, 60), *rows)
        got.append([out, lse, mass[..., :140], kept, kept_len, *rows])
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a, b)


# ---------------------------------------------------------------- together
class Server:
    """A layer's cache with weights and eviction, as a server runs it: two
    tables, of which one holds the sequences and the other what compaction fills."""

    def __init__(self, block, n_kv, n_q, dim, n_seq, width):
        self.n_q, self.n_kv, self.dim, self.n_seq, self.width = n_q, n_kv, dim, n_seq, width
        self.cache = kv8.Cache.empty(2 * n_seq * width, n_kv, dim, block)
        ids = torch.randperm(2 * n_seq * width, generator=torch.Generator().manual_seed(3)).to(torch.int32).cuda()
        self.table, self.spare = (t.contiguous() for t in ids.view(2, n_seq, width))
        self.mass, self.new_mass = (torch.zeros((n_seq, n_kv, width * block), device="cuda") for _ in range(2))
        self.inv, self.amp = kv8.rotary_frequencies(dim // 2, 1e4, "parts", 4.0, original=512)
        self.kv_len = torch.zeros(n_seq, dtype=torch.int32, device="cuda")
        self.scores = kv8.Scores(softcap=30.0, window=4000)

    def step(self, x, q_start, pos, n_tokens):
        """Packed QKV rows in, in place; kv_len counts them already."""
        batch = kv8.Batch(self.table, q_start, self.kv_len, n_tokens)
        q, k, v = x[:, : self.n_q], x[:, self.n_q : self.n_q + self.n_kv], x[:, self.n_q + self.n_kv :]
        kv8.rotary(q, k, self.inv, pos, q, k, interleaved=True, amplitude=self.amp)
        kv8.append(self.cache, batch, k, v)
        out, lse = torch.empty((n_tokens, self.n_q, self.dim), dtype=torch.bfloat16, device="cuda"), torch.empty((n_tokens, self.n_q), device="cuda")
        kv8.attention(self.cache, batch, q, out, scores=self.scores, lse=lse)
        kv8.weigh(self.cache, batch, q, lse, self.mass, scores=self.scores)
        return out, lse

    def evict(self, keep, recent, sinks):
        batch = kv8.Batch(self.table, torch.zeros(self.n_seq + 1, dtype=torch.int32, device="cuda"), self.kv_len, 0)
        kept = torch.empty((self.n_seq, self.n_kv, keep), dtype=torch.int32, device="cuda")
        kept_len = torch.empty(self.n_seq, dtype=torch.int32, device="cuda")
        kv8.select(self.cache, batch, self.mass, kept, kept_len, recent=recent, sinks=sinks)
        kv8.compact(self.cache, batch, kept, kept_len, self.spare, self.mass, self.new_mass)
        self.table, self.spare = self.spare, self.table
        self.mass, self.new_mass = self.new_mass, self.mass
        self.kv_len = kept_len
        return kept


@pytest.mark.parametrize("dim,block", [(64, 16), (128, 32)])
def test_a_conversation_with_evictions(dim, block):
    """Prompts, tokens, evictions, more tokens: attention and weights of every
    step against the oracle over the cache's own values, selection against the
    weights that it had, moved rows against the rows they were."""
    _say(f"conversation with evictions D={dim} block {block}")
    n_q, n_kv, n_seq = 4, 2, 2
    s = Server(block, n_kv, n_q, dim, n_seq, 12)
    rng, true_pos = np.random.default_rng(50), [0, 0]
    mass = np.zeros((n_seq, n_kv, 12 * block))
    for turn, (new, evict) in enumerate([([90, 41], None), ([1, 1], None), ([3, 0], (40, 8, 2)), ([1, 1], None), ([20, 17], (33, 0, 0)), ([1, 1], None)]):
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        pos = torch.tensor([p for a, n in zip(true_pos, new) for p in range(a, a + n)], dtype=torch.int32).cuda()
        true_pos = [a + n for a, n in zip(true_pos, new)]
        s.kv_len += torch.tensor(new, dtype=torch.int32).cuda()
        x = torch.from_numpy(rng.standard_normal((int(sum(new)), n_q + 2 * n_kv, dim))).to(torch.bfloat16).cuda()
        out, lse = s.step(x, torch.from_numpy(start).cuda(), pos, int(sum(new)))
        torch.cuda.synchronize()
        pool = okv8.Pool(s.cache.k.cpu().numpy(), s.cache.v.cpu().numpy(), s.cache.k_scale.double().cpu().numpy(), s.cache.v_scale.double().cpu().numpy())
        lens, table, q = s.kv_len.cpu().numpy(), s.table.cpu().numpy(), _f64(x[:, :n_q])
        slack = np.zeros_like(mass)
        for i in range(n_seq):
            mass[i, :, lens[i] - new[i] : lens[i]] = 0
        for i, t, h, j, sc, w, v, reach, bias in okv8.scored_rows(pool, table, start, lens, q, dim ** -0.5, okv8.Scores(softcap=30.0, window=4000)):
            e = (dim + 3) * U * reach + 300 * U + 3 * U * np.abs(sc).max()
            want, ref = w @ v, sc.max() + np.log(np.exp(sc - sc.max()).sum())
            tol = np.abs(want) * 2.0 ** -8 + (2.0 ** -8 + 2 * e + 300 * U) * (w @ np.abs(v))
            assert np.all(np.abs(_f64(out[t, h]) - want) <= tol), (turn, t, h)
            assert abs(float(lse[t, h]) - ref) <= e + 300 * U + 4 * U * abs(ref)
            mass[i, h // 2, j] += w
            slack[i, h // 2, j] += w * (3 * e + 700 * U + 8 * U * (np.abs(sc) + abs(ref)))
        got = s.mass.double().cpu().numpy()
        for i in range(n_seq):
            n = lens[i]
            assert np.all(np.abs(got[i, :, :n] - mass[i, :, :n]) <= slack[i, :, :n] + 300 * U * mass[i, :, :n] + 1e-30), (turn, i)
            mass[i, :, :n] = got[i, :, :n]
        if evict:
            old = [pool.values(*pool.place(table[i], p)) for i in range(n_seq) for p in range(lens[i])]
            kept = s.evict(*evict).cpu().numpy()
            torch.cuda.synchronize()
            pool = okv8.Pool(s.cache.k.cpu().numpy(), s.cache.v.cpu().numpy(), s.cache.k_scale.double().cpu().numpy(), s.cache.v_scale.double().cpu().numpy())
            for i in range(n_seq):
                n, base = min(lens[i], evict[0]), int(sum(lens[:i]))
                assert int(s.kv_len[i]) == n
                for h in range(n_kv):
                    assert kept[i, h, :n].tolist() == okv8.select(mass[i, h].tolist(), int(lens[i]), *evict)
                    mass[i, h, :n] = mass[i, h, kept[i, h, :n]]
                    for r in range(n):
                        b, row = pool.place(s.table[i].tolist(), r)
                        for a, z in zip(old[base + int(kept[i, h, r])], pool.values(b, row)):
                            scale = max(pool.ks[b, h], pool.vs[b, h])
                            assert np.all(np.abs(a[h] - z[h]) <= np.maximum(np.abs(a[h]) * 2.0 ** -4, scale * 2.0 ** -10))


def test_graphs_of_steps_and_evictions():
    """Captured: a step, and a step with an eviction.  Replayed with other rows,
    lengths and eager work between, every output is the eager calls'."""
    _say("graphs")
    n_q, n_kv, dim, block, n_seq, width = 4, 2, 64, 32, 3, 70

    def fresh():
        s = Server(block, n_kv, n_q, dim, n_seq, width)
        g = torch.Generator().manual_seed(9)
        s.cache.k.copy_(torch.randint(0, 0x50, s.cache.k.shape, generator=g, dtype=torch.uint8))
        s.cache.v.copy_(torch.randint(0, 0x50, s.cache.v.shape, generator=g, dtype=torch.uint8))
        s.cache.k_scale.fill_(0.125), s.cache.v_scale.fill_(0.25)
        s.mass.copy_(torch.rand(s.mass.shape, generator=g))
        return s

    def call(s, x, start, pos, new_len):
        out, lse = s.step(x, start, pos, 3)
        batch = kv8.Batch(s.table, torch.zeros(n_seq + 1, dtype=torch.int32, device="cuda"), s.kv_len, 0)
        kept = torch.empty((n_seq, n_kv, 500), dtype=torch.int32, device="cuda")
        kv8.select(s.cache, batch, s.mass, kept, new_len, recent=32, sinks=4)
        kv8.compact(s.cache, batch, kept, new_len, s.spare, s.mass, s.new_mass)
        return out, lse, kept

    a, e = fresh(), fresh()
    x = torch.zeros((3, n_q + 2 * n_kv, dim), dtype=torch.bfloat16, device="cuda")
    start, pos = torch.arange(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    len_a, len_e = (torch.zeros(n_seq, dtype=torch.int32, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(fresh(), x.clone(), start, pos, len_a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(a, x, start, pos, len_a)
    for turn, lens in enumerate(([2000, 700, 1], [2001, 701, 2], [64, 33, 900], [0, 2240, 501])):
        new = torch.randn(x.shape, generator=torch.Generator().manual_seed(turn)).to(torch.bfloat16).cuda()
        x.copy_(new)
        for s in (a, e):
            s.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        pos.copy_(torch.tensor(lens, dtype=torch.int32) - 1)
        graph.replay()
        want = call(e, new, start, pos, len_e)
        torch.cuda.synchronize()
        for g, w in zip([*got, len_a, a.mass, a.cache.k, a.cache.v, a.cache.k_scale, a.cache.v_scale, a.new_mass],
                        [*want, len_e, e.mass, e.cache.k, e.cache.v, e.cache.k_scale, e.cache.v_scale, e.new_mass]):
            assert torch.equal(g, w), f"replay {turn}"


# ---------------------------------------------------------------- refusals
def test_python_refusals():
    _say("refusals")
    c = Case(16, 2, 64, [20, 3], [2, 1], seed=60)
    q, out = (torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    f32, i32 = dict(device="cuda"), dict(device="cuda", dtype=torch.int32)
    lse, mass = torch.zeros((3, 4), **f32), torch.zeros((2, 2, 32), **f32)
    for x, word in ((kv8.Scores(slopes=torch.zeros(3, **f32)), "slopes of the scores"), (kv8.Scores(first=torch.zeros(4, **i32)), "first of the scores"),
                    (kv8.Scores(prefix=torch.zeros(1, **i32)), "prefix of the scores")):
        with pytest.raises(ValueError, match=word):
            kv8.attention(c.cache, c.batch, q, out, scores=x)
        with pytest.raises(ValueError, match=word):
            kv8.weigh(c.cache, c.batch, q, lse, mass, scores=x)
    for bad in (dict(slopes=torch.zeros(4, **i32)), dict(first=torch.zeros(3, **f32)), dict(prefix=torch.zeros((2, 1), **i32)),
                dict(slopes=torch.zeros(8, **f32)[::2])):
        with pytest.raises(ValueError):
            kv8.Scores(**bad)
    for bad in (torch.zeros((3, 3), **f32), torch.zeros((3, 4), dtype=torch.float64, device="cuda"), torch.zeros((4, 3), **f32).T, torch.zeros((3, 4))):
        with pytest.raises(ValueError, match="lse"):
            kv8.attention(c.cache, c.batch, q, out, lse=bad)
        with pytest.raises(ValueError, match="lse"):
            kv8.weigh(c.cache, c.batch, q, bad, mass)
    kept, kept_len, new = torch.zeros((2, 2, 8), **i32), torch.zeros(2, **i32), torch.zeros((2, 1), **i32)
    for bad in (torch.zeros((2, 2, 31), **f32), torch.zeros((2, 3, 32), **f32), torch.zeros((2, 32), **f32), mass.double(), mass.cpu(),
                torch.zeros((2, 2, 64), **f32)[..., ::2]):
        for call in (lambda: kv8.weigh(c.cache, c.batch, q, lse, bad), lambda: kv8.select(c.cache, c.batch, bad, kept, kept_len),
                     lambda: kv8.compact(c.cache, c.batch, kept, kept_len, new, bad, torch.zeros_like(mass))):
            with pytest.raises(ValueError, match="mass|last dimension"):
                call()
    for k, n in ((kept.float(), kept_len), (kept[:1], kept_len), (kept[..., :0], kept_len), (kept, kept_len[:1]), (kept.transpose(0, 1), kept_len),
                 (kept, kept_len.cpu())):
        with pytest.raises(ValueError, match="kept"):
            kv8.select(c.cache, c.batch, mass, k, n)
        with pytest.raises(ValueError, match="kept"):
            kv8.compact(c.cache, c.batch, k, n, new)
    for recent, sinks in ((9, 0), (0, 9), (5, 4), (-1, 0), (0, -1), (2 ** 32, 0), (0, 2 ** 32 + 1)):
        with pytest.raises(ValueError, match="recent"):
            kv8.select(c.cache, c.batch, mass, kept, kept_len, recent=recent, sinks=sinks)
    for bad in (new.float(), new[:1], torch.zeros((2, 0), **i32), new.cpu()):
        with pytest.raises(ValueError, match="new_table"):
            kv8.compact(c.cache, c.batch, kept, kept_len, bad)
    with pytest.raises(ValueError, match="go together"):
        kv8.compact(c.cache, c.batch, kept, kept_len, new, mass)
    with pytest.raises(_lib.MegakernelError, match="batch's table"):
        kv8.compact(c.cache, c.batch, kept, kept_len, c.batch.table)
    with pytest.raises(_lib.MegakernelError, match="same rows"):
        kv8.compact(c.cache, c.batch, kept, kept_len, new, mass, mass)
    pos, inv, k = torch.zeros(3, **i32), torch.ones(32, **f32), torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    for args in ((q, k, torch.ones(33, **f32), pos, q, k), (q, k, torch.ones(0, **f32), pos, q, k), (q, k, inv, pos[:2], q, k), (q, k, inv.double(), pos, q, k),
                 (q, k[:2], inv, pos, q, k), (q, k.half(), inv, pos, q, k), (q, k, inv, pos, q, q), (q[0], k, inv, pos, q, k)):
        with pytest.raises(ValueError):
            kv8.rotary(*args)
    with pytest.raises(_lib.MegakernelError, match="amplitude"):
        kv8.rotary(q, k, inv, pos, q, k, amplitude=1e300)
    grad = torch.zeros_like(mass, requires_grad=True)
    with pytest.raises(ValueError, match="mass requires a gradient"):
        kv8.weigh(c.cache, c.batch, q, lse, grad)


def test_empty_batches():
    _say("empty batches")
    cache, i32 = kv8.Cache.empty(2, 1, 64, 16), dict(device="cuda", dtype=torch.int32)
    none = kv8.Batch(torch.zeros((0, 1), **i32), torch.zeros(1, **i32), torch.zeros(0, **i32), 0)
    q, lse = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((0, 2), device="cuda")
    mass, kept = torch.zeros((0, 1, 16), device="cuda"), torch.zeros((0, 1, 4), **i32)
    x = kv8.Scores(first=torch.zeros(0, **i32), prefix=torch.zeros(0, **i32))
    kv8.attention(cache, none, q, q, scores=x, lse=lse)
    kv8.weigh(cache, none, q, lse, mass, scores=x)
    kv8.select(cache, none, mass, kept, torch.zeros(0, **i32))
    kv8.compact(cache, none, kept, torch.zeros(0, **i32), torch.zeros((0, 1), **i32), mass, torch.zeros((0, 1, 16), device="cuda"))
    kv8.rotary(q, q, torch.ones(32, device="cuda"), torch.zeros(0, **i32), q, q)
    torch.cuda.synchronize()
