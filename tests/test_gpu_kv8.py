"""GPU parity of the paged 8-bit KV cache's operators with oracle/kv8.py (64 bits).

Tolerances.  Codes, scales and values read back are exact: every step is
exact but the one rounding to e4m3, which both sides do to nearest even.
Norms and attention, u = 2^-24 (half a step of fp32), h = half a step of the
output's type (2^-8 bf16, u fp32):
  norm: |y| h + 24 u (|a| + |b|) for a pair (a, b) of normalised values: the
    mean's sum (8 levels and 16 terms in a lane, halved by the root: 12 u),
    the root, two products and the gain (4 u), the angle's fraction of a turn
    and its sine (5 u), the rotation (3 u);
  attention: |o| h + (2^-8 + 2 D u reach + n u + 16 u) sum_j p_j |v_j|: weights
    rounded to bf16; scores of D products with sum |q k| scale <= reach summed
    in fp32, an error of which enters the weight and the sum; n positions
    summed in fp32; exponentials and divisions.  Beside the largest weight, 1,
    one below 2^-126, fp32's smallest normal number, may be zero: n 2^-126
    times the largest |v| the scales allow, 448 of them.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from megakernel_amd import _lib, kv8
from oracle import fp8
from oracle import kv8 as okv8

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}


def _say(*a):
    print(*a, flush=True)


def _f64(t) -> np.ndarray:
    return t.detach().double().cpu().numpy()


class Case:
    """Sequences over a pool whose blocks are dealt at random; `missing` of
    table entries are outside the pool."""

    def __init__(self, block, n_kv, dim, lens, new, seed, missing=0.0, extra=3, gap=0, width=None, fill=True):
        rng = np.random.default_rng(seed)
        self.rng, self.block, self.n_kv, self.dim = rng, block, n_kv, dim
        need = [-(-c // block) for c in lens]
        n_blocks = sum(need) + extra
        ids = rng.permutation(n_blocks)
        width = width or max(need + [1])
        table, at = rng.choice(np.array([-1, -7, n_blocks, 2 ** 31 - 1]), (len(lens), width)), 0
        for i, k in enumerate(need):
            k = min(k, width)
            table[i, :k] = ids[at : at + k]
            at += k
        if missing:
            drop = rng.random(table.shape) < missing
            table = np.where(drop, rng.choice(np.array([-1, n_blocks, 2 ** 31 - 1]), table.shape), table)
        self.table = table.astype(np.int32)
        self.start = (gap + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
        self.lens, self.tokens = np.array(lens, np.int32), int(gap + sum(new) + gap)
        shape = (n_blocks, n_kv, block, dim)
        if fill:  # finite codes, scales of several sizes
            k = rng.integers(0, 256, shape).astype(np.uint8)
            v = rng.integers(0, 256, (n_blocks, n_kv, dim, block)).astype(np.uint8)
            k[(k & 0x7F) > 0x60], v[(v & 0x7F) > 0x60] = 0x38, 0xB8
            ks, vs = (2.0 ** rng.integers(-6, -2, shape[:2]) for _ in range(2))
        else:  # what an allocation may hold: every code NaN, scales NaN
            k, v = np.full(shape, 0xFF, np.uint8), np.full((n_blocks, n_kv, dim, block), 0x7F, np.uint8)
            ks, vs = np.full(shape[:2], np.nan), np.full(shape[:2], np.nan)
        self.pool = okv8.Pool(k, v, ks, vs)
        self.upload()

    def upload(self):
        p = self.pool
        self.cache = kv8.Cache(*(torch.from_numpy(x).cuda() for x in (p.k, p.v, p.ks.astype(np.float32), p.vs.astype(np.float32))))
        self.batch = kv8.Batch(*(torch.from_numpy(x).cuda() for x in (self.table, self.start, self.lens)), self.tokens)

    def rows(self, heads, dtype, scale=1.0):
        return (torch.from_numpy(self.rng.standard_normal((self.tokens, heads, self.dim))) * scale).to(dtype)

    def same_pool(self):
        c = self.cache
        np.testing.assert_array_equal(c.k_scale.double().cpu().numpy(), self.pool.ks)
        np.testing.assert_array_equal(c.v_scale.double().cpu().numpy(), self.pool.vs)
        np.testing.assert_array_equal(c.k.cpu().numpy(), self.pool.k)
        np.testing.assert_array_equal(c.v.cpu().numpy(), self.pool.v)


# -------------------------------------------------------------------- norms
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dst", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,n_q,n_kv,layout", [(1, 16, 8, "packed"), (37, 5, 1, "packed"), (130, 2, 3, "heads"),
                                                    (64, 16, 8, "in place")])
def test_qk_norm_rope(dim, src, dst, tokens, n_q, n_kv, layout):
    if layout == "in place":
        dst = src
    _say(f"qk_norm_rope D={dim} {src} -> {dst} T={tokens} {n_q}/{n_kv} {layout}")
    g = torch.Generator().manual_seed(tokens * dim + n_q)
    x = torch.randn((tokens, n_q + 2 * n_kv, dim), generator=g) * 3
    x[0, 0] = 0  # an all-zero head
    if tokens > 2:
        x[2] *= 1e-4  # eps counts
    x = x.to(src).cuda()
    qg, kg = ((1 + 0.2 * torch.randn(dim, generator=g)).to(torch.bfloat16).cuda() for _ in range(2))
    inv = torch.tensor([1e6 ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float32).cuda()
    pos = torch.randint(0, 200000, (tokens,), generator=g, dtype=torch.int32)
    pos[0] = 0
    if tokens > 1:
        pos[1] = 2 ** 31 - 1
    pos = pos.cuda()
    q, k = x[:, :n_q], x[:, n_q : n_q + n_kv]
    want = [okv8.norm_rope(_f64(r), _f64(gn), _f64(inv), pos.cpu().numpy(), 1e-6) for r, gn in ((q, qg), (k, kg))]
    rest = x[:, n_q + n_kv :].clone()
    if layout == "packed":
        outs = [torch.full((tokens, h, dim), float("nan"), dtype=dst, device="cuda") for h in (n_q, n_kv)]
    elif layout == "heads":  # [heads][tokens][dim]
        outs = [torch.full((h, tokens, dim), float("nan"), dtype=dst, device="cuda").transpose(0, 1) for h in (n_q, n_kv)]
    else:
        outs = [q, k]
    kv8.qk_norm_rope(q, k, qg, kg, inv, pos, *outs, eps=1e-6)
    torch.cuda.synchronize()
    for got, (y, pair) in zip(outs, want):
        err, tol = np.abs(_f64(got) - y), np.abs(y) * HALF[dst] + 24 * U * pair
        within = bool(np.all(err <= tol))
        assert within, f"worst {np.max(err / np.maximum(tol, 1e-30)):.2f} of the tolerance"
    assert torch.equal(x[:, n_q + n_kv :], rest)  # V of the packed rows is not touched
    assert torch.all(outs[0][0, 0] == 0)


# ----------------------------------------------------- append and read back
APPENDS = [
    # block, n_kv, dim, lens, new, gap
    (16, 1, 64, [1], [1], 0),
    (16, 3, 128, [17, 5, 16], [1, 5, 3], 0),
    (32, 8, 64, [40, 33, 64, 1, 0], [1, 1, 1, 1, 0], 2),
    (32, 2, 128, [100, 31, 65], [100, 7, 34], 1),
    (64, 2, 64, [130, 64], [77, 64], 0),
    (128, 1, 128, [300, 128, 129], [290, 1, 1], 3),
    (128, 2, 64, [127], [100], 0),
]


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", APPENDS, ids=[f"b{c[0]}h{c[1]}d{c[2]}" for c in APPENDS])
def test_append_codes_and_scales(case, src):
    block, n_kv, dim, lens, new, gap = case
    _say(f"append {case} {src}")
    c = Case(block, n_kv, dim, lens, new, seed=sum(lens) + block, gap=gap)
    # rows of every size, so that some blocks' scales grow and others' do not
    size = torch.from_numpy(np.exp(c.rng.uniform(-6, 8, (c.tokens, n_kv, 1))))
    k, v = (c.rows(n_kv, torch.float64) * size).to(src), (c.rows(n_kv, torch.float64) * size * 0.3).to(src)
    if c.tokens > 2:
        k[gap + 1] = 0
        v[gap] = 0
    c.pool.append(c.table, c.start, c.lens, _f64(k), _f64(v))
    kv8.append(c.cache, c.batch, k.cuda(), v.cuda())
    torch.cuda.synchronize()
    c.same_pool()
    kv8.append(c.cache, c.batch, k.cuda(), v.cuda())  # once more: rows take the same codes
    torch.cuda.synchronize()
    c.same_pool()


@pytest.mark.parametrize("dim", [64, 128])
def test_append_encodes_every_code_and_its_borders(dim):
    """Every e4m3 value, the midpoints between neighbours and values beside
    them, at scales to both ends of fp32."""
    _say(f"append every code D={dim}")
    vals = np.sort(np.unique(fp8.e4m3_decode_table()[np.r_[0:0x7F]].astype(np.float64)))
    mid = (vals[1:] + vals[:-1]) / 2
    x = np.concatenate([vals, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    x = np.concatenate([x, -x, [0.0] * (-2 * len(x) % dim)]).reshape(-1, 1, dim)
    for e in (0, -5, 30, -117, -126, 119):
        c = Case(16, 1, dim, [16] * len(x), [1] * len(x), seed=3, fill=False)
        c.lens[:] = 1
        x[:, 0, -1] = 448.0  # every row has the scale 2^e
        rows = torch.from_numpy(np.ldexp(x, e)).float()
        c.upload()
        c.pool.append(c.table, c.start, c.lens, _f64(rows), _f64(rows))
        assert np.all(c.pool.ks[c.table[:, 0]] == 2.0 ** e)
        kv8.append(c.cache, c.batch, rows.cuda(), rows.cuda())
        torch.cuda.synchronize()
        c.same_pool()


def test_append_infinities_nan_and_tiny_rows():
    _say("append inf, nan, tiny")
    c = Case(32, 2, 64, [5, 40], [5, 33], seed=4)
    k, v = c.rows(2, torch.float32), c.rows(2, torch.float32)
    k[0, 0, 3], k[1, 1, 9], v[2, 0, 5], v[7, 1, 63], v[20, 0, 0] = np.inf, -np.inf, np.nan, np.inf, -np.nan
    k[3, 0] = np.inf
    k[6:38, 1] *= 2.0 ** -140  # whole rows among fp32's smallest numbers
    c.pool.append(c.table, c.start, c.lens, _f64(k), _f64(v))
    kv8.append(c.cache, c.batch, k.cuda(), v.cuda())
    torch.cuda.synchronize()
    for got, want in ((c.cache.k, c.pool.k), (c.cache.v, c.pool.v)):  # a NaN may have either sign
        got = got.cpu().numpy()
        np.testing.assert_array_equal(np.where((got & 0x7F) == 0x7F, 0x7F, got), np.where((want & 0x7F) == 0x7F, 0x7F, want))
    np.testing.assert_array_equal(c.cache.k_scale.double().cpu().numpy(), c.pool.ks)
    np.testing.assert_array_equal(c.cache.v_scale.double().cpu().numpy(), c.pool.vs)


def test_append_drops_rows_without_a_place():
    """Missing blocks, rows before position 0, positions past the table, and
    rows of no sequence."""
    _say("append without places")
    c = Case(16, 2, 64, [40, 3, 70, 20], [20, 9, 50, 4], seed=5, missing=0.4, gap=3, width=4)
    k, v = c.rows(2, torch.bfloat16), c.rows(2, torch.bfloat16)
    c.pool.append(c.table, c.start, c.lens, _f64(k), _f64(v))
    kv8.append(c.cache, c.batch, k.cuda(), v.cuda())
    torch.cuda.synchronize()
    c.same_pool()


@pytest.mark.parametrize("dst", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("case", [(16, 1, 64, [1], [1]), (16, 3, 128, [17, 5, 40], [17, 2, 33]), (32, 8, 64, [100, 0, 31], [64, 0, 31]),
                                  (64, 2, 128, [70, 200], [70, 129]), (128, 1, 64, [300, 20], [300, 30])],
                         ids=lambda c: f"b{c[0]}h{c[1]}d{c[2]}" if isinstance(c, tuple) else None)
@pytest.mark.parametrize("missing", [0.0, 0.5])
def test_read(case, dst, missing):
    block, n_kv, dim, lens, new = case
    _say(f"read {case} {dst} missing {missing}")
    c = Case(block, n_kv, dim, lens, new, seed=block + dim, missing=missing, gap=2)
    want = [np.full((c.tokens, n_kv, dim), 7.0) for _ in range(2)]
    c.pool.read(c.table, c.start, c.lens, *want)
    for order in ("tokens", "heads"):
        if order == "tokens":
            got = [torch.full((c.tokens, n_kv, dim), 7.0, dtype=dst, device="cuda") for _ in range(2)]
        else:
            got = [torch.full((n_kv, c.tokens, dim), 7.0, dtype=dst, device="cuda").transpose(0, 1) for _ in range(2)]
        kv8.read(c.cache, c.batch, *got)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            np.testing.assert_array_equal(_f64(g), w)


# ---------------------------------------------------------------- attention
def _check_attention(c: Case, n_q, scale=None, q=None, say="", nan_ok=False, workspace=None):
    if q is None:
        q = c.rows(n_q, torch.bfloat16, 1.5)
    out = torch.full((c.tokens, n_q, c.dim), 5.0, dtype=torch.bfloat16, device="cuda")
    want = np.full((c.tokens, n_q, c.dim), 5.0)
    sc = c.dim ** -0.5 if scale is None else scale
    with np.errstate(invalid="ignore"):
        size, reach = c.pool.attention(c.table, c.start, c.lens, _f64(q), want, sc)
    kv8.attention(c.cache, c.batch, q.cuda(), out, scale=scale, workspace=workspace)
    torch.cuda.synchronize()
    got = _f64(out)
    n = int(max(list(c.lens) + [1]))
    with np.errstate(invalid="ignore"):
        tol = np.abs(want) * 2.0 ** -8 + (2.0 ** -8 + (2 * c.dim * reach + n + 16)[..., None] * U) * size
        tol += n * 2.0 ** -126 * 448 * c.pool.vs.max()
        bad = ~(np.abs(got - want) <= tol)
    if nan_ok:
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        bad &= ~np.isnan(want)
    n_bad = int(bad.sum())
    assert n_bad == 0, f"{say}: {n_bad} outputs off, first at {np.argwhere(bad)[:1]}"
    return q, out


ATTENDS = [
    # block, n_kv, group, dim, lens, new
    (16, 1, 1, 64, [1], [1]),
    (16, 2, 2, 128, [2, 64, 65], [1, 1, 1]),
    (32, 8, 2, 64, [100, 1, 0, 333], [1, 1, 1, 1]),
    (32, 1, 5, 128, [70, 129], [1, 2]),
    (64, 2, 16, 64, [200], [3]),
    (128, 1, 20, 64, [130, 40], [2, 1]),
    (16, 2, 3, 64, [90, 40, 17], [90, 33, 5]),
    (64, 1, 2, 128, [150, 66, 3], [140, 1, 3]),
    (128, 1, 1, 128, [257], [257]),
    (32, 1, 8, 64, [300], [64]),
]


@pytest.mark.parametrize("missing", [0.0, 0.3])
@pytest.mark.parametrize("case", ATTENDS, ids=[f"b{c[0]}h{c[1]}g{c[2]}d{c[3]}n{sum(c[5])}" for c in ATTENDS])
def test_attention(case, missing):
    block, n_kv, group, dim, lens, new = case
    _say(f"attention {case} missing {missing}")
    c = Case(block, n_kv, dim, lens, new, seed=block * dim + sum(lens), missing=missing, gap=1)
    _check_attention(c, n_kv * group)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_splits_of_a_long_context(dim):
    """Few rows over a long axis: many splits, some of them without a position,
    and a hint that is far too short."""
    for lens, hint in (([2100], 0), ([2100], 100), ([1500, 30, 700], 4096)):
        _say(f"attention long D={dim} {lens} hint {hint}")
        c = Case(32, 1, dim, lens, [1] * len(lens), seed=dim, missing=0.1)
        c.batch = kv8.Batch(c.batch.table, c.batch.q_start, c.batch.kv_len, c.tokens, hint)
        _check_attention(c, 2, say=f"hint {hint}")


def test_attention_more_rows_than_positions():
    """Rows whose position is negative see nothing."""
    _say("attention negative positions")
    c = Case(16, 2, 64, [5, 40], [9, 50], seed=8)
    _, out = _check_attention(c, 4)
    assert torch.all(out[:4] == 0) and torch.all(out[9:19] == 0)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_never_sees_what_it_may_not(dim):
    """NaN codes behind the last row, in unused blocks, and in later positions
    of the same tile reach no row that does not see them; those that do are NaN."""
    _say(f"attention NaN D={dim}")
    c = Case(16, 2, dim, [90, 33, 70], [40, 33, 1], seed=9, missing=0.2)
    used = {int(b) for row, n in zip(c.table, c.lens) for j, b in enumerate(row) if j < -(-int(n) // 16) and 0 <= b < c.pool.n_blocks}
    for b in range(c.pool.n_blocks):
        if b not in used:
            c.pool.k[b], c.pool.v[b] = 0x7F, 0xFF
    for row, n in zip(c.table, c.lens):
        b, r = int(row[(n - 1) // 16]), int(n) % 16
        if r and 0 <= b < c.pool.n_blocks:
            c.pool.k[b, :, r:], c.pool.v[b, :, :, r:] = 0xFF, 0x7F
    c.upload()
    _check_attention(c, 4)
    b = int(c.table[0, 70 // 16])  # position 70 of sequence 0: rows from its 20th on see it
    assert 0 <= b < c.pool.n_blocks
    c.pool.v[b, 1, 5, 70 % 16] = 0x7F
    c.pool.v[int(c.table[1, 0]), 0, 9, 3] = 0xFF
    c.upload()
    _, out = _check_attention(c, 4, nan_ok=True)
    assert torch.isnan(out[20, 2, 5]) and not torch.isnan(out[19]).any()
    c.pool.k[b, 0, 70 % 16, 7] = 0x7F  # a NaN key makes the whole row NaN
    c.upload()
    _check_attention(c, 4, nan_ok=True)


def test_attention_large_scores_and_scales():
    """Scores in the hundreds to tens of thousands, whose weights leave fp32's
    range, and scales at both ends."""
    _say("attention extremes")
    c = Case(32, 2, 64, [150, 80], [1, 20], seed=10)
    for ke, ve, qs in ((9, 100, 3.0), (-100, -100, 1.0), (20, 0, 1e-3)):
        c.pool.ks[:], c.pool.vs[:] = 2.0 ** ke, 2.0 ** ve
        c.upload()
        q = c.rows(4, torch.bfloat16, qs)
        # one key decides or two are equal: whole scores matter, so use a
        # scale at which an fp32 score's error stays below one part in 2^10
        _check_attention(c, 4, scale=2.0 ** -10 if ke == 9 else None, q=q, say=f"{ke} {ve}")


def test_attention_strides_and_head_order():
    _say("attention strides")
    c = Case(16, 2, 64, [60, 9], [5, 4], seed=11)
    q, want = _check_attention(c, 4)
    wide = torch.zeros((c.tokens, 9, 96), dtype=torch.bfloat16, device="cuda")
    wide[:, 2:6, 16:80] = q.cuda()
    out = torch.full((4, c.tokens + 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    kv8.attention(c.cache, c.batch, wide[:, 2:6, 16:80], out.transpose(0, 1)[: c.tokens])
    torch.cuda.synchronize()
    assert torch.equal(out.transpose(0, 1)[: c.tokens], want)
    assert torch.all(out[:, c.tokens :] == 3.0)


def test_pool_past_four_gigabytes():
    """Blocks whose codes lie past 2^32 bytes of the pool."""
    _say("pool of 4.5 GB")
    n_blocks, n_kv, block, dim = 18500, 16, 128, 128
    cache = kv8.Cache(*(torch.zeros(s, dtype=torch.uint8, device="cuda") for s in ((n_blocks, n_kv, block, dim), (n_blocks, n_kv, dim, block))),
                      *(torch.ones((n_blocks, n_kv), device="cuda") for _ in range(2)))
    small = Case(block, n_kv, dim, [140], [140], seed=12, extra=0)
    high = torch.tensor([[n_blocks - 1, n_blocks - 2]], dtype=torch.int32, device="cuda")
    small.table = np.array([[0, 1]], np.int32)
    small.upload()
    batch = kv8.Batch(high, small.batch.q_start, small.batch.kv_len, 140)
    k, v, q = small.rows(n_kv, torch.bfloat16), small.rows(n_kv, torch.bfloat16), small.rows(n_kv, torch.bfloat16)
    outs = []
    for c, b in ((small.cache, small.batch), (cache, batch)):
        kv8.append(c, b, k.cuda(), v.cuda())
        out, ko, vo = (torch.empty_like(x, device="cuda") for x in (q, k, v))
        kv8.attention(c, b, q.cuda(), out)
        kv8.read(c, b, ko, vo)
        torch.cuda.synchronize()
        outs.append((out, ko, vo))
    for x, y in zip(*outs):
        assert torch.equal(x, y)
    assert not cache.k[: n_blocks - 2].any() and not cache.v[: n_blocks - 2].any()


# ------------------------------------------------------------ used together
def _layer(c, batch, x, n_q, gains, inv, pos, eps=1e-6):
    """One layer's attention as a server runs it: packed QKV rows in, in place."""
    n_kv = c.n_kv
    q, k, v = x[:, :n_q], x[:, n_q : n_q + n_kv], x[:, n_q + n_kv :]
    kv8.qk_norm_rope(q, k, *gains, inv, pos, q, k, eps=eps)
    kv8.append(c.cache, batch, k, v)
    out = torch.empty((x.shape[0], n_q, c.dim), dtype=torch.bfloat16, device="cuda")
    kv8.attention(c.cache, batch, q, out)
    return out


@pytest.mark.parametrize("dim", [64, 128])
def test_a_conversation_in_steps(dim):
    """A prompt, then token by token, against the oracle fed with the same
    rows: caches bit for bit, attention within its tolerance at every step."""
    _say(f"conversation D={dim}")
    n_q, n_kv, block, total = 4, 2, 16, 61
    c = Case(block, n_kv, dim, [total, total - 20], [1, 1], seed=13, fill=False)
    rng = np.random.default_rng(14)
    gains = [torch.from_numpy(1 + 0.1 * rng.standard_normal(dim)).to(torch.bfloat16).cuda() for _ in range(2)]
    inv = torch.tensor([1e6 ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float32).cuda()
    done = [0, 0]
    for new in ([37, 20], [1, 1], [1, 0], [5, 3], [1, 1], [0, 1], [16, 15]):
        end = [a + b for a, b in zip(done, new)]
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        c.start, c.lens, c.tokens = start, np.array(end, np.int32), int(sum(new))
        batch = kv8.Batch(c.batch.table, torch.from_numpy(start).cuda(), torch.from_numpy(c.lens).cuda(), c.tokens)
        pos = torch.tensor([p for a, b in zip(done, end) for p in range(a, b)], dtype=torch.int32).cuda()
        x = torch.from_numpy(rng.standard_normal((c.tokens, n_q + 2 * n_kv, dim))).to(torch.bfloat16).cuda()
        out = _layer(c, batch, x, n_q, gains, inv, pos)
        torch.cuda.synchronize()
        # x now holds the normed and rotated rows that the cache was given
        c.pool.append(c.table, start, c.lens, _f64(x[:, n_q : n_q + n_kv]), _f64(x[:, n_q + n_kv :]))
        c.same_pool()
        want = np.zeros((c.tokens, n_q, dim))
        size, reach = c.pool.attention(c.table, start, c.lens, _f64(x[:, :n_q]), want, dim ** -0.5)
        tol = np.abs(want) * 2.0 ** -8 + (2.0 ** -8 + (2 * dim * reach + total + 16)[..., None] * U) * size
        within = bool(np.all(np.abs(_f64(out) - want) <= tol))
        assert within, f"step {new}"
        done = end


def test_graph_replays_follow_lengths_and_tables():
    """A captured step, replayed with other lengths, rows and blocks and eager
    work in between, equals the eager call every time."""
    _say("graph")
    n_q, n_kv, dim, block = 4, 2, 64, 32
    c = Case(block, n_kv, dim, [1500, 700], [1, 1], seed=15)
    e = Case(block, n_kv, dim, [1500, 700], [1, 1], seed=15)
    gains = [torch.ones(dim, dtype=torch.bfloat16, device="cuda")] * 2
    inv = torch.tensor([1e6 ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float32).cuda()
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    x = torch.zeros((2, n_q + 2 * n_kv, dim), dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer(c, c.batch, x.clone(), n_q, gains, inv, pos)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    c.upload(), e.upload()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _layer(c, c.batch, x, n_q, gains, inv, pos)
    for step, lens in enumerate(([1500, 700], [1501, 701], [64, 1], [1, 1024], [1502, 702])):
        new = torch.randn(x.shape, generator=torch.Generator().manual_seed(step)).to(torch.bfloat16).cuda()
        x.copy_(new)
        for b in (c.batch, e.batch):
            b.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
            if step == 2:
                b.table.copy_(b.table.flip(0))
        pos.copy_(torch.tensor(lens, dtype=torch.int32) - 1)
        graph.replay()
        want = _layer(e, e.batch, new, n_q, gains, inv, pos)
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {step}"
        assert torch.equal(c.cache.k, e.cache.k) and torch.equal(c.cache.v, e.cache.v)


def test_two_streams_at_once():
    """Two calls in flight, each on its own stream with a workspace of its own."""
    _say("streams")
    cs = [Case(32, 1, 64, [1800], [1], seed=s) for s in (16, 17)]
    qs = [c.rows(2, torch.bfloat16).cuda() for c in cs]
    outs = [torch.empty_like(q) for q in qs]
    want = []
    for c, q in zip(cs, qs):
        o = torch.empty_like(q)
        kv8.attention(c.cache, c.batch, q, o)
        want.append(o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(20):
        for s, c, q, o in zip(streams, cs, qs, outs):
            with torch.cuda.stream(s):
                kv8.attention(c.cache, c.batch, q, o)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_python_refusals():
    _say("refusals")
    c = Case(16, 2, 64, [20], [3], seed=18)
    q, k = c.rows(4, torch.bfloat16).cuda(), c.rows(2, torch.bfloat16).cuda()
    out = torch.empty_like(q)
    with pytest.raises(ValueError, match="shape"):
        kv8.attention(c.cache, c.batch, q[:2], out)
    with pytest.raises(ValueError, match="bfloat16"):
        kv8.attention(c.cache, c.batch, q.float(), out)
    with pytest.raises(ValueError, match="on cpu"):
        kv8.attention(c.cache, c.batch, q, out.cpu())
    with pytest.raises(ValueError, match="contiguous"):
        kv8.append(c.cache, c.batch, k.transpose(0, 2).contiguous().transpose(0, 2), k)
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        kv8.append(c.cache, c.batch, k.half(), k.half())
    with pytest.raises(_lib.MegakernelError, match="multiple"):
        kv8.attention(c.cache, c.batch, q[:, :3].contiguous(), out[:, :3].contiguous())
    with pytest.raises(_lib.MegakernelError, match="overlap"):
        kv8.read(c.cache, c.batch, k[:1].expand(3, 2, 64), k)
    with pytest.raises(_lib.MegakernelError, match="aligned"):
        kv8.append(c.cache, c.batch, torch.zeros((3, 2, 72), dtype=torch.bfloat16, device="cuda")[:, :, 4:68], k)
    with pytest.raises(ValueError, match="int32"):
        kv8.Batch(c.batch.table.long(), c.batch.q_start, c.batch.kv_len, 3)
    with pytest.raises(ValueError, match="blocks of 8"):
        kv8.Cache.empty(4, 2, 64, block=8)
    with pytest.raises(_lib.MegakernelError, match="workspace"):
        c = Case(16, 2, 64, [3000], [3], seed=18)
        kv8.attention(c.cache, c.batch, q, out, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))


def test_empty_batches():
    c = Case(16, 2, 64, [], [], seed=19)
    q = torch.empty((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    k = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    kv8.append(c.cache, c.batch, k, k)
    kv8.read(c.cache, c.batch, k, torch.empty_like(k))
    kv8.attention(c.cache, c.batch, q, torch.empty_like(q))


# --------------------------------------- splits, both kernels, many sequences
def _hint(c: Case, max_kv: int):
    c.batch = kv8.Batch(c.batch.table, c.batch.q_start, c.batch.kv_len, c.tokens, max_kv)
    return c


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("missing", [0.0, 0.2])
def test_attention_splits(dim, missing):
    """Contexts long enough that few rows are split, among short, empty and
    ragged ones; the workspace is needed, and its initial value does not matter."""
    for block, n_kv, group, lens, new in ((32, 1, 2, [4200], [1]), (16, 2, 3, [4100, 30, 2500, 0, 700], [1, 3, 7, 0, 2]),
                                          (128, 1, 16, [5000, 4999], [2, 1])):
        _say(f"attention splits D={dim} block {block} {lens} {new} missing {missing}")
        c = Case(block, n_kv, dim, lens, new, seed=dim + block, missing=missing)
        need = kv8.workspace_bytes(c.cache, c.batch, n_kv * group)
        assert need > 0
        ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN, in any reading
        _, out = _check_attention(c, n_kv * group, say=str(lens), workspace=ws)
        c.rng = np.random.default_rng(5)
        q = c.rows(n_kv * group, torch.bfloat16).cuda()
        a, b = torch.empty_like(q), torch.empty_like(q)
        kv8.attention(c.cache, c.batch, q, a, workspace=ws)
        kv8.attention(c.cache, c.batch, q, b)
        torch.cuda.synchronize()
        assert torch.equal(a, b)  # the same sums in the same order


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hint,n_kv", [(64, 32), (1 << 20, 1)])
def test_attention_of_many_rows_over_many_steps(dim, hint, n_kv):
    """A prompt's last tokens over a context of more steps than a look-up of
    block ids covers, whole (a hint that is far too short) and split."""
    block, lens, new = 16, [2710 if n_kv == 1 else 1310], [131]
    _say(f"attention many steps D={dim} hint {hint}")
    c = _hint(Case(block, n_kv, dim, lens, new, seed=dim, missing=0.05), hint)
    assert (kv8.workspace_bytes(c.cache, c.batch, 8 * n_kv) > 0) == (hint != 64)
    _check_attention(c, 8 * n_kv)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_many_rows_joined_by_waves(dim):
    """More rows than a workgroup each."""
    _say(f"attention joined by waves D={dim}")
    c = _hint(Case(64, 2, dim, [900], [300], seed=31), 1 << 20)
    assert kv8.workspace_bytes(c.cache, c.batch, 16) > 0 and c.tokens * 16 > 4096
    _check_attention(c, 16)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_a_mixed_batch(dim):
    """Single tokens next to prompts, long and short contexts of each."""
    lens, new = [4300, 600, 40, 1500, 0, 300, 2100], [1, 250, 40, 3, 0, 1, 90]
    _say(f"attention mixed D={dim}")
    for hint in (0, 64, 1 << 20):
        c = _hint(Case(32, 1, dim, lens, new, seed=33, missing=0.03, gap=2), hint)
        _check_attention(c, 2, say=f"hint {hint}")


def test_more_sequences_than_a_wave_has_lanes():
    _say("150 sequences")
    rng = np.random.default_rng(34)
    lens = [int(x) for x in rng.integers(0, 90, 150)]
    new = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 6, 150))]
    lens[70], new[70], lens[130], new[130] = 700, 300, 2600, 1
    c = Case(16, 2, 64, lens, new, seed=35, gap=1)
    k, v = c.rows(2, torch.bfloat16), c.rows(2, torch.bfloat16)
    c.pool.append(c.table, c.start, c.lens, _f64(k), _f64(v))
    kv8.append(c.cache, c.batch, k.cuda(), v.cuda())
    torch.cuda.synchronize()
    c.same_pool()
    _check_attention(c, 4)
    want = [np.full((c.tokens, 2, 64), 7.0) for _ in range(2)]
    c.pool.read(c.table, c.start, c.lens, *want)
    got = [torch.full((c.tokens, 2, 64), 7.0, device="cuda") for _ in range(2)]
    kv8.read(c.cache, c.batch, *got)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        np.testing.assert_array_equal(_f64(g), w)


@pytest.mark.parametrize("n_tokens,hint", [(2, 0), (40, 0), (40, 1 << 20)])
def test_graphs_of_split_contexts(n_tokens, hint):
    """Two captured calls, each with the workspace it took, replayed in turn
    and on two streams at once, against the eager call."""
    _say(f"graphs of splits, {n_tokens} tokens")
    cs = [_hint(Case(32, 2, 64, [4500], [n_tokens], seed=s), hint) for s in (36, 37)]
    qs = [c.rows(8, torch.bfloat16).cuda() for c in cs]
    assert all(kv8.workspace_bytes(c.cache, c.batch, 8) > 0 for c in cs)
    want, outs, graphs = [], [], []
    for c, q in zip(cs, qs):
        o = torch.empty_like(q)
        kv8.attention(c.cache, c.batch, q, o)
        torch.cuda.synchronize()
        want.append(o.clone())
        out = torch.empty_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv8.attention(c.cache, c.batch, q, out)
        outs.append(out)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cs]
    for step in range(6):
        for s, g, o in zip(streams, graphs, outs):
            with torch.cuda.stream(s):
                o.fill_(float("nan"))
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w), f"replay {step}"
        eager = torch.empty_like(qs[0])
        kv8.attention(cs[0].cache, cs[0].batch, qs[0], eager)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])


def test_kv8_on_a_side_stream_behind_its_inputs():
    """A stream that waits for the one that wrote the inputs, as with torch's own operators."""
    _say("side stream")
    c = Case(32, 2, 64, [4400], [1], seed=38)
    q = c.rows(4, torch.bfloat16).cuda()
    want, got = torch.empty_like(q), torch.empty_like(q)
    kv8.attention(c.cache, c.batch, q, want)
    side = torch.cuda.Stream()
    late = torch.zeros_like(q)
    torch.cuda.synchronize()
    for _ in range(8):
        late.zero_()
        late.add_(q)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            kv8.attention(c.cache, c.batch, late, got)
        torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# Which kernel takes a sequence goes by the batch's rows times KV heads and by
# the context lengths that it announces: announced as long, these go to the one
# for many rows (split); announced as short, to the one for few.
TILED = [
    # block, n_kv, group, dim, lens, new
    (16, 2, 3, 64, [90, 40, 17], [90, 33, 5]),
    (64, 1, 2, 128, [150, 66, 3], [140, 1, 3]),
    (128, 1, 1, 128, [257], [257]),
    (32, 1, 8, 64, [300], [64]),
    (32, 1, 16, 128, [300, 5, 80], [70, 1, 3]),
    (16, 1, 16, 64, [100, 1100], [66, 33]),
    (64, 2, 4, 64, [600, 0, 129], [300, 0, 129]),
    (128, 1, 3, 64, [1, 500, 64], [1, 400, 64]),
]


@pytest.mark.parametrize("hint", [64, 1 << 20])
@pytest.mark.parametrize("missing", [0.0, 0.3])
@pytest.mark.parametrize("case", TILED, ids=[f"b{c[0]}h{c[1]}g{c[2]}d{c[3]}n{sum(c[5])}" for c in TILED])
def test_attention_tiles(case, missing, hint):
    block, n_kv, group, dim, lens, new = case
    _say(f"attention tiles {case} missing {missing} hint {hint}")
    c = _hint(Case(block, n_kv, dim, lens, new, seed=block * dim + sum(lens), missing=missing, gap=1), hint)
    _check_attention(c, n_kv * group)


# Enough rows times KV heads for the kernel for many rows with short contexts.
WHOLE = [
    (16, 64, 3, 64, [90, 40, 17, 100], [90, 33, 5, 60]),
    (64, 64, 2, 128, [170, 66, 3], [160, 1, 3]),
    (128, 128, 1, 128, [257], [257]),
    (32, 64, 8, 64, [300], [65]),
    (16, 32, 16, 64, [100, 1100], [66, 33]),
    (64, 64, 1, 64, [600, 0, 129], [500, 0, 129]),
    (32, 128, 2, 64, [1, 500], [1, 129]),
]


@pytest.mark.parametrize("missing", [0.0, 0.3])
@pytest.mark.parametrize("case", WHOLE, ids=[f"b{c[0]}h{c[1]}g{c[2]}d{c[3]}n{sum(c[5])}" for c in WHOLE])
def test_attention_tiles_whole(case, missing):
    block, n_kv, group, dim, lens, new = case
    _say(f"attention whole tiles {case} missing {missing}")
    c = _hint(Case(block, n_kv, dim, lens, new, seed=block * dim + sum(lens), missing=missing, gap=1), 64)
    assert kv8.workspace_bytes(c.cache, c.batch, n_kv * group) == 0
    _check_attention(c, n_kv * group)


# The kernel for few rows has eight, four or two waves by the steps and by how
# many row tiles there are.
WAVES = [
    (16, 2, 2, [1500, 900], [3, 9]),       # eight
    (16, 2, 2, [300, 0, 90], [33, 0, 1]),  # four
    (32, 128, 1, [120, 60], [100, 28]),   # two
    (128, 128, 1, [900, 7], [121, 7]),    # two, and steps for all of them
]


@pytest.mark.parametrize("missing", [0.0, 0.3])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("case", WAVES, ids=[f"b{c[0]}h{c[1]}g{c[2]}n{sum(c[4])}" for c in WAVES])
def test_attention_rows_by_waves(case, dim, missing):
    block, n_kv, group, lens, new = case
    _say(f"attention waves {case} D={dim} missing {missing}")
    c = _hint(Case(block, n_kv, dim, lens, new, seed=dim + sum(lens), missing=missing, gap=1), 2 * 64 if block == 32 else max(lens) // 2)
    assert kv8.workspace_bytes(c.cache, c.batch, n_kv * group) == 0
    _check_attention(c, n_kv * group)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("hint,group", [(1 << 20, 2), (64, 30), (64, 78)])
def test_attention_tiles_never_see_what_they_may_not(dim, hint, group):
    """As the rows' test: NaN in unused blocks, behind the last row, and in
    positions that only some rows of a tile see."""
    _say(f"attention tiles NaN D={dim} hint {hint}")
    c = Case(16, 2, dim, [190, 33, 70], [140, 33, 40], seed=9, missing=0.2)
    used = {int(b) for row, n in zip(c.table, c.lens) for j, b in enumerate(row) if j < -(-int(n) // 16) and 0 <= b < c.pool.n_blocks}
    for b in range(c.pool.n_blocks):
        if b not in used:
            c.pool.k[b], c.pool.v[b] = 0x7F, 0xFF
            c.pool.ks[b], c.pool.vs[b] = np.nan, np.inf
    for row, n in zip(c.table, c.lens):
        b, r = int(row[(n - 1) // 16]), int(n) % 16
        if r and 0 <= b < c.pool.n_blocks:
            c.pool.k[b, :, r:], c.pool.v[b, :, :, r:] = 0xFF, 0x7F
    ks, vs = c.pool.ks.copy(), c.pool.vs.copy()

    def check(nan_ok):
        c.upload()
        _hint(c, hint)
        c.pool.vs[:] = np.where(np.isfinite(vs), vs, 0)  # the tolerance's, of what is seen
        out = _check_attention(c, 2 * group, nan_ok=nan_ok)[1]
        c.pool.ks[:], c.pool.vs[:] = ks, vs
        return out

    check(False)
    at = next(p for p in range(100, 180) if c.pool.place(c.table[0], p))  # rows from at - 50 on see it
    b, r = c.pool.place(c.table[0], at)
    c.pool.v[b, 1, 5, r] = 0x7F
    c.pool.v[b, 1, dim - 1, r] = 0xFF
    b1, r1 = c.pool.place(c.table[1], next(p for p in range(3, 33) if c.pool.place(c.table[1], p)))
    c.pool.v[b1, 0, 9, r1] = 0xFF
    out = check(True)
    assert torch.isnan(out[at - 50, 2 * group - 1, 5]) and torch.isnan(out[139, group, dim - 1])
    assert not torch.isnan(out[: at - 50]).any() and not torch.isnan(out[:140, :group]).any()
    c.pool.k[b, 0, r, 7] = 0x7F  # a NaN key makes the whole row NaN
    out = check(True)
    assert torch.isnan(out[at - 50 : 140, :group]).all() and not torch.isnan(out[: at - 50]).any()


def test_attention_tiles_extremes():
    _say("attention tiles extremes")
    c = Case(32, 2, 64, [150, 80], [100, 20], seed=10)
    for ke, ve, qs in ((9, 100, 3.0), (-100, -100, 1.0), (20, 0, 1e-3)):
        c.pool.ks[:], c.pool.vs[:] = 2.0 ** ke, 2.0 ** ve
        c.upload()
        _hint(c, 1 << 20)
        q = c.rows(4, torch.bfloat16, qs)
        _check_attention(c, 4, scale=2.0 ** -10 if ke == 9 else None, q=q, say=f"{ke} {ve}")


def test_attention_tiles_negative_positions_and_rising_maxima():
    """Rows that see nothing in a tile of rows that do; keys that grow with the
    position, so that the running maximum rises at every step."""
    _say("attention tiles negative positions")
    c = Case(16, 1, 64, [50, 700], [90, 300], seed=40)
    for row, n in zip(c.table, c.lens):
        for p in range(int(n)):
            b, r = c.pool.place(row, p)
            c.pool.k[b, :, r] = 0x38
            c.pool.ks[b] = 2.0 ** (p // 16 // 4 - 8)
    c.upload()
    _hint(c, 1 << 20)
    q = c.rows(3, torch.bfloat16, 0.5) + 0.25
    _, out = _check_attention(c, 3, q=q)
    assert torch.all(out[:40] == 0)


def test_more_rows_than_workgroups_of_one_launch():
    """2^25 rows of heads, most of them before position 0: zeros."""
    _say("2^20 tokens")
    tokens = 1 << 20
    c = Case(32, 8, 64, [40], [40], seed=40)
    q = c.rows(32, torch.bfloat16)
    want, out = np.zeros((40, 32, 64)), torch.empty((tokens, 32, 64), dtype=torch.bfloat16, device="cuda")
    size, reach = c.pool.attention(c.table, c.start, c.lens, _f64(q), want, 64 ** -0.5)
    many = torch.zeros((tokens, 32, 64), dtype=torch.bfloat16, device="cuda")
    many[-40:] = q.cuda()
    start = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    batch = kv8.Batch(c.batch.table, start, c.batch.kv_len, tokens)
    kv8.attention(c.cache, batch, many, out)
    torch.cuda.synchronize()
    tol = np.abs(want) * 2.0 ** -8 + (2.0 ** -8 + (2 * 64 * reach + 40 + 16)[..., None] * U) * size
    assert np.all(np.abs(_f64(out[-40:]) - want) <= tol)
    assert not out[:-40].any()


@pytest.mark.parametrize("dim,group", [(64, 71), (64, 64), (128, 66), (128, 33), (128, 32)])
def test_attention_of_more_query_heads_than_the_kernel_for_few_rows_takes(dim, group):
    """A prompt and a short sequence: a single token has more rows than the
    limit between the kernels, or as many."""
    _say(f"attention of {group} query heads per KV head D={dim}")
    for new in ([1020, 4], [1, 1023]):
        c = _hint(Case(64, 1, dim, [1023, 1023], new, seed=group, gap=0), 4096)
        _check_attention(c, group, say=str(new))


@pytest.mark.parametrize("dim", [64, 128])
def test_a_late_key_that_decides_a_row(dim):
    """The first key's score is a row's reference; a key of a later step of the
    same wave, less than 2^8 times as heavy, decides the row.  Weights are
    rounded to bf16, relative h = 2^-8, but their sum is that of the rounded
    ones, so an output is off by its own rounding, |o| h, and by
    h sum_j p_j |v_j - o| (1 + 2 h, as the sum is off by h): near nothing where
    the deciding key's value is the output.  Terms of fp32, 16 u and 2 D u of a
    score of 8, as in the general tolerance."""
    _say(f"late key D={dim}")
    h, block = 2.0 ** -8, 16
    late = 4 * 64 + 5  # waves take every fourth step: positions 0 and 261 are one wave's
    for weight in (1 + 0.97 * h, 128 * (1 + 0.97 * h), 180.37, 3 * (1 + 0.65 * h), 254.6):
        c = Case(block, 1, dim, [late + 1], [1], seed=41)
        c.table[:] = -1
        c.table[0, 0], c.table[0, late // block] = 0, 1
        c.pool.ks[:], c.pool.vs[:] = 1.0, 1.0
        c.pool.k[:] = 0
        c.pool.k[:, :, :, 0] = 0xF7  # -240: the other keys of the two blocks
        c.pool.k[0, 0, 0, 0] = 0x00
        c.pool.k[1, 0, late % block, 0] = 0x50  # 8
        c.pool.v[0, 0, :, 0] = c.pool.v[1, 0, :, late % block] = 0x38 + np.arange(dim) % 8  # 1, 1.125, .. 1.875
        c.pool.v[0, 0, 0, 0] = 0xB8  # and one dimension in which they differ
        c.upload()
        _hint(c, 64)
        assert kv8.workspace_bytes(c.cache, c.batch, 1) == 0
        q = torch.zeros((1, 1, dim), dtype=torch.bfloat16)
        q[..., 0] = 1
        scale, want = float(np.log(weight) / 8), np.zeros((1, 1, dim))
        c.pool.attention(c.table, c.start, c.lens, _f64(q), want, scale)
        out = torch.empty((1, 1, dim), dtype=torch.bfloat16, device="cuda")
        kv8.attention(c.cache, c.batch, q.cuda(), out, scale=scale)
        torch.cuda.synchronize()
        there = [c.pool.place(c.table[0], j) for j in range(late + 1)]
        keys, v = (np.stack([c.pool.values(*at)[i][0] for at in there if at]) for i in (0, 1))
        p = np.exp(keys[:, 0] * scale)  # the first key's is 1
        assert p.max() == p[-1] and abs(p[-1] / weight - 1) < 1e-12
        p /= p.sum()
        o = p @ v
        np.testing.assert_allclose(o, want[0, 0], rtol=1e-9)
        size = p @ np.abs(v)
        tol = np.abs(o) * h + (p @ np.abs(v - o)) * h * (1 + 2 * h) + (16 + 2 * dim * 8) * U * size
        off = np.abs(_f64(out)[0, 0] - o)
        assert np.all(off <= tol), f"weight {weight}: {np.max(off / tol):.2f} of the tolerance"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_rows_at_the_end_of_the_range_are_read_back_finite(dim, src):
    """The type's lowest and largest values, those around the last that fits,
    1.75 * 2^127, and infinities beside them."""
    _say(f"rows of the lowest value D={dim} {src}")
    last = 1.75 * 2.0 ** 127
    values = [torch.finfo(src).min, torch.finfo(src).max, last, last * (1 + 2.0 ** -7), 1.9375 * 2.0 ** 127, last * (1 - 2.0 ** -8)]
    for block in (16, 64):
        c = Case(block, 2, dim, [block + 3, 9], [block + 1, 9], seed=42)
        k, v = c.rows(2, src), c.rows(2, src)
        for i, x in enumerate(values):
            k[i + 2, i % 2, 7 * i], v[i + 1, 1 - i % 2, 9 * i] = x, -x
        v[3, 0, 1], k[0] = np.inf, torch.finfo(src).min
        c.pool.append(c.table, c.start, c.lens, _f64(k), _f64(v))
        assert c.pool.ks.max() == c.pool.vs.max() == 2.0 ** 119
        kv8.append(c.cache, c.batch, k.cuda(), v.cuda())
        torch.cuda.synchronize()
        c.same_pool()
        for dst in (torch.bfloat16, torch.float32):
            want = [np.zeros(k.shape) for _ in range(2)]
            c.pool.read(c.table, c.start, c.lens, *want)
            got = [torch.empty(k.shape, dtype=dst, device="cuda") for _ in range(2)]
            kv8.read(c.cache, c.batch, *got)
            torch.cuda.synchronize()
            for g, w in zip(got, want):
                assert np.isfinite(w).all()
                np.testing.assert_array_equal(_f64(g), w)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,n_kv,hint", [(2, 1, 64), (80, 2, 64), (2, 2, 1 << 20)])
def test_rows_of_the_lowest_value_reach_no_row_that_does_not_see_them(dim, group, n_kv, hint):
    """Padding rows of the type's lowest value behind a sequence's own, and
    codes of 448 that an earlier sequence left behind both.  The sequence's own
    rows are held to the general tolerance (what they see is below 448 * 2^-3),
    those at the padding's positions to nothing."""
    _say(f"lowest value unseen D={dim} group {group} hint {hint}")
    lens, own = [190, 70], [185, 61]
    c = Case(32, n_kv, dim, lens, [140, 40], seed=43)
    c.pool.k[:], c.pool.v[:] = np.where(c.pool.k == 0x60, 0x7E, c.pool.k), np.where(c.pool.v == 0x60, 0x7E, c.pool.v)
    c.upload()
    k, v = (c.rows(n_kv, torch.bfloat16) for _ in range(2))
    for i, n in enumerate(own):
        first = int(c.start[i + 1]) - (lens[i] - n)
        k[first : c.start[i + 1]] = v[first : c.start[i + 1]] = torch.finfo(torch.bfloat16).min
    c.pool.append(c.table, c.start, c.lens, _f64(k), _f64(v))
    kv8.append(c.cache, c.batch, k.cuda(), v.cuda())
    torch.cuda.synchronize()
    c.same_pool()
    _hint(c, hint)
    q = c.rows(n_kv * group, torch.bfloat16, 1.5)
    want, out = np.zeros(q.shape), torch.empty_like(q, device="cuda")
    size, reach = c.pool.attention(c.table, c.start, c.lens, _f64(q), want, dim ** -0.5)
    kv8.attention(c.cache, c.batch, q.cuda(), out)
    torch.cuda.synchronize()
    got = _f64(out)
    for i, n in enumerate(own):
        rows = slice(int(c.start[i]), int(c.start[i + 1]) - (lens[i] - n))
        w, n_seen = want[rows], lens[i]
        tol = np.abs(w) * 2.0 ** -8 + (2.0 ** -8 + (2 * dim * reach[rows] + n_seen + 16)[..., None] * U) * size[rows]
        tol += n_seen * 2.0 ** -126 * 448 * 2.0 ** -3
        n_bad = int((~(np.abs(got[rows] - w) <= tol)).sum())
        assert n_bad == 0, f"sequence {i}: {n_bad} outputs off"


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_tiles_refresh_their_block_ids(dim):
    """attn_tile looks block ids up 16 steps of 64 positions at a time, the
    first two such windows before it starts; a whole context of 79 steps
    refreshes each of their two places at least once.  Three of the KV heads are
    compared, of a pool that has only them."""
    block, n_kv, lens, new = 16, 64, [5003], [449]
    _say(f"attention tiles, 79 steps D={dim}")
    c = _hint(Case(block, n_kv, dim, lens, new, seed=44 + dim, missing=0.05), 64)
    assert kv8.workspace_bytes(c.cache, c.batch, n_kv) == 0  # whole
    q, out = c.rows(n_kv, torch.bfloat16, 1.5), torch.full((c.tokens, n_kv, dim), 5.0, dtype=torch.bfloat16, device="cuda")
    kv8.attention(c.cache, c.batch, q.cuda(), out)
    torch.cuda.synchronize()
    heads, p = [0, 31, 63], c.pool
    some = okv8.Pool(p.k[:, heads], p.v[:, heads], p.ks[:, heads], p.vs[:, heads])
    want = np.zeros((c.tokens, 3, dim))
    size, reach = some.attention(c.table, c.start, c.lens, _f64(q[:, heads]), want, dim ** -0.5)
    tol = np.abs(want) * 2.0 ** -8 + (2.0 ** -8 + (2 * dim * reach + lens[0] + 16)[..., None] * U) * size
    n_bad = int((~(np.abs(_f64(out[:, heads]) - want) <= tol)).sum())
    assert n_bad == 0, f"{n_bad} outputs off"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [33100, 131300])
def test_attention_of_one_row_in_hundreds_of_parts(dim, length):
    """A part is 8 steps of 64 positions at least: 65 parts, one more than
    attn_join reads at once, and 257, of which 256 are the most."""
    _say(f"attention of {length} positions D={dim}")
    c = Case(128, 1, dim, [length], [1], seed=45, missing=0.02)
    assert kv8.workspace_bytes(c.cache, c.batch, 3) > 0
    _check_attention(c, 3)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [20100, 131300])
def test_attention_of_hundreds_of_parts_joined_by_waves(dim, length):
    """A single token over 40 and 256 parts (a wave reads 32 at a time, 16 of
    head_dim 128) beside a prompt, which makes the rows too many for a
    workgroup each."""
    _say(f"attention of {length} positions beside a prompt D={dim}")
    c = _hint(Case(128, 1, dim, [length, 300], [1, 300], seed=46, missing=0.02), 1 << 20)
    assert kv8.workspace_bytes(c.cache, c.batch, 16) > 0 and c.tokens * 16 > 4096
    _check_attention(c, 16)


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_one_tile_in_dozens_of_parts(dim):
    """120 rows of 60 tokens, more than attn_rows takes where contexts may be
    long: 315 steps in parts of 4."""
    _say(f"one tile of 20,100 positions D={dim}")
    c = _hint(Case(64, 1, dim, [20100], [60], seed=47, missing=0.02), 1 << 20)
    assert kv8.workspace_bytes(c.cache, c.batch, 2) > 0
    _check_attention(c, 2)


def test_gradients_that_would_be_lost_are_refused():
    _say("gradients")
    c = Case(16, 2, 64, [20], [3], seed=48)
    q, k = c.rows(4, torch.bfloat16).cuda(), c.rows(2, torch.bfloat16).cuda()
    gain = torch.nn.Parameter(torch.ones(64, dtype=torch.bfloat16, device="cuda"))
    inv, pos = torch.ones(32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    wants = k.clone().requires_grad_()
    calls = [lambda: kv8.qk_norm_rope(q, k, gain, gain, inv, pos, torch.empty_like(q), torch.empty_like(k)),
             lambda: kv8.append(c.cache, c.batch, wants, k), lambda: kv8.read(c.cache, c.batch, torch.empty_like(k), wants),
             lambda: kv8.attention(c.cache, c.batch, torch.nn.Parameter(q), torch.empty_like(q))]
    for call in calls:
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()
    torch.cuda.synchronize()
