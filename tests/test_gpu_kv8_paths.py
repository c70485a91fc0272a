"""GPU parity of the paged 8-bit KV cache's operators on the kernels that long
prompts and large batches run, against oracle/kv8.py (64 bits) with the tolerances
of test_gpu_kv8_more.py.  A window cuts the contexts that the attention's kernel is
chosen by, so each test that means one kernel says so and asks which it is."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from megakernel_amd import kv8
from oracle import fp8
from oracle import kv8 as okv8
from tests import test_gpu_kv8_more as more
from tests.test_gpu_kv8 import U, Case, _f64, _hint, _say

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -126


def _kernels(c, n_q, x):
    return kv8.attention_kernels(c.cache, c.batch, n_q, more._given(x))


def _some(c, every, seed):
    """Every so many of the batch's tokens, and the first and last of each sequence."""
    at = set(range(int(c.start[0]) + seed % every, int(c.start[-1]), every))
    for a, b in zip(c.start[:-1], c.start[1:]):
        at |= {int(a), int(b) - 1} if b > a else set()
    return at


# ------------------------------------------------- the kernel for many rows
KINDS = ["window 1", "window 20", "window 64", "window 129", "documents", "nothing", "prefix", "long prefix", "rising", "all"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block,n_kv,group,dim,lens,new", [(16, 64, 2, 64, [390], [240]), (32, 64, 2, 128, [280], [171]),
                                                           (64, 64, 3, 64, [200, 45, 9], [170, 1, 9]), (16, 64, 3, 128, [190, 45], [131, 2])])
def test_scores_in_tiles_of_128_rows(block, n_kv, group, dim, lens, new, kind):
    """Whole contexts in the kernel for many rows, alone and beside sequences of few."""
    n_q = n_kv * group
    c = Case(block, n_kv, dim, lens, new, seed=block + dim + sum(lens), missing=0.1)
    x = more._scores_of(kind, c, n_q)
    _say(f"tiles {block} {n_kv}x{group} D={dim} {lens} {kind} {_kernels(c, n_q, x)}")
    assert _kernels(c, n_q, x) == ({"tile"} if len(lens) == 1 else {"rows", "tile"})
    more._check(c, n_q, x, tokens=_some(c, 19, KINDS.index(kind)), mass=False)


@pytest.mark.parametrize("dim,n_kv,tokens,window", [(64, 64, 240, 2900), (128, 16, 550, 2100)])
def test_scores_in_split_tiles_under_a_window(dim, n_kv, tokens, window):
    """A window that is long enough for its tiles to be split; blocks before it were
    never written, and hold NaN codes and NaN scales."""
    length, n_q = window + tokens + 500, 2 * n_kv
    c = Case(128, n_kv, dim, [length], [tokens], seed=dim, fill=False)
    x = okv8.Scores(window=window)
    seen = length - tokens + 1 - window  # the first position that some row sees
    for j in range(seen // 128, len(c.table[0])):
        b = int(c.table[0, j])
        c.pool.k[b], c.pool.v[b] = (c.rng.integers(0, 0x60, s).astype(np.uint8) for s in (c.pool.k[b].shape, c.pool.v[b].shape))
        c.pool.ks[b], c.pool.vs[b] = 2.0 ** -6, 2.0 ** -3
    c.table[0, seen // 128 + 3] = -1
    c.upload()
    _say(f"split tiles under a window D={dim} {_kernels(c, n_q, x)}")
    assert {"tile", "tile split"} <= _kernels(c, n_q, x)
    rows = {0, 1, 63, 64, tokens // 2, tokens - 2, tokens - 1}
    more._check(c, n_q, x, tokens=rows, mass=False)
    more._check(c, n_q, okv8.Scores(window=window, softcap=20.0), tokens=rows, mass=False)


@pytest.mark.parametrize("dim,tokens", [(64, 240), (128, 171)])
@pytest.mark.parametrize("block", [16, 32])
def test_tiles_leave_unseen_garbage_out(dim, tokens, block):
    """A fresh pool holds NaN codes and NaN scales; blocks before a window or a
    document were never written, a block that some rows see is missing."""
    length, n_kv, n_q = tokens + 90, 64, 128
    for x, seen in ((okv8.Scores(window=22), 69), (okv8.Scores(window=1), 90), (okv8.Scores(first=np.full(tokens, 70)), 70),
                    (okv8.Scores(window=64, first=np.full(tokens, 33), softcap=9.0), 33)):
        c = Case(block, n_kv, dim, [length], [tokens], seed=22, fill=False)
        for j in range(seen // 16 * 16 // block, len(c.table[0])):
            b = int(c.table[0, j])
            c.pool.k[b], c.pool.v[b] = (c.rng.integers(0, 0x60, s).astype(np.uint8) for s in (c.pool.k[b].shape, c.pool.v[b].shape))
            c.pool.ks[b], c.pool.vs[b] = 2.0 ** -6, 2.0 ** -3
        c.table[0, 160 // block] = -1
        c.upload()
        _say(f"tiles and garbage D={dim} block {block} window {x.window} from {seen} {_kernels(c, n_q, x)}")
        assert _kernels(c, n_q, x) == {"tile"}
        more._check(c, n_q, x, tokens=_some(c, 17, seen), mass=False)


@pytest.mark.parametrize("dim", [64, 128])
def test_split_tiles_leave_garbage_before_documents_out(dim):
    """Documents alone, announced as long: the kernel for many rows, split."""
    c = Case(16, 2, dim, [400], [60], seed=23, fill=False)
    for j in range(128 // 16, len(c.table[0])):
        b = int(c.table[0, j])
        c.pool.k[b], c.pool.v[b], c.pool.ks[b], c.pool.vs[b] = 0x38, 0xB8, 0.5, 0.25
    c.table[0, 12] = -1
    c.upload()
    _hint(c, 1 << 20)
    for first in (128, 131, 143, 201):  # in the first run of 16, and steps further on
        x = okv8.Scores(first=np.where(np.arange(60) % 7, first, 300))
        _say(f"split tiles and garbage D={dim} first {first} {_kernels(c, 4, x)}")
        assert {"tile", "tile split"} <= _kernels(c, 4, x)
        more._check(c, 4, x)


@pytest.mark.parametrize("dim,tokens", [(64, 240), (128, 171)])
def test_tiles_keep_nan_from_rows_that_do_not_see_it(dim, tokens):
    """NaN before a window, before a document and behind a prefix, in steps that
    some rows of a tile see whole, some in part and some not at all."""
    n_kv, n_q, past = 64, 128, 50
    c = Case(16, n_kv, dim, [past + tokens], [tokens], seed=24)
    b = [int(c.table[0, p // 16]) for p in range(past + tokens)]
    c.pool.v[b[70], :, 5, 70 % 16] = 0x7F
    c.pool.v[b[3], 0, 9, 3] = 0xFF
    c.pool.k[b[64], 1, 0, 7] = 0x7F
    c.upload()
    x = okv8.Scores(window=30, prefix=[60])
    _say(f"tiles and NaN D={dim} {_kernels(c, n_q, x)}")
    assert _kernels(c, n_q, x) == {"tile"}
    near = {t for p in (50, 59, 60, 63, 64, 69, 70, 93, 94, 99, 100, 127, 128) for t in (p - past, p - past + 1)} | {tokens - 1}
    _, out, _, _ = more._check(c, n_q, x, nan_ok=True, tokens=near, mass=False)
    assert torch.isnan(out[20:50, :2, 5]).all() and not torch.isnan(out[50:, :2]).any()       # 70 is seen from 70 to 99
    assert not torch.isnan(out[:14, 2:4, 5]).any() and torch.isnan(out[14:44, 2:4]).all()     # key 64, of KV head 1, from 64 to 93
    docs = okv8.Scores(first=np.where(np.arange(past, past + tokens) >= 80, 71, 4))
    assert _kernels(c, n_q, docs) == {"tile"}
    _, out, _, _ = more._check(c, n_q, docs, nan_ok=True, tokens=near, mass=False)
    assert torch.isnan(out[20:30, :, 5]).all() and not torch.isnan(out[30:, 0]).any()


# ---------------------------------------------------- the kernel for few rows
@pytest.mark.parametrize("kind", ["cap", "slopes", "window 129", "documents", "prefix", "all"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n_kv,lens,hint", [(64, [90, 300, 1, 64] * 8, 300), (64, [700, 33, 650, 129, 700], 700), (2, [700, 80, 640], 700)],
                         ids=["two waves", "four waves", "eight waves"])
def test_scores_of_workgroups_of_two_to_eight_waves(n_kv, lens, hint, dim, kind):
    """Many short contexts (2,048 workgroups of at most five steps), more workgroups
    than CUs (320, eleven steps), and few (6)."""
    n_q = 2 * n_kv
    c = _hint(Case(32, n_kv, dim, lens, [1] * len(lens), seed=dim + n_kv, missing=0.05), hint)
    x = more._scores_of(kind, c, n_q)
    _say(f"waves {n_kv} heads {len(lens)} sequences D={dim} {kind} {_kernels(c, n_q, x)}")
    assert _kernels(c, n_q, x) == {"rows"}
    more._check(c, n_q, x)


# --------------------------------------------------------- the join by waves
@pytest.mark.parametrize("kind", ["cap", "slopes", "documents", "nothing", "prefix", "all"])
@pytest.mark.parametrize("dim,n_kv,group,lens,new", [(64, 2, 3, [900], [700]), (128, 2, 3, [900], [700]), (64, 1, 7, [700, 5, 400], [400, 5, 250]),
                                                     (128, 3, 3, [800, 33], [500, 1])])
def test_scores_joined_by_waves(dim, n_kv, group, lens, new, kind):
    """More rows than a workgroup each, four heads of a token to a wave, with heads
    left over; _check() runs every call without and with log-sum-exps."""
    n_q = n_kv * group
    c = _hint(Case(16, n_kv, dim, lens, new, seed=dim + n_q, missing=0.05), 1 << 20)
    x = more._scores_of(kind, c, n_q)
    if kind == "all":
        x.window = 0  # a short window leaves nothing to split
    _say(f"joined by waves D={dim} {n_kv}x{group} {lens} {kind} {_kernels(c, n_q, x)}")
    assert {"tile split", "join by waves"} <= _kernels(c, n_q, x) and n_q % 4
    more._check(c, n_q, x, tokens=_some(c, 11, len(kind)), mass=False)


# ------------------------------------------------------------------- rotary
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("src,dst", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                     (torch.float32, torch.float32)])
@pytest.mark.parametrize("tokens,n_q,n_kv,dim,turned,layout", [
    (4701, 7, 1, 128, 64, "packed"), (4801, 5, 2, 128, 128, "in place"), (1101, 3, 2, 1024, 512, "heads"), (5501, 9, 3, 80, 16, "in place"),
    (9001, 3, 1, 128, 32, "in place"), (5303, 2, 1, 272, 272, "packed")])
def test_rotary_of_four_heads_a_thread(tokens, n_q, n_kv, dim, turned, layout, src, dst, interleaved):
    """Twice as many pieces as a thread takes four heads from on: head counts that are
    no multiple of four and one that is, parts and all of a head, all layouts."""
    assert tokens * (dim // 16) * (n_q + n_kv) > 1 << 18
    more.test_rotary(tokens, n_q, n_kv, dim, turned, layout, src, dst, interleaved)


# -------------------------------------------------------------------- weigh
def _check_weigh(c, n_q, x):
    """lse and weights of every row against 64 bits, one head after the other."""
    q = c.rows(n_q, torch.bfloat16, 1.5)
    given, width = more._given(x), c.table.shape[1] * c.block
    out, lse = torch.empty((c.tokens, n_q, c.dim), dtype=torch.bfloat16, device="cuda"), torch.empty((c.tokens, n_q), device="cuda")
    old = torch.from_numpy(c.rng.random((len(c.lens), c.n_kv, width), dtype=np.float32))
    mass, qc = old.cuda(), q.cuda()
    kv8.attention(c.cache, c.batch, qc, out, scores=given, lse=lse)
    kv8.weigh(c.cache, c.batch, qc, lse, mass, scores=given)
    torch.cuda.synchronize()
    got, got_lse, group, scale = _f64(mass), _f64(lse), n_q // c.n_kv, c.dim ** -0.5
    table = fp8.e4m3_decode_table().astype(np.float64)
    for i, length in enumerate(int(v) for v in c.lens):
        a, b = int(c.start[i]), int(c.start[i + 1])
        ids = c.table[i, : -(-length // c.block)]
        there = np.repeat((ids >= 0) & (ids < c.pool.n_blocks), c.block)[:length]
        ids = np.where((ids >= 0) & (ids < c.pool.n_blocks), ids, 0)
        p, j = np.arange(length - (b - a), length)[:, None], np.arange(length)[None]
        spans = np.array([x.span(i, t, length - b + t, length) for t in range(a, b)])
        seen = (j >= spans[:, :1]) & (j < spans[:, 1:]) & there
        for h in range(c.n_kv):
            keys = (table[c.pool.k[ids, h]] * c.pool.ks[ids, h][:, None, None]).reshape(-1, c.dim)[:length]
            want, tol = np.zeros(length), np.zeros(length)
            want[: length - (b - a)] = _f64(old[i, h, : length - (b - a)])
            tol += ((b - a) * group + 32) * U * np.abs(want)
            for hd in range(h * group, (h + 1) * group):
                qh = _f64(q[a:b, hd])
                s = qh @ keys.T * scale
                reach = (np.abs(qh) @ np.abs(keys).T * scale).max(1)
                if x.softcap:
                    s = x.softcap * np.tanh(s / x.softcap)
                s[~seen] = -np.inf
                top = s.max(1, keepdims=True)
                none = np.isinf(top[:, 0])
                top[none] = 0
                w = np.exp(s - top)
                total = w.sum(1, keepdims=True)
                with np.errstate(divide="ignore"):
                    ref = top + np.log(total)
                w /= np.where(none[:, None], 1, total)
                big = np.abs(np.where(seen, s, 0)).max(1)
                e = (c.dim + 3) * U * reach + 10 * U * x.softcap + 3 * U * big
                ref0 = np.where(none, 0, ref[:, 0])
                tol_lse = e + (length + 16) * U + 4 * U * np.abs(ref0) + length * TINY
                assert np.all((np.abs(got_lse[a:b, hd] - ref[:, 0]) <= tol_lse) | (got_lse[a:b, hd] == ref[:, 0])), (i, hd)
                want += w.sum(0)
                per_row = 2 * e + tol_lse + 4 * U * (big + np.abs(ref0)) + ((b - a) * group + 36) * U
                tol += (w * per_row[:, None]).sum(0) + (b - a) * TINY
            off = np.abs(got[i, h, :length] - want) > tol
            assert not off.any(), (i, h, int(off.sum()), np.argwhere(off)[:3].ravel(), got[i, h, :length][off][:3], want[off][:3], tol[off][:3])
            assert np.array_equal(got[i, h, length:], _f64(old[i, h, length:]))


@pytest.mark.parametrize("x", [okv8.Scores(), okv8.Scores(window=900, softcap=30.0)], ids=["plain", "capped window"])
@pytest.mark.parametrize("dim", [64, 128])
def test_weights_by_waves_that_take_several_steps(dim, x):
    """More steps times KV heads than run at once, few rows: 16 workgroups a head for
    34 times four steps of two sequences."""
    _say(f"weights, waves of several steps D={dim}")
    c = Case(64, 256, dim, [4300, 800], [1, 2], seed=dim, missing=0.02)
    assert -(-4300 // 64) * 2 // 4 > 4096 // 256
    _check_weigh(c, 256, x)


@pytest.mark.parametrize("dim,lens,new,kind", [(64, [1400], [1400], "plain"), (64, [1400], [1400], "capped window"), (128, [1340], [620], "plain"),
                                               (128, [1340], [620], "capped window"), (128, [1340], [620], "documents")])
def test_weights_by_workgroups_that_take_several_steps(dim, lens, new, kind):
    """The same with many rows, more than waves are ever given: 16 workgroups a head
    for 22 (21) steps."""
    _say(f"weights, workgroups of several steps D={dim} {kind}")
    c = Case(32, 256, dim, lens, new, seed=dim + 1, missing=0.02)
    assert -(-lens[0] // 64) > 4096 // 256 and new[0] > (1280 if dim == 64 else 512)
    pos = np.arange(lens[0] - new[0], lens[0])
    _check_weigh(c, 256, {"plain": okv8.Scores(), "capped window": okv8.Scores(window=300, softcap=30.0),
                          "documents": okv8.Scores(first=pos // 211 * 211)}[kind])


@pytest.mark.parametrize("kind", ["plain", "documents", "all"])
@pytest.mark.parametrize("dim,n_kv,group,lens,new", [(64, 64, 1, [620], [330]), (64, 64, 3, [640], [120]), (128, 64, 1, [620], [330]),
                                                     (128, 64, 5, [700], [80]), (64, 8, 2, [4096], [64]), (128, 4, 40, [900, 90], [9, 6])])
def test_weights_by_workgroups(dim, n_kv, group, lens, new, kind):
    """Half as many rows again as workgroups of 64 positions pay from on (a third of the
    steps, or 80), heads that fill a tile, and more than it has rows."""
    n_q, items = n_kv * group, -(-max(lens) // 64) * len(lens) * n_kv
    _say(f"weights by workgroups D={dim} {n_kv}x{group} {lens} {kind}")
    c = Case(16, n_kv, dim, lens, new, seed=dim + group, missing=0.1, gap=1)
    assert sum(new) * group >= 1.5 * len(lens) * (80 if items <= 256 or items == 512 else items / 3)
    more._check(c, n_q, more._scores_of(kind, c, n_q))
