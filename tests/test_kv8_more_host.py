"""Scores, weights, eviction and rotary positions of the paged 8-bit KV cache on
the CPU: the oracle against closed forms, the frequencies, and what the entry
points refuse before any GPU work (the addresses below are never dereferenced)."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from megakernel_amd import _lib, kv8
from oracle import kv8 as okv8
from tests.test_kv8_host import BAD_BATCHES, BAD_CACHES, BAD_ROWS, FAKE, _batch, _cache, _r, _ref, _refused, clib  # noqa: F401


def _x(**kw):
    d = dict(slopes=None, first=None, prefix=None, softcap=0.0, window=0)
    d.update(kw)
    return kv8._CScores(*(d[n] for n, _ in kv8._CScores._fields_))


def _mass(p=4 * FAKE, ts=1024, hs=128, type=0):  # 2 sequences, 8 heads, 128 positions
    return kv8._Rows(p, ts, hs, type)


# ------------------------------------------------------------------ oracle
def _pool(rng, blocks=6, heads=2, block=16, dim=64):
    k, v = rng.integers(0, 0x48, (blocks, heads, block, dim)), rng.integers(0, 0x48, (blocks, heads, dim, block))
    return okv8.Pool(k, v, np.full((blocks, heads), 0.25), np.full((blocks, heads), 0.5))


def test_oracle_scores_without_anything_are_the_causal_attention():
    rng = np.random.default_rng(0)
    pool, table, start, lens = _pool(rng), np.array([[3, -1, 1], [0, 5, -1]]), [0, 3, 4], [40, 20]
    q, out = rng.standard_normal((4, 4, 64)), np.zeros((4, 4, 64))
    pool.attention(table, start, lens, q, out, 0.1)
    n = 0
    for i, t, h, j, s, w, v, reach, bias in okv8.scored_rows(pool, table, start, lens, q, 0.1, okv8.Scores()):
        np.testing.assert_allclose(w @ v, out[t, h], rtol=1e-12)
        assert bias == 0 and abs(s).max() <= reach
        n += 1
    assert n == 16


def test_oracle_spans():
    x = okv8.Scores(window=4, first=[0, 7, 2], prefix=[5])
    assert x.span(0, 0, 9, 100) == (6, 10)
    assert x.span(0, 1, 9, 100) == (7, 10)
    assert x.span(0, 2, 1, 100) == (2, 5) and x.span(0, 0, 1, 3) == (0, 3)
    assert x.span(0, 0, -1, 100) == (0, 0)


def test_oracle_caps_bound_scores_and_slopes_fall_with_distance():
    rng = np.random.default_rng(1)
    pool, q = _pool(rng), rng.standard_normal((1, 2, 64)) * 9
    x = okv8.Scores(softcap=2.0, slopes=[0.5, 0.25])
    for _, _, h, j, s, *_ in okv8.scored_rows(pool, [[0, 1]], [0, 1], [32], q, 1.0, x):
        assert np.all(np.abs(s + [0.5, 0.25][h] * (31 - j)) <= 2.0)


def test_oracle_selection_by_hand():
    m = [5.0, 1.0, 3.0, 3.0, 3.0, math.nan, 9.0, 0.0]
    assert okv8.select(m, 8, 4, 0, 0) == [0, 2, 3, 6]  # of equal weights the lower positions
    assert okv8.select(m, 8, 4, 2, 1) == [0, 2, 6, 7]
    assert okv8.select(m, 8, 8, 2, 1) == list(range(8)) and okv8.select(m, 3, 8, 2, 1) == [0, 1, 2]
    assert okv8.select(m, 6, 5, 0, 0) == [0, 1, 2, 3, 4]  # NaN goes first


def test_oracle_compaction_of_every_row_keeps_values():
    rng = np.random.default_rng(2)
    pool = _pool(rng)
    want = [pool.values(*pool.place([3, 1], p)) for p in range(20)]
    kept = np.broadcast_to(np.arange(20), (1, 2, 20))
    okv8.compact(pool, [[3, 1]], kept, [20], [[0, 4]])
    for p in range(20):
        for a, b in zip(pool.values(*pool.place([0, 4], p)), want[p]):
            # a smaller scale holds the values exactly; none is larger than the old one
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotary_turns_pairs_and_leaves_the_rest(interleaved):
    rng = np.random.default_rng(3)
    x, inv = rng.standard_normal((3, 2, 10)), np.array([1.0, 0.1, 0.01])
    y, _ = okv8.rotary(x, inv, [0, 5, -7], interleaved, 2.0)
    np.testing.assert_array_equal(y[..., 6:], x[..., 6:])
    np.testing.assert_allclose(y[0, :, :6], 2 * x[0, :, :6], rtol=1e-15)
    np.testing.assert_allclose((y[..., :6] ** 2).sum(-1), 4 * (x[..., :6] ** 2).sum(-1), rtol=1e-12)
    a, b = (0, 1) if interleaved else (0, 3)
    z = (x[1, :, a] + 1j * x[1, :, b]) * np.exp(5j) * 2
    np.testing.assert_allclose([y[1, :, a], y[1, :, b]], [z.real, z.imag], rtol=1e-12)


# ------------------------------------------------------------- frequencies
def test_frequencies():
    plain, a = kv8.rotary_frequencies(64, 1e4, device="cpu")
    np.testing.assert_allclose(plain.double().numpy(), 1e4 ** (-np.arange(32) / 32), rtol=2.0 ** -23)
    assert a == 1.0 and plain.dtype == torch.float32
    linear, a = kv8.rotary_frequencies(64, 1e4, "linear", 4.0, device="cpu")
    assert a == 1.0 and torch.equal(linear, plain / 4)
    base, a = kv8.rotary_frequencies(64, 1e4, "base", 4.0, device="cpu")
    assert a == 1.0 and base[0] == plain[0] and abs(base[-1] / plain[-1] * 4 - 1) < 1e-6
    assert torch.all(base <= plain) and torch.all(base >= plain / 4 * (1 - 1e-6))
    parts, a = kv8.rotary_frequencies(64, 1e4, "parts", 4.0, original=2048, device="cpu")
    assert abs(a - (0.1 * math.log(4.0) + 1)) < 1e-12
    turns = 2048 * plain.double() / (2 * math.pi)
    assert torch.equal(parts[turns > 32], plain[turns > 32])
    assert torch.allclose(parts[turns < 1], plain[turns < 1] / 4, rtol=1e-6)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and torch.all(parts[mid] < plain[mid]) and torch.all(parts[mid] > plain[mid] / 4)
    assert kv8.rotary_frequencies(2, device="cpu")[0].tolist() == [1.0]


@pytest.mark.parametrize("args,word", [((3,), "dims 3"), ((0,), "dims 0"), ((64, 0.0), "theta"), ((64, 1e4, "linear", 0.5), "factor"),
                                       ((64, 1e4, "parts", 2.0), "original"), ((64, 1e4, "other"), "scaling 'other'"),
                                       ((64, 1e4, "linear", math.inf), "factor")])
def test_frequencies_that_are_refused(args, word):
    with pytest.raises(ValueError, match=word):
        kv8.rotary_frequencies(*args, device="cpu")


# ---------------------------------------------------------------- refusals
def _calls(lib, cache, batch):
    r, m = _ref(_r()), _ref(_mass())
    return [lambda: lib.megakernel_op_kv8_scored_workspace_bytes(cache, batch, _ref(_x()), 8, 1),
            lambda: lib.megakernel_op_kv8_attention_scored(cache, batch, _ref(_x()), r, _ref(_r(2 * FAKE)), None, 8, 1.0, None, 0, None),
            lambda: lib.megakernel_op_kv8_weigh(cache, batch, _ref(_x()), r, FAKE, m, 8, 1.0, None),
            lambda: lib.megakernel_op_kv8_select(cache, batch, m, 4, 0, 0, FAKE, 2 * FAKE, None),
            lambda: lib.megakernel_op_kv8_compact(cache, batch, FAKE, FAKE, 4, 2 * FAKE, 4, None, None, None)]


@pytest.mark.parametrize("cache,word", BAD_CACHES)
def test_bad_caches(clib, cache, word):  # noqa: F811
    for call in _calls(clib, _ref(cache), _ref(_batch())):
        _refused(clib, call(), word)


@pytest.mark.parametrize("batch,word", BAD_BATCHES)
def test_bad_batches(clib, batch, word):  # noqa: F811
    for call in _calls(clib, _ref(_cache()), _ref(batch)):
        _refused(clib, call(), word)


BAD_SCORES = [(None, "null scores"), (_x(slopes=FAKE + 2), "alignment"), (_x(first=FAKE + 1), "alignment"), (_x(prefix=FAKE + 3), "alignment"),
              (_x(softcap=-1.0), "softcap=-1"), (_x(softcap=float("nan")), "softcap=nan"), (_x(softcap=float("inf")), "softcap=inf"),
              (_x(softcap=1e-20), "softcap"), (_x(softcap=1025.0), "softcap=1025"), (_x(window=-1), "window=-1")]


@pytest.mark.parametrize("x,word", BAD_SCORES)
def test_bad_scores(clib, x, word):  # noqa: F811
    c, b, r = _ref(_cache()), _ref(_batch()), _ref(_r())
    _refused(clib, clib.megakernel_op_kv8_scored_workspace_bytes(c, b, _ref(x), 8, 0), word)
    _refused(clib, clib.megakernel_op_kv8_attention_scored(c, b, _ref(x), r, _ref(_r(2 * FAKE)), None, 8, 1.0, None, 0, None), word)
    _refused(clib, clib.megakernel_op_kv8_weigh(c, b, _ref(x), r, FAKE, _ref(_mass()), 8, 1.0, None), word)


@pytest.mark.parametrize("rows,word", BAD_ROWS)
def test_bad_rows(clib, rows, word):  # noqa: F811
    c, b, x, ok = _ref(_cache()), _ref(_batch()), _ref(_x()), _ref(_r())
    for q, out in ((_ref(rows), ok), (ok, _ref(rows))):
        _refused(clib, clib.megakernel_op_kv8_attention_scored(c, b, x, q, out, None, 8, 1.0, None, 0, None), word)
    _refused(clib, clib.megakernel_op_kv8_weigh(c, b, x, _ref(rows), FAKE, _ref(_mass()), 8, 1.0, None), word)


def test_other_refusals_of_attention_with_scores(clib):  # noqa: F811
    c, b, x, r, far = _ref(_cache()), _ref(_batch()), _ref(_x()), _ref(_r()), _ref(_r(2 * FAKE))
    att = clib.megakernel_op_kv8_attention_scored
    _refused(clib, att(c, b, x, r, far, None, 12, 1.0, None, 0, None), "n_q=12")
    _refused(clib, att(c, b, x, r, r, None, 8, 1.0, None, 0, None), "must not be q")
    _refused(clib, att(c, b, x, r, far, FAKE + 2, 8, 1.0, None, 0, None), "lse")
    for scale in (0.0, -1.0, float("inf"), float("nan"), 3e38):
        _refused(clib, att(c, b, x, r, far, None, 8, scale, None, 0, None), "scale")
    _refused(clib, att(c, b, _ref(_x(softcap=1024.0)), r, far, None, 8, 1e-37, None, 0, None), "too far from softcap")
    _refused(clib, att(c, b, _ref(_x(softcap=2.0 ** -30)), r, far, None, 8, 1e33, None, 0, None), "too far from softcap")
    long = _ref(_batch(table_width=1024))
    plain, more = (clib.megakernel_op_kv8_scored_workspace_bytes(c, long, x, 8, n) for n in (0, 1))
    assert more > plain == clib.megakernel_op_kv8_workspace_bytes(c, long, 8) > 0
    _refused(clib, att(c, long, x, r, far, FAKE, 8, 1.0, FAKE, plain, None), "workspace")
    # a window leaves nothing to split
    assert clib.megakernel_op_kv8_scored_workspace_bytes(c, long, _ref(_x(window=512)), 8, 1) == 0


def test_other_refusals_of_weigh(clib):  # noqa: F811
    c, b, x, r, m = _ref(_cache()), _ref(_batch()), _ref(_x()), _ref(_r()), _ref(_mass())
    w = clib.megakernel_op_kv8_weigh
    _refused(clib, w(c, b, x, r, FAKE, m, 12, 1.0, None), "n_q=12")
    _refused(clib, w(c, b, x, r, None, m, 8, 1.0, None), "lse")
    _refused(clib, w(c, b, x, r, FAKE + 1, m, 8, 1.0, None), "lse")
    _refused(clib, w(c, b, x, _ref(_r(type=0)), FAKE, m, 8, 1.0, None), "bf16 only")
    _refused(clib, w(c, b, x, r, FAKE, m, 8, 0.0, None), "scale")
    for mass, word in BAD_MASSES:
        _refused(clib, w(c, b, x, r, FAKE, _ref(mass), 8, 1.0, None), word)


BAD_MASSES = [(None, "null mass"), (_mass(p=None), "null mass"), (_mass(p=FAKE + 2), "aligned"), (_mass(type=1), "must be fp32"),
              (_mass(type=5), "type 5"), (_mass(hs=127), "overlap"), (_mass(ts=1023), "overlap"), (_mass(ts=-1024), "overlap")]


def test_refusals_of_select(clib):  # noqa: F811
    c, b, m = _ref(_cache()), _ref(_batch()), _ref(_mass())
    sel = clib.megakernel_op_kv8_select
    for mass, word in BAD_MASSES:
        _refused(clib, sel(c, b, _ref(mass), 4, 0, 0, FAKE, 2 * FAKE, None), word)
    for keep, recent, sinks in ((0, 0, 0), (-1, 0, 0), (4, -1, 0), (4, 0, -1), (4, 3, 2), (4, 2 ** 31 - 1, 2 ** 31 - 1), (2 ** 30 + 1, 0, 0)):
        _refused(clib, sel(c, b, m, keep, recent, sinks, FAKE, FAKE, None), f"keep={keep}")
    for kept, lens in ((None, FAKE), (FAKE, None), (FAKE + 2, FAKE), (FAKE, FAKE + 1)):
        _refused(clib, sel(c, b, m, 4, 0, 0, kept, lens, None), "kept")
    _refused(clib, sel(c, b, m, 4, 0, 0, 2 * FAKE, FAKE, None), "must not be kv_len")


def test_refusals_of_compact(clib):  # noqa: F811
    c, b, m, n = _ref(_cache()), _ref(_batch()), _ref(_mass()), _ref(_mass(8 * FAKE))
    com = clib.megakernel_op_kv8_compact
    for kept, lens, new in ((None, FAKE, 2 * FAKE), (FAKE, None, 2 * FAKE), (FAKE, FAKE, None), (FAKE + 1, FAKE, 2 * FAKE)):
        _refused(clib, com(c, b, kept, lens, 4, new, 4, None, None, None), "kept")
    _refused(clib, com(c, b, FAKE, FAKE, 0, 2 * FAKE, 4, None, None, None), "keep=0")
    _refused(clib, com(c, b, FAKE, FAKE, 4, 2 * FAKE, 0, None, None, None), "new_width=0")
    _refused(clib, com(c, b, FAKE, FAKE, 4, 2 * FAKE, 1 << 26, None, None, None), "new_width")
    _refused(clib, com(c, b, FAKE, FAKE, 4, FAKE, 4, None, None, None), "batch's table")
    _refused(clib, com(c, b, FAKE, FAKE, 4, 2 * FAKE, 4, m, None, None), "go together")
    _refused(clib, com(c, b, FAKE, FAKE, 4, 2 * FAKE, 4, None, m, None), "go together")
    _refused(clib, com(c, b, FAKE, FAKE, 4, 2 * FAKE, 4, m, m, None), "same rows")
    for mass, word in BAD_MASSES[1:]:
        _refused(clib, com(c, b, FAKE, FAKE, 4, 2 * FAKE, 4, _ref(mass), n, None), word)
        _refused(clib, com(c, b, FAKE, FAKE, 4, 2 * FAKE, 4, m, _ref(mass), None), word.replace("mass", "new_mass"))


def test_refusals_of_rotary(clib):  # noqa: F811
    r, f32, far = _ref(_r()), _ref(_r(type=0)), _ref(_r(2 * FAKE))

    def call(q=r, k=r, qo=far, ko=_ref(_r(3 * FAKE)), inv=FAKE, pos=FAKE, tokens=5, n_q=8, n_kv=8, dim=64, turned=64, amp=1.0):
        return clib.megakernel_op_rotary(q, k, inv, pos, qo, ko, tokens, n_q, n_kv, dim, turned, 0, amp, None)

    for dim, turned in ((63, 2), (0, 2), (1026, 2), (64, 0), (64, 3), (64, 66), (64, -2)):
        _refused(clib, call(dim=dim, turned=turned), f"head_dim={dim}")
    _refused(clib, call(tokens=-1), "n_tokens=-1")
    _refused(clib, call(n_q=0), "n_q=0")
    _refused(clib, call(n_kv=1025), "n_kv=1025")
    for amp in (float("nan"), float("inf"), -float("inf")):
        _refused(clib, call(amp=amp), "amplitude")
    for bad in (dict(inv=None), dict(pos=None), dict(inv=FAKE + 2), dict(pos=FAKE + 1)):
        _refused(clib, call(**bad), "inv_freq or pos")
    for i, name in enumerate(("q", "k", "qo", "ko")):
        for rows, word in ((None, "null"), (_r(p=None), "null"), (_r(p=FAKE + 1), "2-byte aligned"), (_r(p=FAKE + 2, type=0), "4-byte aligned"),
                           (_r(hs=32), "overlap"), (_r(ts=-512), "overlap"), (_r(type=7), "type 7")):
            _refused(clib, call(**{name: _ref(rows)}), word)
    _refused(clib, call(qo=_ref(_r(2 * FAKE, ts=256))), "overlap")
    _refused(clib, call(k=f32), "one type")
    _refused(clib, call(ko=_ref(_r(3 * FAKE, type=0))), "one type")
    _refused(clib, call(qo=_ref(_r(ts=1024))), "in place")
    _refused(clib, call(ko=far), "same rows")
    _refused(clib, call(k=_ref(_r(2 * FAKE))), "same rows")


def test_empty_calls_do_nothing(clib):  # noqa: F811
    c, x, r, far, m = _ref(_cache()), _ref(_x()), _ref(_r()), _ref(_r(2 * FAKE)), _ref(_mass())
    for b in (_ref(_batch(n_tokens=0)), _ref(_batch(n_tokens=0, n_seq=0))):
        assert clib.megakernel_op_kv8_attention_scored(c, b, x, r, far, FAKE, 8, 1.0, None, 0, None) == 0
        assert clib.megakernel_op_kv8_weigh(c, b, x, r, FAKE, m, 8, 1.0, None) == 0
    none = _ref(_batch(n_seq=0))
    assert clib.megakernel_op_kv8_select(c, none, m, 4, 0, 0, FAKE, 2 * FAKE, None) == 0
    assert clib.megakernel_op_kv8_compact(c, none, FAKE, FAKE, 4, 2 * FAKE, 4, None, None, None) == 0
    assert clib.megakernel_op_rotary(r, r, FAKE, FAKE, far, _ref(_r(3 * FAKE)), 0, 8, 8, 64, 32, 1, 1.0, None) == 0


# ------------------------------------------------------------------ Python
def test_python_refuses_host_tensors(monkeypatch):
    def reached(name, device, *args):
        raise AssertionError(f"{name} was handed host addresses (device {device})")

    monkeypatch.setattr(kv8, "_call", reached)
    i32 = dict(dtype=torch.int32)
    for kw in (dict(slopes=torch.zeros(4)), dict(first=torch.zeros(4, **i32)), dict(prefix=torch.zeros(4, **i32))):
        with pytest.raises(ValueError, match="on the GPU, not on cpu"):
            kv8.Scores(**kw)
    q = torch.zeros((3, 4, 64))
    with pytest.raises(ValueError, match="on the GPU, not on cpu"):
        kv8.rotary(q, q, torch.zeros(32), torch.zeros(3, **i32), q, q)


@pytest.mark.parametrize("kw,word", [(dict(softcap=-1.0), "softcap"), (dict(softcap=math.nan), "softcap"), (dict(softcap=1025.0), "softcap"),
                                     (dict(window=-1), "window"), (dict(window=2 ** 31), "window"), (dict(window=2 ** 32 + 5), "window")])
def test_python_refuses_scores(kw, word):
    with pytest.raises(ValueError, match=word):
        kv8.Scores(**kw)


def test_scores_stay_what_they_were_made_with():
    x = kv8.Scores(softcap=30.0, window=5)
    assert (x._c.softcap, x._c.window, x._c.slopes) == (30.0, 5, None)
    with pytest.raises(AttributeError, match="make another"):
        x.window = 6
