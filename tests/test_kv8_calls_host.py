"""Calls of the paged 8-bit KV cache's operators on the CPU: frequencies for
long contexts against their definition, and what is refused before any GPU work
(the addresses below are never dereferenced)."""
from __future__ import annotations

import math

import numpy as np
import pytest

from megakernel_amd import kv8
from tests.test_kv8_host import FAKE, _batch, _cache, _r, _ref, _refused, clib  # noqa: F401
from tests.test_kv8_more_host import _mass, _x


# ------------------------------------------------------------- frequencies
def _turns(dims, theta, original):
    """How often each pair turns within the original context."""
    return original * theta ** (-2.0 * np.arange(dims // 2) / dims) / (2 * math.pi)


@pytest.mark.parametrize("dims,theta,factor,original,fast,slow", [
    (128, 1e6, 4.0, 32768, 32.0, 1.0), (128, 1e6, 4.0, 8192, 32.0, 1.0), (64, 1e4, 4.0, 2048, 32.0, 1.0), (64, 5e5, 8.0, 8192, 16.0, 2.0),
    (32, 1e4, 2.0, 512, 32.0, 1.0), (16, 10.0, 2.0, 64, 32.0, 1.0), (2, 1e4, 4.0, 4096, 32.0, 1.0), (64, 1e4, 1.0, 2048, 32.0, 1.0),
    (64, 1e4, 4.0, 2, 32.0, 1.0), (8, 1e4, 4.0, 10 ** 9, 32.0, 1.0)])
def test_parts_ramp_over_the_pairs(dims, theta, factor, original, fast, slow):
    """Between the last whole pair that turns more than `fast` times and the first
    that turns less than `slow` times the share falls by equal steps from pair to
    pair; the ends are found here by counting pairs, not by a logarithm."""
    got, amplitude = kv8.rotary_frequencies(dims, theta, "parts", factor, original=original, fast=fast, slow=slow, device="cpu")
    assert amplitude == 0.1 * math.log(factor) + 1
    # pairs beyond the last one go on with the same frequencies, down to dims - 1
    turns = original * theta ** (-2.0 * np.arange(0, 4 * dims) / dims) / (2 * math.pi)
    first = max(int((turns >= fast).sum()) - 1, 0)  # the last pair that is at least as fast
    last = min(int((turns > slow).sum()), dims - 1)
    plain = theta ** (-2.0 * np.arange(dims // 2) / dims)
    share = np.clip((np.arange(dims // 2) - first) / max(last - first, 1e-3), 0, 1)
    want = plain * (1 - share) + plain / factor * share
    np.testing.assert_allclose(got.double().numpy(), want, rtol=2.0 ** -23)


def test_turns_ramp_over_the_turns():
    dims, theta, factor, original = 64, 1e4, 4.0, 2048
    got, amplitude = kv8.rotary_frequencies(dims, theta, "turns", factor, original=original, fast=8.0, slow=2.0, device="cpu")
    assert amplitude == 0.1 * math.log(factor) + 1
    plain = theta ** (-2.0 * np.arange(dims // 2) / dims)
    stay = np.clip((_turns(dims, theta, original) - 2.0) / 6.0, 0, 1)
    np.testing.assert_allclose(got.double().numpy(), plain * stay + plain / factor * (1 - stay), rtol=2.0 ** -23)


@pytest.mark.parametrize("scaling", ["parts", "turns"])
@pytest.mark.parametrize("kw,word", [(dict(original=0), "original 0"), (dict(original=100, fast=1.0, slow=1.0), "fast 1.0"),
                                     (dict(original=100, slow=0.0), "slow 0.0"),
                                     (dict(original=100, fast=math.inf), "fast inf"), (dict(original=100, fast=math.nan), "fast nan")])
def test_ramps_that_are_refused(scaling, kw, word):
    with pytest.raises(ValueError, match=word):
        kv8.rotary_frequencies(64, scaling=scaling, factor=2.0, device="cpu", **kw)


def test_parts_need_pairs_of_different_speeds():
    for theta in (1.0, 0.5):
        with pytest.raises(ValueError, match=f"theta {theta}"):
            kv8.rotary_frequencies(64, theta, "parts", 2.0, original=100, device="cpu")


@pytest.mark.parametrize("dims,theta,scaling,factor,word", [
    (64, 1e4, None, 4.0, "factor 4.0 needs a scaling"), (2, 1e4, "base", 4.0, "dims 2"), (64, 1e4, "base", 1e308, "theta 10000.0"),
    (64, 1e300, "base", 1e10, "theta 1e[+]300"), (4, 1e4, "base", 1e160, "theta 10000.0"),
    (4, 1e-5, "base", 1e155, "theta 1e-05")])
def test_factors_that_would_be_lost(dims, theta, scaling, factor, word):
    with pytest.raises(ValueError, match=word):
        kv8.rotary_frequencies(dims, theta, scaling, factor, device="cpu")


def test_a_factor_of_one_changes_nothing():
    plain, _ = kv8.rotary_frequencies(64, 1e4, device="cpu")
    for scaling in (None, "linear", "base", "parts", "turns"):
        got, amplitude = kv8.rotary_frequencies(64, 1e4, scaling, 1.0, original=2048, device="cpu")
        assert got.equal(plain) and amplitude == 1.0
    assert kv8.rotary_frequencies(2, 1e4, "base", 1.0, device="cpu")[0].tolist() == [1.0]


# --------------------------------------------------- tensors on each other
# n_seq 2, 8 heads of 64, 5 tokens, table 4 blocks of 32; a view that starts
# further on is not the same tensor, but lies on it
def test_select_refuses_outputs_on_its_inputs(clib):  # noqa: F811
    c, b, m = _ref(_cache()), _ref(_batch()), _ref(_mass())
    sel = clib.megakernel_op_kv8_select
    for off in (-4, 4):
        _refused(clib, sel(c, b, m, 4, 0, 0, 2 * FAKE, FAKE + off, None), "kept_len must not be kv_len")
        _refused(clib, sel(c, b, m, 4, 0, 0, 2 * FAKE, 2 * FAKE + 4 * 64 - 4, None), "kept and kept_len")
        _refused(clib, sel(c, b, m, 4, 0, 0, FAKE + off, 2 * FAKE, None), "kept and kv_len")
    _refused(clib, sel(c, b, m, 4, 0, 0, 4 * FAKE + 64, 2 * FAKE, None), "kept and mass")
    _refused(clib, sel(c, b, m, 4, 0, 0, 2 * FAKE, 4 * FAKE + 4 * 2047, None), "kept_len and mass")


def test_compact_refuses_new_tensors_on_old_ones(clib):  # noqa: F811
    c, b, m = _ref(_cache()), _ref(_batch()), _ref(_mass())
    com = clib.megakernel_op_kv8_compact
    for off in (-28, -4, 4, 28):
        _refused(clib, com(c, b, FAKE, FAKE, 4, FAKE + off, 4, None, None, None), "batch's table")
    for off in (-4, 4, 512 * 8 - 4):
        _refused(clib, com(c, b, FAKE, FAKE, 4, 2 * FAKE, 4, m, _ref(_mass(4 * FAKE + off)), None), "mass and new_mass")
    new = _ref(_mass(8 * FAKE))
    _refused(clib, com(c, b, FAKE, FAKE, 4, 8 * FAKE + 16, 4, m, new, None), "new_mass and new_table")
    _refused(clib, com(c, b, 8 * FAKE + 16, FAKE, 4, 2 * FAKE, 4, m, new, None), "new_mass and kept")
    _refused(clib, com(c, b, FAKE, 8 * FAKE, 4, 2 * FAKE, 4, m, new, None), "new_mass and kept_len")


@pytest.mark.parametrize("name", ["rotary", "qk_norm_rope"])
def test_turned_rows_may_lie_on_their_own_inputs_alone(clib, name):  # noqa: F811
    def call(q, k, qo, ko, tokens=5):
        a = [_ref(_r(p)) for p in (q, k, qo, ko)]
        if name == "rotary":
            return clib.megakernel_op_rotary(a[0], a[1], FAKE, FAKE, a[2], a[3], tokens, 8, 8, 64, 64, 0, 1.0, None)
        return clib.megakernel_op_qk_norm_rope(a[0], a[1], FAKE, FAKE, FAKE, FAKE, a[2], a[3], tokens, 8, 8, 64, 1e-6, None)

    q, k, qo, ko = FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE
    for off in (-1024, -64, 16, 128, 4096):
        _refused(clib, call(q, k, q + off, ko), "in place")
        _refused(clib, call(q, k, qo, k + off), "in place")
        _refused(clib, call(q, k, k + off, ko), "q_out and k")
        _refused(clib, call(q, k, qo, q + off), "k_out and q")
        _refused(clib, call(q, k, qo, qo + off), "q_out and k_out")
    assert call(q, k, q + 16, ko, tokens=0) == 0


def test_attention_read_and_weigh_refuse_outputs_on_other_tensors(clib):  # noqa: F811
    c, b, x = _ref(_cache()), _ref(_batch()), _ref(_x())
    att = clib.megakernel_op_kv8_attention_scored
    for off in (-5104, 16, 1024, 5104):  # the last row's last, and first, 16 bytes
        _refused(clib, clib.megakernel_op_kv8_attention(c, b, _ref(_r()), _ref(_r(FAKE + off)), 8, 1.0, None, 0, None), "out and q")
        _refused(clib, clib.megakernel_op_kv8_read(c, b, _ref(_r()), _ref(_r(FAKE + off)), None), "k_out and v_out")
    _refused(clib, att(c, b, x, _ref(_r()), _ref(_r(2 * FAKE)), FAKE + 5116, 8, 1.0, None, 0, None), "lse and q")
    _refused(clib, att(c, b, x, _ref(_r()), _ref(_r(2 * FAKE)), 2 * FAKE - 156, 8, 1.0, None, 0, None), "lse and out")
    w = clib.megakernel_op_kv8_weigh
    _refused(clib, w(c, b, x, _ref(_r()), 4 * FAKE + 64, _ref(_mass()), 8, 1.0, None), "mass and lse")
    _refused(clib, w(c, b, x, _ref(_r(4 * FAKE + 64)), FAKE, _ref(_mass()), 8, 1.0, None), "mass and q")


# ------------------------------------------------------- which kernels run
ROWS, TILE, ROWS_SPLIT, TILE_SPLIT, JOIN_WAVES = 1, 2, 4, 8, 16


@pytest.mark.parametrize("n_kv,dim,batch,x,want", [
    (8, 64, dict(table_width=64, n_seq=1, n_tokens=1), {}, ROWS), (8, 64, dict(table_width=4096, n_seq=1, n_tokens=1), {}, ROWS | ROWS_SPLIT),
    (8, 64, dict(table_width=4096, n_seq=1, n_tokens=1), dict(window=100), ROWS), (8, 128, dict(table_width=256, n_seq=1, n_tokens=4096), {}, TILE),
    (8, 128, dict(table_width=256, n_seq=1, n_tokens=4096), dict(window=64), TILE), (8, 64, dict(table_width=256, n_seq=3, n_tokens=4096), {}, ROWS | TILE),
    (2, 64, dict(table_width=16, n_seq=1, n_tokens=300, max_kv=1 << 20), {}, TILE | TILE_SPLIT | JOIN_WAVES),
    (2, 64, dict(table_width=16, n_seq=1, n_tokens=200, max_kv=1 << 20), dict(softcap=5.0), TILE | TILE_SPLIT)])
def test_kernels_of_an_attention(clib, n_kv, dim, batch, x, want):  # noqa: F811
    c, b = _ref(_cache(n_kv=n_kv, head_dim=dim, block=16)), _ref(_batch(**batch))
    assert clib.megakernel_op_kv8_attention_kernels(c, b, _ref(_x(**x)), 16) == want
    # what is split has partials
    assert (clib.megakernel_op_kv8_scored_workspace_bytes(c, b, _ref(_x(**x)), 16, 0) > 0) == bool(want & (ROWS_SPLIT | TILE_SPLIT))


def test_kernels_of_an_attention_that_is_refused(clib):  # noqa: F811
    q = clib.megakernel_op_kv8_attention_kernels
    _refused(clib, q(None, _ref(_batch()), None, 8), "null cache")
    _refused(clib, q(_ref(_cache()), None, None, 8), "null batch")
    _refused(clib, q(_ref(_cache()), _ref(_batch()), _ref(_x(window=-1)), 8), "window=-1")
    _refused(clib, q(_ref(_cache()), _ref(_batch()), None, 12), "n_q=12")
    assert q(_ref(_cache()), _ref(_batch()), None, 8) == q(_ref(_cache()), _ref(_batch()), _ref(_x()), 8) == 1
