"""The paged 8-bit KV cache's operators on the CPU: the oracle's format against
closed forms, and what the entry points refuse before any GPU work (the
addresses below are never dereferenced)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from megakernel_amd import _lib, kv8
from oracle import fp8
from oracle import kv8 as okv8

FAKE = 0x10000


# ------------------------------------------------------------------ oracle
def test_scale_exponents_by_definition():
    rng = np.random.default_rng(0)
    for a in list(np.exp(rng.uniform(-80, 80, 200))) + [448.0, 448.0000001, 1.75, 2.0 ** -140, 0.0]:
        e = okv8.scale_exp(a)
        assert e >= -126 and a <= 448 * 2.0 ** e
        assert e == -126 or a > 448 * 2.0 ** (e - 1)


def test_append_in_parts_keeps_the_largest_scale_and_rounds_again():
    rng = np.random.default_rng(1)
    B, H, D = 16, 2, 64
    pool = okv8.Pool(np.full((3, H, B, D), 0x7F), np.full((3, H, D, B), 0x7F), np.ones((3, H)), np.ones((3, H)))
    table = np.array([[2, 0]])
    x = rng.standard_normal((20, H, D)) * np.where(np.arange(20) >= 10, 40.0, 1.0)[:, None, None]
    pool.append(table, [0, 10], [10], x[:10], x[:10])
    first = pool.ks.copy()
    pool.append(table, [0, 10], [20], x[10:], x[10:])
    assert np.all(pool.ks[2] > first[2]) and np.all(pool.ks[1] == 1)
    k, v = np.zeros((20, H, D)), np.zeros((20, H, D))
    pool.read(table, [0, 20], [20], k, v)
    np.testing.assert_array_equal(k, v)
    # a code is off by half a step of a value, 2^-4 of it, or of the smallest
    # normal one; rows of the first part were rounded twice
    for t in range(20):
        s = pool.ks[2 if t < 16 else 0][:, None]
        tol = (2 if t < 10 else 1) * np.maximum(np.abs(x[t]) * 2.0 ** -4, s * 2.0 ** -10)
        assert np.all(np.abs(k[t] - x[t]) <= tol * (1 + 2.0 ** -4))
    assert np.all(pool.k[0, :, 4:] == 0x7F)  # rows behind the last stay


def test_oracle_attention_of_equal_keys_is_the_mean():
    B, H, D = 16, 1, 64
    rng = np.random.default_rng(2)
    v = rng.integers(0, 0x60, (2, H, D, B)).astype(np.uint8)
    pool = okv8.Pool(np.full((2, H, B, D), 0x38), v, np.ones((2, H)), np.full((2, H), 2.0))
    q, out = rng.standard_normal((3, 2, D)), np.zeros((3, 2, D))
    pool.attention(np.array([[1, -1, 0]]), [0, 3], [34], q, out, 0.5)
    # positions 0..15 of block 1, 16..31 missing, 32, 33 of block 0
    rows = 2.0 * fp8.e4m3_decode_table().astype(np.float64)[np.concatenate([v[1, 0].T, v[0, 0].T[:2]])]
    np.testing.assert_allclose(out[0], np.stack([rows[:16].mean(0)] * 2), rtol=1e-12)
    np.testing.assert_allclose(out[2], np.stack([rows.mean(0)] * 2), rtol=1e-12)


def test_oracle_rotation_keeps_norms_and_position_zero():
    rng = np.random.default_rng(3)
    x, inv = rng.standard_normal((4, 3, 64)), 1e6 ** (-np.arange(32) / 32)
    y, _ = okv8.norm_rope(x, np.ones(64), inv, [0, 1, 50, 100000], 0.0)
    np.testing.assert_allclose((y * y).sum(-1), 64.0, rtol=1e-12)
    np.testing.assert_allclose(y[0], x[0] / np.sqrt((x[0] ** 2).mean(-1, keepdims=True)), rtol=1e-12)


# ---------------------------------------------------------------- refusals
def _cache(**kw):
    d = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, n_blocks=4, block=32, n_kv=8, head_dim=64)
    d.update(kw)
    return kv8._CCache(*(d[n] for n, _ in kv8._CCache._fields_))


def _batch(**kw):
    d = dict(table=FAKE, q_start=FAKE, kv_len=FAKE, n_seq=2, table_width=4, n_tokens=5, max_kv=0)
    d.update(kw)
    return kv8._CBatch(*(d[n] for n, _ in kv8._CBatch._fields_))


def _r(p=FAKE, ts=512, hs=64, type=1):
    return kv8._Rows(p, ts, hs, type)


def _ref(x):
    return None if x is None else ctypes.byref(x)


@pytest.fixture(scope="module")
def clib():
    import os
    if not os.path.exists(_lib.DEFAULT_LIB):
        from megakernel_amd import launcher
        launcher.compile_shared_library()
    return _lib.load()


BAD_CACHES = [(None, "null cache"), (_cache(k=None), "null cache"), (_cache(v_scale=None), "null cache"),
              (_cache(k=FAKE + 8), "alignment"), (_cache(k_scale=FAKE + 2), "alignment"), (_cache(block=48), "block=48"),
              (_cache(block=0), "block=0"), (_cache(head_dim=96), "head_dim=96"), (_cache(n_blocks=0), "n_blocks=0"),
              (_cache(n_kv=0), "n_kv=0")]
BAD_BATCHES = [(None, "null batch"), (_batch(table=None), "null batch"), (_batch(kv_len=FAKE + 1), "alignment"),
               (_batch(n_seq=-1), "n_seq=-1"), (_batch(n_tokens=-1), "n_tokens=-1"), (_batch(max_kv=-5), "max_kv=-5"),
               (_batch(table_width=0), "table_width=0"), (_batch(table_width=1 << 26), "table_width"),
               (_batch(n_tokens=(1 << 27) + 1), "n_tokens")]
BAD_ROWS = [(None, "null"), (_r(p=None), "null"), (_r(p=FAKE + 2), "aligned"), (_r(ts=516), "aligned"),
            (_r(hs=68), "aligned"), (_r(hs=32), "overlap"), (_r(ts=-512), "overlap"), (_r(type=7), "type 7")]


def _refused(clib, rc, word):
    assert rc == -1
    assert word in _lib.last_error(clib), _lib.last_error(clib)


@pytest.mark.parametrize("cache,word", BAD_CACHES)
def test_bad_caches_are_refused(clib, cache, word):
    b, r = _ref(_batch()), _ref(_r())
    _refused(clib, clib.megakernel_op_kv8_append(_ref(cache), b, r, r, None), word)
    _refused(clib, clib.megakernel_op_kv8_read(_ref(cache), b, r, r, None), word)
    _refused(clib, clib.megakernel_op_kv8_workspace_bytes(_ref(cache), b, 8), word)
    _refused(clib, clib.megakernel_op_kv8_attention(_ref(cache), b, r, _ref(_r(FAKE * 2)), 8, 1.0, None, 0, None), word)


@pytest.mark.parametrize("batch,word", BAD_BATCHES)
def test_bad_batches_are_refused(clib, batch, word):
    c, r = _ref(_cache()), _ref(_r())
    _refused(clib, clib.megakernel_op_kv8_append(c, _ref(batch), r, r, None), word)
    _refused(clib, clib.megakernel_op_kv8_read(c, _ref(batch), r, r, None), word)
    _refused(clib, clib.megakernel_op_kv8_workspace_bytes(c, _ref(batch), 8), word)
    _refused(clib, clib.megakernel_op_kv8_attention(c, _ref(batch), r, _ref(_r(FAKE * 2)), 8, 1.0, None, 0, None), word)


@pytest.mark.parametrize("rows,word", BAD_ROWS)
def test_bad_rows_are_refused(clib, rows, word):
    c, b, ok = _ref(_cache()), _ref(_batch()), _ref(_r())
    for k, v in ((_ref(rows), ok), (ok, _ref(rows))):
        _refused(clib, clib.megakernel_op_kv8_append(c, b, k, v, None), word)
        _refused(clib, clib.megakernel_op_kv8_read(c, b, k, v, None), word)
        _refused(clib, clib.megakernel_op_kv8_attention(c, b, k, v, 8, 1.0, None, 0, None), word)
    for i in range(4):
        q = [_ref(_r()), _ref(_r()), _ref(_r(2 * FAKE)), _ref(_r(2 * FAKE))]
        q[i] = _ref(rows)
        _refused(clib, clib.megakernel_op_qk_norm_rope(q[0], q[1], FAKE, FAKE, FAKE, FAKE, q[2], q[3], 5, 8, 8, 64, 1e-6,
                                                       None), word)


def test_other_refusals(clib):
    c, b = _ref(_cache()), _ref(_batch())
    r, f32, far = _ref(_r()), _ref(_r(type=0)), _ref(_r(2 * FAKE))
    _refused(clib, clib.megakernel_op_kv8_append(c, b, r, f32, None), "one type")
    _refused(clib, clib.megakernel_op_kv8_read(c, b, f32, r, None), "one type")
    _refused(clib, clib.megakernel_op_kv8_read(c, b, _ref(_r(ts=256)), r, None), "overlap")  # 8 heads of 64 a token
    _refused(clib, clib.megakernel_op_kv8_read(c, b, r, _ref(_r(ts=0)), None), "overlap")
    att = clib.megakernel_op_kv8_attention
    _refused(clib, att(c, b, r, far, 12, 1.0, None, 0, None), "n_q=12")
    _refused(clib, att(c, b, r, far, 0, 1.0, None, 0, None), "n_q=0")
    _refused(clib, att(c, b, r, r, 8, 1.0, None, 0, None), "must not be q")
    _refused(clib, att(c, b, f32, far, 8, 1.0, None, 0, None), "bf16 only")
    _refused(clib, att(_ref(_cache(n_kv=1)), _ref(_batch(n_tokens=1 << 27)), _ref(_r(ts=1024)), _ref(_r(2 * FAKE, ts=1024)), 16, 1.0, None, 0, None), "2^30")
    _refused(clib, att(c, b, r, _ref(_r(2 * FAKE, type=0)), 8, 1.0, None, 0, None), "bf16 only")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        _refused(clib, att(c, b, r, far, 8, scale, None, 0, None), "scale")
    long = _batch(table_width=1024)  # 32,768 positions: split, so it needs a workspace
    need = clib.megakernel_op_kv8_workspace_bytes(c, _ref(long), 8)
    assert need > 0
    _refused(clib, att(c, _ref(long), r, far, 8, 1.0, None, 0, None), "workspace")
    _refused(clib, att(c, _ref(long), r, far, 8, 1.0, FAKE, need - 1, None), "workspace")
    _refused(clib, att(c, _ref(long), r, far, 8, 1.0, FAKE + 4, need, None), "workspace")
    norm = clib.megakernel_op_qk_norm_rope

    def call(q=r, k=r, qo=far, ko=far, gain=FAKE, tokens=5, n_q=8, n_kv=8, dim=64, eps=1e-6):
        return norm(q, k, gain, FAKE, FAKE, FAKE, qo, ko, tokens, n_q, n_kv, dim, eps, None)

    _refused(clib, call(dim=32), "head_dim=32")
    _refused(clib, call(tokens=-1), "n_tokens=-1")
    _refused(clib, call(n_q=0), "n_q=0")
    _refused(clib, call(eps=-1.0), "eps")
    _refused(clib, call(eps=float("nan")), "eps")
    _refused(clib, call(gain=None), "gains")
    _refused(clib, call(gain=FAKE + 8), "gains")
    _refused(clib, call(k=f32), "one type")
    _refused(clib, call(ko=_ref(_r(2 * FAKE, type=0))), "one type")
    _refused(clib, call(qo=_ref(_r(ts=1024))), "in place")
    _refused(clib, call(qo=f32, ko=_ref(_r(2 * FAKE, type=0))), "in place")


def test_empty_calls_do_nothing(clib):
    c, r, far = _ref(_cache()), _ref(_r()), _ref(_r(2 * FAKE))
    for b in (_ref(_batch(n_tokens=0)), _ref(_batch(n_tokens=0, n_seq=0))):
        assert clib.megakernel_op_kv8_append(c, b, r, r, None) == 0
        assert clib.megakernel_op_kv8_read(c, b, r, r, None) == 0
        assert clib.megakernel_op_kv8_workspace_bytes(c, b, 8) == 0
        assert clib.megakernel_op_kv8_attention(c, b, r, far, 8, 1.0, None, 0, None) == 0
    assert clib.megakernel_op_qk_norm_rope(r, r, FAKE, FAKE, FAKE, FAKE, far, far, 0, 8, 8, 64, 0.0, None) == 0


def test_python_entry_points_refuse_cpu_tensors():
    codes, scale = torch.zeros((2, 1, 16, 64), dtype=torch.uint8), torch.ones((2, 1))
    with pytest.raises(ValueError, match="on the GPU"):
        kv8.Cache(codes, codes.transpose(2, 3), scale, scale)
    with pytest.raises(ValueError, match="on the GPU"):
        kv8.Batch(torch.zeros((1, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                  torch.zeros(1, dtype=torch.int32), 0)
    q = torch.zeros((1, 1, 64))
    with pytest.raises(ValueError, match="on the GPU"):
        kv8.qk_norm_rope(q, q, q[0, 0], q[0, 0], q[0, 0], q[0, 0], q, q)


def test_outputs_that_are_one_are_refused(clib):
    c, b, far = _ref(_cache()), _ref(_batch()), [_ref(_r(i * FAKE)) for i in range(1, 5)]
    _refused(clib, clib.megakernel_op_kv8_read(c, b, far[0], far[0], None), "same rows")
    for q, k, qo, ko in ((0, 1, 2, 2), (0, 1, 1, 2), (0, 1, 2, 0), (0, 1, 1, 0)):
        _refused(clib, clib.megakernel_op_qk_norm_rope(far[q], far[k], FAKE, FAKE, FAKE, FAKE, far[qo], far[ko], 5, 8, 8, 64,
                                                       1e-6, None), "same rows")


def test_tensors_of_a_cache_or_batch_cannot_be_replaced():
    for cls in (kv8.Cache, kv8.Batch):
        x = cls.__new__(cls)
        x.device = 0
        with pytest.raises(AttributeError, match="make another"):
            x.device = 1
        assert x.device == 0


def test_host_tensors_never_reach_a_launch(monkeypatch):
    """Types, shapes and strides are right, so that only the device can be why a call is refused."""
    def reached(name, device, *args):
        raise AssertionError(f"{name} was handed host addresses (device {device})")

    monkeypatch.setattr(kv8, "_call", reached)
    for dtype in (torch.bfloat16, torch.float32):
        for tokens in (1, 3):
            q, k = torch.zeros((tokens, 4, 64), dtype=dtype), torch.zeros((tokens, 2, 64), dtype=dtype)
            gain, inv = torch.ones(64, dtype=torch.bfloat16), torch.ones(32)
            pos = torch.zeros(tokens, dtype=torch.int32)
            with pytest.raises(ValueError, match="on the GPU, not on cpu"):
                kv8.qk_norm_rope(q, k, gain, gain, inv, pos, q, k)


def test_no_call_is_made_for_a_device_that_is_no_gpu():
    with pytest.raises(ValueError, match="op_kv8_read needs tensors on a GPU"):
        kv8._call("megakernel_op_kv8_read", -1)


@pytest.mark.parametrize("dim,group,n_tokens,max_kv", [(64, 71, 1024, 4096), (128, 66, 1024, 4096), (128, 64, 1040, 1 << 20)])
def test_no_splits_for_few_rows_where_a_token_has_more(clib, dim, group, n_tokens, max_kv):
    """Two sequences of so many tokens are not split, and with more query heads
    per KV head than the kernel for few rows takes, nothing is its own."""
    for n_kv in (1, 2):
        c, b = _cache(head_dim=dim, n_kv=n_kv), _batch(n_tokens=n_tokens, max_kv=max_kv)
        assert clib.megakernel_op_kv8_workspace_bytes(_ref(c), _ref(b), group * n_kv) == 0


def test_scales_stop_where_values_would_leave_fp32():
    top = 448.0 * 2.0 ** 119
    for a, e in ((top / 2, 118), (top, 119), (1.9375 * 2.0 ** 127, 119), (float(np.finfo(np.float32).max), 119)):
        assert okv8.scale_exp(a) == e
        codes = okv8.encode(np.array([a, -a, np.inf]), e)
        np.testing.assert_array_equal(okv8.decode(codes) * 2.0 ** e, [min(a, top), -min(a, top), 448.0 * 2.0 ** e])
        assert np.isfinite(np.float32(448.0 * 2.0 ** e))


def test_tensors_that_require_a_gradient_are_refused_while_torch_records_them():
    rows, gain = torch.zeros((2, 1, 64), requires_grad=True), torch.ones(64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="q requires a gradient.*no_grad"):
        kv8._rows(rows, (2, 1, 64), -1, "q")
    with pytest.raises(ValueError, match="q_gain requires a gradient"):
        kv8._whole(gain, torch.bfloat16, (64,), -1, "q_gain")
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            kv8._rows(rows, (2, 1, 64), -1, "q")
            kv8._whole(gain, torch.bfloat16, (64,), -1, "q_gain")
    kv8._rows(rows.detach(), (2, 1, 64), -1, "q")


@pytest.mark.parametrize("n_tokens,max_kv", [(2 ** 32 + 5, 0), (-1, 0), (2 ** 27 + 1, 0), (5, 2 ** 32 + 64), (5, 2 ** 31), (5, -1)])
def test_sizes_that_32_bits_do_not_hold_are_refused(n_tokens, max_kv):
    """Handed on, 2^32 + 5 rows would be 5."""
    i32 = torch.int32
    with pytest.raises(ValueError, match="n_tokens .* max_kv"):
        kv8.Batch(torch.zeros((1, 1), dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32), n_tokens, max_kv)


def test_a_scale_that_leaves_fp32_in_base_2_is_refused(clib):
    """It would make NaN of every score of zero."""
    c, b, r, far = _ref(_cache()), _ref(_batch()), _ref(_r()), _ref(_r(2 * FAKE))
    _refused(clib, clib.megakernel_op_kv8_attention(c, b, r, far, 8, 3e38, None, 0, None), "scale=3e+38")
