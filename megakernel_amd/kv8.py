"""Operators of a paged 8-bit KV cache over the library's
``megakernel_op_qk_norm_rope``, ``megakernel_op_rotary`` and
``megakernel_op_kv8_*`` entry points.

What a server keeps next to the model: a pool of blocks that sequences share
(:class:`Cache`), the sequences' block tables and lengths (:class:`Batch`),
and the operators that take one layer from its QKV rows to its attention
output: :func:`qk_norm_rope` or :func:`rotary`, :func:`append`,
:func:`attention`, whose scores may be capped, biased by distance or masked
(:class:`Scores`); :func:`read` gives rows of the cache back.  A cache that grows
too long is cut down by what its positions are worth: :func:`weigh` adds up
the attention weights that each gets, :func:`select` chooses the heaviest, and
:func:`compact` moves them to blocks of their own.  The reference has one contiguous bf16 cache
(src/kv_cache.cuh:11-32) and these steps only inside its
kernel (src/attention.cuh).

Tensors are torch tensors on one GPU and belong to the caller, outputs
included; nothing is copied, and no call waits.  Work is enqueued on torch's
current stream of that GPU, so tensors that another stream wrote need that
stream waited for, as with torch's own operators.  Calls can be captured into
a graph: a replay reads lengths and tables anew, while sizes stay fixed.  No
gradients are recorded: while torch records them (outside torch.no_grad()),
tensors that require one are refused.

    cache = kv8.Cache(k, v, k_scale, v_scale)      # or kv8.Cache.empty(...)
    batch = kv8.Batch(table, q_start, kv_len, n_tokens)
    kv8.qk_norm_rope(q, k, q_gain, k_gain, inv_freq, pos, q, k)
    kv8.append(cache, batch, k, v)
    kv8.attention(cache, batch, q, out)

    scores = kv8.Scores(softcap=30.0, window=4096)
    kv8.attention(cache, batch, q, out, scores=scores, lse=lse)
    kv8.weigh(cache, batch, q, lse, mass, scores=scores)
    kv8.select(cache, batch, mass, kept, kept_len, recent=256, sinks=4)
    kv8.compact(cache, batch, kept, kept_len, new_table, mass, new_mass)
"""
from __future__ import annotations

import ctypes
import math
import struct
import sys

import torch
from torch._C import _cuda_getCurrentRawStream as _raw_stream, _cuda_getDevice as _current_device

from . import _lib

_TYPES = {torch.bfloat16: 1, torch.float32: 0}  # MK_TYPE_BF16, MK_TYPE_F32
_BF16 = {torch.bfloat16: 1}


class _Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("token_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong),
                ("type", ctypes.c_int)]


# one _Rows as bytes, in a third of the structure's time
_pack_rows = struct.Struct("@Pqqi0P").pack


class _CCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("n_blocks", ctypes.c_int), ("block", ctypes.c_int),
                ("n_kv", ctypes.c_int), ("head_dim", ctypes.c_int)]


class _CScores(ctypes.Structure):
    _fields_ = [("slopes", ctypes.c_void_p), ("first", ctypes.c_void_p), ("prefix", ctypes.c_void_p),
                ("softcap", ctypes.c_float), ("window", ctypes.c_int)]


class _CBatch(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("q_start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("n_seq", ctypes.c_int), ("table_width", ctypes.c_int), ("n_tokens", ctypes.c_int),
                ("max_kv", ctypes.c_int)]


def _no_grad(t, name: str):
    if torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and none is recorded here: call under torch.no_grad()")


def _whole(t, dtype, shape, device: int, name: str):
    """A contiguous tensor of one type and shape on GPU `device`; None in
    `shape` is any size."""
    if t.requires_grad:
        _no_grad(t, name)
    if t.dtype is dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU, not on {t.device}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{device}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple('any' if n is None else n for n in shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _rows(t, shape, device: int, name: str, types=_TYPES) -> bytes:
    """Rows [tokens][heads][dim] with any token and head stride, as a
    megakernel_rows."""
    if t.requires_grad:
        _no_grad(t, name)
    typ = types.get(t.dtype)
    if typ is None or t.shape != shape or t.get_device() != device:
        if typ is None:
            raise ValueError(f"{name} must be {' or '.join(str(x)[6:] for x in types)}, not {t.dtype}")
        if t.shape != shape:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, not {shape}")
        raise ValueError(f"{name} is on {t.device}, not on cuda:{device}")
    token, head, last = t.stride()
    if last != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous (stride {last})")
    # of a single token or head, the stride says nothing
    return _pack_rows(t.data_ptr(), token if shape[0] > 1 else 0, head if shape[1] > 1 else 0, typ)


_library = None


def _call(name: str, device: int, *args):
    """Enqueue on the current stream of GPU `device`; raises what the library reports."""
    global _library
    if device < 0:
        raise ValueError(f"{name[11:]} needs tensors on a GPU")
    if _library is None:
        _library = _lib.load()
    fn = getattr(_library, name)
    # the handle of torch.cuda.current_stream(device), without the object around it
    if device == _current_device():
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        _lib.check(_library, rc, name[11:])


class _Fixed:
    """The library is handed the tensors' addresses: another tensor in the
    place of one would not be seen, and the first one's memory be reused."""

    def __setattr__(self, name, value):
        if name in self.__dict__:
            raise AttributeError(f"{name} of a {type(self).__name__} stays what it was made with; make another one")
        self.__dict__[name] = value


class Cache(_Fixed):
    """A pool of blocks of one layer: e4m3 codes ``k`` [n_blocks][n_kv][block][head_dim]
    and ``v`` [n_blocks][n_kv][head_dim][block] (uint8), and their power-of-two
    scales [n_blocks][n_kv] (float32).  ``block`` is 16, 32, 64 or 128
    positions, ``head_dim`` 64 or 128.  Blocks need no initial value.
    """

    def __init__(self, k, v, k_scale, v_scale):
        device = k.get_device()
        _whole(k, torch.uint8, (None, None, None, None), device, "k")
        n_blocks, n_kv, block, head_dim = k.shape
        _whole(v, torch.uint8, (n_blocks, n_kv, head_dim, block), device, "v")
        _whole(k_scale, torch.float32, (n_blocks, n_kv), device, "k_scale")
        _whole(v_scale, torch.float32, (n_blocks, n_kv), device, "v_scale")
        if block not in (16, 32, 64, 128) or head_dim not in (64, 128):
            raise ValueError(f"blocks of {block} positions (16, 32, 64 or 128), head_dim {head_dim} (64 or 128)")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_blocks, self.n_kv, self.block, self.head_dim, self.device = n_blocks, n_kv, block, head_dim, device
        self._c = _CCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n_blocks, block, n_kv,
                          head_dim)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, n_blocks: int, n_kv: int, head_dim: int, block: int = 32, device="cuda") -> "Cache":
        codes = [torch.empty(s, dtype=torch.uint8, device=device)
                 for s in ((n_blocks, n_kv, block, head_dim), (n_blocks, n_kv, head_dim, block))]
        return cls(*codes, *(torch.empty((n_blocks, n_kv), dtype=torch.float32, device=device) for _ in range(2)))


class Batch(_Fixed):
    """Rows of several sequences.  Sequence i has rows q_start[i] ..
    q_start[i + 1] - 1 of the row tensors, and these are the newest of its
    kv_len[i] positions.  ``table`` [n_seq][width] names its blocks in order;
    entries outside the pool (-1, say) are missing blocks: attention leaves
    their positions out, :func:`append` drops their rows, :func:`read` gives
    zeros.  All three are int32 tensors on the GPU and are read when a call
    runs, so they may change between calls and replays.

    ``n_tokens`` is the row tensors' first size.  ``max_kv`` only says how long
    contexts are expected to get, from which :func:`attention` chooses its kernels
    and how far to split them; longer ones are right all the same.
    """

    def __init__(self, table, q_start, kv_len, n_tokens: int, max_kv: int = 0):
        if not (0 <= n_tokens <= 1 << 27 and 0 <= max_kv < 1 << 31):  # the library's integers have 32 bits
            raise ValueError(f"n_tokens {n_tokens} (0 to 2^27), max_kv {max_kv} (0 to 2^31 - 1)")
        device = kv_len.get_device()
        _whole(kv_len, torch.int32, (None,), device, "kv_len")
        n_seq = kv_len.shape[0]
        _whole(table, torch.int32, (n_seq, None), device, "table")
        _whole(q_start, torch.int32, (n_seq + 1,), device, "q_start")
        if table.shape[1] < 1:
            raise ValueError("table needs a width of at least 1")
        self.table, self.q_start, self.kv_len = table, q_start, kv_len
        self.n_seq, self.n_tokens, self.max_kv, self.device = n_seq, int(n_tokens), int(max_kv), device
        # of no sequence there are no addresses to hand over, and nothing to do
        self._c = _CBatch(table.data_ptr() or 16, q_start.data_ptr(), kv_len.data_ptr() or 16, n_seq, table.shape[1],
                          self.n_tokens, self.max_kv)
        self._ref = ctypes.byref(self._c)
        self._need: dict[tuple, int] = {}


class Scores(_Fixed):
    """What the scores of :func:`attention` and :func:`weigh` are, and what a
    row sees.  The row at position p and a position j have the score

        softcap * tanh(scale * q.k / softcap) - slopes[head] * |p - j|

    without the tanh where ``softcap`` is 0, and without the bias where there
    are no ``slopes`` (float32 [n_q]; beyond +-2^94 they count as that).  The row sees
    max(0, first[row], p + 1 - window) <= j < max(p + 1, prefix[sequence]):
    ``window`` positions up to its own (0: all), none before its document
    (``first``, int32 [n_tokens]), and of a prefix all (``prefix``, int32
    [n_seq]: how many positions it has).  The tensors are read when a call runs,
    so they may change between calls and replays.
    """

    def __init__(self, softcap: float = 0.0, slopes=None, window: int = 0, first=None, prefix=None):
        given = [t for t in (slopes, first, prefix) if t is not None]
        device = given[0].get_device() if given else None
        for t, name, dtype in ((slopes, "slopes", torch.float32), (first, "first", torch.int32), (prefix, "prefix", torch.int32)):
            if t is not None:
                _whole(t, dtype, (None,), device, name)
        if not (softcap == 0 or 2.0 ** -30 <= softcap <= 1024) or not 0 <= window < 1 << 31:
            raise ValueError(f"softcap {softcap} (0, or 2^-30 to 1024), window {window} (0 to 2^31 - 1)")
        self.slopes, self.first, self.prefix = slopes, first, prefix
        self.softcap, self.window, self.device = float(softcap), int(window), device
        # an empty tensor has no address, and no row asks for what is in it
        self._c = _CScores(*(None if t is None else t.data_ptr() or 16 for t in (slopes, first, prefix)), self.softcap,
                           self.window)
        self._ref = ctypes.byref(self._c)

    def _fits(self, batch: "Batch", n_q: int):
        for t, name, n in ((self.slopes, "slopes", n_q), (self.first, "first", batch.n_tokens), (self.prefix, "prefix", batch.n_seq)):
            if t is not None and t.shape[0] != n:
                raise ValueError(f"{name} of the scores has shape {tuple(t.shape)}, not {(n,)}")
        if self.device is not None and self.device != batch.device:
            raise ValueError(f"the scores are on cuda:{self.device}, not on cuda:{batch.device}")


_plain = None  # Scores() of a call that has none


def _scores(scores: "Scores | None", batch: "Batch", n_q: int) -> Scores:
    global _plain
    if scores is None:
        if _plain is None:
            _plain = Scores()
        return _plain
    scores._fits(batch, n_q)
    return scores


def qk_norm_rope(q, k, q_gain, k_gain, inv_freq, pos, q_out, k_out, eps: float = 1e-6):
    """RMSNorm of every head of q [T][n_q][D] and k [T][n_kv][D] with its gain
    (bf16 [D]), then the rotate-half rotation by ``pos[t] * inv_freq[i]``
    (int32 [T], float32 [D/2]), into q_out and k_out.  D is 64 or 128; inputs
    and outputs are bf16 or fp32 with any token and head strides, so the rows
    may lie in a packed QKV tensor, and an output may be its own input."""
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k are [tokens][heads][head_dim], not {tuple(q.shape)} and {tuple(k.shape)}")
    device = q.get_device()
    if device < 0:  # of other tensors of the host it would be the device that they are expected on
        raise ValueError(f"q must be on the GPU, not on {q.device}")
    tokens, n_q, dim = q.shape
    n_kv = k.shape[1]
    _whole(pos, torch.int32, (tokens,), device, "pos")
    _whole(q_gain, torch.bfloat16, (dim,), device, "q_gain")
    _whole(k_gain, torch.bfloat16, (dim,), device, "k_gain")
    _whole(inv_freq, torch.float32, (dim // 2,), device, "inv_freq")
    qs, ks = (tokens, n_q, dim), (tokens, n_kv, dim)
    rows = (_rows(q, qs, device, "q"), _rows(k, ks, device, "k"), _rows(q_out, qs, device, "q_out"),
            _rows(k_out, ks, device, "k_out"))
    if tokens == 0:
        return
    _call("megakernel_op_qk_norm_rope", device, rows[0], rows[1], q_gain.data_ptr(), k_gain.data_ptr(),
          inv_freq.data_ptr(), pos.data_ptr(), rows[2], rows[3], tokens, n_q, n_kv, dim, eps)


def rotary(q, k, inv_freq, pos, q_out, k_out, interleaved: bool = False, amplitude: float = 1.0):
    """Rotation of every head of q [T][n_q][D] and k [T][n_kv][D] by its token's
    position (int32 [T]), without a norm.  The first 2 * len(inv_freq) dimensions
    of a head are turned, the others copied; pairs are the two halves of the
    turned part, or with ``interleaved`` neighbours.  D is even, at most 1024.
    Inputs and outputs are bf16 or fp32 with any token and head strides, and an
    output may be its own input.  :func:`rotary_frequencies` gives ``inv_freq``
    (float32) and ``amplitude``, what every turned value is multiplied by."""
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"q and k are [tokens][heads][head_dim], not {tuple(q.shape)} and {tuple(k.shape)}")
    device = q.get_device()
    if device < 0:
        raise ValueError(f"q must be on the GPU, not on {q.device}")
    tokens, n_q, dim = q.shape
    n_kv = k.shape[1]
    _whole(pos, torch.int32, (tokens,), device, "pos")
    pairs = inv_freq.numel()
    _whole(inv_freq, torch.float32, (pairs,), device, "inv_freq")
    if not 1 <= pairs <= dim // 2 or dim % 2:
        raise ValueError(f"inv_freq turns {2 * pairs} dimensions of heads of {dim} (2 to all, and heads even)")
    qs, ks = (tokens, n_q, dim), (tokens, n_kv, dim)
    rows = (_rows(q, qs, device, "q"), _rows(k, ks, device, "k"), _rows(q_out, qs, device, "q_out"),
            _rows(k_out, ks, device, "k_out"))
    if tokens == 0:
        return
    _call("megakernel_op_rotary", device, rows[0], rows[1], inv_freq.data_ptr(), pos.data_ptr(), rows[2], rows[3], tokens,
          n_q, n_kv, dim, 2 * pairs, bool(interleaved), amplitude)


def rotary_frequencies(dims: int, theta: float = 1e6, scaling: str | None = None, factor: float = 1.0, original: int = 0,
                       fast: float = 32.0, slow: float = 1.0, device="cuda"):
    """(inv_freq, amplitude) for :func:`rotary` of ``dims`` dimensions: theta^(-2i / dims),
    for contexts ``factor`` times as long as trained for scaled by

    ``"linear"``  positions divided by the factor;
    ``"base"``    theta times factor^(dims / (dims - 2)), which leaves the
                  fastest pair as it is and divides the slowest by the factor;
    ``"parts"``   pairs that turn more than ``fast`` times within the
                  ``original`` context as they are, those that turn less than
                  ``slow`` times divided by the factor, and from the last of the
                  first to the first of the last by equal steps from pair to
                  pair (what Qwen3 and other models are published with for long
                  contexts); the amplitude is 0.1 ln(factor) + 1;
    ``"turns"``   the same with a ramp that is linear in the turns.  Models with
                  this ramp differ in ``fast`` (32 or 4), and some have no
                  amplitude: pass 1.0 to :func:`rotary` for those.

    Computed in double precision, rounded once to float32."""
    if dims < 2 or dims % 2:
        raise ValueError(f"dims {dims} must be even and at least 2")
    if not (theta > 0 and math.isfinite(theta) and factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"theta {theta} (above 0), factor {factor} (at least 1)")
    if scaling is None and factor != 1:
        raise ValueError(f"factor {factor} needs a scaling ('linear', 'base', 'parts' or 'turns')")
    amplitude = 1.0
    if scaling == "base" and factor != 1:
        if dims == 2:
            raise ValueError("dims 2: the base of a single pair scales nothing")
        growth = math.log(factor) * dims / (dims - 2)
        if growth + max(math.log(theta), 0.0) >= math.log(sys.float_info.max):
            raise ValueError(f"theta {theta} times a power of factor {factor} is not finite")
        theta *= factor ** (dims / (dims - 2))
    inv = [theta ** (-2.0 * i / dims) for i in range(dims // 2)]
    if scaling == "linear":
        inv = [f / factor for f in inv]
    elif scaling in ("parts", "turns"):
        if original < 1 or not math.inf > fast > slow > 0:
            raise ValueError(f"original {original} (at least 1), fast {fast} and slow {slow} (fast above slow above 0)")
        if scaling == "turns":
            stay = [min(max((original * f / (2 * math.pi) - slow) / (fast - slow), 0.0), 1.0) for f in inv]
        else:
            if theta <= 1:
                raise ValueError(f"theta {theta} (above 1, or no pair is slower than another)")
            # pair i turns original * theta^(-2i / dims) / 2 pi times: which i has so many turns
            at = [dims * math.log(original / (2 * math.pi * turns)) / (2 * math.log(theta)) for turns in (fast, slow)]
            first = min(max(math.floor(at[0]), 0), dims - 1)
            last = max(min(math.ceil(at[1]), dims - 1), first + 1e-3)  # apart, or there is no ramp
            stay = [1 - min(max((i - first) / (last - first), 0.0), 1.0) for i in range(dims // 2)]
        inv = [f * s + f / factor * (1 - s) for f, s in zip(inv, stay)]
        amplitude = 0.1 * math.log(factor) + 1
    elif scaling not in (None, "base"):
        raise ValueError(f"scaling {scaling!r} (None, 'linear', 'base', 'parts' or 'turns')")
    return torch.tensor(inv, dtype=torch.float64).to(torch.float32).to(device), amplitude


def _one_gpu(cache: Cache, batch: Batch):
    if cache.device != batch.device:
        raise ValueError(f"the batch is on cuda:{batch.device}, not on cuda:{cache.device}")


def append(cache: Cache, batch: Batch, k, v):
    """Quantise rows k, v [n_tokens][n_kv][head_dim] (bf16 or fp32) into their
    blocks.  A block and head has one scale, the smallest power of two that
    fits its rows into e4m3 (2^-126 to 2^119; what is larger saturates at
    448 * 2^119); rows that a block already holds are rounded again where a new
    row makes its scale grow.  A block that a call appends to may
    stand in one table entry only."""
    _one_gpu(cache, batch)
    shape = (batch.n_tokens, cache.n_kv, cache.head_dim)
    a, b = _rows(k, shape, cache.device, "k"), _rows(v, shape, cache.device, "v")
    if batch.n_seq and batch.n_tokens:
        _call("megakernel_op_kv8_append", cache.device, cache._ref, batch._ref, a, b)


def read(cache: Cache, batch: Batch, k_out, v_out):
    """The values of the batch's rows into k_out, v_out [n_tokens][n_kv][head_dim]
    (bf16 or fp32, exact in both).  ``q_start`` of a batch whose rows are whole
    contexts is their lengths' running sum."""
    _one_gpu(cache, batch)
    shape = (batch.n_tokens, cache.n_kv, cache.head_dim)
    a, b = _rows(k_out, shape, cache.device, "k_out"), _rows(v_out, shape, cache.device, "v_out")
    if batch.n_seq and batch.n_tokens:
        _call("megakernel_op_kv8_read", cache.device, cache._ref, batch._ref, a, b)


def workspace_bytes(cache: Cache, batch: Batch, n_q: int, scores: Scores | None = None, lse: bool = False) -> int:
    """Bytes of :func:`attention`'s workspace for these sizes (0: none), with
    scores and a log-sum-exp as the call will have them."""
    scored = scores is not None or lse
    key = (cache.n_kv, cache.head_dim, cache.block, n_q, (scores.window if scores else 0, lse) if scored else None)
    need = batch._need.get(key)
    if need is None:
        lib = _lib.load()
        if scored:
            x = _scores(scores, batch, n_q)
            need = lib.megakernel_op_kv8_scored_workspace_bytes(cache._ref, batch._ref, x._ref, n_q, lse)
        else:
            need = lib.megakernel_op_kv8_workspace_bytes(cache._ref, batch._ref, n_q)
        batch._need[key] = _lib.check(lib, need, "op_kv8_workspace_bytes")
    return need


_KERNELS = ("rows", "tile", "rows split", "tile split", "join by waves")  # bits of MK_KV8_*


def attention_kernels(cache: Cache, batch: Batch, n_q: int, scores: Scores | None = None) -> set[str]:
    """Which kernels :func:`attention` runs for these sizes: "rows" (16 query rows a
    workgroup), "tile" (128), both where sequences with few and many rows may meet;
    "rows split" and "tile split" where contexts are dealt in parts; "join by waves"
    where these are joined by waves, not by a workgroup for each row.  For reading
    profiles, and for tests that mean one of them."""
    _one_gpu(cache, batch)
    lib = _lib.load()
    x = None if scores is None else _scores(scores, batch, n_q)._ref
    bits = _lib.check(lib, lib.megakernel_op_kv8_attention_kernels(cache._ref, batch._ref, x, n_q), "op_kv8_attention_kernels")
    return {name for i, name in enumerate(_KERNELS) if bits >> i & 1}


def attention(cache: Cache, batch: Batch, q, out, scale: float | None = None, workspace=None, scores: Scores | None = None,
              lse=None):
    """Causal attention of q [n_tokens][n_q][head_dim] (bf16) over the cache
    into out: each row sees its sequence's positions up to its own, its own
    among them.  Query head h reads KV head h / (n_q / n_kv); rows that see
    nothing are zeros.  ``scale`` is 1 / sqrt(head_dim) unless given.
    ``scores`` changes what scores are and what rows see (:class:`Scores`).
    ``lse`` (float32 [n_tokens][n_q]) receives the rows' log-sum-exps,
    -infinity for a row that sees nothing.
    ``workspace`` is a uint8 tensor of :func:`workspace_bytes`, one for each
    call that may run at the same time; without one, a call takes its own from
    torch's allocator."""
    if q.dim() != 3:
        raise ValueError(f"q is [tokens][heads][head_dim], not {tuple(q.shape)}")
    _one_gpu(cache, batch)
    device, n_q = cache.device, q.shape[1]
    shape = (batch.n_tokens, n_q, cache.head_dim)
    a, b = _rows(q, shape, device, "q", _BF16), _rows(out, shape, device, "out", _BF16)
    x = None
    if scores is not None or lse is not None:
        x = _scores(scores, batch, n_q)
        if lse is not None:
            _whole(lse, torch.float32, (batch.n_tokens, n_q), device, "lse")
    need = workspace_bytes(cache, batch, n_q, scores, lse is not None)
    if not batch.n_seq or not batch.n_tokens:
        return
    at = size = None
    if workspace is not None:
        _whole(workspace, torch.uint8, (None,), device, "workspace")
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    if workspace is not None:
        at, size = workspace.data_ptr(), workspace.numel()
    if scale is None:
        scale = cache.head_dim ** -0.5
    if x is None:
        _call("megakernel_op_kv8_attention", device, cache._ref, batch._ref, a, b, n_q, scale, at, size or 0)
    else:
        _call("megakernel_op_kv8_attention_scored", device, cache._ref, batch._ref, x._ref, a, b,
              None if lse is None else lse.data_ptr(), n_q, scale, at, size or 0)


def _mass(t, cache: Cache, n_seq: int, positions: int, name: str) -> bytes:
    """Weights [n_seq][n_kv][at least `positions`] as a megakernel_rows."""
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must be torch.float32, not {t.dtype}")
    if t.dim() != 3 or t.shape[2] < positions:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {(n_seq, cache.n_kv, positions)} (or more positions)")
    return _rows(t, (n_seq, cache.n_kv, t.shape[2]), cache.device, name)


def weigh(cache: Cache, batch: Batch, q, lse, mass, scale: float | None = None, scores: Scores | None = None):
    """Add up what each cached position is worth: mass [n_seq][n_kv][positions]
    (float32, any sequence and head strides, at least the table's positions) gains
    the attention weights that the batch's rows give each position, summed over
    rows and the query heads that share a KV head.  ``q``, ``scale`` and ``scores``
    are those of the :func:`attention` that gave ``lse``.  Positions of the batch's
    own rows start from zero, those before them from what mass holds; positions
    past a length stay as they are."""
    if q.dim() != 3:
        raise ValueError(f"q is [tokens][heads][head_dim], not {tuple(q.shape)}")
    _one_gpu(cache, batch)
    device, n_q = cache.device, q.shape[1]
    a = _rows(q, (batch.n_tokens, n_q, cache.head_dim), device, "q", _BF16)
    _whole(lse, torch.float32, (batch.n_tokens, n_q), device, "lse")
    b = _mass(mass, cache, batch.n_seq, batch.table.shape[1] * cache.block, "mass")
    x = _scores(scores, batch, n_q)
    if batch.n_seq and batch.n_tokens:
        _call("megakernel_op_kv8_weigh", device, cache._ref, batch._ref, x._ref, a, lse.data_ptr(), b, n_q,
              cache.head_dim ** -0.5 if scale is None else scale)


def _kept(cache: Cache, batch: Batch, kept, kept_len):
    _whole(kept, torch.int32, (batch.n_seq, cache.n_kv, kept.shape[-1] if kept.dim() else None), cache.device, "kept")
    _whole(kept_len, torch.int32, (batch.n_seq,), cache.device, "kept_len")
    if not 1 <= kept.shape[2] <= 1 << 30:  # the library's integers have 32 bits
        raise ValueError(f"kept has room for {kept.shape[2]} positions (1 to 2^30)")


def select(cache: Cache, batch: Batch, mass, kept, kept_len, recent: int = 0, sinks: int = 0):
    """The positions worth keeping of each sequence and KV head: kept
    [n_seq][n_kv][keep] (int32) receives them in rising order, -1 behind the last,
    and kept_len [n_seq] (int32, another tensor than the batch's lengths) their
    number, min(kv_len, keep).  Of a longer sequence they are its first ``sinks``,
    its last ``recent`` and the heaviest of the others by ``mass`` (:func:`weigh`);
    of equal weights the lower position, and NaN last."""
    _one_gpu(cache, batch)
    _kept(cache, batch, kept, kept_len)
    a = _mass(mass, cache, batch.n_seq, batch.table.shape[1] * cache.block, "mass")
    if recent < 0 or sinks < 0 or recent + sinks > kept.shape[2]:
        raise ValueError(f"recent {recent} and sinks {sinks} (at least 0, together at most {kept.shape[2]}, kept's positions)")
    if batch.n_seq:
        _call("megakernel_op_kv8_select", cache.device, cache._ref, batch._ref, a, kept.shape[2], recent, sinks,
              kept.data_ptr(), kept_len.data_ptr())


def compact(cache: Cache, batch: Batch, kept, kept_len, new_table, mass=None, new_mass=None):
    """Move the kept rows (:func:`select`) to the blocks of new_table
    [n_seq][width] (int32), in order and quantised anew: :func:`read` followed by
    :func:`append` to blocks that start anew.  These blocks are none that the
    batch's table names, and each stands in one entry; the old ones are free
    afterwards.  With ``mass`` and ``new_mass`` ([n_seq][n_kv][the new table's
    positions]) the rows' weights move along.  kept_len counts what was kept
    and no more: the :class:`Batch` of new_table that goes on from there has
    lengths of kept_len plus its own new rows, which are the newest positions
    (of kept_len alone they would be the last kept ones, and replace them), and
    the table has blocks for them.  Its positions are places in the
    cache, so scores that count positions (a window, slopes, documents) count
    kept ones, and the rotation goes on from the sequence's own position."""
    _one_gpu(cache, batch)
    _kept(cache, batch, kept, kept_len)
    device = cache.device
    _whole(new_table, torch.int32, (batch.n_seq, new_table.shape[-1] if new_table.dim() else None), device, "new_table")
    if not 1 <= new_table.shape[1] * cache.block <= 1 << 30:
        raise ValueError(f"new_table has {new_table.shape[1]} blocks of {cache.block} positions (1 to 2^30 positions)")
    if (mass is None) != (new_mass is None):
        raise ValueError("mass and new_mass go together")
    a = b = None
    if mass is not None:
        a = _mass(mass, cache, batch.n_seq, batch.table.shape[1] * cache.block, "mass")
        b = _mass(new_mass, cache, batch.n_seq, new_table.shape[1] * cache.block, "new_mass")
    if batch.n_seq:
        _call("megakernel_op_kv8_compact", device, cache._ref, batch._ref, kept.data_ptr(), kept_len.data_ptr(),
              kept.shape[2], new_table.data_ptr(), new_table.shape[1], a, b)
