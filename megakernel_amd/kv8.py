"""Operators of a paged 8-bit KV cache over the library's
``megakernel_op_qk_norm_rope`` and ``megakernel_op_kv8_*`` entry points.

What a server keeps next to the model: a pool of blocks that sequences share
(:class:`Cache`), the sequences' block tables and lengths (:class:`Batch`),
and the operators that take one layer from its QKV rows to its attention
output: :func:`qk_norm_rope`, :func:`append`, :func:`attention`; :func:`read`
gives rows of the cache back.  The reference has one contiguous bf16 cache
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
"""
from __future__ import annotations

import ctypes
import struct

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


def workspace_bytes(cache: Cache, batch: Batch, n_q: int) -> int:
    """Bytes of :func:`attention`'s workspace for these sizes (0: none)."""
    key = (cache.n_kv, cache.head_dim, cache.block, n_q)
    need = batch._need.get(key)
    if need is None:
        lib = _lib.load()
        need = _lib.check(lib, lib.megakernel_op_kv8_workspace_bytes(cache._ref, batch._ref, n_q), "op_kv8_workspace_bytes")
        batch._need[key] = need
    return need


def attention(cache: Cache, batch: Batch, q, out, scale: float | None = None, workspace=None):
    """Causal attention of q [n_tokens][n_q][head_dim] (bf16) over the cache
    into out: each row sees its sequence's positions up to its own, its own
    among them.  Query head h reads KV head h / (n_q / n_kv); rows that see
    nothing are zeros.  ``scale`` is 1 / sqrt(head_dim) unless given.
    ``workspace`` is a uint8 tensor of :func:`workspace_bytes`, one for each
    call that may run at the same time; without one, a call takes its own from
    torch's allocator."""
    if q.dim() != 3:
        raise ValueError(f"q is [tokens][heads][head_dim], not {tuple(q.shape)}")
    _one_gpu(cache, batch)
    device, n_q = cache.device, q.shape[1]
    shape = (batch.n_tokens, n_q, cache.head_dim)
    a, b = _rows(q, shape, device, "q", _BF16), _rows(out, shape, device, "out", _BF16)
    need = workspace_bytes(cache, batch, n_q)
    if not batch.n_seq or not batch.n_tokens:
        return
    at = size = None
    if workspace is not None:
        _whole(workspace, torch.uint8, (None,), device, "workspace")
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    if workspace is not None:
        at, size = workspace.data_ptr(), workspace.numel()
    _call("megakernel_op_kv8_attention", device, cache._ref, batch._ref, a, b, n_q,
          cache.head_dim ** -0.5 if scale is None else scale, at, size or 0)
