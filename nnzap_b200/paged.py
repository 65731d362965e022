"""Ragged serving over a paged KV cache, on torch CUDA tensors.

Prompt chunks and single tokens of many sequences share one pool of K/V
pages (the reference keeps one contiguous cache per model,
nnmetal/src/transformer.zig:648-700, and prefills token by token, :4032-4068):

* :class:`QKNormRope`: RMSNorm of every query and key head, rotation, and the
  new keys and values into their pages, in one pass;
* :class:`PagedAttention`: causal attention of the new tokens over the pages;
* :func:`token_logprobs`: log probabilities of given tokens, entropy and the
  most probable alternatives, from one read of the logits.

Every call is asynchronous on torch's current stream of the tensors' device
(which need not be the current device); errors found on the device (a page,
slot or token out of range) are reported by :func:`stream_check`.  Tensors that
a call uses must stay alive until its stream has run it, as with any torch
operation (``record_stream`` them if they were allocated on another stream).
The math runs in the CUDA library; this module checks and marshals arguments.
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _capi as capi
from ._capi import check, lib

_DTYPES = {torch.float16: capi.NNZ_DT_F16, torch.bfloat16: capi.NNZ_DT_BF16, torch.float32: capi.NNZ_DT_F32}
_ROPE = {"pairwise": capi.NNZ_ROPE_PAIRWISE, "half_split": capi.NNZ_ROPE_HALF_SPLIT}


# A device's current stream's handle.  (The raw query skips building a Stream object, about a microsecond.)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: torch.cuda.current_stream(device).cuda_stream)
# The library launches on the current device, and the default stream's handle is 0 on every device: a call whose
# tensors are elsewhere makes their device the current one first.
_current_device, _device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device), torch.cuda.device
_current_stream, _capturing = torch.cuda.current_stream, torch.cuda.is_current_stream_capturing


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


class _Own(threading.local):
    """Each thread's own copy of an operator's constant arguments, for a call to complete: the library reads them with
    the GIL released, while another thread may be calling the same operator."""

    def __init__(self, args):
        args = type(args).from_buffer_copy(args)
        self.args = args, C.byref(args)


def _index(t: torch.Tensor, dtype: torch.dtype, shape: tuple, device: torch.device, what: str) -> int:
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous {dtype} tensor of shape {tuple(shape)} on {device}, "
                         f"got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, tokens: int, width: int, kv: "PagedKV", what: str) -> int:
    """Checks a [tokens][width] matrix of the pool's dtype whose rows may be strided; its row stride."""
    if t.dtype is not kv.dtype or t.device != kv.device or t.dim() != 2 or t.shape[0] != tokens or t.shape[1] != width or (
            t.stride(1) != 1 and tokens):
        raise ValueError(f"{what}: expected {kv.dtype} [{tokens}][{width}] with adjacent elements on {kv.device}, "
                         f"got {t.dtype} {tuple(t.shape)} strides {t.stride()} on {t.device}")
    return t.stride(0) if tokens > 1 else max(t.stride(0), width)


class PagedKV:
    """A pool of K and V pages: two equally strided tensors indexed
    ``[page][kv head][token in page][d]``, float16 or bfloat16.  A pool stored
    token by token is passed as ``pool.transpose(1, 2)``."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _need(k.dim() == 4 and k.shape == v.shape, "k and v pages must be equal 4-d tensors [page][kv head][token][d]")
        _need(k.dtype == v.dtype and k.dtype in (torch.float16, torch.bfloat16), "pages must be float16 or bfloat16")
        _need(k.is_cuda and k.device == v.device, "pages must be on one CUDA device")
        _need(k.stride() == v.stride() and k.stride(3) == 1, "k and v pages need equal strides and adjacent elements")
        self.k, self.v = k, v
        self.dtype, self.device, self.index = k.dtype, k.device, k.device.index
        self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = k.shape
        c = capi.NnzPagedKv()
        c.k, c.v, c.dtype = k.data_ptr(), v.data_ptr(), _DTYPES[k.dtype]
        c.num_pages, c.num_kv_heads, c.page_size, c.head_dim = self.num_pages, self.num_kv_heads, self.page_size, self.head_dim
        c.page_stride, c.head_stride, c.token_stride = k.stride(0), k.stride(1), k.stride(2)
        self.c = c
        self._ref = C.byref(c)

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, dtype=torch.float16, device="cuda") -> "PagedKV":
        """A new pool stored head by head."""
        return cls(*(torch.zeros(num_pages, num_kv_heads, page_size, head_dim, dtype=dtype, device=device) for _ in range(2)))


def rope_table(theta: float, head_dim: int, positions: int, device="cuda") -> torch.Tensor:
    """float32 ``[positions][head_dim / 2][2]`` (cos, sin) of position times
    theta^(-2 i / head_dim), evaluated in double precision."""
    _need(positions > 0, "rope_table: positions")
    with _device(device):
        t = torch.empty(positions, head_dim // 2, 2, dtype=torch.float32, device=device)
        check(lib().nnz_rope_table(theta, head_dim, positions, t.data_ptr(), _stream(t.device.index)))
    return t


class QKNormRope:
    """``op(qkv, positions, slots)``: from one matrix of projections (query |
    key | value heads of every new token) to normed and rotated queries
    (returned) and the normed and rotated keys and the values in their pages.

    ``slots[t]`` (int64) is page * page_size + place, negative for a token that
    is not to be written; ``positions`` (int32) index ``table``
    (:func:`rope_table`)."""

    def __init__(self, kv: PagedKV, num_query_heads: int, q_norm: torch.Tensor, k_norm: torch.Tensor, table: torch.Tensor,
                 eps: float = 1e-6, rope_style: str = "pairwise"):
        hd = kv.head_dim
        self.kv, self.num_query_heads = kv, num_query_heads
        self._qd, self._width = num_query_heads * hd, (num_query_heads + 2 * kv.num_kv_heads) * hd
        self._keep = (q_norm, k_norm, table)
        a = capi.NnzNormRopeArgs()
        a.num_query_heads, a.eps, a.rope_style = num_query_heads, eps, _ROPE[rope_style]
        a.q_norm = _index(q_norm, torch.float32, (hd,), kv.device, "q_norm")
        a.k_norm = _index(k_norm, torch.float32, (hd,), kv.device, "k_norm")
        a.rope_table = _index(table, torch.float32, (table.shape[0], hd // 2, 2), kv.device, "table")
        a.table_positions = table.shape[0]
        self._own, self._fn = _Own(a), lib().nnz_qk_norm_rope_paged

    def __call__(self, qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        kv, n = self.kv, qkv.shape[0]
        if _current_device() != kv.index:
            with _device(kv.index):
                return self(qkv, positions, slots, out)
        a, ref = self._own.args
        if out is None:
            out = torch.empty(n, self._qd, dtype=kv.dtype, device=kv.device)
        a.qkv_stride = _rows(qkv, n, self._width, kv, "qkv")
        a.q_stride = _rows(out, n, self._qd, kv, "out")
        a.positions = _index(positions, torch.int32, (n,), kv.device, "positions")
        a.slots = _index(slots, torch.int64, (n,), kv.device, "slots")
        a.qkv, a.q_out, a.tokens = qkv.data_ptr(), out.data_ptr(), n
        rc = self._fn(kv._ref, ref, _stream(kv.index))
        if rc:
            check(rc)
        return out


class Workspace:
    """Memory that a :class:`PagedAttention` call's kernels hand their parts on
    through, and which every call leaves as it found it: one call uses it at a
    time, of whichever operator has it.  A call on another stream than the last
    one's waits for that one on the device (or, the first call, for the zeros),
    and the allocator learns of the stream.  Inside a graph capture it does
    neither: the order of a graph's launches is that of who replays it."""

    def __init__(self, nbytes: int, device: torch.device):
        self.lock = threading.Lock()
        self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        self._last = _current_stream(device)
        self.handle = self._last.cuda_stream       # the stream of the last use

    def move(self, handle: int) -> None:
        """The next use is on the current stream, whose handle this is (under the lock)."""
        if _capturing():
            return
        now = _current_stream(self.buf.device)
        now.wait_stream(self._last)
        self.buf.record_stream(now)
        self._last, self.handle = now, handle


class PagedAttention:
    """``op(q, page_table, q_start, kv_len, max_new)``: causal attention of
    every sequence's new tokens over its pages.

    ``q`` holds the new tokens of all sequences one after the other; sequence
    s has rows ``q_start[s]:q_start[s + 1]`` and ``kv_len[s]`` keys, its new
    tokens' included, on the pages ``page_table[s]`` (negative: absent).
    ``max_new`` is a host-known upper bound of one sequence's new tokens,
    ``scale`` positive (None: 1 / sqrt(head_dim)).

    The object's ``workspace`` serves one call at a time: threads may share the
    object, and a call on another stream waits for the one before.  Operators
    whose calls follow one another (a model's layers) can have one workspace:
    pass the first one's as ``workspace``."""

    def __init__(self, kv: PagedKV, num_query_heads: int, scale: float | None = None, workspace: Workspace | None = None):
        # (0 is the library's word for the default)
        _need(scale is None or 0 < C.c_float(scale).value < float("inf"), f"scale must be positive and finite, got {scale}")
        self.kv, self.num_query_heads = kv, num_query_heads
        self._qd = num_query_heads * kv.head_dim
        with _device(kv.index):      # the workspace follows the device's number of SMs
            n = lib().nnz_paged_attn_workspace(kv._ref, num_query_heads)
            _need(n > 0, f"paged attention over these pages does not take {num_query_heads} query heads")
            self.workspace = Workspace(n, kv.device) if workspace is None else workspace
        buf = self.workspace.buf
        _need(buf.device == kv.device and buf.numel() >= n, f"workspace: expected {n} bytes on {kv.device}, got {buf.numel()} on {buf.device}")
        a = capi.NnzPagedAttnArgs()
        a.num_query_heads, a.scale = num_query_heads, 0.0 if scale is None else scale
        a.workspace, a.workspace_bytes = buf.data_ptr(), n
        self._own, self._fn = _Own(a), lib().nnz_paged_attn

    def __call__(self, q: torch.Tensor, page_table: torch.Tensor, q_start: torch.Tensor, kv_len: torch.Tensor, max_new: int,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        kv, n, seqs = self.kv, q.shape[0], kv_len.shape[0]
        if _current_device() != kv.index:
            with _device(kv.index):
                return self(q, page_table, q_start, kv_len, max_new, out)
        if not 0 <= max_new < 1 << 31:      # (ctypes would wrap it)
            raise ValueError(f"max_new: {max_new}")
        a, ref = self._own.args
        if out is None:   # rows outside every sequence are not written
            out = torch.zeros(n, self._qd, dtype=kv.dtype, device=kv.device)
        a.q_stride = _rows(q, n, self._qd, kv, "q")
        a.out_stride = _rows(out, n, self._qd, kv, "out")
        a.q_start = _index(q_start, torch.int32, (seqs + 1,), kv.device, "q_start")
        a.kv_len = _index(kv_len, torch.int32, (seqs,), kv.device, "kv_len")
        a.table_stride = width = page_table.shape[1]
        a.page_table = _index(page_table, torch.int32, (seqs, width), kv.device, "page_table")
        a.q, a.out, a.tokens, a.num_seqs, a.max_new = q.data_ptr(), out.data_ptr(), n, seqs, max_new
        ws, stream = self.workspace, _stream(kv.index)
        with ws.lock:         # no other call's launch between the kernels of this one
            if stream != ws.handle:
                ws.move(stream)
            rc = self._fn(kv._ref, ref, stream)
        if rc:
            check(rc)
        return out


class TokenLogprobs:
    """What :func:`token_logprobs` returns: views of one allocation, made when they are asked for."""
    __slots__ = ("_f", "_shape", "_rows", "_m", "_k", "top_ids")

    def __init__(self, f, shape, rows, m, k, top_ids):
        self._f, self._shape, self._rows, self._m, self._k, self.top_ids = f, shape, rows, m, k, top_ids

    @property
    def entropy(self) -> torch.Tensor:
        """float32 [rows]"""
        return self._f.as_strided((self._rows,), (1,), 0)

    @property
    def logsumexp(self) -> torch.Tensor:
        """float32 [rows]"""
        return self._f.as_strided((self._rows,), (1,), self._rows)

    @property
    def logprob(self) -> torch.Tensor | None:
        """float32, the given tokens' shape"""
        if self._shape is None:
            return None
        return self._f.as_strided(self._shape, (1,) if len(self._shape) == 1 else (self._m, 1), 2 * self._rows)

    @property
    def top_logprobs(self) -> torch.Tensor | None:
        """float32 [rows][top_k]; ``top_ids`` int32 alike (both None for top_k 0)"""
        if not self._k:
            return None
        return self._f.as_strided((self._rows, self._k), (self._k, 1), (2 + self._m) * self._rows)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities (natural) of ``tokens`` (int32 ``[rows]`` or
    ``[rows][m]``; negative: no token, 0) under softmax(logits), with each
    row's entropy and its ``top_k`` (<= 32) most probable tokens in order,
    equal ones by id.  ``logits`` float32, float16 or bfloat16 ``[rows][n]``,
    rows may be strided; they are not changed."""
    if logits.dim() != 2 or logits.dtype not in _DTYPES or not logits.is_cuda:
        raise ValueError(f"logits: expected float32, float16 or bfloat16 [rows][n] on a CUDA device, got {logits.dtype} "
                         f"{tuple(logits.shape)} on {logits.device}")
    if _current_device() != logits.device.index:
        with _device(logits.device.index):
            return token_logprobs(logits, tokens, top_k)
    rows, n = logits.shape
    _need(n > 0 and (n == 1 or logits.stride(1) == 1), "logits: adjacent elements, at least one")
    _need(0 <= top_k <= 32, "top_k must be 0 .. 32")
    a, dev = capi.NnzLogprobsArgs(), logits.device
    if tokens is None:
        m = 0
    else:
        m = 1 if tokens.dim() == 1 else tokens.shape[1]
        a.tokens = _index(tokens, torch.int32, (rows,) if tokens.dim() == 1 else (rows, m), dev, "tokens")
    f = torch.empty(rows * (2 + m + top_k), dtype=torch.float32, device=dev)     # entropy | logsumexp | logprob | top
    p, ids = f.data_ptr(), None
    a.entropy, a.logsumexp = p, p + 4 * rows
    if m:
        a.num_tokens, a.logprob = m, p + 8 * rows
    if top_k:
        ids = torch.empty((rows, top_k), dtype=torch.int32, device=dev)
        a.top_k, a.top_ids, a.top_logprobs = top_k, ids.data_ptr(), p + 4 * rows * (2 + m)
    a.logits, a.dtype, a.rows, a.n = logits.data_ptr(), _DTYPES[logits.dtype], rows, n
    a.stride = logits.stride(0) if rows > 1 else n
    rc = lib().nnz_token_logprobs(C.byref(a), _stream(dev.index))
    if rc:
        check(rc)
    return TokenLogprobs(f, None if tokens is None else tuple(tokens.shape), rows, m, top_k, ids)


def stream_check(device=None) -> None:
    """Waits for the current stream of ``device`` (None: the current device) and raises what its kernels found wrong
    (``nnz_stream_check``)."""
    with _device(device):
        check(lib().nnz_stream_check(_stream(_current_device())))
