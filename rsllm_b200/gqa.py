"""The grouped-head (GQA) paged KV cache: rotary append, page copies, prefill
and decode attention (``rkv_gqa_*`` of ``include/rsllm_kv_cuda.h``).

For a model with separate K and V heads beside the MLA rows of
``PagedKvPool``: pages hold 64 tokens here too, so the page tables, slots and
planning of ``PrefixKvPool`` (``device=None``, a plan-only pool) serve this
cache; ``GqaKvPool.apply_moves`` does the page copies it decides.
"""
from __future__ import annotations

import functools
import math
import threading
from ctypes import addressof, c_int32

import numpy as np
import torch

from . import _abi
from ._abi import PAGE_TOKENS
from .kvcache import CudaError, InvalidArgument, ShapeMismatch, check, raise_status_bits

# The current stream's handle without a Stream object around it, where this torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

# The current device without torch.cuda.current_device's check that CUDA is initialised (a pool's tensors are on it).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)

_DTYPES = {torch.bfloat16: _abi.GQA_BF16, torch.float16: _abi.GQA_F16}


class RotaryTable:
    """Cosines and sines of rotary positions: ``table`` f32
    ``[rows, rot_dim / 2, 2]`` on the GPU.  ``sections``: the pairs of each
    position axis (default: one axis has them all); ``interleaved``: pairs are
    neighbouring lanes instead of lanes half a rotary width apart."""

    def __init__(self, table: torch.Tensor, sections=None, interleaved: bool = False):
        if not isinstance(table, torch.Tensor) or table.dtype != torch.float32 or table.dim() != 3 or \
                table.shape[2] != 2 or not table.is_contiguous():
            raise ShapeMismatch("RotaryTable: table must be a contiguous float32 [rows, rot_dim / 2, 2] tensor")
        if not table.is_cuda:
            raise ShapeMismatch("RotaryTable: table must be on a CUDA device")
        pairs = table.shape[1]
        sections = (pairs,) if sections is None else tuple(int(x) for x in sections)
        if not 1 <= len(sections) <= 4:
            raise ShapeMismatch("RotaryTable: 1 to 4 sections")
        self.table = table
        self.sections = sections
        self.interleaved = bool(interleaved)
        self._c = _abi.GqaRotary(table.data_ptr(), table.shape[0], 2 * pairs, int(self.interleaved), len(sections),
                                 (c_int32 * 4)(*sections))
        self._p = addressof(self._c)

    @classmethod
    def build(cls, rows: int, rot_dim: int, theta: float = 10000.0, sections=None, interleaved: bool = False,
              device: int | str | torch.device = "cuda") -> "RotaryTable":
        """angle = position * theta ** (-2 i / rot_dim), computed in 64 bits."""
        half = rot_dim // 2
        freq = theta ** (-torch.arange(half, dtype=torch.float64) / half)
        angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
        table = torch.stack((angle.cos(), angle.sin()), dim=-1).float().to(device)
        return cls(table.contiguous(), sections, interleaved)


def _on_its_device(method):
    """The library launches on the current device: for the call, that is the pool's."""

    @functools.wraps(method)
    def call(self, *args, **kwargs):
        if _current_device() == self._index:
            return method(self, *args, **kwargs)
        with torch.cuda.device(self._index):
            return method(self, *args, **kwargs)

    return call


class _Kept(threading.local):
    """Workspaces by stream, of one thread: they go with it."""

    def __init__(self):
        self.by_stream = {}


class GqaKvPool:
    """A grouped-head paged cache on one GPU: ``cache``
    ``[n_layers, n_pages, 2 (K, V), n_kv_heads, 64, head_dim]``, bf16 or f16,
    head_dim 64 or 128.  Storage it makes itself is zeroed.

    Calls run on the cache's device, whichever is current, on its current
    stream or ``stream``.  Threads may call it side by side.  The attentions' workspaces are kept for
    each thread and stream that calls without one (up to 39 MB, with the pool
    or the thread); ``workspace=`` takes the caller's."""

    def __init__(self, n_pages: int, n_kv_heads: int, head_dim: int, n_layers: int = 1,
                 dtype: torch.dtype = torch.bfloat16, device: int | str | torch.device | None = None):
        if not torch.cuda.is_available():
            raise CudaError("GqaKvPool: no CUDA device")
        if min(n_pages, n_kv_heads, n_layers) <= 0:
            raise ShapeMismatch("GqaKvPool: n_pages, n_kv_heads and n_layers must be positive")
        if head_dim not in (64, 128):
            raise ShapeMismatch("GqaKvPool: head_dim must be 64 or 128")
        if dtype not in _DTYPES:
            raise InvalidArgument("GqaKvPool: dtype must be torch.bfloat16 or torch.float16")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self._bind(torch.zeros((n_layers, n_pages, 2, n_kv_heads, PAGE_TOKENS, head_dim), dtype=dtype, device=dev), None)

    @classmethod
    def over(cls, cache: torch.Tensor, status: torch.Tensor | None = None) -> "GqaKvPool":
        """A pool over a cache tensor the caller owns; ``status``: its device
        status word (int32 ``[1]``, zero), made here if not given."""
        if not isinstance(cache, torch.Tensor) or cache.dim() != 6 or cache.shape[2] != 2 or \
                cache.shape[4] != PAGE_TOKENS or cache.shape[5] not in (64, 128) or cache.numel() == 0 or \
                not cache.is_contiguous():
            raise ShapeMismatch("GqaKvPool: cache must be a contiguous [n_layers, n_pages, 2, n_kv_heads, 64, "
                                "64 or 128] tensor")
        if cache.dtype not in _DTYPES:
            raise InvalidArgument("GqaKvPool: cache must be bfloat16 or float16")
        if not cache.is_cuda:
            raise CudaError("GqaKvPool: cache must be on a CUDA device")
        pool = cls.__new__(cls)
        pool._bind(cache, status)
        return pool

    def _bind(self, cache: torch.Tensor, status: torch.Tensor | None) -> None:
        self.lib = _abi.load()
        self.cache = cache
        self.device = cache.device
        self._index = cache.get_device()
        self.dtype = cache.dtype
        self.n_layers, self.n_pages, _, self.n_kv_heads, _, self.head_dim = cache.shape
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=self.device)
        elif status.dtype != torch.int32 or status.numel() != 1 or status.device != self.device:
            raise ShapeMismatch("GqaKvPool: status must be an int32 tensor of one element on the cache's device")
        self.status = status
        self.view = _abi.GqaView(cache.data_ptr(), self.n_pages, self.n_layers, self.n_kv_heads, self.head_dim,
                                 _DTYPES[cache.dtype])
        self._v = addressof(self.view)
        self._s = status.data_ptr()
        self._prefill_ws = self.lib.rkv_gqa_prefill_workspace_bytes(self._v)
        self._decode_ws = {}  # bytes by number of q heads: they do not grow with the sequences
        self._kept = _Kept()
        self._scale = 1.0 / math.sqrt(self.head_dim)

    # -- status ---------------------------------------------------------------
    def take_status(self, stream: torch.cuda.Stream | None = None) -> int:
        """Synchronises, returns and clears the device status bits."""
        (stream or torch.cuda.current_stream(self.device)).synchronize()
        bits = int(self.status.item()) & 0xFFFFFFFF
        self.status.zero_()
        return bits

    def check(self, what: str = "GqaKvPool", stream: torch.cuda.Stream | None = None) -> None:
        raise_status_bits(self.take_status(stream), what)

    # -- argument checks (kept short: a small call's time is the host's) ------------
    def _rows(self, t: torch.Tensor, name: str, heads: int | None = None) -> tuple:
        """(pointer, token stride, head stride, shape) of a [tokens, heads, head_dim] operand."""
        if not isinstance(t, torch.Tensor) or t.dtype is not self.dtype or t.get_device() != self._index:
            raise ShapeMismatch(f"{name}: expected a {self.dtype} tensor on {self.device}")
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ShapeMismatch(f"{name}: expected [tokens, {heads or 'heads'}, {self.head_dim}], got {tuple(shape)}")
        if stride[2] != 1:
            raise ShapeMismatch(f"{name}: the {self.head_dim} elements of a row must be contiguous")
        # a stride that no second row uses may be anything
        return (t.data_ptr(), stride[0] if shape[0] > 1 else shape[1] * shape[2],
                stride[1] if shape[1] > 1 else shape[2], shape)

    def _need(self, t: torch.Tensor, dtype: torch.dtype, name: str, shape: tuple) -> int:
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != self._index:
            raise ShapeMismatch(f"{name}: expected a {dtype} tensor on {self.device}")
        if t.shape != shape or not t.is_contiguous():
            raise ShapeMismatch(f"{name}: expected a contiguous {tuple(shape)} tensor, got {tuple(t.shape)}")
        return t.data_ptr()

    def _table(self, page_table: torch.Tensor, n_seq: int) -> tuple:
        if page_table.dim() != 2:
            raise ShapeMismatch("page_table: expected [n_seq, stride]")
        stride = page_table.shape[1]
        return self._need(page_table, torch.int32, "page_table", (n_seq, stride)), stride

    def _out(self, out: torch.Tensor | None, q: torch.Tensor, shape, name: str, stream) -> tuple:
        """An output like q but contiguous; memory made for a call belongs to the stream that the call runs on."""
        if out is None:
            if stream is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
            else:
                with torch.cuda.stream(stream):
                    out = torch.empty_like(q, memory_format=torch.contiguous_format)
            return out, out.data_ptr()
        return out, self._need(out, self.dtype, name, shape)

    def _workspace(self, workspace: torch.Tensor | None, nbytes: int, stream, handle: int) -> torch.Tensor:
        """The caller's workspace, or one that the pool keeps for this thread and the current stream (of a thread's calls
        on a stream each comes after the one before; another thread's two launches may fall between a call's own);
        with a stream given, or in a graph's capture, memory of the call's own."""
        if workspace is not None:
            if workspace.get_device() != self._index or not workspace.is_contiguous() or \
                    workspace.numel() * workspace.element_size() < nbytes:
                raise ShapeMismatch(f"workspace: expected a contiguous tensor of {nbytes} bytes on {self.device}")
            return workspace
        if stream is not None:
            with torch.cuda.stream(stream):
                return torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        by_stream = self._kept.by_stream
        kept = by_stream.get(handle)
        if kept is None or kept.numel() < nbytes:
            kept = by_stream[handle] = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return kept

    def _stream(self, stream) -> int:
        if stream is not None:
            if stream.device_index != self._index:
                raise InvalidArgument(f"stream: expected one of {self.device}")
            return stream.cuda_stream
        return _raw_stream(self._index) if _raw_stream is not None else \
            torch.cuda.current_stream(self.device).cuda_stream

    # -- append -------------------------------------------------------------------
    @_on_its_device
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor,
               q: torch.Tensor | None = None, rotary: RotaryTable | None = None, pos: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None, stream: torch.cuda.Stream | None = None) -> torch.Tensor | None:
        """Stores k and v ``[tokens, n_kv_heads, head_dim]`` (views with any
        token and head strides that are multiples of 8) at the slots
        ``slot_mapping`` (int32 ``[tokens]``, negative = skip).  With ``rotary``
        k is rotated by the positions ``pos`` (int32 ``[tokens]``, or
        ``[axes, tokens]``), and q ``[tokens, n_q_heads, head_dim]``, if given,
        too: the rotated q is returned (``rkv_gqa_append``)."""
        kp, k_ts, k_hs, shape = self._rows(k, "k", self.n_kv_heads)
        vp, v_ts, v_hs, v_shape = self._rows(v, "v", self.n_kv_heads)
        n = shape[0]
        if v_shape[0] != n:
            raise ShapeMismatch("append: k and v differ in tokens")
        slots = self._need(slot_mapping, torch.int32, "slot_mapping", (n,))
        qp = q_ts = q_hs = heads = op = posp = 0
        if rotary is not None:
            if rotary.table.get_device() != self._index:
                raise ShapeMismatch("append: the rotary table is on another device")
            axes = len(rotary.sections)
            if pos is None:
                raise ShapeMismatch("append: rotary needs pos")
            posp = self._need(pos, torch.int32, "pos", (n,) if axes == 1 and pos.dim() == 1 else (axes, n))
        if q is not None:
            if rotary is None:
                raise InvalidArgument("append: q is only taken with rotary")
            qp, q_ts, q_hs, q_shape = self._rows(q, "q")
            if q_shape[0] != n:
                raise ShapeMismatch("append: q and k differ in tokens")
            heads = q_shape[1]
            q_out, op = self._out(q_out, q, q_shape, "q_out", stream)
        check(self.lib.rkv_gqa_append(self._v, layer, kp, k_ts, k_hs, vp, v_ts, v_hs, n, slots,
                                      rotary._p if rotary is not None else 0, posp, qp, q_ts, q_hs, heads, op, self._s,
                                      self._stream(stream)), "append")
        return q_out if q is not None else None

    # -- attention -----------------------------------------------------------------
    @_on_its_device
    def prefill(self, layer: int, q: torch.Tensor, cu_q: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
                softmax_scale: float | None = None, window: int = 0, sinks: torch.Tensor | None = None,
                out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Causal attention of packed new tokens q ``[tokens, n_q_heads,
        head_dim]`` (sequence s: rows ``cu_q[s]`` to ``cu_q[s + 1]``) over the
        ``kv_lens[s]`` rows of each sequence, which end with the new tokens'
        own (``rkv_gqa_prefill``).  The scale defaults to 1/sqrt(head_dim)."""
        qp, q_ts, q_hs, shape = self._rows(q, "q")
        n, heads = shape[0], shape[1]
        n_seq = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
        lens = self._need(kv_lens, torch.int32, "kv_lens", (n_seq,))
        cu = self._need(cu_q, torch.int32, "cu_q", (n_seq + 1,))
        table, stride = self._table(page_table, n_seq)
        sink = 0 if sinks is None else self._need(sinks, torch.float32, "sinks", (heads,))
        handle = self._stream(stream)
        ws = self._workspace(workspace, self._prefill_ws, stream, handle)
        out, op = self._out(out, q, shape, "out", stream)
        scale = self._scale if softmax_scale is None else softmax_scale
        rc = self.lib.rkv_gqa_prefill(self._v, layer, qp, q_ts, q_hs, n, heads, cu, n_seq, table, stride, lens, window,
                                      sink, scale, ws.data_ptr(), op, self._s, handle)
        if rc:
            check(rc, "prefill")
        return out

    @_on_its_device
    def decode(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, kv_lens: torch.Tensor,
               softmax_scale: float | None = None, window: int = 0, sinks: torch.Tensor | None = None,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Attention of one new token per sequence, q ``[n_seq, n_q_heads,
        head_dim]``, over its ``kv_lens[s]`` rows, the token's own (appended
        before) being the last (``rkv_gqa_decode``)."""
        qp, q_ts, q_hs, shape = self._rows(q, "q")
        n_seq, heads = shape[0], shape[1]
        lens = self._need(kv_lens, torch.int32, "kv_lens", (n_seq,))
        table, stride = self._table(page_table, n_seq)
        sink = 0 if sinks is None else self._need(sinks, torch.float32, "sinks", (heads,))
        if heads not in self._decode_ws:
            self._decode_ws[heads] = max(0, self.lib.rkv_gqa_decode_workspace_bytes(self._v, n_seq, heads))
        handle = self._stream(stream)
        ws = self._workspace(workspace, self._decode_ws[heads], stream, handle)
        out, op = self._out(out, q, shape, "out", stream)
        scale = self._scale if softmax_scale is None else softmax_scale
        rc = self.lib.rkv_gqa_decode(self._v, layer, qp, q_ts, q_hs, n_seq, heads, table, stride, lens, window, sink,
                                     scale, ws.data_ptr(), op, self._s, handle)
        if rc:
            check(rc, "decode")
        return out

    # -- page moves ------------------------------------------------------------------
    @_on_its_device
    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
        """Every layer: page dst[i] <- page src[i] (int32; disjoint sets)."""
        n = src.shape[0] if src.dim() == 1 else -1
        check(self.lib.rkv_gqa_copy_pages(self._v, self._need(src, torch.int32, "src", (n,)),
                                          self._need(dst, torch.int32, "dst", (n,)), n, self._s,
                                          self._stream(stream)), "copy_pages")

    @_on_its_device
    def apply_moves(self, src, dst, stream: torch.cuda.Stream | None = None) -> None:
        """Applies a plan-only pool's page moves (``PrefixKvPool.take_moves``,
        host arrays) in their order: as few ``copy_pages`` calls as keep a page
        that one call writes from being read or written again by it."""
        src, dst = np.asarray(src, dtype=np.int32).ravel(), np.asarray(dst, dtype=np.int32).ravel()
        if src.shape != dst.shape:
            raise ShapeMismatch("apply_moves: src and dst differ in length")
        start, read, written = 0, set(), set()
        for i, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
            if a in written or b in written or b in read:
                self._move(src[start:i], dst[start:i], stream)
                start, read, written = i, set(), set()
            read.add(a)
            written.add(b)
        self._move(src[start:], dst[start:], stream)

    def _move(self, src: np.ndarray, dst: np.ndarray, stream) -> None:
        if not src.size:
            return
        with torch.cuda.stream(stream):  # None: the current one
            both = torch.from_numpy(np.stack((src, dst))).to(self.device)
            self.copy_pages(both[0], both[1], stream)


__all__ = ["GqaKvPool", "RotaryTable"]
