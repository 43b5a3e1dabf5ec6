"""Windowed attention with sinks on the HIP library.

The token at position i of a sequence sees the tokens j <= i with
j > i - window (every j <= i without a window), and the first ``sinks`` tokens
whatever their distance.  No counterpart in the reference; it stands beside
``PagedAttention`` (``real_page.py``) and reads the same cache:

* ``forward``  one new token per sequence over its cached context, the call
  of ``PagedAttention.forward``;
* ``prefill``  several new tokens per sequence over the same cache;
* ``dense``    packed sequences whose keys and values stand beside the queries,
  with gradients (the cached calls have none: a backward pass through them raises).

All take fp16 or bf16 and up to 1024 query heads per kv head.  Every call
runs on the current stream of its tensors' device, never synchronises, and may
be captured into a graph; scratch memory is torch's, allocated per call.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple

import torch

from hip_extends import _lib

from ... import flags
from ..block.common import int32
from ..block.real import LayerBlocksHolder
from .common import AttentionConfig

_DTYPES = {torch.float16: _lib.DW4_F16, torch.bfloat16: _lib.DW4_BF16}


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """The library launches on the current device."""
    if device.type != "cuda":
        raise ValueError("windowed attention runs on a HIP device")
    if device.index is None or device.index == _lib.current_device():
        return _HERE
    return torch.cuda.device(device)


def _dtype(*tensors: torch.Tensor) -> int:
    dtype = _DTYPES.get(tensors[0].dtype)
    if dtype is None or any(t.dtype != tensors[0].dtype for t in tensors):
        raise TypeError("windowed attention runs on fp16 or bf16 tensors of one type")
    return dtype


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [rows, heads, dims] with its heads side by side and rows that the
    kernels can read in 16-byte units; a copy where it is not so."""
    rows, heads, dims = x.shape
    if x.stride(2) != 1 or (heads > 1 and x.stride(1) != dims) or x.data_ptr() % 16 or \
            (rows > 1 and (x.stride(0) % 8 or x.stride(0) < heads * dims)):
        return x.contiguous() if not x.is_contiguous() else x.clone()
    return x


def _stride(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1] * x.shape[2]


def _like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _bound(n: int) -> int:
    """An upper bound as the library takes it (longer than any sequence is as good)."""
    return min(int(n), 2 ** 31 - 1)


def _ints(x: torch.Tensor, count: int, device: torch.device, name: str) -> torch.Tensor:
    if x.dim() != 1 or x.numel() != count or x.device != device:
        raise ValueError(f"{name} must be {count} integers on the queries' device")
    return int32(x, name)


class _NoGradient(torch.autograd.Function):
    """The cached calls have no backward pass: one that reaches them fails instead of
    finding no gradient."""

    @staticmethod
    def forward(ctx, query, output):
        return output.detach()  # (of the same memory: a given output stays outside the graph)

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("windowed attention over a cache has no gradients (WindowAttention.dense has)")


class WindowAttention:
    def __init__(self, config: AttentionConfig, window: Optional[int] = None,
                 sinks: int = 0) -> None:
        if window is not None and window < 1:
            raise ValueError("window must be at least 1, or None")
        if sinks < 0:
            raise ValueError("sinks must not be negative")
        self.cfg = config
        self.scale = self.cfg.head_dim ** -0.5
        self.window = window
        self.sinks = sinks
        # what the library takes: no window is 0, a longer one than any context is none
        self._window = 0 if window is None or window >= 1 << 30 else int(window)
        self._sinks = min(int(sinks), 1 << 30)

    def _check(self, x: torch.Tensor, heads: int, name: str) -> None:
        if x.dim() != 3 or x.shape[1] != heads or x.shape[2] != self.cfg.head_dim:
            raise AssertionError(f"{name} shape does not match the attention config")

    def forward(self, query: torch.Tensor, context_len_max: int, context_lens: torch.Tensor,
                block_tables: torch.Tensor, kv_cacher: LayerBlocksHolder,
                output: Optional[torch.Tensor] = None) -> torch.Tensor:
        """query [seqs, query heads, head_dim], one new token per sequence (its key
        and value cached, ``context_lens`` counting it) -> out of the same shape.
        ``context_len_max``, an upper bound of them, lies within the tables' columns.
        A block table entry that is no block (-1) means that the block was given
        back; an empty context gives zeros."""
        return self._paged(query, None, query.shape[0], 1, context_len_max, context_lens,
                           block_tables, kv_cacher, output)

    def prefill(self, query: torch.Tensor, query_starts: torch.Tensor, query_len_max: int,
                context_len_max: int, context_lens: torch.Tensor, block_tables: torch.Tensor,
                kv_cacher: LayerBlocksHolder,
                output: Optional[torch.Tensor] = None) -> torch.Tensor:
        """query [rows, query heads, head_dim]: sequence s has the rows
        ``query_starts[s]`` to ``query_starts[s + 1]`` (int32 [seqs + 1], ascending), at most
        ``query_len_max`` of them, the last at position ``context_lens[s] - 1``; their
        keys and values are in the cache.  Rows of no sequence are left as they are
        in ``output`` (and undefined where none is given)."""
        return self._paged(query, query_starts, query_starts.numel() - 1, query_len_max,
                           context_len_max, context_lens, block_tables, kv_cacher, output)

    def _paged(self, query, query_starts, num_seqs, query_len_max, context_len_max, context_lens,
               block_tables, kv_cacher, output):
        cfg, info = self.cfg, kv_cacher.block_info
        self._check(query, cfg.num_query_heads, "query")
        dtype, device = _dtype(query), query.device
        if info.head_dim != cfg.head_dim or info.num_key_value_heads != cfg.num_key_value_heads:
            raise AssertionError("the cache's block geometry does not match the attention config")
        if kv_cacher.dtype != query.dtype:
            raise TypeError(f"queries of {query.dtype} over a cache of {kv_cacher.dtype}")
        if kv_cacher.device != device or block_tables.device != device:
            raise ValueError("cache and block tables must be on the queries' device")
        if block_tables.dim() != 2 or block_tables.shape[0] != num_seqs:
            raise ValueError("block_tables must hold one row of block numbers per sequence")
        rows, query_len_max, context_len_max = query.shape[0], _bound(query_len_max), _bound(context_len_max)
        lens = _ints(context_lens, num_seqs, device, "context_lens")
        starts = None if query_starts is None else _ints(query_starts, num_seqs + 1, device, "query_starts")
        if output is None:
            output = _like(query)
        elif output.shape != query.shape or output.dtype != query.dtype or output.device != device:
            raise ValueError("output must have the queries' shape, type and device")
        elif _rows(output) is not output:
            raise ValueError("output rows must be contiguous and 16-byte aligned")
        tables = int32(block_tables, "block_tables")
        with _on(device):
            q = _rows(query)
            nbytes = _lib.window_attention_workspace_size(
                num_seqs, cfg.num_query_heads, cfg.num_key_value_heads, cfg.head_dim,
                flags.BLOCK_SIZE, rows, query_len_max, self._window, self._sinks,
                context_len_max, device.index)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
            _lib.call("dw4_window_attention", dtype, num_seqs, cfg.num_query_heads,
                      cfg.num_key_value_heads, cfg.head_dim, flags.BLOCK_SIZE,
                      min(kv_cacher.layer_key_ptr_table_device.numel(),
                          kv_cacher.layer_val_ptr_table_device.numel()), q.data_ptr(), _stride(q),
                      output.data_ptr(), _stride(output), None if starts is None else starts.data_ptr(),
                      rows, query_len_max, kv_cacher.layer_key_ptr_table_device.data_ptr(),
                      kv_cacher.layer_val_ptr_table_device.data_ptr(), info.head_stride,
                      float(self.scale), self._window, self._sinks, tables.data_ptr(),
                      tables.shape[1], lens.data_ptr(), context_len_max,
                      None if ws is None else ws.data_ptr(), nbytes,
                      _lib.current_stream(device.index))
        if query.requires_grad and torch.is_grad_enabled():
            return _NoGradient.apply(query, output)
        return output

    def dense(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seq_starts: torch.Tensor,
              seq_len_max: int) -> torch.Tensor:
        """Packed sequences: q [rows, query heads, head_dim], k and v [rows, kv heads,
        head_dim], sequence s in the rows ``seq_starts[s]`` to ``seq_starts[s + 1]``
        (int32 [seqs + 1], ascending), each at most ``seq_len_max`` long -> out like q; rows of
        no sequence, and those of a longer one beyond ``seq_len_max``, are zero and get zero
        gradients.  Differentiable in q, k and v (once)."""
        cfg = self.cfg
        self._check(q, cfg.num_query_heads, "q")
        self._check(k, cfg.num_key_value_heads, "k")
        self._check(v, cfg.num_key_value_heads, "v")
        _dtype(q, k, v)
        if k.shape[0] != q.shape[0] or v.shape[0] != q.shape[0]:
            raise AssertionError("q, k and v must have the same rows")
        if k.device != q.device or v.device != q.device:
            raise ValueError("q, k and v must be on one device")
        if seq_starts.numel() < 1:
            raise ValueError("seq_starts must hold one entry more than there are sequences")
        starts = _ints(seq_starts, seq_starts.numel(), q.device, "seq_starts")
        return _WindowDense.apply(q, k, v, starts, _bound(seq_len_max), self)


class _WindowDense(torch.autograd.Function):
    @staticmethod
    def _shape(att: WindowAttention, q: torch.Tensor, starts: torch.Tensor) -> Tuple[int, ...]:
        cfg = att.cfg
        return (_DTYPES[q.dtype], starts.numel() - 1, cfg.num_query_heads, cfg.num_key_value_heads,
                cfg.head_dim)

    @staticmethod
    def forward(ctx, q, k, v, starts, seq_len_max, att):
        device = q.device
        with _on(device):
            q, k, v = _rows(q), _rows(k), _rows(v)
            if starts.numel() == 1 or seq_len_max == 0 or q.shape[0] == 0:
                ctx.empty = True
                ctx.save_for_backward(q, k, v)
                return torch.zeros(q.shape, dtype=q.dtype, device=device)
            out = _like(q)
            need = any(ctx.needs_input_grad[:3])
            lse = torch.empty(q.shape[:2], dtype=torch.float32, device=device) if need else None
            rest = _like(q) if need else None
            _lib.call("dw4_window_attention_dense", *_WindowDense._shape(att, q, starts),
                      q.data_ptr(), _stride(q), k.data_ptr(), _stride(k), v.data_ptr(), _stride(v),
                      out.data_ptr(), _stride(out), None if lse is None else lse.data_ptr(),
                      None if rest is None else rest.data_ptr(), starts.data_ptr(), q.shape[0], seq_len_max, float(att.scale), att._window,
                      att._sinks, _lib.current_stream(device.index))
        ctx.empty = False
        ctx.att, ctx.seq_len_max = att, seq_len_max
        if need:
            ctx.save_for_backward(q, k, v, out, lse, rest, starts)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        if ctx.empty:
            return (*(torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in ctx.saved_tensors),
                    None, None, None)
        q, k, v, out, lse, rest, starts = ctx.saved_tensors
        att, device = ctx.att, q.device
        with _on(device):
            do = _rows(dout)
            dq, dk, dv = _like(q), _like(k), _like(v)
            shape = _WindowDense._shape(att, q, starts)
            nbytes = _lib.window_attention_backward_workspace_size(
                *shape[1:], q.shape[0], ctx.seq_len_max, att._window, att._sinks, device.index)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
            _lib.call("dw4_window_attention_dense_backward", *shape, q.data_ptr(), _stride(q),
                      k.data_ptr(), _stride(k), v.data_ptr(), _stride(v), out.data_ptr(), _stride(out),
                      lse.data_ptr(), rest.data_ptr(), do.data_ptr(), _stride(do), dq.data_ptr(), _stride(dq),
                      dk.data_ptr(), _stride(dk), dv.data_ptr(), _stride(dv), starts.data_ptr(),
                      q.shape[0], ctx.seq_len_max, float(att.scale), att._window, att._sinks,
                      ws.data_ptr(), nbytes, _lib.current_stream(device.index))
        return dq, dk, dv, None, None, None
