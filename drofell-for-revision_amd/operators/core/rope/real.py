"""Rotary positions on the HIP library.

Stands beside ``attention_forward_rope_stage_v2_py`` (``hip_extends/w4a16.py``) and
``LayerBlocksHolder.rope_and_cache``, which keep the reference's fp16 arithmetic over sin / cos
tables (``cuda_extends/exllama/fuse_v2/rope.cu``, paths relative to
``/root/reference/After-Revision-DROFELL``): here rows of any positions, fp16 or bf16, both pair
layouts, a part of the head, scaled frequencies, angles computed from the position (no table, as
exact at far positions as at near ones), and gradients.

* ``forward``         queries and keys turned, differentiable;
* ``forward_cached``  queries turned, keys turned and values as they are into their cache
                      slots, in one launch, for ragged batches of prompts and single tokens.

Every call runs on the current stream of its tensors' device, never synchronises, keeps nothing
and may be captured into a graph.
"""
from __future__ import annotations

import math
from fractions import Fraction
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from hip_extends import _lib

from ... import flags
from ..block.common import int32, no_tangents
from ..block.real import LayerBlocksHolder
from .common import RotaryScaling, rotary_frequencies

_TWO_PI = Fraction(62831853071795864769252867665590057683943, 10 ** 40)
_DTYPES = {torch.float16: _lib.DW4_F16, torch.bfloat16: _lib.DW4_BF16}


def _rows(x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """x [rows, heads, dims] with its heads side by side and rows in 16-byte units (a copy
    where it is not so), and its row stride."""
    rows, heads, dims = x.shape
    width, aligned = heads * dims, x.data_ptr() % 16 == 0
    if aligned and x.is_contiguous():
        return x, width
    if not aligned or x.stride(2) != 1 or (heads > 1 and x.stride(1) != dims) or \
            (rows > 1 and (x.stride(0) % 8 or x.stride(0) < width)):
        return x.clone(memory_format=torch.contiguous_format), width
    return x, x.stride(0) if rows > 1 else width


class RotaryEmbedding:
    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0,
                 interleaved: bool = False, scaling: Optional[RotaryScaling] = None,
                 device: Optional[torch.device] = None) -> None:
        """The first ``rotary_dim`` dims of a head (an even number; all by default) turn, in
        pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1) if ``interleaved``; pair i by
        base^(-2 i / rotary_dim) radians a position, scaled as ``scaling`` says."""
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 8 or head_dim % 8 or head_dim > 512:
            raise ValueError("head_dim must be a multiple of 8 up to 512")
        if rotary_dim < 2 or rotary_dim % 2 or rotary_dim > head_dim:
            raise ValueError("rotary_dim must be even, at least 2 and at most head_dim")
        if not (math.isfinite(base) and base > 1):
            raise ValueError("the base must be above 1")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError("rotary positions run on a HIP device")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, bool(interleaved)
        self.frequencies, self.magnitude = rotary_frequencies(rotary_dim, base, scaling)
        # turns per position as 64-bit fractions: their products with positions wrap at whole turns
        turns = [round(Fraction(f) / _TWO_PI * 2 ** 64) % 2 ** 64 for f in self.frequencies]
        self._turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns],
                                   dtype=torch.int64).to(device)
        self.device = self._turns.device

    def _check(self, *rows: torch.Tensor) -> int:
        dtype, count, dims = rows[0].dtype, rows[0].shape[0], self.head_dim
        for x in rows:
            shape = x.shape
            if len(shape) != 3 or shape[2] != dims or shape[0] != count:
                raise AssertionError(f"q, k and v must be [rows, heads, {dims}], of the same rows")
            if x.dtype != dtype:
                raise TypeError("q, k and v must have one type")
            if x.device != self.device:
                raise ValueError(f"q, k and v must be on {self.device}")
        if dtype not in _DTYPES:
            raise TypeError("rotary positions run on fp16 or bf16")
        no_tangents(*rows)
        if count > 1 << 22 or rows[0].shape[1] > 1 << 14 or rows[1].shape[1] > 1 << 14:
            raise ValueError("a call turns up to 2^22 rows and 2^14 heads")
        return count

    def _positions(self, positions: torch.Tensor, rows: int) -> torch.Tensor:
        if positions.shape != (rows,) or positions.device != self.device:
            raise ValueError(f"positions must be {rows} integers on {self.device}")
        # (every 64-bit number is a position)
        return positions.contiguous() if positions.dtype is torch.int64 else int32(positions, "positions")

    def _form(self, positions: torch.Tensor) -> int:
        return (_lib.DW4_ROTARY_INTERLEAVED if self.interleaved else 0) | \
            (_lib.DW4_ROTARY_POSITIONS64 if positions.dtype is torch.int64 else 0)

    def _turn(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
              inverse: bool) -> Tuple[torch.Tensor, torch.Tensor]:
        if not _lib.is_current(self.device):
            with torch.cuda.device(self.device):
                return self._turn(q, k, positions, inverse)
        (q, ldq), (k, ldk) = _rows(q), _rows(k)
        rows, heads, dims = q.shape
        kv_heads = k.shape[1]
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
        _lib.call("dw4_rotary", _DTYPES[q.dtype], rows, heads, kv_heads, dims, self.rotary_dim, self._form(positions),
                  int(inverse), q.data_ptr(), ldq, k.data_ptr(), ldk, qo.data_ptr(), heads * dims, ko.data_ptr(),
                  kv_heads * dims, positions.data_ptr(), self._turns.data_ptr(), self.magnitude,
                  _lib.current_stream(self.device.index))
        return qo, ko

    def forward(self, q: torch.Tensor, k: torch.Tensor,
                positions: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """q [rows, heads, head_dim] and k [rows, kv heads, head_dim] turned by their rows'
        ``positions`` (integers [rows]; angles are as exact as fp32's up to 2^38) -> new tensors.  Differentiable in q and k
        (once, backward)."""
        pos = self._positions(positions, self._check(q, k))
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
            # (64-bit positions may be counted on before the backward pass)
            return _Rotary.apply(q, k, pos.clone() if pos is positions and pos.dtype is torch.int64 else pos, self)
        return self._turn(q, k, pos, False)

    def forward_cached(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                       slots: torch.Tensor, kv_cacher: LayerBlocksHolder,
                       output: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q turned (returned, or written to ``output``: q itself, or memory apart from q, k and
        v), k turned and v into their cache ``slots`` (integers [rows]; -1: the row is not cached,
        and so is a slot outside the cache's blocks).  k and v stay as they are.  No two rows may
        have one slot.  Without gradients: a backward pass through it, or through an ``output`` that
        required a gradient, raises."""
        if not _lib.is_current(self.device):
            with torch.cuda.device(self.device):
                return self.forward_cached(q, k, v, positions, slots, kv_cacher, output)
        rows, info = self._check(q, k, v), kv_cacher.block_info
        heads, kv_heads, dims = q.shape[1], k.shape[1], self.head_dim
        if v.shape[1] != kv_heads:
            raise AssertionError("k and v must have the same shape")
        if info.head_dim != dims or info.num_key_value_heads != kv_heads:
            raise AssertionError("k and v do not match the cache's block geometry")
        if kv_cacher.dtype != q.dtype:
            raise TypeError(f"rows of {q.dtype} into a cache of {kv_cacher.dtype}")
        if kv_cacher.device != self.device:
            raise ValueError(f"the cache must be on {self.device}")
        pos = self._positions(positions, rows)
        if slots.shape != (rows,) or slots.device != self.device:
            raise ValueError(f"slots must be {rows} integers on {self.device}")
        if slots.dtype is not torch.int64:
            slots = int32(slots, "slots").to(torch.int64)
        elif not slots.is_contiguous():
            slots = slots.contiguous()
        given, ldo = output is not None, heads * dims
        if not given:
            output = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif output.shape != q.shape or output.dtype != q.dtype or output.device != self.device:
            raise ValueError("output must have the queries' shape, type and device")
        else:
            same, ldo = _rows(output)
            if same is not output:
                raise ValueError("output rows must be contiguous and 16-byte aligned")
            if output.requires_grad and output.is_leaf and torch.is_grad_enabled():
                raise RuntimeError("output is a leaf that requires a gradient")
        (q2, ldq), (k2, ldk), (v2, ldv) = _rows(q), _rows(k), _rows(v)
        keys, values = kv_cacher.layer_key_ptr_table_device, kv_cacher.layer_val_ptr_table_device
        _lib.call("dw4_rotary_and_cache", _DTYPES[q.dtype], rows, heads, kv_heads, dims, self.rotary_dim,
                  self._form(pos), q2.data_ptr(), ldq, k2.data_ptr(), ldk, v2.data_ptr(), ldv, output.data_ptr(),
                  ldo, pos.data_ptr(), self._turns.data_ptr(), self.magnitude, slots.data_ptr(),
                  min(keys.numel(), values.numel()), flags.BLOCK_SIZE, keys.data_ptr(), values.data_ptr(),
                  info.head_stride, _lib.current_stream(self.device.index))
        if given:
            increment_version(output)
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or output.requires_grad):
            return _NoGradient.apply(output, output.requires_grad, q, k, v)
        return output


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rotary):
        ctx.rotary = rotary
        ctx.save_for_backward(positions)
        return rotary._turn(q, k, positions, False)

    @staticmethod
    def backward(ctx, dq, dk):
        # (the wrapper that refuses a second derivative takes 3 us, and is needed where one may follow)
        return _Rotary._once(ctx, dq, dk) if torch.is_grad_enabled() else _Rotary._gradients(ctx, dq, dk)

    @staticmethod
    def _gradients(ctx, dq, dk):
        (positions,) = ctx.saved_tensors
        return (*ctx.rotary._turn(dq, dk, positions, True), None, None)

    _once = staticmethod(torch.autograd.function.once_differentiable(_gradients.__func__))


class _NoGradient(torch.autograd.Function):
    """A backward pass that reaches the cached call fails instead of finding no gradient, or by way of
    an output with a history of its own (the queries) that of what was there before."""

    @staticmethod
    def forward(ctx, output, in_place, *inputs):
        if in_place:
            ctx.mark_dirty(output)
            return output
        return output.detach()

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("rotary positions into a cache have no gradients (RotaryEmbedding.forward has)")
