"""Low-rank adapters of many requests beside a shared projection, on the HIP library.

A batch's rows go through one projection (a ``QuantLinear``, a ``MarlinQuantLinear``, or any
other), and each row adds the low-rank product of its own adapter, or of none:

    y_t = W x_t + scaling_a B_a (A_a d(x_t)),   a the row's adapter, d dropout (training).

* ``AdapterRows``     which adapter each row of a batch has, sorted once on the device for all
                      projections of all layers;
* ``LowRankAdapters`` the adapters of one projection, with gradients;
* ``AdaptedLinear``   a projection with its adapters;
* ``CounterDropout``  the adapters' dropout by itself: its mask comes from a counter and is
                      never stored.

The reference's adapters (``operators/core/lora``, paths relative to
``/root/reference/After-Revision-DROFELL``) are dense products of one adapter.

All take fp16 or bf16.  Every call runs on the current stream of its tensors' device, never
synchronises, keeps nothing between calls and may be captured into a graph; scratch memory is
torch's, allocated per call.  Give a training step to a graph when no eager autograd graph over the
same leaves is alive.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import nn
from torch.autograd.graph import increment_version
from torch.nn.modules import module as _modules

from hip_extends import _lib

from ..block.common import int32, no_tangents
from .real import Linear
from .real_marlin import MarlinQuantLinear
from .real_quant import QuantLinear

_DTYPES = {torch.float16: _lib.DW4_F16, torch.bfloat16: _lib.DW4_BF16}


def _whole(x: torch.Tensor) -> torch.Tensor:
    return x if x.is_contiguous() else x.contiguous()


def _matrix(x: torch.Tensor, width: int) -> Tuple[torch.Tensor, int]:
    """x [rows, width] as the kernels read it, in 16-byte units of its rows (a copy where it is not so),
    and its row stride."""
    aligned = x.data_ptr() % 16 == 0
    if aligned and x.is_contiguous():
        return x, width
    if not aligned or x.stride(1) != 1 or x.stride(0) % 8 or x.stride(0) < width:
        return x.clone(memory_format=torch.contiguous_format), width
    return x, x.stride(0)


def _drop(p: float) -> int:
    """A probability as the generator takes it, of 65536."""
    if not 0 <= p <= 1:
        raise ValueError("the probability of dropout lies between 0 and 1")
    return round(p * 65536)


def _seed(seed: Optional[torch.Tensor], device: torch.device) -> torch.Tensor:
    if seed is None:
        raise ValueError("dropout needs a seed (int64 [2], on the device: seed and offset)")
    if seed.dtype != torch.int64 or seed.shape != (2,) or seed.device != device:
        raise ValueError(f"the seed must be int64 [2] on {device}")
    return seed.contiguous()


class AdapterRows:
    """Which adapter each row of a batch has (``adapters``, integers [rows] on the device; a number
    outside 0 .. num_adapters - 1: none), sorted by adapter.  Made once per batch: every
    projection of every layer takes it.  Up to 2^24 rows and 1024 adapters."""

    def __init__(self, adapters: torch.Tensor, num_adapters: int) -> None:
        if adapters.dim() != 1:
            raise ValueError("adapters must hold one integer per row")
        if adapters.shape[0] > 1 << 24 or not 0 <= num_adapters <= 1024:
            raise ValueError("a batch has up to 2^24 rows and 1024 adapters")
        self.num_rows, self.num_adapters, self.device = adapters.shape[0], int(num_adapters), adapters.device
        _lib.is_current(self.device)  # (raises where it is no HIP device)
        self.plan = torch.empty(_lib.adapter_plan_size(self.num_rows, self.num_adapters) // 4, dtype=torch.int32,
                                device=self.device)
        self.update(adapters)

    def update(self, adapters: torch.Tensor) -> None:
        """The same rows with other adapters, in the memory that captured calls read."""
        if adapters.shape != (self.num_rows,) or adapters.device != self.device:
            raise ValueError(f"adapters must be {self.num_rows} integers on {self.device}")
        if not _lib.is_current(self.device):
            with torch.cuda.device(self.device):
                return self.update(adapters)
        index = int32(adapters, "adapters")
        _lib.call("dw4_adapter_plan", self.num_rows, self.num_adapters, index.data_ptr(), self.plan.data_ptr(),
                  self.plan.numel() * 4, _lib.current_stream(self.device.index))
        increment_version(self.plan)  # a backward pass that was to read the old one fails


class LowRankAdapters(nn.Module):
    def __init__(self, in_features: int, out_features: int, rank: int, num_adapters: int,
                 dtype: torch.dtype = torch.float16, device: Optional[torch.device] = None, dropout: float = 0.0,
                 trainable: bool = False) -> None:
        """``rank`` is a multiple of 8 up to 128: adapters of lower rank are filled up with zeros
        (``load``).  ``dropout`` applies to the adapters' input while the module is in training
        mode; its probability counts in steps of 2^-16."""
        super().__init__()
        if dtype not in _DTYPES:
            raise TypeError("adapters are fp16 or bf16")
        if rank < 8 or rank % 8 or rank > 128:
            raise ValueError("the rank must be a multiple of 8 up to 128")
        if any(width < 8 or width % 8 or width > 1 << 20 for width in (in_features, out_features)):
            raise ValueError("in_features and out_features must be multiples of 8 up to 2^20")
        if not 0 < num_adapters <= 1024:
            raise ValueError("there are 1 to 1024 adapters")
        self.in_features, self.out_features, self.rank, self.num_adapters = in_features, out_features, rank, num_adapters
        self.dropout = dropout
        self.a = nn.Parameter(torch.randn(num_adapters, rank, in_features, dtype=torch.float32, device=device)
                              .mul_(in_features ** -0.5).to(dtype), requires_grad=trainable)
        self.b = nn.Parameter(torch.zeros(num_adapters, out_features, rank, dtype=dtype, device=device),
                              requires_grad=trainable)
        self.register_buffer("scaling", torch.ones(num_adapters, dtype=torch.float32, device=device))
        self._shapes = self.a.shape, self.b.shape, self.scaling.shape

    @property
    def dropout(self) -> float:
        return self._dropout

    @dropout.setter
    def dropout(self, p: float) -> None:
        self._dropout, self._dropped = p, _drop(p)

    @torch.no_grad()
    def load(self, index: int, lora_a: torch.Tensor, lora_b: torch.Tensor, scaling: float) -> None:
        """Adapter ``index`` from its matrices A [r, in_features] and B [out_features, r], r up to
        the rank, and its scaling (alpha / r)."""
        r = lora_a.shape[0]
        if not 0 <= index < self.num_adapters:
            raise IndexError(f"there are {self.num_adapters} adapters")
        if r > self.rank or lora_a.shape != (r, self.in_features) or lora_b.shape != (self.out_features, r):
            raise ValueError(f"A and B must be [r, {self.in_features}] and [{self.out_features}, r], r up to {self.rank}")
        if "a" not in self._parameters or "b" not in self._parameters:
            raise RuntimeError("A or B is parametrized: load into what it is made of")
        a, b = torch.zeros_like(self.a[index]), torch.zeros_like(self.b[index])  # (the matrices may be parts of the bank)
        a[:r].copy_(lora_a)
        b[:, :r].copy_(lora_b)
        self.a[index].copy_(a)
        self.b[index].copy_(b)
        self.scaling[index] = scaling

    def forward(self, x: torch.Tensor, base: torch.Tensor, rows: AdapterRows, seed: Optional[torch.Tensor] = None,
                output: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x [..., in_features] and the projection's output ``base`` [..., out_features] ->
        base + each row's adapter's product.  ``seed``: int64 [2] on the device (seed and offset),
        read where dropout applies; another step takes another offset, another projection another
        seed.  Differentiable (once, backward) in x, base, ``a`` and ``b``.  ``output``, without gradients:
        where the result goes: ``base`` itself, or memory apart from it."""
        params = self._parameters  # (attribute look-up on a module takes 0.4 us each)
        try:
            a, b, scaling = params["a"], params["b"], self._buffers["scaling"]
        except KeyError:  # (parametrized)
            a, b, scaling = self.a, self.b, self.scaling
        device, dtype = x.device, x.dtype
        flat = x.dim() == 2 and base.dim() == 2
        x2, base2 = (x, base) if flat else (x.reshape(-1, x.shape[-1]), base.reshape(-1, base.shape[-1]))
        num_rows, width = x2.shape
        if width != self.in_features or base2.shape != (num_rows, self.out_features) or \
                not (flat or x.shape[:-1] == base.shape[:-1]):
            raise ValueError(f"x and base must be [..., {self.in_features}] and [..., {self.out_features}] of the same rows")
        if dtype not in _DTYPES or base.dtype != dtype or a.dtype != dtype or b.dtype != dtype:
            raise TypeError("x, base and the adapters must be of one type, fp16 or bf16")
        if (a.shape, b.shape, scaling.shape) != self._shapes:
            raise ValueError(f"A, B and the scaling must keep the shapes of {self.num_adapters} adapters of rank {self.rank}")
        if base.device != device or a.device != device or b.device != device or scaling.device != device or \
                rows.device != device:
            raise ValueError(f"x, base, the adapters and their rows must be on one device ({device})")
        if num_rows != rows.num_rows or rows.num_adapters != self.num_adapters:
            raise ValueError(f"rows were sorted for {rows.num_rows} rows of {rows.num_adapters} adapters, "
                             f"not for {num_rows} of {self.num_adapters}")
        no_tangents(x, base, a, b, scaling)
        drop = self._dropped if self.training else 0
        seed = _seed(seed, device) if drop else None
        if scaling.dtype != torch.float32:  # (of a module that was made half)
            scaling = scaling.float()
        if torch.is_grad_enabled() and (a.requires_grad or x.requires_grad or b.requires_grad or base.requires_grad):
            if output is not None:
                raise ValueError("output is for calls without gradients")
            out2 = _LowRank.apply(x2, base2, a, b, scaling, rows.plan, drop, seed)
            return out2 if flat else out2.view(base.shape)
        if output is None:
            out2 = _forward(x2, base2, a, b, scaling, rows.plan, drop, seed, None, False)[0]
            return out2 if flat else out2.view(base.shape)
        if output.shape != base.shape or output.dtype != dtype or output.device != device or \
                not output.is_contiguous() or output.data_ptr() % 16:
            raise ValueError("output must be contiguous and 16-byte aligned, of base's shape, type and device")
        if output.requires_grad and torch.is_grad_enabled():
            raise ValueError("output is for calls without gradients, and has one")
        _forward(x2, base2, a, b, scaling, rows.plan, drop, seed, output.view(-1, self.out_features), False)
        increment_version(output)
        return output


def _forward(x, base, a, b, scaling, plan, drop, seed, out, keep):
    """The call itself -> (out, x as the kernels read it, h or None, what the backward pass's call takes).
    (Each property of a tensor takes 0.1 to 0.2 us: they are read once.)"""
    device = x.device
    if not _lib.is_current(device):
        with torch.cuda.device(device):
            return _forward(x, base, a, b, scaling, plan, drop, seed, out, keep)
    rows, k = x.shape
    adapters, n, rank = b.shape
    x, ldx = _matrix(x, k)
    base, ldb = _matrix(base, n)
    a, b, scaling = _whole(a), _whole(b), _whole(scaling)
    nbytes, h_bytes = _lib.adapters_workspace_size(rows, adapters, k, n, rank, False, device.index)
    if out is None:
        out = torch.empty_like(base) if ldb == n else torch.empty_like(base, memory_format=torch.contiguous_format)
    ws = x.new_empty(nbytes // 2)  # (16-bit elements; torch.empty takes 0.6 us more)
    h = x.new_empty(h_bytes // 2) if keep else None
    shape = (_DTYPES[x.dtype], rows, adapters, k, n, rank)
    _lib.call("dw4_adapters", *shape, x.data_ptr(), ldx, base.data_ptr(), ldb, out.data_ptr(), n, a.data_ptr(),
              b.data_ptr(), scaling.data_ptr(), plan.data_ptr(), drop, None if seed is None else seed.data_ptr(),
              None if h is None else h.data_ptr(), ws.data_ptr(), nbytes, _lib.current_stream(device.index))
    if not keep:
        return out, x, h, None
    # worked out here: the backward pass runs in a thread of autograd's, where Python takes twice as long
    nbytes = _lib.adapters_workspace_size(rows, adapters, k, n, rank, True, device.index)[0] if rows else 0
    return out, x, h, (shape, drop, nbytes, device, ldx)


class _LowRank(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, base, a, b, scaling, plan, drop, seed):
        a, b, scaling = _whole(a), _whole(b), _whole(scaling)
        out, x, h, ctx.call = _forward(x, base, a, b, scaling, plan, drop, seed, None, True)
        ctx.save_for_backward(x, a, b, scaling, plan, h, seed)
        return out

    @staticmethod
    def backward(ctx, dout):
        # (the wrapper that refuses a second derivative takes 3 us, and is needed where one may follow)
        return _LowRank._once(ctx, dout) if torch.is_grad_enabled() else _LowRank._gradients(ctx, dout)

    @staticmethod
    def _gradients(ctx, dout):
        x, a, b, scaling, plan, h, seed = ctx.saved_tensors
        shape, drop, nbytes, device, ldx = ctx.call
        need_x, need_base, need_a, need_b = ctx.needs_input_grad[:4]
        dbase = dout if need_base else None
        if shape[1] == 0:
            return (torch.zeros_like(x) if need_x else None, dbase, torch.zeros_like(a) if need_a else None,
                    torch.zeros_like(b) if need_b else None, None, None, None, None)
        if not (need_x or need_a or need_b):
            return None, dbase, None, None, None, None, None, None
        if not _lib.is_current(device):
            with torch.cuda.device(device):
                return _LowRank._gradients(ctx, dout)
        g, ldg = _matrix(dout, shape[4])
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
        da = torch.empty_like(a) if need_a else None
        db = torch.empty_like(b) if need_b else None
        ws = x.new_empty(nbytes // 2)
        _lib.call("dw4_adapters_backward", *shape, x.data_ptr(), ldx, g.data_ptr(), ldg, a.data_ptr(), b.data_ptr(),
                  scaling.data_ptr(), plan.data_ptr(), drop, None if seed is None else seed.data_ptr(), h.data_ptr(),
                  None if dx is None else dx.data_ptr(), shape[3], None if da is None else da.data_ptr(),
                  None if db is None else db.data_ptr(), ws.data_ptr(), nbytes, _lib.current_stream(device.index))
        return dx, dbase, da, db, None, None, None, None

    _once = staticmethod(torch.autograd.function.once_differentiable(_gradients.__func__))


class AdaptedLinear(Linear):
    """A projection with the adapters of many requests: ``forward(x)`` is the projection's,
    ``forward(x, rows)`` adds each row's adapter.  The projection's weight stays frozen (its input
    gradient is its own); the adapters train where they were made trainable."""

    def __init__(self, base: Linear, adapters: LowRankAdapters) -> None:
        nn.Module.__init__(self)
        self.base = base
        self.adapters = adapters

    def forward(self, x: torch.Tensor, rows: Optional[AdapterRows] = None,
                seed: Optional[torch.Tensor] = None) -> torch.Tensor:
        y = self.base(x)
        if rows is None:
            return y
        bank = self.adapters
        if torch.is_grad_enabled() and (y.requires_grad or x.requires_grad or bank.a.requires_grad or bank.b.requires_grad):
            return bank(x, y, rows, seed)
        return bank(x, y, rows, seed, output=y if self._own(y) else None)

    def _own(self, y: torch.Tensor) -> bool:
        """Whether the projection's output is this call's alone, so that the sum may take its place: these
        projections return new memory; of any other, of a hook that saw the output and of a ``forward``
        put in its place nobody knows."""
        base = self.base
        return type(base) in (QuantLinear, MarlinQuantLinear) and not base._forward_hooks and \
            not _modules._global_forward_hooks and "forward" not in base.__dict__ and \
            y.is_contiguous() and y.data_ptr() % 16 == 0


class CounterDropout(nn.Module):
    """Dropout whose mask comes from a counter: element (row, column) of x [..., columns] is zero
    with probability p (in steps of 2^-16), by its 16 bits of Philox 4x32 under the seed; the
    others are scaled to keep the mean.  Nothing but the seed is kept for the backward pass."""

    def __init__(self, p: float) -> None:
        super().__init__()
        self.p = p

    @property
    def p(self) -> float:
        return self._p

    @p.setter
    def p(self, p: float) -> None:
        self._p, self._dropped = p, _drop(p)

    def forward(self, x: torch.Tensor, seed: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``seed``: int64 [2] on the device, seed and offset; another step takes another offset.
        In evaluation mode, or with p 0, x itself."""
        if x.dtype not in _DTYPES:
            raise TypeError("dropout runs on fp16 or bf16")
        if x.dim() < 1 or x.shape[-1] > 1 << 30 or x.numel() >= x.shape[-1] << 31 > 0:
            raise ValueError("x must have columns, up to 2^30, and fewer than 2^31 rows of them")
        if not self.training or self._dropped == 0:
            return x
        return _Dropout.apply(x, _seed(seed, x.device), self._dropped)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def _run(x, seed, drop):
        device = x.device
        if not _lib.is_current(device):
            with torch.cuda.device(device):
                return _Dropout._run(x, seed, drop)
        cols = x.shape[-1]
        rows = x.numel() // cols if cols else 0
        x2 = x if x.dim() == 2 else x.reshape(rows, cols)
        ldx = cols
        if not x2.is_contiguous():
            if x2.stride(1) != 1 or x2.stride(0) < cols:
                x2 = x2.contiguous()
            else:
                ldx = x2.stride(0)
        y = torch.empty_like(x, memory_format=torch.contiguous_format)
        _lib.call("dw4_dropout", _DTYPES[x.dtype], rows, cols, x2.data_ptr(), ldx, y.data_ptr(), cols, drop,
                  seed.data_ptr(), _lib.current_stream(device.index))
        return y

    @staticmethod
    def forward(ctx, x, seed, drop):
        ctx.drop = drop
        ctx.save_for_backward(seed)
        return _Dropout._run(x, seed, drop)

    @staticmethod
    def backward(ctx, dy):
        return _Dropout._once(ctx, dy) if torch.is_grad_enabled() else _Dropout._gradient(ctx, dy)

    @staticmethod
    def _gradient(ctx, dy):
        (seed,) = ctx.saved_tensors
        return _Dropout._run(dy, seed, ctx.drop), None, None

    _once = staticmethod(torch.autograd.function.once_differentiable(_gradient.__func__))
