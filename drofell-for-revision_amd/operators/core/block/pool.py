"""The pool of a stage's cache blocks, kept on the device.

Stands beside ``LayerBlocksHolder`` (``real.py``), which holds one layer's blocks:
a pool spans the layers of a stage, which share block numbers, and gives blocks
to the rows of a running batch (``extend``), lets rows continue other rows
(``fork``: beam steps, parallel samples, shared prompts), takes blocks back
(``free``: finished rows, blocks behind an attention window), copies them
(``copy``), moves the live ones together (``compact``) and says which slots new tokens go
to (``slots``).  No counterpart in the
reference, whose block tables live on the host.

A ``BlockState`` is never changed in place: each call returns the next one, on
the current stream, without waiting for the host, so that a serving loop can be
captured into a graph.  Blocks are handed out from the lowest free number up, in
the order of rows.  Where too few are free, ``shortage`` of the returned state
(int32, on the device) says how many are missing, the state is otherwise the one
given, and nothing is copied.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from hip_extends import _lib

from ... import flags
from .common import int32
from .real import LayerBlocksHolder


class BlockState(NamedTuple):
    block_tables: torch.Tensor  # int32 [rows, blocks per row], -1: none
    context_lens: torch.Tensor  # int32 [rows]
    refs: torch.Tensor          # int32 [blocks of the pool]: table entries that hold each
    shortage: Optional[torch.Tensor] = None  # int32 [1]: blocks missing in the call that gave this state


class SlotMap(NamedTuple):
    """Where the rows' new tokens go (all on the device, token by token, row after row)."""
    query_starts: torch.Tensor  # int32 [rows + 1]: each row's first token
    positions: torch.Tensor     # int32 [tokens]: its position in the row
    slots: torch.Tensor         # int64 [tokens]: its cache slot, -1: none
    rows: torch.Tensor          # int32 [tokens]: its row, -1 behind the last token
    excess: torch.Tensor        # int32 [1]: tokens that the arrays had no room for


class BlockPool:
    def __init__(self, layers: Sequence[LayerBlocksHolder], num_blocks: Optional[int] = None,
                 device: Optional[torch.device] = None) -> None:
        """``layers``: the stage's caches, equally many blocks of one geometry each; none
        for tables and counts alone (then with ``num_blocks`` and ``device``)."""
        self.layers = list(layers)
        if self.layers:
            first = self.layers[0]
            device, blocks = first.device, first.layer_key_ptr_table_device.numel()
            if num_blocks is not None and num_blocks != blocks:
                raise ValueError(f"the layers hold {blocks} blocks, not {num_blocks}")
            num_blocks = blocks
            for layer in self.layers:
                if layer.layer_key_ptr_table_device.numel() != num_blocks or \
                        layer.layer_val_ptr_table_device.numel() != num_blocks:
                    raise ValueError("the layers of a pool hold equally many blocks")
                if layer.device != device:
                    raise ValueError("the layers of a pool are on one device")
                if layer.block_info.bytes_per_block != first.block_info.bytes_per_block:
                    raise ValueError("the layers of a pool have blocks of one size")
                if any(p % 16 for p in layer.layer_key_ptr_table_list + layer.layer_val_ptr_table_list):
                    raise ValueError("blocks must be 16-byte aligned")
            self.part_bytes = first.block_info.bytes_per_block
        elif num_blocks is None or device is None or num_blocks < 0:
            raise ValueError("a pool without layers needs a number of blocks and a device")
        else:
            self.part_bytes = 0
        self.num_blocks = int(num_blocks)
        if torch.device(device).type != "cuda":
            raise ValueError("a block pool lives on a HIP device")
        with torch.cuda.device(device):
            self.device = torch.device("cuda", torch.cuda.current_device())
            self._key_tables, self._value_tables = (
                torch.tensor([t.data_ptr() for t in ts], dtype=torch.int64).to(self.device)
                for ts in ([x.layer_key_ptr_table_device for x in self.layers],
                           [x.layer_val_ptr_table_device for x in self.layers]))

    # ---- states
    def new_state(self, rows: int, blocks_per_row: int) -> BlockState:
        """Rows without tokens, every block free."""
        return BlockState(
            torch.full((rows, blocks_per_row), -1, dtype=torch.int32, device=self.device),
            torch.zeros(rows, dtype=torch.int32, device=self.device),
            torch.zeros(self.num_blocks, dtype=torch.int32, device=self.device))

    def _check(self, state: BlockState) -> Tuple[int, int]:
        tables, lens, refs = state[:3]
        if tables.dim() != 2:
            raise ValueError("block_tables must be [rows, blocks per row]")
        rows, width = tables.shape
        if lens.shape != (rows,) or refs.shape != (self.num_blocks,):
            raise ValueError(f"context_lens must be [{rows}] and refs [{self.num_blocks}]")
        for t in (tables, lens, refs):
            if t.dtype != torch.int32 or t.device != self.device or not t.is_contiguous():
                raise ValueError(f"a block state is contiguous int32 on {self.device}")
        return rows, width

    def _by_row(self, x: torch.Tensor, rows: int, name: str) -> torch.Tensor:
        if x.shape != (rows,) or x.device != self.device:
            raise ValueError(f"{name} must be one integer per row on {self.device}")
        return int32(x, name)

    def _next(self, state: BlockState) -> BlockState:
        return BlockState(torch.empty_like(state.block_tables), torch.empty_like(state.context_lens),
                          torch.empty_like(state.refs),
                          torch.empty(1, dtype=torch.int32, device=self.device))

    @staticmethod
    def _pointers(state: BlockState, new: BlockState, *between: Optional[torch.Tensor]):
        return (state.block_tables.data_ptr(), state.context_lens.data_ptr(), state.refs.data_ptr(),
                *(None if t is None else t.data_ptr() for t in between),
                new.block_tables.data_ptr(), new.context_lens.data_ptr(), new.refs.data_ptr(),
                new.shortage.data_ptr())

    def _layer_args(self):
        return len(self.layers), self._key_tables.data_ptr(), self._value_tables.data_ptr()

    def _workspace(self, rows: int) -> torch.Tensor:
        return torch.empty(_lib.blocks_workspace_size(rows, self.num_blocks), dtype=torch.uint8,
                           device=self.device)

    def _call(self, fn: str, *args) -> None:
        """On the pool's device, on its current stream."""
        index = self.device.index
        if _lib.current_device() == index:
            _lib.call(fn, *args, _lib.current_stream(index))
        else:
            with torch.cuda.device(index):
                _lib.call(fn, *args, _lib.current_stream(index))

    # ---- operators
    def copy(self, pairs: torch.Tensor) -> None:
        """Block pairs[i, 0] copied to pairs[i, 1] in every layer (int32 [n, 2]; a pair with
        a number outside the pool is skipped).  No block may be written twice, or written
        and read."""
        if pairs.dim() != 2 or pairs.shape[1] != 2 or pairs.device != self.device:
            raise ValueError(f"pairs must be integers [n, 2] on {self.device}")
        p = int32(pairs, "pairs")
        n, kt, vt = self._layer_args()
        self._call("dw4_copy_blocks", n, kt, vt, self.num_blocks, self.part_bytes, p.shape[0],
                   p.data_ptr())

    def extend(self, state: BlockState, add: torch.Tensor) -> BlockState:
        """Rows longer by ``add`` tokens (integers [rows], below 0 as 0), with the blocks that
        takes.  A row longer than its table counts the blocks beyond as missing."""
        rows, width = self._check(state)
        n, new, ws = self._by_row(add, rows, "add"), self._next(state), self._workspace(rows)
        self._call("dw4_extend_blocks", rows, width, self.num_blocks, flags.BLOCK_SIZE,
                   *self._pointers(state, new, n), ws.data_ptr(), ws.numel())
        return new

    def slots(self, state: BlockState, new_tokens: torch.Tensor, tokens: int) -> SlotMap:
        """Query starts, positions and cache slots of each row's last ``new_tokens`` tokens
        (integers [rows], counted in ``context_lens`` already: those that ``extend`` has added),
        in arrays of ``tokens`` entries, which the host knows to be enough.  What
        ``WindowAttention.prefill``, ``RotaryEmbedding.forward_cached`` and
        ``kv_tensor_to_slots_with_convert`` take.  Entries behind the last token have position 0,
        slot -1 and row -1.  Where the rows have more tokens, ``excess`` says how many and none is
        mapped.  Up to 8192 rows."""
        rows, width = self._check(state)
        n, tokens = self._by_row(new_tokens, rows, "new_tokens"), int(tokens)
        if not 0 <= tokens <= 1 << 28:
            raise ValueError("tokens lies between 0 and 2^28")
        ints = n.new_empty(rows + 2 + 2 * tokens)
        excess, starts, positions, row_of = torch.split_with_sizes(ints, (1, rows + 1, tokens, tokens))
        slots = n.new_empty(tokens, dtype=torch.int64)
        self._call("dw4_token_slots", rows, width, self.num_blocks, flags.BLOCK_SIZE,
                   state.block_tables.data_ptr(), state.context_lens.data_ptr(), n.data_ptr(), tokens,
                   starts.data_ptr(), positions.data_ptr(), slots.data_ptr(), row_of.data_ptr(),
                   excess.data_ptr())
        return SlotMap(starts, positions, slots, row_of, excess)

    def fork(self, state: BlockState, parents: torch.Tensor) -> BlockState:
        """Row r continues row parents[r] (integers [rows]; outside the rows: it ends).  Full
        blocks are shared; a half-filled last block stays with the first row that
        continues its row, if nothing else holds it, and is copied for the others, in every
        layer, so that each row may write the slots that follow its tokens.  Up to 8192 rows."""
        rows, width = self._check(state)
        p, new, ws = self._by_row(parents, rows, "parents"), self._next(state), self._workspace(rows)
        self._call("dw4_fork_blocks", *self._layer_args(), self.part_bytes, rows, width,
                   self.num_blocks, flags.BLOCK_SIZE, *self._pointers(state, new, p), ws.data_ptr(),
                   ws.numel())
        return new

    def free(self, state: BlockState, window: Optional[int] = None, sinks: int = 0,
             finished: Optional[torch.Tensor] = None) -> BlockState:
        """Blocks given back: those of the rows marked ``finished`` (bool [rows]), and with a
        ``window`` those that no later token sees (``WindowAttention``'s rule, with its
        sinks)."""
        rows, width = self._check(state)
        if (window is not None and window < 1) or sinks < 0:
            raise ValueError("window must be at least 1, or None, and sinks not negative")
        if finished is not None:
            if finished.dtype != torch.bool or finished.shape != (rows,) or finished.device != self.device:
                raise ValueError(f"finished must be one bool per row on {self.device}")
            finished = finished.contiguous()
        new = self._next(state)
        tables, lens, refs, *rest = self._pointers(state, new, finished)
        self._call("dw4_free_blocks", rows, width, self.num_blocks, flags.BLOCK_SIZE, tables, lens,
                   refs, rest[0], min(window or 0, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1), *rest[1:])
        return new

    def compact(self, state: BlockState, held: Optional[torch.Tensor] = None):
        """The live blocks moved, in every layer, into the numbers below their count, which
        is returned too (int32 [1], on the device): the blocks from there on are free, and
        their memory may go elsewhere.  Blocks that ``refs`` counts for a holder outside the
        tables (a cache of prefixes) move like any other: ``held`` gives their numbers (integers
        of any shape), and the numbers they have now (int32) are the third result."""
        rows, width = self._check(state)
        extra = 0
        if held is not None:
            if held.device != self.device:
                raise ValueError(f"held must be integers on {self.device}")
            # as rows of the tables, without tokens
            wide = max(width, 1)
            extra = -(-held.numel() // wide)
            tables = torch.full((rows + extra, wide), -1, dtype=torch.int32, device=self.device)
            tables[:rows, :width] = state.block_tables
            tables[rows:].view(-1)[:held.numel()] = int32(held, "held").reshape(-1)
            lens = torch.cat([state.context_lens, state.context_lens.new_zeros(extra)])
            state = BlockState(tables, lens, state.refs)
        new, ws = self._next(state), self._workspace(rows + extra)
        live = torch.empty(1, dtype=torch.int32, device=self.device)
        self._call("dw4_compact_blocks", *self._layer_args(), self.part_bytes, *state.block_tables.shape,
                   self.num_blocks, *self._pointers(state, new), live.data_ptr(), ws.data_ptr(),
                   ws.numel())
        if held is None:
            return new, live
        now = new.block_tables[rows:].reshape(-1)[:held.numel()].view(held.shape)
        return new._replace(block_tables=new.block_tables[:rows, :width].contiguous(),
                            context_lens=new.context_lens[:rows]), live, now
