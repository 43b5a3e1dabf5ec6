"""CPU tests: the windowed attention and the block pool refuse malformed calls before
anything reaches a device (fake addresses are never dereferenced), and the
oracles agree with independent restatements."""
from __future__ import annotations

import ctypes

import pytest
import torch

from hip_extends import _lib
from operators.core.attention.common import AttentionConfig
from operators.core.attention.real_page import PagedAttention
from operators.core.attention.real_window import WindowAttention
from operators.core.block.common import BlockInfo, int32
from operators.core.block.pool import BlockPool
from operators.core.block.real import LayerBlocksHolder
from oracle import blocks as B
from oracle import window as O

FAKE, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
OK, BAD, UNSUP, MISAL, WORK = (_lib.DW4_OK, _lib.DW4_ERR_INVALID_ARG, _lib.DW4_ERR_UNSUPPORTED,
                               _lib.DW4_ERR_MISALIGNED, _lib.DW4_ERR_WORKSPACE)


def paged(dtype=0, seqs=4, heads=8, kvh=2, hd=128, bs=16, nb=10, q=FAKE, qs=1024, o=FAKE, os=1024, starts=FAKE,
          rows=9, most=5, kp=FAKE, hstride=2048, scale=0.1, window=7, sinks=2, tab=FAKE, width=64, lens=FAKE, ctx=1000,
          ws=FAKE, wsb=0):
    return _lib.load().dw4_window_attention(dtype, seqs, heads, kvh, hd, bs, nb, q, qs, o, os, starts, rows, most, kp, kp,
                                            hstride, scale, window, sinks, tab, width, lens, ctx, ws, wsb, None)


def test_window_attention_refusals():
    assert paged(dtype=2) == UNSUP
    assert paged(hd=72) == UNSUP and paged(bs=8) == UNSUP and paged(heads=9) == UNSUP
    assert paged(seqs=-1) == BAD and paged(rows=-1) == BAD and paged(most=-1) == BAD and paged(window=-1) == BAD
    assert paged(sinks=-1) == BAD and paged(kvh=0) == BAD and paged(nb=-1) == BAD
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert paged(scale=scale) == BAD
    assert paged(q=None) == BAD and paged(o=None) == BAD and paged(kp=None) == BAD and paged(tab=None) == BAD
    assert paged(lens=None) == BAD
    assert paged(starts=None) == BAD                          # one row per sequence only
    assert paged(qs=1016) == BAD and paged(os=1016) == BAD and paged(hstride=2040) == BAD
    assert paged(ctx=64 * 16 + 1) == BAD                      # a table shorter than the context
    assert paged(width=1 << 30) == BAD                        # positions beyond 30 bits
    assert paged(q=ODD) == MISAL and paged(o=ODD) == MISAL and paged(qs=1028) == MISAL
    assert paged(window=0, ws=None) == WORK                   # split over the context
    assert paged(rows=1 << 24, heads=64, kvh=64) == UNSUP     # rows counted in 32 bits
    for empty in (dict(seqs=0), dict(rows=0), dict(most=0)):
        assert paged(**empty) == OK
    out = ctypes.c_size_t(7)
    size = _lib.load().dw4_window_attention_workspace_size
    assert size(4, 8, 2, 128, 16, 9, 5, 7, 2, 1000, None) == BAD
    assert size(4, 8, 2, 128, 8, 9, 5, 7, 2, 1000, ctypes.byref(out)) == UNSUP
    assert size(0, 8, 2, 128, 16, 0, 5, 7, 2, 1000, ctypes.byref(out)) == OK and out.value == 0


def test_window_attention_without_blocks_or_columns():
    """No address is asked for what has no entries (the calls go on to the next refusal)."""
    assert paged(tab=None, width=0, ctx=0, window=0, o=ODD) == MISAL
    assert paged(kp=None, nb=0, o=ODD) == MISAL
    assert paged(tab=None, width=0, ctx=1) == BAD


def test_wide_bounds_are_taken():
    """Lengths bounded by more than there are rows: the limits count the rows (the calls go on to the
    next refusal)."""
    assert paged(most=1 << 30, o=ODD) == MISAL
    assert paged(seqs=1000, rows=5000, most=1 << 20, o=ODD) == MISAL
    assert dense(most=2 ** 31 - 1, q=ODD) == MISAL
    assert dense(back=True, most=2 ** 31 - 1, q=ODD) == MISAL
    assert paged(seqs=1 << 26, rows=1 << 20, most=9) == UNSUP  # (sequence, kv head) pairs in 32 bits


def dense(back=False, dtype=1, seqs=2, heads=8, kvh=4, hd=64, q=FAKE, qs=512, k=FAKE, ks=256, o=FAKE, starts=FAKE, rows=100,
          most=60, scale=0.1, window=0, sinks=0, lse=FAKE, rest=FAKE, do=FAKE, dk=FAKE, dks=256, ws=FAKE, wsb=1 << 20):
    lib = _lib.load()
    if not back:
        return lib.dw4_window_attention_dense(dtype, seqs, heads, kvh, hd, q, qs, k, ks, k, ks, o, 512, lse, rest, starts, rows,
                                              most, scale, window, sinks, None)
    return lib.dw4_window_attention_dense_backward(dtype, seqs, heads, kvh, hd, q, qs, k, ks, k, ks, o, 512, lse, rest, do, 512,
                                                   FAKE, 512, dk, dks, FAKE, 256, starts, rows, most, scale, window, sinks,
                                                   ws, wsb, None)


@pytest.mark.parametrize("back", [False, True])
def test_dense_refusals(back):
    def call(**kw):
        return dense(back, **kw)

    assert call(dtype=-1) == UNSUP and call(hd=48) == UNSUP and call(heads=10, kvh=4) == UNSUP
    assert call(q=None) == BAD and call(k=None) == BAD and call(o=None) == BAD and call(starts=None) == BAD
    assert call(qs=511) == BAD and call(ks=255) == BAD and call(scale=-0.5) == BAD and call(window=-2) == BAD
    assert call(q=ODD) == MISAL and call(k=ODD) == MISAL and call(qs=516) == MISAL and call(ks=260) == MISAL
    for empty in (dict(seqs=0), dict(rows=0), dict(most=0)):
        assert call(**empty) == OK
    assert call(rest=None) == BAD and call(rest=ODD) == MISAL
    if back:
        assert call(lse=None) == BAD and call(do=None) == BAD and call(dk=None) == BAD and call(dks=128) == BAD
        assert call(dk=ODD) == MISAL and call(dks=260) == MISAL
        assert call(ws=None) == WORK and call(wsb=100) == WORK and call(ws=ODD) == MISAL


def test_split_outputs_are_aligned():
    """An odd number of (row, head, part) slots: their maxima and sums, 8 bytes each, are
    followed by 8 bytes more, so that the outputs behind them start at 16-byte units."""
    def size(rows, heads):
        return _lib.window_attention_workspace_size(1, heads, heads, 128, 32, rows, rows, 0, 0, 540)

    slots = 41 * 5 * 3          # 540 tokens in nine steps of 64: three parts
    assert size(41, 5) == slots * 4 * 128 + slots * 8 + 8
    assert size(42, 5) == 42 * 5 * 3 * (4 * 128 + 8)


@pytest.mark.parametrize("seqs,heads,kvh,hd,rows,most,window,sinks", [
    (2, 32, 32, 128, 12000, 6000, 1024, 4), (1, 32, 32, 128, 32768, 32768, 4096, 4), (4, 32, 32, 128, 65536, 16384, 1024, 4),
    (1, 32, 32, 128, 16384, 16384, 128, 4096), (1, 32, 32, 128, 32768, 32768, 256, 1024),
    (64, 64, 8, 128, 65536, 8192, 1024, 4), (1000, 8, 8, 128, 100000, 50000, 1024, 4)])
def test_gradient_workspace_holds_parts_alone(seqs, heads, kvh, hd, rows, most, window, sinks):
    """Where only the sinks' tiles are cut, only their parts take room: a fraction of dk and dv."""
    size = _lib.window_attention_backward_workspace_size(seqs, heads, kvh, hd, rows, most, window, sinks)
    assert size - 4 * rows * heads <= 2 * 2 * rows * kvh * hd / 2


def test_pool_refusals():
    lib = _lib.load()
    out = [ctypes.c_void_p((1 << 20) + 4096 * i) for i in range(1, 9)]

    def extend(rows=4, width=8, blocks=50, bs=16, tab=FAKE, add=FAKE, t2=out[0], short=out[3], ws=out[4], wsb=1 << 16):
        return lib.dw4_extend_blocks(rows, width, blocks, bs, tab, FAKE, FAKE, add, t2, out[1], out[2], short, ws, wsb, None)

    assert extend(rows=-1) == BAD and extend(width=-1) == BAD and extend(blocks=-1) == BAD and extend(bs=24) == UNSUP
    assert extend(tab=None) == BAD and extend(add=None) == BAD and extend(t2=FAKE) == BAD and extend(short=None) == BAD
    assert extend(ws=None) == WORK and extend(wsb=64) == WORK and extend(ws=ODD) == MISAL
    assert extend(blocks=1 << 29) == UNSUP

    def fork(layers=2, kt=FAKE, part=4096, rows=4, parents=FAKE, bs=32):
        return lib.dw4_fork_blocks(layers, kt, kt, part, rows, 8, 50, bs, FAKE, FAKE, FAKE, parents, out[0], out[1], out[2],
                                   out[3], out[4], 1 << 20, None)

    assert fork(layers=-1) == BAD and fork(kt=None) == BAD and fork(part=0) == BAD and fork(part=4100) == MISAL
    assert fork(parents=None) == BAD and fork(rows=9000) == UNSUP and fork(bs=20) == UNSUP

    def free(window=5, sinks=0, bs=16, t2=out[0]):
        return lib.dw4_free_blocks(4, 8, 50, bs, FAKE, FAKE, FAKE, None, window, sinks, t2, out[1], out[2], out[3], None)

    assert free(window=-1) == BAD and free(sinks=-1) == BAD and free(bs=0) == UNSUP and free(t2=None) == BAD

    def compact(live=out[5], part=64):
        return lib.dw4_compact_blocks(1, FAKE, FAKE, part, 4, 8, 50, FAKE, FAKE, FAKE, out[0], out[1], out[2], out[3], live,
                                      out[4], 1 << 16, None)

    assert compact(live=None) == BAD and compact(part=-16) == BAD

    def copy(layers=1, count=3, pairs=FAKE, part=64):
        return lib.dw4_copy_blocks(layers, FAKE, FAKE, 50, part, count, pairs, None)

    assert copy(count=-1) == BAD and copy(pairs=None) == BAD and copy(part=8) == MISAL
    assert copy(count=0) == OK and copy(layers=0) == OK
    size = ctypes.c_size_t(0)
    assert lib.dw4_blocks_workspace_size(-1, 4, ctypes.byref(size)) == BAD
    assert lib.dw4_blocks_workspace_size(4, 4, None) == BAD


def test_python_refusals():
    cfg = AttentionConfig(512, 64, 8, 2, 4)
    for bad in (dict(window=0), dict(window=-3), dict(sinks=-1)):
        with pytest.raises(ValueError):
            WindowAttention(cfg, **bad)
    att = WindowAttention(cfg, 5, 1)
    info = BlockInfo(head_dim=64, num_key_value_heads=2)
    holder = LayerBlocksHolder.create_contigious_cacher(info, 4, torch.device("cpu"))
    lens, tab = torch.ones(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    q = torch.zeros(3, 8, 64, dtype=torch.float16)
    with pytest.raises(AssertionError):
        att.forward(q[:, :4], 1, lens, tab, holder)                      # heads
    with pytest.raises(TypeError):
        att.forward(q.float(), 1, lens, tab, holder)
    with pytest.raises(TypeError):
        att.forward(q.bfloat16(), 1, lens, tab, holder)                  # over an fp16 cache
    with pytest.raises(ValueError):
        att.forward(q, 1, lens[:2], tab, holder)
    with pytest.raises(ValueError):
        att.forward(q, 1, lens.float(), tab, holder)
    with pytest.raises(ValueError):
        att.forward(q, 1, lens, tab[:2], holder)
    with pytest.raises(ValueError):
        att.forward(q, 1, lens, tab, holder, output=q[:2])
    with pytest.raises(ValueError):
        att.forward(q, 1, lens, tab, holder)                             # not on a HIP device
    with pytest.raises(AssertionError):
        other = BlockInfo(head_dim=64, num_key_value_heads=4)
        att.forward(q, 1, lens, tab, LayerBlocksHolder.create_contigious_cacher(other, 4, torch.device("cpu")))
    kv = torch.zeros(3, 2, 64, dtype=torch.float16)
    starts = torch.tensor([0, 3], dtype=torch.int32)
    with pytest.raises(AssertionError):
        att.dense(q, kv[:2], kv, starts, 3)
    with pytest.raises(TypeError):
        att.dense(q, kv.bfloat16(), kv, starts, 3)
    with pytest.raises(ValueError):
        att.dense(q, kv, kv, starts[:0], 3)
    with pytest.raises(ValueError):
        BlockPool([holder])                                              # not on a HIP device
    with pytest.raises(ValueError):
        BlockPool([])
    with pytest.raises(ValueError):
        BlockPool([holder], num_blocks=5)
    with pytest.raises(TypeError):                                       # rows of another type than the cache's
        holder.kv_tensor_to_slots_with_convert(kv.bfloat16(), kv.bfloat16(), torch.arange(3))


def test_bf16_caches_are_refused_where_fp16_is_read():
    info = BlockInfo(head_dim=64, num_key_value_heads=2, dtype=torch.bfloat16)
    holder = LayerBlocksHolder.create_contigious_cacher(info, 4, torch.device("cpu"), torch.bfloat16)
    q = torch.zeros(3, 8, 64, dtype=torch.float16)
    kv = torch.zeros(3, 2, 64, dtype=torch.float16)
    one = torch.ones(3, dtype=torch.int32)
    with pytest.raises(TypeError):
        PagedAttention(AttentionConfig(512, 64, 8, 2, 4)).forward(q, 1, one, torch.zeros(3, 1, dtype=torch.int32), holder)
    with pytest.raises(TypeError):
        holder.rope_and_cache(q, kv, kv, torch.zeros(4, 64), torch.zeros(4, 64), one, torch.zeros(3, 1, dtype=torch.int32))
    with pytest.raises(TypeError):
        holder.kv_tensor_to_slots_with_convert(kv, kv, torch.arange(3))
    with pytest.raises(TypeError):
        WindowAttention(AttentionConfig(512, 64, 8, 2, 4)).forward(q, 1, one, torch.zeros(3, 1, dtype=torch.int32), holder)


def test_cache_type_is_the_backings_or_the_stated_one():
    """A geometry given with bf16 alone says no more than its size: such holders take fp16 rows,
    as before there were bf16 caches; bf16 is what the backing holds or the caller states."""
    info, cpu = BlockInfo(head_dim=64, num_key_value_heads=2, dtype=torch.bfloat16), torch.device("cpu")
    made = LayerBlocksHolder.create_contigious_cacher(info, 4, cpu)
    assert made.dtype == torch.float16 == made.contigious_kv_tenosr[0].dtype
    assert LayerBlocksHolder.create_contigious_cacher(info, 4, cpu, torch.bfloat16).dtype == torch.bfloat16
    none, tables = torch.zeros(4, dtype=torch.int64), [0] * 4
    args = (info, none, none, none, none, tables, tables)
    assert LayerBlocksHolder(*args).dtype == torch.float16
    assert LayerBlocksHolder(*args, dtype=torch.bfloat16).dtype == torch.bfloat16
    with pytest.raises(TypeError):
        LayerBlocksHolder(*args, dtype=torch.float32)
    with pytest.raises(TypeError):
        LayerBlocksHolder(*args, made.contigious_kv_tenosr, dtype=torch.bfloat16)
    q, kv = torch.zeros(0, 8, 64, dtype=torch.float16), torch.zeros(0, 2, 64, dtype=torch.float16)
    for holder in (made, LayerBlocksHolder(*args)):
        with pytest.raises(TypeError):
            holder.kv_tensor_to_slots_with_convert(kv.bfloat16(), kv.bfloat16(), torch.arange(0))
        with pytest.raises(TypeError):
            WindowAttention(AttentionConfig(512, 64, 8, 2, 4)).forward(q.bfloat16(), 1, none[:0], none[:0, None], holder)


def test_caches_of_one_byte_are_refused():
    """Their blocks are half as long as what 16-bit rows take: reading or writing them would
    leave the memory."""
    info = BlockInfo(head_dim=64, num_key_value_heads=2, dtype=torch.float8_e4m3fn)
    holder = LayerBlocksHolder.create_contigious_cacher(info, 4, torch.device("cpu"), torch.float8_e4m3fn)
    bare = LayerBlocksHolder(info, *[getattr(holder, f"layer_{x}_ptr_table_{y}") for y in ("device", "cpu", "list")
                                     for x in ("key", "val")])
    cfg, tab, one = AttentionConfig(512, 64, 8, 2, 4), torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    for h in (holder, bare):
        assert h.dtype == torch.float8_e4m3fn
        with pytest.raises(TypeError):
            h.kv_tensor_from_slots_with_convert_with_create(torch.arange(3))
        for dtype in (torch.float16, torch.bfloat16, torch.float8_e4m3fn):
            q, kv = torch.zeros(3, 8, 64, dtype=dtype), torch.zeros(3, 2, 64, dtype=dtype)
            for call in (lambda: h.kv_tensor_to_slots_with_convert(kv, kv, torch.arange(3)),
                         lambda: h.kv_tensor_from_slots_with_convert(kv, kv, torch.arange(3)),
                         lambda: h.rope_and_cache(q, kv, kv, torch.zeros(4, 64), torch.zeros(4, 64), one, tab),
                         lambda: PagedAttention(cfg).forward(q, 1, one, tab, h),
                         lambda: WindowAttention(cfg).forward(q, 1, one, tab, h)):
                with pytest.raises(TypeError):
                    call()
    with pytest.raises(TypeError):
        LayerBlocksHolder(info, *[getattr(holder, f"layer_{x}_ptr_table_{y}") for y in ("device", "cpu", "list")
                                  for x in ("key", "val")], dtype=torch.float16)


def test_integers_outside_32_bits_stay_outside_every_range():
    """Not cut to their low bits, which may name a block, a row or a length."""
    x = torch.tensor([5, -1, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 40 + 3, -2 ** 32 + 3, -2 ** 63])
    top, low = 2 ** 31 - 1, -2 ** 31
    assert int32(x, "x").tolist() == [5, -1, top, top, top, top, low, low] and int32(x, "x").dtype == torch.int32
    assert int32(x[:3].int(), "x").tolist() == [5, -1, top]
    assert int32(torch.tensor([True, False]), "x").tolist() == [1, 0]
    assert int32(torch.arange(6).view(3, 2).T.int(), "x").is_contiguous()
    for bad in (torch.float32, torch.complex64, torch.uint64):
        with pytest.raises(ValueError):
            int32(torch.zeros(3).to(bad), "x")


def test_oracle_against_a_masked_softmax():
    """oracle/window.py against torch's own softmax and autograd in float64."""
    g = torch.Generator().manual_seed(1)
    n, d, window, sinks = 23, 8, 6, 2
    q, k, v, dout = (torch.randn(n, d, generator=g, dtype=torch.float64) for _ in range(4))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    gap = torch.arange(n)[:, None] - torch.arange(n)
    hidden = (gap < 0) | ((gap >= window) & (torch.arange(n) >= sinks))
    out = torch.softmax((q @ k.T * 0.3).masked_fill(hidden, -torch.inf), 1) @ v
    grads = torch.autograd.grad(out, leaves, dout)
    i = torch.arange(n)
    vals, _, _ = O.gradients(q.detach(), k.detach(), v.detach(), dout, O.visible(i, i, window, sinks), 0.3, torch.float16)
    for a, b in zip(vals, (out.detach(), *grads)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_oracle_pool_keeps_its_counts():
    """Through random steps the counts stay those of the tables, and copies go to free blocks."""
    import random
    rng = random.Random(2)
    rows, width, n, bs = 5, 6, 40, 16
    tables, lens, refs = [[-1] * width for _ in range(rows)], [0] * rows, [0] * n
    for _ in range(200):
        step = rng.choice(["extend", "fork", "free", "compact"])
        free = {p for p in range(n) if refs[p] == 0}
        if step == "extend":
            tables, lens, refs, _ = B.extend(tables, lens, refs, [rng.randint(0, 20) for _ in lens], bs)
        elif step == "fork":
            tables, lens, refs, _, pairs = B.fork(tables, lens, refs, [rng.randint(-1, rows - 1) for _ in lens], bs)
            assert {b for _, b in pairs} <= free and len({b for _, b in pairs}) == len(pairs)
        elif step == "free":
            tables, lens, refs = B.free(tables, lens, refs, bs, rng.choice([0, 9, 40]), 3,
                                        [rng.random() < 0.2 for _ in lens])
        else:
            tables, refs, live, pairs = B.compact(tables, refs)
            assert {b for _, b in pairs} <= free and all(c > 0 for c in refs[:live]) and not any(refs[live:])
        count = [0] * n
        for t in tables:
            for e in t:
                if e >= 0:
                    count[e] += 1
        assert count == refs
