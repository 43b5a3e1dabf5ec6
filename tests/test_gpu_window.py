"""GPU parity of windowed attention (WindowAttention) against oracle/window.py
in float64, element by element within the error that the kernels' roundings
allow (derived there).

Decode and prompts over cache blocks: head sizes, block sizes, groups of 1 to
12 query heads, contexts of no, one and many tokens, sequences without new
tokens, windows of one token and longer than the context, sinks before, across
and behind the window's start, blocks given back, strided queries, outputs'
rows behind the last sequence, non-finite values in places that rows do not
see.  Packed sequences: forward and gradients, shared heads, strided and
broadcast inputs, small fp16 gradients, differences.  Captured and replayed
calls.  Every case prints its name before touching the GPU.
"""
from __future__ import annotations

import pytest
import torch

from operators import flags
from operators.core.attention.common import AttentionConfig
from operators.core.attention.real_page import PagedAttention
from operators.core.attention.real_window import WindowAttention
from operators.core.block.common import BlockInfo
from operators.core.block.real import LayerBlocksHolder
from oracle import window as O

pytestmark = pytest.mark.gpu
HEAD_SIZES = [64, 80, 96, 112, 128, 256]


def say(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


@pytest.fixture(autouse=True)
def block_size_kept():
    old = flags.BLOCK_SIZE
    yield
    flags.BLOCK_SIZE = old


def config(heads, kvh, hd):
    return AttentionConfig(heads * hd, hd, heads, kvh, heads // kvh)


def cache(dev, blocks, kvh, hd, bs, dtype, seed):
    """A layer's blocks with random keys and values, on the device and as CPU copies."""
    flags.BLOCK_SIZE = bs
    info = BlockInfo(head_dim=hd, num_key_value_heads=kvh, dtype=dtype)
    holder = LayerBlocksHolder.create_contigious_cacher(info, blocks, dev, dtype)
    g = torch.Generator().manual_seed(seed)
    kt, vt = holder.contigious_kv_tenosr
    kt.copy_(torch.randn(kt.shape, generator=g))
    vt.copy_(torch.randn(vt.shape, generator=g))
    return holder, g


def tables_of(g, ctxs, bs, blocks, extra=0):
    width = max([1] + [(c + bs - 1) // bs for c in ctxs]) + extra
    order = torch.randperm(blocks, generator=g).tolist()
    t = torch.full((len(ctxs), width), -1, dtype=torch.int32)
    for s, c in enumerate(ctxs):
        for b in range((c + bs - 1) // bs):
            t[s, b] = order.pop()
    return t


def starts_of(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


def check_paged(dev, new, ctxs, heads, kvh, hd, bs, dtype, window, sinks, gone=(), decode=False, spoil=None):
    """One call against the oracle; ``gone``: (sequence, block) entries given back."""
    blocks = sum((c + bs - 1) // bs for c in ctxs) + 3
    holder, g = cache(dev, blocks, kvh, hd, bs, dtype, 11 * len(ctxs) + hd)
    tables = tables_of(g, ctxs, bs, blocks)
    for s, b in gone:
        tables[s, b] = -1
    kt, vt = holder.contigious_kv_tenosr
    if spoil is not None:
        spoil(kt, vt, tables)
    starts = starts_of(new)
    q = torch.randn(starts[-1], heads, hd, generator=g).to(dtype)
    att = WindowAttention(config(heads, kvh, hd), window or None, sinks)
    args = (max([0] + ctxs), torch.tensor(ctxs, dtype=torch.int32, device=dev), tables.to(dev), holder)
    if decode:
        def call():
            return att.forward(q.to(dev), *args)
    else:
        def call():
            return att.prefill(q.to(dev), torch.tensor(starts, dtype=torch.int32, device=dev), max(new), *args)
    out = call()
    again = call()
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))  # deterministic
    ref, bound = O.paged(q.double(), starts, ctxs, tables, kt.cpu(), vt.cpu(), bs, window, sinks, att.scale)
    ok, worst = O.within(out, ref, bound)
    assert ok, f"worst error / bound {worst:.3f}"
    return out, att, q, args


DECODE = [
    # contexts, heads, kv heads, block size, window, sinks
    ([1, 7, 32, 20], 8, 8, 32, 0, 0),
    ([1, 16, 17, 100, 0], 8, 2, 16, 24, 4),     # an empty context
    ([300, 41, 2], 24, 2, 16, 1, 0),            # 12 query heads per kv head, a window of one token
    ([300, 41, 64], 32, 4, 32, 64, 33),         # sinks across a block's end
    ([1500, 2049, 3], 4, 4, 32, 1000, 1),       # split over the length
    ([700], 32, 8, 32, 512, 4),
    ([90, 33, 5000], 8, 1, 16, 40, 70),         # sinks reach into the window of the short ones
    ([130, 129], 80, 2, 32, 0, 3),              # 40 rows per kv head: two row tiles
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("ctxs,heads,kvh,bs,window,sinks", DECODE)
def test_decode(hip_device, ctxs, heads, kvh, bs, window, sinks, dtype):
    say(f"decode {ctxs} {heads}/{kvh} bs={bs} window={window} sinks={sinks} {dtype}")
    check_paged(hip_device, [1] * len(ctxs), ctxs, heads, kvh, 128, bs, dtype, window, sinks, decode=True)


@pytest.mark.parametrize("hd", HEAD_SIZES)
@pytest.mark.parametrize("bs", [16, 32])
def test_decode_head_sizes(hip_device, hd, bs):
    for dtype in (torch.float16, torch.bfloat16):
        say(f"decode hd={hd} bs={bs} {dtype}")
        check_paged(hip_device, [1, 1, 1], [1, 97, 700], 6, 2, hd, bs, dtype, 200, 5, decode=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("ctxs,heads,kvh,hd,bs", [([37, 5, 12, 40], 16, 2, 128, 32), ([3, 64, 20, 33], 18, 3, 80, 16),
                                                  ([9, 30, 2, 50], 16, 4, 256, 32)])
def test_decode_probabilities_in_two_parts(hip_device, ctxs, heads, kvh, hd, bs, dtype):
    """Values that cancel, so that the output's own rounding hides little: within the bound of
    probabilities kept to 2^-16, which one 16-bit part does not hold."""
    say(f"two parts {ctxs} hd={hd} bs={bs} {dtype}")
    blocks = sum((c + bs - 1) // bs for c in ctxs) + 1
    holder, g = cache(hip_device, blocks, kvh, hd, bs, dtype, hd)
    tables = tables_of(g, ctxs, bs, blocks)
    kt, vt = holder.contigious_kv_tenosr
    vt[..., 0::2], vt[..., 1::2] = 1, -1   # by token
    q = torch.randn(len(ctxs), heads, hd, generator=g).to(dtype)
    att = WindowAttention(config(heads, kvh, hd))
    out = att.forward(q.to(hip_device), max(ctxs), torch.tensor(ctxs, dtype=torch.int32, device=hip_device),
                      tables.to(hip_device), holder)
    torch.cuda.synchronize()
    ref, bound = O.paged(q.double(), range(len(ctxs) + 1), ctxs, tables, kt.cpu(), vt.cpu(), bs, 0, 0, att.scale, rounded_p=False)
    ok, worst = O.within(out, ref, bound)
    assert ok, f"worst error / bound {worst:.3f}"
    # (one part: the same from probabilities rounded to the type)
    ratios = []
    for s, ctx in enumerate(ctxs):
        k, v, _ = O.slots_to_rows(kt.cpu(), vt.cpu(), tables[s], ctx, bs)
        for h in range(heads):
            x = h // (heads // kvh)
            seen = torch.ones(1, ctx, dtype=torch.bool)
            _, _, p = O.attend(q[s:s + 1, h].double(), k[:, x].double(), v[:, x].double(), seen, att.scale)
            rough = p.to(dtype).double() @ v[:, x].double()
            ratios.append(float(((rough - ref[s, h]).abs() / bound[s, h]).max()))
    assert max(ratios) > 1


PREFILL = [
    # new tokens, contexts, heads, kv heads, block size, window, sinks
    ([7, 1, 0, 3], [100, 1, 50, 3], 8, 2, 16, 0, 0),           # few rows: the rows kernel
    ([5, 2], [9, 900], 8, 2, 32, 30, 4),
    ([64, 1, 0, 33], [64, 1, 40, 300], 8, 2, 32, 0, 0),        # the tile kernel
    ([130, 257], [130, 400], 4, 4, 16, 0, 0),
    ([130, 257], [130, 400], 4, 4, 32, 50, 3),
    ([200, 90], [333, 90], 12, 1, 32, 1, 0),                   # 12 rows per token, a window of one
    ([200], [900], 4, 2, 16, 64, 70),
    ([40], [2500], 8, 8, 32, 0, 0),                            # split over the length
    ([300, 300], [300, 1000], 2, 2, 32, 100000, 2),            # a window longer than the context
    ([70], [20], 4, 2, 32, 0, 0),                              # more new tokens than context: rows that see nothing
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("new,ctxs,heads,kvh,bs,window,sinks", PREFILL)
def test_prefill(hip_device, new, ctxs, heads, kvh, bs, window, sinks, dtype):
    say(f"prefill {new} of {ctxs} {heads}/{kvh} bs={bs} window={window} sinks={sinks} {dtype}")
    check_paged(hip_device, new, ctxs, heads, kvh, 128, bs, dtype, window, sinks)


def test_prefill_in_an_odd_number_of_slots(hip_device):
    """Odd heads, rows and parts: the parts' outputs start behind maxima and sums that do not
    fill whole 16-byte units."""
    for n, dtype in ((41, torch.float16), (1, torch.bfloat16)):
        say(f"odd heads, rows and parts, {n} new tokens")
        check_paged(hip_device, [n], [540], 5, 5, 128, 32, dtype, 0, 0)


@pytest.mark.parametrize("hd", HEAD_SIZES)
@pytest.mark.parametrize("bs", [16, 32])
def test_prefill_head_sizes(hip_device, hd, bs):
    for dtype in (torch.float16, torch.bfloat16):
        say(f"prefill hd={hd} bs={bs} {dtype}")
        check_paged(hip_device, [100, 9], [150, 300], 4, 2, hd, bs, dtype, 70, 3)


@pytest.mark.parametrize("decode", [True, False])
def test_blocks_given_back(hip_device, decode):
    """Entries of -1 behind the window are never read; one inside it hides its tokens."""
    new, ctxs = ([1, 1], [600, 400]) if decode else ([90, 40], [600, 400])
    first = [(c - n + 1 - 64) // 16 for n, c in zip(new, ctxs)]
    behind = [(s, b) for s in range(2) for b in range(1, first[s])]
    for bs, gone in ((16, behind), (16, behind + [(0, 35), (1, 24)]), (32, [(0, 17), (1, 12), (1, 11)])):
        say(f"blocks given back, decode={decode}, block {bs}, {len(gone)} gone")
        check_paged(hip_device, new, ctxs, 8, 2, 128, bs, torch.float16, 64, 4, gone=gone, decode=decode)


def test_every_visible_block_missing(hip_device):
    say("rows whose mask leaves nothing")
    for decode in (True, False):
        new = [1, 1] if decode else [40, 3]
        out, *_ = check_paged(hip_device, new, [64, 64], 4, 2, 128, 32, torch.bfloat16, 0, 0,
                              gone=[(0, 0), (0, 1)], decode=decode)
        assert not out[:new[0]].any() and out[new[0]:].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("decode", [True, False])
def test_nonfinite_in_unseen_places(hip_device, decode, dtype):
    """Slots behind the context, tokens before the window and, for the rows of a prompt
    before them, later tokens hold NaN and infinities."""
    bs, ctxs = 32, [75, 300]
    new = [1, 1] if decode else [20, 70]

    def spoil(kt, vt, tables):
        for s, c in enumerate(ctxs):
            last = int(tables[s, (c - 1) // bs])
            kt[last, :, :, c % bs:] = torch.nan
            vt[last, :, :, c % bs:] = torch.inf
        # before the window of every new token of sequence 1, behind its sinks
        t = 300 - new[1] - 40 - 3
        blk = int(tables[1, t // bs])
        kt[blk, :, :, t % bs] = torch.nan
        vt[blk, :, 0::2, t % bs] = -torch.inf
        vt[blk, :, 1::2, t % bs] = torch.nan

    say(f"non-finite values unseen, decode={decode} {dtype}")
    check_paged(hip_device, new, ctxs, 8, 2, 128, bs, dtype, 40, 4, decode=decode, spoil=spoil)


@pytest.mark.parametrize("hd,bs", [(128, 32), (80, 16), (256, 32)])
def test_nonfinite_of_later_tokens(hip_device, hd, bs):
    """A token's infinities reach the rows that see it and no others."""
    ctxs, heads, kvh = [200], 4, 2
    holder, g = cache(hip_device, 20, kvh, hd, bs, torch.float16, 5)
    tables = tables_of(g, ctxs, bs, 20)
    kt, vt = holder.contigious_kv_tenosr
    q = torch.randn(120, heads, hd, generator=g).half().to(hip_device)
    att = WindowAttention(config(heads, kvh, hd), 50, 2)
    args = (torch.tensor([0, 120], dtype=torch.int32, device=hip_device), 120, 200,
            torch.tensor(ctxs, dtype=torch.int32, device=hip_device), tables.to(hip_device), holder)
    say(f"an infinite value inside a prompt hd={hd} bs={bs}")
    clean = att.prefill(q, *args)
    blk = int(tables[0, 130 // bs])
    vt[blk, 0, 3, 130 % bs] = torch.inf
    vt[blk, 0, 5, 130 % bs] = -torch.inf
    vt[blk, 0, 7, 130 % bs] = torch.nan
    out = att.prefill(q, *args)
    torch.cuda.synchronize()
    pos = torch.arange(80, 200, device=hip_device)
    hit = (pos >= 130) & (pos < 180)
    assert torch.equal(out[~hit], clean[~hit])
    assert torch.equal(out[hit][:, 2:], clean[hit][:, 2:])          # the other kv head
    o = out[hit][:, :2]
    assert (o[..., 3] == torch.inf).all() and (o[..., 5] == -torch.inf).all() and o[..., 7].isnan().all()
    rest = [d for d in range(hd) if d not in (3, 5, 7)]
    assert torch.equal(o[..., rest], clean[hit][:, :2][..., rest])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hd,bs,token", [(128, 32, 140), (64, 16, 140), (256, 32, 140), (128, 32, 195), (80, 16, 101)])
def test_nonfinite_values_that_rows_see(hip_device, hd, bs, token, dtype):
    """Decode and a few new tokens: an infinity gives infinity, a NaN NaN, in the dims that hold
    them and nowhere else, whether every row sees the whole step of tokens (140), or some of it
    is behind the context (195) or before the window (101)."""
    holder, g = cache(hip_device, 20, 2, hd, bs, dtype, 5)
    tables = tables_of(g, [200], bs, 20)
    kt, vt = holder.contigious_kv_tenosr
    att = WindowAttention(config(4, 2, hd), 100, 2)
    lens = torch.tensor([200], dtype=torch.int32, device=hip_device)
    for n in (1, 3):
        say(f"visible non-finite values, token {token}, {n} rows, hd={hd} bs={bs} {dtype}")
        q = torch.randn(n, 4, hd, generator=g).to(dtype).to(hip_device)
        starts = torch.tensor([0, n], dtype=torch.int32, device=hip_device)

        def call():
            return att.prefill(q, starts, n, 200, lens, tables.to(hip_device), holder)

        clean = call()
        kept = vt.clone()
        blk = int(tables[0, token // bs])
        for dim, value in ((3, torch.inf), (5, -torch.inf), (7, torch.nan), (hd - 1, torch.inf)):
            vt[blk, 0, dim, token % bs] = value
        out = call()
        vt.copy_(kept)
        torch.cuda.synchronize()
        hit = torch.arange(200 - n, 200) < token + 100
        assert hit.any()
        o = out[hit][:, :2]
        assert (o[..., 3] == torch.inf).all() and (o[..., 5] == -torch.inf).all()
        assert o[..., 7].isnan().all() and (o[..., hd - 1] == torch.inf).all()
        rest = [d for d in range(hd) if d not in (3, 5, 7, hd - 1)]
        assert torch.equal(o[..., rest], clean[hit][:, :2][..., rest])
        assert torch.equal(out[:, 2:], clean[:, 2:]) and torch.equal(out[~hit], clean[~hit])


def test_rows_behind_the_last_sequence_and_strides(hip_device):
    """Queries inside a wider tensor, an output with a stride of its own, rows that
    belong to no sequence."""
    for new, ctxs in (([3, 2], [40, 77]), ([60, 45], [60, 177])):
        say(f"strides and padding rows {new}")
        holder, g = cache(hip_device, 30, 2, 128, 16, torch.bfloat16, 3)
        tables = tables_of(g, ctxs, 16, 30, extra=2)
        starts = starts_of(new)
        total = starts[-1] + 9
        wide = torch.randn(total, 8 + 4, 128, generator=g).bfloat16()
        att = WindowAttention(config(8, 2, 128), 33, 2)
        buf = torch.full((total, 10, 128), 7.0, dtype=torch.bfloat16, device=hip_device)
        q = wide.to(hip_device)[:, 2:10]
        out = att.prefill(q, torch.tensor(starts, dtype=torch.int32, device=hip_device), max(new), max(ctxs),
                          torch.tensor(ctxs, dtype=torch.int32, device=hip_device), tables.to(hip_device), holder,
                          output=buf[:, 1:9])
        torch.cuda.synchronize()
        kt, vt = holder.contigious_kv_tenosr
        ref, bound = O.paged(wide[:, 2:10].double(), starts, ctxs, tables, kt.cpu(), vt.cpu(), 16, 33, 2, att.scale)
        n = starts[-1]
        ok, worst = O.within(out[:n], ref[:n], bound[:n])
        assert ok, worst
        assert (buf[n:] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, 9] == 7).all()


def test_no_window_is_paged_attention(hip_device):
    """Without window and sinks: the results of PagedAttention, within both kernels' roundings."""
    say("no window against PagedAttention")
    ctxs = [300, 41, 129]
    out, att, q, args = check_paged(hip_device, [1] * 3, ctxs, 8, 2, 128, 32, torch.float16, 0, 0, decode=True)
    ref = PagedAttention(att.cfg).forward(q.to(hip_device), *args)
    torch.cuda.synchronize()
    assert torch.allclose(out.float(), ref.float(), rtol=2 ** -10, atol=2 ** -13)


def test_fp16_rows_of_a_geometry_given_with_bf16(hip_device):
    """A holder whose geometry says bf16 but whose blocks were not made so takes, gives back and
    attends over fp16 rows."""
    flags.BLOCK_SIZE = 16
    info = BlockInfo(head_dim=64, num_key_value_heads=2, dtype=torch.bfloat16)
    made = LayerBlocksHolder.create_contigious_cacher(info, 5, hip_device)
    k, v = made.contigious_kv_tenosr
    bare = LayerBlocksHolder(info, made.layer_key_ptr_table_device, made.layer_val_ptr_table_device,
                             made.layer_key_ptr_table_cpu, made.layer_val_ptr_table_cpu,
                             made.layer_key_ptr_table_list, made.layer_val_ptr_table_list)
    g = torch.Generator().manual_seed(3)
    rows = [torch.randn(70, 2, 64, generator=g).half().to(hip_device) for _ in range(2)]
    q = torch.randn(1, 4, 64, generator=g).half().to(hip_device)
    slots = torch.arange(70, device=hip_device)
    tables = torch.arange(5, dtype=torch.int32, device=hip_device)[None]
    lens = torch.tensor([70], dtype=torch.int32, device=hip_device)
    for holder in (made, bare):
        say(f"fp16 rows, geometry given with bf16, backing: {holder.is_contigious}")
        k.zero_(), v.zero_()
        holder.kv_tensor_to_slots_with_convert(*rows, slots)
        back = holder.kv_tensor_from_slots_with_convert_with_create(slots)
        a = PagedAttention(config(4, 2, 64)).forward(q, 70, lens, tables, holder)
        b = WindowAttention(config(4, 2, 64)).forward(q, 70, lens, tables, holder)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(back, rows))
        ref, bound = O.paged(q.cpu().double(), [0, 1], [70], tables.cpu(), k.cpu(), v.cpu(), 16, 0, 0, 64 ** -0.5)
        ok, worst = O.within(b, ref, bound)
        assert ok, worst
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -10, atol=2 ** -13)


def test_bf16_rows_come_back(hip_device):
    """Rows written to a bf16 cache and read back, bit for bit, infinities and NaN among them."""
    for hd, kvh, bs in ((128, 8, 32), (80, 3, 16), (256, 1, 32)):
        say(f"bf16 rows hd={hd} bs={bs}")
        flags.BLOCK_SIZE = bs
        info = BlockInfo(head_dim=hd, num_key_value_heads=kvh, dtype=torch.bfloat16)
        holder = LayerBlocksHolder.create_contigious_cacher(info, 9, hip_device, torch.bfloat16)
        g = torch.Generator().manual_seed(hd)
        rows = [torch.randint(-2 ** 15, 2 ** 15, (77, kvh, hd), generator=g).to(torch.int16).view(torch.bfloat16).to(hip_device)
                for _ in range(2)]
        slots = torch.randperm(9 * bs, generator=g)[:77].to(hip_device)
        holder.kv_tensor_to_slots_with_convert(*rows, slots)
        back = holder.kv_tensor_from_slots_with_convert_with_create(slots)
        torch.cuda.synchronize()
        for x, y in zip(back, rows):
            assert x.dtype == torch.bfloat16 and torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_long_position_and_large_cache_offsets(hip_device):
    """A stream far beyond its window, its early blocks given back, and blocks whose byte
    offset in the cache passes 2^32."""
    bs, kvh, hd = 32, 32, 128
    page = kvh * hd * bs * 2
    blocks = (1 << 32) // page + 40
    flags.BLOCK_SIZE = bs
    info = BlockInfo(head_dim=hd, num_key_value_heads=kvh)
    holder = LayerBlocksHolder.create_contigious_cacher(info, blocks, hip_device)
    kt, vt = holder.contigious_kv_tenosr
    g = torch.Generator().manual_seed(1)
    ctx, window = 1_000_003, 100
    tables = torch.full((1, (ctx + bs - 1) // bs), -1, dtype=torch.int32)
    used = list(range((ctx - 150) // bs, (ctx + bs - 1) // bs)) + [0]
    for i, b in enumerate(used):
        blk = blocks - 1 - 2 * i
        tables[0, b] = blk
        kt[blk] = torch.randn(kt.shape[1:], generator=g).half().to(hip_device)
        vt[blk] = torch.randn(vt.shape[1:], generator=g).half().to(hip_device)
    ids = [int(tables[0, b]) for b in used]
    small = torch.full_like(tables, -1)
    for i, b in enumerate(used):
        small[0, b] = i
    kc, vc = kt[ids].cpu(), vt[ids].cpu()
    att = WindowAttention(config(kvh, kvh, hd), window, 4)
    for n in (1, 40):
        say(f"position {ctx}, {n} new tokens")
        q = torch.randn(n, kvh, hd, generator=g).half()
        out = att.prefill(q.to(hip_device), torch.tensor([0, n], dtype=torch.int32, device=hip_device), n, ctx,
                          torch.tensor([ctx], dtype=torch.int32, device=hip_device), tables.to(hip_device), holder)
        torch.cuda.synchronize()
        # the oracle over the kept tokens alone
        keep = torch.cat([torch.arange(0, bs), torch.arange((ctx - 150) // bs * bs, ctx)])
        k, v, held = [x for x in O.slots_to_rows(kc, vc, small[0], ctx, bs)]
        seen = O.visible(torch.arange(ctx - n, ctx), keep, window, 4)
        for h in (0, 31):
            o, spread, _ = O.attend(q[:, h].double(), k[keep, h].double(), v[keep, h].double(), seen, att.scale)
            ok, worst = O.within(out[:, h], o, O.out_bound(o, spread, len(keep), torch.float16))
            assert ok, worst


TRAIN = [
    # lengths, heads, kv heads, head size, window, sinks
    ([1], 2, 2, 64, 0, 0),
    ([2, 1, 3], 4, 2, 128, 0, 0),
    ([333, 1, 40], 4, 1, 80, 50, 3),
    ([130, 200], 6, 2, 96, 1, 0),
    ([257], 2, 2, 112, 0, 0),
    ([300, 64], 4, 4, 128, 64, 40),
    ([260], 12, 1, 64, 33, 140),      # sinks over more than a tile of tokens
    ([150, 33], 2, 1, 256, 70, 2),
    ([400], 24, 2, 64, 100000, 1),
    ([2000, 30], 2, 1, 64, 40, 5),    # the sinks' rows, far beyond a window's, in parts
]


def leaves(g, lens, heads, kvh, hd, dtype, extra=0):
    n = sum(lens) + extra
    return [torch.randn(n, h, hd, generator=g).to(dtype) for h in (heads, kvh, kvh, heads)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("lens,heads,kvh,hd,window,sinks", TRAIN)
def test_dense_and_gradients(hip_device, lens, heads, kvh, hd, window, sinks, dtype):
    say(f"dense {lens} {heads}/{kvh} hd={hd} window={window} sinks={sinks} {dtype}")
    g = torch.Generator().manual_seed(sum(lens) + hd)
    extra = 5  # rows of no sequence
    q, k, v, dout = leaves(g, lens, heads, kvh, hd, dtype, extra)
    att = WindowAttention(config(heads, kvh, hd), window or None, sinks)
    starts = torch.tensor(starts_of(lens), dtype=torch.int32, device=hip_device)
    dev = [t.to(hip_device).requires_grad_(True) for t in (q, k, v)]

    def call():
        out = att.dense(*dev, starts, max(lens))
        return (out.detach(), *torch.autograd.grad(out, dev, dout.to(hip_device)))

    got, again = call(), call()
    torch.cuda.synchronize()
    for a, b in zip(got, again):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))  # deterministic
    ref, bounds = O.dense(*[t[:sum(lens)].double() for t in (q, k, v, dout)], lens, window, sinks, att.scale, dtype)
    for name, y, r, b in zip(("out", "dq", "dk", "dv"), got, ref, bounds):
        ok, worst = O.within(y[:sum(lens)], r, b)
        assert ok, f"{name}: worst error / bound {worst:.3f}"
        assert not y[sum(lens):].any()
    with torch.no_grad():
        assert torch.equal(att.dense(*dev, starts, max(lens)), got[0])


@pytest.mark.parametrize("hd", [64, 80, 128, 256])
@pytest.mark.parametrize("group", [8, 16, 32, 64])
def test_gradients_of_wide_groups(hip_device, group, hd):
    """Groups of as many heads as a step, a copy's turn or half a turn has rows, and more."""
    test_dense_and_gradients(hip_device, [140, 37], 2 * group, 2, hd, 90, 3, torch.bfloat16 if group < 32 else torch.float16)


@pytest.mark.parametrize("heads,n", [(1023, 4200), (1000, 6200)])
def test_gradients_of_far_tokens_of_wide_groups(hip_device, heads, n):
    """Groups whose rows at far tokens an inexact division by the group's size (one product
    with ceil(2^32 / heads)) counts to the next token: the last head's rows from token 4120
    on with 1023 heads, 6100 with 1000.  Only that head has an output gradient, so that its
    part of dk and dv is not lost among the others'."""
    hd, window, tail = 64, 6, 150
    say(f"{n} tokens of {heads} heads on one")
    g = torch.Generator(device=hip_device).manual_seed(heads)
    q, k, v, dout = (torch.randn(n, h, hd, generator=g, device=hip_device, dtype=torch.float16).to(torch.bfloat16)
                     for h in (heads, 1, 1, 1))
    full = torch.zeros_like(q)
    full[:, -1:] = dout
    att = WindowAttention(config(heads, 1, hd), window)
    dev = [t.requires_grad_(True) for t in (q, k, v)]
    out = att.dense(*dev, torch.tensor([0, n], dtype=torch.int32, device=hip_device), n)
    dq, dk, dv = torch.autograd.grad(out, dev, full)
    torch.cuda.synchronize()
    # the last tokens as a sequence of their own, less those whose window starts before it
    x = [t[n - tail:].detach().double().cpu() for t in (q[:, -1:], k, v, dout)]
    ref, bounds = O.dense(*x, [tail], window, 0, att.scale, torch.bfloat16)
    for name, y, r, b in zip(("out", "dq", "dk", "dv"), (out[:, -1:].detach(), dq[:, -1:], dk, dv), ref, bounds):
        ok, worst = O.within(y[n - tail + window:], r[window:], b[window:])
        assert ok, f"{name}: worst error / bound {worst:.3f}"


@pytest.mark.parametrize("lens,most,heads,kvh,hd,sinks", [([100, 30], 64, 4, 2, 128, 0), ([5, 700, 1], 1, 2, 1, 80, 2),
                                                          ([1500, 900], 1000, 20, 20, 64, 3)])
def test_rows_beyond_the_stated_length(hip_device, lens, most, heads, kvh, hd, sinks):
    """Sequences longer than the call says: their further rows are zeros, in the output and
    in every gradient, whatever the memory held; the others are those of shorter sequences."""
    say(f"{lens} tokens said to be {most}")
    g = torch.Generator().manual_seed(6)
    q, k, v, dout = leaves(g, lens, heads, kvh, hd, torch.bfloat16)
    att = WindowAttention(config(heads, kvh, hd), 40, sinks)
    starts = starts_of(lens)
    dev = [t.to(hip_device).requires_grad_(True) for t in (q, k, v)]
    spoilt = [torch.full_like(t, torch.nan, device=hip_device) for t in (q, q, k, v) for _ in range(3)]
    del spoilt  # torch gives this memory out again
    out = att.dense(*dev, torch.tensor(starts, dtype=torch.int32, device=hip_device), most)
    grads = torch.autograd.grad(out, dev, dout.to(hip_device))
    torch.cuda.synchronize()
    keep = torch.cat([torch.arange(a, min(b, a + most)) for a, b in zip(starts, starts[1:])])
    rest = torch.ones(sum(lens), dtype=torch.bool)
    rest[keep] = False
    ref, bounds = O.dense(*[t[keep].double() for t in (q, k, v, dout)], [min(n, most) for n in lens], 40, sinks,
                          att.scale, torch.bfloat16)
    for name, y, r, b in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), ref, bounds):
        assert not y.cpu()[rest].any(), name
        ok, worst = O.within(y.cpu()[keep], r, b)
        assert ok, f"{name}: worst error / bound {worst:.3f}"


def test_small_fp16_gradients(hip_device):
    """Output gradients of a mean loss, far below fp16's normal range after the product
    with the probabilities: as exact, relative to their size, as gradients of size one.  The
    scale is a power of two, so the oracle's bounds scale with it; results go out in
    fp16, whose smallest step the bounds hold."""
    lens, heads, kvh, hd = [300], 4, 2, 128
    g = torch.Generator().manual_seed(4)
    q, k, v, dout = leaves(g, lens, heads, kvh, hd, torch.float16)
    small = (dout.float() * 2.0 ** -11).half()
    att = WindowAttention(config(heads, kvh, hd), 200, 2)
    starts = torch.tensor([0, 300], dtype=torch.int32, device=hip_device)
    dev = [t.to(hip_device).requires_grad_(True) for t in (q, k, v)]
    say("small fp16 gradients")
    grads = torch.autograd.grad(att.dense(*dev, starts, 300), dev, small.to(hip_device))
    torch.cuda.synchronize()
    ref, bounds = O.dense(*[t.double() for t in (q, k, v, small)], lens, 200, 2, att.scale, torch.float16)
    for name, y, r, b in zip(("dq", "dk", "dv"), grads, ref[1:], bounds[1:]):
        ok, worst = O.within(y, r, b)
        assert ok, f"{name}: {worst:.3f}"


@pytest.mark.parametrize("lens,heads,kvh,hd,window,sinks", [
    ([2000, 40], 20, 20, 64, 40, 140),   # sink tiles in parts, the others whole
    ([1500], 6, 3, 128, 30, 200),        # both in parts, of different numbers
])
def test_gradients_of_cut_sink_tiles(hip_device, lens, heads, kvh, hd, window, sinks):
    test_dense_and_gradients(hip_device, lens, heads, kvh, hd, window, sinks, torch.bfloat16)


def check_gradients(dev, q, k, v, dout, lens, window, sinks):
    """dq, dk, dv of packed fp16 sequences against the oracle, element by element."""
    heads, kvh, hd = q.shape[1], k.shape[1], q.shape[2]
    att = WindowAttention(config(heads, kvh, hd), window or None, sinks)
    starts = torch.tensor(starts_of(lens), dtype=torch.int32, device=dev)
    x = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(att.dense(*x, starts, max(lens)), x, dout.to(dev))
    torch.cuda.synchronize()
    ref, bounds = O.dense(*[t.double() for t in (q, k, v, dout)], lens, window, sinks, att.scale, q.dtype)
    for name, y, r, b in zip(("dq", "dk", "dv"), grads, ref[1:], bounds[1:]):
        ok, worst = O.within(y, r, b)
        assert ok, f"{name}: worst error / bound {worst:.3f}"


@pytest.mark.parametrize("hd,kvh,lens,window", [(256, 1, [2, 40, 3], 0), (128, 2, [300, 2, 5], 70), (64, 1, [4, 700], 0)])
def test_fp16_gradients_of_large_values(hip_device, hd, kvh, lens, window):
    """Values of one size and alternating sign by token, every dim of a token alike, under output
    gradients of one: dO . V is 2^22, far beyond fp16, where dq and dk, with small keys
    and queries, are not."""
    say(f"fp16 gradients of large values, {lens} tokens, head size {hd}")
    g = torch.Generator().manual_seed(hd)
    q, k, v, dout = leaves(g, lens, 2, kvh, hd, torch.float16)
    q, k = (q.float() * 0.02).half(), (k.float() * 0.02).half()
    v[:] = min(2.0 ** 22 / hd, 65504)
    v[::2] *= -1
    check_gradients(hip_device, q, k, v, torch.ones_like(dout), lens, window, 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("lens,heads,kvh,hd,window,sinks", [([16, 40], 4, 4, 128, 0, 0), ([300], 6, 2, 64, 0, 0),
                                                            ([700, 33], 4, 4, 80, 200, 4), ([150], 10, 2, 256, 60, 0)])
def test_gradients_with_keys_of_a_common_part(hip_device, lens, heads, kvh, hd, window, sinks, dtype):
    """Keys that share a vector eight times as large as what tells them apart, as a bias makes
    them: dS sums to zero over a row's tokens, so that the shared part must not reach dq,
    and an error of delta, which every token of a row gets, must not bring it back.

    In the 2-norm over many elements: the result's own rounding is one (relative u / sqrt(3)
    of a mantissa of 1, 0.42 u on average).  Of the rest the largest is delta's error from the
    forward's 16-bit probabilities, at most u / sqrt(3) = 0.58 u of what tells the keys apart, as
    dq is: together sqrt(0.42^2 + 0.58^2) / 0.42 = 1.7.  Uncorrected it is 0.58 u times 8 beside
    0.42 u, 5 and more."""
    say(f"keys of a common part {lens} {heads}/{kvh} hd={hd} window={window} {dtype}")
    g = torch.Generator().manual_seed(hd)
    q, k, v, dout = leaves(g, lens, heads, kvh, hd, dtype)
    k = (k.float() + 8 * torch.randn(1, kvh, hd, generator=g)).to(dtype)
    att = WindowAttention(config(heads, kvh, hd), window or None, sinks)
    x = [t.to(hip_device).requires_grad_(True) for t in (q, k, v)]
    out = att.dense(*x, torch.tensor(starts_of(lens), dtype=torch.int32, device=hip_device), max(lens))
    grads = torch.autograd.grad(out, x, dout.to(hip_device))
    torch.cuda.synchronize()
    ref, bounds = O.dense(*[t.double() for t in (q, k, v, dout)], lens, window, sinks, att.scale, dtype)
    for name, y, r, b in zip(("dq", "dk", "dv"), grads, ref[1:], bounds[1:]):
        ok, worst = O.within(y, r, b)
        assert ok, f"{name}: worst error / bound {worst:.3f}"
        ratio = float((y.double().cpu() - r).norm() / (r.to(dtype).double() - r).norm())
        assert ratio < 1.7, f"{name}: {ratio:.2f} times its own rounding"


@pytest.mark.parametrize("where", ["first", "last", "middle"])
@pytest.mark.parametrize("n,window,hd,low", [(2048, 512, 128, -10), (1024, 200, 64, -12), (512, 64, 128, -10), (300, 0, 80, -12)])
def test_uneven_fp16_gradients(hip_device, n, window, hd, low, where):
    """Eight rows with output gradients of size one among rows of 2^-10 or 2^-12, as at the end of a
    masked loss: the others' gradients are as exact as without them."""
    say(f"uneven fp16 gradients {n} tokens, window {window}, 2^{low}, large ones {where}")
    g = torch.Generator().manual_seed(n + low)
    q, k, v, dout = leaves(g, [n], 2, 1, hd, torch.float16)
    at = {"first": 0, "last": n - 8, "middle": n // 2}[where]
    size = torch.full((n, 1, 1), 2.0 ** low)
    size[at:at + 8] = 1
    check_gradients(hip_device, q, k, v, (dout.float() * size).half(), [n], window, 0)


def test_gradients_against_differences(hip_device):
    """(f(x + h d) - f(x - h d)) / 2 h in float64 of the oracle's forward against the
    kernels' gradient along d: the formula itself, not the oracle's."""
    lens, heads, kvh, hd = [37, 20], 4, 2, 64
    g = torch.Generator().manual_seed(9)
    q, k, v, dout = leaves(g, lens, heads, kvh, hd, torch.float16)
    att = WindowAttention(config(heads, kvh, hd), 12, 3)
    starts = torch.tensor(starts_of(lens), dtype=torch.int32, device=hip_device)
    dev = [t.to(hip_device).requires_grad_(True) for t in (q, k, v)]
    say("gradients against differences")
    grads = torch.autograd.grad(att.dense(*dev, starts, 37), dev, dout.to(hip_device))
    x = [t.double() for t in (q, k, v)]
    _, bounds = O.dense(*x, dout.double(), lens, 12, 3, att.scale, torch.float16)

    def loss(parts):
        res, _ = O.dense(*parts, dout.double(), lens, 12, 3, att.scale, torch.float16)
        return float((res[0] * dout.double()).sum())

    h = 1e-5
    for i in range(3):
        d = torch.randn(x[i].shape, generator=g, dtype=torch.float64)
        plus, minus = [list(x), list(x)]
        plus[i], minus[i] = x[i] + h * d, x[i] - h * d
        slope = (loss(plus) - loss(minus)) / (2 * h)
        along = float((grads[i].double().cpu() * d).sum())
        # the kernel's allowed error along d, and the differences' own (h^2 and 1e-16 / h of the loss)
        allowed = float((bounds[i + 1] * d.abs()).sum()) + 1e-4 * abs(slope) + 1e-6
        assert abs(slope - along) <= allowed, (i, slope, along, allowed)


def test_strided_and_broadcast_inputs(hip_device):
    """q, k, v as views of one projection's output, an output gradient that is broadcast,
    keys broadcast over their heads."""
    n, heads, kvh, hd = 70, 4, 2, 128
    g = torch.Generator().manual_seed(2)
    both = torch.randn(n, (heads + 2 * kvh) * hd, generator=g).half().to(hip_device).requires_grad_(True)
    att = WindowAttention(config(heads, kvh, hd), 30, 1)
    starts = torch.tensor([0, n], dtype=torch.int32, device=hip_device)

    def split(t):
        x = t.view(n, heads + 2 * kvh, hd)
        return x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]

    say("strided inputs")
    grad, = torch.autograd.grad(att.dense(*split(both), starts, n).sum(), both)
    x = [t.detach().double().cpu() for t in split(both)]
    ref, bounds = O.dense(*x, torch.ones(n, heads, hd, dtype=torch.float64), [n], 30, 1, att.scale, torch.float16)
    for y, r, b in zip(split(grad), ref[1:], bounds[1:]):
        ok, worst = O.within(y, r, b)
        assert ok, worst
    say("broadcast keys")
    q, k, v, dout = [t.to(hip_device) for t in leaves(g, [n], heads, kvh, hd, torch.float16)]
    one = k[:, :1].contiguous().requires_grad_(True)
    grad, = torch.autograd.grad(att.dense(q, one.expand(n, kvh, hd), v, starts, n), one, dout)
    ref, bounds = O.dense(q.double().cpu(), one.detach().double().cpu().expand(n, kvh, hd), v.double().cpu(),
                          dout.double().cpu(), [n], 30, 1, att.scale, torch.float16)
    total = ref[2].sum(1, keepdim=True)
    # torch sums the two heads' gradients in fp16: one more rounding
    ok, worst = O.within(grad, total, bounds[2].sum(1, keepdim=True) + 2.0 ** -11 * total.abs() * 2)
    assert ok, worst


@pytest.mark.parametrize("far", ["q", "k and v"])
def test_rows_far_apart(hip_device, far):
    """Rows 16 MiB and more apart, whose offsets within a step pass 31 bits."""
    n, heads, kvh, hd, stride = 140, 2, 1, 64, (1 << 23) + 64
    g = torch.Generator().manual_seed(5)
    q, k, v, dout = leaves(g, [n], heads, kvh, hd, torch.bfloat16)
    say(f"rows of {far} {2 * stride} bytes apart")
    flat = torch.empty(n * stride, dtype=torch.bfloat16, device=hip_device)

    def spread(x, at):
        y = flat.as_strided(x.shape, (stride, hd, 1), at)
        y.copy_(x)
        return y

    x = [t.to(hip_device) for t in (q, k, v)]
    d = dout.to(hip_device)
    if far == "q":
        x[0], d = spread(q, 0), spread(dout, 1024)
    else:
        x[1], x[2] = spread(k, 0), spread(v, 1024)
    x = [t.requires_grad_(True) for t in x]
    att = WindowAttention(config(heads, kvh, hd), 50, 2)
    out = att.dense(*x, torch.tensor([0, n], dtype=torch.int32, device=hip_device), n)
    grads = torch.autograd.grad(out, x, d)
    torch.cuda.synchronize()
    ref, bounds = O.dense(*[t.double() for t in (q, k, v, dout)], [n], 50, 2, att.scale, torch.bfloat16)
    for name, y, r, b in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), ref, bounds):
        ok, worst = O.within(y, r, b)
        assert ok, f"{name}: worst error / bound {worst:.3f}"


def test_misaligned_inputs(hip_device):
    """Tensors that start at 2 bytes past a 16-byte unit, and rows of odd strides: the
    results of aligned ones."""
    n, heads, kvh, hd = 50, 4, 2, 128
    g = torch.Generator().manual_seed(5)
    plain = [t.to(hip_device) for t in leaves(g, [n], heads, kvh, hd, torch.float16)]
    att = WindowAttention(config(heads, kvh, hd), 20, 1)
    starts = torch.tensor([0, n], dtype=torch.int32, device=hip_device)
    holder, _ = cache(hip_device, 4, kvh, hd, 32, torch.float16, 2)
    tables = torch.arange(4, dtype=torch.int32, device=hip_device)[None]
    lens = torch.tensor([90], dtype=torch.int32, device=hip_device)

    def moved(t, pad):
        row = t.shape[1] * t.shape[2] + pad
        buf = torch.empty(n * row + 1, dtype=t.dtype, device=hip_device)
        y = buf[1:].as_strided(t.shape, (row, t.shape[2], 1))
        y.copy_(t)
        return y

    results = []
    for place in (lambda t: t, lambda t: moved(t, 0), lambda t: moved(t, 3)):
        say("misaligned inputs")
        x = [place(t).requires_grad_(True) for t in plain[:3]]
        out = att.dense(*x, starts, n)
        results.append([out.detach(), *torch.autograd.grad(out, x, place(plain[3])),
                        att.prefill(x[0].detach(), starts, n, 90, lens, tables, holder)])
    torch.cuda.synchronize()
    for r in results[1:]:
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(r, results[0]))
    with pytest.raises(ValueError):
        att.prefill(plain[0], starts, n, 90, lens, tables, holder, output=moved(plain[0], 0))


@pytest.mark.parametrize("heads,kvh", [(100, 1), (130, 2), (333, 1)])
def test_wide_groups_over_a_cache(hip_device, heads, kvh):
    """More query heads per kv head than a tile has rows, in tiles that end inside a token's heads."""
    for dtype in (torch.float16, torch.bfloat16):
        say(f"{heads} heads on {kvh} over a cache {dtype}")
        check_paged(hip_device, [1, 1], [70, 300], heads, kvh, 64, 32, dtype, 100, 3, decode=True)
        check_paged(hip_device, [5, 17], [70, 300], heads, kvh, 64, 16, dtype, 100, 3)


@pytest.mark.parametrize("group", [65, 77, 100, 255])
def test_gradients_of_groups_that_no_step_holds(hip_device, group):
    test_dense_and_gradients(hip_device, [90, 37], 2 * group, 2, 64, 50, 3, torch.bfloat16)


def test_captured_and_replayed(hip_device):
    """Decode, prompt and a training step in graphs, replayed with changed inputs between
    eager calls of other sizes."""
    dev = hip_device
    holder, g = cache(dev, 80, 2, 128, 32, torch.float16, 8)
    ctxs = [1500, 600]
    tables = tables_of(g, ctxs, 32, 80).to(dev)
    att = WindowAttention(config(8, 2, 128), 900, 4)
    lens = torch.tensor(ctxs, dtype=torch.int32, device=dev)
    q1 = torch.randn(2, 8, 128, generator=g).half().to(dev)
    q2 = torch.randn(90, 8, 128, generator=g).half().to(dev)
    starts = torch.tensor([0, 40, 90], dtype=torch.int32, device=dev)
    t = [x.to(dev).requires_grad_(True) for x in leaves(g, [200, 50], 8, 2, 128, torch.float16)[:3]]
    dout = torch.randn(250, 8, 128, generator=g).half().to(dev)
    ts = torch.tensor([0, 200, 250], dtype=torch.int32, device=dev)

    def step():
        out = att.dense(*t, ts, 200)
        return [out.detach(), *torch.autograd.grad(out, t, dout)]

    def everything():
        return [att.forward(q1, 1500, lens, tables, holder),
                att.prefill(q2, starts, 50, 1500, lens, tables, holder), *step()]

    say("captured and replayed")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = everything()
    for r in range(4):
        with torch.no_grad():
            q1.normal_()
            q2.normal_()
            t[0].normal_()
            lens.copy_(torch.tensor([1500 - 100 * r, 600 - 7 * r], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in kept]
        want = everything()  # eager, between the replays
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), r


def test_no_gradient_through_a_cache(hip_device):
    """Queries that require a gradient: the call runs, also into a given output, and a backward
    pass through it raises."""
    holder, g = cache(hip_device, 4, 2, 64, 32, torch.float16, 1)
    att = WindowAttention(config(4, 2, 64), 8, 1)
    lens = torch.tensor([40, 7], dtype=torch.int32, device=hip_device)
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=hip_device)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device=hip_device)
    q = torch.randn(2, 4, 64, generator=g).half().to(hip_device)
    say("no gradient through a cache")
    want = att.forward(q, 40, lens, tables, holder)
    x = q.clone().requires_grad_(True)
    given = torch.empty_like(q)
    for y in (att.forward(x, 40, lens, tables, holder), att.prefill(x * 1, starts, 1, 40, lens, tables, holder),
              att.forward(x, 40, lens, tables, holder, output=given)):
        assert torch.equal(y.detach(), want)
        with pytest.raises(RuntimeError, match="no gradients"):
            y.sum().backward()
    assert given.data_ptr() == y.data_ptr() and not given.requires_grad and x.grad is None
    both = (att.forward(x, 40, lens, tables, holder) + x).sum()  # beside a path that has gradients
    with pytest.raises(RuntimeError, match="no gradients"):
        both.backward()
    with torch.no_grad():
        assert not att.forward(x, 40, lens, tables, holder).requires_grad


def test_two_streams(hip_device):
    """Two calls of one object at once, each on a stream of its own."""
    dev = hip_device
    holder, g = cache(dev, 200, 2, 128, 32, torch.float16, 8)
    att = WindowAttention(config(8, 2, 128), 900, 4)
    sets = []
    for ctxs in ([1500, 600], [2500]):
        tables = tables_of(g, ctxs, 32, 200).to(dev)
        q = torch.randn(len(ctxs), 8, 128, generator=g).half().to(dev)
        sets.append((q, max(ctxs), torch.tensor(ctxs, dtype=torch.int32, device=dev), tables, holder))
    want = [att.forward(*s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    say("two streams")
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(att.forward(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in got[i]:
            assert torch.equal(y, want[i])


def test_tables_without_columns_and_caches_without_blocks(hip_device):
    """Empty contexts give zeros also where there is no table entry, or no block, at all."""
    dev = hip_device
    att = WindowAttention(config(4, 2, 64), 8, 1)
    lens = torch.zeros(2, dtype=torch.int32, device=dev)
    starts = torch.tensor([0, 1, 41], dtype=torch.int32, device=dev)
    for blocks, width in ((2, 0), (0, 0), (0, 3)):
        holder, _ = cache(dev, blocks, 2, 64, 32, torch.float16, 1)
        tab = torch.full((2, width), -1, dtype=torch.int32, device=dev)
        q = torch.ones(41, 4, 64, dtype=torch.float16, device=dev)
        say(f"{blocks} blocks, tables of {width} columns")
        out = torch.ones_like(q)
        assert not att.forward(q[:2], 0, lens, tab, holder, output=out[:2]).any()
        out.fill_(1)
        assert not att.prefill(q, starts, 40, 0, lens, tab, holder, output=out).any()


def test_wide_bounds(hip_device):
    """Bounds far above the lengths, past 32 bits too: the same results."""
    dev = hip_device
    holder, g = cache(dev, 10, 2, 64, 32, torch.bfloat16, 1)
    att = WindowAttention(config(4, 2, 64), 20, 1)
    starts = torch.tensor([0, 50, 51], dtype=torch.int32, device=dev)
    lens = torch.tensor([60, 90], dtype=torch.int32, device=dev)
    tables = torch.arange(6, dtype=torch.int32, device=dev).view(2, 3)
    q, k, v, dout = [t.to(dev) for t in leaves(g, [50, 1], 4, 2, 64, torch.bfloat16)]
    x = [t.requires_grad_(True) for t in (q, k, v)]
    results = []
    for most in (50, 51, 2 ** 20, 2 ** 31 - 1, 2 ** 32, 2 ** 40):
        say(f"bound {most}")
        out = att.dense(*x, starts, most)
        results.append([att.prefill(q.detach(), starts, most, 90, lens, tables, holder), out.detach(),
                        *torch.autograd.grad(out, x, dout)])
    torch.cuda.synchronize()
    for r in results[1:]:
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(r, results[0]))


def test_empty_calls(hip_device):
    say("empty calls")
    dev = hip_device
    holder, _ = cache(dev, 2, 2, 64, 32, torch.float16, 1)
    att = WindowAttention(config(4, 2, 64), 8, 1)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    q = torch.empty(0, 4, 64, dtype=torch.float16, device=dev)
    tab = torch.zeros(0, 3, dtype=torch.int32, device=dev)
    assert att.forward(q, 0, none, tab, holder).shape == (0, 4, 64)
    assert att.prefill(q, torch.zeros(1, dtype=torch.int32, device=dev), 0, 0, none, tab, holder).shape == (0, 4, 64)
    x = torch.ones(3, 4, 64, dtype=torch.float16, device=dev, requires_grad=True)
    kv = torch.ones(3, 2, 64, dtype=torch.float16, device=dev, requires_grad=True)
    out = att.dense(x, kv, kv, torch.zeros(1, dtype=torch.int32, device=dev), 0)
    out.sum().backward()
    assert not out.any() and not x.grad.any() and not kv.grad.any()
