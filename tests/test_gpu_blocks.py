"""GPU parity of the cache-block pool (BlockPool) against oracle/blocks.py: whole
numbers equal, block contents bit for bit.

Growing, forking, freeing and compacting random states of one row to some
hundred, tables with holes, blocks shared by rows and held from outside, rows
that end, pools without room (the state then stays as it was), captured and
replayed calls; and a serving run of them together with prompts and decode
steps of windowed attention, against attention over the rows' own tokens.
Every case prints its name before touching the GPU.
"""
from __future__ import annotations

import random

import pytest
import torch

from operators import flags
from operators.core.attention.common import AttentionConfig
from operators.core.attention.real_window import WindowAttention
from operators.core.block.common import BlockInfo
from operators.core.block.pool import BlockPool, BlockState
from operators.core.block.real import LayerBlocksHolder
from oracle import blocks as B
from oracle import window as O

pytestmark = pytest.mark.gpu


def say(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


@pytest.fixture(autouse=True)
def block_size_kept():
    old = flags.BLOCK_SIZE
    yield
    flags.BLOCK_SIZE = old


def make_pool(dev, blocks, layers=2, kvh=2, hd=64, bs=16, dtype=torch.float16, seed=0):
    flags.BLOCK_SIZE = bs
    info = BlockInfo(head_dim=hd, num_key_value_heads=kvh, dtype=dtype)
    held = [LayerBlocksHolder.create_contigious_cacher(info, blocks, dev, dtype) for _ in range(layers)]
    g = torch.Generator(device=dev).manual_seed(seed)
    for h in held:
        for t in h.contigious_kv_tenosr:
            t.normal_(generator=g)
    return (BlockPool(held) if layers else BlockPool([], blocks, dev)), held


def contents(held):
    return [t.clone() for h in held for t in h.contigious_kv_tenosr]


def random_state(rng, rows, width, blocks, bs, shared=True):
    """Tables of rows with lengths anywhere up to their width, some full blocks shared, some
    entries missing (given back), some blocks held from outside."""
    order = list(range(blocks))
    rng.shuffle(order)
    tables, lens, refs = [], [], [0] * blocks
    for r in range(rows):
        n = rng.randint(0, width * bs)
        row = []
        for b in range(-(-n // bs)):
            full = (b + 1) * bs <= n
            if shared and r and full and rng.random() < 0.3 and b < len(tables[-1]) and tables[-1][b] >= 0 and \
                    (b + 1) * bs <= lens[-1]:
                row.append(tables[-1][b])
            elif full and rng.random() < 0.15:
                row.append(-1)
            elif order:
                row.append(order.pop())
            else:
                row.append(-1)
        lens.append(n)
        tables.append(row + [-1] * (width - len(row)))
    for row in tables:
        for e in row:
            if e >= 0:
                refs[e] += 1
    for p in rng.sample(range(blocks), blocks // 10):
        refs[p] += 1
    return tables, lens, refs


def to_state(dev, tables, lens, refs, width):
    t = torch.tensor(tables, dtype=torch.int32).view(len(lens), width).to(dev)
    return BlockState(t, torch.tensor(lens, dtype=torch.int32).to(dev), torch.tensor(refs, dtype=torch.int32).to(dev))


def check_state(got, tables, lens, refs, shortage):
    torch.cuda.synchronize()
    assert got.shortage.tolist() == [shortage]
    assert got.context_lens.tolist() == lens
    assert got.block_tables.tolist() == tables
    assert got.refs.tolist() == refs


SIZES = [(1, 1, 3, 16), (1, 7, 20, 32), (5, 9, 60, 16), (33, 12, 600, 32), (130, 40, 6000, 16), (1100, 3, 2500, 32)]


@pytest.mark.parametrize("rows,width,blocks,bs", SIZES)
def test_extend(hip_device, rows, width, blocks, bs):
    rng = random.Random(rows)
    pool, _ = make_pool(hip_device, blocks, layers=0, bs=bs)
    tables, lens, refs = random_state(rng, rows, width, blocks, bs)
    state = to_state(hip_device, tables, lens, refs, width)
    room = [width * bs - n for n in lens]
    free = sum(c == 0 for c in refs)
    for name, add in (("fits", [rng.randint(-3, min(m, 2 * bs)) if i < free // 2 else 0 for i, m in enumerate(room)]),
                      ("none", [0] * rows), ("too long", [m + 1 + (i == 0) * 40 for i, m in enumerate(room)])):
        say(f"extend {rows} rows, {blocks} blocks of {bs}: {name}")
        got = pool.extend(state, torch.tensor(add, dtype=torch.int32, device=hip_device))
        check_state(got, *B.extend(tables, lens, refs, add, bs))
    assert state.block_tables.tolist() == tables and state.refs.tolist() == refs  # the given state is kept


@pytest.mark.parametrize("rows,width,blocks,bs", SIZES)
def test_fork(hip_device, rows, width, blocks, bs):
    rng = random.Random(rows + 1)
    pool, held = make_pool(hip_device, blocks, layers=2 if blocks <= 600 else 1, kvh=1, bs=bs)
    tables, lens, refs = random_state(rng, rows, width, blocks, bs)
    state = to_state(hip_device, tables, lens, refs, width)
    for name, parents in (("itself", list(range(rows))), ("one for all", [rows // 2] * rows),
                          ("random", [rng.randint(-1, rows) for _ in range(rows)])):
        say(f"fork {rows} rows, {blocks} blocks of {bs}: {name}")
        before = contents(held)
        got = pool.fork(state, torch.tensor(parents, dtype=torch.int64, device=hip_device))
        *want, pairs = B.fork(tables, lens, refs, parents, bs)
        check_state(got, *want)
        for src, dst in pairs:
            for t in before:
                t[dst] = t[src]
        assert all(torch.equal(a, b) for a, b in zip(contents(held), before))


def test_fork_without_room(hip_device):
    """Two copies wanted, one block free: nothing changes."""
    say("fork without room")
    pool, held = make_pool(hip_device, 4, bs=16)
    tables, lens, refs = [[0, 1], [2, -1], [-1, -1]], [20, 5, 0], [1, 1, 1, 0]
    state = to_state(hip_device, tables, lens, refs, 2)
    before = contents(held)
    got = pool.fork(state, torch.tensor([0, 0, 0], device=hip_device))
    check_state(got, tables, lens, refs, 1)
    assert all(torch.equal(a, b) for a, b in zip(contents(held), before))
    got = pool.fork(state, torch.tensor([0, 0, -1], device=hip_device))
    *want, _ = B.fork(tables, lens, refs, [0, 0, -1], 16)
    check_state(got, *want)


@pytest.mark.parametrize("rows,width,blocks,bs", SIZES)
def test_free(hip_device, rows, width, blocks, bs):
    rng = random.Random(rows + 2)
    pool, _ = make_pool(hip_device, blocks, layers=0, bs=bs)
    tables, lens, refs = random_state(rng, rows, width, blocks, bs)
    state = to_state(hip_device, tables, lens, refs, width)
    done = [rng.random() < 0.2 for _ in range(rows)]
    for window, sinks, finished in ((None, 0, done), (1, 0, done), (bs, 0, None), (bs + 1, 4, done), (7, bs, None),
                                    (40, bs + 1, None), (10 ** 9, 0, None), (2 ** 40, 2 ** 40, None)):
        say(f"free {rows} rows of {width} blocks of {bs}: window {window}, sinks {sinks}")
        f = None if finished is None else torch.tensor(finished, device=hip_device)
        got = pool.free(state, window, sinks, f)
        check_state(got, *B.free(tables, lens, refs, bs, window if window and window < 2 ** 31 else 0,
                                 sinks, finished or [False] * rows), 0)


@pytest.mark.parametrize("rows,width,blocks,bs", SIZES + [(3, 2, 4000, 16), (40, 5, 200, 32)])
def test_compact(hip_device, rows, width, blocks, bs):
    rng = random.Random(rows + 3)
    pool, held = make_pool(hip_device, blocks, layers=2 if blocks <= 600 else 1, kvh=1, bs=bs)
    tables, lens, refs = random_state(rng, rows, width, blocks, bs)
    state = to_state(hip_device, tables, lens, refs, width)
    say(f"compact {rows} rows, {blocks} blocks of {bs}")
    before = contents(held)
    got, live = pool.compact(state)
    want_tables, want_refs, want_live, pairs = B.compact(tables, refs)
    check_state(got, want_tables, lens, want_refs, 0)
    assert live.tolist() == [want_live]
    for src, dst in pairs:
        for t in before:
            t[dst] = t[src]
    assert all(torch.equal(a, b) for a, b in zip(contents(held), before))
    again, live = pool.compact(got)  # already together: nothing moves
    check_state(again, want_tables, lens, want_refs, 0)
    assert all(torch.equal(a, b) for a, b in zip(contents(held), before))


@pytest.mark.parametrize("rows,width,blocks,count", [(5, 9, 200, 30), (1, 7, 40, 1), (3, 4, 50, 0), (0, 4, 60, 9), (4, 0, 60, 9)])
def test_compact_tells_where_held_blocks_went(hip_device, rows, width, blocks, count):
    """Blocks counted for a holder outside the tables: their contents are found at the numbers
    returned; numbers that are no block stay what they are."""
    rng = random.Random(blocks)
    pool, layers = make_pool(hip_device, blocks, layers=2, kvh=1)
    tables, lens, refs = random_state(rng, rows, width, blocks, 16)
    free = [p for p in range(blocks) if refs[p] == 0]
    held = rng.sample(free, count)
    for p in held:
        refs[p] += 1
    if count > 2:
        held[0], held[2] = -1, blocks       # (their old blocks stay counted)
    say(f"compact with {count} blocks held outside, {rows} rows of {width}")
    before = contents(layers)
    got, live, now = pool.compact(to_state(hip_device, tables, lens, refs, width),
                                  torch.tensor(held, dtype=torch.int64, device=hip_device))
    want_tables, want_refs, want_live, pairs = B.compact(tables, refs)
    check_state(got, want_tables, lens, want_refs, 0)
    assert got.block_tables.shape == (rows, width) and live.tolist() == [want_live]
    to = dict(pairs)
    assert now.dtype == torch.int32 and now.tolist() == [to.get(p, p) for p in held]
    for old, p in zip(held, now.tolist()):
        if 0 <= old < blocks:
            assert p < want_live
            assert all(torch.equal(a[p], b[old]) for a, b in zip(contents(layers), before))
    # the state goes on into other calls
    pool.extend(got, torch.zeros(rows, dtype=torch.int32, device=hip_device))


@pytest.mark.parametrize("kvh,hd,bs,dtype", [(1, 64, 16, torch.float16), (3, 80, 16, torch.bfloat16),
                                             (32, 128, 32, torch.float16), (2, 256, 32, torch.bfloat16)])
def test_copy(hip_device, kvh, hd, bs, dtype):
    pool, held = make_pool(hip_device, 30, layers=3, kvh=kvh, hd=hd, bs=bs, dtype=dtype)
    before = contents(held)
    pairs = [[3, 9], [4, 0], [-1, 5], [7, 30], [3, 11], [8, 8], [29, 28]]
    say(f"copy blocks of {kvh} x {hd} x {bs}")
    pool.copy(torch.tensor(pairs, device=hip_device))
    pool.copy(torch.zeros(0, 2, dtype=torch.int32, device=hip_device))
    torch.cuda.synchronize()
    for src, dst in pairs:
        if 0 <= src < 30 and 0 <= dst < 30:
            for t in before:
                t[dst] = t[src]
    assert all(torch.equal(a, b) for a, b in zip(contents(held), before))


def test_numbers_past_32_bits(hip_device):
    """64-bit numbers of no block and no row, whose low 32 bits name one, and tokens by the
    billion: skipped, ended, missing."""
    pool, held = make_pool(hip_device, 6, bs=16)
    before = contents(held)
    say("numbers past 32 bits")
    pool.copy(torch.tensor([[2 ** 32, 3], [1, 2 ** 33 + 4], [-2 ** 32 + 2, 5]], device=hip_device))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(contents(held), before))
    tables, lens, refs = [[0, 1], [2, -1]], [20, 5], [1, 1, 1, 0, 0, 0]
    state = to_state(hip_device, tables, lens, refs, 2)
    *want, _ = B.fork(tables, lens, refs, [-1, 1], 16)
    check_state(pool.fork(state, torch.tensor([2 ** 32, 1], device=hip_device)), *want)
    got = pool.extend(state, torch.tensor([2 ** 32, 2 ** 40 + 1], device=hip_device))
    assert got.shortage.item() > 2 ** 27 and got.context_lens.tolist() == lens and got.block_tables.tolist() == tables
    got = pool.extend(state, torch.tensor([-2 ** 32 + 9, 0], device=hip_device))
    check_state(got, tables, lens, refs, 0)


def test_separately_allocated_blocks(hip_device):
    """Layers whose blocks were allocated one by one (pointer tables without contiguous backing)."""
    flags.BLOCK_SIZE = 16
    info = BlockInfo(head_dim=64, num_key_value_heads=2)
    layers, parts = [], []
    for _ in range(2):
        ks = [torch.randn(info.key_block_shape, device=hip_device).half() for _ in range(6)]
        vs = [torch.randn(info.value_block_shape, device=hip_device).half() for _ in range(6)]
        kp, vp = [t.data_ptr() for t in ks], [t.data_ptr() for t in vs]
        kc, vc = torch.tensor(kp), torch.tensor(vp)
        layers.append(LayerBlocksHolder(info, kc.to(hip_device), vc.to(hip_device), kc, vc, kp, vp))
        parts += [ks, vs]
    say("separately allocated blocks")
    want = [[t.clone() for t in p] for p in parts]
    BlockPool(layers).copy(torch.tensor([[1, 4], [5, 0]], device=hip_device))
    torch.cuda.synchronize()
    for p, w in zip(parts, want):
        w[4], w[0] = w[1], w[5]
        assert all(torch.equal(a, b) for a, b in zip(p, w))


def test_captured_and_replayed(hip_device):
    """A loop's step over one set of state buffers, replayed with other inputs between eager calls."""
    dev, bs, rows, width, blocks = hip_device, 16, 9, 12, 200
    rng = random.Random(5)
    pool, held = make_pool(dev, blocks, layers=2, kvh=1, bs=bs)
    tables, lens, refs = random_state(rng, rows, width, blocks, bs)
    state = to_state(dev, tables, lens, refs, width)
    parents = torch.arange(rows, dtype=torch.int32, device=dev)
    add = torch.zeros(rows, dtype=torch.int32, device=dev)
    done = torch.zeros(rows, dtype=torch.bool, device=dev)

    def step():
        a = pool.fork(state, parents)
        b = pool.extend(a, add)
        c = pool.free(b, 50, 4, done)
        d, live = pool.compact(c)
        return a, b, c, d, live

    say("captured pool calls")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for r in range(4):
        t2, l2, r2 = random_state(rng, rows, width, blocks, bs)
        fresh = to_state(dev, t2, l2, r2, width)
        state.block_tables.copy_(fresh.block_tables)
        state.context_lens.copy_(fresh.context_lens)
        state.refs.copy_(fresh.refs)
        p = [rng.randint(-1, rows - 1) for _ in range(rows)]
        n = [rng.randint(0, max(0, width * bs - l2[x])) if x >= 0 else 0 for x in p]
        f = [rng.random() < 0.3 for _ in range(rows)]
        parents.copy_(torch.tensor(p, dtype=torch.int32))
        add.copy_(torch.tensor(n, dtype=torch.int32))
        done.copy_(torch.tensor(f))
        start = contents(held)
        graph.replay()
        torch.cuda.synchronize()
        after = contents(held)
        *a, pairs = B.fork(t2, l2, r2, p, bs)
        b = B.extend(*a[:3], n, bs)
        c = B.free(*b[:3], bs, 50, 4, f)
        d = B.compact(c[0], c[2])
        for got, want in zip(kept, (a, b, (*c, 0), (d[0], c[1], d[1], 0))):
            check_state(got, *want)
        assert kept[4].tolist() == [d[2]]
        for src, dst in pairs + d[3]:
            for t in start:
                t[dst] = t[src]
        assert all(torch.equal(x, y) for x, y in zip(after, start)), r
        eager = pool.fork(state, parents)  # eager work between the replays
        check_state(eager, *a)


def test_serving_run(hip_device):
    """Prompts, beams and decode steps of two layers over one pool: extend, write, prefill,
    free, fork, decode, compact -- each row's attention against its own tokens."""
    dev, bs, heads, kvh, hd, window, sinks = hip_device, 16, 4, 2, 64, 40, 3
    dtype = torch.bfloat16
    pool, held = make_pool(dev, 60, layers=2, kvh=kvh, hd=hd, bs=bs, dtype=dtype)
    att = WindowAttention(AttentionConfig(heads * hd, hd, heads, kvh, heads // kvh), window, sinks)
    g = torch.Generator().manual_seed(3)
    rows, width = 4, 12
    state = pool.new_state(rows, width)
    history = [[(torch.zeros(0, kvh, hd), torch.zeros(0, kvh, hd)) for _ in range(rows)] for _ in held]

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    def advance(state, new):
        """New tokens of each row: blocks, keys and values, attention; checked per row and layer."""
        state = pool.extend(state, ints(new))
        assert state.shortage.item() == 0
        lens, tables = state.context_lens.tolist(), state.block_tables.tolist()
        slots = [tables[r][t // bs] * bs + t % bs for r in range(rows) for t in range(lens[r] - new[r], lens[r])]
        assert min(slots, default=0) >= 0
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        for layer, h in enumerate(held):
            k, v = (torch.randn(sum(new), kvh, hd, generator=g).to(dtype) for _ in range(2))
            h.kv_tensor_to_slots_with_convert(k.to(dev), v.to(dev), torch.tensor(slots, device=dev))
            q = torch.randn(sum(new), heads, hd, generator=g).to(dtype)
            args = (max(lens), state.context_lens, state.block_tables, h)
            if all(n == 1 for n in new):
                out = att.forward(q.to(dev), *args)
            else:
                out = att.prefill(q.to(dev), ints(starts), max(new), *args)
            torch.cuda.synchronize()
            for r in range(rows):
                a, b = starts[r], starts[r + 1]
                hk, hv = history[layer][r]
                hk, hv = torch.cat([hk, k[a:b].float()]), torch.cat([hv, v[a:b].float()])
                history[layer][r] = (hk, hv)
                if a == b:
                    continue
                seen = O.visible(torch.arange(lens[r] - new[r], lens[r]), torch.arange(lens[r]), window, sinks)
                for x in range(heads):
                    o, spread, _ = O.attend(q[a:b, x].double(), hk[:, x // 2].double(), hv[:, x // 2].double(), seen, att.scale)
                    ok, worst = O.within(out[a:b, x], o, O.out_bound(o, spread, lens[r], dtype))
                    assert ok, (r, layer, worst)
        return state

    say("serving run")
    state = advance(state, [50, 0, 21, 0])                       # two prompts
    state = advance(state, [33, 0, 30, 0])                       # their next chunks
    state = pool.free(state, window, sinks)                      # behind the window
    assert (state.block_tables == -1).sum() > 0
    for parents in ([0, 0, 2, 2], [1, 0, 3, 3], [0, 0, 0, 2]):   # beams
        state = pool.fork(state, ints(parents))
        assert state.shortage.item() == 0
        for h in history:
            h[:] = [h[p] for p in parents]
        for _ in range(9):
            state = advance(state, [1] * rows)
        state = pool.free(state, window, sinks)
    state = pool.free(state, finished=torch.tensor([False, True, False, False], device=dev))
    for h in history:
        h[1] = (h[1][0][:0], h[1][1][:0])
    state, live = pool.compact(state)
    assert live.item() == int((state.refs > 0).sum()) == len({e for t in state.block_tables.tolist() for e in t if e >= 0})
    assert state.block_tables.max().item() < live.item()
    state = advance(state, [5, 17, 0, 2])
    state = pool.free(state, finished=torch.ones(rows, dtype=torch.bool, device=dev))
    assert not state.refs.any() and (state.block_tables == -1).all()


def test_empty_states(hip_device):
    """No rows, tables without columns, a pool without blocks."""
    say("empty states")
    for rows, width, blocks in ((0, 4, 10), (3, 0, 10), (3, 4, 0), (0, 0, 0)):
        pool, _ = make_pool(hip_device, blocks, layers=0)
        state = pool.new_state(rows, width)
        ints = torch.zeros(rows, dtype=torch.int32, device=hip_device)
        for got in (pool.extend(state, ints), pool.fork(state, ints), pool.free(state, 4, 1), pool.compact(state)[0]):
            check_state(got, [[-1] * width] * rows, [0] * rows, [0] * blocks, 0)
        if rows:
            got = pool.extend(state, ints + 5)
            want = 0 if width and blocks >= rows else max(rows - blocks, 0) + (0 if width else rows)
            assert got.shortage.item() == want


@pytest.mark.parametrize("blocks", [2047, 32768, 32769, 70001])
def test_many_blocks(hip_device, blocks):
    """Runs of counts that just fit what is read at once, and that take several reads."""
    rng = random.Random(blocks)
    rows, width, bs = 60, blocks // 80, 16
    pool, _ = make_pool(hip_device, blocks, layers=0, bs=bs)
    tables, lens, refs = random_state(rng, rows, width, blocks, bs)
    state = to_state(hip_device, tables, lens, refs, width)
    say(f"{blocks} blocks")
    add = [rng.randint(0, min(width * bs - n, 5 * bs)) for n in lens]
    check_state(pool.extend(state, torch.tensor(add, dtype=torch.int32, device=hip_device)), *B.extend(tables, lens, refs, add, bs))
    parents = [rng.randint(-1, rows - 1) for _ in range(rows)]
    check_state(pool.fork(state, torch.tensor(parents, device=hip_device)), *B.fork(tables, lens, refs, parents, bs)[:4])
    got, live = pool.compact(state)
    want_tables, want_refs, want_live, _ = B.compact(tables, refs)
    check_state(got, want_tables, lens, want_refs, 0)
    assert live.tolist() == [want_live]


def test_two_streams(hip_device):
    """Two states of one pool worked on at once."""
    rng = random.Random(8)
    pool, _ = make_pool(hip_device, 3000, layers=0, bs=16)
    cases = []
    for rows in (20, 50):
        tables, lens, refs = random_state(rng, rows, 30, 3000, 16)
        add = [rng.randint(0, 5) if n < 30 * 16 - 5 else 0 for n in lens]
        cases.append((to_state(hip_device, tables, lens, refs, 30), torch.tensor(add, dtype=torch.int32, device=hip_device),
                      B.extend(tables, lens, refs, add, 16)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    say("two streams")
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(pool.extend(*cases[i][:2]))
    for i in range(2):
        for y in got[i]:
            check_state(y, *cases[i][2])
