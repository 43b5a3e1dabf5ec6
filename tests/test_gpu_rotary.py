"""GPU parity of rotary positions (RotaryEmbedding) against oracle/rotary.py in float64 within the
error that the kernels' roundings allow (derived there), and of slot maps (BlockPool.slots) against
oracle/blocks.py, whole numbers equal.

Both pair layouts, parts of the head down to two dims, odd pair counts, every scaling, positions of
zero, below zero and up to 2^31 - 1, strided rows, gradients; keys and values in cache slots bit for
bit beside untouched ones, runs of slots that start and end anywhere, scattered and missing slots;
states with holes; captured and replayed calls; a batch of requests with adapters through
projections, positions, cache and attention.  Every case prints its name before touching the GPU.
"""
from __future__ import annotations

import random

import pytest
import torch

from operators import flags
from operators.core.attention.common import AttentionConfig
from operators.core.attention.real_window import WindowAttention
from operators.core.block.common import BlockInfo
from operators.core.block.pool import BlockPool
from operators.core.block.real import LayerBlocksHolder
from operators.core.linear.adapters import AdaptedLinear, AdapterRows, LowRankAdapters
from operators.core.rope.common import RotaryScaling, rotary_frequencies
from operators.core.rope.real import RotaryEmbedding
from oracle import blocks as B
from oracle import rotary as O
from test_gpu_adapters import quant
from test_gpu_blocks import SIZES, make_pool, random_state, to_state

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def say(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


@pytest.fixture(autouse=True)
def block_size_kept():
    old = flags.BLOCK_SIZE
    yield
    flags.BLOCK_SIZE = old


def check(got, want, err, what):
    d = (got.cpu().double() - want).abs()
    worst = (d - err).max().item() if d.numel() else -1.0
    assert not d.isnan().any() and worst <= 0, f"{what}: {worst} beyond the bound"


def turned(x, positions, rotary, inverse=False):
    return O.turned(x, positions, rotary.frequencies, rotary.magnitude, rotary.rotary_dim, rotary.interleaved, inverse)


FORMS = [  # head dim, rotary dim, interleaved
    (128, 128, False), (128, 128, True), (64, 32, False), (64, 32, True), (80, 80, False), (80, 20, False), (96, 48, True),
    (112, 112, False), (256, 64, False), (128, 2, True), (128, 2, False), (64, 50, True), (64, 50, False), (8, 8, False),
    (8, 4, True), (512, 512, False)]
SCALINGS = [None, RotaryScaling("linear", 4.0), RotaryScaling("ntk", 8.0), RotaryScaling("wavelength", 8.0, 8192),
            RotaryScaling("yarn", 16.0, 4096), RotaryScaling("yarn", 4.0, magnitude=1.25)]
FAR = [0, 1, -1, 2, 4095, 131071, 2 ** 20 + 3, -70000, 2 ** 30 + 7, 2 ** 31 - 1, -2 ** 31]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,rd,interleaved", FORMS)
def test_forward_and_gradients(hip_device, hd, rd, interleaved, dtype):
    g = torch.Generator().manual_seed(hd + rd)
    for rows, heads, kvh in ((1, 1, 1), (11, 3, 2), (70, 8, 1), (5, 2, 5)):
        say(f"rotary {rows} rows, {heads}/{kvh} heads of {hd}, {rd} turning, interleaved {interleaved} {dtype}")
        scaling = SCALINGS[(rows + hd) % len(SCALINGS)]
        if rd == 2 and scaling is not None and scaling.kind == "ntk":
            scaling = None
        rotary = RotaryEmbedding(hd, rd, interleaved=interleaved, scaling=scaling, device=hip_device)
        q, k, dq, dk = (torch.randn(rows, h, hd, generator=g).to(dtype) for h in (heads, kvh, heads, kvh))
        pos = torch.randint(0, 100000, (rows,), generator=g)
        pos[:min(rows, len(FAR))] = torch.tensor(FAR)[:rows]
        a, b = q.to(hip_device).requires_grad_(True), k.to(hip_device).requires_grad_(True)
        qo, ko = rotary.forward(a, b, pos.to(hip_device))
        grads = torch.autograd.grad((qo, ko), (a, b), (dq.to(hip_device), dk.to(hip_device)))
        for name, got, x, inverse in (("q", qo, q, False), ("k", ko, k, False), ("dq", grads[0], dq, True), ("dk", grads[1], dk, True)):
            check(got.detach(), *turned(x, pos, rotary, inverse), name)
        with torch.no_grad():
            again = rotary.forward(a, b, pos.to(hip_device, torch.int32))
        assert torch.equal(again[0], qo) and torch.equal(again[1], ko)
        assert torch.equal(a.detach().cpu(), q)  # not in place


def test_gradients_against_differences(hip_device):
    """Turning is linear: a step's difference is the gradient's product with it, but for roundings."""
    say("rotary differences")
    g = torch.Generator().manual_seed(1)
    rotary = RotaryEmbedding(64, 32, interleaved=True, scaling=RotaryScaling("yarn", 8.0), device=hip_device)
    q, k, dq = (torch.randn(9, 4, 64, generator=g).to(F16) for _ in range(3))
    pos = torch.randint(0, 5000, (9,), generator=g).to(hip_device)
    leaf = q.to(hip_device).requires_grad_(True)
    out = rotary.forward(leaf, k.to(hip_device), pos)[0]
    (grad,) = torch.autograd.grad(out, leaf, dq.to(hip_device))
    moved = (q + torch.randn(q.shape, generator=g).to(F16)).to(F16)
    after = rotary.forward(moved.to(hip_device), k.to(hip_device), pos)[0]
    step, grad = moved.double() - q.double(), grad.double().cpu()
    got = ((after.double().cpu() - out.detach().double().cpu()) * dq.double()).sum()
    room = 2.0 ** -11 * 1.01 * (((after.abs() + out.abs()).detach().double().cpu() * dq.double().abs()).sum() + (grad.abs() * step.abs()).sum())
    assert (got - (grad * step).sum()).abs() <= room


def test_frequencies():
    """Each scaling against its definition; the fast pairs stay and the slow ones are stretched."""
    plain, one = rotary_frequencies(128, 10000.0)
    assert one == 1.0 and plain[0] == 1.0 and abs(plain[32] - 0.01) < 1e-15
    assert rotary_frequencies(128, 10000.0, RotaryScaling("linear", 4.0))[0] == [f / 4 for f in plain]
    ntk = rotary_frequencies(128, 10000.0, RotaryScaling("ntk", 4.0))[0]
    assert ntk[0] == 1.0 and abs(ntk[-1] / (plain[-1] / 4) - 1) < 1e-12
    for kind in ("wavelength", "yarn"):
        got, m = rotary_frequencies(128, 10000.0, RotaryScaling(kind, 8.0, 4096))
        assert got[0] == plain[0] and abs(got[-1] / (plain[-1] / 8) - 1) < 1e-12
        assert all(f / 8 * (1 - 1e-12) <= x <= f for x, f in zip(got, plain)) and got == sorted(got, reverse=True)
        assert m == (1.0 if kind == "wavelength" else 0.1 * torch.log(torch.tensor(8.0, dtype=torch.float64)).item() + 1.0)


def cache(dev, blocks, kvh, hd, bs, dtype, g):
    flags.BLOCK_SIZE = bs
    holder = LayerBlocksHolder.create_contigious_cacher(BlockInfo(hd, kvh, dtype), blocks, dev, dtype)
    for t in holder.contigious_kv_tenosr:
        t.copy_(torch.randn(t.shape, generator=g))
    return holder, [t.cpu().clone() for t in holder.contigious_kv_tenosr]


def slots_of(g, rows, blocks, bs, kind):
    total = blocks * bs
    if kind == "scattered":
        s = torch.randperm(total, generator=g)[:rows]
    else:  # runs from anywhere in blocks in any order
        s, order = [], torch.randperm(blocks, generator=g).tolist()
        while len(s) < rows and order:
            first, n = int(torch.randint(0, bs, (1,), generator=g)), int(torch.randint(1, 3 * bs, (1,), generator=g))
            for i in range(first, first + n):
                if i % bs == 0 or i == first:
                    if not order:
                        break
                    block = order.pop()
                s.append(block * bs + i % bs)
        s = torch.tensor(s[:rows])
        rows = len(s)
    s = s.clone()
    if rows > 4:
        s[rows // 3] = -1
        s[-1] = total + 5  # outside the cache
    return s


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,rd,interleaved,bs,kvh,rows,kind", [
    (128, 128, False, 16, 2, 1, "runs"), (128, 128, False, 32, 2, 45, "scattered"), (64, 64, True, 16, 1, 333, "runs"),
    (80, 20, False, 32, 3, 100, "runs"), (112, 50, True, 16, 2, 70, "scattered"), (256, 256, False, 32, 1, 90, "runs"),
    (64, 64, False, 16, 1, 2500, "runs"), (96, 48, True, 32, 2, 2100, "runs"), (512, 512, False, 16, 1, 2100, "runs"), (512, 40, True, 32, 1, 9, "scattered"), (128, 2, False, 16, 1, 2049, "scattered")])
def test_into_the_cache(hip_device, hd, rd, interleaved, bs, kvh, rows, kind, dtype):
    say(f"rotary into the cache: {rows} rows, {kvh} heads of {hd}, {rd} turning, blocks of {bs}, {kind} {dtype}")
    g = torch.Generator().manual_seed(rows + hd)
    heads = 2 * kvh
    holder, pages = cache(hip_device, rows // bs + 9, kvh, hd, bs, dtype, g)
    slots = slots_of(g, rows, rows // bs + 9, bs, kind)
    rows = len(slots)
    rotary = RotaryEmbedding(hd, rd, interleaved=interleaved, scaling=SCALINGS[1], device=hip_device)
    merged = torch.randn(rows, (heads + 2 * kvh) * hd, generator=g).to(dtype)
    q, k, v = (t.view(rows, -1, hd) for t in merged.split([heads * hd, kvh * hd, kvh * hd], 1))
    pos = torch.randint(0, 50000, (rows,), generator=g)
    dev = merged.to(hip_device)
    qd, kd, vd = (t.view(rows, -1, hd) for t in dev.split([heads * hd, kvh * hd, kvh * hd], 1))
    out = rotary.forward_cached(qd, kd, vd, pos.to(hip_device), slots.to(hip_device), holder)
    check(out, *turned(q, pos, rotary), "q")
    assert torch.equal(dev.cpu(), merged)
    # the cache: the turned keys as forward() gives them, bit for bit, everything else as it was
    turned_k = rotary.forward(qd, kd, pos.to(hip_device))[1].cpu()
    check(turned_k, *turned(k, pos, rotary), "k")
    there = (slots >= 0) & (slots < pages[0].shape[0] * bs)
    block, off = slots[there] // bs, slots[there] % bs
    pages[0][block, :, :, off] = turned_k[there].view(-1, kvh, hd // 8, 8)
    pages[1][block, :, :, off] = v[there]
    for name, got, want in zip("kv", holder.contigious_kv_tenosr, pages):
        assert torch.equal(got.cpu().view(torch.int16), want.view(torch.int16)), name
    # in place of the queries, with 32-bit slots; contiguous inputs give the same
    qc = qd.contiguous()
    assert rotary.forward_cached(qc, kd.contiguous(), vd.contiguous(), pos.to(hip_device), slots.to(hip_device, torch.int32),
                                 holder, output=qc) is qc
    assert torch.equal(qc, out)


def test_cached_calls_and_refusals(hip_device):
    say("cached rotary: refusals, empty calls, no gradients")
    dev, g = hip_device, torch.Generator().manual_seed(0)
    holder, pages = cache(dev, 4, 2, 64, 16, F16, g)
    rotary = RotaryEmbedding(64, device=dev)
    q, k = torch.randn(6, 4, 64, generator=g).to(dev, F16), torch.randn(6, 2, 64, generator=g).to(dev, F16)
    pos, slots = torch.arange(6, device=dev), torch.arange(6, device=dev)
    for args, kind in (((q.bfloat16(), k.bfloat16(), k.bfloat16(), pos, slots, holder), TypeError),
                       ((q, k, k.bfloat16(), pos, slots, holder), TypeError),
                       ((q.float(), k.float(), k.float(), pos, slots, holder), TypeError),
                       ((q, k[:, :1], k[:, :1], pos, slots, holder), AssertionError),
                       ((q, k, k[:5], pos, slots, holder), AssertionError), ((q, k, k, pos[:5], slots, holder), ValueError),
                       ((q, k, k, pos, slots[:5], holder), ValueError), ((q, k, k, pos.float(), slots, holder), ValueError),
                       ((q, k, k, pos, slots.double(), holder), ValueError), ((q, k, k, pos.cpu(), slots, holder), ValueError),
                       ((q, k, k, pos, slots, holder, q[:3]), ValueError)):
        with pytest.raises(kind):
            rotary.forward_cached(*args)
    assert rotary.forward_cached(q[:0], k[:0], k[:0], pos[:0], slots[:0], holder).shape == (0, 4, 64)
    a, b = rotary.forward(q[:0], k[:0], pos[:0])
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    assert all(torch.equal(t.cpu(), p) for t, p in zip(holder.contigious_kv_tenosr, pages))
    out = rotary.forward_cached(q.requires_grad_(True), k, k, pos, slots, holder)
    with pytest.raises(RuntimeError, match="no gradients"):
        out.sum().backward()
    with pytest.raises(AssertionError):
        rotary.forward(q, k[:3], pos)


def test_missing_gradients_are_zero(hip_device):
    say("a gradient of q alone")
    rotary = RotaryEmbedding(64, device=hip_device)
    q = torch.randn(5, 2, 64, device=hip_device, dtype=F16).requires_grad_(True)
    k = torch.randn(5, 1, 64, device=hip_device, dtype=F16).requires_grad_(True)
    qo, _ = rotary.forward(q, k, torch.arange(5, device=hip_device))
    dq, dk = torch.autograd.grad(qo, (q, k), torch.ones(1, 1, 1, device=hip_device, dtype=F16).expand(5, 2, 64))
    assert dq.abs().sum() > 0 and not dk.any()


@pytest.mark.parametrize("rows,width,blocks,bs", SIZES)
def test_slots(hip_device, rows, width, blocks, bs):
    rng = random.Random(rows + 7)
    pool, _ = make_pool(hip_device, blocks, layers=0, bs=bs)
    tables, lens, refs = random_state(rng, rows, width, blocks, bs)
    state = to_state(hip_device, tables, lens, refs, width)
    for name, new in (("some", [rng.randint(-2, max(1, n)) for n in lens]), ("one each", [1] * rows), ("all", [n + 5 for n in lens]),
                      ("none", [0] * rows)):
        need = sum(max(min(n, m), 0) for n, m in zip(new, lens))
        for tokens in {need, need + 13, max(need - 1, 0), 0}:
            say(f"slots of {rows} rows, blocks of {bs}: {name}, {need} in {tokens}")
            got = pool.slots(state, torch.tensor(new, device=hip_device), tokens)
            want = B.slots(tables, lens, refs, new, tokens, bs)
            assert got.excess.tolist() == [want[4]]
            for x, y in zip(got, want[:4]):
                assert x.tolist() == y
    assert state.block_tables.tolist() == tables


def test_slots_of_many_and_of_no_rows(hip_device):
    say("slots of 8192 rows, and of none")
    pool, _ = make_pool(hip_device, 9000, layers=0, bs=16)
    rng = random.Random(3)
    lens = [rng.randint(0, 16) for _ in range(8192)]
    tables = [[i] if n else [-1] for i, n in enumerate(lens)]
    refs = [int(i < 8192 and lens[i] > 0) if i < 8192 else 0 for i in range(9000)]
    state = to_state(hip_device, tables, lens, refs, 1)
    new = [rng.randint(0, 3) for _ in lens]
    got = pool.slots(state, torch.tensor(new, device=hip_device), 24000)
    want = B.slots(tables, lens, refs, new, 24000, 16)
    for x, y in zip(got, (*want[:4], [want[4]])):
        assert x.tolist() == y
    empty = pool.slots(pool.new_state(0, 4), torch.empty(0, dtype=torch.int32, device=hip_device), 5)
    assert empty.query_starts.tolist() == [0] and empty.slots.tolist() == [-1] * 5 and empty.excess.tolist() == [0]
    with pytest.raises(ValueError):
        pool.slots(state, torch.tensor(new, device=hip_device), -1)
    with pytest.raises(ValueError):
        pool.slots(state, torch.tensor(new[:5], device=hip_device), 5)
    with pytest.raises(RuntimeError):  # more rows than the call takes
        big = pool.new_state(8193, 1)
        pool.slots(big, torch.zeros(8193, dtype=torch.int32, device=hip_device), 1)


def test_captured_step(hip_device):
    """Slots, rotary and cache writes of a decode step in one graph, replayed as rows grow."""
    say("captured rotary step")
    dev, g = hip_device, torch.Generator().manual_seed(2)
    flags.BLOCK_SIZE = 16
    holder, _ = cache(dev, 40, 2, 64, 16, BF16, g)
    pool = BlockPool([holder])
    rotary = RotaryEmbedding(64, device=dev)
    q, k, v = (torch.zeros(5, h, 64, device=dev, dtype=BF16) for h in (4, 2, 2))
    one = torch.ones(5, dtype=torch.int32, device=dev)
    state = pool.extend(pool.new_state(5, 8), torch.tensor([3, 16, 1, 30, 15], device=dev))
    tables, lens, refs = (t.clone() for t in state[:3])
    held = type(state)(tables, lens, refs)

    def step():
        new = pool.extend(held, one)
        m = pool.slots(new, one, 5)
        out = rotary.forward_cached(q, k, v, m.positions, m.slots, holder)
        for mine, t in zip((tables, lens, refs), new):
            mine.copy_(t)
        return out, m

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, m = step()
    want = [3, 16, 1, 30, 15]
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert m.positions.tolist() == [n + i for n in want]
        check(out, *turned(q.cpu(), m.positions.cpu(), rotary), f"replay {i}")
        got = holder.kv_tensor_from_slots_with_convert_with_create(m.slots)
        torch.cuda.synchronize()
        assert torch.equal(got[0], rotary.forward(q, k, m.positions)[1]) and torch.equal(got[1], v)


def test_requests_with_adapters_through_a_stage(hip_device):
    """The run of them: ragged prompts and then a decode step of requests with different adapters,
    through adapted q, k and v projections, slots, positions and cache, and attention over it; against
    the same in float64 from the 16-bit values that each step hands to the next."""
    say("requests with adapters through a stage")
    dev, hidden, heads, kvh, hd = hip_device, 256, 4, 2, 64
    flags.BLOCK_SIZE = 16
    g = torch.Generator().manual_seed(9)
    holder, _ = cache(dev, 64, kvh, hd, 16, F16, g)
    pool, rotary = BlockPool([holder]), RotaryEmbedding(hd, scaling=RotaryScaling("yarn", 4.0, 64), device=dev)
    att = WindowAttention(AttentionConfig(hidden, hd, heads, kvh, heads // kvh))
    projections = []
    for i, n in enumerate((heads * hd, kvh * hd, kvh * hd)):
        bank = LowRankAdapters(hidden, n, 8, 3, device=dev)
        for j in range(3):
            bank.load(j, torch.randn(8, hidden, generator=g) * 0.06, torch.randn(n, 8, generator=g) * 0.3, 0.7)
        projections.append(AdaptedLinear(quant(dev, hidden, n, seed=20 + i), bank))
    adapters = torch.tensor([1, -1, 0, 2, 1], device=dev)
    history = [[] for _ in range(5)]
    state = pool.new_state(5, 8)
    for step, new in enumerate(([17, 5, 40, 1, 33], [1, 1, 1, 1, 1], [2, 0, 30, 1, 0])):
        tokens = sum(new) + (3 if step == 2 else 0)  # a padded batch
        new_t = torch.tensor(new, device=dev)
        state = pool.extend(state, new_t)
        assert state.shortage.tolist() == [0]
        m = pool.slots(state, new_t, tokens)
        row_of = m.rows.long()
        index = torch.where(row_of >= 0, adapters[row_of.clamp(min=0)], -1)
        rows = AdapterRows(index, 3)
        x = torch.randn(tokens, hidden, generator=g).to(dev, F16)
        with torch.no_grad():
            q, k, v = (p(x, rows).view(tokens, -1, hd) for p in projections)
            qr = rotary.forward_cached(q, k, v, m.positions, m.slots, holder)
            out = att.prefill(qr, m.query_starts, max(new), 128, state.context_lens, state.block_tables, holder)
        kr = rotary.forward(q, k, m.positions)[1]
        for p, y in zip(projections, (q, k, v)):  # the adapters' part, on top of the projection's
            base = p.base(x).double().cpu()
            a, b, s = p.adapters.a.detach().double().cpu(), p.adapters.b.detach().double().cpu(), p.adapters.scaling.double().cpu()
            for t, i in enumerate(index.tolist()):
                want = base[t] + (s[i] * (b[i] @ (a[i] @ x[t].double().cpu())) if i >= 0 else 0)
                assert torch.allclose(y[t].flatten().double().cpu(), want, rtol=2.0 ** -10, atol=2.0 ** -10), (t, i)
        at = 0
        for r, n in enumerate(new):
            for t in range(at, at + n):
                history[r].append((kr[t].double().cpu(), v[t].double().cpu()))
            keys, values = (torch.stack(z, 1).repeat_interleave(heads // kvh, 0) if z else None
                            for z in zip(*history[r])) if history[r] else (None, None)
            for i in range(n):
                seen = len(history[r]) - n + i + 1
                logits = torch.einsum("hd,htd->ht", qr[at + i].double().cpu(), keys[:, :seen]) * hd ** -0.5
                want = torch.einsum("ht,htd->hd", logits.softmax(1), values[:, :seen])
                # the bound of windowed attention's own tests is finer; here the wiring is what counts
                assert (out[at + i].double().cpu() - want).abs().max() <= 2.0 ** -9 * values.abs().max()
            at += n


def test_forward_mode_derivatives_are_refused(hip_device):
    say("forward-mode derivatives")
    g = torch.Generator().manual_seed(4)
    holder, pages = cache(hip_device, 4, 2, 64, 16, F16, g)
    rotary = RotaryEmbedding(64, device=hip_device)
    q, k = torch.randn(6, 4, 64, generator=g).to(hip_device, F16), torch.randn(6, 2, 64, generator=g).to(hip_device, F16)
    pos = torch.arange(6, device=hip_device)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(k, torch.ones_like(k))
        for call in (lambda: rotary.forward(q, dual, pos), lambda: rotary.forward_cached(q, k, dual, pos, pos, holder),
                     lambda: rotary.forward_cached(q, dual, k, pos, pos, holder, output=q)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        rotary.forward(q, k, pos)
    assert all(torch.equal(t.cpu(), p) for t, p in zip(holder.contigious_kv_tenosr, pages))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,rd,interleaved", [(128, 128, False), (64, 32, True), (64, 50, False)])
def test_positions_of_64_bits(hip_device, hd, rd, interleaved, dtype):
    """64-bit positions are what they are, also those that 32 bits do not hold."""
    say(f"64-bit positions, heads of {hd}, {rd} turning, interleaved {interleaved} {dtype}")
    g = torch.Generator().manual_seed(hd)
    wide = [2 ** 31, 2 ** 31 + 4097, -2 ** 31 - 1, 2 ** 32, 2 ** 33 + 5, -2 ** 35 - 7, 2 ** 38 - 1, 2 ** 31 - 1, 0]
    pos = torch.tensor(wide)
    rotary = RotaryEmbedding(hd, rd, interleaved=interleaved, scaling=SCALINGS[4], device=hip_device)
    q, k, v, dq, dk = (torch.randn(9, h, hd, generator=g).to(dtype) for h in (4, 2, 2, 4, 2))
    there = pos.to(hip_device)
    a, b = q.to(hip_device).requires_grad_(True), k.to(hip_device).requires_grad_(True)
    qo, ko = rotary.forward(a, b, there)
    there += 1  # (the next step's, before the backward pass)
    grads = torch.autograd.grad((qo, ko), (a, b), (dq.to(hip_device), dk.to(hip_device)))
    for name, got, x, inverse in (("q", qo, q, False), ("k", ko, k, False), ("dq", grads[0], dq, True), ("dk", grads[1], dk, True)):
        check(got.detach(), *turned(x, pos, rotary, inverse), name)
    holder, pages = cache(hip_device, 2, 2, hd, 16, dtype, g)
    every_other = torch.stack([pos, pos * 0], 1).to(hip_device)[:, 0]
    out = rotary.forward_cached(a.detach(), b.detach(), v.to(hip_device), every_other, torch.arange(9, device=hip_device), holder)
    assert torch.equal(out, qo)
    got = holder.contigious_kv_tenosr[0].cpu()[0, :, :, :9].permute(2, 0, 1, 3).reshape(9, 2, hd)
    assert torch.equal(got, ko.detach().cpu())


def test_turned_in_place_of_queries_with_a_gradient(hip_device):
    """Queries that were overwritten no longer lead to what they were made of."""
    say("in place of queries that require a gradient")
    g = torch.Generator().manual_seed(6)
    holder, _ = cache(hip_device, 4, 2, 64, 16, F16, g)
    rotary = RotaryEmbedding(64, device=hip_device)
    leaf = torch.randn(6, 4, 64, generator=g).to(hip_device, F16).requires_grad_(True)
    k = torch.randn(6, 2, 64, generator=g).to(hip_device, F16)
    pos = torch.arange(6, device=hip_device)
    want = rotary.forward(leaf.detach(), k, pos)[0]
    for made in (lambda: leaf * 1, lambda: (leaf.view(6, 256) * 1).view(6, 4, 64)):
        q = made()
        out = rotary.forward_cached(q, k, k, pos, pos, holder, output=q)
        assert torch.equal(out, want) and torch.equal(q, want)
        for t in (out, q):
            with pytest.raises(RuntimeError, match="no gradients"):
                t.sum().backward()
    into = torch.empty_like(want)
    out = rotary.forward_cached(leaf * 1, k, k, pos, pos, holder, output=into)
    assert torch.equal(into, want) and not into.requires_grad
    with pytest.raises(RuntimeError, match="no gradients"):
        out.sum().backward()
    other = leaf * 1
    rotary.forward_cached(want.clone(), k, k, pos, pos, holder, output=other)
    with pytest.raises(RuntimeError, match="no gradients"):
        other.sum().backward()
    with pytest.raises(RuntimeError, match="leaf"):
        rotary.forward_cached(leaf, k, k, pos, pos, holder, output=leaf)
    assert torch.equal(rotary.forward(leaf.detach(), k, pos)[0], want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,rd,interleaved,rows", [(128, 128, False, 70), (80, 20, True, 9), (64, 64, False, 1)])
def test_queries_of_a_merged_product_in_place(hip_device, hd, rd, interleaved, rows, dtype):
    """The queries' part of merged rows turned where it stands, keys and values beside it unchanged; the gradients
    of such parts."""
    say(f"merged rows in place: {rows} rows, heads of {hd}, {rd} turning, interleaved {interleaved} {dtype}")
    g = torch.Generator().manual_seed(rows)
    heads, kvh = 4, 2
    holder, pages = cache(hip_device, rows // 16 + 2, kvh, hd, 16, dtype, g)
    rotary = RotaryEmbedding(hd, rd, interleaved=interleaved, device=hip_device)
    merged = torch.randn(rows, (heads + 2 * kvh) * hd, generator=g).to(dtype)
    pos = torch.randint(0, 9000, (rows,), generator=g)
    dev = merged.to(hip_device)
    q, k, v = (t.view(rows, -1, hd) for t in dev.split([heads * hd, kvh * hd, kvh * hd], 1))
    want = rotary.forward(q, k, pos.to(hip_device))
    assert rotary.forward_cached(q, k, v, pos.to(hip_device), torch.arange(rows, device=hip_device), holder, output=q) is q
    check(q, *turned(merged[:, :heads * hd].reshape(rows, heads, hd), pos, rotary), "q")
    assert torch.equal(q, want[0]) and torch.equal(dev[:, heads * hd:].cpu(), merged[:, heads * hd:])
    got = holder.kv_tensor_from_slots_with_convert_with_create(torch.arange(rows, device=hip_device))
    assert torch.equal(got[0], want[1]) and torch.equal(got[1], v)
    leaf = merged.to(hip_device).requires_grad_(True)
    parts = [t.view(rows, -1, hd) for t in leaf.split([heads * hd, kvh * hd, kvh * hd], 1)]
    grads = torch.randn(merged.shape, generator=g).to(dtype)
    dq, dk = (t.reshape(rows, -1, hd) for t in grads.split([heads * hd, kvh * hd, kvh * hd], 1)[:2])
    given = [t.view(rows, -1, hd) for t in grads.to(hip_device).split([heads * hd, kvh * hd, kvh * hd], 1)]
    (dx,) = torch.autograd.grad(rotary.forward(*parts[:2], pos.to(hip_device)), leaf, given[:2])
    for name, x, first in (("dq", dq, 0), ("dk", dk, heads)):
        check(dx[:, first * hd:(first + x.shape[1]) * hd].view(rows, -1, hd), *turned(x, pos, rotary, True), name)
    assert not dx[:, (heads + kvh) * hd:].any()
