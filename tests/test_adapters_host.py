"""CPU tests: adapters, dropout, rotary positions and slot maps refuse malformed calls before anything
reaches a device (fake addresses are never dereferenced), and the generator's oracle gives the
published numbers."""
from __future__ import annotations

import ctypes
import math
from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from hip_extends import _lib
from operators.core.linear.adapters import AdaptedLinear, AdapterRows, CounterDropout, LowRankAdapters
from operators.core.linear.real import Linear
from operators.core.linear.real_quant import QuantLinear
from operators.core.rope.common import RotaryScaling, rotary_frequencies
from operators.core.rope.real import RotaryEmbedding
from oracle import adapters as O
from oracle import blocks as B
from oracle import rotary as R

FAKE, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
OK, BAD, UNSUP, MISAL, WORK = (_lib.DW4_OK, _lib.DW4_ERR_INVALID_ARG, _lib.DW4_ERR_UNSUPPORTED,
                               _lib.DW4_ERR_MISALIGNED, _lib.DW4_ERR_WORKSPACE)


def adapters(dtype=0, rows=50, count=3, k=64, n=32, rank=16, x=FAKE, ldx=64, base=FAKE, ldb=32, out=FAKE, ldo=32, a=FAKE, b=FAKE,
             scaling=FAKE, plan=FAKE, drop=0, seed=None, h=None, ws=FAKE, wsb=0):
    return _lib.load().dw4_adapters(dtype, rows, count, k, n, rank, x, ldx, base, ldb, out, ldo, a, b, scaling, plan, drop, seed,
                                    h, ws, wsb, None)


def backward(dtype=1, rows=50, count=3, k=64, n=32, rank=16, x=FAKE, ldx=64, g=FAKE, ldg=32, a=FAKE, b=FAKE, scaling=FAKE,
             plan=FAKE, drop=0, seed=None, h=FAKE, dx=FAKE, lddx=64, da=FAKE, db=FAKE, ws=FAKE, wsb=0):
    return _lib.load().dw4_adapters_backward(dtype, rows, count, k, n, rank, x, ldx, g, ldg, a, b, scaling, plan, drop, seed, h,
                                             dx, lddx, da, db, ws, wsb, None)


def test_adapter_refusals():
    for call in (adapters, backward):
        assert call() == WORK                                     # a workspace that is too small
        assert call(ws=None, wsb=1 << 30) == WORK
        assert call(ws=ODD, wsb=1 << 30) == MISAL
        assert call(dtype=2) == UNSUP and call(rank=12) == UNSUP and call(rank=136) == UNSUP
        assert call(k=60, ldx=64) == UNSUP and call(n=28) == UNSUP
        assert call(rows=-1) == BAD and call(count=-1) == BAD and call(rank=0) == BAD and call(k=0) == BAD
        assert call(count=1025) == UNSUP and call(rows=(1 << 24) + 1) == UNSUP and call(k=(1 << 20) + 8, ldx=1 << 21) == UNSUP
        assert call(x=None) == BAD and call(a=None) == BAD and call(b=None) == BAD and call(scaling=None) == BAD
        assert call(plan=None) == BAD and call(plan=ODD) == MISAL
        assert call(x=ODD) == MISAL and call(ldx=68) == MISAL and call(ldx=56) == BAD and call(a=ODD) == MISAL
        assert call(drop=-1) == BAD and call(drop=65537) == BAD and call(drop=5) == BAD  # dropout without a seed
        assert call(drop=5, seed=FAKE) == WORK
        assert call(count=0, a=None, b=None, scaling=None) == WORK  # no adapters, no weights
    assert adapters(rows=0, x=None, plan=None) == OK
    assert adapters(base=None) == BAD and adapters(out=None) == BAD and adapters(ldo=24) == BAD and adapters(base=ODD) == MISAL
    assert adapters(h=ODD) == MISAL
    assert adapters(ldo=40, wsb=1 << 30) == BAD                   # in place of base, but other rows
    assert backward(rows=0) == BAD and backward(h=None) == BAD and backward(h=ODD) == MISAL
    assert backward(g=None) == BAD and backward(g=ODD) == MISAL and backward(dx=ODD) == MISAL and backward(lddx=56) == BAD
    assert backward(da=ODD) == MISAL and backward(db=ODD) == MISAL
    assert backward(dx=None, da=None, db=None) == OK


def test_plan_and_workspace_sizes():
    lib, out, h = _lib.load(), ctypes.c_size_t(7), ctypes.c_size_t(7)
    assert lib.dw4_adapter_plan_size(0, 5, ctypes.byref(out)) == OK and out.value == 0
    assert lib.dw4_adapter_plan_size(10, 5, None) == BAD and lib.dw4_adapter_plan_size(-1, 5, ctypes.byref(out)) == BAD
    assert lib.dw4_adapter_plan_size(10, 1025, ctypes.byref(out)) == UNSUP
    assert lib.dw4_adapter_plan_size(1 << 24, 1024, ctypes.byref(out)) == OK and out.value < 1 << 28
    need = _lib.adapter_plan_size(100, 4)
    assert lib.dw4_adapter_plan(100, 4, FAKE, FAKE, need - 1, None) == WORK
    assert lib.dw4_adapter_plan(100, 4, FAKE, ODD, need, None) == MISAL
    assert lib.dw4_adapter_plan(100, 4, None, FAKE, need, None) == BAD and lib.dw4_adapter_plan(100, 4, FAKE, None, need, None) == BAD
    assert lib.dw4_adapter_plan(0, 4, None, None, 0, None) == OK
    size = lib.dw4_adapters_workspace_size
    assert size(0, 4, 64, 64, 16, 1, ctypes.byref(out), ctypes.byref(h)) == OK and out.value == 0 and h.value == 0
    assert size(10, 4, 64, 64, 16, 0, None, None) == BAD and size(10, 4, 64, 64, 15, 0, ctypes.byref(out), None) == UNSUP
    assert size(10, 4, 64, 64, 16, 0, ctypes.byref(out), None) == OK and out.value > 0


def test_dropout_refusals():
    call = _lib.load().dw4_dropout
    assert call(2, 4, 8, FAKE, 8, FAKE, 8, 5, FAKE, None) == UNSUP
    assert call(0, -1, 8, FAKE, 8, FAKE, 8, 5, FAKE, None) == BAD and call(0, 4, 8, FAKE, 8, FAKE, 8, 5, None, None) == BAD
    assert call(0, 4, 8, None, 8, FAKE, 8, 5, FAKE, None) == BAD and call(0, 4, 8, FAKE, 7, FAKE, 8, 5, FAKE, None) == BAD
    assert call(0, 4, 8, FAKE, 8, FAKE, 8, 65537, FAKE, None) == BAD
    assert call(0, 0, 8, None, 8, None, 8, 5, FAKE, None) == OK and call(0, 4, 0, None, 0, None, 0, 5, FAKE, None) == OK


def rotary(dtype=0, rows=9, heads=4, kvh=2, hd=64, rd=64, inter=0, q=FAKE, qs=256, k=FAKE, ks=128, qo=FAKE, qos=256, ko=FAKE, kos=128,
           pos=FAKE, turns=FAKE, m=1.0):
    return _lib.load().dw4_rotary(dtype, rows, heads, kvh, hd, rd, inter, 0, q, qs, k, ks, qo, qos, ko, kos, pos, turns, m, None)


def cached(dtype=0, rows=9, heads=4, kvh=2, hd=64, rd=64, q=FAKE, qs=256, k=FAKE, ks=128, v=FAKE, vs=128, qo=FAKE, qos=256, pos=FAKE,
           turns=FAKE, m=1.0, slots=FAKE, nb=4, bs=16, kp=FAKE, vp=FAKE, hs=1024):
    return _lib.load().dw4_rotary_and_cache(dtype, rows, heads, kvh, hd, rd, 0, q, qs, k, ks, v, vs, qo, qos, pos, turns, m, slots, nb,
                                            bs, kp, vp, hs, None)


def test_rotary_refusals():
    for call in (rotary, cached):
        assert call(dtype=2) == UNSUP and call(rows=-1) == BAD and call(heads=-1) == BAD and call(hd=0) == BAD
        assert call(rd=0) == BAD and call(rd=66) == BAD and call(rd=7) == UNSUP and call(hd=60, rd=60) == UNSUP
        assert call(hd=520, qs=4 * 520, qos=4 * 520, ks=2 * 520, rd=64) == UNSUP
        assert call(m=float("nan")) == BAD and call(m=float("inf")) == BAD
        assert call(q=None) == BAD and call(k=None) == BAD and call(qo=None) == BAD and call(pos=None) == BAD
        assert call(turns=None) == BAD and call(qs=248) == BAD and call(q=ODD) == MISAL and call(ks=132) == MISAL
        assert call(rows=(1 << 24) + 1) == UNSUP and call(rows=1 << 24, heads=64, qs=4096, qos=4096) == UNSUP
        assert call(rows=0, q=None) == OK
    assert rotary(heads=0, kvh=0) == OK and rotary(ko=None) == BAD and rotary(kos=120) == BAD
    assert cached(v=None) == BAD and cached(slots=None) == BAD and cached(kp=None) == BAD and cached(vp=None) == BAD
    assert cached(bs=8) == UNSUP and cached(nb=-1) == BAD and cached(hs=1016) == BAD and cached(hs=1028) == MISAL
    assert cached(kvh=0) == BAD and cached(heads=0) == BAD and cached(v=ODD) == MISAL


def test_slot_refusals():
    def call(rows=5, width=4, nb=9, bs=16, tables=FAKE, lens=FAKE, new=FAKE, tokens=7, starts=FAKE, pos=FAKE, slots=FAKE, row=FAKE,
             excess=FAKE):
        return _lib.load().dw4_token_slots(rows, width, nb, bs, tables, lens, new, tokens, starts, pos, slots, row, excess, None)
    assert call(rows=-1) == BAD and call(width=-1) == BAD and call(nb=-1) == BAD and call(tokens=-1) == BAD
    assert call(bs=24) == UNSUP and call(rows=8193) == UNSUP and call(tokens=(1 << 28) + 1) == UNSUP
    for name in ("tables", "lens", "new", "starts", "pos", "slots", "row", "excess"):
        assert call(**{name: None}) == BAD


def test_modules_refuse_what_the_kernels_do_not_take():
    for kwargs in (dict(rank=12), dict(rank=0), dict(rank=136), dict(in_features=60), dict(out_features=0), dict(num_adapters=0),
                   dict(num_adapters=1025), dict(dropout=1.5), dict(dropout=-0.1)):
        with pytest.raises(ValueError):
            LowRankAdapters(**{**dict(in_features=64, out_features=64, rank=8, num_adapters=2), **kwargs})
    with pytest.raises(TypeError):
        LowRankAdapters(64, 64, 8, 2, dtype=torch.float32)
    with pytest.raises(ValueError):
        CounterDropout(1.01)
    bank = LowRankAdapters(64, 64, 8, 2)
    assert not bank.a.requires_grad and LowRankAdapters(64, 64, 8, 2, trainable=True).b.requires_grad
    assert set(bank.state_dict()) == {"a", "b", "scaling"}
    for args in ((60,), (64, 63), (64, 66), (64, 0), (520,)):
        with pytest.raises(ValueError):
            RotaryEmbedding(*args, device="cuda")
    with pytest.raises(ValueError):
        RotaryEmbedding(64, device="cpu")
    with pytest.raises(ValueError):
        RotaryEmbedding(64, base=0.5)
    for args in (("other", 2.0), ("linear", 0.5), ("yarn", float("inf")), ("yarn", 2.0, 0), ("wavelength", 2.0, 4096, 4.0, 4.0)):
        with pytest.raises(ValueError):
            RotaryScaling(*args)
    with pytest.raises(ValueError):
        rotary_frequencies(2, 10000.0, RotaryScaling("ntk", 2.0))


def test_the_generator_gives_its_published_numbers():
    """Known answers of Philox 4x32 with 10 rounds, published with it."""
    for counter, key, want in (((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                               ((O.WORD,) * 4, (O.WORD,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                               ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                                (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(O.philox(counter, key)) == want


def test_oracles_agree_with_autograd():
    g = torch.Generator().manual_seed(1)
    x, base, dout = (torch.randn(6, w, generator=g).half() for w in (16, 8, 8))
    a, b, s = torch.randn(2, 8, 16, generator=g).half(), torch.randn(2, 8, 8, generator=g).half(), torch.rand(2, generator=g)
    index = torch.tensor([0, 1, -1, 1, 0, 7])
    mask = O.kept(6, 16, 20000, 3, 4)
    leaves = [t.double().requires_grad_(True) for t in (x, a, b)]
    z = torch.where(mask, leaves[0] * (65536 / 45536), 0.0)
    rows = [base[t].double() + (s[i].double() * (leaves[2][i] @ (leaves[1][i] @ z[t])) if 0 <= i < 2 else 0)
            for t, i in enumerate(index.tolist())]
    out = torch.stack(rows)
    want = (out, *torch.autograd.grad(out, leaves, dout.double()))
    got, _ = O.low_rank(x, base, a, b, s, index, dout, mask, 20000)
    assert all(torch.allclose(u, v, rtol=1e-12, atol=1e-12) for u, v in zip(got, want))
    y, _ = R.turned(torch.randn(3, 2, 8, generator=g).half(), torch.tensor([0, 5, -9]), [1.0, 0.5], 1.0, 4, True)
    back, _ = R.turned(y.half(), torch.tensor([0, 5, -9]), [1.0, 0.5], 1.0, 4, True, inverse=True)
    assert y.shape == (3, 2, 8) and torch.isfinite(back).all()
    assert B.slots([[4, -1]], [20], [0] * 9, [6], 8, 16) == ([0, 6], [14, 15, 16, 17, 18, 19, 0, 0], [78, 79, -1, -1, -1, -1, -1, -1],
                                                            [0] * 6 + [-1] * 2, 0)


def test_sizes_beyond_32_bits_are_refused():
    """Sizes that a 32-bit argument would wrap around to small ones."""
    one = torch.zeros(1, dtype=torch.int32)
    for rows, count in (((1 << 24) + 1, 4), ((1 << 32) + 5, 4), (9, 1025), (9, -1)):
        with pytest.raises(ValueError):
            AdapterRows(one.expand(rows), count)
    for kwargs in (dict(in_features=(1 << 20) + 8), dict(out_features=(1 << 32) + 8)):
        with pytest.raises(ValueError):
            LowRankAdapters(**{**dict(in_features=64, out_features=64, rank=8, num_adapters=2), **kwargs})
    x, seed = torch.zeros(1, dtype=torch.float16), torch.zeros(2, dtype=torch.int64)
    for shape in (((1 << 32) + 8,), (3, (1 << 30) + 1), ((1 << 31), 1), ((1 << 32) + 1, 8)):
        with pytest.raises(ValueError):
            CounterDropout(0.5)(x.expand(shape), seed)
    call = _lib.load().dw4_dropout
    assert call(0, 1, (1 << 30) + 1, FAKE, 1 << 31, FAKE, 1 << 31, 5, FAKE, None) == UNSUP
    for test in (rotary, cached):
        assert test(rows=(1 << 22) + 1) == UNSUP and test(rows=1 << 22, heads=32, qs=2048, qos=2048) == UNSUP


class _Passes(Linear):
    def __init__(self):
        torch.nn.Module.__init__(self)

    def forward(self, x):
        return x


def test_a_projection_that_returns_its_input_keeps_it():
    """The adapters' sum goes into the projection's output unless that is the caller's input."""
    seen = []

    class Bank(torch.nn.Module):
        a = b = torch.zeros(1)

        def forward(self, x, y, rows, seed=None, output=None):
            seen.append(output)
            return y

    x = torch.zeros(4, 64, dtype=torch.float16)
    AdaptedLinear(_Passes(), Bank())(x, rows=object())
    assert seen == [None]


def cpu_rotary(head_dim):
    """A RotaryEmbedding whose checks run on the CPU."""
    r = object.__new__(RotaryEmbedding)
    r.device, r.head_dim, r.rotary_dim, r.interleaved, r.magnitude = torch.device("cpu"), head_dim, head_dim, False, 1.0
    return r


class _Doubles(_Passes):
    def forward(self, x):
        return x * 2


def test_forward_mode_derivatives_are_refused():
    """A result without its tangent would be a wrong derivative, and one written into the projection's
    output would keep the projection's tangent alone."""
    rows = SimpleNamespace(device=torch.device("cpu"), num_rows=4, num_adapters=2, plan=None)
    x, t = torch.randn(4, 64).half(), torch.randn(4, 64).half()
    rotary, pos = cpu_rotary(8), torch.arange(4)
    for trainable in (False, True):
        bank = LowRankAdapters(64, 64, 8, 2, trainable=trainable)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, t)
            for args in ((dual, x), (x, dual)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    bank(*args, rows)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                AdaptedLinear(_Doubles(), bank)(dual, rows)
            turned = forward_ad.make_dual(bank.a.detach(), torch.ones_like(bank.a))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.func.functional_call(bank, {"a": turned}, (x, x, rows))
            q, plain = dual.view(4, 8, 8), x.view(4, 8, 8)
            for pair in ((q, plain), (plain, q)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    rotary.forward(*pair, pos)
            with pytest.raises(ValueError):  # without tangents: no HIP device
                bank(x, x, rows)


@pytest.mark.parametrize("name", ["a", "b"])
def test_loading_into_parametrized_adapters_is_refused(name):
    """What a parametrization gives is a tensor of the moment: matrices copied there are lost."""
    bank = LowRankAdapters(64, 32, 8, 2)
    torch.nn.utils.parametrize.register_parametrization(bank, name, torch.nn.Identity())
    before = {k: t.clone() for k, t in bank.state_dict().items()}
    with pytest.raises(RuntimeError, match="parametrized"):
        bank.load(0, torch.ones(8, 64), torch.ones(32, 8), 2.0)
    assert all(torch.equal(t, before[k]) for k, t in bank.state_dict().items())


def test_loading_parts_of_the_bank():
    """An adapter from the bank itself, in its own place with another scaling or moved up in rank, and
    from another's place."""
    bank = LowRankAdapters(64, 32, 16, 2)
    with torch.no_grad():
        bank.b.normal_()
    a, b = bank.a.detach().clone(), bank.b.detach().clone()
    bank.load(0, bank.a[0], bank.b[0], 3.0)
    assert torch.equal(bank.a, a) and torch.equal(bank.b, b) and bank.scaling.tolist() == [3.0, 1.0]
    bank.load(0, bank.a[0, 5:], bank.b[0, :, 5:], 2.0)
    assert torch.equal(bank.a[0, :11], a[0, 5:]) and torch.equal(bank.b[0, :, :11], b[0, :, 5:])
    assert not bank.a[0, 11:].any() and not bank.b[0, :, 11:].any()
    bank.load(1, bank.a[0, :11], bank.b[0, :, :11], 2.0)
    assert torch.equal(bank.a[1], bank.a[0]) and torch.equal(bank.b[1], bank.b[0])


class _Slice(_Passes):
    def forward(self, x):
        return x.flatten()[64:192].view(2, 64)  # begins inside x


class _Keeps(_Passes):
    def __init__(self):
        super().__init__()
        self.kept = torch.zeros(2, 64, dtype=torch.float16)

    def forward(self, x):
        return self.kept


def test_sums_take_the_place_of_new_outputs_alone(monkeypatch):
    """A projection's output is overwritten where it is known to be the call's own: not where it lies in
    the input, where the projection keeps it, or where a hook has seen it."""
    seen = []

    class Bank(torch.nn.Module):
        a = b = torch.zeros(1)

        def forward(self, x, y, rows, seed=None, output=None):
            seen.append(output is y)
            return y

    x = torch.zeros(4, 64, dtype=torch.float16)

    def taken(base):
        AdaptedLinear(base, Bank())(x, rows=object())
        return seen.pop()

    assert not taken(_Slice()) and not taken(_Keeps()) and not taken(_Doubles())
    monkeypatch.setattr(QuantLinear, "forward", lambda self, x: x * 2)
    quant = QuantLinear(64, 64, 64, False, False)
    assert taken(quant)
    hook = quant.register_forward_hook(lambda module, args, y: None)
    assert not taken(quant)
    hook.remove()
    assert taken(quant)
    hook = torch.nn.modules.module.register_module_forward_hook(lambda module, args, y: None)
    try:
        assert not taken(quant)
    finally:
        hook.remove()
    quant.forward = lambda x: x
    assert not taken(quant)


def test_forms_of_rotary_calls():
    lib = _lib.load()
    for form in (4, -1, 1 << 20):
        assert rotary(inter=form) == BAD
        assert lib.dw4_rotary_and_cache(0, 9, 4, 2, 64, 64, form, FAKE, 256, FAKE, 128, FAKE, 128, FAKE, 256, FAKE, FAKE, 1.0, FAKE, 4, 16,
                                        FAKE, FAKE, 1024, None) == BAD
    for form in range(4):
        assert rotary(rows=0, inter=form) == OK


def test_replaced_adapters_keep_their_shapes():
    """A parametrization, a functional call or an assignment may bring other tensors than the module was
    made with: the kernels would read past them."""
    rows = SimpleNamespace(device=torch.device("cpu"), num_rows=4, num_adapters=2, plan=None)
    bank, x = LowRankAdapters(64, 32, 8, 2), torch.zeros(4, 64).half()
    base = torch.zeros(4, 32).half()
    for name, shape in (("a", (1, 8, 64)), ("a", (2, 8, 32)), ("a", (2, 16, 64)), ("a", (8, 64)), ("b", (1, 32, 8)), ("b", (2, 32, 16)),
                        ("b", (2, 24, 8)), ("scaling", (1,)), ("scaling", (2, 1))):
        other = torch.zeros(shape, dtype=torch.float32 if name == "scaling" else torch.float16)
        with pytest.raises(ValueError, match="shapes"):
            torch.func.functional_call(bank, {name: other}, (x, base, rows))
    for name in ("a", "b", "scaling"):
        with pytest.raises(ValueError, match="one device"):
            torch.func.functional_call(bank, {name: getattr(bank, name).detach().to("meta")}, (x, base, rows))


def test_an_output_with_a_gradient_is_refused():
    """What is written over would keep the gradient of what was there."""
    rows = SimpleNamespace(device=torch.device("cpu"), num_rows=4, num_adapters=2, plan=None)
    bank, x = LowRankAdapters(64, 32, 8, 2), torch.zeros(4, 64).half()
    base, into = torch.zeros(4, 32).half(), torch.zeros(4, 32).half().requires_grad_(True)
    for output in (into, into * 1):
        with pytest.raises(ValueError, match="without gradients"):
            bank(x, base, rows, output=output)


def test_the_probability_of_dropout_may_change():
    drop, bank = CounterDropout(0.5), LowRankAdapters(64, 32, 8, 2, dropout=0.5)
    x = torch.zeros(4, 64).half()
    drop.p = 0.0
    assert drop(x) is x and drop.p == 0.0  # no seed is read
    bank.dropout = 0.25
    assert bank.dropout == 0.25 and bank._dropped == 16384
    for change in (lambda: setattr(drop, "p", 1.5), lambda: setattr(bank, "dropout", -0.5)):
        with pytest.raises(ValueError):
            change()
    assert drop.p == 0.0 and bank.dropout == 0.25


def test_backward_workspaces_hold_what_is_written():
    """Shares of gradients are for adapters of more than 512 rows: beside the turned weights a batch of few rows
    an adapter needs little."""
    for rows, count, rank, k, n in ((1024, 1024, 64, 4096, 11008), (512, 2, 128, 4096, 4096), (1, 1024, 8, 64, 64)):
        turned = 2 * count * rank * (k + n)
        need, _ = _lib.adapters_workspace_size(rows, count, k, n, rank, True)
        several = rows // 512 + min(count, rows // 513) if rows > 512 else 0
        # beside them: planes and packed operands, some 16 planes of 32 rows an adapter with rows
        positions = 32 * (rows // 32 + min(count + 1, rows))
        assert turned <= need <= turned + 4 * several * rank * (k + n) + positions * max(rank, 16) * (16 * 4 + 12) + 4096


def test_gradients_beyond_a_launch_are_refused():
    """A launch of 2^32 threads or more, which banks and batches within the other limits would need."""
    size, out = _lib.load().dw4_adapters_workspace_size, ctypes.c_size_t(0)
    for rows, count, k, n, rank in ((2000, 1024, 1 << 20, 64, 8), (2000, 512, 1 << 19, 1 << 19, 72), (1 << 24, 64, 1 << 20, 64, 8),
                                    (1 << 24, 64, 64, 1 << 20, 8)):
        assert size(rows, count, k, n, rank, 1, ctypes.byref(out), None) == UNSUP
        assert size(rows, count, k, n, rank, 0, ctypes.byref(out), None) == OK
        assert backward(rows=rows, count=count, k=k, n=n, rank=rank, ldx=k, ldg=n, lddx=k, wsb=1 << 62) == UNSUP
    assert size(2000, 500, 1 << 19, 1 << 19, 8, 1, ctypes.byref(out), None) == OK


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k,n,rank,adapters,order", O.WIDE)
def test_whole_numbers_tell_what_is_missing(rows, k, n, rank, adapters, order, dtype):
    """The whole-number cases are exact, and show the last columns, a part of the reduced axis or the second part
    of h or dh missing."""
    x, base, a, b, s, dout = O.whole_case(rows, k, n, rank, adapters, dtype, 13)
    index = torch.arange(rows) % adapters

    def results(x=x, dout=dout, one_part=False):
        """(out, db), (dx, da) with x, or dout, as the first products see them."""
        out, dx = base.double().clone(), torch.zeros(rows, k).double()
        da, db = torch.zeros(adapters, rank, k).double(), torch.zeros(adapters, n, rank).double()
        for i in range(adapters):
            t = index == i
            f = 2 * float(s[i])
            h, dh = f * (x[t].double() @ a[i].double().T), f * (dout[t].double() @ b[i].double())
            if one_part:
                h, dh = h.to(dtype).double(), dh.to(dtype).double()
            out[t] += h @ b[i].double().T
            db[i], dx[t], da[i] = whole[1][t].double().T @ h, dh @ a[i].double(), dh.T @ whole[0][t].double()
        return (out, db), (dx, da)

    whole = (x, dout)
    want = results()
    # exact: sums of absolute values in their units
    for i in range(adapters):
        h, dh = x.double().abs() @ a[i].double().abs().T, dout.double().abs() @ b[i].double().abs()
        small = x.double() @ a[i].double().T, dout.double() @ b[i].double()
        assert max(h.max(), dh.max()) < 2 ** 24 and max(v.abs().max() for v in small) < 2 ** 16
        for sums in (small[0].abs() @ b[i].double().abs().T + 100 / s[i], dout.double().abs().T @ small[0].abs(),
                     small[1].abs() @ a[i].double().abs(), small[1].abs().T @ x.double().abs()):
            assert sums.max() < 2 ** 24
    assert all(v.abs().max() < torch.finfo(torch.float16).max for pair in want for v in pair)

    def differ(got, i):
        return all(not torch.equal(g.to(dtype), w.to(dtype)) for g, w in zip(got[i], want[i]))

    lost = torch.ones(k).to(dtype)
    lost[-8:] = 0
    assert differ(results(x=x * lost), 0)
    lost = torch.ones(n).to(dtype)
    lost[-8:] = 0
    assert differ(results(dout=dout * lost), 1)
    if k > 4000:
        lost = torch.ones(k).to(dtype)
        lost[256:320] = 0
        assert differ(results(x=x * lost), 0)
        assert differ(results(one_part=True), 0)
    if n > 4000:
        lost = torch.ones(n).to(dtype)
        lost[256:320] = 0
        assert differ(results(dout=dout * lost), 1)
        assert differ(results(one_part=True), 1)


def test_scalings_by_their_definitions():
    """Each pair's frequency from wavelengths and from the places of the blend worked out by hand, apart from the
    implementation."""
    plain = [10000.0 ** (-i / 64) for i in range(64)]

    def same(got, want):
        assert len(got) == len(want) and all(abs(g / w - 1) < 1e-12 for g, w in zip(got, want))

    same(rotary_frequencies(128, 10000.0)[0], plain)
    same(rotary_frequencies(128, 10000.0, RotaryScaling("linear", 2.5))[0], [f / 2.5 for f in plain])
    # the last of 64 pairs is divided by the factor: base' ^ (-126/128) = base ^ (-126/128) / factor
    stretched = (10000.0 ** (126 / 128) * 8.0) ** (128 / 126)
    same(rotary_frequencies(128, 10000.0, RotaryScaling("ntk", 8.0))[0], [stretched ** (-i / 64) for i in range(64)])
    # by wavelength: below L / high as they are, above L / low divided, between them in turns
    for length, low, high, factor in ((8192, 1.0, 4.0, 8.0), (4096, 0.5, 16.0, 32.0)):
        want = []
        for f in plain:
            wave = 2 * math.pi / f
            share = 1.0 if wave < length / high else 0.0 if wave > length / low else (length / wave - low) / (high - low)
            want.append((1 - share) * f / factor + share * f)
        assert 0 < sum(w not in (f, f / factor) for w, f in zip(want, plain)) < 30
        same(rotary_frequencies(128, 10000.0, RotaryScaling("wavelength", factor, length, low=low, high=high))[0], want)
    # by index: 64 ln(4096 / 64 pi) / ln 10000 = 20.9, 64 ln(4096 / 2 pi) / ln 10000 = 45.03: whole up to pair 20, divided from 46
    # on, in 26 equal steps between
    got, magnitude = rotary_frequencies(128, 10000.0, RotaryScaling("yarn", 8.0, 4096))
    same(got, [f * (1 - min(max(i - 20, 0), 26) / 26 * (1 - 1 / 8)) for i, f in enumerate(plain)])
    assert abs(magnitude - 1.2079441541679836) < 1e-15
    # 16 of a head: 8 ln(1024 / 64 pi) / ln 500000 = 0.99, 8 ln(1024 / 2 pi) / ln 500000 = 3.1
    got, magnitude = rotary_frequencies(16, 500000.0, RotaryScaling("yarn", 4.0, 1024, magnitude=0.5))
    same(got, [500000.0 ** (-i / 8) * (1 - min(i, 4) / 4 * 0.75) for i in range(8)])
    assert magnitude == 0.5
