"""AdamW with moments in 8 bits, without a GPU: what the format's definition gives, what is refused, how the optimiser's Python face keeps its state."""
import ctypes as C
import math
import os
import sys
from array import array

import pytest

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import adamw_reference as ref  # noqa: E402

from cswap_amd import _lib  # noqa: E402
from cswap_amd.adamw8 import AdamW8, _dense_order, unpack_moments  # noqa: E402


@pytest.mark.parametrize("signed", [True, False])
def test_a_held_moment_is_within_a_code_of_its_value(signed):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(64 * 32, generator=g) * torch.exp(3 * torch.randn(64 * 32, generator=g)))
    x = x if signed else x.square()
    codes, scales = ref.pack(x, ref.offsets(x.numel(), 7, signed), signed)
    back = ref.unpack(codes, scales, x.numel(), signed)
    unit = ref.power(scales.int() - 127).repeat_interleave(32)
    step = (x.double().abs() + ref.least(signed) * unit) / 8             # a code's step is an eighth of its power of two, which is at most this
    assert bool(((back - x.double()).abs() <= step).all())
    assert int(codes.long().amax()) <= 248


@pytest.mark.parametrize("signed", [True, False])
def test_what_a_code_stands_for_is_held_as_that_code(signed):
    codes = torch.arange(0, 121 if signed else 248, dtype=torch.uint8)
    scales = torch.full((-(-codes.numel() // 32),), 120, dtype=torch.uint8)
    full = torch.nn.functional.pad(codes, (0, -codes.numel() % 32))
    # every group has its largest value, which sets the scale (code 248 of v stands for 2^7 - 2^-24, which is 2^7 in fp32: of the next scale)
    full[::32] = 120 if signed else 247
    values = ref.unpack(full, scales, full.numel(), signed).float()
    assert bool(torch.isfinite(values).all())
    for step in (1, 2, 1000):
        again, same = ref.pack(values, ref.offsets(values.numel(), step, signed), signed)
        assert torch.equal(same, scales) and torch.equal(again, full)    # nothing is cut off, so no offset carries


def test_over_the_steps_a_value_is_held_by_its_two_codes_in_proportion():
    """A value between two codes, held again and again: the mean of what it is held as is the value, to 1 / steps of a code's step."""
    x = torch.full((32,), 0.4)
    x[0] = 1.0
    total, steps = torch.zeros(32, dtype=torch.float64), 512
    for t in range(1, steps + 1):
        codes, scales = ref.pack(x, ref.offsets(32, t, False), False)
        total += ref.unpack(codes, scales, 32, False)
    # discrepancy of a Weyl sequence with a badly approximable factor: a few over the number of terms
    assert float((total / steps - x.double()).abs().amax()) <= 0.4 / 8 * 8 / steps


def test_a_second_moment_decays():
    """v' = 0.999 v moves by about a hundredth of a code's step, which rounding to nearest drops each time.  An offset that falls into that share
    of [0, 1) makes it fall by a code; the waits for one are between a third of the mean wait and three times it (a rotation's waits for an
    interval take three values, the longest the sum of the others), so after 1000 steps log v has fallen by 1/3 to 3, give or take a code."""
    v = torch.full((32,), 0.7)
    v[1:] = torch.linspace(0.05, 1.0, 31)
    factor = ref.single(torch.tensor(0.999, dtype=torch.float64))
    held, stuck = v.clone(), v.clone()
    for t in range(1, 1001):
        codes, scales = ref.pack(ref.single(held.double() * factor).float(), ref.offsets(32, t, False), False)
        held = ref.unpack(codes, scales, 32, False).float()
        codes, scales = ref.pack(ref.single(stuck.double() * factor).float(), ref.NEAREST, False)
        stuck = ref.unpack(codes, scales, 32, False).float()
    assert bool((held <= v * math.exp(-1 / 3) * 9 / 8).all()) and bool((held >= v * math.exp(-3) * 7 / 8).all())
    assert bool((stuck >= v * 15 / 16 * 15 / 16).all())


def table(**kw):
    row = dict(param=1 << 20, grad=1 << 20, m=1 << 20, v=1 << 20, master=0, n=32, dtype=0)
    row.update(kw)
    return array("Q", row.values())


GOOD = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0)


@pytest.mark.parametrize("row,bits,options,step,code", [
    ({}, 16, {}, 1, -1), ({}, 8, {}, 0, -1), ({"dtype": 3}, 8, {}, 1, -1), ({"param": 0}, 8, {}, 1, -1), ({"grad": 0}, 8, {}, 1, -1),
    ({"param": (1 << 20) + 2}, 32, {}, 1, -1), ({"m": 0}, 8, {}, 1, -1), ({"m": (1 << 20) + 4}, 8, {}, 1, -1), ({"v": (1 << 20) + 2}, 32, {}, 1, -1),
    ({"master": (1 << 20) + 2, "dtype": 1}, 32, {}, 1, -1), ({"n": (1 << 34) - 31}, 8, {}, 1, -2),
    ({}, 8, {"lr": -1.0}, 1, -1), ({}, 8, {"lr": math.nan}, 1, -1), ({}, 8, {"beta1": 1.0}, 1, -1), ({}, 8, {"beta2": -0.1}, 1, -1),
    ({}, 8, {"eps": 0.0}, 1, -1), ({}, 8, {"weight_decay": -1.0}, 1, -1), ({}, 8, {"lr": math.inf}, 1, -1)])
def test_argument_errors_do_not_launch(row, bits, options, step, code):
    t = table(**row)
    o = _lib.AdamwOptions(*{**GOOD, **options}.values())
    assert _lib.lib().cswap_adamw_step(t.buffer_info()[0], 1, bits, C.byref(o), step, None) == code


def test_argument_errors_of_the_other_calls_do_not_launch():
    L, o = _lib.lib(), _lib.AdamwOptions(*GOOD.values())
    t = table()
    at = t.buffer_info()[0]
    assert L.cswap_adamw_step(None, 1, 8, C.byref(o), 1, None) == -1
    assert L.cswap_adamw_step(at, 1, 8, None, 1, None) == -1
    assert L.cswap_adamw_step_counted(at, 1, 8, C.byref(o), None, None, 1 << 20, None) == -1
    assert L.cswap_adamw_step_counted(at, 1, 8, C.byref(o), (1 << 20) + 4, None, 1 << 20, None) == -1
    assert L.cswap_adamw_step_counted(at, 1, 8, C.byref(o), 1 << 20, (1 << 20) + 1, 1 << 20, None) == -1
    assert L.cswap_adamw_step_counted(at, 1, 8, C.byref(o), 1 << 20, None, None, None) == -1
    for f in (L.cswap_adamw_pack, L.cswap_adamw_unpack):
        assert f(None, 1, None) == -1
        for bad in ([0, 8, 8, 8, 1], [4, 2, 8, 8, 1], [4, 4, 0, 8, 1], [4, 4, 8, 12, 1]):
            row = array("Q", bad)
            assert f(row.buffer_info()[0], 1, None) == -1
        row = array("Q", [4, 4, 8, 8, 1 << 34])
        assert f(row.buffer_info()[0], 1, None) == -2
        assert f(None, 0, None) == 0
    empty = table(param=0, n=0)
    assert L.cswap_adamw_step(empty.buffer_info()[0], 1, 8, C.byref(o), 1, None) == 0       # a tensor of no values is no work
    assert L.cswap_adamw_step(None, 0, 8, C.byref(o), 1, None) == 0


def test_moment_bytes():
    L = _lib.lib()
    assert [L.cswap_adamw_moment_bytes(n) for n in (0, 1, 32, 33, 1000)] == [0, 33, 33, 66, 33 * 32]


@pytest.mark.parametrize("kw", [{"lr": -1.0}, {"betas": (1.0, 0.9)}, {"betas": (0.9, 1.5)}, {"eps": 0.0}, {"weight_decay": -1.0}, {"bits": 4},
                                {"lr": torch.tensor(1e-3)}, {"lr": torch.tensor(1e-3), "capturable": True}])
def test_options_are_refused(kw):
    with pytest.raises(ValueError):
        AdamW8([torch.nn.Parameter(torch.zeros(4))], **kw)
    with pytest.raises(ValueError):
        AdamW8([{"params": [torch.nn.Parameter(torch.zeros(4))], **kw}])


def test_types_and_places_are_refused():
    with pytest.raises(TypeError):
        AdamW8([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))])
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    optimizer = AdamW8([p])
    with pytest.raises(ValueError, match="device memory"):
        optimizer.step()
    assert torch.equal(p.detach(), torch.zeros(4))


def test_a_step_without_gradients_does_nothing():
    p = torch.nn.Parameter(torch.zeros(4))
    optimizer = AdamW8([p])
    assert optimizer.step(lambda: 3.0) == 3.0
    assert not optimizer.state and unpack_moments(optimizer) == []


def test_options_by_group_and_copies_of_an_optimiser():
    import copy

    a, b = (torch.nn.Parameter(torch.zeros(4)) for _ in range(2))
    optimizer = AdamW8([{"params": [a], "bits": 32, "lr": 1.0}, {"params": [b]}], lr=2.0)
    again = copy.deepcopy(optimizer)
    for o in (optimizer, again):
        assert [(g["bits"], g["lr"]) for g in o.param_groups] == [(32, 1.0), (8, 2.0)]
    saved = optimizer.state_dict()
    other = AdamW8([{"params": [a]}, {"params": [b], "bits": 32}])
    other.load_state_dict(saved)
    assert [(g["bits"], g["lr"]) for g in other.param_groups] == [(8, 1.0), (32, 2.0)]       # how it holds its state stays its own
    plain = torch.optim.AdamW([a], lr=0.5, amsgrad=True)
    with pytest.raises(ValueError, match="amsgrad"):
        AdamW8([a]).load_state_dict(plain.state_dict())


def test_which_layouts_fill_their_memory():
    t = torch.zeros(4, 6, 5, 3)
    assert _dense_order(t) and _dense_order(t.to(memory_format=torch.channels_last)) and _dense_order(t.permute(2, 0, 3, 1))
    assert _dense_order(torch.zeros(1, 5, 1)) and _dense_order(torch.zeros(())) and _dense_order(torch.zeros(3, 4).t())
    assert not _dense_order(t[:, :5]) and not _dense_order(t[..., ::2]) and not _dense_order(torch.zeros(4).expand(3, 4))


def test_a_parameter_twice_is_refused():
    a, b = (torch.nn.Parameter(torch.zeros(4)) for _ in range(2))
    for given in ([a, b, a], iter([a, b, a])):
        with pytest.raises(ValueError, match="twice"), pytest.warns(UserWarning, match="duplicate"):
            AdamW8(given)
    optimizer = AdamW8([a])
    with pytest.raises(ValueError):
        optimizer.add_param_group({"params": [a]})
    assert len(optimizer.param_groups) == 1


@pytest.mark.parametrize("kept", [{"step": 3}, {"exp_avg": torch.zeros(4), "exp_avg_sq": torch.zeros(4)},
                                  {"step": 3, "exp_avg": torch.zeros(4)}, {"step": 3, "exp_avg": [0.0] * 4, "exp_avg_sq": [0.0] * 4}])
def test_states_without_moments_are_refused(kept):
    a = torch.nn.Parameter(torch.zeros(4))
    optimizer = AdamW8([a], lr=0.5)
    saved = AdamW8([a]).state_dict()
    saved["state"] = {0: kept}
    with pytest.raises(ValueError, match="expected step"):
        optimizer.load_state_dict(saved)
    assert not optimizer.state and optimizer.param_groups[0]["lr"] == 0.5


def test_parameters_on_another_device_make_that_device_current(monkeypatch):
    import contextlib

    from cswap_amd import adamw8, api, q8

    current, launched = [0], []

    @contextlib.contextmanager
    def device(d):
        was, current[0] = current[0], d.index
        yield
        current[0] = was

    class OnDevice1(torch.Tensor):
        is_cuda = property(lambda self: True)
        device = property(lambda self: torch.device("cuda", 1))

    class Lib:
        cswap_adamw_moment_bytes = staticmethod(_lib.lib().cswap_adamw_moment_bytes)

        @staticmethod
        def cswap_adamw_step(*a):
            launched.append((current[0], a[1], a[4], a[-1]))
            return 0

    monkeypatch.setattr(q8, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(api, "_raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(adamw8, "lib", lambda: Lib)
    made = torch.zeros
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: made(*a, **kw).as_subclass(OnDevice1))
    p = torch.nn.Parameter(made(64).as_subclass(OnDevice1))
    p.grad = made(64).as_subclass(OnDevice1)
    optimizer = AdamW8([p])
    optimizer.step(), optimizer.step()
    assert launched == [(1, 1, 1, 1001), (1, 1, 2, 1001)] and current == [0]
