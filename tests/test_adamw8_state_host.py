"""AdamW8 and the state that its caller replaces, changes or clears, without a GPU: which step and which moments a launch is given."""
import ctypes as C
from collections import defaultdict

import pytest

torch = pytest.importorskip("torch")

from cswap_amd import _lib, adamw8, q8  # noqa: E402
from cswap_amd.adamw8 import AdamW8, unpack_moments  # noqa: E402


class OnDevice(torch.Tensor):
    is_cuda = property(lambda self: True)


@pytest.fixture
def launches(monkeypatch):
    """What the library's calls are given: of steps (number, [(param, exp_avg, exp_avg_sq, master)]), of conversions ("unpack", [codes of exp_avg])."""
    made = []

    def words(at, count, each):
        return [(C.c_uint64 * each).from_address(at + 8 * each * i)[:] for i in range(count)]

    class Lib:
        cswap_adamw_moment_bytes = staticmethod(_lib.lib().cswap_adamw_moment_bytes)
        cswap_adamw_factors_bytes = staticmethod(_lib.lib().cswap_adamw_factors_bytes)

        @staticmethod
        def cswap_adamw_step(table, count, bits, options, step, stream):
            made.append((step, [(p, m, v, master) for p, g, m, v, master, n, kind in words(table, count, 7)]))
            return 0

        @staticmethod
        def cswap_adamw_step_counted(table, count, bits, options, counter, lr, factors, stream):
            at = C.c_longlong.from_address(counter)
            at.value += 1
            return Lib.cswap_adamw_step(table, count, bits, options, at.value, stream)

        @staticmethod
        def cswap_adamw_unpack(table, count, stream):
            made.append(("unpack", [m8 for m, v, m8, v8, n in words(table, count, 5)]))
            return 0

        cswap_adamw_pack = cswap_adamw_unpack

    convert = adamw8._convert
    monkeypatch.setattr(adamw8, "lib", lambda: Lib)
    monkeypatch.setattr(adamw8, "_convert", lambda rows, name, device: convert(rows, name, 0))
    monkeypatch.setattr(q8, "_stream_of", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return made


def parameter(n, dtype=torch.float32):
    p = torch.nn.Parameter(torch.ones(n, dtype=dtype).as_subclass(OnDevice))
    p.grad = torch.ones(n, dtype=dtype).as_subclass(OnDevice)
    return p


def held(optimizer, *params):
    """A launch's rows of these parameters, from the optimiser's state."""
    return [(p.data_ptr(), *(optimizer.state[p][k].data_ptr() for k in ("exp_avg", "exp_avg_sq")),
             optimizer.state[p]["master"].data_ptr() if "master" in optimizer.state[p] else 0) for p in params]


def steps(optimizer, count):
    for _ in range(count):
        optimizer.step()


CLEARS = {"clear": lambda o: o.state.clear(), "another": lambda o: setattr(o, "state", defaultdict(dict)),
          "empty": lambda o: o.state.update({p: {} for p in o.state}), "pop": lambda o: [o.state.pop(p) for p in list(o.state)]}


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("how", sorted(CLEARS))
def test_a_state_that_was_cleared_begins_anew(launches, how, capturable):
    a, b = parameter(40), parameter(100, torch.bfloat16)
    optimizer = AdamW8([a, b], master=True, capturable=capturable)
    steps(optimizer, 6)
    b.data.fill_(3.0)
    CLEARS[how](optimizer)
    optimizer.step()
    assert launches[-1] == (1, held(optimizer, a, b)) and len(launches) == 7
    assert not any(optimizer.state[p][k].any() for p in (a, b) for k in ("exp_avg", "exp_avg_sq"))
    assert torch.equal(optimizer.state[b]["master"], torch.full((100,), 3.0))
    assert [int(s["step"]) for s in optimizer.state_dict()["state"].values()] == [1, 1]
    optimizer.step()
    assert launches[-1] == (2, held(optimizer, a, b))


@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_that_was_replaced_is_the_one_that_is_used(launches, bits):
    a, b = parameter(40), parameter(100)
    optimizer = AdamW8([a, b], bits=bits)
    steps(optimizer, 3)
    optimizer.state[a] = {k: v.clone() if isinstance(v, torch.Tensor) else 10 if k == "step" else v for k, v in optimizer.state[a].items()}
    if bits == 8:
        unpack_moments(optimizer)
        assert launches[-1] == ("unpack", [optimizer.state[p]["exp_avg"].data_ptr() for p in (a, b)])
    del launches[:]
    optimizer.step()
    assert launches == [(11, held(optimizer, a)), (4, held(optimizer, b))]
    assert [optimizer.state[p]["step"] for p in (a, b)] == [11, 4]


def test_a_step_that_was_set_is_the_one_that_is_counted_on(launches):
    a, b = parameter(40), parameter(100)
    optimizer = AdamW8([a, b])
    steps(optimizer, 3)
    for p in (a, b):
        optimizer.state[p]["step"] = 1000
    optimizer.step()
    assert launches[-1] == (1001, held(optimizer, a, b))
    optimizer.state[b]["step"] = 7
    del launches[:]
    optimizer.step()
    assert launches == [(1002, held(optimizer, a)), (8, held(optimizer, b))]
    optimizer.state[b]["step"] = torch.tensor(1002.0)               # as torch's optimisers count
    del launches[:]
    optimizer.step()
    assert launches == [(1003, held(optimizer, a, b))] and optimizer.state[b]["step"] == 1003


def test_a_counter_that_was_set_is_the_one_that_is_counted_on(launches):
    a, b = parameter(40), parameter(100)
    optimizer = AdamW8([a, b], capturable=True)
    steps(optimizer, 3)
    assert optimizer.state[a]["step"] is optimizer.state[b]["step"]
    optimizer.state[b]["step"] = torch.full((1,), 7)
    del launches[:]
    optimizer.step()
    assert launches == [(4, held(optimizer, a)), (8, held(optimizer, b))]
    for wrong in (torch.tensor(20.0), torch.tensor([20], dtype=torch.int32), 20):     # a float, or four bytes: no counter to count on in place
        optimizer.state[b]["step"] = wrong
        del launches[:]
        optimizer.step()
        assert launches[1] == (21, held(optimizer, b)), wrong
        assert optimizer.state[b]["step"].dtype is torch.int64 and int(optimizer.state[b]["step"]) == 21


def test_a_group_keeps_its_plan_while_another_changes(launches):
    a, b = parameter(40), parameter(100)
    optimizer = AdamW8([{"params": [a]}, {"params": [b], "bits": 32}])
    steps(optimizer, 2)
    del optimizer.state[b]
    del launches[:]
    optimizer.step()
    assert launches == [(3, held(optimizer, a)), (1, held(optimizer, b))]
    b.grad, kept = None, b.grad
    optimizer.step()
    b.grad = kept
    del launches[:]
    optimizer.step()
    assert launches == [(5, held(optimizer, a)), (2, held(optimizer, b))]


@pytest.mark.parametrize("bits,capturable", [(8, False), (8, True), (32, False)])
def test_autograd_is_told_what_a_step_writes(launches, bits, capturable):
    a, b, idle = parameter(40), parameter(100, torch.bfloat16), parameter(8)
    idle.grad = None
    optimizer = AdamW8([a, b, idle], bits=bits, master=True, capturable=capturable)
    optimizer.step()

    def versions():
        kept = [optimizer.state[p].get(k) for p in (a, b) for k in ("exp_avg", "exp_avg_sq", "master")]
        return [t._version for t in (a, b, *kept) if t is not None]

    was, others = versions(), [t._version for t in (idle, a.grad, b.grad)]
    optimizer.step()
    assert len(was) == 7 and all(now > then for now, then in zip(versions(), was))
    assert [t._version for t in (idle, a.grad, b.grad)] == others


def test_a_backward_pass_after_a_step_is_refused_as_after_torchs(launches):
    x = torch.ones(2, 4, requires_grad=True)
    w = torch.nn.Parameter(torch.ones(4, 4).as_subclass(OnDevice))
    for optimizer in (torch.optim.AdamW([w]), AdamW8([w])):
        y = (x @ w).sum()
        w.grad = torch.ones_like(w)
        optimizer.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.parametrize("bits", [8, 32])
def test_autograd_is_told_where_moments_are_unpacked_to(launches, bits):
    a, b = parameter(40), parameter(100)
    optimizer = AdamW8([a, b], bits=bits)
    optimizer.step()
    out = [[torch.zeros(p.shape) for _ in range(2)] for p in (a, b)]
    unpack_moments(optimizer, out)
    assert all(t._version == 1 for pair in out for t in pair)
    held8 = [optimizer.state[p][k]._version for p in (a, b) for k in ("exp_avg", "exp_avg_sq")]
    unpack_moments(optimizer)
    assert [optimizer.state[p][k]._version for p in (a, b) for k in ("exp_avg", "exp_avg_sq")] == held8


def test_steps_in_inference_mode(launches):
    a = parameter(40)
    optimizer = AdamW8([a])
    with torch.inference_mode():
        optimizer.step()
    was = a._version
    optimizer.step()                                # its moments are inference tensors, which have no version
    assert a._version > was and [s for s, _ in launches] == [1, 2]


@pytest.mark.parametrize("bits", [8, 32])
def test_moments_that_moved_are_written_where_they_are(launches, bits):
    """A program that takes its optimiser's state elsewhere and back through ``.data``: the tensors are the same ones, their memory is not."""
    a, b = parameter(40), parameter(100, torch.bfloat16)
    optimizer = AdamW8([a, b], bits=bits, master=True)
    optimizer.step()
    old = []
    for p, key in ((a, "exp_avg"), (a, "exp_avg_sq"), (b, "exp_avg"), (b, "exp_avg_sq"), (b, "master")):
        kept = optimizer.state[p][key]
        old.append(kept.data)                       # so that its place is not given out again
        kept.data = kept.data.clone()
        if bits == 8:
            unpack_moments(optimizer)
            assert launches[-1] == ("unpack", [optimizer.state[p]["exp_avg"].data_ptr() for p in (a, b)])
        optimizer.step()
        assert launches[-1][1] == held(optimizer, a, b), key
    assert launches[-1][0] == 6


def test_a_counter_that_moved_is_counted_on_where_it_is(launches):
    a = parameter(40)
    optimizer = AdamW8([a], capturable=True)
    steps(optimizer, 2)
    old, counter = optimizer.state[a]["step"].data, optimizer.state[a]["step"]
    counter.data = counter.data.clone()
    optimizer.step()
    assert int(counter) == 3 and int(old) == 2


class Numbered(OnDevice):
    def get_device(self):
        return 0


def test_what_lies_in_host_memory_is_refused_before_a_launch(launches):
    a, b = (torch.nn.Parameter(torch.ones(n).as_subclass(Numbered)) for n in (40, 100))
    a.grad, b.grad = (torch.ones(n).as_subclass(Numbered) for n in (40, 100))
    optimizer = AdamW8([a, b])
    optimizer.step()
    b.grad = torch.ones(100)                        # a gradient that stayed behind
    with pytest.raises(ValueError, match="gradient"):
        optimizer.step()
    b.grad = torch.ones(100).as_subclass(Numbered)
    other = torch.nn.Parameter(torch.ones(100))
    other.grad = torch.ones(100)
    host = AdamW8([other])
    host.state[other].update(optimizer.state[b])
    with pytest.raises(ValueError, match="device memory"):
        host.step()
    assert len(launches) == 1 and optimizer.state[a]["step"] == 1


def traced(call, p):
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(g):
        p.grad = g
        call()
        return g * 2

    return make_fx(f)(p.grad)


@pytest.mark.parametrize("name", ["step", "first_step", "unpack", "load"])
def test_traces_are_refused(launches, name):
    p = parameter(40)
    optimizer = AdamW8([p])
    if name != "first_step":
        optimizer.step()
    saved = optimizer.state_dict()
    call = {"step": optimizer.step, "first_step": optimizer.step, "unpack": lambda: unpack_moments(optimizer),
            "load": lambda: AdamW8([p], bits=32).load_state_dict(saved)}[name]
    count = len(launches)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        traced(call, p)
    p.grad = torch.ones(40).as_subclass(OnDevice)
    with pytest.raises(RuntimeError, match="cannot be traced" if name != "load" else "constant"):       # torch refuses what loading does before it converts
        torch.jit.trace(lambda g: (call(), g * 2)[1], torch.ones(40), check_trace=False)
    assert len(launches) == count and optimizer.state[p].get("step", 0) == (0 if name == "first_step" else 1)


def test_forward_mode_is_refused(launches):
    from torch.autograd import forward_ad

    p = parameter(40)
    optimizer = AdamW8([p])
    optimizer.step()
    with forward_ad.dual_level():
        optimizer.step()                                             # nothing here has a tangent
        p.grad = forward_ad.make_dual(torch.ones(40).as_subclass(OnDevice), torch.ones(40).as_subclass(OnDevice))
        with pytest.raises(RuntimeError, match="forward-mode"):
            optimizer.step()
    assert [s for s, _ in launches] == [1, 2]


def test_hooks_on_loading_are_heard(launches):
    """What a hook before loading gives back is what is loaded, and a hook after it sees the state as it then is."""
    a, b = parameter(40), parameter(100, torch.bfloat16)
    saved = {"state": {i: {"step": torch.tensor(5.0), "exp_avg": torch.full((n,), 1.0), "exp_avg_sq": torch.full((n,), 2.0)} for i, n in enumerate((40, 100))},
             "param_groups": torch.optim.AdamW([torch.nn.Parameter(torch.zeros(1)) for _ in range(2)], lr=0.25).state_dict()["param_groups"]}
    wrapped = {"optimizer": saved}
    optimizer = AdamW8([a, b], bits=32, master=True)
    seen = []
    hooks = [optimizer.register_load_state_dict_pre_hook(lambda o, given: given["optimizer"]),
             optimizer.register_load_state_dict_pre_hook(lambda o, given: {**given, "state": {i: {**s, "exp_avg": s["exp_avg"] * 3} for i, s in given["state"].items()}}),
             optimizer.register_load_state_dict_post_hook(lambda o: seen.append([(type(s["step"]), s["exp_avg"].dtype, float(s["exp_avg"][0])) for s in o.state.values()]))]
    optimizer.load_state_dict(wrapped)
    assert seen == [[(int, torch.float32, 3.0)] * 2]
    for p in (a, b):
        s = optimizer.state[p]
        assert s["step"] == 5 and bool((s["exp_avg"] == 3).all()) and bool((s["exp_avg_sq"] == 2).all()) and s["exp_avg"].dtype is torch.float32
    assert optimizer.param_groups[0]["lr"] == 0.25 and optimizer.param_groups[0]["bits"] == 32
    assert torch.equal(optimizer.state[b]["master"], torch.ones(100)) and float(saved["state"][0]["exp_avg"][0]) == 1.0
    # a hook may change what it is given in place; what it gives is checked as what a caller gives
    for hook in hooks:
        hook.remove()
    first = optimizer.register_load_state_dict_pre_hook(lambda o, given: given["param_groups"][0].update(amsgrad=True))
    with pytest.raises(ValueError, match="amsgrad"):
        optimizer.load_state_dict(saved)
    first.remove()
    saved["param_groups"][0]["amsgrad"] = False
    optimizer.load_state_dict(saved)
    optimizer.load_state_dict(optimizer.state_dict())
    assert len(seen) == 1 and optimizer.state[a]["step"] == 5


def test_hooks_on_loading_are_the_callers_alone_after_it(launches):
    a = parameter(40)
    optimizer = AdamW8([a])
    optimizer.step()
    saved = optimizer.state_dict()
    for given in (saved, {**saved, "param_groups": []}):
        try:
            optimizer.load_state_dict(given)
        except ValueError:
            assert given is not saved
    other = torch.optim.Optimizer.load_state_dict
    del optimizer.state[a]
    other(optimizer, saved)                                          # torch's own, with nothing of ours left behind
    assert optimizer.state[a]["exp_avg"].dtype is torch.float32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loading_moments_of_8_bits_makes_them_in_no_other_type(launches, dtype):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Made(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if isinstance(out, torch.Tensor):
                made.append((out.dtype, out.numel()))
            return out

    a, b, made = parameter(4000, dtype), parameter(7000, dtype), []
    optimizer = AdamW8([a, b])
    optimizer.step()
    for i, p in enumerate((a, b)):
        optimizer.state[p]["exp_avg"].fill_(i + 1), optimizer.state[p]["exp_avg_sq"].fill_(i + 10)
    saved = optimizer.state_dict()
    other = AdamW8([a, b])
    with Made():
        other.load_state_dict(saved)
    assert made and all(kind is torch.uint8 for kind, n in made if n >= 4000), made
    for p in (a, b):
        for key in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(other.state[p][key], optimizer.state[p][key]) and other.state[p][key] is not optimizer.state[p][key]
    # what belongs to no parameter is handed on as torch hands it on
    saved["state"]["extra"] = {}
    other.load_state_dict(saved)
    assert other.state["extra"] == {} and other.state[a]["step"] == 1


@pytest.mark.parametrize("lr", [torch.tensor(0.25), torch.tensor(0.25, dtype=torch.float64), 0.25])
def test_options_that_torchs_optimiser_holds_as_tensors_are_loaded(launches, lr):
    """``torch.optim.AdamW`` may count and hold its learning rate on the device; a loaded one goes on as its own ``capturable`` says."""
    a = parameter(40)
    plain = torch.optim.AdamW([torch.nn.Parameter(torch.ones(40))], lr=0.5)
    saved = plain.state_dict()
    saved["state"][0] = {"step": torch.tensor(3.0), "exp_avg": torch.ones(40), "exp_avg_sq": torch.ones(40)}
    saved["param_groups"][0].update(lr=lr, capturable=True)
    optimizer = AdamW8([a], bits=32)
    optimizer.load_state_dict(saved)
    group = optimizer.param_groups[0]
    assert type(group["lr"]) is float and group["lr"] == 0.25 and group["capturable"] is False
    optimizer.step()
    assert launches == [(4, held(optimizer, a))]
    counted = AdamW8([a], bits=32, capturable=True)
    counted.load_state_dict(saved)
    given = counted.param_groups[0]["lr"]
    if isinstance(lr, torch.Tensor):
        assert given.dtype is torch.float32 and float(given) == 0.25 and given.device == a.device and given is not lr
    else:
        assert given == 0.25
