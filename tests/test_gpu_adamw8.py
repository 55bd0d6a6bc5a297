"""AdamW over many tensors on the GPU: moments to the byte against tests/adamw_reference.py, parameters within the bound that its roundings give."""
import copy
import math
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import adamw_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
BETAS, EPS = (0.9, 0.999), 1e-8


def mod():
    from cswap_amd import adamw8

    return adamw8


def bound(p, size, dtype, steps=1):
    """What the kernel's p' may be off by.  The change goes through the root (2^-23), its factor and the sum with eps (2^-24 each, eps itself
    2^-24), the reciprocal (2^-23), two products and the factor lr / (1 - b1^t) (2^-24 each): 11 * 2^-24 of it; p (1 - lr wd) is two roundings
    off; the sum is rounded once, and once to its type.  m' and v' have the reference's bits, or (held in fp32 over several steps) their own."""
    return steps * (12 * 2.0 ** -24 * size + p.abs() * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype is F16 else 2.0 ** -149))


def gradient(shape, dtype, seed, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * torch.exp(torch.randn(shape, generator=g)) * scale).to(dtype)


class Model:
    """Parameters on the GPU and their step by the definition, on the CPU."""

    def __init__(self, shapes, dtypes, bits, master=False, **kw):
        self.kw = dict(lr=1e-2, weight_decay=0.1, **kw)
        self.bits = bits
        self.p = [gradient(s, d, 100 + i, 0.5) for i, (s, d) in enumerate(zip(shapes, dtypes))]
        self.params = [torch.nn.Parameter(p.clone().cuda()) for p in self.p]
        self.optimizer = mod().AdamW8(self.params, betas=BETAS, eps=EPS, bits=bits, master=master, **self.kw)
        self.m = [torch.zeros(p.numel()) for p in self.p]
        self.v = [torch.zeros(p.numel()) for p in self.p]
        self.t = 0

    def step(self, grads, check=True):
        self.t += 1
        before = [(s["master"] if "master" in (s := self.optimizer.state.get(p, {})) else p.detach()).cpu().clone() for p in self.params]
        for p, g in zip(self.params, grads):
            p.grad = g.cuda()
        self.optimizer.step()
        for k, (p, g) in enumerate(zip(self.params, grads)):
            n, s = g.numel(), self.optimizer.state[p]
            m, v = ref.moments(self.m[k], self.v[k], g.reshape(-1), BETAS)
            if self.bits == 8:
                mh, vh = ref.pack_pair(m.float(), v.float(), ref.offsets(n, self.t, True), ref.offsets(n, self.t, False))
                assert torch.equal(s["exp_avg"].cpu(), ref.room(*mh)), k
                assert torch.equal(s["exp_avg_sq"].cpu(), ref.room(*vh)), k
                self.m[k], self.v[k] = ref.unpack(*mh, n, True).float(), ref.unpack(*vh, n, False).float()
            else:
                self.m[k], self.v[k] = m.float(), v.float()
                assert torch.equal(s["exp_avg"].cpu().reshape(-1), self.m[k]) and torch.equal(s["exp_avg_sq"].cpu().reshape(-1), self.v[k])
            want, size = ref.update(before[k].reshape(-1).double(), m, v, self.t, self.kw["lr"], BETAS, EPS, self.kw["weight_decay"])
            if check:
                got = s.get("master", p).detach().cpu().reshape(-1)
                assert bool(((got.double() - want).abs() <= bound(want, size, got.dtype)).all()), k
                if "master" in s:
                    assert torch.equal(p.detach().cpu(), s["master"].cpu().to(p.dtype))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_steps_of_tensors_of_any_size(dtype, bits):
    shapes = [(1,), (7,), (31,), (32,), (33,), (8, 4), (3, 5, 7), (2047,), (2048,), (2049,), (193, 65), ()]
    model = Model(shapes, [dtype] * len(shapes), bits)
    for t in range(4):
        model.step([gradient(s, dtype, 10 * t + i) for i, s in enumerate(shapes)])


@pytest.mark.parametrize("bits,master", [(8, False), (8, True), (32, True)])
def test_more_tensors_than_a_launch_takes_of_all_types(bits, master):
    count = 150
    shapes = [(1 + 37 * i % 500,) for i in range(count)]
    dtypes = [(F32, BF16, F16)[i % 3] for i in range(count)]
    model = Model(shapes, dtypes, bits, master)
    for t in range(2):
        model.step([gradient(s, d, 1000 * t + i) for i, (s, d) in enumerate(zip(shapes, dtypes))])
    assert all(("master" in model.optimizer.state[p]) == (master and p.dtype is not F32) for p in model.params)


def test_master_copies_gather_steps_below_the_last_place():
    for master in (False, True):
        p = torch.nn.Parameter(torch.ones(64, dtype=BF16).cuda())
        optimizer = mod().AdamW8([p], lr=1e-4, weight_decay=0.0, master=master)
        p.grad = torch.ones_like(p)
        for _ in range(100):
            optimizer.step()
        # each step is 1e-4, a bf16 one's step below 1 2^-8: 2^-9 is half of it
        assert float(p.detach()[0]) == (1.0 if not master else float(torch.tensor(0.99).to(BF16)))


@pytest.mark.parametrize("bits", [8, 32])
def test_values_at_the_ends_of_the_range(bits):
    fi = torch.finfo(F32)
    rows = [[0.0] * 32, [1e-30] * 32, [1e-20, 1e-21] * 16, [1e18] * 32, [-1e18, 1e-3] * 16, [1.0] + [2.0 ** -k for k in range(1, 32)],
            [-1.0] + [-(2.0 ** -(k + 16)) for k in range(1, 32)], [0.0, -0.0] * 16, [fi.tiny, -fi.tiny] * 16]
    g = torch.tensor(rows).reshape(-1)
    model = Model([(len(rows) * 32,)], [F32], bits)
    model.step([g])
    model.step([torch.zeros_like(g)])
    model.step([-g])
    assert bool(torch.isfinite(model.params[0]).all())


def test_a_gradient_that_is_not_finite_reaches_its_group_alone():
    p = torch.nn.Parameter(torch.ones(100).cuda())
    optimizer = mod().AdamW8([p], lr=0.1)
    p.grad = torch.full_like(p, 0.5)
    p.grad[40], p.grad[99] = math.nan, math.inf
    optimizer.step()
    at = torch.zeros(100, dtype=torch.bool)
    at[[40, 99]] = True
    assert torch.equal(torch.isnan(p.detach()).cpu(), at)            # in the step itself the element alone
    (m, v), = mod().unpack_moments(optimizer)
    bad = torch.zeros(100, dtype=torch.bool)
    bad[32:64] = bad[96:] = True
    assert torch.equal(torch.isnan(m).cpu(), bad) and torch.equal(torch.isnan(v).cpu(), bad)
    s = optimizer.state[p]
    assert s["exp_avg"][32:64].eq(0).all() and s["exp_avg"][96:128].eq(0).all()
    p32 = torch.nn.Parameter(torch.ones(100).cuda())
    o32 = mod().AdamW8([p32], lr=0.1, bits=32)
    p32.grad = p.grad
    o32.step()
    o32.step()
    assert torch.equal(torch.isnan(p32.detach()).cpu(), at)


def test_a_first_moment_without_a_second_is_dropped():
    """A neighbour 2^17 times as large: v's code is 0 there, m's would not be."""
    g = torch.full((32,), 2.0 ** -17)
    g[0] = 1.0
    model = Model([(32,)], [F32], 8)
    for t in range(1, 30):
        model.step([g])
        codes, _ = ref.split(model.optimizer.state[model.params[0]]["exp_avg"].cpu(), 32)
        second, _ = ref.split(model.optimizer.state[model.params[0]]["exp_avg_sq"].cpu(), 32)
        assert bool((codes[second == 0] == 0).all())
    # and what was dropped costs no more than a step of the learning rate's size, whatever the neighbour's size
    model.step([torch.zeros(32)])


@pytest.mark.parametrize("bits", [8, 32])
def test_parameters_and_gradients_of_other_layouts(bits):
    w = gradient((8, 6, 3, 3), F32, 1, 0.5)
    g = gradient((8, 6, 3, 3), F32, 2)
    results = []
    for layout in (torch.contiguous_format, torch.channels_last):
        for g_layout in (torch.contiguous_format, torch.channels_last):
            p = torch.nn.Parameter(w.clone().to(memory_format=layout).cuda())
            p.grad = g.to(memory_format=g_layout).cuda()
            optimizer = mod().AdamW8([p], bits=bits)
            optimizer.step()
            optimizer.step()
            (m, v), = mod().unpack_moments(optimizer)
            assert m.stride() == p.stride()
            results.append((layout, p.detach().cpu(), m.cpu(), v.cpu()))
    for layout, *values in results:
        same = results[0 if layout is torch.contiguous_format or bits == 32 else 2]
        assert all(torch.equal(a, b) for a, b in zip(values, same[1:]))


def test_views_that_start_at_any_element():
    flat = torch.zeros(4000, dtype=BF16).cuda()
    guard = flat.clone()
    starts = [1, 104, 1003, 2501]
    sizes = [100, 777, 1400, 1499]
    params = []
    for s, n in zip(starts, sizes):
        p = torch.nn.Parameter(flat[s:s + n])
        p.grad = gradient((n + 1,), BF16, n).cuda()[1:]
        params.append(p)
    single = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(params, single):
        q.grad = p.grad.clone()
    a, b = mod().AdamW8(params), mod().AdamW8(single)
    for _ in range(2):
        a.step(), b.step()
    for p, q in zip(params, single):
        assert torch.equal(p.detach(), q.detach())
        assert torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])
    there = torch.zeros(4000, dtype=torch.bool)
    for s, n in zip(starts, sizes):
        there[s:s + n] = True
    assert torch.equal(flat.cpu()[~there], guard.cpu()[~there])       # what lies between is left alone


def test_parameters_that_have_no_gradient_in_a_step_keep_their_count():
    a, b = (torch.nn.Parameter(torch.ones(40).cuda()) for _ in range(2))
    optimizer = mod().AdamW8([a, b], lr=0.1)
    plain = torch.nn.Parameter(torch.ones(40).cuda())
    other = mod().AdamW8([plain], lr=0.1)
    for t in range(5):
        a.grad = torch.full_like(a, 0.1 * (t + 1))
        b.grad = torch.full_like(b, 0.3) if t in (1, 2, 4) else None
        before = b.detach().clone()
        optimizer.step()
        if b.grad is None:
            assert torch.equal(b.detach(), before)
        else:
            plain.grad = b.grad
            other.step()
    assert optimizer.state[a]["step"] == 5 and optimizer.state[b]["step"] == 3
    assert torch.equal(b.detach(), plain.detach())


@pytest.mark.parametrize("bits", [8, 32])
def test_state_dicts_go_on_where_they_stopped(bits):
    shapes, dtypes = [(40,), (3, 50), (1,)], [F32, BF16, F16]
    first = Model(shapes, dtypes, bits, True)
    for t in range(3):
        first.step([gradient(s, d, 7 * t + i) for i, (s, d) in enumerate(zip(shapes, dtypes))])
    saved = copy.deepcopy(first.optimizer.state_dict())
    params = [torch.nn.Parameter(p.detach().clone()) for p in first.params]
    again = mod().AdamW8(params, bits=bits, master=True)
    again.load_state_dict(saved)
    grads = [gradient(s, d, 99 + i) for i, (s, d) in enumerate(zip(shapes, dtypes))]
    for p, g in zip(params, grads):
        p.grad = g.cuda()
    again.step()
    first.step(grads)
    for p, q in zip(params, first.params):
        assert torch.equal(p.detach(), q.detach())
        for key in ("exp_avg", "exp_avg_sq", "master"):
            assert key not in again.state[p] or torch.equal(again.state[p][key], first.optimizer.state[q][key])
        assert again.state[p]["step"] == 4


def test_states_of_torchs_own_optimiser_are_taken_and_other_widths():
    w = gradient((6, 40, 3), F32, 5, 0.5)
    p = torch.nn.Parameter(w.clone().cuda())
    plain = torch.optim.AdamW([p], lr=1e-2, weight_decay=0.1)
    for t in range(3):
        p.grad = gradient((6, 40, 3), F32, t).cuda()
        plain.step()
    m, v = (plain.state[p][k].detach().cpu().reshape(-1) for k in ("exp_avg", "exp_avg_sq"))
    q = torch.nn.Parameter(p.detach().clone())
    small = mod().AdamW8([q])
    small.load_state_dict(plain.state_dict())
    assert small.state[q]["step"] == 3 and small.param_groups[0]["lr"] == 1e-2
    mh, vh = ref.pack_pair(m, v, ref.NEAREST, ref.NEAREST)
    assert torch.equal(small.state[q]["exp_avg"].cpu(), ref.room(*mh)) and torch.equal(small.state[q]["exp_avg_sq"].cpu(), ref.room(*vh))
    wide = mod().AdamW8([q], bits=32)
    wide.load_state_dict(small.state_dict())
    assert torch.equal(wide.state[q]["exp_avg"].cpu().reshape(-1), ref.unpack(*mh, m.numel(), True).float())
    assert torch.equal(wide.state[q]["exp_avg_sq"].cpu().reshape(-1), ref.unpack(*vh, m.numel(), False).float())
    # a parameter of another layout: the values are the same ones
    last = torch.nn.Parameter(p.detach().view(6, 40, 3, 1).permute(0, 2, 3, 1))     # [6, 3, 1, 40], channels first in memory
    saved = small.state_dict()
    saved["state"][0] = {**saved["state"][0], "strides": (120, 1, 3, 3)}
    moved = torch.nn.Parameter(p.detach().view(6, 40, 3).permute(0, 2, 1).contiguous().view(6, 3, 1, 40))
    assert last.shape == moved.shape
    saved["state"][0]["strides"] = last.stride()
    other = mod().AdamW8([moved], bits=32)
    other.load_state_dict(saved)
    assert torch.equal(other.state[moved]["exp_avg"].cpu().view(6, 3, 40).permute(0, 2, 1).reshape(-1), ref.unpack(*mh, m.numel(), True).float())


def test_a_captured_step_counts_on():
    lr = torch.tensor(0.05).cuda()
    params = [torch.nn.Parameter(gradient((n,), d, n, 0.5).cuda()) for n, d in ((100, F32), (3000, BF16))]
    eager = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(params, eager):
        p.grad = torch.zeros_like(p)
        q.grad = torch.zeros_like(q)
    optimizer = mod().AdamW8(params, lr=lr, capturable=True)
    other = mod().AdamW8(eager, lr=0.05)

    def gradients(t):
        for i, (p, q) in enumerate(zip(params, eager)):
            g = gradient(p.shape, p.dtype, 10 * t + i).cuda()
            p.grad.copy_(g), q.grad.copy_(g)

    gradients(0)
    optimizer.step(), other.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        optimizer.step()
    for t in range(1, 6):
        gradients(t)
        if t == 3:
            lr.fill_(0.01)
            other.param_groups[0]["lr"] = float(lr)
        graph.replay()
        torch.cuda.synchronize()
        other.step()
        for p, q in zip(params, eager):
            assert int(optimizer.state[p]["step"]) == t + 1
            assert torch.equal(optimizer.state[p]["exp_avg"], other.state[q]["exp_avg"])
            assert torch.equal(optimizer.state[p]["exp_avg_sq"], other.state[q]["exp_avg_sq"])
            # lr comes from fp32 and the powers from the device's pow: the factors may differ in the last place
            scale = q.detach().double().abs() + 4 * 0.05
            assert bool(((p.detach().double() - q.detach().double()).abs() <= (t + 1) * (2.0 ** -20 + torch.finfo(p.dtype).eps) * scale).all())
    torch.randn(1000, device="cuda").sum().item()


def test_captures_that_would_go_wrong_are_refused():
    a, b = (torch.nn.Parameter(torch.ones(40).cuda()) for _ in range(2))
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    plain, first = mod().AdamW8([a]), mod().AdamW8([b], capturable=True)
    plain.step()
    for optimizer, text in ((plain, "capturable"), (first, "first step")):
        with pytest.raises(RuntimeError, match=text):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                optimizer.step()
    torch.cuda.synchronize()
    both = mod().AdamW8([a, b], capturable=True)
    both.step()
    b.grad = None
    with pytest.raises(RuntimeError, match="shares the count"):
        both.step()
    assert int(both.state[a]["step"]) == 1


def test_another_stream_and_gradients_of_each_step():
    p = torch.nn.Parameter(gradient((5000,), BF16, 1, 0.5).cuda())
    q = torch.nn.Parameter(p.detach().clone())
    a, b = mod().AdamW8([p]), mod().AdamW8([q])
    side = torch.cuda.Stream()
    for t in range(3):
        g = gradient((5000,), BF16, t).cuda()
        p.grad = g
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a.step()
        torch.cuda.current_stream().wait_stream(side)
        q.grad = g.clone()
        b.step()
    assert torch.equal(p.detach(), q.detach()) and torch.equal(a.state[p]["exp_avg_sq"], b.state[q]["exp_avg_sq"])


def test_what_changes_under_the_optimiser_is_seen():
    p = torch.nn.Parameter(torch.ones(64).cuda())
    p.grad = torch.ones_like(p)
    optimizer = mod().AdamW8([p], lr=0.1)
    optimizer.step()
    old = p.detach()
    p.data = torch.full((64,), 5.0).cuda()                      # other memory
    optimizer.step()
    assert float(old[0]) > 0.8 and float(p.detach()[0]) < 5.0
    optimizer.state[p]["exp_avg"] = optimizer.state[p]["exp_avg"][:33]
    with pytest.raises(ValueError, match="moment"):
        optimizer.step()
    optimizer.state[p]["exp_avg"] = torch.zeros(66, dtype=torch.uint8).cuda()
    optimizer.step()
    w = torch.nn.Parameter(torch.ones(2, 4, 3, 3).cuda())
    w.grad = torch.ones_like(w)
    optimizer = mod().AdamW8([w])
    optimizer.step()
    w.data = w.data.to(memory_format=torch.channels_last)
    with pytest.raises(RuntimeError, match="strides"):
        optimizer.step()
    gap = torch.nn.Parameter(torch.ones(4, 8).cuda()[:, :6])
    gap.grad = torch.ones_like(gap)
    with pytest.raises(ValueError, match="fill"):
        mod().AdamW8([gap]).step()
    e = torch.nn.Embedding(10, 4, sparse=True).cuda()
    e(torch.tensor([1]).cuda()).sum().backward()
    with pytest.raises(RuntimeError, match="sparse"):
        mod().AdamW8(e.parameters()).step()


def test_a_tensor_beyond_32_bits_of_values():
    """Element numbers wrap in the offsets, and in nothing else."""
    n = (1 << 32) + 40
    p = torch.nn.Parameter(torch.zeros(n, dtype=BF16, device="cuda"))
    p.grad = torch.zeros_like(p)
    tail = gradient((104,), BF16, 3)
    p.grad[n - 104:] = tail.cuda()
    optimizer = mod().AdamW8([p], lr=0.5, weight_decay=0.0)
    optimizer.step()
    m, v = ref.moments(torch.zeros(104), torch.zeros(104), tail, BETAS)
    at = (torch.arange(128, dtype=torch.int64) + n - 104) % (1 << 32)
    mh, vh = ref.pack_pair(m.float(), v.float(), (at * ref.A + ref.B) % (1 << 32), (at * ref.B + ref.A) % (1 << 32))
    groups = -(-n // 32)
    for key, (codes, scales) in (("exp_avg", mh), ("exp_avg_sq", vh)):
        held = optimizer.state[p][key]
        assert torch.equal(held[groups * 32 - 128:groups * 32].cpu(), codes) and torch.equal(held[-4:].cpu(), scales)
        assert not held[:groups * 32 - 128].any()
    assert bool(p.detach()[n - 104:].ne(0).all()) and not bool(p.detach()[:n - 104].any())


def test_options_that_change_under_way():
    p = torch.nn.Parameter(torch.ones(200).cuda())
    p.grad = torch.ones_like(p)
    optimizer = mod().AdamW8([p], lr=0.1)
    optimizer.step()
    optimizer.param_groups[0]["bits"] = 32                     # moments that are there are not read as what they are not
    with pytest.raises(ValueError, match="moment"):
        optimizer.step()
    optimizer.param_groups[0]["bits"] = 8
    optimizer.param_groups[0]["capturable"] = True
    optimizer.step()
    assert int(optimizer.state[p]["step"]) == 2 and optimizer.state[p]["step"].is_cuda
    optimizer.param_groups[0]["capturable"] = False
    optimizer.step()
    assert optimizer.state[p]["step"] == 3 and isinstance(optimizer.state[p]["step"], int)
    square = torch.nn.Parameter(torch.ones(64, 64).cuda())
    square.grad = torch.ones_like(square)
    optimizer = mod().AdamW8([square], bits=32)
    optimizer.step()
    square.data = square.data[:32]                             # at the same place, fewer values
    with pytest.raises((TypeError, ValueError)):
        optimizer.step()


# ---------------------------------------------------------------- what no other test calls
def test_groups_that_were_loaded_at_one_step_count_apart():
    """Each group's launch counts its own steps on: a counter of two groups would count twice."""
    params = [torch.nn.Parameter(gradient((n,), F32, n, 0.5).cuda()) for n in (100, 200)]
    first = mod().AdamW8([{"params": [p]} for p in params], capturable=True)
    for p in params:
        p.grad = torch.ones_like(p)
    first.step()
    again = mod().AdamW8([{"params": [p]} for p in params], capturable=True)
    again.load_state_dict(copy.deepcopy(first.state_dict()))
    again.step()
    assert [int(again.state[p]["step"]) for p in params] == [2, 2]
    again.step()
    assert [int(again.state[p]["step"]) for p in params] == [3, 3]


def test_what_one_group_refuses_is_refused_before_a_step_of_another():
    a = torch.nn.Parameter(torch.ones(40).cuda())
    gap = torch.nn.Parameter(torch.ones(4, 8).cuda()[:, :6])
    e = torch.nn.Embedding(10, 4, sparse=True).cuda()
    e(torch.tensor([1]).cuda()).sum().backward()
    gap.grad = torch.ones_like(gap)
    for bad, error in ((gap, ValueError), (e.weight, RuntimeError)):
        a.grad = torch.ones_like(a)
        optimizer = mod().AdamW8([{"params": [a]}, {"params": [bad]}])
        with pytest.raises(error):
            optimizer.step()
        assert bool((a.detach() == 1).all()) and optimizer.state[a].get("step", 0) == 0 and not optimizer.state[a]["exp_avg"].any()


def test_parameters_that_share_memory_are_refused():
    room = torch.zeros(100).cuda()
    a, b, c = torch.nn.Parameter(room[:64]), torch.nn.Parameter(room[63:80]), torch.nn.Parameter(room[80:])
    for p in (a, b, c):
        p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match="share memory"):
        mod().AdamW8([a, c, b]).step()
    assert not room.any()
    mod().AdamW8([b, c]).step()                                  # next to each other
    assert bool(room[63:].ne(0).all())


def test_a_parameter_that_no_longer_fills_its_memory_is_refused():
    room = torch.ones(8, 8).cuda()
    p = torch.nn.Parameter(room.clone())
    p.grad = torch.ones_like(p)
    optimizer = mod().AdamW8([p], bits=32)
    optimizer.step()
    s, wide = optimizer.state[p], torch.ones(8, 9).cuda()
    p.data = wide[:, :8]
    p.grad = torch.ones_like(p)
    for k in ("exp_avg", "exp_avg_sq"):
        s[k] = torch.zeros(8, 9).cuda()[:, :8]
    with pytest.raises(ValueError, match="fill"):
        optimizer.step()
    assert bool((wide == 1).all())


def test_capturable_set_within_a_capture_is_refused():
    p = torch.nn.Parameter(torch.ones(40).cuda())
    p.grad = torch.ones_like(p)
    optimizer = mod().AdamW8([p])
    optimizer.step()
    optimizer.param_groups[0]["capturable"] = True
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            optimizer.step()
    torch.cuda.synchronize()
    optimizer.step()
    assert int(optimizer.state[p]["step"]) == 2


def test_master_set_within_a_capture_is_refused():
    p = torch.nn.Parameter(torch.ones(40).cuda().to(BF16))
    p.grad = torch.ones_like(p)
    optimizer = mod().AdamW8([p], capturable=True)
    optimizer.step()
    optimizer.param_groups[0]["master"] = True
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            optimizer.step()
    torch.cuda.synchronize()
    optimizer.step()
    assert int(optimizer.state[p]["step"]) == 2 and "master" in optimizer.state[p]


def test_master_copies_that_are_asked_for_and_given_up_under_way():
    p = torch.nn.Parameter(torch.ones(300).cuda().to(BF16))
    optimizer = mod().AdamW8([p], lr=2.0 ** -12, weight_decay=0.0)
    group = optimizer.param_groups[0]

    def steps(count):
        for _ in range(count):
            p.grad = torch.ones_like(p)
            optimizer.step()

    steps(4)
    assert bool((p.detach() == 1).all()) and "master" not in optimizer.state[p]      # below bf16's last place
    group["master"] = True
    steps(20)                                                                        # 20 of 2^-12: 1.25 of 2^-8
    assert optimizer.state[p]["master"].dtype is F32 and bool((p.detach() < 1).all())
    at = p.detach().clone()
    group["master"] = False
    steps(1)
    assert "master" not in optimizer.state[p] and torch.equal(p.detach(), at)


def test_two_captured_steps_of_two_optimisers():
    """Two graphs, replayed in turn and on two streams: each has its counter and its factors."""
    makes = [torch.nn.Parameter(gradient((n,), d, n, 0.5).cuda()) for n, d in ((5000, F32), (700, BF16))]
    eager = [torch.nn.Parameter(p.detach().clone()) for p in makes]
    optimizers = [mod().AdamW8([p], lr=0.01 * (i + 1), capturable=True) for i, p in enumerate(makes)]
    others = [mod().AdamW8([p], lr=0.01 * (i + 1), capturable=True) for i, p in enumerate(eager)]
    for i, (p, q) in enumerate(zip(makes, eager)):
        p.grad = gradient(p.shape, p.dtype, i).cuda()
        q.grad = p.grad.clone()
    graphs, streams = [], []
    for optimizer in optimizers:
        optimizer.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            optimizer.step()
        graphs.append(graph), streams.append(torch.cuda.Stream())
    torch.cuda.synchronize()
    for t in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        torch.randn(1000, device="cuda").sum().item()
    for other in others:
        for _ in range(5):
            other.step()
    for p, q, a, b in zip(makes, eager, optimizers, others):
        assert int(a.state[p]["step"]) == int(b.state[q]["step"]) == 5
        assert torch.equal(p.detach(), q.detach()) and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])


@pytest.mark.parametrize("bits", [8, 32])
def test_an_optimiser_whose_state_was_cleared_is_a_new_one(bits):
    shapes, dtypes = [(40,), (300,), (7, 9)], [F32, BF16, F16]
    model = Model(shapes, dtypes, bits, True)
    for t in range(3):
        model.step([gradient(s, d, 10 * t + i) for i, (s, d) in enumerate(zip(shapes, dtypes))])
    model.optimizer.state.clear()
    params = [torch.nn.Parameter(p.detach().clone()) for p in model.params]
    fresh = mod().AdamW8(params, betas=BETAS, eps=EPS, bits=bits, master=True, **model.kw)
    for t in range(2):
        for i, (p, q) in enumerate(zip(params, model.params)):
            p.grad = gradient(p.shape, p.dtype, 50 * t + i).cuda()
            q.grad = p.grad.clone()
        fresh.step(), model.optimizer.step()
    a, b = fresh.state_dict()["state"], model.optimizer.state_dict()["state"]
    for i, (p, q) in enumerate(zip(params, model.params)):
        assert torch.equal(p.detach(), q.detach()) and a[i]["step"] == b[i]["step"] == 2
        for key in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(a[i][key], b[i][key])


def test_a_backward_pass_through_weights_that_a_step_has_moved_is_refused():
    from cswap_amd import hooks, layers8

    x = torch.randn(64, 32, device="cuda", requires_grad=True)
    net = torch.nn.Sequential(torch.nn.Linear(32, 64), torch.nn.Linear(64, 8)).cuda()
    for kind in (torch.nn.Linear, layers8.Linear8):
        for layer in net:
            layer.__class__ = kind
        optimizer = mod().AdamW8(net.parameters())
        loss = net(x).square().sum()
        loss.backward(retain_graph=True)
        optimizer.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        net(x).sum().backward()                                      # a forward pass of its own
    view = net[0].weight.t()
    key = hooks.swap_saved_tensors._key(view)
    optimizer.step()
    assert hooks.swap_saved_tensors._key(view) != key
    (m, v), *_ = out = [[torch.empty_like(p) for _ in range(2)] for p in net.parameters()]
    mod().unpack_moments(optimizer, out)
    assert m._version == v._version == 1


def test_loading_takes_no_room_beyond_what_is_kept():
    n = 1 << 24
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = torch.ones_like(p)
    first = mod().AdamW8([p])
    first.step()
    saved = {k: v for k, v in first.state_dict().items()}
    saved["state"] = {0: {k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in saved["state"][0].items()}}
    again = mod().AdamW8([p])
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    again.load_state_dict(saved)
    assert torch.cuda.max_memory_allocated() - before <= 2 * (n * 33 // 32) + (2 << 20)      # two moments, and the allocator's rounding
    assert all(torch.equal(again.state[p][k], first.state[p][k]) for k in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("eps", [1e-30, 1e-20])
@pytest.mark.parametrize("bits", [8, 32])
def test_second_moments_below_the_normal_range_with_a_small_eps(bits, eps):
    """Gradients whose squares fp32 holds as subnormal numbers: the step is the learning rate, not m / eps."""
    rows = [[2.0 ** -k] * 32 for k in range(50, 68)] + [[-3e-19] * 32, [2.0 ** -50, -2.0 ** -62] * 16, [0.0] * 32]
    g = torch.tensor(rows).reshape(-1)
    p = torch.nn.Parameter(torch.full_like(g, 0.5).cuda())
    p.grad = g.cuda()
    optimizer = mod().AdamW8([p], lr=1e-2, betas=BETAS, eps=eps, weight_decay=0.0, bits=bits)
    optimizer.step()
    m, v = ref.moments(torch.zeros_like(g), torch.zeros_like(g), g, BETAS)
    assert bool((v[:32] > 2.0 ** -126).all()) and bool(((v[64:18 * 32] > 0) & (v[64:18 * 32] < 2.0 ** -110)).all()) and int((v == 0).sum()) == 32
    want, size = ref.update(torch.full_like(g, 0.5).double(), m, v, 1, 1e-2, BETAS, eps, 0.0)
    assert float((want - 0.5).abs().max()) <= 0.25                      # v is a few bits there, but no step is m / eps
    assert bool(((p.detach().cpu().double() - want).abs() <= bound(want, size, F32)).all())


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("bits", [8, 32])
def test_a_state_that_goes_to_the_host_and_comes_back(bits, capturable):
    """As programs do that need the room between steps: with other tensors, or with other memory for the same ones."""
    params = [torch.nn.Parameter(gradient((n,), d, n, 0.5).cuda()) for n, d in ((300, F32), (3000, BF16))]
    stay = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = (mod().AdamW8(some, bits=bits, master=True, capturable=capturable) for some in (params, stay))

    def step(t, refused=False):
        for i, (p, q) in enumerate(zip(params, stay)):
            p.grad = gradient(p.shape, p.dtype, 10 * t + i).cuda()
            q.grad = p.grad.clone()
        if refused:
            with pytest.raises(ValueError, match="moment"):
                a.step()
        else:
            a.step(), b.step()

    def move(to, data):
        for s in a.state.values():
            for k, v in s.items():
                if isinstance(v, torch.Tensor):
                    if data:
                        v.data = v.data.to(to)
                    else:
                        s[k] = v.to(to)

    step(0), step(1)
    for t, data in ((2, False), (3, True)):
        move("cpu", data)
        filler = torch.full((1 << 20,), 0x55, dtype=torch.uint8, device="cuda")         # where the moments were
        step(t, refused=True)
        move("cuda", data)
        step(t)
        assert bool((filler == 0x55).all())
    for p, q in zip(params, stay):
        assert torch.equal(p.detach(), q.detach()) and int(a.state[p]["step"]) == int(b.state[q]["step"]) == 4
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(a.state[p][k], b.state[q][k])
