"""Group norm with an activation function, channels last, on the GPU: every output within the bounds of tests/group_norm_reference.py, checkpoints to
the byte; layers, streams, graphs."""
import math
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import group_norm_reference as gref  # noqa: E402
import q8_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = ("y", "mean", "rstd", "dx", "dw", "db")


def q8():
    from cswap_amd import q8 as m

    return m


def images(n, c, spatial, dtype, seed, scale=1.0, shift=0.0):
    """[N, P, C] on the CPU, and the same as [N, C, ...] channels last on the GPU."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, math.prod(spatial), c, generator=g, dtype=torch.float64) * torch.exp(0.7 * torch.randn(c, generator=g, dtype=torch.float64))
    x = (x * scale + shift).to(dtype)
    return x, x.cuda().view(n, *spatial, c).movedim(-1, 1)


def flat(t):
    return t.detach().movedim(1, -1).flatten(1, -2) if t.dim() > 2 else t.detach().unsqueeze(1)


def params(c, seed):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.3 * torch.randn(c, generator=g)), 0.3 * torch.randn(c, generator=g)


def run(x, dy, groups, w, b, kind, checkpoint, eps=1e-5):
    m = q8()
    y, mean, rstd, held = m.group_norm(x, groups, w, b, eps, act=kind, checkpoint=checkpoint)
    return (y, mean, rstd, *m.group_norm_backward(dy, held, mean, rstd, groups, w, b, act=kind)), held


def compare(cpu, gpu, groups, w, b, kind, checkpoint, eps=1e-5):
    (xc, dyc), (x, dy) = cpu, gpu
    outs, held = run(x, dy, groups, w.cuda(), b.cuda(), kind, checkpoint, eps)
    dtype = xc.dtype
    if checkpoint:
        codes, scales = ref.pack(xc.reshape(-1, xc.shape[-1]))
        assert torch.equal(held.codes.cpu(), codes) and torch.equal(held.scales.cpu(), scales)
    args = (xc.double(), gref.held(xc) if checkpoint else xc.double(), dyc.double(), w.double(), b.double(), groups, eps, kind)
    want, err = gref.outputs(*args), gref.errors(*args, dtype)
    for name, got, v, e, t in zip(NAMES, outs, want, err, (dtype, F32, F32, dtype, w.dtype, w.dtype)):
        assert got.dtype == t
        if name in ("y", "dx"):
            assert got.shape == x.shape
            got = flat(got)
        ref.check(got, v, e, t, name)
    return outs


@pytest.mark.parametrize("checkpoint", [True, False])
@pytest.mark.parametrize("kind", [None, "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_types_and_functions(dtype, kind, checkpoint):
    n, c, spatial, groups = 3, 64, (9, 11), 8
    (xc, x), (dyc, dy) = images(n, c, spatial, dtype, 1), images(n, c, spatial, dtype, 2, 0.1)
    w, b = params(c, 3)
    compare((xc, dyc), (x, dy), groups, w.to(dtype), b.to(dtype), kind, checkpoint)
    if dtype is not F32:
        compare((xc, dyc), (x, dy), groups, w, b, kind, checkpoint)         # fp32 parameters of a 16-bit model


# channels: one, fewer than a chunk, odd, those whose lanes are no power of two, the widest; groups of one channel, of all, across chunks
SHAPES = [(1, 1, (1,), 1), (2, 1, (37,), 1), (3, 7, (5, 3), 7), (2, 9, (4, 4), 3), (5, 24, (1, 1), 3), (2, 33, (16, 9), 11), (1, 96, (35, 35), 24),
          (2, 288, (17, 17), 24), (7, 320, (3, 5), 32), (130, 32, (2, 2), 32), (2, 512, (8, 8), 1), (1, 1000, (9, 9), 8), (2, 2048, (4, 4), 32),
          (1, 2049, (3, 3), 3), (2, 4096, (3, 3), 2048), (1, 4095, (40,), 5), (1, 8, (200, 200), 2), (600, 16, (3,), 4), (2, 12, (2, 3, 4, 5), 6),
          (1, 64, (64, 64), 32)]


@pytest.mark.parametrize("checkpoint", [True, False])
@pytest.mark.parametrize("n,c,spatial,groups", SHAPES)
def test_shapes(n, c, spatial, groups, checkpoint):
    dtype, kind = ((F32, "silu"), (BF16, "gelu"), (F16, None))[(n + c) % 3]
    (xc, x), (dyc, dy) = images(n, c, spatial, dtype, c), images(n, c, spatial, dtype, c + 1, 0.1)
    w, b = params(c, 4)
    compare((xc, dyc), (x, dy), groups, w, b, kind, checkpoint, eps=1e-3)


def test_every_function_where_channels_are_no_whole_chunks():
    for kind in (None, "gelu", "gelu_tanh", "silu"):
        (xc, x), (dyc, dy) = images(2, 42, (7, 5), F32, 8), images(2, 42, (7, 5), F32, 9, 0.1)
        compare((xc, dyc), (x, dy), 6, *params(42, 4), kind, True)


def test_a_mean_far_from_zero_and_no_parameters():
    (xc, x), (dyc, dy) = images(2, 48, (12, 12), F32, 5, shift=1000.0), images(2, 48, (12, 12), F32, 6)
    m = q8()
    y, mean, rstd, held = m.group_norm(x, 6, checkpoint=False)
    assert held is x
    dx, dw, db = m.group_norm_backward(dy, held, mean, rstd, 6)
    one, zero = torch.ones(48, dtype=torch.float64), torch.zeros(48, dtype=torch.float64)
    args = (xc.double(), xc.double(), dyc.double(), one, zero, 6, 1e-5, None)
    for name, got, want, err in zip(NAMES, (flat(y), mean, rstd, flat(dx), dw, db), gref.outputs(*args), gref.errors(*args, F32)):
        ref.check(got, want, err, F32, name)


def test_a_first_value_far_from_the_others():
    """Sums are taken about the first value that a thread meets, which may be any value."""
    (xc, x), (dyc, dy) = images(1, 32, (16, 16), F32, 5), images(1, 32, (16, 16), F32, 6)
    xc[0, 0, :] = 1e4
    x = xc.cuda().view(1, 16, 16, 32).movedim(-1, 1)
    compare((xc, dyc), (x, dy), 4, *params(32, 1), "silu", False)


def test_a_sample_that_is_not_finite_leaves_the_others_groups():
    (xc, x), (dyc, dy) = images(3, 64, (6, 6), F32, 5), images(3, 64, (6, 6), F32, 6)
    w, b = (t.cuda() for t in params(64, 1))
    clean, _ = run(x, dy, 8, w, b, "silu", False)
    bad = x.clone()
    bad[1, 20, 3, 3] = math.nan
    bad[2, 40, 0, 0] = math.inf
    for checkpoint in (False, True):
        outs, _ = run(bad, dy, 8, w, b, "silu", checkpoint)
        y, dx = flat(outs[0]).unflatten(-1, (8, 8)), flat(outs[3]).unflatten(-1, (8, 8))
        want = flat(clean[0]).unflatten(-1, (8, 8))
        for n in range(3):
            for g in range(8):
                hit = (n, g) in ((1, 2), (2, 5))
                assert bool(torch.isnan(y[n, :, g]).all()) == hit and bool(torch.isnan(dx[n, :, g]).any()) == (hit or (checkpoint and (n, g // 4) in ((1, 0), (2, 1))))
                if not hit:
                    assert torch.equal(y[n, :, g], want[n, :, g])


def test_images_with_gaps_and_what_lies_between():
    n, c, h, w_ = 2, 40, 5, 6
    (xc, x), (dyc, dy) = images(n, c, (h, w_), BF16, 1), images(n, c, (h, w_), BF16, 2)
    w, b = (t.cuda() for t in params(c, 3))
    want, _ = run(x, dy, 5, w, b, "gelu", True)
    wide = torch.full((n, h, w_, 53), 7.0, dtype=BF16, device="cuda")
    wide[..., 3:43] = x.movedim(1, -1)
    gaps = wide[..., 3:43].movedim(-1, 1)
    wide_dy = torch.zeros_like(wide)
    wide_dy[..., 5:45] = dy.movedim(1, -1)
    for checkpoint in (True, False):
        got, held = run(gaps, wide_dy[..., 5:45].movedim(-1, 1), 5, w, b, "gelu", checkpoint)
        assert got[0].movedim(1, -1).is_contiguous()
        if checkpoint:
            assert all(torch.equal(a, e) for a, e in zip(got, want))
    assert bool((wide[..., :3] == 7).all()) and bool((wide[..., 43:] == 7).all())


def test_no_samples():
    m = q8()
    x = torch.empty(0, 4, 4, 32, device="cuda").movedim(-1, 1)
    y, mean, rstd, held = m.group_norm(x, 4)
    dx, dw, db = m.group_norm_backward(torch.empty_like(x), held, mean, rstd, 4)
    assert y.shape == x.shape and mean.shape == (0, 4) and dx.shape == x.shape
    assert torch.equal(dw, torch.zeros(32, device="cuda")) and torch.equal(db, dw)


def test_the_same_call_twice_gives_the_same_bits():
    (_, x), (_, dy) = images(4, 128, (40, 40), BF16, 1), images(4, 128, (40, 40), BF16, 2)
    w, b = (t.cuda() for t in params(128, 3))
    a, _ = run(x, dy, 16, w, b, "silu", True)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(run(x, dy, 16, w, b, "silu", True)[0], a))


def test_more_values_than_32_bits_count():
    """2^32 values and more: the last sample is that of a call of its own."""
    n, c, p, groups = 33, 64, 2097152 - 1, 4                           # 4.43e9 values
    x = torch.empty(n, p, c, dtype=BF16, device="cuda")
    x[:-1] = 0
    last = torch.randn(p, c, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(BF16)
    x[-1] = last
    y, mean, rstd, held = q8().group_norm(x.movedim(-1, 1), groups, act="silu")
    y1, mean1, rstd1, held1 = q8().group_norm(last[None].movedim(-1, 1), groups, act="silu")
    # tiles differ with the number of samples, and with them the order of sums: 64 + p / 8 roundings at most, in fact a few hundred
    assert torch.allclose(mean[-1], mean1[0], atol=1e-6) and torch.allclose(rstd[-1], rstd1[0], rtol=1e-5)
    assert bool((mean[:-1] == 0).all())
    assert torch.equal(held.codes[-p:], held1.codes) and torch.equal(held.scales[-p:], held1.scales)
    assert float((y[-1].float() - y1[0].float()).abs().max()) <= 2.0 ** -8 * 8
    assert not y[:-1].any()
    dx, dw, db = q8().group_norm_backward(x.movedim(-1, 1), held, mean, rstd, groups, act="silu")
    dx1, _, _ = q8().group_norm_backward(last[None].movedim(-1, 1), held1, mean1, rstd1, groups, act="silu")
    assert float((dx[-1].float() - dx1[0].float()).abs().max()) <= 2.0 ** -8 * 8


# ---------------------------------------------------------------- layers
def differences(f, x, h=1e-5):
    g = torch.zeros_like(x)
    flat_x, out = x.reshape(-1), g.view(-1)
    for i in range(flat_x.numel()):
        v = flat_x[i].item()
        flat_x[i] = v + h
        up = f(x)
        flat_x[i] = v - h
        out[i] = (up - f(x)) / (2 * h)
        flat_x[i] = v
    return g


def test_gradients_are_the_functions():
    from cswap_amd import layers8

    g = torch.Generator().manual_seed(0)
    x = torch.randint(-127, 128, (2, 3, 32), generator=g).double() / 64        # held exactly: multiples of 1/64 below 2, one of 1 or more
    x[..., 0] = 1.25
    assert torch.equal(gref.held(x), x)
    dy = torch.randn(2, 3, 32, generator=g, dtype=torch.float64)
    w, b = (t.double() for t in params(32, 1))
    leaves = [t.to(F32).cuda().requires_grad_() for t in (x.movedim(-1, 1), w, b)]
    layers8.group_norm(leaves[0], 4, leaves[1], leaves[2], act="silu").backward(dy.movedim(-1, 1).to(F32).cuda())

    def loss(x, w, b):
        return float((gref.outputs(x, x, dy, w, b, 4, 1e-5, "silu")[0] * dy).sum())

    wants = (differences(lambda v: loss(v, w, b), x.clone()).movedim(-1, 1), differences(lambda v: loss(x, v, b), w.clone()),
             differences(lambda v: loss(x, w, v), b.clone()))
    for leaf, want in zip(leaves, wants):
        assert float((leaf.grad.double().cpu() - want).abs().max()) <= 4e-6 * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_a_converted_model_gives_what_torch_gives(dtype):
    from cswap_amd import layers8
    from torch import nn

    torch.manual_seed(0)
    make = lambda: nn.Sequential(nn.Conv2d(3, 32, 3, padding=1), nn.GroupNorm(8, 32), nn.SiLU(), nn.Conv2d(32, 24, 3), nn.GroupNorm(3, 24))  # noqa: E731
    plain = make().cuda().to(dtype)
    ours = make().cuda().to(dtype)
    ours.load_state_dict(plain.state_dict())
    assert type(layers8.checkpoint_layers(ours)[1]) is nn.GroupNorm            # only where it is asked for
    assert type(layers8.checkpoint_layers(ours, group_norm=True)[1]) is layers8.GroupNorm8
    ours = ours.to(memory_format=torch.channels_last)
    x = torch.randn(4, 3, 16, 16, device="cuda", dtype=dtype)
    out, want = ours(x.to(memory_format=torch.channels_last)), plain(x)
    tol = 1e-3 if dtype is F32 else 0.05                                        # torch's convolutions of the two layouts differ by themselves
    assert float((out - want).detach().float().abs().max()) <= tol * max(1.0, float(want.detach().float().abs().max()))
    dy = torch.randn_like(want)
    out.backward(dy)
    want.backward(dy)
    for p, q in zip(ours.parameters(), plain.parameters()):
        # activations off by 2^-7 of their group's largest: gradients agree in direction
        a, e = p.grad.float().flatten(), q.grad.float().flatten()
        assert float((a @ e) / (a.norm() * e.norm() + 1e-30)) > 0.99 or float(e.norm()) < 1e-2
    # images of any layout, with an activation function, without gradients
    fused = layers8.GroupNorm8(8, 32, act="silu", device="cuda", dtype=dtype)
    z = torch.randn(2, 32, 5, 7, device="cuda", dtype=dtype)
    with torch.no_grad():
        a, e = fused(z), fused(z.to(memory_format=torch.channels_last))
    assert torch.equal(a, e) and torch.equal(fused(z), a)
    y = nn.functional.silu(nn.functional.group_norm(z.float(), 8, eps=1e-5))
    assert float((a.float() - y).abs().max()) <= (1e-5 if dtype is F32 else 2.0 ** -8 * float(y.abs().max()) + 1e-5)


def test_what_autograd_holds_and_hooks_leave_alone():
    from cswap_amd import layers8

    x = torch.randn(4, 64, 32, 32, device="cuda", dtype=BF16).to(memory_format=torch.channels_last).requires_grad_()
    w, b = (t.cuda().to(BF16).requires_grad_() for t in params(64, 1))
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = layers8.group_norm(x, 8, w, b, act="silu")
    assert sum(t.numel() * t.element_size() for t in kept) <= x.numel() * 33 / 32 + 3000
    y.sum().backward()
    assert x.grad.is_contiguous(memory_format=torch.channels_last)
    grad, = torch.autograd.grad(layers8.group_norm(x, 8, w, b).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_streams_and_graphs():
    from cswap_amd import layers8

    torch.manual_seed(0)
    x = torch.randn(3, 64, 20, 20, device="cuda", dtype=BF16).to(memory_format=torch.channels_last)
    dy = torch.randn(3, 64, 20, 20, device="cuda", dtype=BF16).to(memory_format=torch.channels_last)
    w, b = (t.cuda() for t in params(64, 1))

    def step(x, dy):
        leaf, p, q = x.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()
        y = layers8.group_norm(leaf, 8, p, q, act="gelu")
        return (y.detach(), *torch.autograd.grad(y, (leaf, p, q), dy))

    want = [t.clone() for t in step(x, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    sx, sdy = x.clone(), dy.clone()
    with torch.cuda.stream(side):
        step(sx, sdy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sdy)
    for k in range(4):
        sx.copy_(x * (k + 1)), sdy.copy_(dy.roll(k, 0))
        graph.replay()
        torch.cuda.synchronize()
        eager = step(sx.clone(), sdy.clone())
        assert all(torch.equal(a, e) for a, e in zip(out, eager))


# ---------------------------------------------------------------- what no other test calls
def test_statistics_beyond_32_bits():
    """More than 2^32 groups in all, of one value each: its mean is the value itself, and y is beta."""
    n, c = (1 << 21) + 3, 2048
    x = torch.zeros(n, c, dtype=BF16, device="cuda")
    ends = torch.randn(6, c, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(BF16)
    x[:3], x[-3:] = ends[:3], ends[3:]
    y, mean, rstd, _ = q8().group_norm(x, c, eps=0.25, checkpoint=False)
    assert torch.equal(mean[:3], ends[:3].float()) and torch.equal(mean[-3:], ends[3:].float())
    assert not y.any() and bool((rstd == 2.0).all()) and not mean[3:-3].any()


def test_layers_of_no_samples_of_no_positions_and_of_expanded_gradients():
    from cswap_amd import layers8

    w, b = (t.cuda().requires_grad_() for t in params(40, 1))
    for shape in ((0, 40, 3, 5), (0, 40)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = layers8.group_norm(x, 5, w, b, act="silu")
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert y.shape == shape and dx.shape == shape and not dw.any() and not db.any()
    with pytest.raises(ValueError, match="without values"):
        layers8.group_norm(torch.empty(2, 40, 0, 3, device="cuda"), 5, w, b)
    # [N, C]: groups of a row; images of one channel, one position, channels first
    for shape, groups in (((6, 40), 5), ((6, 40, 7), 8), ((3, 40, 1, 1), 4), ((1, 40, 2, 3, 2), 10)):
        x = torch.randn(shape, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
        y = layers8.group_norm(x, groups, w, b)
        want = torch.nn.functional.group_norm(x, groups, w, b)
        # fp32 both: a mean and a variance of up to 120 values, two products, each some roundings of values below 8
        assert float((y - want).detach().abs().max()) <= 64 * 2.0 ** -24 * 8
        got = torch.autograd.grad(y.sum(), (x, w, b), retain_graph=True)                    # one value, expanded
        full = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert all(torch.equal(a, e) for a, e in zip(got, full)) and got[0].shape == shape
    one = torch.randn(4, 1, 9, 9, device="cuda")
    y = layers8.group_norm(one, 1)
    assert float((y - torch.nn.functional.group_norm(one, 1)).abs().max()) <= 64 * 2.0 ** -24 * 8


def test_two_graphs_that_share_their_memory_and_calls_on_two_streams():
    (_, x), (_, dy) = images(2, 64, (50, 40), BF16, 1), images(2, 64, (50, 40), BF16, 2)
    w, b = (t.cuda() for t in params(64, 3))
    names = ("gelu", "silu")
    for kind in names:
        run(x, dy, 8, w, b, kind, True)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in names], []
    for graph, kind in zip(graphs, names):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if outs else None):
            outs.append(run(x, dy, 8, w, b, kind, True)[0])
    for k in range(4):
        x.mul_(1.5), dy.neg_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for kind, out in zip(names, outs):
            assert all(torch.equal(a, e) for a, e in zip(out, run(x, dy, 8, w, b, kind, True)[0]))
    want = [run(x, dy, 8, w, b, kind, True)[0] for kind in names]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in names]
    for _ in range(5):
        got = []
        for kind, stream in zip(names, streams):
            with torch.cuda.stream(stream):
                got.append(run(x, dy, 8, w, b, kind, True)[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for p, q in zip(got, want) for a, e in zip(p, q))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_parameters_and_images_that_start_at_any_element(dtype):
    for n, c, spatial, groups in ((2, 64, (6, 7), 8), (3, 30, (5, 4), 5), (1, 64, (100, 90), 4)):
        (_, x), (_, dy) = images(n, c, spatial, dtype, 1), images(n, c, spatial, dtype, 2)
        w, b = (t.to(dtype).cuda() for t in params(c + 3, 3))
        shifted = []
        for t in (x, dy):
            room = torch.empty(t.numel() + 3, dtype=dtype, device="cuda")[1:-2].view(n, *spatial, c).movedim(-1, 1)
            shifted.append(room.copy_(t))
        want, _ = run(x, dy, groups, w[1:-2].clone(), b[1:-2].clone(), "silu", True)
        got, _ = run(*shifted, groups, w[1:-2], b[1:-2], "silu", True)
        assert all(torch.equal(a, e) for a, e in zip(got, want))
