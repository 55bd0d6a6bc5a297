"""Products in 8-bit floating point on the GPU: codes and scales exactly, results within the bounds of tests/f8_reference.py, whole numbers to the bit;
layers, streams, graphs."""
import math
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import f8_reference as fref  # noqa: E402
import q8_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def f8():
    from cswap_amd import f8 as m

    return m


def values(rows, cols, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64) * torch.exp(torch.randn(cols, generator=g, dtype=torch.float64))
    return (x * scale).to(dtype)


def whole(rows, cols, seed, most=8):
    return torch.randint(-most, most + 1, (rows, cols), generator=torch.Generator().manual_seed(seed)).double()


# ---------------------------------------------------------------- format
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("n,k", [(1, 1), (16, 16), (127, 129), (128, 128), (200, 300), (1000, 193), (130, 520)])
def test_weights_are_laid_out_as_defined(dtype, n, k):
    w = values(n, k, dtype, n + k)
    held = f8().f8_weight(w.cuda())
    want, scales = fref.held(w, 128)
    assert torch.equal(held.scales.cpu(), scales)
    assert torch.equal(f8().f8_weight_values(held, F32).cpu().double(), want)
    full = held.codes.view(torch.uint8)
    assert torch.equal(held.turned.view(torch.uint8), full.t())
    assert not full[n:].any() and not full[:, k:].any()
    plain = f8().f8_weight(w.cuda(), backward=False)
    assert plain.turned is None and torch.equal(plain.codes.view(torch.uint8), full)


def special(dtype):
    fi = torch.finfo(dtype)
    least = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[dtype]
    rows = [[0.0] * 130, [-0.0] * 130, [fi.max] * 130, [least] * 130, [fi.tiny, -least] * 65, [448.0] * 130, [449.0] + [1.0] * 129, [-448.5, 3.0] * 65,
            [2.0 ** -k for k in range(130)], [240.0, 17.0, 18.0, 19.0, 20.0, 21.0, 22.0, 23.0, 24.0, 25.0] * 13, [1.0] + [2.0 ** -18 * i / 4 for i in range(129)]]
    return torch.tensor(rows, dtype=torch.float64).to(dtype)


@pytest.mark.parametrize("rows_of", [1, 40])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_activations_are_held_as_defined(dtype, rows_of):
    """The unit matrix gives back what the codes stand for: one product of a value with 1, in fp32 exactly."""
    x = torch.cat([special(dtype), values(5, 130, dtype, 3)]).repeat(rows_of, 1) if rows_of > 1 else torch.cat([special(dtype), values(5, 130, dtype, 3)])
    one = f8().f8_weight(torch.eye(130).cuda())
    want = fref.held(x, 1)[0]
    fits = want.abs() <= torch.finfo(F32).max
    y = f8().f8_linear(x.cuda(), one, out_dtype=F32).cpu().double()
    # what is below fp32's normal range may be flushed by the matrix instructions
    small = want.abs() < 2.0 ** -126
    assert torch.equal(torch.where(small | ~fits, 0.0, y), torch.where(small | ~fits, 0.0, want))
    assert bool((y[small] .abs()<= 2.0 ** -126).all())
    back = f8().f8_linear_backward(x.cuda(), one, out_dtype=F32).cpu().double()
    assert torch.equal(torch.isnan(back), torch.isnan(y)) and torch.equal(back.nan_to_num(7.0), y.nan_to_num(7.0))    # a row beyond fp32: infinity times 0


def test_values_that_are_not_finite():
    for bad in (math.nan, math.inf, -math.inf):
        for rows in (3, 70):
            x, w = values(rows, 300, BF16, 1), values(200, 300, BF16, 2)
            x[2, 290] = bad
            for out in (BF16, F32):
                y = f8().f8_linear(x.cuda(), f8().f8_weight(w.cuda()), out_dtype=out)
                clean = f8().f8_linear(values(rows, 300, BF16, 1).cuda(), f8().f8_weight(w.cuda()), out_dtype=out)
                assert bool(torch.isnan(y[2]).all())
                keep = [i for i in range(rows) if i != 2]
                assert torch.equal(y[keep], clean[keep])
            w[130, 5] = bad
            y = f8().f8_linear(values(rows, 300, BF16, 1).cuda(), f8().f8_weight(w.cuda()))
            assert bool(torch.isnan(y[:, 128:]).all()) and torch.equal(y[:, :128], clean[:, :128].to(BF16) if out is BF16 else f8().f8_linear(
                values(rows, 300, BF16, 1).cuda(), f8().f8_weight(values(200, 300, BF16, 2).cuda()))[:, :128])


# ---------------------------------------------------------------- products
SIZES = [(1, 16, 16), (1, 1, 1), (1, 4096, 1024), (2, 17, 129), (15, 100, 300), (16, 128, 128), (17, 1000, 193), (32, 33, 4100), (33, 130, 40), (50, 4100, 4200), (64, 256, 256), (100, 300, 520),
         (129, 127, 640), (257, 1000, 193), (1000, 5, 1030), (700, 520, 130), (1576, 1000, 193), (2050, 129, 384), (300, 4100, 256),
         (4100, 8300, 200), (16400, 4000, 136)]                       # the last two: the largest tiles, everything cut off somewhere


@pytest.mark.parametrize("rows,n,k", SIZES)
def test_whole_numbers_are_exact(rows, n, k):
    """Products of whole numbers up to 8 span 6 bits and sums stay below 2^24: every form gives them exactly, rounded once."""
    x, w, b = whole(rows, k, 1), whole(n, k, 2), whole(1, n, 3, 100)[0]
    dev = torch.device("cuda")
    xg, wg = x.to(dev), w.to(dev)
    want = (xg.float() @ wg.float().t()).double() if max(rows, n) > 2000 else (x @ w.t()).to(dev)      # fp32 products of whole numbers are exact, too
    held = f8().f8_weight(wg.to(F32))
    for dtype in (BF16, F16) if k < 1000 else (BF16,):
        for out in (dtype, F32):
            y = f8().f8_linear(xg.to(dtype), held, b.to(dev, F32), out_dtype=out)
            assert y.dtype is out and torch.equal(y, (want + b.to(dev)).to(F32).to(out)), (dtype, out)
    d = whole(rows, n, 4).to(dev)
    want = (d.float() @ wg.float()).double() if max(rows, n) > 2000 else (d.cpu() @ w).to(dev)
    for out in (BF16, F32):
        assert torch.equal(f8().f8_linear_backward(d.to(BF16), held, out_dtype=out), want.to(F32).to(out)), out


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,n,k", [s for s in SIZES if max(s) <= 2100])
def test_products(dtype, rows, n, k):
    x, w, dy = values(rows, k, dtype, 1), values(n, k, dtype, 2, k ** -0.5), values(rows, n, dtype, 3, 0.1)
    b = values(1, n, dtype, 4)[0]
    held = f8().f8_weight(w.cuda())
    for out in {dtype, F32}:
        y, cut, exact = fref.linear(x, w, b)
        ref.check(f8().f8_linear(x.cuda(), held, b.cuda(), out_dtype=out), y, exact if out is F32 else cut, out, "y")
        y, cut, exact = fref.linear(dy, w, None, turned=True)
        ref.check(f8().f8_linear_backward(dy.cuda(), held, out_dtype=out), y, exact if out is F32 else cut, out, "dx")


def test_results_in_16_bits_are_near_those_in_32():
    """What an instruction cuts off is small against the rounding of the result: a sum of 64 cut products is off by at most 64 * 2^-13 of the
    largest, and of many sums those cuts are as a rule 2^-14 of it."""
    x, w = values(300, 1024, F16, 1), values(500, 1024, F16, 2)
    held = f8().f8_weight(w.cuda())
    for rows in (300, 5):
        a, e = f8().f8_linear(x[:rows].cuda(), held).double(), f8().f8_linear(x[:rows].cuda(), held, out_dtype=F32).double()
        assert float((a - e).norm() / e.norm()) <= 2.0 ** -12 + 2.0 ** -11


def test_rows_with_gaps_leading_dimensions_and_no_rows():
    x, w = values(60, 200, BF16, 1), values(77, 200, BF16, 2)
    held = f8().f8_weight(w.cuda())
    want = f8().f8_linear(x.cuda(), held)
    wide = torch.full((60, 231), math.nan, dtype=BF16, device="cuda")
    wide[:, 5:205] = x.cuda()
    assert torch.equal(f8().f8_linear(wide[:, 5:205], held), want)
    assert torch.equal(f8().f8_linear(wide[:, 5:205][:7], held), f8().f8_linear(x[:7].cuda(), held))
    assert torch.equal(f8().f8_linear(x.cuda().view(3, 4, 5, 200), held), want.view(3, 4, 5, 77))
    assert torch.equal(f8().f8_linear(x[0].cuda(), held), f8().f8_linear(x[:1].cuda(), held)[0])
    big = torch.zeros(77, 250, dtype=BF16, device="cuda")
    big[:, 3:203] = w.cuda()
    assert torch.equal(f8().f8_weight(big[:, 3:203]).codes.view(torch.uint8), held.codes.view(torch.uint8))
    assert f8().f8_linear(torch.empty(0, 200, dtype=BF16, device="cuda"), held).shape == (0, 77)
    assert f8().f8_linear_backward(torch.empty(4, 0, 77, dtype=BF16, device="cuda"), held).shape == (4, 0, 200)


def test_more_codes_than_32_bits_count():
    """Activations of more than 2^32 codes: rows far in are those of a call of their own."""
    rows, k = (1 << 32) // 8192 + 300, 8192
    x = torch.zeros(rows, k, dtype=BF16, device="cuda")
    tail = values(300, k, BF16, 1).cuda()
    x[-300:] = tail
    held = f8().f8_weight(values(40, k, BF16, 2).cuda())
    y = f8().f8_linear(x, held, out_dtype=F32)
    assert torch.equal(y[-300:], f8().f8_linear(tail, held, out_dtype=F32)) and not y[:-300].any()
    assert torch.equal(f8().f8_linear(x, held)[-300:], f8().f8_linear(tail, held))


def test_twice_gives_the_same_bits():
    x, held = values(1000, 700, BF16, 1).cuda(), f8().f8_weight(values(900, 700, BF16, 2).cuda())
    y = f8().f8_linear(x, held)
    assert all(torch.equal(f8().f8_linear(x, held), y) for _ in range(3))


# ---------------------------------------------------------------- layers
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_layer_is_the_kernels_in_a_row(dtype):
    from cswap_amd import layers8, q8

    x, w, b = (t.cuda().requires_grad_() for t in (values(60, 200, dtype, 1), values(96, 200, dtype, 2), values(1, 96, dtype, 3)[0]))
    dy = values(60, 96, dtype, 4).cuda()
    held8 = f8().f8_weight(w.detach())
    y = layers8.linear_f8(x.view(3, 20, 200), w, b)
    assert torch.equal(y.view(60, 96), f8().f8_linear(x.detach(), held8, b.detach()))
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy.view(3, 20, 96))
    assert torch.equal(dx, f8().f8_linear_backward(dy, held8))
    want = q8.q8_weight_grad(dy, q8.q8_compress(x.detach()))
    assert torch.equal(dw, want[0]) and torch.equal(db, want[1])
    # some of them, with what is there already, and none
    held = layers8.hold(x)
    y = layers8.linear_f8(x, w, b, held=held, weight8=held8)
    assert torch.equal(torch.autograd.grad(y, w, dy, retain_graph=True)[0], dw) and torch.equal(torch.autograd.grad(y, x, dy)[0], dx)
    y = layers8.linear_f8(x.detach(), w.detach(), b)
    assert torch.allclose(torch.autograd.grad(y, b, dy)[0].float(), db.float(), rtol=1e-2, atol=1e-2)
    y = layers8.linear_f8(x, w.detach(), None)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], dx)
    with torch.no_grad():
        assert torch.equal(layers8.linear_f8(x, w, b), f8().f8_linear(x, held8, b))
    with pytest.raises(ValueError, match="weight8"):
        layers8.linear_f8(x, w, b, weight8=f8().f8_weight(w.detach(), backward=False))
    with pytest.raises(ValueError, match="weight8"):
        layers8.linear_f8(x, w, b, weight8=f8().f8_weight(w.detach()[:50]))
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(layers8.linear_f8(x, w, b).sum(), x, create_graph=True)
        g.sum().backward()


def test_gradients_are_the_functions():
    """At values that the codes hold exactly the gradients are those of x @ w.T + b, which is linear in each: exact differences."""
    from cswap_amd import layers8

    x, w, b, dy = whole(5, 40, 1), whole(7, 40, 2), whole(1, 7, 3)[0], whole(5, 7, 4)
    leaves = [t.to(F32).cuda().requires_grad_() for t in (x, w, b)]
    layers8.linear_f8(*leaves).backward(dy.to(F32).cuda())
    assert torch.equal(leaves[0].grad.cpu().double(), dy @ w) and torch.equal(leaves[1].grad.cpu().double(), dy.t() @ x)
    assert torch.equal(leaves[2].grad.cpu().double(), dy.sum(0))

    def loss(x, w, b):
        return float(((x @ w.t() + b) * dy).sum())

    for at, leaf in zip((0, 1, 2), leaves):
        for i in (0, 3):
            up = [t.clone() for t in (x, w, b)]
            up[at].view(-1)[i] += 1.0
            assert loss(*up) - loss(x, w, b) == float(leaf.grad.view(-1)[i])


def test_under_autocast_on_another_stream_and_in_a_graph():
    from cswap_amd import layers8

    torch.manual_seed(0)
    layer = layers8.checkpoint_layers(torch.nn.Sequential(torch.nn.Linear(300, 200), torch.nn.GELU(), torch.nn.Linear(200, 100)), f8=True).cuda()
    assert [type(m).__name__ for m in layer] == ["LinearF8", "GELU8", "LinearF8"]
    x = torch.randn(70, 300, device="cuda")

    def step(x):
        with torch.autocast("cuda", dtype=BF16):
            y = layer(x)
        assert y.dtype is BF16
        return (y.detach(), *torch.autograd.grad(y.float().square().sum(), list(layer.parameters())))

    want = [t.clone() for t in step(x)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.synchronize()
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    sx = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx)
    for k in range(4):
        sx.copy_(x.roll(k, 0) * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        eager = step(sx.clone())
        assert all(torch.equal(a, e) for a, e in zip(out, eager))


def test_a_training_step_of_all_three():
    """Convolutions with group norms, linear layers in 8-bit floating point and the 8-bit optimiser, eager and captured: the same parameters."""
    from cswap_amd import adamw8, layers8
    from torch import nn

    def build():
        torch.manual_seed(0)
        net = nn.Sequential(nn.Conv2d(3, 32, 3, padding=1), nn.GroupNorm(8, 32), nn.SiLU(), nn.Conv2d(32, 64, 3, stride=2), nn.GroupNorm(8, 64), nn.SiLU(),
                            nn.AdaptiveAvgPool2d(2), nn.Flatten(), nn.Linear(256, 128), nn.GELU(), nn.LayerNorm(128), nn.Linear(128, 10))
        net = layers8.checkpoint_layers(net, group_norm=True, f8=True).cuda().to(BF16).to(memory_format=torch.channels_last)
        return net, adamw8.AdamW8(net.parameters(), lr=1e-3, master=True, capturable=True)

    x = torch.randn(16, 3, 20, 20, device="cuda").to(BF16).to(memory_format=torch.channels_last)
    t = torch.randint(0, 10, (16,), device="cuda")

    def step(net, optimizer):
        loss = nn.functional.cross_entropy(net(x).float(), t)
        loss.backward()
        optimizer.step()
        for p in net.parameters():
            p.grad.zero_()
        return loss

    torch.backends.cudnn.deterministic = True
    try:
        a, oa = build()
        b, ob = build()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                step(a, oa)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(a, oa)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            torch.randn(100, device="cuda").sum().item()
        for _ in range(6):
            step(b, ob)
        torch.cuda.synchronize()
    finally:
        torch.backends.cudnn.deterministic = False
    for p, q in zip(a.parameters(), b.parameters()):
        assert bool(torch.isfinite(p).all())
        assert int(oa.state[p]["step"]) == int(ob.state[q]["step"]) == 6
        # the convolutions' gradients are torch's, whose order of sums may differ from run to run: six steps of 1e-3, at most all the other way
        assert float((p.detach().float() - q.detach().float()).abs().max()) <= 2 * 6 * 1e-3 * 4 + 2.0 ** -8 * float(p.detach().float().abs().max())


# ---------------------------------------------------------------- what no other test calls
def test_two_graphs_that_share_their_memory():
    x = values(300, 260, BF16, 1).cuda()
    held = f8().f8_weight(values(400, 260, BF16, 2).cuda())
    dy = values(300, 400, BF16, 3).cuda()
    f8().f8_linear(x, held), f8().f8_linear_backward(dy, held)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    with torch.cuda.graph(graphs[0]):
        outs.append(f8().f8_linear(x, held))
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        outs.append(f8().f8_linear_backward(dy, held))
    for k in range(4):
        x.mul_(1.25), dy.neg_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], f8().f8_linear(x, held)) and torch.equal(outs[1], f8().f8_linear_backward(dy, held))


def test_calls_on_two_streams_at_once():
    x = [values(700, 520, BF16, i).cuda() for i in range(4)]
    held = f8().f8_weight(values(600, 520, BF16, 9).cuda())
    want = [f8().f8_linear(t, held) for t in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in x]
    for _ in range(5):
        got = []
        for t, stream in zip(x, streams):
            with torch.cuda.stream(stream):
                got.append(f8().f8_linear(t, held))
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_layers_of_no_rows_and_of_expanded_gradients():
    from cswap_amd import layers8

    w, b = values(24, 40, F32, 1).cuda().requires_grad_(), values(1, 24, F32, 2)[0].cuda().requires_grad_()
    for shape in ((0, 40), (0, 3, 40), (2, 0, 40)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = layers8.linear_f8(x, w, b)
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert y.shape == (*shape[:-1], 24) and dx.shape == shape and not dw.any() and not db.any()
    x = values(50, 40, F32, 3).cuda().requires_grad_()
    wide = torch.zeros(24, 60, device="cuda")
    wide[:, 5:45] = w.detach()
    for weight in (w, wide[:, 5:45].requires_grad_(), w.detach().t().contiguous().t().requires_grad_()):
        y = layers8.linear_f8(x, weight, b)
        got = torch.autograd.grad(y.sum(), (x, weight, b), retain_graph=True)                # one value, expanded
        want = torch.autograd.grad(y, (x, weight, b), torch.ones_like(y))
        assert all(torch.equal(a, e) for a, e in zip(got, want))
    with torch.no_grad():
        assert torch.equal(layers8.linear_f8(x, wide[:, 5:45], b), f8().f8_linear(x, f8().f8_weight(w), b))


def test_signs_that_are_turned_in_a_view_are_refused():
    z = torch.complex(values(1, 1, F32, 1), values(1, 1, F32, 2)).cuda().conj().imag
    held = f8().f8_weight(values(1, 1, F32, 3).cuda())
    assert z.is_neg() and z.is_contiguous()
    for call in (lambda: f8().f8_weight(z), lambda: f8().f8_linear(z, held), lambda: f8().f8_linear_backward(z, held)):
        with pytest.raises(ValueError, match="sign"):
            call()


def test_hooks_on_saved_tensors_leave_the_layers_as_they_are():
    """What the layers keep is in 8 bits already: the hooks that hold or swap activations give the same gradients."""
    from cswap_amd import hooks, layers8, swap
    from torch import nn

    engine = swap.SwapEngine(pinned_bytes=64 << 20, device_bytes=64 << 20)

    torch.manual_seed(0)
    net = nn.Sequential(nn.Conv2d(3, 32, 3, padding=1), nn.GroupNorm(4, 32), nn.Flatten(), nn.Linear(32 * 36, 96), nn.Linear(96, 8))
    net = layers8.checkpoint_layers(net, group_norm=True, f8=True).cuda().to(memory_format=torch.channels_last)
    assert [type(m).__name__ for m in net] == ["Conv2d", "GroupNorm8", "Flatten", "LinearF8", "LinearF8"]
    x = torch.randn(5, 32, 6, 6, device="cuda").to(memory_format=torch.channels_last)
    tail = net[1:]                                                                            # torch's convolution keeps its own input

    dy = torch.randn(5, 8, device="cuda")
    want = torch.autograd.grad(tail(x), list(tail.parameters()), dy)
    for ctx in (hooks.hold_saved_tensors(min_bytes=0), hooks.swap_saved_tensors(engine, policy=swap.NONE, min_bytes=4)):
        with ctx:
            y = tail(x)
        got = torch.autograd.grad(y, list(tail.parameters()), dy)
        assert ctx.stats.get("held", 0) == 0 and all(torch.equal(a, e) for a, e in zip(got, want))
        ctx.close()
    engine.close()


@pytest.mark.parametrize("dtype,rows,n,k,kind", [(F16, 8200, 8003, 400, F32), (BF16, 8192, 8192, 512, BF16), (BF16, 9000, 7999, 300, None), (F16, 4100, 4200, 4200, F16),
                                                 (BF16, 8200, 8100, 4200, BF16), (F16, 17000, 4352, 100, F32)], ids=str)
def test_whole_numbers_in_many_large_tiles(dtype, rows, n, k, kind):
    """Sums of products of 0 and +-1 are exact in fp32, so that results are the exact ones rounded once; rows further apart than they are long keep
    what lies between them.  More tiles than compute units, ends inside a tile on either side, even and odd numbers of stages."""
    from cswap_amd._lib import lib

    g = torch.Generator(device="cuda").manual_seed(rows + k)
    x = torch.randint(-1, 2, (rows, k), generator=g, device="cuda").float()
    w = torch.randint(-1, 2, (n, k), generator=g, device="cuda").float()
    x[:, 0] = w[0, :] = 1                                           # every block has a value, and one scale
    bias = None if kind is None else torch.randint(-9, 10, (n,), generator=g, device="cuda").to(kind)
    want = x @ w.t() if bias is None else x @ w.t() + bias.float()
    held = f8().f8_weight(w.to(dtype))
    assert torch.equal(f8().f8_linear(x.to(dtype), held, bias), want.to(dtype))
    del x
    dy = torch.randint(-1, 2, (rows, n), generator=g, device="cuda").float()
    assert torch.equal(f8().f8_linear_backward(dy.to(dtype), held), (dy @ w).to(dtype))
    # gaps between rows of the result
    xs, pitch = (want[:, :k] * 0 + 1).to(dtype), n + 5
    y = torch.full((rows, pitch), -7.0, dtype=dtype, device="cuda")
    room = lib().cswap_f8_linear_workspace_bytes(rows, k)
    ws = torch.empty(room, dtype=torch.uint8, device="cuda")
    code = {F32: 0, BF16: 1, F16: 2}[dtype]
    assert lib().cswap_f8_linear(xs.data_ptr(), code, rows, k, 0, held.codes.data_ptr(), held.scales.data_ptr(), n, 0, 0, 0, y.data_ptr(), code, pitch, ws.data_ptr(),
                                 room, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(y[:, :n], w.sum(1).to(dtype).expand(rows, n)) and bool((y[:, n:] == -7).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
def test_biases_and_rows_that_start_at_any_element(dtype):
    room = values(1, 4400, dtype, 5)[0].cuda()
    for rows, n, k in ((1, 200, 130), (16, 77, 256), (40, 200, 130), (300, 333, 300), (4200, 4300, 256)):
        wide = values(rows, k + 3, dtype, 1).cuda()
        held = f8().f8_weight(values(n, k, dtype, 2).cuda())
        plain = f8().f8_linear(wide[:, 1:k + 1].contiguous(), held, room[1:n + 1].clone())
        assert torch.equal(f8().f8_linear(wide[:, 1:k + 1], held, room[1:n + 1]), plain)
        w = values(n, k + 3, dtype, 2).cuda()
        again = f8().f8_weight(w[:, 1:k + 1])
        want = f8().f8_weight(w[:, 1:k + 1].contiguous())
        assert torch.equal(again.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(again.turned.view(torch.uint8), want.turned.view(torch.uint8))
        assert torch.equal(again.scales, want.scales)


def test_a_captured_training_step_is_the_eager_one_to_the_bit():
    """Group norm, linear layers in 8-bit floating point, activation functions, layer norm and the 8-bit optimiser make their sums in fixed orders: steps on
    inputs of their own, captured and eager, leave the same parameters and the same moments."""
    from cswap_amd import adamw8, layers8
    from torch import nn

    def build():
        torch.manual_seed(0)
        net = nn.Sequential(nn.GroupNorm(4, 32), nn.SiLU(), nn.Flatten(), nn.Linear(32 * 36, 200), nn.GELU(), nn.LayerNorm(200), nn.Linear(200, 10))
        net = layers8.checkpoint_layers(net, group_norm=True, f8=True).cuda().to(BF16)
        assert [type(m).__name__ for m in net] == ["GroupNorm8", "SiLU8", "Flatten", "LinearF8", "GELU8", "LayerNorm8", "LinearF8"]
        return net, adamw8.AdamW8(net.parameters(), lr=1e-2, master=True, capturable=True)

    g = torch.Generator(device="cuda").manual_seed(5)
    inputs = [torch.randn(40, 32, 6, 6, generator=g, device="cuda").to(BF16).to(memory_format=torch.channels_last) for _ in range(7)]
    targets = [torch.randn(40, 10, generator=g, device="cuda") for _ in inputs]
    x, t = inputs[0].clone(memory_format=torch.channels_last), targets[0].clone()

    def step(net, optimizer):
        (net(x).float() - t).square().sum().backward()
        optimizer.step()
        for p in net.parameters():
            p.grad.zero_()

    def kept(net, optimizer):
        return [v.clone() for p in net.parameters() for v in (p.detach(), *(s for s in optimizer.state[p].values() if isinstance(s, torch.Tensor)))]

    eager, captured = build(), build()
    start = [p.detach().clone() for p in eager[0].parameters()]
    wanted = []
    for k in range(7):
        x.copy_(inputs[k]), t.copy_(targets[k])
        step(*eager)
        wanted.append(kept(*eager))
    side = torch.cuda.Stream()
    for k in range(3):
        x.copy_(inputs[k]), t.copy_(targets[k])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*captured)
        torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(*captured)
    for k in range(3, 7):
        x.copy_(inputs[k]), t.copy_(targets[k])
        graph.replay()
        torch.cuda.synchronize()
        torch.randn(1000, device="cuda").sum().item()
        assert all(torch.equal(a, e) for a, e in zip(kept(*captured), wanted[k], strict=True)), k
    assert all(bool((p != q).any()) for p, q in zip(captured[0].parameters(), start))
    assert all(any(bool((a != b).any()) for a, b in zip(wanted[k], wanted[k + 1])) for k in range(6))
