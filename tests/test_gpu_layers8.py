"""Layers that keep their inputs in 8 bits: gradients against the formulas, against differences and against the
kernels called one by one; streams, graphs and the saved-tensor hooks."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import q8_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
DEV = "cuda"


def randn(*shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).to(dtype).to(DEV)


def exactly_held(rows, cols, seed=0):
    """Values that a checkpoint holds exactly: multiples of 1/64 below 2, one of them 1 or more in each group."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-127, 128, (rows, cols), generator=g).double() / 64
    x[:, ::32] = 1.25
    assert torch.equal(ref.held(x), x)
    return x


def differences(f, x, h=1e-5):
    """The gradient of the number f(x) by central differences, 64 bits."""
    g = torch.zeros_like(x)
    flat, out = x.view(-1), g.view(-1)
    for i in range(flat.numel()):
        v = flat[i].item()
        flat[i] = v + h
        up = f(x)
        flat[i] = v - h
        out[i] = (up - f(x)) / (2 * h)
        flat[i] = v
    return g


def close(got, want, tol, what):
    got = got.detach().double().cpu()
    assert float((got - want).abs().max()) <= tol * max(1.0, float(want.abs().max())), what


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_activation_gradient_is_the_functions(kind):
    from cswap_amd import layers8

    x = exactly_held(2, 40)
    dy = randn(2, 40, seed=1).cpu().double()
    leaf = x.to(F32).to(DEV).requires_grad_()
    layers8.activation(leaf, kind).backward(dy.to(F32).to(DEV))
    # differences of 64-bit values are off by h^2 and 2^-53 / h, both below 1e-9: what is left is fp32
    close(leaf.grad, differences(lambda v: float((ref.act(v, kind)[0] * dy).sum()), x.clone()), 1e-6, kind)


def test_layer_norm_gradients_are_the_functions():
    from cswap_amd import layers8

    x, dy = exactly_held(3, 40, 2), randn(3, 40, seed=3).cpu().double()
    w, b = randn(40, seed=4).cpu().double(), randn(40, seed=5).cpu().double()
    leaves = [t.to(F32).to(DEV).requires_grad_() for t in (x, w, b)]
    layers8.layer_norm(*leaves).backward(dy.to(F32).to(DEV))

    def loss(x, w, b):
        return float((ref.norm(x, x, dy, w, b, 1e-5)[0] * dy).sum())

    close(leaves[0].grad, differences(lambda v: loss(v, w, b), x.clone()), 2e-6, "dx")
    close(leaves[1].grad, differences(lambda v: loss(x, v, b), w.clone()), 2e-6, "dw")
    close(leaves[2].grad, differences(lambda v: loss(x, w, v), b.clone()), 2e-6, "db")


def test_linear_gradients_are_the_functions():
    from cswap_amd import layers8

    x, dy = exactly_held(6, 40, 6), randn(6, 5, seed=7).cpu().double()
    w, b = randn(5, 40, seed=8).cpu().double(), randn(5, seed=9).cpu().double()
    leaves = [t.to(F32).to(DEV).view(*s).requires_grad_() for t, s in ((x, (2, 3, 40)), (w, (5, 40)), (b, (5,)))]
    y = layers8.linear(*leaves)
    assert y.shape == (2, 3, 5)
    y.backward(dy.to(F32).to(DEV).view(2, 3, 5))
    close(leaves[0].grad.view(6, 40), dy @ w, 1e-5, "dx")
    close(leaves[1].grad, differences(lambda v: float(((x @ v.t() + b) * dy).sum()), w.clone()), 1e-5, "dw")
    close(leaves[2].grad, differences(lambda v: float(((x @ w.t() + v) * dy).sum()), b.clone()), 1e-5, "db")


def block(cols=96, hidden=224, dtype=F32, seed=10):
    from torch import nn

    torch.manual_seed(seed)
    return nn.Sequential(nn.LayerNorm(cols), nn.Linear(cols, hidden), nn.GELU(), nn.Linear(hidden, cols), nn.SiLU()).to(DEV).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_a_block_of_layers_is_the_kernels_in_a_row(dtype):
    """Forward and backward of a norm and two linear layers with activations, converted in place, to the bit what the
    functions give one by one, and near what the layers give without checkpoints."""
    from cswap_amd import layers8, q8
    from torch.nn import functional as F

    plain, model = block(dtype=dtype), layers8.checkpoint_layers(block(dtype=dtype))
    assert [type(m).__name__ for m in model] == ["LayerNorm8", "Linear8", "GELU8", "Linear8", "SiLU8"]
    assert list(model.state_dict()) == list(plain.state_dict())
    x, dy = randn(4, 37, 96, dtype=dtype, seed=11), randn(4, 37, 96, dtype=dtype, seed=12, scale=0.01)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    ya, yb = model(a), plain(b)
    ya.backward(dy)
    yb.backward(dy)
    norm, one, _, two, _ = model
    with torch.no_grad():
        h0, mean, rstd, held0 = q8.layer_norm(x, norm.weight, norm.bias)
        h1 = F.linear(h0, one.weight, one.bias)
        h2, held2 = q8.q8_act(h1, "gelu")
        h3 = F.linear(h2, two.weight, two.bias)
        y, held4 = q8.q8_act(h3, "silu")
        d3 = q8.q8_act_backward(dy, held4, "silu")
        dw2, db2 = q8.q8_weight_grad(d3, q8.q8_compress(h2))
        d1 = q8.q8_act_backward(d3 @ two.weight, held2, "gelu")
        dw1, db1 = q8.q8_weight_grad(d1, q8.q8_compress(h0))
        dx, dg, dn = q8.layer_norm_backward(d1 @ one.weight, held0, mean, rstd, norm.weight)
    for got, want in ((ya, y), (a.grad, dx), (norm.weight.grad, dg), (norm.bias.grad, dn), (one.weight.grad, dw1),
                      (one.bias.grad, db1), (two.weight.grad, dw2), (two.bias.grad, db2)):
        assert torch.equal(got, want)
    # every input is off by at most 2^-7 of the largest of 32 neighbours: a gradient's direction hardly moves
    for p, q in zip([a.grad, *(p.grad for p in model.parameters())], [b.grad, *(p.grad for p in plain.parameters())]):
        assert float(torch.nn.functional.cosine_similarity(p.double().flatten(), q.double().flatten(), dim=0)) > 0.998
    assert float((ya.detach().double() - yb.detach().double()).abs().max()) <= 8 * torch.finfo(dtype).eps * float(yb.detach().abs().max())


def test_what_autograd_holds():
    """A block's saved activations in bytes: one and a 32nd a value of each layer's input."""
    from cswap_amd import layers8

    rows, cols, hidden = 4096, 256, 1024
    x = randn(rows, cols, dtype=BF16)
    saved = {}
    for name, model in (("plain", block(cols, hidden, BF16)), ("8 bits", layers8.checkpoint_layers(block(cols, hidden, BF16)))):
        sizes = {}

        def pack(t):
            if t.numel() >= rows * cols:
                sizes[t.data_ptr()] = t.numel() * t.element_size()
            return t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = model(x.clone().requires_grad_())
        saved[name] = sum(sizes.values())
        y.sum().backward()
    values = rows * (cols + cols + hidden + hidden + cols)
    assert saved["8 bits"] == values * 33 // 32
    assert saved["plain"] >= 2 * values


def test_a_shared_checkpoint_and_partial_gradients():
    from cswap_amd import layers8, q8

    x = randn(50, 72, seed=13, dtype=BF16)
    w = [randn(40, 72, seed=14 + i, dtype=BF16).requires_grad_() for i in range(3)]
    leaf = x.clone().requires_grad_()
    held = layers8.hold(leaf)
    ys = [layers8.linear(leaf, v, None, held=held) for v in w]
    dys = [randn(50, 40, seed=20 + i, dtype=BF16) for i in range(3)]
    torch.autograd.backward(ys, dys)
    for v, dy in zip(w, dys):
        assert torch.equal(v.grad, q8.q8_weight_grad(dy, q8.q8_compress(x), bias=False)[0])
    # a frozen weight keeps nothing of x; a frozen input gets no gradient
    b = randn(40, seed=30, dtype=BF16).requires_grad_()
    y = layers8.linear(leaf.detach().requires_grad_(), w[0].detach(), b)
    assert all(t.dtype != torch.int8 for t in y.grad_fn.saved_tensors)
    y.backward(dys[0])
    assert torch.allclose(b.grad.float(), dys[0].float().sum(0), rtol=2 ** -7, atol=1e-2)
    with torch.no_grad():
        assert layers8.linear(x, w[0], b).grad_fn is None
        assert layers8.activation(x).grad_fn is None and layers8.layer_norm(x).grad_fn is None
    with pytest.raises(ValueError):
        layers8.linear(leaf, w[0], None, held=layers8.hold(x[:40]))


def test_without_gradients_nothing_is_made(monkeypatch):
    """Where gradients are off, parameters that could have them make no checkpoint, and results are the same."""
    from cswap_amd import layers8, q8

    model = layers8.checkpoint_layers(block(dtype=BF16))
    x = randn(30, 96, dtype=BF16, seed=35)
    want = model(x).detach()
    monkeypatch.setattr(q8, "_empty_checkpoint", None)
    with torch.no_grad():
        assert torch.equal(model(x), want)
        with torch.autocast("cuda", dtype=BF16):
            assert model(x.float()).dtype == BF16
    with torch.inference_mode():
        assert torch.equal(model(x), want)


def test_gradients_that_are_views():
    """What sum() and a transposition hand to backward: expanded and strided gradients, and inputs that are views."""
    from cswap_amd import layers8

    x = randn(33, 96, seed=40).requires_grad_()
    for f in (lambda v: layers8.activation(v), lambda v: layers8.layer_norm(v)):
        for view in (lambda v: v, lambda v: v.t().contiguous().t(), lambda v: v[::2], lambda v: v[:, 5:70]):
            a, b = (x.detach().clone().requires_grad_() for _ in range(2))
            f(view(a)).sum().backward()
            f(view(b).contiguous()).sum().backward()
            assert torch.equal(a.grad, b.grad)
            a.grad = b.grad = None
            out = f(view(a))
            out.t().backward(torch.ones(out.shape[1], out.shape[0], device=DEV).t().contiguous().t())
            f(view(b).contiguous()).backward(torch.ones_like(out))
            assert torch.equal(a.grad, b.grad)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_under_autocast(dtype):
    from cswap_amd import layers8

    plain, model = block(), layers8.checkpoint_layers(block())
    x = randn(64, 96, seed=41)
    grads = []
    for m in (plain, model):
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", dtype=dtype):
            y = m(leaf)
        assert y.dtype == dtype
        y.float().sum().backward()
        assert leaf.grad.dtype == F32 and all(p.grad.dtype == F32 for p in m.parameters())
        grads.append([leaf.grad, *(p.grad for p in m.parameters())])
    for p, q in zip(*grads):
        assert float(torch.nn.functional.cosine_similarity(p.double().flatten(), q.double().flatten(), dim=0)) > 0.998


def test_double_backward_and_other_types_are_refused():
    from cswap_amd import layers8

    x = randn(4, 32).requires_grad_()
    g, = torch.autograd.grad(layers8.activation(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with pytest.raises(TypeError):
        layers8.activation(x.double())
    with pytest.raises(ValueError):
        layers8.activation(x.cpu())


def test_layers_over_several_dimensions_and_those_left_alone():
    from cswap_amd import layers8
    from torch import nn

    m = layers8.checkpoint_layers(nn.Sequential(nn.LayerNorm((6, 8)), nn.GELU("tanh"), nn.SiLU(inplace=True), nn.LayerNorm(20000),
                                                nn.Linear(8, 8, bias=False))).to(DEV)
    assert [type(c).__name__ for c in m] == ["LayerNorm8", "GELU8", "SiLU", "LayerNorm", "Linear8"]
    x = randn(5, 6, 8, seed=42)
    want = torch.nn.functional.layer_norm(x.double(), (6, 8), m[0].weight.double(), m[0].bias.double())
    assert float((m[0](x).detach().double() - want.detach()).abs().max()) < 1e-5
    want = torch.nn.functional.gelu(x.double(), approximate="tanh")
    assert float((m[1](x).double() - want).abs().max()) < 1e-6
    with pytest.raises(ValueError):
        m[0](x[..., :4])


# ---------------------------------------------------------------- streams and graphs
def test_on_another_stream():
    from cswap_amd import q8

    x = randn(4096, 768, dtype=BF16, seed=50)
    dy = randn(4096, 512, dtype=BF16, seed=51)
    want = q8.q8_weight_grad(dy, q8.q8_compress(x))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        held = q8.q8_compress(x)
        got = q8.q8_weight_grad(dy, held)
    held.record_stream(torch.cuda.current_stream())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_graphs_of_the_whole_run():
    """Two captured training steps of a block's kernels, replayed in turn with eager work between them: every replay
    gives what the eager calls give."""
    from cswap_amd import q8

    x = torch.zeros(1000, 192, device=DEV, dtype=BF16)
    dy = torch.zeros(1000, 320, device=DEV, dtype=BF16)
    weight, gain = randn(320, 192, dtype=BF16, seed=60), randn(192, dtype=BF16, seed=61)

    def step():
        h, mean, rstd, held = q8.layer_norm(x, gain, gain)
        y, kept = q8.q8_act(torch.nn.functional.linear(h, weight), "silu")
        d = q8.q8_act_backward(dy, kept, "silu")
        dw, db = q8.q8_weight_grad(d, q8.q8_compress(h))
        return [y, dw, db, *q8.layer_norm_backward(d @ weight, held, mean, rstd, gain)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for turn in range(6):
        x.copy_(randn(1000, 192, dtype=BF16, seed=70 + turn))
        dy.copy_(randn(1000, 320, dtype=BF16, seed=80 + turn))
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(outs[turn % 2], want)), turn


# ---------------------------------------------------------------- saved-tensor hooks
def test_hooks_hold_what_a_model_saves():
    from cswap_amd.hooks import hold_saved_tensors

    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 32, 3, padding=1), torch.nn.ReLU(), torch.nn.Conv2d(32, 16, 3, padding=1),
                                torch.nn.Tanh(), torch.nn.Flatten(), torch.nn.Linear(16 * 15 * 15, 10)).to(DEV)
    x = randn(8, 3, 15, 15, seed=90)
    grads = []
    for ctx in (None, hold_saved_tensors(min_bytes=1 << 10)):
        model.zero_grad()
        if ctx is None:
            loss = model(x).square().sum()
        else:
            with ctx:
                loss = model(x).square().sum()
        loss.backward()
        grads.append([p.grad.clone() for p in model.parameters()])
    assert ctx.stats["held"] >= 3 and ctx.stats["bytes_held"] * 3.8 < ctx.stats["bytes_in"]
    for p, q in zip(*grads):
        assert float(torch.nn.functional.cosine_similarity(p.double().flatten(), q.double().flatten(), dim=0)) > 0.998


def test_hooks_give_back_what_a_checkpoint_stands_for():
    from cswap_amd.hooks import hold_saved_tensors

    x = randn(300, 17, seed=91)
    a = x.clone().requires_grad_()
    with hold_saved_tensors(min_bytes=0):
        y = (a * 1.0).tanh()                                        # tanh saves its result
    y.backward(torch.ones_like(y))
    kept = ref.held(y.detach().reshape(1, -1), keep_sign=True).view(300, 17)
    want = 1 - kept ** 2
    assert float((a.grad.cpu().double() - want).abs().max()) <= 4 * ref.U


def test_swapping_and_checkpoints_in_one_model():
    """Layers with checkpoints under the swapping hooks: their checkpoints pass through, what else is saved is swapped."""
    from cswap_amd import layers8
    from cswap_amd.hooks import swap_saved_tensors
    from cswap_amd.swap import NONE, SwapEngine

    eng = SwapEngine(pinned_bytes=64 << 20, device_bytes=64 << 20)
    x = randn(2048, 96, seed=92)
    grads = []
    for swapped in (False, True):
        model = torch.nn.Sequential(layers8.checkpoint_layers(block()), torch.nn.Tanh(), torch.nn.Softmax(-1)).to(DEV)
        leaf = x.clone().requires_grad_()
        if swapped:
            ctx = swap_saved_tensors(eng, policy=NONE, min_bytes=1 << 16)
            with ctx:
                y = model(leaf)
            y.square().sum().backward()
            assert ctx.stats["swapped"] >= 1
            ctx.close()
        else:
            model(leaf).square().sum().backward()
        grads.append([leaf.grad, *(p.grad for p in model.parameters())])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    eng.close()
