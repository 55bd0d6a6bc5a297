"""What the saved-tensor hooks hold in 8 bits: signs, probabilities, masks and weights, against 64-bit forms."""
import math
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


def held_few(x):
    """What the hooks hold of a tensor: groups of 32 through the whole of it, rounded to nearest, and where one or two of a
    group's values would become 0 these as one step with their sign."""
    flat = x.detach().cpu().reshape(1, -1)
    codes, scales = ref.pack(flat)
    signed, _ = ref.pack(flat, True)
    lost = ((codes == 0) & (signed != 0)).view(-1, 32)
    few = (lost.sum(1, keepdim=True) <= 2).expand(-1, 32).reshape(codes.shape)
    return ref.unpack(torch.where(few, signed, codes), scales, flat.shape[1]).view(x.shape)


def what_is_held(t):
    """What backward gets for a contiguous, non-leaf ``t``."""
    from cswap_amd.hooks import hold_saved_tensors

    class Keep(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            ctx.save_for_backward(x)
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            seen.append(ctx.saved_tensors[0].detach().clone())
            return g

    seen = []
    leaf = t.clone().requires_grad_()
    x = leaf * 1.0
    ctx = hold_saved_tensors(min_bytes=0)
    with ctx:
        y = Keep.apply(x)
    assert ctx.stats["held"] == 1
    y.backward(torch.ones_like(y))
    return seen[0]


# ---------------------------------------------------------------- signs
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_many_small_values_beside_a_large_one_are_not_raised(dtype):
    """A value that rounds to 0 beside two more such or fewer is held as one step with its sign, off by less than a step,
    2^-6 of the largest; among more it is held as 0, and every error is at most 2^-7 of the largest."""
    x = torch.zeros(70, 32, dtype=torch.float64)
    x[:, 5] = 64.0
    for row in range(70):
        small = row % 35
        x[row, [i for i in range(32) if i != 5][:small]] = 1e-3 if row < 35 else -1e-3
    x = x.to(dtype)
    got = what_is_held(x.to(DEV)).cpu().double()
    for row in range(70):
        there = min(row % 35, 31)
        want = (1.0 if row < 35 else -1.0) if there <= 2 else 0.0
        small = (x[row] != 0) & (x[row].abs() < 1)
        assert bool((got[row][small] == want).all()) and bool((got[row][x[row] == 0] == 0).all()), row


@pytest.mark.parametrize("sigma", [1.0, 3.0, 9.0, 16.0])
def test_softmax_keeps_its_sums_and_gradient(sigma):
    """Held to the byte as defined, whose 64-bit form has rows that sum to 0.99 to 1.01 and a gradient that is off by less
    than 2 % for these inputs (with a sign for every value: up to 1.48, and 34 %)."""
    from cswap_amd.hooks import hold_saved_tensors

    x, dy = randn(200, 512, seed=1, scale=sigma), randn(200, 512, seed=2)
    probs = torch.softmax(x, -1)
    held = what_is_held(probs).cpu().double()
    assert torch.equal(held, held_few(probs))
    assert 0.97 < float(held.sum(1).min()) and float(held.sum(1).max()) < 1.02 and abs(float(held.sum(1).mean()) - 1) < 0.01
    leaf = x.clone().requires_grad_()
    with hold_saved_tensors(min_bytes=0):
        p = torch.softmax(leaf * 1.0, -1)
    p.backward(dy)
    d, probs, got = dy.cpu().double(), probs.cpu().double(), leaf.grad.cpu().double()
    exact = probs * (d - (probs * d).sum(1, keepdim=True))
    want = held * (d - (held * d).sum(1, keepdim=True))              # softmax's gradient of what is held
    size = held * (d.abs() + (held * d.abs()).sum(1, keepdim=True))
    assert bool(((got - want).abs() <= 520 * ref.U * size + 2.0 ** -149).all())
    assert float((want - exact).norm() / exact.norm()) < 0.02


def test_attention_through_the_hooks():
    """Probabilities are saved by the softmax and by the product behind it: neither's gradient is biased."""
    from cswap_amd.hooks import hold_saved_tensors

    q, k, v = (randn(4, 100, 64, seed=3 + i, scale=s) for i, s in enumerate((2.0, 2.0, 1.0)))
    dy = randn(4, 100, 64, seed=6)
    grads = []
    for dtype, ctx in ((torch.float64, None), (F32, hold_saved_tensors(min_bytes=1 << 10))):
        a, b, c = (t.cpu().double().requires_grad_() if ctx is None else t.clone().requires_grad_() for t in (q, k, v))
        if ctx is None:
            y = torch.softmax(a @ b.transpose(-1, -2).contiguous() / 8.0, -1) @ c
            y.backward(dy.cpu().double())
        else:
            with ctx:
                y = torch.softmax(torch.matmul(a, b.transpose(-1, -2).contiguous()) / 8.0, -1) @ c
            y.backward(dy)
            assert ctx.stats["held"] >= 2
        grads.append([t.grad.cpu().double() for t in (a, b, c)])
    for want, got in zip(*grads):
        assert float((got - want).norm() / want.norm()) < 0.03


@pytest.mark.parametrize("inplace", [False, True])
def test_a_relus_gradient_is_exact_beside_outliers(inplace):
    """A ReLU's own result keeps the sign of every value, however many are small beside the largest; the operator that
    takes it next gets values rounded to nearest."""
    from cswap_amd.hooks import hold_saved_tensors

    x = randn(64, 256, seed=7)
    x[:, ::32] *= 1000.0
    dy = randn(64, 256, seed=8)
    leaf, scale = x.clone().requires_grad_(), torch.ones(256, device=DEV, requires_grad=True)
    ctx = hold_saved_tensors(min_bytes=0)
    with ctx:
        y = torch.nn.functional.relu(leaf * 1.0, inplace=inplace)
        z = y * scale                                               # saves y, too
    z.backward(dy)
    assert ctx.stats["held"] == 2
    assert torch.equal(leaf.grad, torch.where(x > 0, dy, torch.zeros_like(dy)))
    kept, d = held_few(torch.relu(x)), dy.cpu().double()
    err = (scale.grad.cpu().double() - (d * kept).sum(0)).abs()      # 64 products, summed in fp32 in any order
    assert bool((err <= 65 * ref.U * (d * kept).abs().sum(0)).all())


def test_signs_on_request():
    """``keep_sign``: nothing that is not 0 becomes 0, for backward passes that divide by what they saved."""
    from cswap_amd.hooks import hold_saved_tensors

    x = torch.full((8, 64), 1e-4, device=DEV)
    x[:, ::32] = 1.0
    leaf = x.clone().requires_grad_()
    with hold_saved_tensors(min_bytes=0, keep_sign=True):
        y = torch.log(leaf * 1.0)
    y.backward(torch.ones_like(y))
    assert bool((leaf.grad[:, ::32] == 1).all()) and bool((leaf.grad[:, 1:32] == 64).all())


# ---------------------------------------------------------------- masks
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", [(8, 64), (5, 45)])
def test_minus_infinity_is_held_beside_its_neighbours(dtype, shape):
    """Masked places stay minus infinity; the others are held as if those were not there.  NaN and plus infinity make their
    group NaN."""
    x = randn(*shape, dtype=dtype, seed=9, scale=3.0)
    x[1, ::3] = -math.inf
    x[2] = -math.inf
    x[3, 7] = -math.inf
    got = what_is_held(x).cpu().double()
    masked = torch.isinf(x.cpu())
    want = held_few(x.masked_fill(masked.to(DEV), 0.0))
    assert torch.equal(got, torch.where(masked, torch.full_like(want, -math.inf), want.to(dtype).double()))
    x.view(-1)[40], x.view(-1)[100] = math.nan, math.inf
    nan = torch.isnan(what_is_held(x).cpu()).view(-1).nonzero().flatten().tolist()
    assert nan == [*range(32, 64), *range(96, 128)]


def test_masked_logits_have_finite_gradients():
    """logsumexp saves its masked input: gradients within what the held logits, off by 2^-7 of the largest of 32, give."""
    from cswap_amd.hooks import hold_saved_tensors

    x = randn(16, 96, seed=10)
    mask = torch.rand(16, 96, generator=torch.Generator().manual_seed(11)) < 0.3
    mask[:, 5] = False
    leaf = x.clone().requires_grad_()
    ctx = hold_saved_tensors(min_bytes=1 << 10)
    with ctx:
        y = torch.logsumexp(leaf.masked_fill(mask.to(DEV), -math.inf), -1)
    y.sum().backward()
    assert ctx.stats["held"] == 1
    got, want = leaf.grad.cpu().double(), torch.softmax(x.cpu().double().masked_fill(mask, -math.inf), -1)
    assert bool((got[mask] == 0).all())
    off = 2.0 ** -7 * group_max(x.cpu().double().masked_fill(mask, 0.0).view(-1)).view(16, 96)
    assert bool(((got - want).abs() <= want * (torch.expm1(2 * off) + 200 * ref.U)).all())


@pytest.mark.parametrize("lowest", [-math.inf, torch.finfo(F32).min])
def test_log_probabilities_are_kept_as_they_are(lowest):
    """log_softmax saves its result for its exponential: masked or not, the gradient is that without the hooks."""
    from cswap_amd.hooks import hold_saved_tensors

    x, target = randn(64, 1000, seed=12), torch.arange(64, device=DEV)
    x[:, 500::7] = lowest
    grads = []
    for ctx in (None, hold_saved_tensors(min_bytes=0)):
        leaf = x.clone().requires_grad_()
        if ctx is None:
            loss = torch.nn.functional.cross_entropy(leaf, target)
        else:
            with ctx:
                loss = torch.nn.functional.cross_entropy(leaf, target)
        loss.backward()
        grads.append(leaf.grad)
    assert bool(torch.isfinite(grads[0]).all()) and torch.equal(*grads)


def group_max(x):
    """For every value of a 1-D tensor the largest magnitude among its 32."""
    n = x.numel()
    g = torch.nn.functional.pad(x.abs(), (0, -n % 32)).view(-1, 32)
    return g.amax(1, keepdim=True).expand_as(g).reshape(-1)[:n]


# ---------------------------------------------------------------- weights
@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_weights_pass_through_under_autocast(dtype):
    """Layers with checkpoints, hooks and autocast together: the hooks have nothing to hold, and every gradient is to the
    bit that without them."""
    from cswap_amd import layers8
    from cswap_amd.hooks import hold_saved_tensors
    from torch import nn

    x = randn(128, 96, seed=13)
    grads = []
    for hooked in (False, True):
        torch.manual_seed(14)
        model = nn.Sequential(nn.LayerNorm(96), nn.Linear(96, 224), nn.GELU(), nn.Linear(224, 96), nn.SiLU()).to(DEV)
        layers8.checkpoint_layers(model)
        leaf = x.clone().requires_grad_()
        ctx = hold_saved_tensors(min_bytes=1 << 10)
        with torch.autocast("cuda", dtype=dtype):
            if hooked:
                with ctx:
                    y = model(leaf)
            else:
                y = model(leaf)
        assert ctx.stats["held"] == 0
        y.float().square().sum().backward()
        grads.append([leaf.grad, *(p.grad for p in model.parameters())])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_weights_that_are_computed_pass_through():
    """A norm over several dimensions takes its weight as a view, a linear layer one that was made of others."""
    from cswap_amd import layers8
    from cswap_amd.hooks import hold_saved_tensors

    x, w = randn(32, 6, 16, seed=15), randn(40, 96, seed=16)
    grads = []
    for ctx in (None, hold_saved_tensors(min_bytes=0)):
        norm = layers8.checkpoint_layers(torch.nn.LayerNorm((6, 16))).to(DEV)
        with torch.no_grad():
            norm.weight.copy_(randn(6, 16, seed=17))
        leaves = x.clone().requires_grad_(), w.clone().requires_grad_()

        def forward():
            return layers8.linear(norm(leaves[0]).view(32, 96), leaves[1] * 0.3, None)

        if ctx is None:
            y = forward()
        else:
            with ctx:
                y = forward()
            assert ctx.stats["held"] == 0
        y.square().sum().backward()
        grads.append([norm.weight.grad, norm.bias.grad, *(t.grad for t in leaves)])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_weights_of_torchs_own_layers_pass_through():
    """A convolution's weight, cast by autocast, and a view of a parameter; their inputs are held."""
    from cswap_amd.hooks import hold_saved_tensors

    conv = torch.nn.Conv2d(8, 16, 3).to(DEV)
    x = randn(2, 8, 12, 12, seed=18).requires_grad_()
    shapes = []

    class Watch(hold_saved_tensors):
        def _eligible(self, t):
            take = super()._eligible(t)
            if take:
                shapes.append(tuple(t.shape))
            return take

    with Watch(min_bytes=0):
        with torch.autocast("cuda", dtype=BF16):
            conv(x * 1.0)
        torch.matmul((x * 1.0).view(-1, 16), conv.weight.view(16, 72))
    assert (16, 8, 3, 3) not in shapes and (16, 72) not in shapes
    assert (2, 8, 12, 12) in shapes and (144, 16) in shapes


def test_tensors_of_other_layouts_are_saved_as_usual():
    from cswap_amd.hooks import hold_saved_tensors

    dense, eye = randn(6, 8, seed=19), torch.eye(6, device=DEV)
    for make in (lambda: eye.to_sparse_csr(), lambda: eye.to_sparse()):
        grads = []
        for ctx in (hold_saved_tensors(min_bytes=0), torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t)):
            s, d = make().requires_grad_(), dense.clone().requires_grad_()
            with ctx:
                y = torch.sparse.mm(s * 2.0, d)
            y.sum().backward()
            grads.append(d.grad)
        assert torch.equal(*grads)
    nested = torch.nested.nested_tensor([dense, dense[:3]])
    for ctx in (hold_saved_tensors(min_bytes=0), torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t)):
        leaf = nested.clone().detach().requires_grad_()
        with ctx:
            y = torch.relu(leaf * 2.0)
        torch.nested.to_padded_tensor(y, 0.0).sum().backward()
        grads.append(torch.nested.to_padded_tensor(leaf.grad, 0.0))
    assert torch.equal(*grads[2:])


# ---------------------------------------------------------------- the codec that the hooks use, by itself
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_rows_with_gaps_and_padding(dtype):
    """The hooks hold tensors as one row; the functions take rows, with groups that begin at each."""
    from cswap_amd import q8

    x = randn(9, 130, dtype=dtype, seed=20)
    x[2, 5:60], x[3, 64:96] = -math.inf, 0.0
    x[3, 70], x[4, 0] = -math.inf, 1e4
    big = torch.full((9, 141), math.nan, dtype=dtype, device=DEV)
    big[:, 3:133] = x
    got = q8._give_back(q8.q8_compress(big[:, 3:133], keep_sign=q8._HOLD)).cpu().double()
    masked = torch.isinf(x.cpu())
    rows = x.masked_fill(masked.to(DEV), 0.0)
    want = torch.cat([held_few(r) for r in rows]).view(9, 130).to(dtype).double()
    assert torch.equal(got, want.masked_fill(masked, -math.inf))


def test_in_a_graph():
    """Recorded, and replayed with eager work between: every replay holds and gives back what the eager calls do."""
    from cswap_amd import q8

    x = torch.zeros(300, 193, device=DEV)

    def there_and_back():
        return q8._give_back(q8.q8_compress(x, flat=True, keep_sign=q8._HOLD))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there_and_back()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = there_and_back()
    for turn in range(4):
        x.copy_(randn(300, 193, seed=21 + turn))
        x[turn] = -math.inf
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, there_and_back()) and bool((out[turn] == -math.inf).all())
