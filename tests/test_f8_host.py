"""Products in 8-bit floating point without a GPU: the reference is torch's own e4m3, sizes, refusals."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import f8_reference as fref  # noqa: E402

from cswap_amd import _lib, f8, layers8  # noqa: E402

A = 1 << 20


def test_the_reference_rounds_as_e4m3_does():
    x = torch.randn(40, 300, dtype=torch.float64) * torch.exp(3 * torch.randn(40, 300, dtype=torch.float64))
    x = x.float()
    for rows in (1, 128):
        value, scales = fref.held(x, rows)
        unit = torch.exp2(scales.double() - 127).repeat_interleave(rows, 0)[:40].repeat_interleave(128, 1)[:, :300]
        codes = (x.double() / unit).float().to(torch.float8_e4m3fn)
        assert torch.equal(codes.double() * unit, value)
        assert float((x.double() / unit).abs().max()) <= 448 and bool(((value - x.double()).abs() <= torch.maximum(x.double().abs() / 16, unit * 2.0 ** -10)).all())


def test_scales_at_the_border():
    x = torch.zeros(4, 128)
    x[0, 0], x[1, 0], x[2, 0], x[3, 5] = 448.0, 448.0 * (1 + 2.0 ** -23), 1.75, 2.0 ** -140
    assert fref.held(x, 1)[1].flatten().tolist() == [127, 128, 119, 1]


def pack(w=A, dtype=0, n=4, k=4, stride=0, codes=A, turned=A, scales=A):
    return _lib.lib().cswap_f8_pack_weight(w, dtype, n, k, stride, codes, turned, scales, None)


def linear(x=A, dtype=0, rows=40, k=4, stride=0, codes=A, scales=A, n=4, turned=0, bias=A, kind=0, y=A, out=0, y_stride=0, ws=A, room=1 << 30):
    return _lib.lib().cswap_f8_linear(x, dtype, rows, k, stride, codes, scales, n, turned, bias, kind, y, out, y_stride, ws, room, None)


def test_argument_errors_do_not_launch():
    for kw in (dict(w=0), dict(w=A + 2), dict(dtype=3), dict(n=0), dict(k=0), dict(stride=3), dict(codes=0), dict(codes=A + 8), dict(turned=A + 8), dict(scales=0)):
        assert pack(**kw) == -1, kw
    for kw in (dict(n=(1 << 20) + 1), dict(k=(1 << 20) + 1)):
        assert pack(**kw) == -2 and linear(**kw) == -2, kw
    assert linear(rows=1 << 31) == -2
    for kw in (dict(x=0), dict(x=A + 2), dict(dtype=3), dict(out=-1), dict(kind=5), dict(k=0), dict(n=0), dict(stride=2), dict(y_stride=3), dict(codes=0), dict(codes=A + 4),
               dict(scales=0), dict(turned=2), dict(bias=A + 2), dict(y=0), dict(y=A + 1), dict(ws=0), dict(ws=A + 8)):
        assert linear(**kw) == -1, kw
    assert linear(room=10) == -4
    assert linear(rows=0, x=0, y=0, codes=0, scales=0, bias=0, ws=0) == 0


def test_workspaces():
    f = _lib.lib().cswap_f8_linear_workspace_bytes
    assert f(0, 100) == 0 and f(1, 100) == 0 and f(100, 0) == 0
    assert f(1000, 129) == 2 * 1024 * 129                                         # whole tiles of 256 rows
    assert f(1 << 31, 128) == 0 and f(100, (1 << 20) + 1) == 0


def test_weights_have_the_arrays_of_their_shape():
    codes, scales = torch.zeros(256, 128, dtype=torch.float8_e4m3fn), torch.zeros(2, 1, dtype=torch.uint8)
    held = f8.F8Weight(codes, scales, (200, 100), torch.bfloat16)
    assert held.turned is None and tuple(held.shape) == (200, 100)
    assert tuple(f8.f8_weight_values(held).shape) == (200, 100)
    turned = torch.zeros(128, 256, dtype=torch.float8_e4m3fn)
    f8.F8Weight(codes, scales, (200, 100), torch.bfloat16, turned)
    for bad in ((codes[:128], scales), (codes, scales.t()), (codes.view(torch.uint8), scales), (codes, scales.int()), (codes, scales, codes)):
        with pytest.raises(ValueError):
            f8.F8Weight(bad[0], bad[1], (200, 100), torch.bfloat16, *bad[2:])
    with pytest.raises(TypeError):
        f8.F8Weight(codes, scales, (200, 100), torch.float64)
    with pytest.raises(ValueError, match="backward=False"):
        f8.f8_linear_backward(torch.zeros(3, 200), held)
    with pytest.raises(ValueError, match="device memory"):
        f8.f8_linear(torch.zeros(3, 100), held)
    with pytest.raises(ValueError, match="device memory"):
        f8.f8_weight(torch.zeros(3, 100))
    with pytest.raises(TypeError):
        f8.f8_linear(torch.zeros(3, 100, dtype=torch.float64), held)


def test_which_layers_are_converted():
    from torch import nn

    model = nn.Sequential(nn.Linear(3, 4), nn.GELU())
    assert [type(m) for m in layers8.checkpoint_layers(model, f8=True)] == [layers8.LinearF8, layers8.GELU8]
    model = nn.Sequential(nn.Linear(3, 4))
    assert type(layers8.checkpoint_layers(model)[0]) is layers8.Linear8


def test_sizes_beyond_a_launch_are_refused():
    M = 1 << 20
    for kw in (dict(n=1 << 18, k=1 << 18), dict(n=M, k=1 << 16)):
        assert pack(**kw, stride=M) == -2, kw
        assert linear(rows=1, **kw) == -2, kw
    for kw in (dict(rows=1 << 28, k=1), dict(rows=(1 << 27) + 1, k=129), dict(rows=(1 << 24) - 15, k=2048), dict(rows=1 << 29, n=1 << 9)):
        assert linear(**kw) == -2, kw
    f = _lib.lib().cswap_f8_linear_workspace_bytes
    assert f(1 << 28, 1) == 0 and f((1 << 28) - 16, 1) == (1 << 28) * 129


def test_tensors_on_another_device_make_that_device_current(monkeypatch):
    import contextlib

    from cswap_amd import api, q8

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
        cswap_f8_linear_workspace_bytes = staticmethod(_lib.lib().cswap_f8_linear_workspace_bytes)

        @staticmethod
        def cswap_f8_pack_weight(*a):
            launched.append(("weight", current[0], a[-1]))
            return 0

        @staticmethod
        def cswap_f8_linear(*a):
            launched.append(("product", current[0], a[-1]))
            return 0

    made = torch.empty
    monkeypatch.setattr(q8, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(api, "_raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(f8, "lib", lambda: Lib)
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: made(*a, **kw).as_subclass(OnDevice1))
    held = f8.f8_weight(torch.zeros(30, 40).as_subclass(OnDevice1))
    f8.f8_linear(torch.zeros(20, 40).as_subclass(OnDevice1), held)
    f8.f8_linear_backward(torch.zeros(20, 30).as_subclass(OnDevice1), held)
    assert launched == [("weight", 1, 1001), ("product", 1, 1001), ("product", 1, 1001)] and current == [0]
    monkeypatch.undo()
    with pytest.raises(ValueError):
        f8.f8_linear(torch.zeros(20, 40), held)                     # a tensor elsewhere than the weights


def watched():
    codes, scales = torch.zeros(128, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8)
    held = f8.F8Weight(codes, scales, (40, 40), torch.float32, codes.clone())
    plain = torch.zeros(4, 40)
    return {"weight": f8.f8_weight, "product": lambda x: f8.f8_linear(x, held), "bias": lambda x: f8.f8_linear(plain, held, x[0]),
            "backward": lambda x: f8.f8_linear_backward(x, held), "layer": lambda x: layers8.linear_f8(x, torch.zeros(40, 40), weight8=held),
            "layer_weight": lambda x: layers8.linear_f8(plain, x)}


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", sorted(watched()))
def test_traces_and_forward_mode_are_refused(name):
    from torch.autograd import forward_ad

    x = torch.randn(4, 40)
    with torch.no_grad():
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            watched()[name](forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(watched()[name], x, check_trace=False)


def test_the_products_that_are_tested_run_every_form():
    """Whatever the rule that chooses a form becomes, each has a product of its own in either type of results, and large tiles have even and odd numbers
    of blocks and fewer and more tiles than compute units."""
    import f8_tile_cases as tiles

    form = _lib.lib().cswap_test_f8_linear_form
    for want, bits, rows, n, k in tiles.CASES:
        assert [form(rows, n, k, out) for out in ((1, 2) if bits == 16 else (0,))] == [want] * (2 if bits == 16 else 1), (want, bits, rows, n, k)
        assert n % 32 and (rows % 32 or want < 128) and k % 128
    assert {(f, b) for f, b, *_ in tiles.CASES} == {(f, b) for f in (0, 32, 64, 128, 192, 256) for b in (16, 32)}
    for f in (192, 256):
        for bits in (16, 32):
            kinds = {(-(-k // 128) % 2, -(-rows // 256) * -(-n // f) > 256) for g, b, rows, n, k in tiles.CASES if (g, b) == (f, bits)}
            assert kinds == {(0, False), (0, True), (1, False), (1, True)}, (f, bits)
    assert form(0, 5, 5, 0) == 0 and form(40, 0, 5, 0) == -1 and form(1 << 31, 5, 5, 0) == -1
    x = tiles.blocks(300, 300, 1, "cpu", 1)
    assert set(x.abs().unique().tolist()) == {0.0, 1.0, 2.0, 4.0, 8.0} and fref.held(x, 1)[0].equal(x.double())
    assert set(fref.held(x, 1)[1].flatten().tolist()) == {119, 120, 121, 122}


def test_layers_that_hold_their_input_become_layers_of_8_bit_products_too():
    """One call after the other on a model, in whatever order, gives what one call with both gives; classes derived from either are left alone."""
    from torch import nn

    class Mine(layers8.Linear8):
        pass

    model = nn.Sequential(nn.Linear(3, 4), Mine(4, 4), nn.GELU(), nn.LayerNorm(4))
    weights = [p.data_ptr() for p in model.parameters()]
    layers8.checkpoint_layers(model)
    assert [type(m) for m in model] == [layers8.Linear8, Mine, layers8.GELU8, layers8.LayerNorm8]
    layers8.checkpoint_layers(model, f8=True)
    assert [type(m) for m in model] == [layers8.LinearF8, Mine, layers8.GELU8, layers8.LayerNorm8]
    layers8.checkpoint_layers(model)                                # what is there stays
    assert [type(m) for m in model] == [layers8.LinearF8, Mine, layers8.GELU8, layers8.LayerNorm8]
    assert [p.data_ptr() for p in model.parameters()] == weights
    wide = nn.Linear(3, 4)
    wide.__class__ = layers8.Linear8
    wide.weight = nn.Parameter(torch.empty(0, 3))
    assert type(layers8.checkpoint_layers(wide, f8=True)) is layers8.Linear8


def test_codes_of_another_weight_are_refused_with_and_without_gradients():
    codes, scales = torch.zeros(128, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8)
    held = f8.F8Weight(codes, scales, (40, 30), torch.float32, codes.clone())
    x, w = torch.zeros(4, 30), torch.zeros(50, 30, requires_grad=True)
    for mode in (torch.no_grad, torch.enable_grad):
        with mode(), pytest.raises(ValueError, match="weight8"):
            layers8.linear_f8(x, w, None, weight8=held)
