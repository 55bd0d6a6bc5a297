"""Traces and forward-mode derivatives, of which the kernels' outputs know nothing, are refused: host checks, no GPU."""
import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad  # noqa: E402

pytestmark = pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")


def checkpoint(rows=4, cols=40, dtype=torch.float32):
    from cswap_amd.q8 import Checkpoint8

    g = -(-cols // 32)
    return Checkpoint8(torch.zeros(rows, g * 32, dtype=torch.int8), torch.zeros(rows, g, dtype=torch.uint8), (rows, cols), dtype)


def calls():
    from cswap_amd import q8

    held, s = checkpoint(), torch.zeros(4)
    return {"compress": q8.q8_compress, "act": q8.q8_act, "act_backward": lambda x: q8.q8_act_backward(x, held),
            "norm": q8.layer_norm, "norm_weight": lambda x: q8.layer_norm(torch.zeros(4, 40), x[0]),
            "norm_backward": lambda x: q8.layer_norm_backward(x, held, s, s),
            "norm_backward_of_x": lambda x: q8.layer_norm_backward(torch.zeros(4, 40), x, s, s),
            "weight_grad": lambda x: q8.q8_weight_grad(x, held),
            "decompress": lambda x: q8.q8_decompress(held, out=x)}


@pytest.mark.parametrize("name", sorted(calls()))
def test_forward_mode_is_refused(name):
    x = torch.randn(4, 40)
    with forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match="forward-mode"):
            calls()[name](forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(ValueError, match="device memory"):          # a tensor without a tangent is one like any other
            calls()[name](x)
    with pytest.raises(ValueError, match="device memory"):
        calls()[name](x)


@pytest.mark.parametrize("name", sorted(calls()))
def test_traces_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx

    def f(x):
        calls()[name](x)
        return x

    x = torch.randn(4, 40)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, x, check_trace=False)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f)(x)


@pytest.mark.parametrize("layer", ["activation", "layer_norm"])
def test_layers_refuse_where_gradients_are_off(layer):
    from cswap_amd import layers8

    x = torch.randn(4, 40)
    with torch.no_grad():
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            getattr(layers8, layer)(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(getattr(layers8, layer), x, check_trace=False)


@pytest.mark.parametrize("layer", ["activation", "layer_norm", "linear"])
def test_layers_refuse_a_trace_where_gradients_are_on(layer):
    from cswap_amd import layers8

    x, w = torch.randn(4, 40, requires_grad=True), torch.randn(8, 40, requires_grad=True)
    inputs = (x, w) if layer == "linear" else (x,)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(getattr(layers8, layer), inputs, check_trace=False)


def test_modes_that_only_look_are_not_refused():
    from torch.utils.flop_counter import FlopCounterMode

    with FlopCounterMode(display=False), torch.no_grad():
        for f in calls().values():
            with pytest.raises(ValueError, match="device memory"):
                f(torch.randn(4, 40))
