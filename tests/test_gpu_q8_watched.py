"""Layers with checkpoints and the hooks under a trace and under forward-mode differentiation."""
import pytest

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")]

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad  # noqa: E402


@pytest.mark.parametrize("grad", [True, False])
def test_a_block_is_not_traced(grad):
    from cswap_amd import layers8
    from torch import nn

    model = layers8.checkpoint_layers(nn.Sequential(nn.Linear(96, 224), nn.GELU(), nn.LayerNorm(224))).cuda()
    x = torch.randn(37, 96, device="cuda")
    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(model, x, check_trace=False)
    assert not model(x).isnan().any()                                # nothing of the trace is left


def test_forward_mode_beside_kernels():
    from cswap_amd import layers8
    from cswap_amd.hooks import hold_saved_tensors

    x = torch.randn(8, 64, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for on in (True, False):
            with torch.set_grad_enabled(on):
                for f in (layers8.activation, layers8.layer_norm, lambda t: layers8.linear(t, x.clone().requires_grad_(on))):
                    if on or f in (layers8.activation, layers8.layer_norm):
                        with pytest.raises(RuntimeError):
                            f(dual)
        assert torch.equal(layers8.activation(x), layers8.activation(x))
        # forward over reverse: what torch saves with a tangent is left to torch
        grads = []
        for ctx in (hold_saved_tensors(min_bytes=0), torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t)):
            leaf = x.clone().requires_grad_()
            with ctx:
                y = torch.tanh(forward_ad.make_dual(leaf, torch.ones_like(x)) * 1.0)
            grads.append(torch.autograd.grad(y.sum(), leaf)[0])
        assert float((forward_ad.unpack_dual(grads[0]).primal - forward_ad.unpack_dual(grads[1]).primal).abs().max()) < 2.0 ** -5
