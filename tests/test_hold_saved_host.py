"""What the saved-tensor hooks take and what their calls refuse: host checks, no GPU."""
import pytest

torch = pytest.importorskip("torch")

ARG, UNSUPPORTED = -1, -2
A = 1 << 20          # an aligned address that is never followed


def test_the_hooks_codec_refuses_what_the_codec_does():
    from cswap_amd import _lib

    pack, unpack = _lib.lib().cswap_q8_pack, _lib.lib().cswap_q8_unpack_held
    assert pack(None, 0, 4, 32, 0, 2, A, A, None) == ARG and pack(A, 3, 4, 32, 0, 2, A, A, None) == ARG
    assert pack(A, 0, 4, 0, 0, 2, A, A, None) == ARG and pack(A, 0, 1 << 29, 32, 0, 2, A, A, None) == UNSUPPORTED
    assert unpack(None, A, 4, 32, A, 0, 0, None) == ARG and unpack(A + 4, A, 4, 32, A, 0, 0, None) == ARG
    assert unpack(A, None, 4, 32, A, 0, 0, None) == ARG and unpack(A, A, 4, 32, None, 0, 0, None) == ARG
    assert unpack(A, A, 4, 32, A, 7, 0, None) == ARG and unpack(A, A, 4, 0, A, 0, 0, None) == ARG
    assert unpack(A, A, 4, 32, A, 0, 31, None) == ARG and unpack(A, A, 1 << 29, 32, A, 0, 0, None) == UNSUPPORTED
    assert unpack(None, None, 0, 32, None, 0, 0, None) == 0


def test_layers_save_their_weights_as_leaves():
    """Hooks take what is no leaf: a weight that was cast or computed is none, but is no activation either."""
    from cswap_amd import layers8
    from cswap_amd.q8 import Checkpoint8

    x, w = torch.randn(4, 32, requires_grad=True), torch.randn(8, 32, requires_grad=True)
    held = Checkpoint8(torch.zeros(4, 32, dtype=torch.int8), torch.ones(4, 1, dtype=torch.uint8), (4, 32), torch.float32)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(t), t)[1], lambda t: t):
        scaled = w.to(torch.float64).to(torch.float32)
        layers8.linear(x, scaled, None, held=held)                   # its checkpoint is kept with it
        layers8.linear(x, scaled.detach(), torch.zeros(8, requires_grad=True))
    weights = [t for t in seen if t.shape == (8, 32)]
    assert len(weights) == 2 and all(t.is_leaf and t.data_ptr() in (scaled.data_ptr(),) for t in weights)


def test_what_is_a_weight():
    from cswap_amd.hooks import _is_weight

    p, x = torch.nn.Parameter(torch.zeros(4, 8)), torch.zeros(4, 8, requires_grad=True)
    for weight in (p.view(8, 4), p[1:], p.flatten(), p.to(torch.bfloat16), p.half()):
        assert _is_weight(weight)
    for other in (x.view(8, 4), x.half(), p * 2, (p * 2).half(), torch.relu(x), p @ x.t()):
        assert not _is_weight(other)


def test_a_weight_that_changed_before_backward_is_noticed():
    from cswap_amd import layers8
    from cswap_amd.q8 import Checkpoint8

    x, w = torch.randn(4, 32, requires_grad=True), torch.randn(8, 32, requires_grad=True)
    held = Checkpoint8(torch.zeros(4, 32, dtype=torch.int8), torch.ones(4, 1, dtype=torch.uint8), (4, 32), torch.float32)
    y = layers8.linear(x, w, None, held=held)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


# ---------------------------------------------------------------- sizes
def test_what_is_too_large_is_saved_as_usual():
    """The codec's limit is 2^31 - 1 pieces of 8 values, in whole groups of 32."""
    from cswap_amd import _lib, q8
    from cswap_amd.hooks import hold_saved_tensors

    most = q8.MAX_VALUES
    pack = _lib.lib().cswap_q8_pack
    assert pack(None, 0, 1, most, 0, 2, A, A, None) == ARG           # would run
    assert pack(None, 0, 1, most + 1, 0, 2, A, A, None) == UNSUPPORTED

    class Large:
        is_cuda, dtype, is_leaf, grad_fn, _base = True, torch.float32, False, None, None
        layout, is_nested = torch.strided, False

        def __init__(self, n):
            self.n = n

        def is_contiguous(self):
            return True

        def dim(self):
            return 1

        def numel(self):
            return self.n

        def element_size(self):
            return 4

    hooks = hold_saved_tensors()
    assert hooks._eligible(Large(most)) and not hooks._eligible(Large(most + 1))


def test_layers_that_the_kernels_cannot_take_are_left_alone():
    from cswap_amd import layers8
    from torch import nn

    def kinds(*layers):
        with torch.device("meta"):
            return [type(m).__name__ for m in layers8.checkpoint_layers(nn.Sequential(*(f() for f in layers)))]

    most = 1 << 20
    assert kinds(lambda: nn.Linear(most, 2), lambda: nn.Linear(most + 1, 2), lambda: nn.Linear(2, most), lambda: nn.Linear(2, most + 1)) \
        == ["Linear8", "Linear", "Linear8", "Linear"]
    assert kinds(lambda: nn.Linear(0, 3), lambda: nn.Linear(3, 0), lambda: nn.LayerNorm(0), lambda: nn.LayerNorm((4, 0))) \
        == ["Linear", "Linear", "LayerNorm", "LayerNorm"]
    assert kinds(lambda: nn.LayerNorm(16384), lambda: nn.LayerNorm(16385), nn.GELU, nn.SiLU, lambda: nn.SiLU(inplace=True)) \
        == ["LayerNorm8", "LayerNorm", "GELU8", "SiLU8", "SiLU"]


def test_linear_refuses_in_the_forward_pass():
    from cswap_amd import layers8
    from cswap_amd.q8 import Checkpoint8

    x = torch.zeros(1, 2, requires_grad=True)
    with pytest.raises(ValueError, match="features"):
        layers8.linear(x, torch.zeros((1 << 20) + 1, 2, requires_grad=True))
    w = torch.zeros(3, 2, requires_grad=True, device="meta")
    held = Checkpoint8(torch.zeros(1, 32, dtype=torch.int8), torch.zeros(1, 1, dtype=torch.uint8), (1, 2), torch.float32)
    with pytest.raises(ValueError, match="on cpu, x is"):
        layers8.linear(x.detach().to("meta"), w, None, held=held)


def test_a_view_with_its_sign_turned_is_refused():
    """The imaginary part of a conjugate is a view whose values in memory have the other sign."""
    from cswap_amd import layers8
    from cswap_amd.q8 import _row_stride

    t = torch.randn(4, 1, dtype=torch.complex64).conj().imag
    with pytest.raises(ValueError, match="sign"):
        _row_stride(t, "t")
    assert torch.equal(layers8._rows(t), t) and not layers8._rows(t).is_neg()
