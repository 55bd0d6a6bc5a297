"""Group norm without a GPU: sizes, refusals, and that the reference is torch's own function."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import group_norm_reference as gref  # noqa: E402

from cswap_amd import _lib, layers8, q8  # noqa: E402

A = 1 << 20     # an address that nothing reads


def forward(act=3, x=A, dtype=0, n=2, p=16, c=64, groups=8, stride=0, gamma=A, beta=A, kind=0, eps=1e-5, y=A, mean=A, rstd=A, codes=A, scales=A, ws=A,
            room=1 << 20):
    return _lib.lib().cswap_group_norm_forward(act, x, dtype, n, p, c, groups, stride, gamma, beta, kind, eps, y, 0, mean, rstd, codes, scales, ws, room, None)


def backward(act=3, dy=A, dtype=0, n=2, p=16, c=64, groups=8, stride=0, x=0, codes=A, scales=A, mean=A, rstd=A, gamma=A, beta=A, kind=0, dx=A, dw=A, db=A,
             ws=A, room=1 << 30):
    return _lib.lib().cswap_group_norm_backward(act, dy, dtype, n, p, c, groups, stride, x, 0, codes, scales, mean, rstd, gamma, beta, kind, dx, 0, dw, db, ws,
                                                room, None)


def test_argument_errors_do_not_launch():
    bad = [dict(act=4), dict(act=-1), dict(dtype=3), dict(kind=3), dict(c=0), dict(p=0), dict(groups=0), dict(groups=7), dict(stride=63), dict(stride=-64)]
    for kw in bad + [dict(x=0), dict(x=A + 2), dict(y=0), dict(mean=A + 2), dict(rstd=0), dict(codes=0), dict(scales=0), dict(codes=A + 4), dict(eps=-1.0),
                     dict(gamma=A + 1), dict(beta=A + 1)]:
        assert forward(**kw) == -1, kw
    for kw in bad + [dict(dy=0), dict(dx=A + 2), dict(mean=0), dict(rstd=A + 1), dict(x=A), dict(codes=0, scales=0), dict(scales=0), dict(dw=A + 1),
                     dict(db=A + 1), dict(gamma=A + 2), dict(ws=0), dict(ws=A + 4)]:
        assert backward(**kw) == -1, kw
    for kw in (dict(c=4104), dict(c=4096, groups=4096), dict(n=1 << 31), dict(p=1 << 31), dict(n=1 << 20, p=1 << 11)):
        assert forward(**kw) == -2 and backward(**kw) == -2, kw
    assert backward(room=100) == -4
    assert forward(p=100000, room=100) == -4 and forward(p=100000, ws=0) == -1
    assert forward(n=0, x=0, y=0, mean=0, rstd=0, codes=0, scales=0, gamma=0, beta=0) == 0
    assert backward(n=0, dy=0, dx=0, mean=0, rstd=0, dw=0, db=0) == 0


def test_workspaces():
    f = _lib.lib().cswap_group_norm_workspace_bytes
    assert f(2, 16, 64, 8, 0) == 0 and f(0, 16, 64, 8, 1) == 0 and f(2, 16, 64, 7, 1) == 0 and f(2, 16, 5000, 8, 1) == 0
    assert f(2, 16, 64, 8, 1) == 2 * 2 * 64 * 4                                   # a share for each sample
    tiles = f(1, 1 << 16, 64, 8, 0) // (8 * 8)
    assert 1 < tiles <= 512 and f(1, 1 << 16, 64, 8, 1) == tiles * (8 * 8 + 2 * 64 * 4)
    assert all(f(n, p, c, 1, 1) <= max(4 * n, 4096) * (8 + 2 * c * 4) for n in (1, 3, 700) for p in (1, 7, 1000, 1 << 20) for c in (1, 8, 257, 4096))


def test_the_reference_is_the_function():
    x, dy = torch.randn(3, 5, 12, dtype=torch.float64), torch.randn(3, 5, 12, dtype=torch.float64)
    w, b = torch.randn(12, dtype=torch.float64), torch.randn(12, dtype=torch.float64)
    for kind, f in ((None, lambda t: t), ("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu)):
        leaves = [t.clone().requires_grad_() for t in (x.movedim(-1, 1), w, b)]
        y = f(torch.nn.functional.group_norm(leaves[0], 3, leaves[1], leaves[2], 1e-3))
        y.backward(dy.movedim(-1, 1))
        got = gref.outputs(x, x, dy, w, b, 3, 1e-3, kind)
        assert torch.allclose(got[0].movedim(-1, 1), y.detach(), atol=1e-12)
        for a, leaf in zip((got[3].movedim(-1, 1), got[4], got[5]), leaves):
            assert torch.allclose(a, leaf.grad, atol=1e-11)


def test_which_images_are_taken():
    t = torch.zeros(2, 3, 4, 5)
    for bad in (t, t.to(memory_format=torch.channels_last)[:, :, :, ::2][:, :, ::3], torch.zeros(3), torch.zeros(2, 0, 3, 3), torch.zeros(2, 3, 0, 3)):
        with pytest.raises(ValueError):
            q8._images(bad, "images")
    last = t.to(memory_format=torch.channels_last)
    assert q8._images(last, "") == (2, 20, 3, 0)
    assert q8._images(torch.zeros(2, 4, 5, 8)[..., 1:4].movedim(-1, 1), "") == (2, 20, 3, 8)
    assert q8._images(last[:, :, 1:], "")[:3] == (2, 15, 3) if last[:, :, 1:].stride(0) == 45 else True
    assert q8._images(torch.zeros(7, 6), "") == (7, 1, 6, 0) and q8._images(torch.zeros(1, 1, 9), "") == (1, 9, 1, 0)
    assert q8._images(torch.zeros(5, 9, 1).movedim(-1, 1), "") == (5, 9, 1, 0)
    with pytest.raises(ValueError):
        q8._images(torch.zeros(1, 5, 3).expand(4, 5, 3).movedim(-1, 1), "")     # overlapping samples


def test_tensors_that_are_refused():
    x = torch.zeros(2, 4, 4, 8).movedim(-1, 1)
    with pytest.raises(ValueError, match="device memory"):
        q8.group_norm(x, 2)
    with pytest.raises(TypeError):
        q8.group_norm(x.double(), 2)
    with pytest.raises(ValueError, match="activation"):
        q8.group_norm(x, 2, act="relu")
    with pytest.raises(ValueError, match="activation"):
        layers8.GroupNorm8(2, 8, act="relu")
    with pytest.raises(ValueError, match="channels"):
        layers8.GroupNorm8(2, 8)(torch.zeros(2, 6, 3, 3))
    with pytest.raises(ValueError, match="device memory"):
        layers8.GroupNorm8(2, 8)(x)


def test_which_layers_are_converted():
    from torch import nn

    model = nn.Sequential(nn.GroupNorm(2, 8), nn.GroupNorm(1, 8192), nn.GroupNorm(4096, 4096), nn.Linear(3, 3))
    layers8.checkpoint_layers(model)
    assert [type(m) for m in model] == [nn.GroupNorm] * 3 + [layers8.Linear8]
    layers8.checkpoint_layers(model, group_norm=True)
    assert [type(m) for m in model] == [layers8.GroupNorm8, nn.GroupNorm, nn.GroupNorm, layers8.Linear8]
    assert model[0].act is None


def test_more_samples_than_a_launch_has_room_for():
    assert forward(n=(1 << 22) + 1) == -2 and backward(n=(1 << 22) + 1) == -2
    assert _lib.lib().cswap_group_norm_workspace_bytes((1 << 22) + 1, 1, 8, 1, 1) == 0


def watched():
    held = q8.Checkpoint8(torch.zeros(12, 64, dtype=torch.int8), torch.zeros(12, 2, dtype=torch.uint8), (4, 3, 40), torch.float32)
    plain, s = torch.zeros(4, 3, 40).movedim(-1, 1), torch.zeros(4, 5)
    return {"forward": lambda x: q8.group_norm(x, 5), "weight": lambda x: q8.group_norm(plain, 5, x[0, :, 0]),
            "backward": lambda x: q8.group_norm_backward(x, held, s, s, 5), "backward_of_x": lambda x: q8.group_norm_backward(plain, x, s, s, 5),
            "layer": lambda x: layers8.group_norm(x, 5)}


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("name", sorted(watched()))
def test_traces_and_forward_mode_are_refused(name):
    from torch.autograd import forward_ad

    x = torch.randn(4, 3, 40).movedim(-1, 1)
    with torch.no_grad():
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            watched()[name](forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(watched()[name], x, check_trace=False)
