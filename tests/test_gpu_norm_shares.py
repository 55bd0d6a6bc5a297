"""Layer norm of enough rows that several workgroups share them, each taking more than one turn, in every form of more
than 1024 values a row: against the 64-bit form."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import q8_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def values(rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64) * torch.exp(torch.randn(cols, generator=g, dtype=torch.float64))
    return (x * scale).to(dtype)


# backward: 256 workgroups of 4 rows (up to 2048 values), 2 (4096) and 1; forward: 1024 workgroups of 2 and 1, 512, 256
@pytest.mark.parametrize("checkpoint", [True, False])
@pytest.mark.parametrize("dtype,rows,cols", [(F32, 2100, 1500), (BF16, 2100, 1025), (F16, 2050, 2048), (F32, 1030, 3000),
                                             (BF16, 1025, 2049), (F16, 600, 4096), (F32, 600, 4100), (BF16, 520, 8192),
                                             (BF16, 300, 16384), (F32, 260, 8193)], ids=str)
def test_shares_and_turns(dtype, rows, cols, checkpoint):
    from cswap_amd import q8
    from cswap_amd._lib import lib

    assert lib().cswap_layer_norm_workspace_bytes(rows, cols) > 2 * 4 * cols         # more than one workgroup
    x, dy = values(rows, cols, dtype, 1), values(rows, cols, dtype, 2, 0.1)
    w, b = values(1, cols, F32, 3)[0], values(1, cols, F32, 4)[0]
    y, mean, rstd, held = q8.layer_norm(x.cuda(), w.cuda(), b.cuda(), 1e-5, checkpoint=checkpoint)
    dx, dw, db = q8.layer_norm_backward(dy.cuda(), held, mean, rstd, w.cuda())
    if checkpoint:
        codes, scales = ref.pack(x)
        assert torch.equal(held.codes.cpu(), codes) and torch.equal(held.scales.cpu(), scales)
    args = (x.double(), ref.held(x) if checkpoint else x.double(), dy.double(), w.double(), b.double(), 1e-5)
    for name, got, want, err, t in zip(("y", "mean", "rstd", "dx", "dw", "db"), (y, mean, rstd, dx, dw, db), ref.norm(*args),
                                       ref.norm_error(*args), (dtype, F32, F32, dtype, F32, F32)):
        assert got.dtype == t
        ref.check(got, want, err, t, name)


def test_the_weights_gradient_of_many_long_rows():
    """Two thousand million values: dw against 64-bit sums of what the kernel's own mean and deviation give."""
    from cswap_amd import q8

    rows, cols, step = 500_003, 4100, 1 << 15
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.empty(rows, cols, dtype=BF16, device="cuda").normal_(generator=g)
    dy = torch.empty(rows, cols, dtype=BF16, device="cuda").normal_(generator=g)
    w = torch.ones(cols, dtype=F32, device="cuda")
    _, mean, rstd, held = q8.layer_norm(x, w, None)
    _, dw, db = q8.layer_norm_backward(dy, held, mean, rstd, w)
    del x
    want, want_b, size, size_b = (torch.zeros(cols, dtype=torch.float64, device="cuda") for _ in range(4))
    for at in range(0, rows, step):
        part = q8.Checkpoint8(held.codes[at:at + step], held.scales[at:at + step], (min(step, rows - at), cols), BF16)
        d = dy[at:at + step].double()
        mu, r = mean[at:at + step].double()[:, None], rstd[at:at + step].double()[:, None]
        kept = q8.q8_decompress(part, dtype=F32).double()
        want += (d * (kept - mu) * r).sum(0)
        size += (d.abs() * (kept.abs() + mu.abs()) * r).sum(0)
        want_b += d.sum(0)
        size_b += d.abs().sum(0)
    # 256 shares of 1954 rows or one less, one after the other in a lane, and 300 joins; h has two roundings, its product one
    assert bool(((dw.double() - want).abs() <= 2300 * ref.U * size).all())
    assert bool(((db.double() - want_b).abs() <= 2300 * ref.U * size_b).all())
