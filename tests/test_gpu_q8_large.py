"""Offsets beyond 32 bits: tensors of more than 2^32 values, against the same kernels on pieces of them and, for the
weight gradient, against 64-bit sums."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24


def filled(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for at in range(0, rows, 1 << 17):
        x[at:at + (1 << 17)] = torch.randn(min(1 << 17, rows - at), cols, generator=g, device="cuda", dtype=torch.bfloat16)
    return x


@pytest.fixture(autouse=True)
def memory_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cols", [4128, 4100])          # one row of pieces, and rows with padding
def test_codec_and_activation(cols):
    from cswap_amd import q8

    rows = (1 << 20) + 37
    x = filled(rows, cols, 1)
    assert x.numel() > 1 << 32
    y, held = q8.q8_act(x, "silu")
    back = q8.q8_decompress(held)
    dx = q8.q8_act_backward(y, held, "silu")
    for lo, hi in ((0, 1000), (1 << 19, (1 << 19) + 1000), ((1 << 31) // cols - 500, (1 << 31) // cols + 500),
                   ((1 << 32) // cols - 500, (1 << 32) // cols + 500), (rows - 1000, rows)):
        yp, hp = q8.q8_act(x[lo:hi], "silu")
        assert torch.equal(held.codes[lo:hi], hp.codes) and torch.equal(held.scales[lo:hi], hp.scales)
        assert torch.equal(y[lo:hi], yp) and torch.equal(back[lo:hi], q8.q8_decompress(hp))
        assert torch.equal(dx[lo:hi], q8.q8_act_backward(yp, hp, "silu"))


def test_layer_norm():
    from cswap_amd import q8

    rows, cols = (1 << 20) + 37, 4100
    x = filled(rows, cols, 2)
    w = torch.randn(cols, device="cuda", dtype=torch.bfloat16)
    y, mean, rstd, held = q8.layer_norm(x, w, w)
    dx, dw, db = q8.layer_norm_backward(y, held, mean, rstd, w, None)
    for lo, hi in ((0, 500), ((1 << 32) // cols - 250, (1 << 32) // cols + 250), (rows - 500, rows)):
        yp, mp, rp, hp = q8.layer_norm(x[lo:hi], w, w)
        assert torch.equal(y[lo:hi], yp) and torch.equal(mean[lo:hi], mp) and torch.equal(held.codes[lo:hi], hp.codes)
        assert torch.equal(dx[lo:hi], q8.layer_norm_backward(yp, hp, mp, rp, w)[0])
    want = sum(y[at:at + (1 << 17)].double().sum(0) for at in range(0, rows, 1 << 17))
    size = sum(y[at:at + (1 << 17)].double().abs().sum(0) for at in range(0, rows, 1 << 17))
    # a share has 4097 rows one after the other in a lane, the joins are 300 more; then one rounding to bf16
    assert bool(((db.double() - want).abs() <= 4400 * U * size + 2.0 ** -8 * want.abs()).all())
    assert bool(torch.isfinite(dw).all())


def test_weight_grad():
    """Whole numbers whose sums stay below 2^24: every order of fp32 additions gives the exact result."""
    from cswap_amd import q8

    rows, n, k = (1 << 20) + 37, 4100, 96
    g = torch.Generator(device="cuda").manual_seed(3)
    dy = torch.randint(-1, 2, (rows, n), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    x = torch.randint(-2, 3, (rows, k), generator=g, device="cuda", dtype=torch.int8).to(torch.bfloat16)
    assert dy.numel() > 1 << 32
    held = q8.q8_compress(x)
    assert torch.equal(q8.q8_decompress(held), x)
    dw, db = q8.q8_weight_grad(dy, held, out_dtype=torch.float32)
    want, want_b = torch.zeros(n, k, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
    for at in range(0, rows, 1 << 15):
        d = dy[at:at + (1 << 15)].double()
        want += torch.mm(d.t().contiguous(), x[at:at + (1 << 15)].double())
        want_b += d.sum(0)
    assert torch.equal(dw.double(), want) and torch.equal(db.double(), want_b)
