"""Rows of more than 2^32 values, several of them and with gaps between: the same as each row by itself."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

COLS = (1 << 32) + 8          # no multiple of 32: rows with padding


@pytest.fixture(autouse=True)
def memory_back():
    yield
    torch.cuda.empty_cache()


def filled(rows, pitch):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.empty(rows * pitch, dtype=torch.bfloat16, device="cuda")
    for at in range(0, rows * pitch, 1 << 29):
        x[at:at + (1 << 29)].normal_(generator=g)
    return x.view(rows, pitch)


@pytest.mark.parametrize("pitch", [COLS, COLS + 6])
def test_two_rows_are_two_checkpoints(pitch):
    from cswap_amd import q8

    x = filled(2, pitch)[:, :COLS]
    held = q8.q8_compress(x)
    for r in range(2):
        one = q8.q8_compress(x[r])
        assert torch.equal(held.codes[r], one.codes[0]) and torch.equal(held.scales[r], one.scales[0])
        assert bool(one.codes[0, COLS - 8:COLS].any()) and not bool(one.codes[0, COLS:].any())
        del one
    out = torch.zeros(2, COLS, dtype=torch.bfloat16, device="cuda")
    q8.q8_decompress(held, out=out)
    del x
    for r in range(2):
        one = q8.Checkpoint8(held.codes[r:r + 1], held.scales[r:r + 1], (COLS,), torch.bfloat16)
        assert torch.equal(out[r], q8.q8_decompress(one))


def test_activations_of_two_rows():
    from cswap_amd import q8

    x = filled(2, COLS)
    y, held = q8.q8_act(x, "silu")
    assert torch.equal(held.codes[1], q8.q8_compress(x[1]).codes[0])
    dx = q8.q8_act_backward(y, held, "silu")
    for r in range(2):
        yr, hr = q8.q8_act(x[r], "silu")
        assert torch.equal(y[r], yr)
        assert torch.equal(dx[r], q8.q8_act_backward(yr, hr, "silu"))
        del yr, hr
