"""Every form of the 8-bit floating point product, with blocks whose scales differ from row to row and from block to block: exact results, rounded once."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import f8_tile_cases as tiles  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
KIND = {F32: 0, BF16: 1, F16: 2}


@pytest.mark.parametrize("turned", [False, True], ids=["plain", "turned"])
@pytest.mark.parametrize("form,bits,rows,n,k", tiles.CASES)
def test_scales_of_every_row_and_block(form, bits, rows, n, k, turned):
    """Products of 0 and +-1 times 1 to 64 are whole numbers, of one size within a block, and sums of their magnitudes at most 64 k: exact in fp32 in any
    order.  Gaps between rows of the result and rows behind the last keep what was there."""
    from cswap_amd import f8
    from cswap_amd._lib import lib

    assert 64 * k < 1 << 24
    x = tiles.blocks(rows, k, 1, "cuda", rows + k)
    w = tiles.blocks(k, n, 128, "cuda", n) if turned else tiles.blocks(n, k, 128, "cuda", n)
    bias = torch.randint(-9, 10, (n,), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").float()
    want = x @ (w if turned else w.t()) + bias
    held = f8.f8_weight(w)
    codes = held.turned if turned else held.codes
    for out in (BF16, F16) if bits == 16 else (F32,):
        assert lib().cswap_test_f8_linear_form(rows, n, k, KIND[out]) == form
        given = x.to(F16 if out is F16 else BF16)
        y = torch.full((rows + 2, n + 3), -7.5, dtype=out, device="cuda")
        room = lib().cswap_f8_linear_workspace_bytes(rows, k)
        ws = torch.full((room,), 0x7f, dtype=torch.uint8, device="cuda")           # codes of NaN behind the last row
        assert lib().cswap_f8_linear(given.data_ptr(), KIND[given.dtype], rows, k, 0, codes.data_ptr(), held.scales.data_ptr(), n, int(turned), bias.data_ptr(), 0,
                                     y.data_ptr(), KIND[out], n + 3, ws.data_ptr() if room else 0, room, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert torch.equal(y[:rows, :n], want.to(out)), out
        assert bool((y[rows:] == -7.5).all()) and bool((y[:, n:] == -7.5).all())
        got = f8.f8_linear_backward(given, held, out_dtype=out) if turned else f8.f8_linear(given, held, bias, out_dtype=out)
        assert torch.equal(got, (want - bias if turned else want).to(out))
