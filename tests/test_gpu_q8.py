"""8-bit activation checkpoints on the GPU against their 64-bit forms: codes and scales to the byte, everything else
within the bounds that tests/q8_reference.py derives."""
import math
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import q8_reference as ref  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def q8():
    from cswap_amd import q8 as m

    return m


def values(rows, cols, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, dtype=torch.float64) * torch.exp(torch.randn(cols, generator=g, dtype=torch.float64))
    return (x * scale).to(dtype)


# ---------------------------------------------------------------- codec
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (7, 193), (2, 768), (1000, 1), (4, 16391), (257, 100)])
def test_codes_and_scales_are_those_of_the_definition(dtype, rows, cols):
    x = values(rows, cols, dtype, rows + cols)
    held = q8().q8_compress(x.cuda())
    codes, scales = ref.pack(x)
    assert torch.equal(held.scales.cpu(), scales)
    assert torch.equal(held.codes.cpu(), codes)
    want = ref.unpack(codes, scales, cols)
    for out in TYPES:
        back = q8().q8_decompress(held, dtype=out)
        assert torch.equal(back.cpu(), want.to(F32).to(out))         # q 2^e is an fp32 value exactly, rounded once from there
    err = (x.double() - want).abs()
    unit = ref.power_of_two(scales.long() - 127).repeat_interleave(32, 1)[:, :cols]
    assert bool((err <= torch.where(x.double().abs() > 127 * unit, unit, unit / 2)).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_codec_at_the_ends_of_the_range(dtype):
    fi = torch.finfo(dtype)
    least = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[dtype]
    rows = [[0.0] * 40, [-0.0] * 40, [fi.max] * 40, [-fi.max, 1.0] * 20, [least] * 40, [fi.tiny, -least] * 20,
            [math.inf] + [1.0] * 39, [1.0] * 39 + [-math.inf], [1.0, math.nan] + [2.0] * 38,
            [127.5, -127.5, 127.49, 126.5, 64.5, 63.5, 0.5, 1.5] * 5, [128.0, 127.75, -127.9, 1.0] * 10, [1e-30] + [3.0] * 39,
            [1.5 * 2.0 ** -127] * 40, [2.0 ** -127, -2.0 ** -126, 2.0 ** -120, 2.0 ** -121] * 10]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    held = q8().q8_compress(x.cuda())
    codes, scales = ref.pack(x)
    assert torch.equal(held.scales.cpu(), scales)
    assert torch.equal(held.codes.cpu(), codes)
    back = q8().q8_decompress(held).cpu()
    want = ref.unpack(codes, scales, 40).to(F32).to(dtype)
    assert torch.equal(torch.isnan(back), torch.isnan(want)) and torch.equal(back.nan_to_num(7.0), want.nan_to_num(7.0))
    assert not torch.isnan(back[6, 32:]).any() and torch.isnan(back[6, :32]).all()   # the other group is untouched


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_codec_of_rows_with_gaps_and_odd_starts(dtype):
    x = values(9, 130, dtype)
    big = torch.zeros(9, 141, dtype=dtype).cuda()
    view = big[:, 3:133]
    view.copy_(x)
    held = q8().q8_compress(view)
    assert torch.equal(held.codes.cpu(), ref.pack(x)[0])
    big.fill_(5.0)
    q8().q8_decompress(held, out=view)
    assert torch.equal(view.cpu(), ref.held(x).to(F32).to(dtype))
    assert bool((big[:, :3] == 5).all()) and bool((big[:, 133:] == 5).all())         # what lies between rows is left alone


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_signs_that_are_kept(dtype):
    """What is not 0 has a code that is not 0, with its sign; the other codes are the same."""
    x = values(50, 130, dtype, 31)
    x[::3, ::7] = 0.0
    x[1::3, 1::5] *= 1e-4
    x[0, 64:96] = torch.finfo(dtype).tiny
    x[0, 64], x[0, 65] = 1.0, -torch.finfo(dtype).tiny
    plain, kept = q8().q8_compress(x.cuda()), q8().q8_compress(x.cuda(), keep_sign=True)
    assert torch.equal(plain.scales, kept.scales)
    a, b, sign = plain.codes.cpu().int(), kept.codes.cpu().int(), torch.zeros(50, 160, dtype=torch.int32)
    sign[:, :130] = torch.sign(x.float()).int()
    assert int((sign[a == 0] != 0).sum()) > 100
    assert torch.equal(b, torch.where(a == 0, sign, a))
    assert torch.equal(torch.sign(q8().q8_decompress(kept).float()).cpu(), torch.sign(x.float()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_signs_that_are_kept(dtype):
    """What is not 0 has a code that is not 0, with its sign; the other codes are the same."""
    x = values(50, 130, dtype, 31)
    x[::3, ::7] = 0.0
    x[1::3, 1::5] *= 1e-4
    x[0, 64:96] = torch.finfo(dtype).tiny
    x[0, 64], x[0, 65] = 1.0, -torch.finfo(dtype).tiny
    plain, kept = q8().q8_compress(x.cuda()), q8().q8_compress(x.cuda(), keep_sign=True)
    assert torch.equal(plain.scales, kept.scales)
    a, b, sign = plain.codes.cpu().int(), kept.codes.cpu().int(), torch.zeros(50, 160, dtype=torch.int32)
    sign[:, :130] = torch.sign(x.float()).int()
    assert int((sign[a == 0] != 0).sum()) > 100
    assert torch.equal(b, torch.where(a == 0, sign, a))
    assert torch.equal(torch.sign(q8().q8_decompress(kept).float()).cpu(), torch.sign(x.float()))


def test_flat_checkpoints():
    x = values(6, 4 * 5, F32).view(6, 4, 5)
    held = q8().q8_compress(x.cuda(), flat=True)
    assert held.codes.shape == (1, 128) and held.shape == (6, 4, 5)
    assert torch.equal(held.codes.cpu(), ref.pack(x.reshape(1, -1))[0])
    assert torch.equal(q8().q8_decompress(held).cpu(), ref.held(x.reshape(1, -1)).to(F32).view(6, 4, 5))
    even = values(6, 64, F32)
    a, b = q8().q8_compress(even.cuda(), flat=True), q8().q8_compress(even.cuda())
    assert torch.equal(a.codes.view(-1), b.codes.view(-1)) and torch.equal(a.scales.view(-1), b.scales.view(-1))


def test_no_rows():
    m = q8()
    x = torch.empty(0, 48, device="cuda")
    held = m.q8_compress(x)
    assert held.codes.shape == (0, 64) and m.q8_decompress(held).shape == (0, 48)
    y, held = m.q8_act(x)
    assert y.shape == (0, 48) and m.q8_act_backward(x, held).shape == (0, 48)
    w = torch.ones(48, device="cuda")
    y, mean, rstd, held = m.layer_norm(x, w, w)
    dx, dw, db = m.layer_norm_backward(x, held, mean, rstd, w)
    assert dx.shape == (0, 48) and not dw.any() and not db.any()
    dw, db = m.q8_weight_grad(torch.empty(0, 33, device="cuda"), held)
    assert dw.shape == (33, 48) and not dw.any() and not db.any()


# ---------------------------------------------------------------- activation functions
@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 33), (64, 256), (5, 1111)])
def test_activation_functions(kind, dtype, rows, cols):
    x, dy = values(rows, cols, dtype, 1, 3.0), values(rows, cols, dtype, 2)
    y, held = q8().q8_act(x.cuda(), kind)
    assert torch.equal(held.codes.cpu(), ref.pack(x)[0]) and torch.equal(held.scales.cpu(), ref.pack(x)[1])
    xd, kept = x.double(), ref.held(x)
    ref.check(y, ref.act(xd, kind)[0], ref.act_error(xd, kind, dtype)[0], dtype, "y")
    dx = q8().q8_act_backward(dy.cuda(), held, kind)
    d = dy.double()
    ref.check(dx, d * ref.act(kept, kind)[1], d.abs() * (ref.act_error(kept, kind, dtype)[1] + 2 * ref.U), dtype, "dx")


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_activation_functions_far_out(kind):
    """Every exponent of fp32, infinities and NaN: the limits where the formula's products are 0 * inf."""
    e = torch.arange(-140, 128, dtype=torch.float64)
    x = torch.cat([2.0 ** e * s for s in (1.0, -1.0, 1.7, -1.7)]).to(F32)
    x = x[torch.isfinite(x)]
    rows = x.repeat_interleave(32).view(-1, 32)                     # one value a group, so that it is held closely
    y, held = q8().q8_act(rows.cuda(), kind)
    want = ref.act(rows.double(), kind)[0]
    far = rows.double().abs() > 1e4                                 # 64 bits overflow there, too: the limits are x and 0
    want = torch.where(far, rows.double().clamp(min=0), want)
    err = torch.where(far, torch.full_like(want, 1e-34), ref.act_error(rows.double().clamp(-1e4, 1e4), kind, F32)[0])
    ref.check(y, want, err, F32, "y")
    kept = ref.held(rows)
    dx = q8().q8_act_backward(torch.ones_like(rows).cuda(), held, kind)
    far = kept.abs() > 1e4
    want = torch.where(far, (kept > 0).double(), ref.act(kept.clamp(-1e4, 1e4), kind)[1])
    err = torch.where(far, torch.full_like(want, 4 * ref.U), ref.act_error(kept.clamp(-1e4, 1e4), kind, F32)[1])
    ref.check(dx, want, err, F32, "dx")
    odd = torch.tensor([[math.inf] * 32, [-math.inf] * 32, [math.nan] * 32], dtype=F32)
    y, held = q8().q8_act(odd.cuda(), kind)
    y = y.cpu()
    assert bool((y[0] == math.inf).all()) and bool((y[1].abs() < 1e-34).all()) and bool(torch.isnan(y[2]).all())
    assert bool(torch.isnan(q8().q8_act_backward(torch.ones_like(odd).cuda(), held, kind)).all())


# ---------------------------------------------------------------- layer norm
@pytest.mark.parametrize("checkpoint", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (33, 100), (17, 128), (70, 193), (9, 512), (1, 768), (65, 777), (5, 1500),
                                       (3, 2049), (6, 4096), (4, 5001), (3, 8200), (2, 16384)])
def test_layer_norm(dtype, rows, cols, checkpoint):
    x = (values(rows, cols, dtype, 3).double() + 0.5).to(dtype)
    dy = values(rows, cols, dtype, 4, 0.1)
    pd = F32 if cols % 2 else dtype
    w, b = values(1, cols, pd, 5)[0], values(1, cols, pd, 6)[0]
    m = q8()
    y, mean, rstd, held = m.layer_norm(x.cuda(), w.cuda(), b.cuda(), 1e-5, checkpoint=checkpoint)
    dx, dw, db = m.layer_norm_backward(dy.cuda(), held, mean, rstd, w.cuda())
    if checkpoint:
        assert torch.equal(held.codes.cpu(), ref.pack(x)[0]) and torch.equal(held.scales.cpu(), ref.pack(x)[1])
    args = (x.double(), ref.held(x) if checkpoint else x.double(), dy.double(), w.double(), b.double(), 1e-5)
    for name, got, want, err, t in zip(("y", "mean", "rstd", "dx", "dw", "db"), (y, mean, rstd, dx, dw, db), ref.norm(*args),
                                       ref.norm_error(*args), (dtype, F32, F32, dtype, pd, pd)):
        assert got.dtype == t
        ref.check(got, want, err, t, name)


@pytest.mark.parametrize("rows", [300, 5000])
def test_layer_norm_of_many_rows_twice_gives_the_same_bits(rows):
    m = q8()
    x, dy = values(rows, 200, BF16, 7).cuda(), values(rows, 200, BF16, 8).cuda()
    w = values(1, 200, BF16, 9)[0].cuda()
    outs = []
    for _ in range(2):
        y, mean, rstd, held = m.layer_norm(x, w, w)
        outs.append([y, *m.layer_norm_backward(dy, held, mean, rstd, w)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    args = (x.cpu().double(), ref.held(x.cpu()), dy.cpu().double(), w.cpu().double(), w.cpu().double(), 1e-5)
    want, err = ref.norm(*args), ref.norm_error(*args)
    for name, got, at in zip(("y", "dx", "dw", "db"), outs[0], (0, 3, 4, 5)):
        ref.check(got, want[at], err[at], BF16, name)


@pytest.mark.parametrize("checkpoint", [True, False])
@pytest.mark.parametrize("dtype,rows,cols", [(BF16, 8197, 513), (F16, 8192, 768), (BF16, 9001, 700), (BF16, 8191, 640)], ids=str)
def test_layer_norm_of_many_rows_of_513_to_768_values(dtype, rows, cols, checkpoint):
    m = q8()
    x, dy = values(rows, cols, dtype, 41), values(rows, cols, dtype, 42, 0.1)
    w, b = values(1, cols, F32, 43)[0], values(1, cols, F32, 44)[0]
    y, mean, rstd, held = m.layer_norm(x.cuda(), w.cuda(), b.cuda(), 1e-5, checkpoint=checkpoint)
    dx, dw, db = m.layer_norm_backward(dy.cuda(), held, mean, rstd, w.cuda())
    if checkpoint:
        assert torch.equal(held.codes.cpu(), ref.pack(x)[0]) and torch.equal(held.scales.cpu(), ref.pack(x)[1])
    args = (x.double(), ref.held(x) if checkpoint else x.double(), dy.double(), w.double(), b.double(), 1e-5)
    for name, got, want, err, t in zip(("y", "mean", "rstd", "dx", "dw", "db"), (y, mean, rstd, dx, dw, db), ref.norm(*args),
                                       ref.norm_error(*args), (dtype, F32, F32, dtype, F32, F32)):
        assert got.dtype == t
        ref.check(got, want, err, t, name)


def test_layer_norm_without_parameters_and_with_a_large_mean():
    m = q8()
    x = (values(20, 300, F32, 10).double() + 1000.0).to(F32)
    dy = values(20, 300, F32, 11)
    one, zero = torch.ones(300, dtype=torch.float64), torch.zeros(300, dtype=torch.float64)
    y, mean, rstd, held = m.layer_norm(x.cuda(), None, None, checkpoint=False)
    dx, dw, db = m.layer_norm_backward(dy.cuda(), held, mean, rstd, None)
    args = (x.double(), x.double(), dy.double(), one, zero, 1e-5)
    for name, got, want, err in zip(("y", "mean", "rstd", "dx", "dw", "db"), (y, mean, rstd, dx, dw, db), ref.norm(*args),
                                    ref.norm_error(*args)):
        ref.check(got, want, err, F32, name)


def test_layer_norm_of_a_row_that_is_not_finite_leaves_the_others():
    m = q8()
    x, dy = values(8, 96, F32, 12), values(8, 96, F32, 13)
    clean = x.clone()
    x[3, 40] = math.nan
    x[5, 95] = math.inf
    w = values(1, 96, F32, 14)[0].cuda()
    y, mean, rstd, held = m.layer_norm(x.cuda(), w, w)
    dx, _, _ = m.layer_norm_backward(dy.cuda(), held, mean, rstd, w)
    y2, mean2, rstd2, held2 = m.layer_norm(clean.cuda(), w, w)
    dx2, _, _ = m.layer_norm_backward(dy.cuda(), held2, mean2, rstd2, w)
    good = [0, 1, 2, 4, 6, 7]
    assert torch.equal(y[good], y2[good]) and torch.equal(dx[good], dx2[good])
    assert bool(torch.isnan(y[[3, 5]]).all()) and bool(torch.isnan(dx[[3, 5]]).all())


# ---------------------------------------------------------------- weight gradient
GRADS = [(1, 1, 1), (1, 130, 40), (7, 33, 65), (64, 256, 256), (31, 100, 193), (333, 129, 257), (1000, 300, 96), (2050, 64, 128),
         (700, 520, 130), (4100, 17, 300), (128, 128, 128), (515, 1000, 193),
         (2050, 2900, 2850), (8200, 1500, 1400)]    # the larger tiles, the rows not split and split, everything cut off somewhere


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,n,k", GRADS)
def test_weight_grad(dtype, rows, n, k):
    x, dy = values(rows, k, dtype, 15), values(rows, n, dtype, 16, 0.1)
    held = q8().q8_compress(x.cuda())
    d, kept = dy.double(), ref.held(x)
    want, err = ref.weight_grad(d, kept), ref.weight_grad_error(d, kept)
    for out in (dtype, F32):
        dw, db = q8().q8_weight_grad(dy.cuda(), held, out_dtype=out)
        ref.check(dw, want[0], err[0], out, "dw")
        ref.check(db, want[1], err[1], out, "db")
    dw2, none = q8().q8_weight_grad(dy.cuda(), held, bias=False, out_dtype=F32)
    assert none is None and torch.equal(dw, dw2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_weight_grad_of_rows_with_gaps_and_odd_starts(dtype):
    x, dy = values(300, 70, dtype, 17), values(300, 150, dtype, 18)
    big = torch.full((300, 171), math.nan, dtype=dtype).cuda()
    big[:, 5:155] = dy.cuda()
    held = q8().q8_compress(x.cuda())
    dw, db = q8().q8_weight_grad(big[:, 5:155], held)
    d, kept = dy.double(), ref.held(x)
    want, err = ref.weight_grad(d, kept), ref.weight_grad_error(d, kept)
    ref.check(dw, want[0], err[0], dtype, "dw")
    ref.check(db, want[1], err[1], dtype, "db")


def test_weight_grad_keeps_the_last_bits_of_fp32():
    """One row of x that is not 0 and a dy whose 24 bits are all in use: a result is one product, cut into three
    that are summed with two roundings, and rounded to fp32."""
    g = torch.Generator().manual_seed(19)
    dy = (torch.randint(1 << 23, 1 << 24, (200, 64), generator=g).double() * 2.0 ** -23).to(F32)
    x = torch.zeros(200, 96, dtype=F32)
    x[77] = torch.randint(-127, 128, (96,), generator=g).to(F32)
    x[77, 0::32] = 127.0
    kept = ref.held(x)
    assert torch.equal(kept, x.double())
    dw, _ = q8().q8_weight_grad(dy.cuda(), q8().q8_compress(x.cuda()))
    want = dy.double().t() @ kept
    ref.check(dw, want, 2 * ref.U * want.abs(), F32, "dw")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,n,k", [(3001, 777, 333), (16384, 768, 768), (16000, 300, 2000), (200, 5000, 70), (20001, 603, 701), (100003, 33, 17)])
def test_weight_grad_of_whole_numbers_is_exact(dtype, rows, n, k):
    """Sums below 2^24: every order of fp32 additions gives the exact result, and a value left out or taken twice shows."""
    g = torch.Generator().manual_seed(rows + n + k)
    x, dy = torch.randint(-9, 10, (rows, k), generator=g), torch.randint(-9, 10, (rows, n), generator=g)
    x[:, ::32] = 9
    dw, db = q8().q8_weight_grad(dy.to(dtype).cuda(), q8().q8_compress(x.to(dtype).cuda()), out_dtype=F32)
    assert torch.equal(dw.cpu(), (dy.float().t() @ x.float()))
    assert torch.equal(db.cpu(), dy.sum(0).float())


@pytest.mark.parametrize("rows,n,k", [(12000, 8, 2048), (30000, 64, 300), (9001, 49, 1000), (20011, 33, 131), (70, 17, 4000),
                                      (700, 1, 257)])
def test_weight_grad_of_few_outputs_in_fp32(rows, n, k):
    """dy has 24 bits, whose three parts each matter, and a row of x at most one value that is not 0: a sum is off by one
    rounding for each part of each product that is not 0 (parts have dy's sign, so their magnitudes add up to its own)."""
    g = torch.Generator().manual_seed(rows + n + k)
    dy = (torch.randint(-(1 << 24) + 1, 1 << 24, (rows, n), generator=g).double() * 2.0 ** -23).to(F32)
    x = torch.zeros(rows, k)
    x[torch.arange(rows), torch.randint(0, k, (rows,), generator=g)] = 3.0
    held = q8().q8_compress(x.cuda())
    dw, db = q8().q8_weight_grad(dy.cuda(), held)
    kept = ref.held(x)
    terms = 2 + 3 * int((x != 0).sum(0).max())
    ref.check(dw, dy.double().t() @ kept, terms * ref.U * (dy.double().abs().t() @ kept.abs()), F32, "dw")
    ref.check(db, dy.double().sum(0), ref.weight_grad_error(dy.double(), kept)[1], F32, "db")


def test_weight_grad_of_subnormal_values():
    """fp16 below 2^-14 in either operand, bf16 and fp32 below 2^-126: nothing is flushed."""
    g = torch.Generator().manual_seed(24)
    small = torch.randint(-1000, 1001, (200, 70), generator=g).double() * 2.0 ** -24
    for x, dy in ((values(200, 70, F16, 25), small[:, :40].to(F16)), (small.to(F16), values(200, 40, F16, 26))):
        dw, db = q8().q8_weight_grad(dy.cuda(), q8().q8_compress(x.cuda()), out_dtype=F32)
        d, kept = dy.double(), ref.held(x)
        ref.check(dw, ref.weight_grad(d, kept)[0], ref.weight_grad_error(d, kept)[0], F32, "dw")
        ref.check(db, ref.weight_grad(d, kept)[1], ref.weight_grad_error(d, kept)[1], F32, "db")
    for dtype in (BF16, F32):
        dy = (torch.randint(1, 128, (1, 40), generator=g).double() * 2.0 ** -133).to(dtype)
        dw, db = q8().q8_weight_grad(dy.cuda(), q8().q8_compress(torch.full((1, 32), 64.0, dtype=dtype).cuda()), out_dtype=F32)
        assert torch.equal(dw.cpu().double(), dy.double().t() * torch.full((1, 32), 64.0, dtype=torch.float64))
        assert torch.equal(db.cpu().double(), dy.double()[0])


def test_weight_grad_of_values_that_are_not_finite():
    x, dy = values(100, 96, F32, 20), values(100, 40, F32, 21)
    x[50, 33] = math.nan                                             # columns 32 to 63 of every row of dw
    dy[3, 7] = math.nan
    dy[4, 9] = math.inf
    dw, db = q8().q8_weight_grad(dy.cuda(), q8().q8_compress(x.cuda()))
    bad = ~torch.isfinite(dw.cpu())
    want = torch.zeros(40, 96, dtype=torch.bool)
    want[:, 32:64] = True
    want[7], want[9] = True, True
    assert torch.equal(bad, want)
    assert (~torch.isfinite(db.cpu())).nonzero().flatten().tolist() == [7, 9]


def test_weight_grad_of_leading_dimensions_twice_gives_the_same_bits():
    x, dy = values(6 * 50, 72, BF16, 22).view(6, 50, 72), values(6 * 50, 40, BF16, 23).view(6, 50, 40)
    held = q8().q8_compress(x.cuda())
    a, b = q8().q8_weight_grad(dy.cuda(), held), q8().q8_weight_grad(dy.cuda(), held)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    d, kept = dy.double().view(300, 40), ref.held(x.view(300, 72))
    ref.check(a[0], ref.weight_grad(d, kept)[0], ref.weight_grad_error(d, kept)[0], BF16, "dw")
