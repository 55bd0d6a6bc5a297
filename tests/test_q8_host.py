"""What the 8-bit checkpoints refuse, and their sizes: host checks, no GPU."""
import pytest

torch = pytest.importorskip("torch")

ARG, UNSUPPORTED, NOMEM = -1, -2, -4
A = 1 << 20          # an aligned address that is never followed


def L():
    from cswap_amd import _lib

    return _lib.lib()


def test_sizes():
    for cols, pitch, groups in ((1, 32, 1), (32, 32, 1), (33, 64, 2), (193, 224, 7), (16384, 16384, 512)):
        assert L().cswap_q8_code_pitch(cols) == pitch and L().cswap_q8_scale_pitch(cols) == groups
    assert L().cswap_layer_norm_workspace_bytes(0, 100) == 0
    assert L().cswap_layer_norm_workspace_bytes(10, 16385) == 0
    assert L().cswap_layer_norm_workspace_bytes(1, 100) == 0            # one workgroup takes all rows
    assert L().cswap_layer_norm_workspace_bytes(100000, 100) >= 2 * 2 * 4 * 100
    assert L().cswap_q8_weight_grad_workspace_bytes(1, 10, 0, 5) == 0


def test_codec_refuses():
    pack, unpack = L().cswap_q8_pack, L().cswap_q8_unpack
    assert pack(None, 0, 4, 32, 0, 0, A, A, None) == ARG
    assert pack(A, 0, 4, 32, 0, 0, None, A, None) == ARG
    assert pack(A, 0, 4, 32, 0, 0, A, None, None) == ARG
    assert pack(A, 0, 4, 32, 0, 0, A + 4, A, None) == ARG          # codes are 8-byte aligned
    assert pack(A + 2, 0, 4, 32, 0, 0, A, A, None) == ARG          # fp32 values 4-byte aligned
    assert pack(A + 1, 1, 4, 32, 0, 0, A, A, None) == ARG
    assert pack(A, 3, 4, 32, 0, 0, A, A, None) == ARG
    assert pack(A, 0, 4, 0, 0, 0, A, A, None) == ARG
    assert pack(A, 0, 4, 32, 31, 0, A, A, None) == ARG             # rows overlap
    assert pack(A, 0, 4, 32, -32, 0, A, A, None) == ARG
    assert pack(A, 0, 1 << 40, 32, 0, 0, A, A, None) == UNSUPPORTED
    assert pack(A, 0, 1, 1 << 40, 0, 0, A, A, None) == UNSUPPORTED
    assert pack(A, 0, 1 << 29, 32, 0, 0, A, A, None) == UNSUPPORTED  # 2^31 pieces
    assert pack(None, 0, 0, 32, 0, 0, None, None, None) == 0
    assert unpack(None, A, 4, 32, A, 0, 0, None) == ARG
    assert unpack(A, A, 4, 32, None, 0, 0, None) == ARG
    assert unpack(A, A, 4, 32, A, 7, 0, None) == ARG
    assert unpack(None, None, 0, 32, None, 0, 0, None) == 0


def test_activations_refuse():
    fwd, bwd = L().cswap_q8_act_forward, L().cswap_q8_act_backward
    assert fwd(3, A, 0, 4, 32, 0, A, 0, A, A, None) == ARG
    assert fwd(-1, A, 0, 4, 32, 0, A, 0, A, A, None) == ARG
    assert fwd(0, A, 0, 4, 32, 0, None, 0, A, A, None) == ARG
    assert fwd(0, A, 0, 4, 32, 0, A, 8, A, A, None) == ARG
    assert fwd(0, A, 0, 4, 32, 0, A, 0, A, None, None) == ARG   # codes and scales, or neither
    assert fwd(0, A, 0, 4, 32, 0, A, 0, None, A, None) == ARG
    assert fwd(0, None, 0, 0, 32, 0, None, 0, None, None, None) == 0
    assert bwd(0, A, 0, 4, 32, 0, None, A, A, 0, None) == ARG
    assert bwd(5, A, 0, 4, 32, 0, A, A, A, 0, None) == ARG
    assert bwd(0, None, 0, 0, 32, 0, None, None, None, 0, None) == 0


def test_layer_norm_refuses():
    fwd, bwd = L().cswap_layer_norm_forward, L().cswap_layer_norm_backward
    ok = [A, 0, 4, 32, 0, A, A, 0, 1e-5, A, 0, A, A, A, A, None]

    def f(**kw):
        a = list(ok)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return fwd(*a)

    assert f(_0=None) == ARG and f(_1=9) == ARG and f(_3=0) == ARG and f(_4=5) == ARG and f(_7=-1) == ARG
    assert f(_8=-1.0) == ARG and f(_8=float("nan")) == ARG and f(_9=None) == ARG and f(_11=None) == ARG and f(_12=None) == ARG
    assert f(_13=None) == ARG and f(_14=None) == ARG and f(_5=A + 1) == ARG
    assert f(_3=16385) == UNSUPPORTED
    assert f(_2=0, _0=None) == 0
    room = L().cswap_layer_norm_workspace_bytes(4000, 32)
    good = [A, 0, 4000, 32, 0, None, 0, A, A, A, A, A, 0, A, 0, A, A, A, room, None]

    def b(**kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return bwd(*a)

    assert b(_0=None) == ARG and b(_5=A) == ARG and b(_7=None) == ARG and b(_8=None) == ARG and b(_9=None) == ARG
    assert b(_10=None) == ARG and b(_12=4) == ARG and b(_13=None) == ARG and b(_17=None) == ARG
    assert b(_7=None, _8=None) == ARG                           # neither x nor its checkpoint
    assert b(_18=room - 1) == NOMEM
    assert b(_3=16385) == UNSUPPORTED


def test_weight_grad_refuses():
    assert L().cswap_q8_weight_grad_workspace_bytes(1, 64, 48, 40) == 0      # results leave from the tiles
    room = L().cswap_q8_weight_grad_workspace_bytes(1, 20000, 48, 40)
    good = [A, 1, 20000, 48, 0, A, A, 40, A, A, 1, A, room, None]

    def f(**kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return L().cswap_q8_weight_grad(*a)

    assert f(_0=None) == ARG and f(_1=5) == ARG and f(_3=0) == ARG and f(_4=47) == ARG and f(_5=None) == ARG and f(_6=None) == ARG
    assert f(_7=0) == ARG and f(_8=None) == ARG and f(_9=A + 1) == ARG and f(_10=-2) == ARG and f(_11=None) == ARG
    assert f(_12=room - 1) == NOMEM
    assert f(_3=(1 << 20) + 1) == UNSUPPORTED and f(_7=(1 << 20) + 1) == UNSUPPORTED


def test_weight_grad_layout():
    """Tiles (1000s: 0 small, 1 middle, 2 large) and splits as they measured best, and the same in the workspace's size."""
    plan, room = L().cswap_test_weight_grad_plan, L().cswap_q8_weight_grad_workspace_bytes
    f32, bf16 = 0, 1
    for rows, n, k in ((1, 1, 1), (64, 256, 256), (512, 2048, 2048), (512, 768, 4096), (0, 100, 100)):
        assert plan(bf16, rows, n, k) == 1 and room(bf16, rows, n, k) == 0
    for rows, n, k in ((2048, 4096, 4096), (8192, 4096, 4096), (4096, 4096, 4096)):
        assert plan(bf16, rows, n, k) == 2001 and plan(f32, rows, n, k) == 2001
    for rows, n, k in ((16384, 4096, 1024), (32768, 1024, 1024), (8192, 2048, 2048)):
        assert plan(bf16, rows, n, k) >= 2004
    for rows, n, k in ((8192, 768, 768), (2048, 2048, 2048), (2048, 768, 4096)):
        assert 1002 <= plan(f32, rows, n, k) < 2000
    for rows, n, k in ((8192, 256, 256), (32768, 256, 256), (4100, 17, 300)):
        assert 2 <= plan(bf16, rows, n, k) <= 64
    for dtype in (f32, bf16):
        for rows, n, k in ((5000, 300, 100), (70000, 33, 65), (16384, 768, 768), (1 << 20, 128, 128)):
            form, splits = divmod(plan(dtype, rows, n, k), 1000)
            assert 2 <= splits <= 512 and room(dtype, rows, n, k) == 4 * splits * (n * k + n * -(-k // (128, 256, 256)[form]))


def test_weight_grad_layout_of_few_outputs():
    """Narrow tiles (3000s) where an fp32 dY has no more columns than they."""
    plan, room = L().cswap_test_weight_grad_plan, L().cswap_q8_weight_grad_workspace_bytes
    for rows, n, k in ((12000, 8, 2048), (30000, 64, 300), (9001, 33, 1000)):
        form, splits = divmod(plan(0, rows, n, k), 1000)
        assert form == 3 and room(0, rows, n, k) == 4 * splits * (n * k + n * -(-k // 256))
        assert plan(1, rows, n, k) < 3000
    for rows, n, k in ((30000, 65, 300), (30000, 192, 2048), (30000, 64, 128)):
        assert plan(0, rows, n, k) < 3000


# ---------------------------------------------------------------- the torch side
def checkpoint(shape, rows, cols, dtype=torch.float32):
    from cswap_amd.q8 import Checkpoint8

    g = -(-cols // 32)
    return Checkpoint8(torch.zeros(rows, g * 32, dtype=torch.int8), torch.zeros(rows, g, dtype=torch.uint8), shape, dtype)


def test_checkpoints_have_the_arrays_of_their_shape():
    from cswap_amd.q8 import Checkpoint8

    assert (lambda h: (h.rows, h.cols))(checkpoint((2, 3, 40), 6, 40)) == (6, 40)
    assert (lambda h: (h.rows, h.cols))(checkpoint((2, 3, 40), 1, 240)) == (1, 240)       # flat
    assert checkpoint((2, 3, 40), 6, 40).nbytes == 6 * 64 + 6 * 2
    codes, scales = torch.zeros(6, 64, dtype=torch.int8), torch.zeros(6, 2, dtype=torch.uint8)
    for c, s, shape in ((codes, scales, (6, 65)), (codes, scales, (5, 40)), (codes[:, :32], scales, (6, 40)),
                        (codes, scales[:, :1], (6, 40)), (codes.int(), scales, (6, 40)), (codes, scales.int(), (6, 40)),
                        (codes.t(), scales, (64, 6)), (codes[0], scales, (6, 40))):
        with pytest.raises(ValueError):
            Checkpoint8(c, s, shape, torch.float32)
    with pytest.raises(TypeError):
        Checkpoint8(codes, scales, (6, 40), torch.float64)


def test_tensors_that_are_refused():
    from cswap_amd import q8

    x = torch.zeros(4, 40)
    held = checkpoint((4, 40), 4, 40)
    for call in (lambda: q8.q8_compress(x), lambda: q8.q8_decompress(held), lambda: q8.q8_act(x), lambda: q8.q8_act_backward(x, held),
                 lambda: q8.layer_norm(x), lambda: q8.layer_norm_backward(x, held, x, x), lambda: q8.q8_weight_grad(x, held)):
        with pytest.raises(ValueError, match="device memory"):
            call()
    with pytest.raises(TypeError):
        q8.q8_compress(x.double())
    with pytest.raises(ValueError):
        q8.q8_act(x, "relu")


def test_a_tensor_on_another_device_makes_that_device_current(monkeypatch):
    """The launch is on the tensor's device: where another is current, the call is made again with it current."""
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

    x = torch.zeros(4, 40).as_subclass(OnDevice1)
    monkeypatch.setattr(q8, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(api, "_raw_stream", lambda index: 1000 + index)
    monkeypatch.setattr(q8, "_empty_checkpoint", lambda t, rows, cols, device: checkpoint((4, 40), rows, cols))

    class Lib:
        @staticmethod
        def cswap_q8_pack(*a):
            launched.append((current[0], a[-1]))
            return 0

    monkeypatch.setattr(q8, "lib", lambda: Lib)
    q8.q8_compress(x)
    assert launched == [(1, 1001)] and current == [0]


def test_row_strides():
    from cswap_amd.q8 import _row_stride

    t = torch.zeros(4, 6, 10)
    assert _row_stride(t, "t") == 0
    assert _row_stride(t[:, :, :7], "t") == 10
    assert _row_stride(t[:, 2:3, :], "t") == 60
    assert _row_stride(t[:, :1, 3:4], "t") == 60
    assert _row_stride(t[1], "t") == 0
    for bad in (t.transpose(1, 2), t[:, :3, :], t[:, :, ::2], torch.zeros(1, 10).expand(4, 10), torch.zeros(4, 1).expand(4, 10)):
        with pytest.raises(ValueError):
            _row_stride(bad, "t")
