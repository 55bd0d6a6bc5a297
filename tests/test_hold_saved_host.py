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
