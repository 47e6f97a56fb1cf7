"""CPU: sizes whose tile counts would pass 32 bits are refused before anything is counted."""
import pytest

A = 1 << 20   # an aligned address that is never read: every call here is refused first


@pytest.mark.parametrize("big", ["M", "N", "K"])
@pytest.mark.parametrize("size", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 1016])
def test_linear_refuses_sizes_near_2_31(big, size):
    from edge_maskgit_b200._lib import lib
    call = dict(dtype=1, x=A, ldx=1 << 32, w=A, ldw=1 << 32, M=4, N=8, K=64, bias=None, act=0, resid=None, ldr=0, y=A,
                ldy=1 << 32, st=None)
    call[big] = size - size % 8 if big == "K" else size
    assert lib.mgc_linear(*call.values()) == -1
    assert "2^31 - 1024" in lib.mgc_last_error().decode()
