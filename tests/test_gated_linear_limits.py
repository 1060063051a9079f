"""What the gated projection refuses, it refuses before the forward pass: a training forward whose backward pass could not run is refused itself.  By the sizes alone: no operand is there
(the pointers are never read), so this runs without a GPU."""
import pytest

from cagc import _lib

NOWHERE = 4096


def forward(n, dtype, saved):
    lib = _lib.load()
    rc = lib.cagc_gated_linear_fwd(None, NOWHERE if saved else None, None, None, None, None, None, None, 1, n, 8, 8, 8, dtype, dtype, 0, 1.0, None)
    return rc, lib.cagc_last_error().decode()


def backward(n, dtype):
    lib = _lib.load()
    rc = lib.cagc_gated_linear_bwd(NOWHERE, None, None, None, None, None, None, None, 1, n, 8, 8, 8, n, dtype, 0, 1.0, None)
    return rc, lib.cagc_last_error().decode()


@pytest.mark.parametrize("dtype, size", [(0, 4), (1, 2), (3, 2)])
def test_columns(dtype, size):
    most = ((7 << 20) // size - 16) // 2      # 2n values of dz, and a chunk, within 7 MiB
    for n in (most + 1, 1 << 24, 1 << 26):
        rc, why = forward(n, dtype, saved=True)
        assert rc != 0 and "n too large" in why
        assert "n too large" in backward(n, dtype)[1]
        assert "null pointer" in forward(n, dtype, saved=False)[1]      # without the backward pass there is no such limit
    assert "null pointer" in forward(most, dtype, saved=True)[1] and "null pointer" in backward(most, dtype)[1]
