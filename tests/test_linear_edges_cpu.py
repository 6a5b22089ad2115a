"""CPU: what the linear-layer operators refuse, and what their host side does
when a call fails."""

import numpy as np
import pytest

import thork_b200 as tk
from thork_b200 import runtime as rt

K = tk.kernels
LONG = (1 << 23) + 16  # longer than a product may sum over


# ---------------------------------------------------------------- contractions
@pytest.mark.parametrize("make", [
    lambda: K.linear(4, 64, LONG), lambda: K.linear(4, 64, LONG, tk.dt.float8_e4m3),
    lambda: K.grouped_matmul(1, 32, 8, LONG), lambda: K.grouped_matmul(1, 32, 16, LONG, tk.dt.float8_e4m3)])
def test_contractions_that_a_kernel_cannot_finish_are_refused(make):
    with pytest.raises(ValueError, match="contraction over K"):
        make()


def test_gradients_refuse_the_contractions_that_they_compute():
    x = np.zeros(8, np.uint16)  # the sizes are refused before the arrays are looked at
    for f, rows in ((K.linear_backward(LONG, 8, 8), "M"), (K.grouped_matmul_backward(2, LONG, 8, 8), "T")):
        args = (None, x, None, x, x, None) if rows == "M" else (None, x, x, x, None, x)
        with pytest.raises(ValueError, match=f"contraction over {rows}="):
            f(*args)
    for f, args in ((K.linear_backward(8, LONG, 8), (x, None, None, x, None, x)),
                    (K.grouped_matmul_backward(2, 8, LONG, 8), (x, None, x, None, x, x))):
        with pytest.raises(ValueError, match="contraction over N="):
            f(*args)


def test_c_entry_points_refuse_long_contractions_and_only_those():
    L = rt.lib()

    def bad(rc, text):
        assert rc == rt.ERR_INVALID and text in rt.last_error(), rt.last_error()

    bad(L.thork_linear_bf16(16, 32, 48, None, None, None, 4, 64, LONG, 0, 0, None), "contraction over K")
    bad(L.thork_linear_e4m3(16, 32, 48, None, None, None, 4, 64, LONG, 1.0, 1.0, 0, 0, None), "contraction over K")
    bad(L.thork_grouped_gemm_bf16(16, 32, 48, 64, None, 2, 4, 64, LONG, 0, 0, None), "contraction over K")
    bad(L.thork_grouped_gemm_e4m3(16, 32, 48, 64, None, 2, 4, 64, LONG, 1.0, None, 0, 0, None), "contraction over K")
    bwd, gbwd = L.thork_linear_backward_bf16, L.thork_grouped_gemm_backward_bf16
    bad(bwd(16, None, None, 64, None, 96, None, None, 4, LONG, 64, 0, None), "contraction over N")
    bad(bwd(None, 32, None, 64, 80, None, None, None, LONG, 64, 64, 0, None), "contraction over M")
    bad(gbwd(16, None, 64, None, 96, 48, None, None, 2, 4, LONG, 64, 0, None), "contraction over N")
    bad(gbwd(None, 32, 64, 80, None, 48, None, None, 2, LONG, 64, 64, 0, None), "contraction over T")
    # a long size that nothing sums over passes this check (and fails a later one here)
    bad(L.thork_linear_bf16(16, 32, 48, None, None, None, LONG, 64, 64, 7, 0, None), "activation")
    bad(bwd(16, None, None, 64, None, 96, None, None, LONG, 64, 64, 7, None), "activation")
    bad(bwd(None, 32, None, 64, 80, None, None, None, 4, LONG, 64, 7, None), "activation")
