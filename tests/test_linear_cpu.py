"""The linear-layer operators' refusals (CPU): sizes, types, activations and
arguments are checked before a device is touched."""

import numpy as np
import pytest

import thork_b200 as tk
from thork_b200 import runtime as rt
from thork_b200.kernels._library import Operand

K = tk.kernels


@pytest.mark.parametrize("make", [
    lambda: K.linear(0, 64, 64), lambda: K.linear(4, 60, 64), lambda: K.linear(4, 64, 20),
    lambda: K.linear(4, 72, 64, tk.dt.float8_e4m3), lambda: K.linear(4, 64, 64, activation="tanh"),
    lambda: K.linear((1 << 30) + 1, 64, 64), lambda: K.linear_backward(-1, 64, 64),
    lambda: K.linear_backward(4, 64, 12), lambda: K.grouped_matmul(0, 4, 64, 64),
    lambda: K.grouped_matmul(1025, 4, 64, 64), lambda: K.grouped_matmul(2, 0, 64, 64),
    lambda: K.grouped_matmul(2, 4, 64, 72, tk.dt.float8_e4m3),
    lambda: K.grouped_matmul_backward(2, 4, 64, 64, activation="swish")])
def test_bad_sizes_and_activations(make):
    with pytest.raises(ValueError):
        make()


@pytest.mark.parametrize("make", [
    lambda: K.linear(4, 64, 64, tk.dt.float32), lambda: K.linear_backward(4, 64, 64, tk.dt.float8_e4m3),
    lambda: K.grouped_matmul(2, 4, 64, 64, tk.dt.float16),
    lambda: K.grouped_matmul_backward(2, 4, 64, 64, tk.dt.float8_e4m3)])
def test_bad_types(make):
    with pytest.raises(TypeError):
        make()


def test_arguments_that_do_not_go_together():
    z = np.zeros((4, 64), np.uint16)
    w = np.zeros((64, 64), np.uint16)
    off = np.zeros(3, np.int32)
    with pytest.raises(TypeError):
        K.linear(4, 64, 64)(None, z, w)
    with pytest.raises(ValueError):
        K.linear(4, 64, 64)(z, z, w, scale_a=2.0)
    with pytest.raises(ValueError):
        K.linear_backward(4, 64, 64, activation="silu")(z, None, None, z, z, w)
    with pytest.raises(ValueError):
        K.linear_backward(4, 64, 64)(z, None, None, z, z, w, preact=z)
    with pytest.raises(TypeError):
        K.linear_backward(4, 64, 64)(z, w, None, z, None, w)
    with pytest.raises(TypeError):
        K.grouped_matmul(2, 4, 64, 64)(z, z, w, None)
    with pytest.raises(ValueError):
        K.grouped_matmul(2, 4, 64, 64)(z, z, w, off, scale_b=np.ones(2, np.float32))
    with pytest.raises(TypeError):
        K.grouped_matmul_backward(2, 4, 64, 64)(None, w, z, None, None, off)


def test_operand_checks():
    o = Operand("A", tk.dt.bfloat16, (4, 64))
    o.check(np.zeros((4, 64), np.uint16), 0)
    with pytest.raises(TypeError):
        o.check([1, 2], 0)
    with pytest.raises(TypeError):
        o.check(np.zeros((4, 64), np.float32), 0)
    with pytest.raises(ValueError):
        o.check(np.zeros((4, 63), np.uint16), 0)
    with pytest.raises(ValueError):
        o.check(np.zeros((64, 4), np.uint16).T, 0)

    class Elsewhere:
        ptr, nbytes, _dev = 4096, 512, 1

    d = rt.DeviceArray((4, 64), np.uint16, buffer=Elsewhere())
    o.check(d, 1)
    with pytest.raises(ValueError, match="device 1"):
        o.check(d, 0)
    Elsewhere.ptr = 0
    with pytest.raises(ValueError, match="freed"):
        o.check(d, 1)


def test_borrowed_streams_stay_their_owners(monkeypatch):
    destroyed = []
    monkeypatch.setattr(rt.lib(), "thork_stream_destroy", destroyed.append, raising=False)
    s = rt.Stream.from_handle(0)
    assert s.handle is None  # the legacy default stream
    s.close()
    s = rt.Stream.from_handle(4096)
    assert s.handle == 4096
    s.close()
    assert s.handle is None and not destroyed


def test_c_entry_points_refuse_before_touching_a_device():
    L = rt.lib()

    def bad(rc, text):
        assert rc == rt.ERR_INVALID
        assert text in rt.last_error(), rt.last_error()

    lin = L.thork_linear_bf16
    bad(lin(None, 32, 48, None, None, None, 4, 64, 64, 0, 0, None), "A is NULL")
    bad(lin(16, 32, None, None, None, None, 4, 64, 64, 0, 0, None), "out is NULL")
    bad(lin(16, 32, 48, 8, None, None, 4, 64, 64, 0, 0, None), "bias must be 16-byte aligned")
    bad(lin(16, 32, 48, None, 8, None, 4, 64, 64, 0, 0, None), "residual must be 16-byte aligned")
    bad(lin(16, 32, 16, None, None, None, 4, 64, 64, 0, 0, None), "same array")
    bad(lin(16, 32, 48, None, 64, 64, 4, 64, 64, 0, 0, None), "same array")
    bad(lin(16, 32, 48, None, None, None, 4, 60, 64, 0, 0, None), "multiples of 8")
    bad(lin(16, 32, 48, None, None, None, 0, 64, 64, 0, 0, None), "positive")
    bad(lin(16, 32, 48, None, None, None, (1 << 30) + 1, 64, 64, 0, 0, None), "at most 2^30")
    bad(lin(16, 32, 48, None, None, None, 4, 64, 64, 5, 0, None), "activation")
    bad(lin(16, 32, 48, None, None, None, 4, 64, 64, 0, 2, None), "flags")
    bad(L.thork_linear_e4m3(16, 32, 48, None, None, None, 4, 72, 64, 1.0, 1.0, 0, 0, None), "multiples of 16")
    bwd = L.thork_linear_backward_bf16
    bad(bwd(16, 32, 48, 64, 80, 96, None, None, 4, 64, 64, 4, None), "preact and dpre")
    bad(bwd(16, 32, 48, 64, 80, 96, 112, 128, 4, 64, 64, 0, None), "preact and dpre")
    bad(bwd(16, 32, 48, None, 80, 96, None, None, 4, 64, 64, 0, None), "dout is NULL")
    bad(bwd(16, 32, 48, 64, None, 96, None, None, 4, 64, 64, 0, None), "A is NULL")
    bad(bwd(16, 32, 48, 64, 80, 96, 112, 64, 4, 64, 64, 1, None), "same array")
    g = L.thork_grouped_gemm_bf16
    bad(g(16, 32, 48, None, None, 2, 4, 64, 64, 0, 0, None), "offsets")
    bad(g(16, 32, 48, 6, None, 2, 4, 64, 64, 0, 0, None), "offsets")
    bad(g(16, 32, 48, 64, None, 0, 4, 64, 64, 0, 0, None), "E=0")
    bad(g(16, 32, 48, 64, None, 1025, 4, 64, 64, 0, 0, None), "E=1025")
    bad(L.thork_grouped_gemm_e4m3(16, 32, 48, 64, None, 2, 4, 64, 64, 1.0, 6, 0, 0, None), "scale_b")
    bad(L.thork_grouped_gemm_backward_bf16(16, 32, 48, 64, 80, None, None, None, 2, 4, 64, 64, 0, None),
        "offsets")
