"""GPU: every kernel, tile height and split that the linear-layer operators
choose from, against the 64-bit forms (shapes in linear_choices.py, tolerances
derived in linear_ref.py)."""

import numpy as np
import pytest

import linear_choices as C
import thork_b200 as tk
from linear_ref import act, act_err, bits, close, product, sizes_to_offsets, wide
from oracle import oracle

pytestmark = pytest.mark.gpu
rt = tk.runtime
NAN = 0x7FC0  # what an output holds before the call: an unwritten element fails


@pytest.fixture(autouse=True)
def _status():
    assert rt.sm_count() == C.SMS  # the choices are those of this many
    yield
    assert rt.kernel_status() == 0


def _e4m3(rng, *shape, std=1.0):
    q, scale = tk.dt.quantize_e4m3(rng.standard_normal(shape, dtype=np.float32) * np.float32(std))
    return q, scale, oracle.e4m3_bits_to_f32(q).astype(np.float64)


def _linear(m, n, k, dtype):
    rng = np.random.default_rng(m + n + k)
    bi, re = bits(rng, n, std=0.5), bits(rng, m, n)
    out, pre = np.full((m, n), NAN, np.uint16), np.full((m, n), NAN, np.uint16)
    if dtype == tk.dt.float8_e4m3:
        a, sa, wa = _e4m3(rng, m, k)
        b, sb, wb = _e4m3(rng, k, n, std=1.2 / np.sqrt(k))
        kw = dict(scale_a=sa, scale_b=sb)
    else:
        a, b, sa, sb, kw = bits(rng, m, k), bits(rng, k, n, std=1.2 / np.sqrt(k)), 1.0, 1.0, {}
        wa, wb = wide(a), wide(b)
    tk.kernels.linear(m, n, k, dtype, activation="silu")(out, a, b, bias=bi, residual=re, preact=pre, **kw)
    z, err = product(wa, wb)
    s = sa * sb
    # the scale's and the bias's rounding
    z, err = z * s + wide(bi), err * s + 2.0 ** -22 * (np.abs(z) * s + np.abs(wide(bi)))
    close(pre, z, err, "preact")
    y = act(z, "silu") + wide(re)
    close(out, y, act_err(z, err) + 2.0 ** -24 * np.abs(y), "out")


@pytest.mark.parametrize("m,n,k", C.FULL + C.PRODUCT)
def test_products(m, n, k):
    _linear(m, n, k, tk.dt.bfloat16)


@pytest.mark.parametrize("m,n,k", C.FULL + C.PRODUCT_E4M3)
def test_products_e4m3(m, n, k):
    _linear(m, n, k, tk.dt.float8_e4m3)


@pytest.mark.parametrize("m,n,k", C.FULL + C.PRODUCT)
def test_input_gradients(m, n, k):
    """dA[m, n] = dout[m, k] B[n, k]^T: the weights are read as they are stored."""
    rng = np.random.default_rng(m + n + k)
    dout, b = bits(rng, m, k, std=1 / 64), bits(rng, n, k, std=1.2 / np.sqrt(n))
    da = np.full((m, n), NAN, np.uint16)
    tk.kernels.linear_backward(m, k, n)(da, None, None, dout, None, b)
    close(da, *product(wide(dout), wide(b).T), "dA")


@pytest.mark.parametrize("m,n,k", C.WEIGHTS)
def test_weight_gradients(m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, dout, b = bits(rng, m, k), bits(rng, m, n, std=1 / 64), bits(rng, k, n)
    db = np.full((k, n), NAN, np.uint16)
    tk.kernels.linear_backward(m, n, k)(None, db, None, dout, a, None)
    want = product(wide(a).T, wide(dout))
    close(db, *want, "dB")
    # behind the other product of the call, without a wait of its own before it
    both = np.full((k, n), NAN, np.uint16)
    tk.kernels.linear_backward(m, n, k)(np.zeros((m, k), np.uint16), both, None, dout, a, b)
    np.testing.assert_array_equal(both, db)


def _offsets(e, t):
    """Sizes that leave one group empty and two rows of no group, where there
    are so many."""
    first, behind = (1, 1) if t > 4 else (0, 0)
    rows = t - first - behind
    sizes = [rows // 3, 0, rows - rows // 3]
    assert e == len(sizes)
    return sizes_to_offsets(sizes, first)


def _check_groups(off, got, before, want):
    for i in range(len(off) - 1):
        r = slice(off[i], off[i + 1])
        if off[i + 1] > off[i]:
            close(got[r], *want(i, r), f"group {i}")
    rest = np.ones(len(got), bool)
    rest[off[0]:off[-1]] = False
    np.testing.assert_array_equal(got[rest], before[rest])


@pytest.mark.parametrize("e,t,n,k", C.GROUPS)
def test_grouped_products_and_input_gradients(e, t, n, k):
    rng = np.random.default_rng(t + n + k)
    off = _offsets(e, t)
    a, b = bits(rng, t, k), bits(rng, e, k, n, std=1.2 / np.sqrt(k))
    before = bits(rng, t, n)
    out = before.copy()
    tk.kernels.grouped_matmul(e, t, n, k, activation="gelu")(out, a, b, off)

    def want(i, r):
        z, err = product(wide(a[r]), wide(b[i]))
        return act(z, "gelu"), act_err(z, err)

    _check_groups(off, out, before, want)
    # the same product as a gradient: dA[t, n] = dout[t, k] W[e, n, k]^T
    w = np.ascontiguousarray(b.transpose(0, 2, 1))
    da = before.copy()
    tk.kernels.grouped_matmul_backward(e, t, k, n)(da, None, a, None, w, off)
    _check_groups(off, da, before, lambda i, r: product(wide(a[r]), wide(b[i])))


@pytest.mark.parametrize("e,t,n,k", C.GROUPS_E4M3)
def test_grouped_products_e4m3(e, t, n, k):
    rng = np.random.default_rng(t + n + k)
    off = _offsets(e, t)
    a, sa, wa = _e4m3(rng, t, k)
    b, _, wb = _e4m3(rng, e, k, n)
    sb = (0.5 + rng.random(e)).astype(np.float32) / 448
    before = bits(rng, t, n)
    out = before.copy()
    tk.kernels.grouped_matmul(e, t, n, k, tk.dt.float8_e4m3, activation="silu")(
        out, a, b, off, scale_a=sa, scale_b=sb)

    def want(i, r):
        s = sa * float(sb[i])
        z, err = product(wa[r], wb[i])
        z, err = z * s, err * s + 2.0 ** -22 * np.abs(z) * s
        return act(z, "silu"), act_err(z, err)

    _check_groups(off, out, before, want)
