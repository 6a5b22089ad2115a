"""GPU: tk.kernels.linear and tk.kernels.linear_backward against their 64-bit
forms (tolerances derived in linear_ref.py)."""

import numpy as np
import pytest

import thork_b200 as tk
from linear_ref import (ACTS, act, act_err, bits, close, product, slope, slope_err, wide)
from oracle import oracle

pytestmark = pytest.mark.gpu
rt = tk.runtime


@pytest.fixture(autouse=True)
def _status():
    yield
    assert rt.kernel_status() == 0


def _forward(m, n, k, activation, bias, residual, preact, seed=0, **kw):
    rng = np.random.default_rng(seed)
    a, b = bits(rng, m, k), bits(rng, k, n, std=1.2 / np.sqrt(k))
    bi = bits(rng, n, std=0.5) if bias else None
    re = bits(rng, m, n) if residual else None
    pre = np.full((m, n), 0x7FC0, np.uint16) if preact else None
    out = np.full((m, n), 0x7FC0, np.uint16)  # NaN bits: an unwritten element fails
    tk.kernels.linear(m, n, k, activation=activation, **kw)(out, a, b, bias=bi, residual=re, preact=pre)
    z, err = product(wide(a), wide(b))
    if bias:
        z = z + wide(bi)
        err = err + 2.0 ** -24 * np.abs(z)
    if preact:
        close(pre, z, err, "preact")
    y, err = act(z, activation), act_err(z, err)
    if residual:
        y = y + wide(re)
        err = err + 2.0 ** -24 * np.abs(y)
    close(out, y, err, "out")


@pytest.mark.parametrize("activation", ACTS)
@pytest.mark.parametrize("m,n,k", [(5, 264, 136), (300, 264, 200)])
def test_linear_activations(m, n, k, activation):
    _forward(m, n, k, activation, True, True, True)


# few rows (every tile height and both sides of each), split contractions,
# pairs of both widths, sizes that end inside every tile
SHAPES = [(1, 8, 8), (1, 4096, 1024), (2, 128, 64), (16, 1000, 4096), (17, 256, 72), (32, 136, 2048),
          (33, 520, 512), (64, 1024, 640), (65, 264, 1032), (100, 2304, 512), (128, 128, 4096),
          (129, 8, 8), (256, 256, 64), (257, 264, 328), (777, 1544, 1032), (512, 128, 1000),
          (1000, 4104, 256), (2304, 2304, 192)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_shapes(m, n, k):
    _forward(m, n, k, "none", False, False, False, seed=1)
    _forward(m, n, k, "silu", True, True, True, seed=2, static_weights=True)


@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("bias,residual,preact", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_linear_optional_arguments(m, bias, residual, preact):
    _forward(m, 392, 264, "relu", bias, residual, preact, seed=3)


@pytest.mark.parametrize("m,n,k", [(1, 528, 272), (20, 256, 1040), (48, 1040, 512), (128, 400, 2048),
                                   (300, 528, 272), (1030, 2064, 384)])
def test_linear_e4m3(m, n, k):
    rng = np.random.default_rng(4)
    qa, sa = tk.dt.quantize_e4m3(rng.standard_normal((m, k), dtype=np.float32))
    qb, sb = tk.dt.quantize_e4m3(rng.standard_normal((k, n), dtype=np.float32) / np.float32(np.sqrt(k)))
    bi, re = bits(rng, n), bits(rng, m, n)
    out, pre = (np.full((m, n), 0x7FC0, np.uint16) for _ in range(2))
    tk.kernels.linear(m, n, k, tk.dt.float8_e4m3, activation="gelu_tanh")(
        out, qa, qb, bias=bi, residual=re, preact=pre, scale_a=sa, scale_b=sb)
    z, err = product(oracle.e4m3_bits_to_f32(qa).astype(np.float64), oracle.e4m3_bits_to_f32(qb).astype(np.float64))
    s = sa * sb
    z, err = z * s + wide(bi), err * s + 2.0 ** -22 * (np.abs(z) * s + np.abs(wide(bi)))
    close(pre, z, err, "preact")
    y = act(z, "gelu_tanh") + wide(re)
    close(out, y, act_err(z, err) + 2.0 ** -24 * np.abs(y), "out")


@pytest.mark.parametrize("m", [7, 300])
def test_linear_residual_in_place_and_device_arrays(m):
    """out may be the residual; repeated asynchronous calls on a stream of the
    user's own agree with host calls bit for bit."""
    n, k = 520, 264
    rng = np.random.default_rng(5)
    a, b, re = bits(rng, m, k), bits(rng, k, n, std=0.05), bits(rng, m, n)
    f = tk.kernels.linear(m, n, k, activation="relu")
    want = np.zeros((m, n), np.uint16)
    f(want, a, b, residual=re)
    da, db, dr = (rt.to_device(x) for x in (a, b, re))
    s = rt.Stream()
    f(dr, da, db, residual=dr, stream=s, sync=False)
    s.synchronize()
    np.testing.assert_array_equal(dr.to_host(), want)
    other = rt.Stream.from_handle(s.handle)
    out = rt.empty((m, n), np.uint16)
    dr = rt.to_device(re)
    f(out, da, db, residual=dr, stream=other, sync=False)
    other.close()  # borrowed: the stream stays usable
    s.synchronize()
    np.testing.assert_array_equal(out.to_host(), want)
    host = re.copy()
    f(host, a, b, residual=host)
    np.testing.assert_array_equal(host, want)


@pytest.mark.parametrize("m", [4, 64, 400])
def test_linear_special_values_stay_in_their_rows(m):
    """A row with NaN or infinity spoils that row alone; relu keeps NaN."""
    n, k = 264, 200
    rng = np.random.default_rng(6)
    a, b = bits(rng, m, k), bits(rng, k, n, std=0.1)
    f = tk.kernels.linear(m, n, k, activation="relu")
    clean, out = (np.zeros((m, n), np.uint16) for _ in range(2))
    f(clean, a, b)
    a[1, 3] = 0x7FC0
    a[2, 5] = 0x7F80
    f(out, a, b)
    keep = np.arange(m) > 2
    keep[0] = True
    np.testing.assert_array_equal(out[keep], clean[keep])
    assert np.isnan(oracle.bf16_bits_to_f32(out[1])).all()
    # +inf times weights of either sign: relu leaves 0 or +inf
    assert np.isin(oracle.bf16_bits_to_f32(out[2]), [0.0, np.inf]).all()


@pytest.mark.parametrize("m,n,k", [(1, 1024, 8192), (16, 512, 4096), (300, 512, 512)])
def test_linear_repeats_bit_for_bit_on_two_streams(m, n, k):
    rng = np.random.default_rng(7)
    a, b = rt.to_device(bits(rng, m, k)), rt.to_device(bits(rng, k, n, std=0.02))
    f = tk.kernels.linear(m, n, k, activation="silu", static_weights=True)
    streams = [rt.Stream(), rt.Stream()]
    outs = [rt.empty((m, n), np.uint16) for _ in range(8)]
    for i, o in enumerate(outs):
        f(o, a, b, stream=streams[i % 2], sync=False)
    for s in streams:
        s.synchronize()
    first = outs[0].to_host()
    for o in outs[1:]:
        np.testing.assert_array_equal(o.to_host(), first)


def test_linear_output_past_2_31_elements():
    """Rows whose elements lie beyond 2^31 (a 4.3 GB output): the first and the
    last rows against the formula, on the product and on the bias gradient's
    kernel."""
    n, k = 14336, 8
    m = (1 << 31) // n + 200
    rng = np.random.default_rng(10)
    a, b = bits(rng, m, k), bits(rng, k, n)
    A, B, out, dout = rt.to_device(a), rt.to_device(b), rt.empty((m, n), np.uint16), rt.empty((m, n), np.uint16)
    f = tk.kernels.linear(m, n, k, activation="relu")
    f(out, A, B, preact=dout)

    def rows(x, r0, r1):
        got = np.empty((r1 - r0, n), np.uint16)
        rt.copy_dtoh(got, x.ptr + r0 * n * 2)
        return got

    for r0, r1 in ((0, 70), (m - 130, m)):
        z, err = product(wide(a[r0:r1]), wide(b))
        close(rows(out, r0, r1), np.maximum(z, 0), err, f"rows {r0}..{r1}")
    # dpre = dout * (preact > 0) with dout = preact is the output again
    dpre, dbias = rt.empty((m, n), np.uint16), rt.empty((n,), np.float32)
    tk.kernels.linear_backward(m, n, k, activation="relu")(None, None, dbias, dout, None, None, dout, dpre)
    for r0, r1 in ((0, 70), (m - 130, m)):
        np.testing.assert_array_equal(oracle.bf16_bits_to_f32(rows(dpre, r0, r1)),
                                      oracle.bf16_bits_to_f32(rows(out, r0, r1)))


# ---------------------------------------------------------------- backward
def _backward(m, n, k, activation, seed=0):
    rng = np.random.default_rng(seed)
    a, b = bits(rng, m, k), bits(rng, k, n, std=1.2 / np.sqrt(k))
    dout = bits(rng, m, n, std=1 / 64)
    bent = activation != "none"
    pre = bits(rng, m, n, std=1.5) if bent else None
    dpre = np.full((m, n), 0x7FC0, np.uint16) if bent else None
    da, db = np.full((m, k), 0x7FC0, np.uint16), np.full((k, n), 0x7FC0, np.uint16)
    dbias = np.full((n,), np.nan, np.float32)
    tk.kernels.linear_backward(m, n, k, activation=activation)(da, db, dbias, dout, a, b, pre, dpre)
    g = wide(dout)
    err = np.zeros_like(g)
    if bent:
        z = wide(pre)
        err = np.abs(g) * slope_err(z)
        g = g * slope(z, activation)
        close(dpre, g, err, "dpre")
    # the bias gradient sums the unrounded dpre in fp32: each addition rounds
    # the partial sum, at most the sum of magnitudes
    mags = np.abs(g).sum(0)
    tol = err.sum(0) + (m + 40) * 2.0 ** -24 * mags
    assert (np.abs(dbias - g.sum(0)) <= tol).all(), "dbias"
    # the products read dpre as rounded to bf16
    gz = wide(dpre) if bent else g
    close(da, *product(gz, wide(b).T), "dA")
    close(db, *product(wide(a).T, gz), "dB")


@pytest.mark.parametrize("activation", ACTS)
def test_linear_backward_activations(activation):
    _backward(200, 264, 136, activation)


@pytest.mark.parametrize("m,n,k", [(1, 8, 8), (1, 256, 512), (13, 136, 264), (40, 1024, 128),
                                   (100, 520, 1032), (128, 64, 64), (257, 328, 264), (1000, 776, 520),
                                   (2500, 136, 2304), (640, 2304, 2304), (2604, 184, 152), (3001, 520, 264),
                                   (4100, 72, 1000), (6000, 1032, 520)])
def test_linear_backward_shapes(m, n, k):
    _backward(m, n, k, "silu", seed=1)
    _backward(m, n, k, "none", seed=2)


def test_linear_backward_leaves_out_what_is_not_asked_for():
    m, n, k = 70, 136, 72
    rng = np.random.default_rng(3)
    a, b, dout = bits(rng, m, k), bits(rng, k, n), bits(rng, m, n)
    f = tk.kernels.linear_backward(m, n, k)
    whole = [np.zeros((m, k), np.uint16), np.zeros((k, n), np.uint16), np.zeros(n, np.float32)]
    f(*whole, dout, a, b)
    for i in range(3):
        some = [np.zeros_like(w) if j == i else None for j, w in enumerate(whole)]
        f(*some, dout, a if i == 1 else None, b if i == 0 else None)
        np.testing.assert_array_equal(some[i], whole[i])


@pytest.mark.parametrize("activation", ["gelu", "gelu_tanh", "silu"])
def test_linear_backward_against_differences(activation):
    """<gradient, direction> against a central difference of the 64-bit loss
    sum(dout * act(A B + bias)) along random directions.  The kernels' own
    forward pass supplies preact, so its rounding (2^-8 of z) moves the
    slope by at most |slope'| <= 1.1 times that; dpre, dA and dB each add a
    rounding of 2^-8.  Per element the errors are bounded; along a direction
    they add as magnitudes at most."""
    m, n, k = 48, 72, 40
    rng = np.random.default_rng(8)
    a, b, bi = bits(rng, m, k), bits(rng, k, n, std=0.2), bits(rng, n, std=0.5)
    dout = bits(rng, m, n)
    out, pre, dpre = (np.zeros((m, n), np.uint16) for _ in range(3))
    tk.kernels.linear(m, n, k, activation=activation)(out, a, b, bias=bi, preact=pre)
    da, db, dbias = np.zeros((m, k), np.uint16), np.zeros((k, n), np.uint16), np.zeros(n, np.float32)
    tk.kernels.linear_backward(m, n, k, activation=activation)(da, db, dbias, dout, a, b, pre, dpre)
    A, B, C, G = wide(a), wide(b), wide(bi), wide(dout)

    def loss(t, ua, ub, uc):
        return float((G * act((A + t * ua) @ (B + t * ub) + C + t * uc, activation)).sum())

    z = A @ B + C
    g_err = np.abs(G) * (1.1 * 2.0 ** -8 * np.abs(z) + 2.0 ** -8 * 1.13 + 2.0 ** -16)
    for which in range(3):
        u = [np.zeros_like(A), np.zeros_like(B), np.zeros_like(C)]
        u[which] = rng.standard_normal(u[which].shape)
        h = 1e-5
        want = (loss(h, *u) - loss(-h, *u)) / (2 * h)
        got = float((wide(da) * u[0]).sum() + (wide(db) * u[1]).sum() + (dbias.astype(np.float64) * u[2]).sum())
        carried = np.abs(g_err * (np.abs(u[0]) @ np.abs(B) + np.abs(A) @ np.abs(u[1]) + np.abs(u[2]))).sum()
        rounded = 2.0 ** -8 * ((np.abs(wide(da)) * np.abs(u[0])).sum() + (np.abs(wide(db)) * np.abs(u[1])).sum())
        assert abs(got - want) <= carried + rounded + 1e-5 * abs(want) + 1e-6


def test_training_step_of_two_layers():
    """Forward and backward of x + W2 gelu(W1 x + b1) + b2, every array on the
    device and every call on one stream without a wait in between."""
    t, d, f = 192, 136, 520
    rng = np.random.default_rng(9)
    x, w1, w2 = bits(rng, t, d), bits(rng, d, f, std=0.09), bits(rng, f, d, std=0.05)
    b1, b2, dy = bits(rng, f, std=0.3), bits(rng, d, std=0.3), bits(rng, t, d, std=0.1)
    D = {n: rt.to_device(v) for n, v in dict(x=x, w1=w1, w2=w2, b1=b1, b2=b2, dy=dy).items()}
    h, z, dz, dh = (rt.empty((t, f), np.uint16) for _ in range(4))
    y, dx = rt.empty((t, d), np.uint16), rt.empty((t, d), np.uint16)
    dw1, dw2 = rt.empty((d, f), np.uint16), rt.empty((f, d), np.uint16)
    db1, db2 = rt.empty((f,), np.float32), rt.empty((d,), np.float32)
    s = rt.Stream()
    kw = dict(stream=s, sync=False)
    L = tk.kernels
    L.linear(t, f, d, activation="gelu")(h, D["x"], D["w1"], bias=D["b1"], preact=z, **kw)
    L.linear(t, d, f)(y, h, D["w2"], bias=D["b2"], residual=D["x"], **kw)
    L.linear_backward(t, d, f)(dh, dw2, db2, D["dy"], h, D["w2"], **kw)
    L.linear_backward(t, f, d, activation="gelu")(dx, dw1, db1, dh, D["x"], D["w1"], z, dz, **kw)
    s.synchronize()
    # each stage against the formula on what the stage before left
    zz, err = product(wide(x), wide(w1))
    zz = zz + wide(b1)
    close(z.to_host(), zz, err + 2.0 ** -23 * np.abs(zz), "z")
    close(h.to_host(), act(zz, "gelu"), act_err(zz, err), "h")
    H = wide(h.to_host())
    yy, err = product(H, wide(w2))
    yy = yy + wide(b2) + wide(x)
    close(y.to_host(), yy, err + 2.0 ** -22 * (np.abs(yy) + 8), "y")
    close(dh.to_host(), *product(wide(dy), wide(w2).T), "dh")
    close(dw2.to_host(), *product(H.T, wide(dy)), "dw2")
    gz = wide(dh.to_host()) * slope(wide(z.to_host()), "gelu")
    close(dz.to_host(), gz, np.abs(wide(dh.to_host())) * slope_err(wide(z.to_host())), "dz")
    DZ = wide(dz.to_host())
    close(dx.to_host(), *product(DZ, wide(w1).T), "dx")
    close(dw1.to_host(), *product(wide(x).T, DZ), "dw1")
    assert np.abs(db1.to_host() - gz.sum(0)).max() <= 1e-4
    assert np.abs(db2.to_host() - wide(dy).sum(0)).max() <= 1e-4


@pytest.mark.parametrize("t,d,f", [(8, 264, 520), (160, 136, 392), (700, 520, 1032)])
def test_long_chains_without_a_wait_repeat_those_with_one(t, d, f):
    """Twelve layers forward (the residual updated in place) and backward, each
    call's inputs written by the call before it and its outputs read by the
    next: queued without a wait, every array is bit for bit what the same calls
    give one by one.  The kernels of a stream overlap, so a missing wait for the
    previous kernel would show here."""
    rng = np.random.default_rng(12)
    layers = 12
    w1 = [rt.to_device(bits(rng, d, f, std=0.06)) for _ in range(3)]
    w2 = [rt.to_device(bits(rng, f, d, std=0.03)) for _ in range(3)]
    x0, dy0 = bits(rng, t, d), bits(rng, t, d, std=0.1)
    L = tk.kernels
    up, down = L.linear(t, f, d, activation="silu", static_weights=True), L.linear(t, d, f, static_weights=True)
    up_b, down_b = L.linear_backward(t, f, d, activation="silu"), L.linear_backward(t, d, f)
    s = rt.Stream()

    def chain(sync):
        x, dy = rt.to_device(x0), rt.to_device(dy0)
        h, z, dz, dh = (rt.empty((t, f), np.uint16) for _ in range(4))
        dx, dw1, dw2, db = (rt.empty((t, d), np.uint16), rt.empty((d, f), np.uint16),
                            rt.empty((f, d), np.uint16), rt.empty((f,), np.float32))
        kw = dict(stream=s, sync=sync)
        seen = []
        for i in range(layers):
            up(h, x, w1[i % 3], preact=z, **kw)
            down(x, h, w2[i % 3], residual=x, **kw)
            down_b(dh, dw2, None, dy, h, w2[i % 3], **kw)
            up_b(dx, dw1, db, dh, x, w1[i % 3], z, dz, **kw)
            dy, dx = dx, dy
        s.synchronize()
        seen += [v.to_host() for v in (x, dy, h, z, dz, dh, dw1, dw2, db)]
        return seen

    want = chain(True)
    for _ in range(3):
        for a, b in zip(chain(False), want):
            np.testing.assert_array_equal(a, b)
