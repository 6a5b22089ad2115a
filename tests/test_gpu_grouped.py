"""GPU: tk.kernels.grouped_matmul and its backward pass against their 64-bit
forms, group by group (tolerances derived in linear_ref.py)."""

import numpy as np
import pytest

import thork_b200 as tk
from linear_ref import act, act_err, bits, close, product, sizes_to_offsets, slope, slope_err, wide
from oracle import oracle

pytestmark = pytest.mark.gpu
rt = tk.runtime

# sizes per expert, first row, rows of the buffer behind the last group
GROUPS = {
    "one": ([5], 0, 0),
    "empty": ([0, 0, 0], 0, 4),
    "single rows": ([1, 0, 1, 1], 0, 0),
    "thin": ([0, 3, 16, 17, 0, 1, 40, 2], 0, 5),
    "first offset": ([7, 0, 9], 6, 3),
    "sixteens": ([15, 16, 17, 31, 32, 33, 47, 48, 49, 80, 95], 0, 0),
    "tiles": ([64, 65, 128, 127, 63, 1], 0, 0),
    "wide": ([300, 0, 257, 256, 513], 0, 11),
    "skewed": ([1000, 2, 0, 130], 1, 1),
    "many": ([(i * 7) % 23 for i in range(70)], 0, 9),
    "most": ([i % 3 for i in range(1024)], 2, 1),
}


@pytest.fixture(autouse=True)
def _status():
    yield
    assert rt.kernel_status() == 0


def _layout(name):
    sizes, first, behind = GROUPS[name]
    off = sizes_to_offsets(sizes, first)
    return off, int(off[-1]) + behind


def _inside(off, t):
    return (np.arange(t) >= off[0]) & (np.arange(t) < off[-1])


@pytest.mark.parametrize("n,k", [(136, 72), (264, 1032)])
@pytest.mark.parametrize("name", sorted(GROUPS))
def test_grouped_matmul(name, n, k):
    off, t = _layout(name)
    e = len(off) - 1
    rng = np.random.default_rng(1)
    a, b = bits(rng, t, k), bits(rng, e, k, n, std=1.2 / np.sqrt(k))
    a[~_inside(off, t)] = 0x7FC0  # NaN in rows of no group must not spread
    for activation, keep in (("none", False), ("silu", True)):
        out = bits(rng, t, n)
        pre = bits(rng, t, n) if keep else None
        before, before_pre = out.copy(), None if pre is None else pre.copy()
        tk.kernels.grouped_matmul(e, t, n, k, activation=activation)(out, a, b, off, preact=pre)
        for i in range(e):
            r = slice(off[i], off[i + 1])
            z, err = product(wide(a[r]), wide(b[i]))
            if keep:
                close(pre[r], z, err, f"preact of group {i}") if z.size else None
            if z.size:
                close(out[r], act(z, activation), act_err(z, err), f"group {i}")
        rest = ~_inside(off, t)
        np.testing.assert_array_equal(out[rest], before[rest])
        if keep:
            np.testing.assert_array_equal(pre[rest], before_pre[rest])


@pytest.mark.parametrize("name", ["thin", "wide", "many", "tiles"])
@pytest.mark.parametrize("scaled", [True, False])
def test_grouped_matmul_e4m3(name, scaled):
    off, t = _layout(name)
    e, n, k = len(off) - 1, 272, 208
    rng = np.random.default_rng(2)
    qa, sa = tk.dt.quantize_e4m3(rng.standard_normal((t, k), dtype=np.float32))
    qb = np.stack([tk.dt.quantize_e4m3(rng.standard_normal((k, n), dtype=np.float32))[0] for _ in range(e)])
    sb = (0.5 + rng.random(e)).astype(np.float32) / 1000 if scaled else None
    out = bits(rng, t, n)
    before = out.copy()
    tk.kernels.grouped_matmul(e, t, n, k, tk.dt.float8_e4m3, activation="gelu_tanh")(
        out, qa, qb, off, scale_a=sa, scale_b=sb)
    A, B = oracle.e4m3_bits_to_f32(qa).astype(np.float64), oracle.e4m3_bits_to_f32(qb).astype(np.float64)
    for i in range(e):
        r = slice(off[i], off[i + 1])
        s = sa * (float(sb[i]) if scaled else 1.0)
        z, err = product(A[r], B[i])
        z, err = z * s, err * s + 2.0 ** -22 * np.abs(z) * s
        if z.size:
            close(out[r], act(z, "gelu_tanh"), act_err(z, err), f"group {i}")
    rest = ~_inside(off, t)
    np.testing.assert_array_equal(out[rest], before[rest])


@pytest.mark.parametrize("n,k", [(136, 72), (520, 264)])
@pytest.mark.parametrize("name", sorted(GROUPS))
def test_grouped_backward(name, n, k):
    off, t = _layout(name)
    e = len(off) - 1
    rng = np.random.default_rng(3)
    a, b = bits(rng, t, k), bits(rng, e, k, n, std=1.2 / np.sqrt(k))
    dout, z = bits(rng, t, n, std=1 / 64), bits(rng, t, n, std=1.5)
    rest = ~_inside(off, t)
    a[rest] = dout[rest] = z[rest] = 0x7FC0  # NaN behind the groups must not enter a sum
    for activation in ("none", "gelu_tanh"):
        bent = activation != "none"
        da, dz = bits(rng, t, k), bits(rng, t, n) if bent else None
        # dz of the rows of no group keeps NaN too: the weight gradient's last
        # rows of a group are loaded together with it
        if bent:
            dz[rest] = 0x7FC0
        before, before_dz = da.copy(), dz.copy() if bent else None
        db = np.full((e, k, n), 0x7FC0, np.uint16)
        tk.kernels.grouped_matmul_backward(e, t, n, k, activation=activation)(
            da, db, dout, a, b, off, z if bent else None, dz)
        for i in range(e):
            r = slice(off[i], off[i + 1])
            g = wide(dout[r])
            if bent and g.size:
                want = g * slope(wide(z[r]), activation)
                close(dz[r], want, np.abs(g) * slope_err(wide(z[r])), f"dpre of group {i}")
            gz = wide(dz[r]) if bent else g
            if g.size:
                close(da[r], *product(gz, wide(b[i]).T), f"dA of group {i}")
                close(db[i], *product(wide(a[r]).T, gz), f"dB of group {i}")
            else:
                assert (db[i] == 0).all(), f"dB of the empty group {i}"
        np.testing.assert_array_equal(da[rest], before[rest])
        if bent:
            np.testing.assert_array_equal(dz[rest], before_dz[rest])


def test_group_with_nan_leaves_the_others_gradients_alone():
    """The last k-block of a group's weight gradient also loads the next
    group's first rows: a NaN there must not count."""
    off = sizes_to_offsets([70, 40, 3])
    e, t, n, k = 3, 113, 136, 136
    rng = np.random.default_rng(4)
    a, b, dout = bits(rng, t, k), bits(rng, e, k, n), bits(rng, t, n)
    f = tk.kernels.grouped_matmul_backward(e, t, n, k)
    clean = np.zeros((e, k, n), np.uint16)
    f(None, clean, dout, a, None, off)
    a[70:110] = 0x7FC0
    dout[70:110] = 0xFF80
    got = np.zeros((e, k, n), np.uint16)
    f(None, got, dout, a, None, off)
    np.testing.assert_array_equal(got[[0, 2]], clean[[0, 2]])
    assert np.isnan(oracle.bf16_bits_to_f32(got[1])).all()


@pytest.mark.parametrize("name", ["thin", "wide"])
def test_captured_calls_replay_with_other_sizes(name):
    """A forward and a backward call captured into a graph, replayed after the
    offsets and the inputs changed in place, agree with direct calls bit for
    bit: nothing about the sizes is read by the host."""
    torch = pytest.importorskip("torch")
    off, t = _layout(name)
    e, n, k = len(off) - 1, 136, 264
    rng = np.random.default_rng(7)
    T = lambda x: torch.from_numpy(x.view(np.int16)).cuda().view(torch.bfloat16)  # noqa: E731
    W = lambda x, d=np.uint16: rt.wrap_pointer(x.data_ptr(), tuple(x.shape), d, owner=x)  # noqa: E731
    a, b, dout = T(bits(rng, t, k)), T(bits(rng, e, k, n, std=0.1)), T(bits(rng, t, n))
    offsets = torch.from_numpy(off).cuda()
    new = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    out, z, dz, da, db = new(t, n), new(t, n), new(t, n), new(t, k), new(e, k, n)
    f = tk.kernels.grouped_matmul(e, t, n, k, activation="silu")
    g = tk.kernels.grouped_matmul_backward(e, t, n, k, activation="silu")

    def both():
        s = rt.Stream.from_handle(torch.cuda.current_stream().cuda_stream)
        o = W(offsets, np.int32)
        f(W(out), W(a), W(b), o, preact=W(z), stream=s, sync=False)
        g(W(da), W(db), W(dout), W(a), W(b), o, W(z), W(dz), stream=s, sync=False)

    both()  # the first call allocates the status word
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    sizes = np.diff(off)[::-1]  # the same rows dealt out otherwise, and other values
    offsets.copy_(torch.from_numpy(sizes_to_offsets(sizes, int(off[0]))))
    a.copy_(T(bits(rng, t, k)))
    results = []
    for run in (both, graph.replay):
        for x in (out, z, dz, da, db):
            x.zero_()
        run()
        torch.cuda.synchronize()
        results.append([x.view(torch.int16).cpu().numpy() for x in (out, z, dz, da, db)])
    for x, y in zip(*results):
        np.testing.assert_array_equal(x, y)
    assert any(r.any() for r in results[0])


def test_offsets_that_are_wrong_are_clamped_and_reported():
    e, t, n, k = 4, 40, 136, 72
    rng = np.random.default_rng(5)
    a, b = bits(rng, t, k), bits(rng, e, k, n)
    off = np.array([-5, 10, 7, 1000, 20], np.int32)  # reads as 0, 10, 10, 40, 40
    want = np.zeros((t, n), np.uint16)
    f = tk.kernels.grouped_matmul(e, t, n, k)
    f(want, a, b, np.array([0, 10, 10, 40, 40], np.int32))
    assert rt.kernel_status() == 0
    out = np.zeros((t, n), np.uint16)
    f(out, a, b, off)
    assert rt.kernel_status() & 0xFF == 2
    np.testing.assert_array_equal(out, want)
    # the backward pass clamps alike
    dout = bits(rng, t, n)
    got = []
    for o in (off, np.array([0, 10, 10, 40, 40], np.int32)):
        da, db = np.zeros((t, k), np.uint16), np.zeros((e, k, n), np.uint16)
        dz, z = np.zeros((t, n), np.uint16), out
        tk.kernels.grouped_matmul_backward(e, t, n, k, activation="silu")(da, db, dout, a, b, o, z, dz)
        got.append((da, db, dz))
        assert rt.kernel_status() & 0xFF == (2 if o is off else 0)
    for x, y in zip(*got):
        np.testing.assert_array_equal(x, y)


def test_every_row_in_one_group():
    """The largest group that the buffer allows, with kernels chosen for a few
    rows a group."""
    e, t, n, k = 32, 500, 136, 72
    rng = np.random.default_rng(8)
    a, b = bits(rng, t, k), bits(rng, e, k, n, std=0.1)
    for at in (0, 17, 31):
        off = np.where(np.arange(e + 1) <= at, 0, t).astype(np.int32)
        out = np.zeros((t, n), np.uint16)
        tk.kernels.grouped_matmul(e, t, n, k)(out, a, b, off)
        close(out, *product(wide(a), wide(b[at])), f"group {at}")


def test_expert_layers_forward_and_backward():
    """Two grouped layers with an activation between, forward and backward,
    asynchronously on one stream, with offsets that live on the device."""
    sizes = [30, 0, 100, 7, 260]
    off = sizes_to_offsets(sizes)
    e, t, d, f = len(sizes), int(off[-1]), 136, 264
    rng = np.random.default_rng(6)
    x, w1, w2 = bits(rng, t, d), bits(rng, e, d, f, std=0.1), bits(rng, e, f, d, std=0.06)
    dy = bits(rng, t, d, std=0.1)
    D = {n: rt.to_device(v) for n, v in dict(x=x, w1=w1, w2=w2, dy=dy, off=off).items()}
    h, z, dz, dh = (rt.empty((t, f), np.uint16) for _ in range(4))
    y, dx = rt.empty((t, d), np.uint16), rt.empty((t, d), np.uint16)
    dw1, dw2 = rt.empty((e, d, f), np.uint16), rt.empty((e, f, d), np.uint16)
    s = rt.Stream()
    kw = dict(stream=s, sync=False)
    K = tk.kernels
    K.grouped_matmul(e, t, f, d, activation="silu")(h, D["x"], D["w1"], D["off"], preact=z, **kw)
    K.grouped_matmul(e, t, d, f)(y, h, D["w2"], D["off"], **kw)
    K.grouped_matmul_backward(e, t, d, f)(dh, dw2, D["dy"], h, D["w2"], D["off"], **kw)
    K.grouped_matmul_backward(e, t, f, d, activation="silu")(dx, dw1, dh, D["x"], D["w1"], D["off"], z, dz, **kw)
    s.synchronize()
    for i in range(e):
        r = slice(off[i], off[i + 1])
        if sizes[i] == 0:
            assert (dw1.to_host()[i] == 0).all() and (dw2.to_host()[i] == 0).all()
            continue
        H, DH, DZ = (wide(v.to_host()[r]) for v in (h, dh, dz))
        zz, err = product(wide(x[r]), wide(w1[i]))
        close(h.to_host()[r], act(zz, "silu"), act_err(zz, err), "h")
        close(y.to_host()[r], *product(H, wide(w2[i])), "y")
        close(dh.to_host()[r], *product(wide(dy[r]), wide(w2[i]).T), "dh")
        close(dw2.to_host()[i], *product(H.T, wide(dy[r])), "dw2")
        zb = wide(z.to_host()[r])
        close(dz.to_host()[r], DH * slope(zb, "silu"), np.abs(DH) * slope_err(zb), "dz")
        close(dx.to_host()[r], *product(DZ, wide(w1[i]).T), "dx")
        close(dw1.to_host()[i], *product(wide(x[r]).T, DZ), "dw1")


@pytest.mark.parametrize("sizes", [[2, 0, 1, 5], [30, 0, 100, 7, 260], [1, 16, 17, 300, 0, 64]])
def test_long_chains_without_a_wait_repeat_those_with_one(sizes):
    """Layers of experts forward and backward, queued without a wait, against
    the same calls one by one, bit for bit (see the dense form)."""
    off = sizes_to_offsets(sizes)
    e, t, d, f = len(sizes), int(off[-1]), 264, 392
    rng = np.random.default_rng(13)
    w1, w2 = rt.to_device(bits(rng, e, d, f, std=0.06)), rt.to_device(bits(rng, e, f, d, std=0.05))
    o = rt.to_device(off)
    x0, dy0 = bits(rng, t, d), bits(rng, t, d, std=0.1)
    K = tk.kernels
    up, down = K.grouped_matmul(e, t, f, d, activation="gelu"), K.grouped_matmul(e, t, d, f)
    up_b = K.grouped_matmul_backward(e, t, f, d, activation="gelu")
    down_b = K.grouped_matmul_backward(e, t, d, f)
    s = rt.Stream()

    def chain(sync):
        x, y, dy = rt.to_device(x0), rt.empty((t, d), np.uint16), rt.to_device(dy0)
        h, z, dz, dh = (rt.empty((t, f), np.uint16) for _ in range(4))
        dx, dw1, dw2 = rt.empty((t, d), np.uint16), rt.empty((e, d, f), np.uint16), rt.empty((e, f, d), np.uint16)
        kw = dict(stream=s, sync=sync)
        for _ in range(8):
            up(h, x, w1, o, preact=z, **kw)
            down(y, h, w2, o, **kw)
            down_b(dh, dw2, dy, h, w2, o, **kw)
            up_b(dx, dw1, dh, x, w1, o, z, dz, **kw)
            x, y, dy, dx = y, x, dx, dy
        s.synchronize()
        return [v.to_host() for v in (x, dy, h, z, dz, dh, dw1, dw2)]

    want = chain(True)
    for _ in range(3):
        for a, b in zip(chain(False), want):
            np.testing.assert_array_equal(a, b)
