"""GPU: calls of the linear-layer operators in unusual company: slow kernels
before them, status words, extreme values (tolerances derived in
linear_ref.py)."""

import ctypes
import math

import numpy as np
import pytest

import thork_b200 as tk
from linear_ref import BF16, act, act_err, bits, close, product, wide
from oracle import oracle

pytestmark = pytest.mark.gpu
rt = tk.runtime


@pytest.fixture(autouse=True)
def _status():
    yield
    assert rt.kernel_status() == 0


# Lets its successor start at once and then takes `ns` nanoseconds, as a
# barrier between GPUs does while a peer is late.  The loop ends by count too.
SLOW = """
extern "C" __global__ void slow(unsigned long long ns) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  unsigned long long t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  for (int i = 0; i < 40000; ++i) {
    __nanosleep(100000);
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t - t0 > ns) break;
  }
}
"""


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (5, 264, 2056), (48, 512, 1024)])
def test_a_product_behind_a_slow_kernel_waits_for_it(m, n, k):
    """A product of few rows starts beside the kernel before it; its one-second
    limit must not count the time that that kernel takes (1.4 s here)."""
    rng = np.random.default_rng(1)
    a, b = bits(rng, m, k), bits(rng, k, n, std=0.05)
    A, B, out = rt.to_device(a), rt.to_device(b), rt.empty((m, n), np.uint16)
    out.zero()
    f = tk.kernels.linear(m, n, k, activation="silu", static_weights=True)
    s = rt.Stream()
    f(out, A, B, stream=s)  # the kernels are loaded
    out.zero(s)
    slow = rt.compile_source(SLOW).function("slow")
    rt.launch(slow, (1, 1, 1), (32, 1, 1), [ctypes.c_ulonglong(1_400_000_000)], stream=s)
    f(out, A, B, stream=s, sync=False)
    s.synchronize()
    assert rt.kernel_status() == 0
    z, err = product(wide(a), wide(b))
    close(out.to_host(), act(z, "silu"), act_err(z, err), "out")


def _threes(*shape):
    d = rt.empty(shape, np.uint16)
    rt.check(rt.lib().thork_memset(d.ptr, 0x40, d.nbytes, None))  # 0x4040: 3.0
    return d


LONGEST = 1 << 23


def _all_of_it(out):
    """2^23 products of 9, summed by tensor cores, which may cut a product to
    the running sum's last bit (74.5e6 measured without a split, 75.5e6 with
    one).  The sum stays below 2^27, so that bit is at most 8, and of each 9 at
    least 8 is added; 2^26 and 9 2^23 are bf16 numbers."""
    got = wide(out.to_host())
    assert ((got >= 8.0 * LONGEST) & (got <= 9.0 * LONGEST)).all(), got


@pytest.mark.parametrize("rows", [2, 32])
def test_the_longest_contraction_of_a_product(rows):
    """One tile, whose accumulator is waited for through 131072 blocks
    (swap_kernel splits them; rows_kernel, which 32 rows a group go to, does
    not)."""
    a, b = _threes(rows, LONGEST), _threes(1, LONGEST, 8)
    out = rt.empty((rows, 8), np.uint16)
    out.zero()
    tk.kernels.grouped_matmul(1, rows, 8, LONGEST)(out, a, b, np.array([0, rows], np.int32))
    _all_of_it(out)


def test_the_longest_contraction_of_a_gradient():
    a, dout = _threes(LONGEST, 8), _threes(LONGEST, 8)
    db = rt.empty((1, 8, 8), np.uint16)
    for call in (lambda: tk.kernels.grouped_matmul_backward(1, LONGEST, 8, 8)(
                     None, db, dout, a, None, np.array([0, LONGEST], np.int32)),
                 lambda: tk.kernels.linear_backward(LONGEST, 8, 8)(None, db, None, dout, a, None)):
        db.zero()
        call()
        _all_of_it(db)


def _stream_status(stream):
    v = ctypes.c_uint(0)
    rt.check(rt.lib().thork_stream_status(ctypes.byref(v), stream.handle))
    return v.value


@pytest.mark.parametrize("t", [40, 600])
def test_what_a_kernel_reports_is_read_behind_its_stream(t):
    """The operators report to a word of their own, which a call that
    synchronises looks at (wrong offsets stay in it, an expired wait is
    raised); kernel_status shows and clears it."""
    e, n, k = 4, 136, 72
    rng = np.random.default_rng(2)
    A, B, out = rt.to_device(bits(rng, t, k)), rt.to_device(bits(rng, e, k, n)), rt.empty((t, n), np.uint16)
    good = rt.to_device(np.array([0, 10, 10, 30, t], np.int32))
    bad = rt.to_device(np.array([0, 10, 7, 30, 5 * t], np.int32))
    f = tk.kernels.grouped_matmul(e, t, n, k)
    s = rt.Stream()
    f(out, A, B, good, stream=s, sync=False)
    assert _stream_status(s) == 0
    f(out, A, B, bad, stream=s, sync=False)
    assert _stream_status(s) == 2 | 0x40 << 8
    f(out, A, B, good, stream=s)
    assert rt.kernel_status(clear=False) == 2 | 0x40 << 8
    assert rt.kernel_status() == 2 | 0x40 << 8
    assert rt.kernel_status() == 0 and _stream_status(s) == 0
    # a word planted on the device, as another kernel's expired wait leaves it,
    # is that kernel's caller's to read
    rt.copy_htod(rt.status_pointer(), np.array([1 | 0x14 << 8], np.uint32))
    f(out, A, B, good, stream=s)
    assert rt.kernel_status() == 1 | 0x14 << 8


@pytest.mark.parametrize("which", ["linear ragged 777", "linear backward 200", "grouped backward odd"])
def test_measured_calls_follow_the_current_stream(which):
    """The calls of perf/operators.py on one state: eager, on another stream,
    captured and replayed, with a buffer replaced."""
    import importlib.util
    import os

    torch = pytest.importorskip("torch")
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("measured_operators", path)
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    case = next(c for c in ops.listed() if c["name"] == which)
    state = ops.prepare(case, 3)
    before = {name: x.clone() for name, x in ops.run(state).items()}

    def fresh():
        for x in ops.run(state).values():  # rows behind the last group keep their values
            if "e" not in case:
                x.zero_()

    fresh()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.run(state)
    side.synchronize()  # the call's own stream: its results are there
    for name, x in got.items():
        assert torch.equal(x, before[name]), name
    fresh()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.run(state)
    graph.replay()
    torch.cuda.synchronize()
    for name, x in got.items():
        assert torch.equal(x, before[name]), name
    state["A"] = state["A"].clone()
    for name, x in ops.run(state).items():
        assert torch.equal(x, before[name]), name
    assert state["call"]["buffers"][0] is state["A"]


# ---------------------------------------------------------------- activations on a grid
# Relative error of an activation beside the output's rounding: the exponent of
# its exponential is a product of three factors, up to 126, rounded twice or
# three times (3 2^-24 126 ln 2 = 1.6e-5 of the value); Phi's tail adds its
# approximation's 5e-5; exponential, reciprocal and the rest add a few 2^-22.
# Together below 2^-13.  Exponentials and sigmoids below 2^-126 may be 0.
ACT_REL = 2.0 ** -13
TINY = 2.0 ** -125
_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def _grid(last):
    """Every bf16 value of magnitude 2^-20 to `last`, both signs."""
    top = int(oracle.f32_to_bf16_bits(np.array([last], np.float32))[0])
    up = np.arange(0x3580, top + 1, dtype=np.uint16)
    return np.concatenate([up, up | 0x8000])


def _gate(z, activation):
    """(gate, its derivative) of an activation z * gate(z), without cancellation."""
    if activation == "gelu":
        return 0.5 * _erfc(-z / math.sqrt(2)), np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    u, du = z, 1.0
    if activation == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        u, du = c * (z + 0.044715 * z ** 3), c * (1 + 3 * 0.044715 * z * z)
    e = np.exp(-np.abs(u))
    return np.where(u > 0, 1, e) / (1 + e), du * e / (1 + e) ** 2


@pytest.mark.parametrize("rows", [24, 4096])
@pytest.mark.parametrize("activation,last", [("gelu", 14.0), ("gelu_tanh", 9.0), ("silu", 100.0)])
def test_activations_are_relatively_accurate(activation, last, rows):
    """z = A B with one non-zero product, exact; z * gate(z) keeps its relative
    accuracy down the negative tail, where it is far below one."""
    bits_z = _grid(last)
    a = np.zeros((rows, 8), np.uint16)
    b = np.full((8, 256), 0x3F80, np.uint16)  # 1
    f = tk.kernels.linear(rows, 256, 8, activation=activation)
    for first in range(0, len(bits_z), rows):
        part = bits_z[first:first + rows]
        if rows < 100 and first // rows % 8:
            continue  # few rows go to another kernel; an eighth of the grid does
        a[:len(part), 0] = part
        out, pre = np.zeros((rows, 256), np.uint16), np.zeros((rows, 256), np.uint16)
        f(out, a, b, preact=pre)
        out, pre = out[:len(part)], pre[:len(part)]
        np.testing.assert_array_equal(pre, np.repeat(part[:, None], 256, 1))
        z = wide(part)
        gate, _ = _gate(z, activation)
        want = z * gate
        tol = (BF16 + ACT_REL) * np.abs(want) + TINY * np.abs(z)
        off = np.abs(wide(out) - want[:, None])
        worst = np.argmax(off.max(1) - tol)
        assert (off <= tol[:, None]).all(), f"z = {z[worst]}: {wide(out)[worst].max()}, not {want[worst]}"


@pytest.mark.parametrize("activation,last", [("gelu", 14.0), ("gelu_tanh", 9.0), ("silu", 100.0)])
def test_slopes_are_relatively_accurate(activation, last):
    """gate + z gate', each term to ACT_REL of itself (the sum passes zero).
    Where the gate is close to 1, 1 - gate is off by a rounding of 2^-24, which
    z and the inner derivative (at most 3 |z| + 3 for these z) multiply."""
    bits_z = _grid(last)
    m, n = 64, 256
    for first in range(0, len(bits_z), m * n):
        part = bits_z[first:first + m * n]
        pre = np.zeros(m * n, np.uint16)
        pre[:len(part)] = part
        dout = np.full((m, n), 0x3F80, np.uint16)
        dpre = np.zeros((m, n), np.uint16)
        tk.kernels.linear_backward(m, n, 8, activation=activation)(
            None, None, None, dout, None, None, pre.reshape(m, n), dpre)
        z = wide(part)
        gate, slope = _gate(z, activation)
        want = gate + z * slope
        got = wide(dpre).reshape(-1)[:len(part)]
        terms = gate + np.abs(z * slope)
        near_one = 0.0 if activation == "gelu" else 2.0 ** -23 * np.abs(z) * (3 * np.abs(z) + 3) * (gate > 0.5)
        tol = BF16 * np.abs(want) + 1.01 * (ACT_REL * terms + near_one + TINY * (3 * np.abs(z) + 3) ** 2)
        worst = np.argmax(np.abs(got - want) - tol)
        assert (np.abs(got - want) <= tol).all(), f"z = {z[worst]}: {got[worst]}, not {want[worst]} +- {tol[worst]}"


@pytest.mark.parametrize("activation", ["relu", "gelu", "gelu_tanh", "silu"])
def test_the_largest_values(activation):
    """From 2^8 to bf16's largest number an activation is z or 0 and its slope
    1 or 0 (the next terms are below e^-200): nothing overflows on the way."""
    up = np.arange(0x4380, 0x7F80, dtype=np.uint16)
    part = np.concatenate([up, up | 0x8000])
    z = wide(part)
    rows = len(part)
    a = np.zeros((rows, 8), np.uint16)
    a[:, 0] = part
    out = np.zeros((rows, 8), np.uint16)
    tk.kernels.linear(rows, 8, 8, activation=activation)(out, a, np.full((8, 8), 0x3F80, np.uint16))
    np.testing.assert_array_equal(wide(out), np.repeat(np.maximum(z, 0)[:, None], 8, 1))
    dout, dpre = np.full((rows, 8), 0x3F80, np.uint16), np.zeros((rows, 8), np.uint16)
    tk.kernels.linear_backward(rows, 8, 8, activation=activation)(
        None, None, None, dout, None, None, np.repeat(part[:, None], 8, 1), dpre)
    np.testing.assert_array_equal(wide(dpre), np.repeat((z > 0)[:, None].astype(np.float64), 8, 1))


def test_host_memory_is_not_wrapped():
    torch = pytest.importorskip("torch")
    host, pinned = np.zeros(64, np.uint16), rt.pinned_empty((64,), np.uint16)
    for x in (host, pinned):
        with pytest.raises(ValueError, match="not device memory"):
            rt.wrap_pointer(x.ctypes.data, x.shape, x.dtype)
    t = torch.arange(64, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    # into the middle of an allocation, and of the framework's own memory
    np.testing.assert_array_equal(rt.wrap_pointer(t[16:].data_ptr(), (48,), np.int32, owner=t).to_host(),
                                  np.arange(16, 64))
    d = rt.to_device(host)
    assert rt.wrap_pointer(d.ptr, (64,), np.uint16).ptr == d.ptr


def test_two_threads_with_streams_of_their_own():
    """Forward, backward and grouped calls of the same handles from two threads
    at once, each on its own stream and arrays, repeat the calls of one."""
    import threading

    t, n, k, e = 300, 264, 520, 3
    rng = np.random.default_rng(5)
    host = dict(a=bits(rng, t, k), b=bits(rng, k, n, std=0.05), w=bits(rng, e, k, n, std=0.05),
                dout=bits(rng, t, n, std=0.1), off=np.array([0, 100, 117, 290], np.int32))
    L = tk.kernels
    fwd, bwd = L.linear(t, n, k, activation="gelu"), L.linear_backward(t, n, k, activation="gelu")
    few = L.linear(7, n, k, activation="silu", static_weights=True)
    grp, grp_b = L.grouped_matmul(e, t, n, k), L.grouped_matmul_backward(e, t, n, k)

    def work(times, results):
        D = {name: rt.to_device(x) for name, x in host.items()}
        z, dz, out, gout = (rt.empty((t, n), np.uint16) for _ in range(4))
        small, x7 = rt.empty((7, n), np.uint16), rt.to_device(host["a"][:7])
        da, db, dw = rt.empty((t, k), np.uint16), rt.empty((k, n), np.uint16), rt.empty((e, k, n), np.uint16)
        dbias = rt.empty((n,), np.float32)
        gout.zero()
        s = rt.Stream()
        rt.synchronize()
        kw = dict(stream=s, sync=False)
        for _ in range(times):
            fwd(out, D["a"], D["b"], preact=z, **kw)
            few(small, x7, D["b"], **kw)
            bwd(da, db, dbias, D["dout"], D["a"], D["b"], z, dz, **kw)
            grp(gout, D["a"], D["w"], D["off"], **kw)
            grp_b(None, dw, D["dout"], D["a"], None, D["off"], **kw)
        s.synchronize()
        results.append([x.to_host(stream=s) for x in (out, z, small, da, db, dbias, dz, gout, dw)])

    want, got = [], []
    work(1, want)
    threads = [threading.Thread(target=work, args=(40, got)) for _ in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert len(got) == 2
    for result in got:
        for x, y in zip(result, want[0]):
            np.testing.assert_array_equal(x, y)


def test_a_first_call_that_is_captured():
    """In a process whose library has been used otherwise before, an operator's
    first call may be one that is captured: it allocates nothing."""
    import os
    import subprocess
    import sys

    pytest.importorskip("torch")
    code = """
import numpy as np, torch, thork_b200 as tk
rt = tk.runtime
rt.status_pointer()
A, B, O = (torch.randn(64, 64, device="cuda").bfloat16() for _ in range(3))
a, b, o = (rt.wrap_pointer(t.data_ptr(), (64, 64), np.uint16, owner=t) for t in (A, B, O))
f, graph = tk.kernels.linear(64, 64, 64), torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    f(o, a, b, stream=rt.Stream.from_handle(torch.cuda.current_stream().cuda_stream), sync=False)
O.zero_()
graph.replay()
torch.cuda.synchronize()
first = O.clone()
f(o, a, b)
assert torch.equal(first, O) and O.any() and rt.kernel_status() == 0
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
