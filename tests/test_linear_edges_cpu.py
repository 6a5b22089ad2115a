"""CPU: what the linear-layer operators refuse, and what their host side does
when a call fails."""

import ctypes

import numpy as np
import pytest

import linear_choices as C
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


# ---------------------------------------------------------------- the host side of a call
class _Fake:
    """The runtime under a call, without a device: a stream, buffers and
    copies that record what happens in order."""

    def __init__(self, monkeypatch, status=0):
        self.log, self.status, self.allocated = [], status, 0
        fake = self

        class Buffer:
            def __init__(self, nbytes):
                fake.allocated += 1
                self.ptr, self.nbytes, self._dev = 4096 * fake.allocated, nbytes, 0

            def free(self):
                fake.log.append("free")
                self.ptr = 0

        class Stream:
            handle = 4096

            def synchronize(self):
                fake.log.append("synchronize")

        def read(ref, *_):
            ref._obj.value = fake.status
            return 0

        def stream_status(ref, handle):
            fake.log.append("synchronize")
            return read(ref)

        def kernel_status(ref, clear):
            read(ref)
            if clear:
                fake.status = 0
            return 0

        self.Buffer, self.stream = Buffer, Stream()
        monkeypatch.setattr(rt, "get_device", lambda: 0)
        monkeypatch.setattr(rt, "DeviceBuffer", Buffer)
        monkeypatch.setattr(rt, "copy_htod", lambda *a, **k: self.log.append("in"))
        monkeypatch.setattr(rt, "copy_dtoh", lambda *a, **k: self.log.append("out"))
        for name, f in (("thork_stream_status", stream_status), ("thork_kernel_status", kernel_status)):
            monkeypatch.setattr(rt.lib(), name, f, raising=False)

    def kernel(self, monkeypatch, name, rc=0):
        def launch(*args):
            self.log.append("launch")
            return rc
        monkeypatch.setattr(rt.lib(), name, launch, raising=False)

    def array(self, *shape):
        d = rt.DeviceArray(shape, np.uint16, buffer=self.Buffer(2 * int(np.prod(shape))))
        return d


def test_an_expired_wait_is_raised_by_calls_that_synchronise(monkeypatch):
    expired = 1 | 0x53 << 8
    fake = _Fake(monkeypatch, expired)
    fake.kernel(monkeypatch, "thork_linear_bf16")
    f = K.linear(4, 64, 64)
    out, a, b = fake.array(4, 64), fake.array(4, 64), fake.array(64, 64)
    f(out, a, b, stream=fake.stream, sync=False)  # an asynchronous call reads nothing
    assert fake.log == ["launch"] and fake.status == expired
    with pytest.raises(rt.CudaError, match="bounded wait expired at site 83") as e:
        f(out, a, b, stream=fake.stream)
    assert e.value.code == rt.ERR_KERNEL and fake.status == 0  # raised once
    f(out, a, b, stream=fake.stream)
    # another thread's call that cleared the word in between
    fake.status = expired
    monkeypatch.setattr(rt, "kernel_status", lambda clear=True: 0)
    with pytest.raises(rt.CudaError, match="bounded wait expired at site 83"):
        f(out, a, b, stream=fake.stream)
    # host arrays: the call synchronises in any case
    host = np.zeros((4, 64), np.uint16)
    with pytest.raises(rt.CudaError, match="bounded wait"):
        f(host, a, b, stream=fake.stream, sync=False)


def test_wrong_offsets_stay_in_the_status_word(monkeypatch):
    bad_offsets = 2 | 0x40 << 8
    fake = _Fake(monkeypatch, bad_offsets)
    fake.kernel(monkeypatch, "thork_grouped_gemm_bf16")
    x, w = np.zeros((4, 64), np.uint16), np.zeros((2, 64, 64), np.uint16)
    K.grouped_matmul(2, 4, 64, 64)(x.copy(), x, w, np.array([0, 9, 4], np.int32), stream=fake.stream)
    assert fake.status == bad_offsets


def test_a_gathered_result_is_an_operand(monkeypatch):
    """The arrays that a fused gather returns borrow its slots; they feed a
    linear layer like any other array of the device."""
    from thork_b200.dist import _View
    fake = _Fake(monkeypatch)
    fake.kernel(monkeypatch, "thork_linear_bf16")
    gathered = rt.DeviceArray((4, 64), np.uint16, buffer=_View(1 << 20, 512))
    f = K.linear(4, 64, 64)
    f(fake.array(4, 64), gathered, fake.array(64, 64), stream=fake.stream)
    assert fake.log == ["launch", "synchronize"]
    f._operands[1].check(gathered, 0)
    with pytest.raises(ValueError, match="device 0"):
        f._operands[1].check(gathered, 1)


def _call_linear(fake, **kw):
    host = [np.zeros(s, np.uint8) for s in ((4, 64), (64, 64))]
    K.linear(4, 64, 64, tk.dt.float8_e4m3)(np.zeros((4, 64), np.uint16), *host, stream=fake.stream, **kw)


def test_a_call_that_fails_waits_for_its_copies_before_it_frees(monkeypatch):
    """Copies of host arrays are queued before the launch is refused: their
    buffers go back to the pool only when the stream has finished."""
    fake = _Fake(monkeypatch)
    fake.kernel(monkeypatch, "thork_linear_e4m3", rc=rt.ERR_INVALID)
    with pytest.raises(rt.CudaError):
        _call_linear(fake)
    assert fake.log == ["in", "in", "launch", "synchronize", "free", "free", "free"]

    fake.log.clear()

    def raises(*args):
        raise TypeError("scale_a")

    monkeypatch.setattr(rt.lib(), "thork_linear_e4m3", raises, raising=False)
    with pytest.raises(TypeError):
        _call_linear(fake, scale_a="one")
    assert fake.log == ["in", "in", "synchronize", "free", "free", "free"]


def test_an_operand_refused_after_others_were_copied_waits_too(monkeypatch):
    fake = _Fake(monkeypatch)
    fake.kernel(monkeypatch, "thork_linear_bf16")
    x, w = np.zeros((4, 64), np.uint16), np.zeros((64, 63), np.uint16)
    with pytest.raises(ValueError):
        K.linear(4, 64, 64)(x.copy(), x, w, stream=fake.stream)
    assert fake.log == ["in", "synchronize", "free", "free"]


def test_only_memory_of_the_current_device_is_wrapped(monkeypatch):
    where = {4096: 0, 8192: 1, 12288: -1}

    def pointer_device(ptr, ref):
        ref._obj.value = where[ptr]
        return 0

    monkeypatch.setattr(rt, "get_device", lambda: 0)
    monkeypatch.setattr(rt.lib(), "thork_pointer_device", pointer_device, raising=False)
    owner = object()
    a = rt.wrap_pointer(4096, (4, 64), np.uint16, owner=owner)
    assert (a.ptr, a.shape, a.nbytes, a.buffer._dev) == (4096, (4, 64), 512, 0)
    with pytest.raises(ValueError, match="memory of device 1"):
        rt.wrap_pointer(8192, (4, 64), np.uint16)
    with pytest.raises(ValueError, match="not device memory"):
        rt.wrap_pointer(12288, (4, 64), np.uint16)
    assert rt.wrap_pointer(0, (0, 64), np.uint16).size == 0
    monkeypatch.setattr(rt, "get_device", lambda: 1)
    assert rt.wrap_pointer(8192, (4, 64), np.uint16).buffer._dev == 1


def test_host_outputs_are_writeable_and_apart(monkeypatch):
    fake = _Fake(monkeypatch)
    fake.kernel(monkeypatch, "thork_linear_bf16")
    x, w, out = (np.zeros(s, np.uint16) for s in ((4, 64), (64, 64), (8, 64)))
    f = K.linear(4, 64, 64)
    frozen = np.frombuffer(bytes(4 * 64 * 2), np.uint16).reshape(4, 64)
    with pytest.raises(ValueError, match="'out' is written, but the array is read-only"):
        f(frozen, x, w, stream=fake.stream)
    f(out[:4], frozen, w, residual=frozen, stream=fake.stream)  # inputs may be read-only
    with pytest.raises(ValueError, match="'preact' shares memory with another output"):
        f(out[:4], x, w, preact=out[:4], stream=fake.stream)
    with pytest.raises(ValueError, match="'preact' shares memory"):
        f(out[:4], x, w, preact=out[2:6], stream=fake.stream)
    f(out[:4], x, w, preact=out[4:], residual=out[:4], stream=fake.stream)  # in place, and a neighbour


# ---------------------------------------------------------------- the choice of kernel
def _near(values, step):
    return sorted({max(step, int(v) // step * step) for v in values})


@pytest.mark.parametrize("form", range(5))
def test_every_choice_of_kernel_is_among_the_tested_shapes(form):
    """Over a grid of sizes the rules choose no kernel, tile height or split
    that the GPU tests' shapes do not reach as well."""
    tested = {
        C.BF16: C.FULL + C.PRODUCT, C.E4M3: C.FULL + C.PRODUCT_E4M3, C.GRADIENT: C.WEIGHTS,
        C.GROUPED_BF16: C.GROUPS, C.GROUPED_E4M3: C.GROUPS_E4M3}[form]
    step = 16 if form in (C.E4M3, C.GROUPED_E4M3) else 8
    if form >= C.GROUPED_BF16:
        covered = {C.choice(form, t, n, k, e) for e, t, n, k in tested}
        reached = {C.choice(form, t, n, k, e) for e in (1, 2, 3, 8, 24, 64, 256, 1024)
                   for t in (1, 2, 3, 7, 15, 30, 64, 100, 200, 500, 513, 8192)
                   for n in (16, 128, 1000 // step * step, 4096) for k in (16, 320, 512, 1024, 2048, 14336)}
    else:
        covered = {C.choice(form, *s) for s in tested}
        sizes = _near([8, 72, 136, 264, 400, 520, 656, 784, 1024, 1544, 2048, 2800, 4096, 5504, 8192, 14336], step)
        rows = [1, 9, 16, 17, 32, 33, 50, 64, 65, 96, 128, 129, 200, 256, 400, 600, 800, 1200, 2000, 4096, 8192, 65536]
        reached = {C.choice(form, m, n, k) for m in rows for n in sizes for k in sizes}
    assert reached <= covered, reached - covered
    assert len(reached) >= {C.BF16: 12, C.E4M3: 12, C.GRADIENT: 6}.get(form, 9)


def test_the_choice_refuses_bad_sizes():
    L = rt.lib()
    x, y = ctypes.c_int(), ctypes.c_int()
    for args in ((5, 4, 64, 64, 1, 148), (0, 0, 64, 64, 1, 148), (0, 4, 60, 64, 1, 148), (0, 4, 64, 64, 0, 148),
                 (0, 4, 64, 64, 1, 1)):
        assert L.thork_linear_choice(*args, ctypes.byref(x), ctypes.byref(y)) == rt.ERR_INVALID
    assert L.thork_linear_choice(0, 4, 64, 64, 1, 148, None, ctypes.byref(y)) == rt.ERR_INVALID
