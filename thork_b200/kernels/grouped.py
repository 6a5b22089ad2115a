"""``tk.kernels.grouped_matmul`` and ``tk.kernels.grouped_matmul_backward``:
matrix products grouped by expert, with group sizes that only the device
knows, and their gradients.

No reference counterpart (see ``linear``).  The rows of ``A`` are sorted by
expert; ``offsets`` (int32, ``E + 1`` values, on the device or a NumPy array)
says where each expert's rows begin, so nothing about the sizes is read back
to the host and a call can be captured into a graph that later sizes reuse.
"""

from .. import dtypes as dt
from .. import runtime as rt
from ._library import Operand, run_operands
from .linear import MAX_CONTRACTION, activation_code, check_contraction, check_preact, check_sizes

MAX_GROUPS = 1024


def _check(what: str, dtype: dt.Dtype, E: int, T: int, N: int, K: int) -> None:
    check_sizes(what, dtype, N, K, E=E, T=T)
    if E > MAX_GROUPS:
        raise ValueError(f"{what}: E={E} must be at most {MAX_GROUPS}")


class grouped_matmul:
    """``k(out, A, B, offsets, preact=None)``: for every expert ``e``, with
    ``r = offsets[e] .. offsets[e + 1]``,

        z[r] = A[r] @ B[e];  out[r] = act(z[r])

    for ``A[T, K]``, ``B[E, K, N]`` and ``out[T, N]``.  Experts may be empty,
    and rows outside every group (behind the last, or before the first) are
    left as they were in ``out`` and ``preact``.  ``offsets`` do not decrease
    and lie in ``[0, T]``; others are clamped so that nothing outside the
    arrays is touched, and recorded in ``tk.runtime.kernel_status()``.

    With ``dtype=tk.dt.float8_e4m3`` the call takes ``scale_a`` (a number) and
    ``scale_b`` (float32 ``[E]``, one per expert, or ``None`` for ones):
    ``z[r] = scale_a * scale_b[e] * (A[r] @ B[e])``.  ``activation`` and
    ``preact`` are as for ``tk.kernels.linear``.  K is at most 2^23.

    ``static_weights`` may be given as to ``tk.kernels.linear`` and changes
    nothing: which expert's weights a tile needs is known only when the
    previous kernel, which may write ``offsets``, has finished.
    """

    name = "grouped_matmul"

    def __init__(self, E: int, T: int, N: int, K: int, dtype: dt.Dtype = dt.bfloat16,
                 activation: str = "none", static_weights: bool = False):
        E, T, N, K = int(E), int(T), int(N), int(K)
        _check("grouped_matmul", dtype, E, T, N, K)
        check_contraction("grouped_matmul", "K", K)
        self._fp8 = dtype == dt.float8_e4m3
        self._sizes = (E, T, N, K)
        self._act = (activation_code(activation, "grouped_matmul"), int(bool(static_weights)))
        self._operands = (
            Operand("out", dt.bfloat16, (T, N), written=True, partly=True), Operand("A", dtype, (T, K)),
            Operand("B", dtype, (E, K, N)), Operand("offsets", dt.int32, (E + 1,)),
            Operand("preact", dt.bfloat16, (T, N), written=True, partly=True),
            Operand("scale_b", dt.float32, (E,)))

    def __call__(self, out, A, B, offsets, preact=None, scale_a: float = 1.0, scale_b=None, stream=None,
                 sync: bool = True) -> None:
        if out is None or A is None or B is None or offsets is None:
            raise TypeError("grouped_matmul: out, A, B and offsets are required")
        if not self._fp8 and (scale_a != 1.0 or scale_b is not None):
            raise ValueError("grouped_matmul: scale_a and scale_b go with float8_e4m3 operands")
        L = rt.lib()

        def launch(p, s):
            if self._fp8:
                return L.thork_grouped_gemm_e4m3(p[1], p[2], p[0], p[3], p[4], *self._sizes, scale_a, p[5],
                                                 *self._act, s)
            return L.thork_grouped_gemm_bf16(p[1], p[2], p[0], p[3], p[4], *self._sizes, *self._act, s)

        run_operands(self._operands, (out, A, B, offsets, preact, scale_b), launch, self.name, stream, sync)


class grouped_matmul_backward:
    """``k(dA, dB, dout, A, B, offsets, preact=None, dpre=None)``: the gradients
    of ``tk.kernels.grouped_matmul`` (bf16): on each group's rows ``r``

        dpre[r] = dout[r] * act'(preact[r])
        dA[r] = dpre[r] @ B[e]^T;  dB[e] = A[r]^T @ dpre[r]

    ``dB[E, K, N]`` is written whole (zeros for an empty expert); rows outside
    every group are left as they were in ``dA`` and ``dpre``.  ``dA`` or ``dB``
    may be ``None``; ``preact`` and ``dpre`` are as for
    ``tk.kernels.linear_backward``.  N is at most 2^23 for ``dA``, T for ``dB``.
    """

    name = "grouped_matmul_backward"

    def __init__(self, E: int, T: int, N: int, K: int, dtype: dt.Dtype = dt.bfloat16,
                 activation: str = "none"):
        E, T, N, K = int(E), int(T), int(N), int(K)
        _check("grouped_matmul_backward", dtype, E, T, N, K)
        if dtype != dt.bfloat16:
            raise TypeError(f"grouped_matmul_backward: unsupported dtype {dtype!r}")
        self._tail = (E, T, N, K, activation_code(activation, "grouped_matmul_backward"))
        self._bent = activation != "none"
        b16 = dt.bfloat16
        self._operands = (
            Operand("dA", b16, (T, K), written=True, partly=True),
            Operand("dB", b16, (E, K, N), written=True), Operand("dout", b16, (T, N)),
            Operand("A", b16, (T, K)), Operand("B", b16, (E, K, N)),
            Operand("offsets", dt.int32, (E + 1,)), Operand("preact", b16, (T, N)),
            Operand("dpre", b16, (T, N), written=True, partly=True))

    def __call__(self, dA, dB, dout, A, B, offsets, preact=None, dpre=None, stream=None,
                 sync: bool = True) -> None:
        check_preact(self.name, self._bent, preact, dpre)
        if dout is None or offsets is None or (dB is not None and A is None) or (dA is not None and B is None):
            raise TypeError("grouped_matmul_backward: dout and offsets are required, A for dB and B for dA")
        T, N = self._tail[1:3]
        if T > MAX_CONTRACTION and dB is not None:
            check_contraction(self.name, "T", T)
        if N > MAX_CONTRACTION and dA is not None:
            check_contraction(self.name, "N", N)
        fn = rt.lib().thork_grouped_gemm_backward_bf16
        run_operands(self._operands, (dA, dB, dout, A, B, offsets, preact, dpre),
                     lambda p, s: fn(*p, *self._tail, s), self.name, stream, sync)
