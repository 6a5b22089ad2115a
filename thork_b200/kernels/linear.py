"""``tk.kernels.linear`` and ``tk.kernels.linear_backward``: a linear layer with
its bias, activation and residual in the product's epilogue, and its gradients.

No reference counterpart: the reference's pre-built product is the plain
``src/thork/kernels/matmul.py:17-71``.  Layouts, types and calls follow
``tk.kernels.matmul``: row-major ``A[M, K]`` and ``B[K, N]``, bf16 or float8
e4m3 operands, fp32 sums, bf16 outputs, NumPy arrays (copied in and back) or
DeviceArrays (used in place, with ``stream=`` and ``sync=False`` for
asynchronous calls).
"""

from .. import dtypes as dt
from .. import runtime as rt
from ._library import Operand, run_operands

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def activation_code(activation: str, what: str) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"{what}: unknown activation {activation!r}; one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[activation]


# what a product may sum over: an epilogue's bounded wait spans its tile's whole
# contraction (csrc/linear.cu, kMaxContraction)
MAX_CONTRACTION = 1 << 23


def check_contraction(what: str, name: str, size: int) -> None:
    if size > MAX_CONTRACTION:
        raise ValueError(f"{what}: a contraction over {name}={size} is more than 2^23")


def check_sizes(what: str, dtype: dt.Dtype, N: int, K: int, **positive) -> None:
    for name, v in {**positive, "N": N, "K": K}.items():
        if not 0 < v <= 1 << 30:
            raise ValueError(f"{what}: {name}={v} must be positive and at most 2^30")
    align = {dt.bfloat16: 8, dt.float8_e4m3: 16}.get(dtype)
    if align is None:
        raise TypeError(f"{what}: unsupported dtype {dtype!r}")
    if N % align or K % align:
        raise ValueError(f"{what}({dtype.name}): K and N must be multiples of {align}; got N={N}, K={K}")


class linear:
    """``k(out, A, B, bias=None, residual=None, preact=None)`` for

        z = A[M, K] @ B[K, N] + bias[N];  out[M, N] = act(z) + residual[M, N]

    ``activation``: ``"none"``, ``"relu"``, ``"gelu"`` (through erf),
    ``"gelu_tanh"`` or ``"silu"``.  ``preact``, when given, receives ``z`` in
    bf16 for ``linear_backward``.  ``out`` may be the residual itself.  With
    ``dtype=tk.dt.float8_e4m3`` the call takes ``scale_a`` and ``scale_b`` and
    ``z = scale_a * scale_b * (A @ B) + bias``; everything but A and B stays
    bf16.  K and N are multiples of 8 (e4m3: 16), M is any positive number; K
    is at most 2^23.

    ``static_weights``: B is written by no earlier kernel on the stream
    (decode weights), so that a product of few rows may start fetching it
    before the previous kernel has finished.
    """

    name = "linear"

    def __init__(self, M: int, N: int, K: int, dtype: dt.Dtype = dt.bfloat16,
                 activation: str = "none", static_weights: bool = False):
        M, N, K = int(M), int(N), int(K)
        check_sizes("linear", dtype, N, K, M=M)
        check_contraction("linear", "K", K)
        act, flags = activation_code(activation, "linear"), int(bool(static_weights))
        self._fp8 = dtype == dt.float8_e4m3
        self._operands = (
            Operand("out", dt.bfloat16, (M, N), written=True), Operand("A", dtype, (M, K)),
            Operand("B", dtype, (K, N)), Operand("bias", dt.bfloat16, (N,)),
            Operand("residual", dt.bfloat16, (M, N)),
            Operand("preact", dt.bfloat16, (M, N), written=True))
        self._tail = (M, N, K)
        self._act = (act, flags)

    def __call__(self, out, A, B, bias=None, residual=None, preact=None, scale_a: float = 1.0,
                 scale_b: float = 1.0, stream=None, sync: bool = True) -> None:
        if out is None or A is None or B is None:
            raise TypeError("linear: out, A and B are required")
        if self._fp8:
            fn, scales = rt.lib().thork_linear_e4m3, (scale_a, scale_b)
        else:
            if scale_a != 1.0 or scale_b != 1.0:
                raise ValueError("linear: scale_a and scale_b go with float8_e4m3 operands")
            fn, scales = rt.lib().thork_linear_bf16, ()

        def launch(p, s):
            return fn(p[1], p[2], p[0], p[3], p[4], p[5], *self._tail, *scales, *self._act, s)

        run_operands(self._operands, (out, A, B, bias, residual, preact), launch, self.name, stream, sync)


class linear_backward:
    """``k(dA, dB, dbias, dout, A, B, preact=None, dpre=None)``: the gradients
    of ``tk.kernels.linear`` (bf16) from ``dout[M, N]``,

        dpre = dout * act'(preact);  dbias[N] = sum over rows of dpre
        dA[M, K] = dpre @ B^T;       dB[K, N] = A^T @ dpre

    ``dout`` is also the residual's gradient.  Any of ``dA``, ``dB`` and
    ``dbias`` may be ``None`` and is then not computed.  With an activation
    the call needs ``preact`` as the forward pass left it and ``dpre``, an
    [M, N] output that the two products read; without one ``dpre`` is ``dout``
    and both stay ``None``.  ``dbias`` is float32 (its sum is taken before
    ``dpre`` is rounded), the other outputs are bf16.  N is at most 2^23 for
    ``dA``, M for ``dB``.
    """

    name = "linear_backward"

    def __init__(self, M: int, N: int, K: int, dtype: dt.Dtype = dt.bfloat16, activation: str = "none"):
        M, N, K = int(M), int(N), int(K)
        check_sizes("linear_backward", dtype, N, K, M=M)
        if dtype != dt.bfloat16:
            raise TypeError(f"linear_backward: unsupported dtype {dtype!r}")
        self._tail = (M, N, K, activation_code(activation, "linear_backward"))
        self._bent = activation != "none"
        b16 = dt.bfloat16
        self._operands = (
            Operand("dA", b16, (M, K), written=True), Operand("dB", b16, (K, N), written=True),
            Operand("dbias", dt.float32, (N,), written=True), Operand("dout", b16, (M, N)),
            Operand("A", b16, (M, K)), Operand("B", b16, (K, N)), Operand("preact", b16, (M, N)),
            Operand("dpre", b16, (M, N), written=True))

    def __call__(self, dA, dB, dbias, dout, A, B, preact=None, dpre=None, stream=None,
                 sync: bool = True) -> None:
        check_preact(self.name, self._bent, preact, dpre)
        if dout is None or (dB is not None and A is None) or (dA is not None and B is None):
            raise TypeError("linear_backward: dout is required, A for dB and B for dA")
        M, N = self._tail[:2]
        if M > MAX_CONTRACTION and dB is not None:
            check_contraction(self.name, "M", M)
        if N > MAX_CONTRACTION and dA is not None:
            check_contraction(self.name, "N", N)
        fn = rt.lib().thork_linear_backward_bf16
        run_operands(self._operands, (dA, dB, dbias, dout, A, B, preact, dpre),
                     lambda p, s: fn(*p, *self._tail, s), self.name, stream, sync)


def check_preact(what: str, bent: bool, preact, dpre) -> None:
    if bent and (preact is None or dpre is None):
        raise ValueError(f"{what}: an activation needs preact and dpre")
    if not bent and (preact is not None or dpre is not None):
        raise ValueError(f"{what}: preact and dpre go with an activation")
