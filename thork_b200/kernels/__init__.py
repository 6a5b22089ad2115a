"""thork_b200.kernels — pre-built kernels with launch geometry chosen for you
(reference ``src/thork/kernels/__init__.py``)::

    mm = tk.kernels.matmul(4096, 4096, 4096, dtype=tk.dt.bfloat16)
    mm(C, A, B)

    add = tk.kernels.matrix_add((1024, 1024))
    add(C, A, B)

    tm = tk.kernels.tile_matmul(4096, 4096, 4096, ncta=2)   # written in tk.kittens
    tm(C, A, B)

    up = tk.kernels.linear(4096, 14336, 4096, activation="gelu")
    up(H, X, W, bias=b, preact=Z)                            # H = gelu(X @ W + b)

    ex = tk.kernels.grouped_matmul(8, 4096, 14336, 4096)
    ex(Y, X, W, offsets)                                     # rows of group e times W[e]
"""

from .grouped import grouped_matmul, grouped_matmul_backward
from .linear import linear, linear_backward

from .matmul import matmul
from .matrix_add import matrix_add
from .tile_matmul import tile_matmul

__all__ = ["grouped_matmul", "grouped_matmul_backward", "linear", "linear_backward", "matmul",
           "matrix_add", "tile_matmul"]
