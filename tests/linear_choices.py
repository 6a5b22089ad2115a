"""Shapes that between them reach every kernel and split that the linear-layer
operators choose from (on B200's 148 SMs), most of them odd to the tiles.

The choice is the library's own (``thork_linear_choice``); that no choice is
left out is tested on the CPU, the results on the GPU."""

import ctypes

from thork_b200 import runtime as rt

BF16, E4M3, GRADIENT, GROUPED_BF16, GROUPED_E4M3 = range(5)
SMS = 148


def choice(form, m, n, k, e=1):
    """(rows a tile, split) of swap_kernel; (0, 0) for the kernels of many rows."""
    tile, split = ctypes.c_int(-1), ctypes.c_int(-1)
    rt.check(rt.lib().thork_linear_choice(form, m, n, k, e, SMS, ctypes.byref(tile), ctypes.byref(split)))
    return tile.value, split.value


# served batches of full-size layers, around every tile height
FULL = [(m, 4096, 4096) for m in (1, 16, 31, 63, 64, 65, 100, 128, 129, 200, 256, 257)]
FULL += [(96, 4096, 14336), (512, 512, 8192)]

PRODUCT = [(1, 32, 8), (1, 32, 136), (17, 32, 200), (1, 32, 392), (17, 32, 392), (1, 32, 904), (17, 32, 944),
           (17, 5640, 200), (973, 144, 552), (18, 2888, 424), (549, 144, 392), (17, 1360, 920), (660, 32, 928),
           (746, 672, 1512), (33, 3576, 392), (710, 264, 912), (34, 1856, 944), (884, 144, 1360), (65, 4048, 920),
           (713, 648, 2024), (67, 2320, 1416), (963, 272, 3344), (300, 520, 72), (1100, 4136, 136)]

PRODUCT_E4M3 = [(1, 32, 16), (1, 32, 272), (18, 32, 416), (1, 32, 784), (17, 32, 784), (1, 32, 1808), (17, 32, 1808),
                (17, 5488, 400), (993, 144, 1040), (19, 2960, 784), (1089, 32, 800), (17, 1392, 1936),
                (683, 32, 1808), (1412, 272, 3248), (35, 3696, 784), (943, 272, 1440), (34, 1936, 1840),
                (875, 144, 2592), (70, 4592, 1888), (2305, 144, 3856), (65, 2288, 2832), (1126, 272, 5792),
                (300, 528, 80), (1100, 4112, 144)]

# rows summed over, columns, rows of the gradient
WEIGHTS = [(193, 32, 8), (1498, 392, 1128), (387, 32, 8), (654, 32, 72), (897, 32, 8), (926, 32, 72),
           (947, 4144, 72), (1933, 136, 2232), (982, 2320, 72), (2346, 280, 1352), (100, 520, 1032), (3001, 2312, 1288)]

# groups, rows of the buffer, columns, contraction
GROUPS = [(3, 2, 32, 8), (3, 10, 32, 208), (3, 5, 32, 472), (3, 5, 32, 976), (3, 72, 32, 8), (3, 62, 32, 200),
          (3, 19, 32, 496), (3, 27, 32, 1048), (3, 300, 264, 200)]
GROUPS_E4M3 = [(3, 1, 32, 16), (3, 11, 32, 400), (3, 7, 32, 912), (3, 5, 32, 1952), (3, 16, 32, 16), (3, 49, 32, 416),
               (3, 71, 32, 912), (3, 20, 32, 1968), (3, 300, 272, 400)]
