"""Sizes of the linear layer that between them reach every variant its launchers choose, and what tells one from another."""
import ctypes as C
import math
import random

from forward_amd import lib

# (m, n, k, operands on 16-byte boundaries, with an activation); the last seven are ordinary widths
SIZES = [(1, 1, 1, 0, 1), (20, 8, 8, 1, 0), (36, 8, 14, 1, 1), (1, 1, 12485, 0, 0), (20, 8, 13036, 1, 1),
         (33, 35, 6570, 1, 0), (2444, 10, 8, 1, 0), (9703, 1, 8, 1, 0), (40, 8672, 8, 1, 0), (38, 21, 10608, 1, 1),
         (974, 8, 1028, 0, 0), (33, 8381, 1, 1, 0), (38, 5058, 342, 1, 1), (2368, 2312, 8, 1, 1), (13962, 39, 198, 1, 0),
         (611, 2553, 1, 1, 1), (36, 2224, 1688, 0, 1), (1, 105, 19848, 1, 1), (77, 14126, 88, 1, 1), (136, 72, 12656, 1, 1),
         (18934, 2, 263, 0, 1), (198, 6634, 70, 1, 0), (82, 12360, 10, 1, 1), (13092, 10, 100, 1, 1), (58, 4794, 816, 1, 1),
         (6868, 102, 72, 1, 1), (3456, 8, 2234, 1, 1), (124, 36, 12584, 1, 1), (1028, 5414, 38, 1, 1),
         (2400, 8, 2728, 1, 0), (17520, 46, 8, 1, 1), (4, 2430, 3264, 1, 1), (4, 5592, 1464, 1, 1), (556, 54, 9040, 1, 1),
         (132, 410, 3522, 1, 0), (6098, 88, 78, 0, 1), (546, 40, 8602, 1, 0), (2188, 200, 396, 1, 0), (1830, 4338, 8, 1, 0),
         (2, 5378, 2054, 1, 1), (4456, 3336, 40, 1, 0), (35, 1, 1, 1, 1), (8333, 1, 1, 0, 0), (2318, 2326, 38, 0, 0),
         (65, 459, 17332, 1, 0), (19230, 10, 72, 1, 1), (110, 2786, 2964, 0, 0), (296, 54, 18098, 1, 0),
         (4, 320, 16400, 1, 1), (272, 8, 16904, 1, 1), (2719, 1, 2724, 1, 1), (104, 624, 7880, 1, 0),
         (1048, 228, 4171, 0, 0), (336, 17376, 12, 1, 1), (304, 20, 16960, 1, 0), (66, 4178, 6298, 1, 1),
         (4, 6574, 2288, 1, 1), (2736, 2808, 120, 1, 0), (104, 2973, 4112, 1, 0), (3460, 2836, 200, 1, 1),
         (3980, 6368, 132, 1, 0), (92, 4436, 5744, 1, 1), (6408, 4480, 80, 1, 0), (6648, 132, 1268, 1, 1),
         (7398, 146, 1056, 1, 1), (18046, 144, 432, 1, 0), (4488, 6952, 80, 1, 0), (7845, 2, 9658, 1, 0),
         (400, 4886, 2784, 1, 0), (8248, 40, 6464, 1, 1), (74, 11216, 6624, 1, 1), (46, 8588, 6452, 1, 1),
         (68, 10916, 9092, 1, 0), (144, 5652, 4628, 1, 1), (11240, 140, 5652, 1, 1), (10952, 168, 5584, 1, 1),
         (76, 8996, 8432, 1, 1), (132, 4396, 11992, 1, 1), (10888, 4472, 148, 1, 1), (6537, 10925, 144, 1, 1),
         (4547, 320, 1216, 1, 0), (6921, 3920, 384, 1, 1), (5196, 2376, 1536, 1, 0), (1465, 2400, 192, 1, 1),
         (2048, 1024, 1024, 1, 1), (384, 1024, 4096, 1, 0), (512, 768, 768, 0, 1)]


def plan(m, n, k, what, act, dtype, on_boundary):
    p = lib.LinearPlan()
    lib.check(lib.dll.fwdmi_linear_plan(m, n, k, what, act, dtype, on_boundary, C.byref(p)))
    return p


def variants(m, n, k, on_boundary, act):
    """The variants that y, dx, dw and both gradients together take in fp32 and in the 16-bit types (which plan alike)."""
    found = set()
    for dtype in (lib.F32, lib.F16):
        for what in range(4):
            p = plan(m, n, k, what, lib.ACT_GELU if act else lib.ACT_NONE, dtype, on_boundary)
            if p.tile_rows:
                found.add((what, dtype, p.tile, p.tile_rows, p.tile_columns, p.splits > 1, p.direct, p.end))
    return found


def drawn(count, seed):
    """Sizes from 1 to 20000 along each axis, even over their logarithm, of every divisibility."""
    rng = random.Random(seed)
    while count:
        step = rng.choice([1, 2, 4, 8, 64])
        m, n, k = (max(step, int(math.exp(rng.uniform(0, math.log(20000)))) // step * step) for _ in range(3))
        if m * n * k <= 6e10:
            count -= 1
            yield m, n, k, int(rng.random() < 0.7), rng.choice([0, 1])
