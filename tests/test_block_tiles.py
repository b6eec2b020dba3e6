"""Every way that the tiles' products run: five launches (the gate, its backward, y, dx, the three weight gradients), tiles of
256, 128 and 64 with two and with four LDS buffers, sums of 1, 2, an odd and an even count of steps, and sums split over 2 to
16 and over 32 and more workgroups. The sizes are odd ones for which the library chooses these; a test without a GPU reads its
choices, so that another rule cannot leave a way untested."""
import ctypes as ct

import pytest
import torch

# (rows, in, hidden, out)
FLOAT32 = [(20, 16, 32, 20), (17, 36, 33, 18), (22, 17, 69, 20), (22, 22, 100, 16), (18, 653, 1155, 296), (429, 22, 35, 37),
           (34, 18, 34, 21), (71, 18, 33, 18), (22, 18, 39, 67), (17, 100, 45, 19), (111, 18, 35, 22), (4101, 20, 1225, 97),
           (20, 25, 4306, 1144), (849, 65, 4805, 16), (1199, 33, 5229, 20), (4079, 19, 422, 23), (2021, 1099, 65, 792),
           (15180, 458, 149, 715), (1565, 20, 7600, 99), (65, 3331, 1370, 19), (34, 1102, 872, 55), (4078, 19, 34, 17),
           (847, 33, 1242, 17), (1116, 22, 35, 1859), (1445, 111, 32, 1438), (131, 1907, 7452, 41), (65, 603, 1356, 218),
           (1667, 1220, 33, 18), (1233, 35, 65, 1635), (2345, 892, 32, 29), (98, 970, 977, 28), (2940, 17, 727, 35),
           (33, 1811, 1316, 134), (1122, 18, 97, 1861), (2818, 22, 33, 1806), (1540, 32, 32, 3317), (1645, 33, 1620, 21),
           (18, 2139, 2707, 41), (1072, 17, 1974, 103), (3305, 1555, 32, 23), (3582, 1448, 33, 29), (1834, 1106, 101, 43),
           (2702, 69, 977, 18), (2005, 16, 2745, 38), (33, 1571, 3698, 30), (4249, 43, 32, 2819), (100, 1148, 2117, 93),
           (4248, 26, 33, 2854), (8175, 324, 70, 27), (2012, 46, 97, 2575), (1755, 100, 1499, 16), (1327, 19, 3862, 68),
           (65, 40, 2696, 3528), (3135, 16, 3988, 19), (3557, 3480, 33, 49), (5571, 2302, 32, 16), (4909, 36, 66, 2605),
           (3207, 18, 3990, 34), (3597, 67, 1810, 18), (1481, 3430, 102, 19), (97, 2240, 2566, 25), (4954, 60, 100, 2448),
           (1866, 98, 3439, 16), (2594, 19, 4721, 72), (2716, 4354, 65, 17), (3924, 3183, 97, 53), (136, 3426, 3256, 44),
           (3312, 3433, 133, 64), (138, 339, 7160, 3630), (2047, 1031, 2049, 1023)]
SIXTEEN = [(20, 21, 32, 21), (18, 17, 70, 25), (22, 25, 132, 19), (18, 17, 199, 19), (76, 26, 39, 130), (17, 2460, 1575, 85),
           (31, 68, 33, 16), (18, 21, 41, 193), (25, 197, 41, 30), (129, 16, 54, 137), (193, 26, 32, 131), (653, 130, 5880, 31),
           (21, 1139, 8145, 45), (1676, 26, 66, 1195), (4867, 130, 592, 23), (2301, 18, 921, 130), (17, 19, 8251, 1260),
           (72, 1121, 8593, 17), (10768, 1116, 129, 398), (668, 204, 5575, 21), (9515, 198, 74, 29), (17, 848, 1107, 40),
           (4641, 143, 65, 1702), (2992, 17, 1355, 136), (9662, 443, 65, 173), (135, 269, 8626, 174), (1198, 38, 32, 1681),
           (70, 20, 5874, 2168), (65, 1055, 834, 170), (2278, 29, 33, 1457), (2231, 917, 33, 18), (599, 16, 1715, 129),
           (2710, 1103, 33, 24), (8518, 29, 32, 168), (2450, 19, 68, 1296), (668, 70, 1502, 143), (18, 53, 4370, 2089),
           (450, 17, 135, 4100), (198, 262, 3005, 34), (2668, 32, 33, 3101), (13619, 527, 197, 100), (1047, 33, 194, 1953),
           (323, 73, 4486, 133), (650, 18, 3108, 193), (719, 2738, 131, 95), (195, 1251, 1145, 131), (2446, 3289, 33, 170),
           (890, 29, 200, 3481), (1142, 129, 1954, 65), (2140, 20, 1481, 200), (899, 2181, 205, 27), (1905, 1603, 130, 39),
           (3366, 2317, 65, 107), (4423, 18, 130, 1809), (1032, 75, 3585, 154), (2618, 1173, 193, 21), (214, 24, 7216, 807),
           (4211, 17, 2045, 145), (2588, 21, 193, 3116), (2670, 17, 3114, 199), (9771, 131, 791, 18), (6797, 132, 1236, 65),
           (129, 2848, 5614, 52), (139, 46, 6465, 5846), (2047, 1031, 4097, 1023)]
MORE_BUFFERS = 512   # workgroups of 64 x 64 tiles that take four LDS buffers


class Tile(ct.Structure):
    _fields_ = [("side", ct.c_int), ("splits", ct.c_int)]


class Layout(ct.Structure):
    _fields_ = ([(n, ct.c_int64) for n in ("ldx", "ldh", "ldy")] +
                [(n, ct.c_size_t) for n in ("h", "dg", "du", "kept", "x", "wg", "wu", "wd", "dy", "part", "bytes", "kept_bytes")] +
                [(n, Tile) for n in ("gate", "gate_back", "y", "dx", "dw")] +
                [("fits", ct.c_bool), ("narrow", ct.c_bool), ("dx_sum", ct.c_size_t), ("narrow_parts", ct.c_int),
                 ("narrow_slices", ct.c_int), ("few", ct.c_bool), ("narrow_groups", ct.c_int)])


def ways(layout, rows, i, h, o, dtype):
    """{(launch, tile, steps or splits)} of a forward and a backward without kept."""
    size = 4 if dtype == 0 else 2
    step, up = 128 // size, lambda n: -(-n // (16 // size)) * (16 // size)
    fwd, bwd = layout(rows, i, h, o, dtype, False, False), layout(rows, i, h, o, dtype, True, True)
    assert not (fwd.narrow or fwd.few or bwd.narrow) and fwd.fits and bwd.fits
    assert fwd.ldx == up(i) and fwd.ldh == up(h) and fwd.ldy == up(o)   # the structure here is the library's
    found = set()
    for name, t, products, k in (("gate", fwd.gate, [(rows, 2 * up(h))], up(i)), ("y", fwd.y, [(rows, o)], up(h)),
                                 ("gate_back", bwd.gate_back, [(rows, up(h))], o), ("dx", bwd.dx, [(rows, i)], h),
                                 ("dw", bwd.dw, [(h, i), (h, i), (o, h)], rows)):
        groups = sum(-(-m // t.side) * -(-n // t.side) for m, n in products) * t.splits
        tile = "64, four buffers" if t.side == 64 and groups <= MORE_BUFFERS else str(t.side)
        steps = -(-k // step)
        found.add((name, tile, "split" if 1 < t.splits <= 16 else "split much" if t.splits > 16 else
                   f"{steps} steps" if steps < 3 else "odd steps" if steps % 2 else "even steps"))
    return found


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_the_sizes_take_every_way(dtype):
    from nest_splat import _lib as L
    layout = L.lib()._ZN4nest12gated_layoutEliiiibb
    layout.restype, layout.argtypes = Layout, [ct.c_int64] + [ct.c_int] * 4 + [ct.c_bool] * 2
    found = set()
    for size in FLOAT32 if dtype == 0 else SIXTEEN:
        found |= ways(layout, *size, dtype)
    tiles, steps = ("256", "128", "64", "64, four buffers"), ("1 steps", "2 steps", "odd steps", "even steps")
    want = {(n, t, s) for n in ("gate", "gate_back", "y", "dx", "dw") for t in tiles for s in steps}
    want |= {(n, t, "split") for n in ("y", "dx", "dw") for t in tiles}
    want |= {(n, t, "split much") for n in ("y", "dx", "dw") for t in tiles[2:]}
    want |= {("dx", "128", "split much"), ("dw", "128", "split much")}
    if dtype == 0:
        want |= {("y", "128", "split much"), ("dx", "256", "split much"), ("dw", "256", "split much")}
    assert not want - found, sorted(want - found)


@pytest.mark.gpu
@pytest.mark.parametrize("size", FLOAT32, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients_float32(size):
    from nest_splat import blocks
    from test_gpu_blocks import ffn_case, ffn_check
    ffn_check(blocks, *ffn_case(*size, torch.float32), ("silu", "gelu", "relu")[FLOAT32.index(size) % 3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", SIXTEEN, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients_16_bit(size, dtype):
    from nest_splat import blocks
    from test_gpu_blocks import ffn_case, ffn_check
    ffn_check(blocks, *ffn_case(*size, dtype), ("gelu", "silu", "relu")[SIXTEEN.index(size) % 3])
