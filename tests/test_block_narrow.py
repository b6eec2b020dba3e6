"""The rule that keeps narrow 16-bit rows on the chip, and every way that its kernels run under it: padded widths of 32 to 128
features, 1 to 8 waves that share the hidden features, one, two and more launches of a backward, hidden features that fill a
launch's slices and that do not, workgroups of one turn and of several."""
import ctypes as ct

import pytest
import torch

from test_block_tiles import Layout

# (rows, in, hidden, out)
SIZES = [(64, 22, 132, 45), (64, 28, 8, 10), (64, 40, 8, 91), (64, 58, 8, 44), (64, 61, 128, 46), (64, 98, 64, 54),
         (64, 105, 8, 55), (64, 107, 32, 111), (64, 115, 65, 3), (65, 13, 67, 23), (65, 62, 32, 73), (65, 64, 65, 46),
         (65, 68, 65, 20), (65, 68, 128, 53), (65, 85, 64, 91), (65, 92, 33, 78), (65, 116, 33, 68), (66, 8, 33, 16),
         (66, 123, 128, 91), (67, 22, 397, 18), (67, 27, 130, 14), (68, 1, 64, 43), (69, 22, 32, 21), (71, 12, 128, 14),
         (75, 21, 64, 18), (80, 35, 256, 5), (192, 5, 512, 32), (226, 24, 511, 7), (1236, 23, 256, 17), (15897, 28, 722, 22),
         (17548, 19, 768, 23), (20801, 15, 639, 7), (29852, 13, 259, 10), (29989, 55, 512, 56), (30883, 45, 457, 31),
         (32436, 6, 643, 62), (33113, 91, 8, 74), (33133, 45, 8, 30), (37920, 59, 767, 19), (40611, 63, 382, 50),
         (47613, 19, 384, 2), (48250, 30, 272, 64), (49353, 7, 766, 21), (50992, 16, 384, 60), (51763, 27, 511, 45),
         (52996, 9, 768, 60), (68278, 21, 8, 13), (89465, 91, 375, 76), (90083, 46, 248, 86), (91088, 62, 382, 78),
         (94746, 70, 256, 55), (99204, 87, 255, 66), (107567, 5, 384, 94), (110527, 90, 192, 50), (112955, 42, 189, 92),
         (112967, 68, 191, 62), (163202, 22, 253, 105), (170892, 101, 378, 93), (170907, 25, 255, 101), (182361, 2, 382, 103),
         (191278, 118, 256, 51), (208704, 104, 384, 123), (227129, 72, 192, 105), (229308, 44, 187, 98), (243122, 11, 191, 109),
         (324408, 87, 32, 124)]


@pytest.fixture(scope="module")
def layout():
    from nest_splat import _lib as L
    f = L.lib()._ZN4nest12gated_layoutEliiiibb
    f.restype, f.argtypes = Layout, [ct.c_int64] + [ct.c_int] * 4 + [ct.c_bool] * 2
    return f


# a forward and backward in us, kept on the chip and in tiles
TIMED = [(64, 32, 128, 29, 38), (640000, 32, 128, 125, 636), (64, 32, 256, 31, 38), (64, 32, 1024, 67, 39), (8192, 32, 1024, 131, 71),
         (65536, 32, 2048, 371, 1005), (640000, 64, 128, 179, 680), (65536, 64, 1024, 254, 512), (8192, 64, 512, 103, 49),
         (64, 64, 2048, 211, 42), (1024, 64, 8192, 955, 80), (640000, 64, 1024, 1551, 4550), (64, 128, 256, 65, 36),
         (8192, 128, 512, 205, 55), (65536, 128, 1024, 608, 543), (640000, 128, 256, 981, 1448), (64, 128, 8192, 2317, 42),
         (8192, 128, 8192, 3358, 591), (65536, 128, 8192, 4849, 3858)]


@pytest.mark.parametrize("rows,features,hidden,narrow,tiles", TIMED)
def test_the_rule_takes_the_faster_way(layout, rows, features, hidden, narrow, tiles):
    for dtype in (1, 2):
        for backward in (False, True):
            assert layout(rows, features, hidden, features, dtype, backward, False).narrow == (narrow < tiles)
    assert not layout(rows, features, hidden, features, 0, False, False).narrow


def test_rows_and_features_that_never_stay(layout):
    assert not layout(63, 32, 64, 32, 2, False, False).narrow and layout(64, 32, 64, 32, 2, False, False).narrow
    for i, o in ((129, 16), (16, 129)):
        assert not layout(640000, i, 64, o, 2, False, False).narrow


def test_the_sizes_take_every_way(layout):
    found = set()
    for rows, i, h, o in SIZES:
        l = layout(rows, i, h, o, 2, True, True)
        assert l.narrow, (rows, i, h, o)
        ki = -(-max(i, o) // 32)
        full, per = 32 * l.narrow_slices, -(-h // l.narrow_parts)
        last = h - (l.narrow_parts - 1) * per
        groups = (8 if ki <= 2 else 4) // l.narrow_slices
        found |= {(ki, "turns" if rows > 256 * 32 * groups else "one turn"),
                  (ki, l.narrow_slices, min(l.narrow_parts, 3), "filled" if per == full and last == per else "ends" if per < full else "last ends")}
    want = {(ki, t) for ki in (1, 2, 3, 4) for t in ("one turn", "turns")}
    for ki, slices in ((1, (1, 2, 4, 8)), (2, (2, 4, 8)), (3, (1, 2, 4)), (4, (1, 2, 4))):
        want |= {(ki, s, 1, e) for s in slices for e in ("filled", "ends")}
        want |= {(ki, slices[-1], n, e) for n in (2, 3) for e in ("filled", "ends", "last ends")}
        want |= {(ki, slices[-2], 3, e) for e in ("filled", "ends", "last ends")}
    assert not want - found, sorted(want - found, key=str)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(size, dtype):
    from nest_splat import blocks
    from test_gpu_blocks import ffn_case, ffn_check
    ffn_check(blocks, *ffn_case(*size, dtype), ("gelu", "relu", "silu")[SIZES.index(size) % 3])
    torch.cuda.empty_cache()
