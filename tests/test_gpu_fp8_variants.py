"""Every form of the 8-bit product's tiled kernel, over its whole output: each tile, K whole and in slices, one tile a
workgroup and several, K that ends inside a block and K that does not, rows of out that start on no line. Which form a size
takes is chosen by an estimate, so each case says what it is there for and asserts that it gets it (on 256 compute units).

The sizes are the smallest of at least four blocks of K a slice among 1.5 million drawn up to 5e10 multiply-adds. What is
missing here (bf16: several tiles a workgroup with K in slices on wide tiles) none of them took."""
import ctypes

import pytest

from helpers import BF16, F32
from test_gpu_fp8 import check_gemm

pytestmark = pytest.mark.gpu

# rows and columns of the tile, K in slices, several tiles a workgroup; m, n, k
BF16_CASES = [
    (128, 128, 0, 0, 65, 7623, 575), (128, 128, 0, 0, 67, 8083, 512), (128, 128, 0, 1, 796, 9257, 512),
    (128, 128, 0, 1, 4891, 1595, 535), (128, 128, 1, 0, 34, 17, 3981), (128, 128, 1, 0, 35, 17, 4096),
    (128, 128, 1, 1, 1291, 1129, 10880), (128, 192, 0, 0, 259, 10925, 523), (128, 192, 0, 0, 262, 10915, 512),
    (128, 192, 0, 1, 776, 12383, 512), (128, 192, 0, 1, 1057, 10245, 517), (128, 192, 1, 0, 33, 11127, 2471),
    (128, 192, 1, 0, 33, 11409, 2432), (128, 192, 1, 1, 1542, 2435, 7967), (128, 192, 1, 1, 1558, 2461, 8064),
    (128, 256, 0, 0, 514, 11007, 512), (128, 256, 0, 0, 523, 10883, 531), (128, 256, 0, 1, 1284, 11297, 515),
    (128, 256, 0, 1, 1305, 11215, 512), (128, 256, 1, 0, 17, 8459, 9856), (128, 256, 1, 0, 17, 8701, 9799),
    (128, 256, 1, 0, 600, 4096, 10240), (256, 128, 0, 0, 5486, 971, 523), (256, 128, 0, 0, 6551, 783, 512),
    (256, 128, 0, 1, 1537, 9235, 512), (256, 128, 0, 1, 2371, 6445, 529), (256, 128, 1, 0, 132, 6433, 5707),
    (256, 128, 1, 0, 135, 6503, 5760), (256, 192, 0, 0, 643, 11251, 512), (256, 192, 0, 0, 656, 11391, 525),
    (256, 192, 0, 1, 1676, 10415, 512), (256, 192, 0, 1, 2060, 8647, 519), (256, 192, 0, 1, 8192, 4608, 1152),
    (256, 192, 1, 0, 136, 8473, 7019), (256, 192, 1, 0, 137, 8489, 7424), (256, 256, 0, 0, 919, 12411, 512),
    (256, 256, 0, 0, 1154, 9851, 529), (256, 256, 0, 1, 2058, 11597, 512), (256, 256, 0, 1, 2231, 10943, 517),
    (256, 256, 1, 0, 129, 12291, 8960), (256, 256, 1, 0, 134, 12311, 8481)]
F32_CASES = [
    (128, 128, 0, 0, 65, 12313, 561), (128, 128, 0, 0, 69, 12337, 640), (128, 128, 0, 1, 796, 9257, 512),
    (128, 128, 0, 1, 4891, 1595, 535), (128, 128, 1, 0, 33, 17, 5539), (128, 128, 1, 0, 34, 17, 5120),
    (128, 128, 1, 1, 1287, 1025, 8767), (128, 128, 1, 1, 1296, 1051, 7552), (128, 192, 0, 0, 259, 10925, 523),
    (128, 192, 0, 0, 262, 10915, 512), (128, 192, 0, 1, 776, 12383, 512), (128, 192, 0, 1, 1057, 10245, 517),
    (128, 192, 1, 0, 33, 12005, 2701), (128, 192, 1, 0, 35, 9689, 3200), (128, 192, 1, 1, 1537, 2439, 5563),
    (128, 192, 1, 1, 1607, 2473, 6016), (128, 256, 0, 0, 514, 11007, 512), (128, 256, 0, 0, 523, 10883, 531),
    (128, 256, 0, 1, 1284, 11297, 515), (128, 256, 0, 1, 1305, 11215, 512), (128, 256, 1, 0, 35, 12337, 3623),
    (128, 256, 1, 0, 40, 12361, 3200), (128, 256, 1, 1, 259, 8271, 10695), (128, 256, 1, 1, 261, 8199, 11136),
    (256, 128, 0, 0, 5486, 971, 523), (256, 128, 0, 0, 6551, 783, 512), (256, 128, 0, 1, 919, 12411, 512),
    (256, 128, 0, 1, 1154, 9851, 529), (256, 128, 1, 0, 131, 8471, 3456), (256, 128, 1, 0, 135, 9001, 2961),
    (256, 128, 1, 1, 129, 12291, 8960), (256, 128, 1, 1, 138, 12399, 9523), (256, 192, 0, 0, 643, 11251, 512),
    (256, 192, 0, 0, 656, 11391, 525), (256, 192, 0, 1, 1695, 11675, 512), (256, 192, 0, 1, 2823, 7047, 515),
    (256, 192, 1, 0, 134, 8211, 5511), (256, 192, 1, 0, 135, 8227, 5120), (256, 192, 1, 1, 391, 9377, 10155),
    (256, 192, 1, 1, 404, 9221, 10240)]


def check(dtype, rows, cols, sliced, walked, m, n, k):
    import burnisher_amd as bh
    plan = bh.GemmFp8Plan()
    bh.call("bh_gemm_fp8_describe", m, n, k, BF16 if dtype == "bfloat16" else F32, 1, 0, ctypes.byref(plan))
    got = (plan.in_lds, plan.tile_rows, plan.tile_cols, plan.slices > 1, plan.tiles > plan.workgroups)
    assert got == (1, rows, cols, bool(sliced), bool(walked)), "this size has another form now: it needs another size"
    check_gemm(m, n, k, act=m % 3, with_bias=True, dtype=dtype)


@pytest.mark.parametrize("rows,cols,sliced,walked,m,n,k", BF16_CASES)
def test_bf16(hip, rows, cols, sliced, walked, m, n, k):
    check("bfloat16", rows, cols, sliced, walked, m, n, k)


@pytest.mark.parametrize("rows,cols,sliced,walked,m,n,k", F32_CASES)
def test_f32(hip, rows, cols, sliced, walked, m, n, k):
    check("float32", rows, cols, sliced, walked, m, n, k)


@pytest.mark.parametrize("m,n,k", [(1104, 1120, 7736), (506, 1102, 4814), (829, 1791, 7442)])
def test_as_many_tiles_as_run_at_once(hip, m, n, k):
    # a number of workgroups that is no multiple of eight, in slices
    check_gemm(m, n, k, with_bias=True)
