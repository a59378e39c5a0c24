"""bh_quantize_fp8 and bh_gemm_fp8 on the GPU against plain forms.

The quantiser is two IEEE divisions, one fp32 product and one conversion a value, so its codes and
scales equal the same operations in torch bit for bit. The product is checked against 64 bits on the
same codes and scales, with tolerances that count roundings:
  - an fp32 sum of K products, in any order: at most 2^-23 of the summed magnitudes per addition;
  - an fp32 output: the codes are multiplied exactly, so that and the epilogue is all;
  - a bf16 output: half a step, 2^-8 of the value, and the 8-bit matrix instruction, which adds eight
    neighbouring products at a time and drops of each less than 2^-13 of the largest of the eight.
"""
import math

import pytest

from helpers import BF16, F32

pytestmark = pytest.mark.gpu

FLOOR = 2.0 ** -96


def blocks_of(x, block_rows):
    """x padded to whole blocks, as [row blocks, block_rows, column blocks, 128] in fp32."""
    import torch
    rows, cols = x.shape
    nr, nc = -(-rows // block_rows), -(-cols // 128)
    p = torch.zeros(nr * block_rows, nc * 128, device=x.device)
    p[:rows, :cols] = x.float()
    return p.view(nr, block_rows, nc, 128)


def quantize_plain(x, block_rows):
    import torch
    rows, cols = x.shape
    b = blocks_of(x, block_rows)
    amax = b.abs().amax(dim=(1, 3))
    amax = torch.where(amax < FLOOR, torch.full_like(amax, FLOOR), amax)   # keeps a NaN
    top = torch.full_like(amax, 448.0)   # a tensor: torch replaces a division by a number by a product
    codes = (b * (top / amax)[:, None, :, None]).reshape(-1, b.shape[2] * 128)[:rows]
    codes[:, cols:] = 0   # the tail of a row is zeros even where its block holds a NaN
    codes = codes[:, :(cols + 15) // 16 * 16].to(torch.float8_e4m3fn)
    scales = amax / top
    return codes.contiguous(), scales.t().contiguous() if block_rows == 1 else scales


def quantize(x, block_rows, guard=0):
    """The library's codes and scales of the matrix x (a view with any row stride)."""
    import torch
    import burnisher_amd as bh
    rows, cols = x.shape
    assert x.stride(1) == 1 or cols == 1
    kp = (cols + 15) // 16 * 16
    codes = torch.full((rows * kp + guard,), 0x55, dtype=torch.uint8, device="cuda")
    shape = (-(-cols // 128), rows) if block_rows == 1 else (-(-rows // 128), -(-cols // 128))
    scales = torch.full((shape[0] * shape[1] + guard,), -7.0, device="cuda")
    bh.call("bh_quantize_fp8", x.data_ptr(), x.stride(0), codes.data_ptr(), scales.data_ptr(), rows, cols, block_rows,
            BF16 if x.dtype == torch.bfloat16 else F32, bh.stream_ptr())
    if guard:
        assert (codes[rows * kp:] == 0x55).all() and (scales[-guard:] == -7.0).all(), "written past the end"
    n = shape[0] * shape[1]
    return codes[:rows * kp].view(rows, kp).view(torch.float8_e4m3fn), scales[:n].view(shape)


def same_bits(a, b):
    import torch
    def num(t):   # one NaN for all
        f = t.float()
        return torch.where(torch.isnan(f), torch.full_like(f, 1e30), f)
    return torch.equal(num(a), num(b))


def normal(shape, seed, dtype, std=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 127), (16, 128), (17, 129), (130, 520), (257, 1155),
                                       (128, 2048), (600, 640)])
def test_quantize_is_the_formula_bit_for_bit(hip, dtype, block_rows, rows, cols):
    import torch
    x = normal((rows, cols), rows * 31 + cols, getattr(torch, dtype))
    x[:, ::7] *= 30
    got = quantize(x, block_rows, guard=64)
    want = quantize_plain(x, block_rows)
    assert got[0].view(torch.uint8)[:, cols:].eq(0).all(), "the tail of a row is not zero"
    assert same_bits(got[0], want[0])
    assert torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_rows_of_a_wider_tensor_and_unaligned_ones(hip, dtype, block_rows):
    import torch
    wide = normal((70, 777), 5, getattr(torch, dtype))
    for view in (wide[:, :300], wide[3:, 1:400], wide[:, 8:8 + 256], wide[1:2, 5:6]):
        got, want = quantize(view, block_rows, guard=16), quantize_plain(view, block_rows)
        assert same_bits(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_zeros_tiny_infinite_and_nan_blocks(hip, block_rows):
    import torch
    x = torch.zeros(640, 140, device="cuda")
    x[130:260] = normal((130, 140), 1, torch.float32) * 1e-35     # below the floor: codes stay small
    x[300, 3], x[400, 130] = math.inf, math.nan
    x[520, 2] = 3e38
    x[521, 2] = 1.5e-45                                            # the smallest fp32
    got, want = quantize(x, block_rows, guard=8), quantize_plain(x, block_rows)
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])
    rows = 1 if block_rows == 1 else 128
    finite = torch.isfinite(got[1].t() if block_rows == 1 else got[1])
    assert not finite[300 // rows, 0] and not finite[400 // rows, 1] and finite[0].all()
    assert got[1][torch.isfinite(got[1])].gt(0).all()


def test_quantize_every_bf16_value(hip):
    # all 2^16 patterns, one a row with 448 beside it, so the factor is 1 where the value is not larger
    import torch
    bits = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16).view(torch.bfloat16)
    x = torch.stack([bits, torch.full_like(bits, 448.0)], dim=1).contiguous()
    got, want = quantize(x, 1), quantize_plain(x, 1)
    assert same_bits(got[0], want[0]) and same_bits(got[1], want[1])


# ---- the product ---------------------------------------------------------------------------------

def operands(m, n, k, seed, kind="normal"):
    import torch
    a, b = normal((m, k), seed, torch.float32), normal((n, k), seed + 1, torch.float32, 0.02)
    if kind == "outliers":
        a[:, ::37] *= 50
        b[::5] *= 20
    return quantize_plain(a, 1) + quantize_plain(b, 128)


def run_gemm(a, sa, b, sb, bias, k, act=0, dtype="bfloat16", workspace=True, guard=64):
    import torch
    import burnisher_amd as bh
    m, n = a.shape[0], b.shape[0]
    buf = torch.full((m * n + guard,), -3.0, dtype=getattr(torch, dtype), device="cuda")
    need = bh.lib().bh_gemm_fp8_workspace_bytes(m, n, k)
    assert need >= 0
    # what an earlier call left in the workspace must not matter
    ws = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device="cuda")
    bh.call("bh_gemm_fp8", a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), bh.ptr(bias), buf.data_ptr(), m, n,
            k, act, BF16 if dtype == "bfloat16" else F32, ws.data_ptr() if workspace else None,
            need if workspace else 0, bh.stream_ptr())
    assert (buf[m * n:] == -3.0).all(), "written past the end"
    return buf[:m * n].view(m, n)


def gemm_plain(a, sa, b, sb, bias, k, act, dtype):
    """(64-bit result, tolerance) of one product."""
    import torch
    m, n = a.shape[0], b.shape[0]
    blocks = -(-k // 128)
    x, y = a[:, :k].double(), b[:, :k].double()
    total = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(total)
    drop = torch.zeros_like(total)
    eights = lambda t: t.abs().view(t.shape[0], -1, 8).amax(2)  # noqa: E731
    a8, b8 = a.double(), b.double()   # rows of whole sixteens, zero at the end
    of = torch.arange(n, device="cuda") // 128
    for j in range(blocks):
        c = slice(j * 128, min(j * 128 + 128, k))
        s = sa[j].double()[:, None] * sb[of, j].double()
        xj, yj = x[:, c].contiguous(), y[:, c].t().contiguous()
        total += xj @ yj * s
        size += xj.abs() @ yj.abs() * s
        c = slice(j * 128, min(j * 128 + 128, a.shape[1]))
        drop += 8 * 2.0 ** -13 * (eights(a8[:, c]) @ eights(b8[:, c]).t().contiguous()) * s
    tol = (k + 3 * blocks + 2) * 2.0 ** -23 * size + (drop if dtype == "bfloat16" else 0)
    if bias is not None:
        total += bias.double()
        tol += 2.0 ** -23 * total.abs()
    v = total
    if act == 1:
        u2 = 2 * math.sqrt(2 / math.pi) * (total + 0.044715 * total ** 3)
        v = total / (1 + torch.exp(-u2))
        # slope at most 1.13; the exponent's few fp32 roundings grow with its size (below 88, where exp ends)
        tol = 1.13 * tol + v.abs() * (u2.abs().clamp(max=90) + 8) * 2.0 ** -22
    elif act == 2:
        v = total / (1 + torch.exp(-total))
        tol = 1.1 * tol + v.abs() * (total.abs().clamp(max=90) + 8) * 2.0 ** -22
    tol = tol + v.abs() * (2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -23) + 1e-30
    return v, tol


def check_gemm(m, n, k, act=0, with_bias=False, dtype="bfloat16", kind="normal", workspace=True):
    import torch
    a, sa, b, sb = operands(m, n, k, m * 7 + n * 3 + k, kind)
    bias = normal((n,), 3, getattr(torch, dtype)) if with_bias else None
    got = run_gemm(a, sa, b, sb, bias, k, act, dtype, workspace)
    want, tol = gemm_plain(a, sa, b, sb, bias, k, act, dtype)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: " \
        f"{got[tuple(bad.nonzero()[0])]} for {want[tuple(bad.nonzero()[0])]}"
    return got


GEMM_SIZES = [(1, 1, 1), (1, 4096, 4096), (1, 16, 10240), (2, 130, 15), (5, 17, 129), (16, 384, 2048), (17, 100, 300),
              (33, 257, 1152), (64, 128, 128), (65, 1000, 260), (77, 4608, 1152), (120, 1152, 4608), (128, 256, 4096),
              (200, 128, 640), (257, 129, 2001), (300, 4100, 272), (600, 4096, 1024), (1024, 3456, 1152), (1155, 333, 777),
              (2049, 1152, 128), (4096, 64, 256)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("m,n,k", GEMM_SIZES)
def test_gemm_sizes(hip, m, n, k, dtype):
    check_gemm(m, n, k, dtype=dtype)


# one and several blocks of K, few and many tiles; test_gpu_fp8_variants.py reaches every form
TILE_SIZES = [(454, 3853, 16), (33, 39, 5011), (817, 4616, 170), (272, 3733, 3941), (929, 1287, 2911), (1843, 4127, 330),
              (521, 3680, 4188), (2763, 2222, 200), (404, 4285, 5927), (1592, 802, 5735), (2256, 3619, 330),
              (2951, 3411, 16), (2875, 4239, 330), (4500, 4300, 160), (2048, 2048, 2048)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("m,n,k", TILE_SIZES)
def test_gemm_tiles(hip, m, n, k, dtype):
    check_gemm(m, n, k, dtype=dtype, with_bias=k % 2 == 1)


# rows of out that start on lines of 128 bytes and rows that do not, tiles inside and across the edge
ROW_SIZES = [(195, 4360, 272), (235, 4288, 272), (131, 280, 4005), (141, 256, 5008), (2816, 1416, 256), (1697, 2432, 256),
             (266, 3904, 3968), (1836, 4160, 384), (2736, 2200, 256), (2304, 3592, 256), (2495, 3264, 256), (2736, 4424, 256),
             (2816, 4608, 256), (2637, 2952, 256), (515, 3588, 4224), (1318, 4420, 256), (385, 4160, 3749), (2927, 2820, 256)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("m,n,k", ROW_SIZES)
def test_gemm_output_rows_of_any_alignment(hip, m, n, k, dtype):
    import torch
    import burnisher_amd as bh
    got = check_gemm(m, n, k, act=2, with_bias=True, dtype=dtype)
    a, sa, b, sb = operands(m, n, k, m * 7 + n * 3 + k)
    bias = normal((n,), 3, getattr(torch, dtype))
    need = max(16, bh.lib().bh_gemm_fp8_workspace_bytes(m, n, k))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for shift in (16 // got.element_size(), 1):
        buf = torch.full((m * n + 64,), -3.0, dtype=got.dtype, device="cuda")
        out = buf[shift:shift + m * n]
        bh.call("bh_gemm_fp8", a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), bias.data_ptr(), out.data_ptr(), m,
                n, k, 2, BF16 if dtype == "bfloat16" else F32, ws.data_ptr(), need, bh.stream_ptr())
        assert torch.equal(out.view(m, n), got)
        assert (buf[:shift] == -3.0).all() and (buf[shift + m * n:] == -3.0).all(), "written outside"


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("m,n,k", [(1, 300, 400), (40, 129, 256), (333, 640, 520), (2048, 256, 128)])
def test_gemm_epilogues(hip, m, n, k, act, dtype):
    check_gemm(m, n, k, act=act, with_bias=True, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("m,n,k", [(4, 256, 4096), (600, 512, 10240), (512, 1024, 1024)])
def test_gemm_outliers_and_no_workspace(hip, m, n, k, dtype):
    check_gemm(m, n, k, dtype=dtype, kind="outliers")
    check_gemm(m, n, k, dtype=dtype, workspace=False)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("m,n,k", [(3, 300, 300), (300, 257, 400), (500, 1028, 640), (300, 130, 8192)])
def test_gemm_bias_of_any_alignment(hip, m, n, k, dtype):
    import torch
    a, sa, b, sb = operands(m, n, k, 5)
    wide = normal((n + 9,), 3, getattr(torch, dtype))
    for shift in (1, 3, 8):
        bias = wide[shift:shift + n]
        want, tol = gemm_plain(a, sa, b, sb, bias, k, 1, dtype)
        assert ((run_gemm(a, sa, b, sb, bias, k, 1, dtype).double() - want).abs() <= tol).all()


def test_gemm_of_an_empty_sum_is_the_epilogue_of_the_bias(hip):
    import torch
    one = torch.zeros(64, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(64, device="cuda")
    bias = normal((5,), 1, torch.float32)
    for m in (3, 200):
        got = run_gemm(one[:16].view(1, 16).expand(m, 16), scale, one[:16].view(1, 16).expand(5, 16), scale, bias, 0,
                       dtype="float32")
        assert torch.equal(got, bias.expand(m, 5))


def test_gemm_of_matrices_without_columns_takes_no_addresses(hip):
    import torch
    import burnisher_amd as bh
    bias = normal((5,), 1, torch.float32)
    for m in (3, 200):
        out = torch.full((m, 5), 9.0, device="cuda")
        bh.call("bh_gemm_fp8", None, None, None, None, bias.data_ptr(), out.data_ptr(), m, 5, 0, 0, F32, None, 0,
                bh.stream_ptr())
        assert torch.equal(out, bias.expand(m, 5))


def test_gemm_stays_inside_its_workspace_and_refuses_a_small_one(hip):
    import torch
    import burnisher_amd as bh
    m, n, k = 600, 256, 8192
    need = bh.lib().bh_gemm_fp8_workspace_bytes(m, n, k)
    assert need > 0
    a, sa, b, sb = operands(m, n, k, 1)
    out = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    ws = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device="cuda")

    def call(at, size):
        return bh.lib().bh_gemm_fp8(a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), None, out.data_ptr(), m, n,
                                    k, 0, BF16, at, size, bh.stream_ptr())

    used = 4 * m * n * 2   # at least two slices
    assert call(ws.data_ptr(), used // 2) != 0 and b"this call needs" in bh.lib().bh_last_error()
    assert call(ws.data_ptr() + 8, need) != 0 and b"16-byte" in bh.lib().bh_last_error()
    torch.cuda.synchronize()
    assert not out.any() and (ws == 0x5a).all(), "a refused call wrote"
    assert call(ws.data_ptr(), need) == 0
    assert (ws[need:] == 0x5a).all(), "written past the workspace"
    assert torch.equal(out, run_gemm(a, sa, b, sb, None, k))


def test_gemm_small_whole_numbers_are_exact(hip):
    # integers up to 8 with power-of-two scales: every product and sum is exact in either instruction
    import torch
    for m, n, k in ((3, 70, 500), (700, 300, 500)):
        g = torch.Generator(device="cuda").manual_seed(9)
        a = torch.randint(-8, 9, (m, 512), generator=g, device="cuda").float()
        b = torch.randint(-8, 9, (n, 512), generator=g, device="cuda").float()
        a[:, k:], b[:, k:] = 0, 0
        sa = torch.pow(2.0, torch.randint(-3, 4, (4, m), generator=g, device="cuda").float())
        sb = torch.pow(2.0, torch.randint(-3, 4, (-(-n // 128), 4), generator=g, device="cuda").float())
        want = torch.zeros(m, n, dtype=torch.float64, device="cuda")
        for j in range(4):
            c = slice(j * 128, j * 128 + 128)
            want += a[:, c].double().contiguous() @ b[:, c].t().double().contiguous() * sa[j].double()[:, None] * \
                sb[torch.arange(n, device="cuda") // 128, j].double()
        a8, b8 = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
        assert torch.equal(run_gemm(a8, sa, b8, sb, None, k, dtype="float32").double(), want)
        assert torch.equal(run_gemm(a8, sa, b8, sb, None, k), want.to(torch.bfloat16))


@pytest.mark.parametrize("m", [3, 40, 300, 2048])
def test_gemm_whose_large_products_cancel(hip, m):
    # of every eight columns two products are +-448 * 448 and the other six whole numbers below 2^7: an fp32 output
    # has the exact sum, a bf16 one is off by at most what the contract lets each eight lose, 8 * 2^-13 * 448 * 448, and
    # its rounding. In the second half of the output's columns nothing cancels and the sum keeps its relative accuracy.
    import torch
    n, k = 200, 384
    g = torch.Generator(device="cuda").manual_seed(m)
    a, b = (torch.randint(-8, 9, (rows, k), generator=g, device="cuda").float() for rows in (m, n))
    a[:, 0::8], a[:, 1::8], b[:, 0::8], b[:, 1::8] = 448, 448, 448, -448
    b[n // 2:, 1::8] = 448
    want = a.double() @ b.t().double().contiguous()
    a8, b8 = a.to(torch.float8_e4m3fn), b.to(torch.float8_e4m3fn)
    sa, sb = torch.ones(3, m, device="cuda"), torch.ones(2, 3, device="cuda")
    off = (run_gemm(a8, sa, b8, sb, None, k, dtype="float32").double() - want).abs()
    # Whole numbers below 2^24 are exact in fp32. Where the products cancel any part of the sum is: at most 48 * 448^2
    # = 9.6e6 and the small ones. Where they do not, a block's sum is (16 * 2 * 448^2 = 6.4e6) and the sum of two, but not
    # that of all three, 1.9e7: its addition rounds by half a step, 2^-24 of it.
    alike = slice(n // 2, n)
    assert off[:, :n // 2].max() == 0 and (off <= 2.0 ** -24 * want.abs()).all()
    off = (run_gemm(a8, sa, b8, sb, None, k).double() - want).abs()
    lost = k / 8 * 8 * 2.0 ** -13 * 448 * 448
    assert (off <= lost + 2.0 ** -8 * (want.abs() + lost)).all()
    # each eight adds up to at least 2 * 448^2 - 6 * 64 and loses below 2^-10 * 448^2
    assert (off[:, alike] <= (2.0 ** -11 * (1 + 2.0 ** -8) + 2.0 ** -8 * (1 + 2.0 ** -10)) * want[:, alike].abs()).all()


@pytest.mark.parametrize("m", [2, 40, 300])
def test_gemm_keeps_a_nan_and_an_infinite_scale_in_their_rows(hip, m):
    import torch
    a, sa, b, sb = operands(m, 200, 384, 4)
    clean = run_gemm(a, sa, b, sb, None, 384)
    sa[1, 1] = math.inf
    got = run_gemm(a, sa, b, sb, None, 384)
    assert not torch.isfinite(got[1]).any()
    keep = torch.arange(m, device="cuda") != 1
    assert torch.equal(got[keep], clean[keep])
    sb[1, 0] = math.nan
    got = run_gemm(a, sa, b, sb, None, 384)
    assert torch.isnan(got[:, 128:]).all() and torch.equal(got[keep][:, :128], clean[keep][:, :128])


@pytest.mark.parametrize("m,n,k", [(1, 512, 2048), (300, 512, 2048), (600, 256, 8192)])
def test_gemm_in_a_graph_and_on_two_streams(hip, m, n, k):
    import torch
    import burnisher_amd as bh
    sets = [operands(m, n, k, s) for s in (1, 2)]
    need = max(16, bh.lib().bh_gemm_fp8_workspace_bytes(m, n, k))
    out = [torch.zeros(m, n, dtype=torch.bfloat16, device="cuda") for _ in sets]
    ws = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in sets]

    def call(i, stream):
        a, sa, b, sb = sets[i]
        bh.call("bh_gemm_fp8", a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), None, out[i].data_ptr(), m, n, k,
                0, BF16, ws[i].data_ptr(), need, bh.stream_ptr(stream))

    want = [run_gemm(*s, None, k) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for i in (0, 1):
            call(i, streams[i])
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0, torch.cuda.current_stream())
    for seed in (5, 6, 7):
        for t, fresh in zip(sets[0], operands(m, n, k, seed)):
            t.copy_(fresh)
        out[0].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], run_gemm(*sets[0], None, k)), "a replay differs from the call"


def within(got, want_tol):
    want, tol = want_tol
    return ((got.double() - want).abs() <= tol).all()


def test_matrices_beyond_32_bits(hip):
    import torch
    import burnisher_amd as bh
    # 530432 rows of 8192: 8.7 GB of bf16, 4.3 GB of codes, as the activations and as the weights of a product
    rows, k, tail = 1024 * 518, 8192, 300
    piece = normal((1024, k), 1, torch.bfloat16)
    x = piece.repeat(518, 1)
    small, small_s = quantize_plain(normal((40, k), 2, torch.float32, 0.02), 128)
    q, sq = quantize(x, 1)
    want, want_s = quantize_plain(piece, 1)
    for at in (0, rows - 1024):
        assert same_bits(q[at:at + 1024], want) and torch.equal(sq[:, at:at + 1024], want_s)
    out = run_gemm(q, sq, small, small_s, None, k)
    assert within(out[-tail:], gemm_plain(q[-tail:], sq[:, -tail:].contiguous(), small, small_s, None, k, 0, "bfloat16"))
    q, sq = quantize(x, 128)
    want, want_s = quantize_plain(piece, 128)
    for at in (0, rows - 1024):
        assert same_bits(q[at:at + 1024], want) and torch.equal(sq[at // 128:at // 128 + 8], want_s)
    few, few_s = quantize_plain(normal((3, k), 3, torch.float32), 1)
    out = run_gemm(few, few_s, q, sq, None, k)
    assert within(out[:, -384:], gemm_plain(few, few_s, q[-384:], sq[-3:], None, k, 0, "bfloat16"))
    del x, q, out
    # 4.6 GB of output
    m, n, k = 70000, 33000, 130
    a, sa, b, sb = operands(m, n, k, 4)
    out = run_gemm(a, sa, b, sb, None, k)
    assert within(out[-200:], gemm_plain(a[-200:], sa[:, -200:].contiguous(), b, sb, None, k, 0, "bfloat16"))
    bh.check(0)


def test_quantized_projection_of_a_wide_activation(hip):
    # as a program uses them: weights quantised once, activations per call, the product against the
    # unquantised one; an e4m3 rounding is at most 2^-4 of a value, so the error of a sum of K products of two
    # rounded factors stays below (2 * 2^-4 + 2^-8) of the summed magnitudes, plus the output's own
    import torch
    m, n, k = 300, 520, 1000
    x, w = normal((m, k), 1, torch.bfloat16), normal((n, k), 2, torch.bfloat16, 0.02)
    qw, sw = quantize(w, 128)
    qx, sx = quantize(x, 1)
    got = run_gemm(qx, sx, qw, sw, None, k).double()
    want = x.double() @ w.t().double().contiguous()
    size = x.double().abs() @ w.t().double().abs().contiguous()
    # a value below 2^-6 of e4m3's normal range rounds by at most 2^-10 of a unit: 2^-10 * amax / 448 each
    small = 2.0 ** -10 / 448 * (x.double().abs().amax(1)[:, None] * w.double().abs().sum(1) +
                                w.double().abs().amax() * x.double().abs().sum(1)[:, None])
    assert ((got - want).abs() <= (2 * 2.0 ** -4 + 2.0 ** -7) * size + 2 * small + 2.0 ** -8 * want.abs()).all()


def test_the_default_stream_is_the_current_one(hip):
    import torch
    import burnisher_amd as bh
    other = torch.cuda.Stream()
    assert bh.stream_ptr() == torch.cuda.current_stream().cuda_stream
    assert bh.stream_ptr(other) == other.cuda_stream
    with torch.cuda.stream(other):
        assert bh.stream_ptr() == other.cuda_stream
