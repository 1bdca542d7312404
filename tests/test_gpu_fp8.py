"""Casts to 8 bits and the block-scaled product on the GPU against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

import simdyolo_b200 as sy
from tests import device_ops as D

pytestmark = pytest.mark.gpu


def spread(rows, cols, seed, dtype=torch.float32):
    """Values over a wide range of sizes: per-row and per-column factors, some zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    x = x * torch.exp(torch.randn(1, cols, generator=g))
    x[torch.rand(rows, cols, generator=g) < 0.02] = 0
    return x.to(dtype)


# ------------------------------------------------------------------ casts: equal to the definition, bit for bit

@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 300), (3, 127), (127, 5), (128, 128), (129, 257), (200, 640)])
def test_cast_both_ways(rows, cols, dtype, block_rows, fmt):
    x = spread(rows, cols, rows * 1000 + cols, dtype)
    q, e = D.cast_reference(x, fmt, block_rows)
    qt, et = D.cast_reference(x.T, fmt, block_rows)
    one = D.quantize(x.cuda(), fmt, block_rows)
    h, t = D.quantize(x.cuda(), fmt, block_rows, both=True)
    for got in (one, h):
        assert torch.equal(got.exponents(), e)
        assert torch.equal(got.data().view(torch.uint8), q.view(torch.uint8))
    assert torch.equal(t.exponents(), et)
    assert torch.equal(t.data().view(torch.uint8), qt.view(torch.uint8))
    assert torch.equal(D.dequantize(h, torch.float32).cpu().double(), D.values(q, e, block_rows))
    assert torch.equal(D.dequantize(t, dtype).cpu(), D.values(qt, et, block_rows).float().to(dtype))


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("offset, pitch", [(0, 208), (1, 201), (8, 216)])
def test_cast_of_strided_rows(offset, pitch, block_rows):
    base = spread(40, pitch + 16, 5, torch.bfloat16).cuda()
    x = base.view(-1)[offset:].as_strided((40, 200), (pitch, 1))
    q, e = D.cast_reference(x.cpu(), "e4m3", block_rows)
    h, t = D.quantize(x, "e4m3", block_rows, both=True)
    assert torch.equal(h.data().view(torch.uint8), q.view(torch.uint8)) and torch.equal(h.exponents(), e)
    qt, _ = D.cast_reference(x.cpu().T, "e4m3", block_rows)
    assert torch.equal(t.data().view(torch.uint8), qt.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("both", [False, True])
def test_cast_of_extreme_values(fmt, both):
    x = torch.zeros(130, 300)
    x[0, :130] = torch.finfo(torch.float32).max
    x[1, 5] = torch.finfo(torch.float32).smallest_normal
    x[1, 200] = 2.0 ** -149
    x[2, 3], x[2, 4], x[2, 5], x[2, 6] = float("inf"), -float("inf"), float("nan"), 3.0
    x[3, 128:256] = float("nan")
    x[4, :4] = torch.tensor([448.0, 449.0, 57344.0, 57345.0])
    x[5, 0], x[5, 130] = 448.0, 57344.0
    x[6, 0], x[6, 130] = -448.0 * (1 + 2.0 ** -23), 57344.0 * (1 + 2.0 ** -23)
    x[7, 0], x[7, 1] = 1.0, -0.0
    for block_rows in (1, 128):
        q, e = D.cast_reference(x, fmt, block_rows)
        h = D.quantize(x.cuda(), fmt, block_rows, both=both)
        h = h[0] if both else h
        assert torch.equal(h.exponents(), e)
        a, b = h.data().float(), q.float()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_cast_of_blocks_without_a_finite_value(dtype, block_rows, fmt):
    """Rows and columns of a block with nothing but NaN or infinities have scale 1, in both orientations."""
    nan, inf = float("nan"), float("inf")
    x = spread(300, 260, 8, dtype)
    x[:128, 3], x[128:256, 4], x[:, 5] = nan, inf, -inf
    x[256:, 6], x[:128, 140], x[:127, 141] = inf, torch.tensor([nan, inf] * 64), nan
    x[7, :128], x[140, 128:256], x[299, 256:] = nan, -inf, inf
    x[:128, 128:256] = nan if block_rows == 128 else x[:128, 128:256]
    for got, want in zip(D.quantize(x.cuda(), fmt, block_rows, both=True), (x, x.T)):
        q, e = D.cast_reference(want, fmt, block_rows)
        assert torch.equal(got.exponents(), e)
        a, b = got.data().float(), q.float()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])


def test_dequantize_takes_any_scale_byte_and_leaves_the_rows_padding():
    h = D.Held(4, 130, "e4m3", 1)
    h.q[:] = torch.arange(4 * h.q.shape[1], dtype=torch.int64, device="cuda").view(4, -1).remainder(127).to(torch.uint8)
    h.scale[:] = 127
    h.scale[1, 0], h.scale[2, 0], h.scale[3, 1] = 0, 255, 254
    out = D.dequantize(h, torch.float32, pitch=140).cpu()
    assert (out[:, 130:] == 7).all()
    assert out[2, :128].isnan().all() and not out[2, 128:].isnan().any()
    want = h.values()
    want[2, :128] = float("nan")
    assert torch.equal(out[1, :130].double(), want[1].float().double())
    assert torch.equal(out[3, :130].double(), want[3].float().double())


# ------------------------------------------------------------------ products

def operands(m, n, k, a_fmt="e4m3", b_fmt="e4m3", a_block=1, b_block=128, seed=0):
    a = D.quantize(spread(m, k, seed + 1).cuda(), a_fmt, a_block)
    b = D.quantize(spread(n, k, seed + 2).cuda(), b_fmt, b_block)
    return a, b


def check(a, b, dtype, got, start=None):
    va, vb = a.values(), b.values()
    want = va @ vb.T
    bound = D.product_bound(va, vb, dtype, want)
    if start is not None:
        want = want + start.double().cpu()
        bound = bound + D.HALF_STEP[dtype] * want.abs()
    got = got.double().cpu()
    if dtype == torch.float16:
        fits = want.abs() < 65000
        got, want, bound = got[fits], want[fits], bound[fits] + 2.0 ** -25   # below 2^-14 the step is 2^-24
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()


@pytest.mark.parametrize("m, n, k", [
    (1, 1, 1), (1, 16, 128), (1, 300, 1000), (2, 129, 127), (16, 128, 129), (17, 257, 513), (33, 1000, 2000),
    (65, 130, 4100), (127, 255, 640), (128, 128, 128), (129, 64, 200), (200, 33, 8000), (300, 1, 384), (513, 300, 256),
    (1000, 1000, 700), (2300, 2500, 300), (1500, 5200, 2300), (2100, 4100, 640)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_product_sizes(m, n, k, dtype):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, b = operands(m, n, k)
    check(a, b, dtype, D.matmul(a, b, dtype, status=status))
    assert status.item() == 0


@pytest.mark.parametrize("a_fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("b_fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("a_block, b_block", [(1, 1), (1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("m, n, k", [(40, 300, 900), (300, 40, 900), (260, 390, 520)])
def test_product_formats_and_blocks(m, n, k, a_fmt, b_fmt, a_block, b_block):
    a, b = operands(m, n, k, a_fmt, b_fmt, a_block, b_block)
    check(a, b, torch.float16, D.matmul(a, b, torch.float16))
    check(a, b, torch.float32, D.matmul(a, b, torch.float32))


@pytest.mark.parametrize("m, n, k", [(5, 300, 1100), (300, 5, 1100), (300, 500, 300)])
@pytest.mark.parametrize("pad", [0, 3, 4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_product_into_strided_rows_leaves_the_rest(m, n, k, pad, dtype):
    a, b = operands(m, n, k)
    buf = torch.full((m + 2, n + pad), 7.0, dtype=dtype, device="cuda")
    D.matmul(a, b, dtype, out=buf)
    check(a, b, dtype, buf[:m, :n])
    assert (buf[m:] == 7).all() and (buf[:, n:] == 7).all()


@pytest.mark.parametrize("m, n, k", [(3, 200, 3000), (200, 3, 3000), (400, 300, 500), (130, 140, 0)])
def test_product_accumulates(m, n, k):
    start = torch.randn(m, n, generator=torch.Generator().manual_seed(3))
    out = start.cuda()
    if k == 0:
        e = torch.empty(16, dtype=torch.uint8, device="cuda")
        for add, want in ((True, start), (False, start * 0)):
            sy.matmul_fp8_device(e.data_ptr(), e.data_ptr(), 0, 1, e.data_ptr(), e.data_ptr(), 0, 1, m, n, 0,
                                 out.data_ptr(), sy.SY_TYPE_F32, n, add, stream=D.stream())
            assert torch.equal(out.cpu(), want)
        return
    a, b = operands(m, n, k)
    D.matmul(a, b, torch.float32, out=out, accumulate=True)
    check(a, b, torch.float32, out, start)


# FP32 outputs of many tiles: 128, 192, 224 and 240 columns per tile, along the output's rows and across them.
@pytest.mark.parametrize("m, n, k", [(2853, 1452, 532), (658, 3364, 546), (3674, 972, 515), (3643, 1128, 653),
                                     (1721, 2139, 512), (537, 3733, 527), (790, 3834, 518), (2274, 1677, 644),
                                     (2274, 1676, 4700), (2274, 1677, 4700)])
def test_wide_products_in_fp32(m, n, k):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, b = operands(m, n, k)
    buf = torch.full((m + 1, n + 5), 7.0, device="cuda")
    D.matmul(a, b, torch.float32, out=buf, status=status)
    check(a, b, torch.float32, buf[:m, :n])
    D.matmul(a, b, torch.float32, out=buf, accumulate=True, status=status)
    assert (buf[m:] == 7).all() and (buf[:, n:] == 7).all() and status.item() == 0
    start = torch.randn(m, n, generator=torch.Generator().manual_seed(3))
    out = start.cuda()
    D.matmul(a, b, torch.float32, out=out, accumulate=True, status=status)
    check(a, b, torch.float32, out, start)
    assert status.item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("m, n, k", [(3785, 904, 527), (537, 3736, 527), (3883, 776, 538), (1552, 2480, 645),
                                     (1552, 2477, 645), (1000, 4096, 1300)])
def test_wide_products_in_16_bits(m, n, k, dtype):
    a, b = operands(m, n, k)
    buf = torch.full((m + 1, n + 8), 7.0, dtype=dtype, device="cuda")
    D.matmul(a, b, dtype, out=buf)
    check(a, b, dtype, buf[:m, :n])
    assert (buf[m:] == 7).all() and (buf[:, n:] == 7).all()


def test_product_is_the_same_every_time():
    a, b = operands(7, 900, 8000)
    first = D.matmul(a, b, torch.float32)
    for _ in range(5):
        assert torch.equal(D.matmul(a, b, torch.float32), first)


@pytest.mark.parametrize("m, n", [(4, 300), (300, 200)])
def test_nan_reaches_its_own_row_and_column_only(m, n):
    x, w = spread(m, 500, 1), spread(n, 500, 2)
    x[2, 77], w[5, 400] = float("nan"), float("nan")
    a, b = D.quantize(x.cuda(), "e4m3", 1), D.quantize(w.cuda(), "e4m3", 1)
    out = D.matmul(a, b, torch.float32).cpu()
    bad = torch.zeros(m, n, dtype=torch.bool)
    bad[2], bad[:, 5] = True, True
    assert torch.equal(out.isnan(), bad)


def test_unused_bytes_of_the_operands_do_not_matter():
    """Bytes past a row's end and scales past its last block hold anything."""
    a, b = operands(30, 140, 130)
    want = D.matmul(a, b, torch.float32)
    for h in (a, b):
        h.q[:, h.cols:] = 0x7f
        h.scale[:, -(-h.cols // 128):] = 0xff
    assert torch.equal(D.matmul(a, b, torch.float32), want)


def test_host_form():
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((50, 300)).astype(np.float32), rng.standard_normal((300, 70)).astype(np.float32)
    for fmt in ("e4m3", "e5m2"):
        qa, ea = D.cast_reference(torch.from_numpy(x), fmt, 1)
        qb, eb = D.cast_reference(torch.from_numpy(w.T.copy()), fmt, 128)
        va, vb = D.values(qa, ea, 1), D.values(qb, eb, 128)
        got = torch.from_numpy(sy.matmul_fp8(x, w, D.FORMATS[fmt][0])).double()
        assert ((got - va @ vb.T).abs() <= D.product_bound(va, vb, torch.float32, va @ vb.T)).all()


def test_host_pointers_are_refused():
    x = np.zeros((4, 256), np.float32)
    h = D.Held(4, 256, "e4m3", 1)
    with pytest.raises(sy.InvalidArgument, match="memory of the device"):
        sy.quantize_fp8_device(x.ctypes.data, sy.SY_TYPE_F32, 256, 4, 256, 0, 1, h.q.data_ptr(), h.scale.data_ptr())


def test_graph_replays_follow_their_inputs_and_streams():
    """Two captured chains (cast, product) on two streams, replayed with new inputs in the same buffers."""
    chains = []
    for seed in (1, 2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            x = spread(20, 700, seed).cuda()
            w = D.quantize(spread(300, 700, seed + 5).cuda(), "e4m3", 128)
            out = torch.empty(20, 300, device="cuda")
            D.matmul(D.quantize(x, "e4m3", 1), w, torch.float32, out=out)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                h = D.quantize(x, "e4m3", 1)
                D.matmul(h, w, torch.float32, out=out)
        chains.append((s, g, x, w, out, h))
    torch.cuda.synchronize()
    for turn in range(3):
        fresh = [spread(20, 700, 10 * turn + i).cuda() for i in range(2)]
        torch.cuda.synchronize()
        for (s, g, x, *_), f in zip(chains, fresh):
            with torch.cuda.stream(s):
                x.copy_(f)
                g.replay()
        torch.cuda.synchronize()
        for (_, _, x, w, out, h), f in zip(chains, fresh):
            assert torch.equal(out, D.matmul(D.quantize(f, "e4m3", 1), w, torch.float32))


def test_a_linear_layers_gradients_against_formula_and_differences():
    """y = x w^T in 8 bits with its three products, and differences of the loss sum(dy * y) of the cast operands:
    linear in each operand, so a difference is exact but for the rounding of its terms."""
    t, n, k = 96, 160, 200
    x, w, dy = spread(t, k, 1).cuda(), spread(n, k, 2).cuda() / 14, spread(t, n, 3).cuda()
    hx, hxt = D.quantize(x, "e4m3", 1, both=True)
    hw, hwt = D.quantize(w, "e4m3", 128, both=True)
    hd, hdt = D.quantize(dy, "e5m2", 1, both=True)
    y, dx, dw = D.matmul(hx, hw, torch.float32), D.matmul(hd, hwt, torch.float32), D.matmul(hdt, hxt, torch.float32)
    check(hx, hw, torch.float32, y)
    check(hd, hwt, torch.float32, dx)
    check(hdt, hxt, torch.float32, dw)
    vw, vd = hw.values(), hd.values()
    loss = lambda v: (vd * (v @ vw.T)).sum()
    vx = hx.values()
    bound = D.product_bound(vd, hwt.values(), torch.float32, vd @ vw)
    for i, j in [(0, 0), (50, 130), (95, 199)]:
        step = torch.zeros_like(vx)
        step[i, j] = 1.0
        diff = (loss(vx + step) - loss(vx - step)) / 2
        assert abs(dx[i, j].item() - diff) <= bound[i, j] + 1e-9 * loss(vx.abs()).abs()


# Long sums of one sign.  Accumulators truncate: an addition (32 products) loses at most 2 * 2^-23 of its partial sum.  They
# end after 16 blocks of K for FP32 results and at most 32 for 16-bit ones, 64 and 128 additions, whatever K is: at most
# 2^-16 and 2^-15 of the sum; adding up to K / (128 * 16) of them and eight splits rounds by 2^-24 each; then the output's rounding,
# half a step at the result's own size.
def long_sum_bound(k, dtype, want):
    full = dtype == torch.float32
    loss = (2.0 ** -16 if full else 2.0 ** -15) + (k / 2048 + 8) * 2.0 ** -24
    bits = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}[dtype]
    half_step = 2.0 ** (torch.floor(torch.log2(want)) - bits)
    if dtype == torch.float16:
        # f16's exponents end at -14: below 2^-14 (the smallest sums here are 9e-8) its values are multiples of 2^-24
        half_step = half_step.clamp(min=2.0 ** -25)
    return want * loss + half_step


def one_sign(rows, cols, seed, scale):
    return spread(rows, cols, seed).abs() * scale


def check_long(m, n, k, dtype, rows, accumulate=False):
    a = D.quantize(one_sign(m, k, 1, 2.0 ** -9).cuda(), "e4m3", 1)
    b = D.quantize(one_sign(n, k, 2, 2.0 ** -9).cuda(), "e4m3", 1)
    start = torch.rand(m, n, generator=torch.Generator().manual_seed(4)) if accumulate else None
    out = start.cuda() if accumulate else None
    got = D.matmul(a, b, dtype, out=out, accumulate=accumulate)[:rows].cpu().double()
    a.q, a.scale, a.rows = a.q[:rows], a.scale[:rows], rows
    want = a.values() @ b.values().T
    bound = long_sum_bound(k, dtype, want)
    if accumulate:
        want = want + start[:rows].double()
        bound = bound + 2.0 ** -24 * want
    assert want.max() < 60000
    assert ((got - want).abs() <= bound).all(), ((got - want) / want).mean()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n, k", [(4, 8, 1 << 21), (3, 40, 400000), (64, 576, 40960), (300, 300, 20001), (130, 1000, 20000),
                                     (1200, 1300, 9000)])
def test_long_sums_of_few_tiles_do_not_drift(m, n, k, dtype):
    check_long(m, n, k, dtype, min(m, 64))


@pytest.mark.parametrize("m, n, k", [(3, 40, 400000), (300, 301, 20001), (1200, 1300, 9000)])
def test_long_sums_of_few_tiles_added_to_the_output(m, n, k):
    check_long(m, n, k, torch.float32, min(m, 64), accumulate=True)


# 16-bit outputs of many tiles whose K is more than one accumulator takes: 128, 192, 224 and 240 columns per tile, along
# the output's rows and across them.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("m, n, k", [(1025, 3888, 4825), (3720, 520, 4750), (1167, 2712, 4948), (1158, 3176, 4821),
                                     (963, 3715, 4313), (3747, 522, 4940), (3736, 776, 4159), (776, 3755, 4628),
                                     (3718, 904, 4514), (909, 3718, 4883), (3204, 1208, 4217)])
def test_wide_products_of_long_sums_in_16_bits(m, n, k, dtype):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, b = operands(m, n, k)
    buf = torch.full((m + 1, n + 8), 7.0, dtype=dtype, device="cuda")
    D.matmul(a, b, dtype, out=buf, status=status)
    check(a, b, dtype, buf[:m, :n])
    assert (buf[m:] == 7).all() and (buf[:, n:] == 7).all() and status.item() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("m, n, k", [(2048, 2048, 65536), (2047, 2041, 65536), (2560, 2048, 8192)])
def test_long_sums_of_many_tiles_do_not_drift(m, n, k, dtype):
    check_long(m, n, k, dtype, 8)
