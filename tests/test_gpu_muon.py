"""Newton-Schulz orthogonalisation and the Muon step on the GPU against their definitions in 64 bits.

Tolerances (relative 2-norm of a whole matrix).  22-bit operands: an iteration's three products each round two
operands to 2^-22 and drop lo * lo (2^-22), so five iterations are within 5 * 3 * 3 * 2^-22 = 1.1e-5 in the
directions whose singular values the iteration flattens, which hold nearly all of a random matrix's norm; twice
that covers the FP32 accumulation.  11-bit operands: the same count with 2^-11 / 2 per rounding (no dropped term)
is 5 * 3 * 2 * 2^-12 = 7.3e-3.  Outputs add half a step of their type.
"""
import numpy as np
import pytest
import torch

import simdyolo_b200 as sy
from tests import device_ops as D

pytestmark = pytest.mark.gpu
SPLIT_TOL, SINGLE_TOL = 2.2e-5, 7.3e-3


def update(rows, cols, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    k = min(8, rows, cols)
    low = torch.randn(rows, k, generator=g) @ torch.randn(k, cols, generator=g)
    return (1e-3 * (low + torch.randn(rows, cols, generator=g))).to(dtype)


SHAPES = [(1, 1), (1, 300), (300, 1), (2, 2), (17, 5), (64, 576), (80, 720), (127, 129), (128, 128), (129, 640),
          (576, 64), (700, 333), (130, 2304), (512, 512), (129, 129), (128, 3000), (4500, 140), (300, 9000), (1100, 1030),
          (3500, 3400)]


@pytest.mark.parametrize("rows, cols", SHAPES)
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_orthogonalize_shapes(rows, cols, out):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    u = update(rows, cols, rows + cols)
    got = D.orthogonalize(u.cuda(), out, status=status)
    tol = SPLIT_TOL if out == torch.float32 else SINGLE_TOL + D.HALF_STEP[out]
    assert D.rel(got, D.orthogonal_reference(u)) <= tol
    assert status.item() == 0


# Where the products run on pairs a 16-bit result is the FP32 one rounded: SPLIT_TOL plus half a step.
@pytest.mark.parametrize("rows, cols, out", [(r, c, t) for r, c in ((2, 2), (4, 2), (9, 9), (33, 2000), (64, 64), (576, 64))
                                             for t in (torch.bfloat16, torch.float16)] +
                         [(r, c, torch.float16) for r, c in ((65, 65), (128, 300), (700, 333))])
def test_orthogonalize_rounds_once(rows, cols, out):
    for seed in range(4):
        u = update(rows, cols, seed)
        assert D.rel(D.orthogonalize(u.cuda(), out), D.orthogonal_reference(u)) <= SPLIT_TOL + D.HALF_STEP[out]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows, cols", [(64, 200), (200, 64)])
def test_orthogonalize_reads_types_and_strides_and_leaves_padding(dtype, rows, cols):
    base = torch.zeros(rows, cols + 13, dtype=dtype)
    base[:, 1:cols + 1] = update(rows, cols, 4).to(dtype)
    x = base.cuda()[:, 1:cols + 1]
    got = D.orthogonalize(x, torch.float32, pitch=cols + 3)
    assert D.rel(got[:, :cols], D.orthogonal_reference(base[:, 1:cols + 1])) <= SPLIT_TOL
    assert (got[:, cols:] == 7).all()


@pytest.mark.parametrize("steps", [1, 2, 3, 6])
def test_orthogonalize_steps(steps):
    u = update(90, 150, 1)
    assert D.rel(D.orthogonalize(u.cuda(), torch.float32, steps), D.orthogonal_reference(u, steps)) <= SPLIT_TOL


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30, 3e37])
def test_orthogonalize_does_not_depend_on_the_scale(scale):
    u = update(100, 180, 2).double() * 1e3
    u = (u / u.abs().max() * scale).float()
    assert D.rel(D.orthogonalize(u.cuda(), torch.float32), D.orthogonal_reference(u)) <= SPLIT_TOL


def test_orthogonalize_of_zero_and_of_values_that_are_not_finite():
    z = torch.zeros(70, 90, device="cuda")
    for out in (torch.float32, torch.bfloat16):
        assert (D.orthogonalize(z, out) == 0).all()
    for v in (float("nan"), float("inf")):
        z[3, 4] = v
        assert D.orthogonalize(z, torch.bfloat16).isnan().all()


def test_orthogonalize_a_few_strong_directions():
    """A matrix of rank 3 (its other singular values are zero) and one diagonal matrix with a wide spectrum."""
    g = torch.Generator().manual_seed(0)
    low = torch.randn(200, 3, generator=g) @ torch.randn(3, 300, generator=g)
    diag = torch.diag(2.0 ** -torch.arange(64, dtype=torch.float32))
    # the null directions of `low` hold only its own FP32 rounding (2^-24), which the iteration raises 485 times
    assert D.rel(D.orthogonalize(low.cuda(), torch.float32), D.orthogonal_reference(low)) <= SPLIT_TOL + 485 * 2.0 ** -22
    assert D.rel(D.orthogonalize(diag.cuda(), torch.float32), D.orthogonal_reference(diag)) <= SPLIT_TOL


def lists(shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = [torch.randn(r, c, generator=g) / c ** 0.5 for r, c in shapes]
    m = [update(r, c, seed + i) for i, (r, c) in enumerate(shapes)]
    d = [update(r, c, seed + 100 + i) for i, (r, c) in enumerate(shapes)]
    return w, m, d


def check_muon(shapes, opts, options, tol_o, seed=0):
    w, m, d = lists(shapes, seed)
    cw, cm, cd = ([x.cuda() for x in v] for v in (w, m, d))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    keep = D.muon(cw, cm, cd, options, status)
    for i in range(len(shapes)):
        want_w, want_m = D.muon_reference(w[i], m[i], d[i], **opts)
        # the step may be off by tol_o of itself, the weight by two FP32 roundings
        step = (want_w - w[i].double() * (1 - opts["lr"] * opts.get("weight_decay", 0.0))).norm()
        off = (cw[i].cpu().double() - want_w).norm()
        assert off <= tol_o * step + 3 * 2.0 ** -24 * (want_w.norm() + step), shapes[i]
        assert D.rel(cm[i], want_m) <= 3 * 2.0 ** -24
        assert torch.equal(cd[i].cpu(), d[i])
    assert status.item() == 0
    return keep


@pytest.mark.parametrize("opts", [
    dict(lr=0.02), dict(lr=0.02, momentum=0.9, weight_decay=0.1, nesterov=False),
    dict(lr=0.5, momentum=0.0, rms=1.0, grad_scale=0.125, steps=3)])
@pytest.mark.parametrize("precision, tol", [(sy.SY_PRECISION_3XTF32, SPLIT_TOL), (sy.SY_PRECISION_TF32, SINGLE_TOL)])
def test_muon_list(opts, precision, tol):
    shapes = [(64, 576), (1, 7), (300, 40), (80, 80), (129, 130), (5, 1)]
    check_muon(shapes, opts, sy.muon_options(precision=precision, **opts), tol)


@pytest.mark.parametrize("shapes", [[(8 + i, 200 - 2 * i) for i in range(70)], [(130 + i, 140 + 3 * i) for i in range(37)],
                                    [(130 + 40 * (i % 2), 60 + 37 * i) for i in range(40)], [(900, 1300), (1000, 2049), (2000, 300)]])
def test_muon_of_longer_lists_and_larger_matrices(shapes):
    check_muon(shapes, dict(lr=0.02), sy.muon_options(0.02), SPLIT_TOL)


def test_muon_list_equals_its_matrices_one_by_one():
    shapes = [(64, 300), (150, 70), (256, 256)]
    w, m, d = lists(shapes, 9)
    o = sy.muon_options(0.02)
    cw, cm, cd = ([x.cuda() for x in v] for v in (w, m, d))
    keep = [D.muon(cw, cm, cd, o)]
    for i in range(3):
        a, b = w[i].cuda(), m[i].cuda()
        keep.append(D.muon([a], [b], [cd[i]], o))
        assert torch.equal(a, cw[i]) and torch.equal(b, cm[i])


def test_muon_skips_empty_matrices_and_reports_values_that_are_not_finite():
    w, m, d = ([x.cuda() for x in v] for v in lists([(16, 20), (30, 8)], 3))
    e = torch.zeros(0, 4, device="cuda")
    d[1][3, 3] = float("inf")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    keep = D.muon([w[0], e, w[1]], [m[0], e, m[1]], [d[0], e, d[1]], sy.muon_options(0.02), status)
    assert status.item() == sy.SY_ERR_NONFINITE
    assert w[0].isfinite().all() and w[1].isnan().all()
    del keep


@pytest.mark.parametrize("shapes", [[(64, 200), (100, 60)], [(200, 300), (64, 200), (140, 131)]])
def test_graphs_with_their_own_workspaces_replay_side_by_side(shapes):
    o = sy.muon_options(0.02, weight_decay=0.01)
    runs = []
    for seed in (1, 2):
        w, m, d = ([x.cuda() for x in v] for v in lists(shapes, seed))
        t = sy.muon_tensors([(a.data_ptr(), b.data_ptr(), c.data_ptr(), *a.shape) for a, b, c in zip(w, m, d)])
        work = torch.empty(sy.muon_workspace(t, o), dtype=torch.uint8, device="cuda")
        s = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            sy.muon_update_device(t, o, work.data_ptr(), work.numel(), stream=torch.cuda.current_stream().cuda_stream)
        runs.append((s, g, w, m, d, work, t))
    del t   # the list is read during the call
    eager = [[[x.clone() for x in v] for v in r[2:5]] for r in runs]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, g, *_ in runs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for r, (w, m, d) in zip(runs, eager):
        keep = [D.muon(w, m, d, o) for _ in range(3)]
        torch.cuda.synchronize()
        for a, b in zip(r[2], w):
            assert torch.equal(a, b)
        del keep


def test_workspace_of_any_alignment():
    w, m, d = ([x.cuda() for x in v] for v in lists([(50, 90)], 5))
    w2, m2 = w[0].clone(), m[0].clone()
    o = sy.muon_options(0.02)
    keep = D.muon(w, m, d, o)
    t = sy.muon_tensors([(w2.data_ptr(), m2.data_ptr(), d[0].data_ptr(), 50, 90)])
    need = sy.muon_workspace(t, o)
    work = torch.full((need + 77,), 0x7f, dtype=torch.uint8, device="cuda")
    sy.muon_update_device(t, o, work.data_ptr() + 7, need, stream=D.stream())
    assert torch.equal(w2, w[0])
    assert (work[:7] == 0x7f).all() and (work[7 + need:] == 0x7f).all()
    del keep


def test_host_form_matches_the_device_form():
    w, m, d = lists([(60, 100)], 6)
    o = sy.muon_options(0.02, weight_decay=0.05)
    cw, cm = w[0].cuda(), m[0].cuda()
    keep = D.muon([cw], [cm], [d[0].cuda()], o)
    hw, hm, hg = (x[0].numpy().copy() for x in (w, m, d))
    sy.muon_update(hw, hm, hg, o)
    assert np.array_equal(hw, cw.cpu().numpy()) and np.array_equal(hm, cm.cpu().numpy())
    hg[0, 0] = np.nan
    with pytest.raises(sy.NonFinite):
        sy.muon_update(hw, hm, hg, o)
    del keep


def test_an_8_bit_layer_trained_by_muon():
    """Forward, backward and update as a training step runs them, on one stream, against the same in 64 bits."""
    t, n, k = 256, 160, 192
    g = torch.Generator().manual_seed(1)
    x, target = torch.randn(t, k, generator=g), torch.randn(t, n, generator=g)
    w, m = torch.randn(n, k, generator=g) / k ** 0.5, torch.zeros(n, k)
    cx, ct, cw, cm = x.cuda(), target.cuda(), w.cuda(), m.cuda()
    o = sy.muon_options(0.02)
    keep = []
    for _ in range(3):
        hx, hxt = D.quantize(cx, "e4m3", 1, both=True)
        y = D.matmul(hx, D.quantize(cw, "e4m3", 128), torch.float32)
        hd, hdt = D.quantize(y - ct, "e5m2", 1, both=True)
        dw = D.matmul(hdt, hxt, torch.float32)
        before, mom = cw.cpu(), cm.cpu()
        keep.append(D.muon([cw], [cm], [dw], o))
        want, want_m = D.muon_reference(before, mom, dw.cpu(), 0.02)
        step = (want - before.double()).norm()
        assert (cw.cpu().double() - want).norm() <= SPLIT_TOL * step + 3 * 2.0 ** -24 * (want.norm() + step)
        assert D.rel(cm, want_m) <= 3 * 2.0 ** -24
        want_dw = hdt.values() @ hxt.values().T
        assert ((dw.cpu().double() - want_dw).abs() <= D.product_bound(hdt.values(), hxt.values(), torch.float32, want_dw)).all()


def spectrum(rows, cols, kind, seed=0):
    """A matrix whose singular values fall over three decades, as 1 / i^2, or from eight equal ones to 1 % of them."""
    g = torch.Generator().manual_seed(seed)
    basis = lambda n: torch.linalg.qr(torch.randn(n, n, generator=g, dtype=torch.float64))[0]
    k = min(rows, cols)
    i = torch.arange(k, dtype=torch.float64)
    s = {"decades": 10.0 ** (-3 * i / (k - 1)), "squares": 1 / (i + 1) ** 2,
         "eight": torch.where(i < 8, 1.0, 0.01).double()}[kind]
    return ((basis(rows)[:, :k] * s) @ basis(cols)[:, :k].T).float()


# The weak directions of such a matrix carry the operands' roundings, raised up to 485 times.  An operand of 22 bits is off
# by at most 2^-21 of its size (2^-22 for the pair, as much for the dropped lo lo), which orthogonal_bound follows through
# the iterations; a 16-bit result is the FP32 result rounded, bit for bit.
@pytest.mark.parametrize("kind", ["decades", "squares", "eight"])
@pytest.mark.parametrize("rows, cols", [(65, 65), (128, 300), (300, 128), (129, 129), (700, 333), (256, 512)])
def test_orthogonalize_of_steep_spectra_rounds_once(rows, cols, kind):
    u = spectrum(rows, cols, kind)
    want = D.orthogonal_reference(u)
    full = D.orthogonalize(u.cuda(), torch.float32)
    assert (full.cpu().double() - want).norm() <= D.orthogonal_bound(u, 2.0 ** -21)
    for out in (torch.bfloat16, torch.float16):
        assert torch.equal(D.orthogonalize(u.cuda(), out), full.to(out))


@pytest.mark.parametrize("rows, cols, steps", [(130, 140, 1), (260, 700, 2), (900, 200, 3), (400, 400, 4), (300, 2000, 16)])
def test_bf16_results_of_tiled_matrices_are_the_fp32_ones_rounded(rows, cols, steps):
    u = update(rows, cols, 3).cuda()
    assert torch.equal(D.orthogonalize(u, torch.bfloat16, steps, pitch=cols + 5)[:, :cols],
                       D.orthogonalize(u, torch.float32, steps).bfloat16())


@pytest.mark.parametrize("rows, cols", [(3, 2000003), (1500001, 2)])
def test_orthogonalize_very_long_matrices(rows, cols):
    u = update(rows, cols, 11)
    assert D.rel(D.orthogonalize(u.cuda(), torch.float32), D.orthogonal_reference(u)) <= SPLIT_TOL


@pytest.mark.parametrize("shapes", [[(128, 1024)] + [(128, 320)] * 31, [(128, 1024)] * 8 + [(320, 128)] * 24,
                                    [(128, 1024)] * 15 + [(128, 320)] * 4, [(16, 64)] * 32 + [(120, 300)] * 32])
def test_muon_lists_whose_matrices_fit_one_or_four_ctas_but_not_two(shapes):
    """128 x 320 takes 230,400 bytes of shared memory on one CTA and 232,448 on two, which need room for an exchange."""
    check_muon(shapes, dict(lr=0.02), sy.muon_options(0.02), SPLIT_TOL)


@pytest.mark.parametrize("shape", [(64, 200), (200, 300)])
def test_a_report_of_an_earlier_call_is_kept(shape):
    """Calls that share a status word: a value that is not finite does not hide an earlier SY_ERR_DEVICE."""
    w, m, d = ([x.cuda() for x in v] for v in lists([shape], 3))
    d[0][1, 1] = float("nan")
    for before, after in ((0, sy.SY_ERR_NONFINITE), (sy.SY_ERR_DEVICE, sy.SY_ERR_DEVICE)):
        status = torch.full((1,), before, dtype=torch.int32, device="cuda")
        keep = D.muon(w, m, d, sy.muon_options(0.02), status)
        assert status.item() == after
        del keep


# ------------------------------------------------------------------ 11-bit operands (SY_PRECISION_TF32)

def orthogonal_in_fp16(u, steps=5):
    """The iteration in 64 bits with X, A and B rounded to fp16 as the kernels hold them: X times a power of two that puts
    its entries near 1 (at most 2^15), A and B times 2^14."""
    x = u.double()
    if x.shape[0] > x.shape[1]:
        return orthogonal_in_fp16(u.T, steps).T
    p = 2.0 ** min(15, int(np.floor(0.5 * np.log2(x.numel()))))
    half = lambda v, f: (v * f).half().double() / f
    x = half(x / x.norm(), p)
    for i in range(steps):
        a = half(x @ x.T, 2.0 ** 14)
        b = half(D.NS[1] * a + D.NS[2] * (a @ a), 2.0 ** 14)
        x = D.NS[0] * x + b @ x
        if i + 1 < steps:
            x = half(x, p)
    return x


# Kernel and restatement round at the same places, so they differ where a sum that the tensor core forms in FP32 (off by
# d = 2^-20 of itself at most: 512 products of 11-bit values at K = 512, half a place of 2^-24 lost per 16) falls on the
# other side of a rounding.  That happens with probability d / step (step 2^-10 of the value) and costs a step: a
# root-mean-square error of sqrt(d * step) = 2^-15 per operand, which orthogonal_bound follows through the iterations
# at the steepest slope.  The bound has to leave an update without its orthogonalisation (error 1) far outside.
@pytest.mark.parametrize("kind", ["decades", "squares", "eight", "white"])
@pytest.mark.parametrize("rows, cols", [(64, 64), (64, 576), (80, 720), (120, 50), (200, 300), (300, 140)])
def test_muon_in_11_bits_follows_its_roundings(rows, cols, kind):
    u = update(rows, cols, 5) if kind == "white" else spectrum(rows, cols, kind)
    want = orthogonal_in_fp16(u)
    w, m = torch.zeros(rows, cols, device="cuda"), torch.zeros(rows, cols, device="cuda")
    o = sy.muon_options(1.0, momentum=0.0, rms=max(rows, cols) ** -0.5, precision=sy.SY_PRECISION_TF32)
    keep = D.muon([w], [m], [u.cuda()], o)
    off, bound = (-w.cpu().double() - want).norm(), D.orthogonal_bound(u, 2.0 ** -15)
    assert bound < 0.15 * want.norm()
    assert off <= bound, off / want.norm()
    del keep
