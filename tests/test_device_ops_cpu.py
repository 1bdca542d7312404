"""Refusals of the operators on device memory, checked before anything touches a GPU (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

import simdyolo_b200 as sy

P = 1 << 20   # a well-aligned address that the refused calls never reach


def quantize(**kw):
    a = dict(x=P, x_type=sy.SY_TYPE_BF16, x_pitch=256, rows=4, cols=256, fmt=sy.SY_FP8_E4M3, block_rows=1, q=P, scale=P,
             qt=0, scale_t=0)
    a.update(kw)
    sy.quantize_fp8_device(**a)


def dequantize(**kw):
    a = dict(q=P, scale=P, rows=4, cols=256, fmt=sy.SY_FP8_E5M2, block_rows=128, out=P, out_type=sy.SY_TYPE_F32,
             out_pitch=256)
    a.update(kw)
    sy.dequantize_fp8_device(**a)


def matmul(**kw):
    a = dict(a=P, a_scale=P, a_fmt=sy.SY_FP8_E4M3, a_block_rows=1, b=P, b_scale=P, b_fmt=sy.SY_FP8_E4M3,
             b_block_rows=128, m=16, n=32, k=256, out=P, out_type=sy.SY_TYPE_BF16, out_pitch=32)
    a.update(kw)
    sy.matmul_fp8_device(**a)


def orthogonalize(**kw):
    a = dict(x=P, x_type=sy.SY_TYPE_F32, x_pitch=64, rows=32, cols=64, steps=5, out=P, out_type=sy.SY_TYPE_BF16,
             out_pitch=64, workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    sy.orthogonalize_device(**a)


def muon(entry=(P, P, P, 32, 64), bytes=1 << 30, workspace=P, **kw):
    sy.muon_update_device(sy.muon_tensors([entry]), sy.muon_options(**{"lr": 0.02, **kw}), workspace, bytes)


@pytest.mark.parametrize("call, kw, match", [
    (quantize, dict(x_type=7), "element type"),
    (quantize, dict(rows=-1), "negative"),
    (quantize, dict(x_pitch=255), "pitch"),
    (quantize, dict(x_pitch=1 << 62), "pitch"),
    (quantize, dict(fmt=2), "format"),
    (quantize, dict(block_rows=64), "block_rows"),
    (quantize, dict(qt=P), "together"),
    (quantize, dict(scale_t=P), "together"),
    (quantize, dict(x=0), "null"),
    (quantize, dict(x=P + 1), "aligned"),
    (quantize, dict(q=P + 8), "aligned"),
    (quantize, dict(scale=P + 2), "aligned"),
    (quantize, dict(qt=P + 4, scale_t=P), "aligned"),
    (dequantize, dict(q=0), "null"),
    (dequantize, dict(out_type=-1), "element type"),
    (dequantize, dict(out=P + 2), "aligned"),
    (dequantize, dict(out_pitch=128), "pitch"),
    (dequantize, dict(block_rows=0), "block_rows"),
    (matmul, dict(m=-1), "negative"),
    (matmul, dict(k=-1), "negative"),
    (matmul, dict(out_pitch=31), "pitch"),
    (matmul, dict(accumulate=True), "accumulate"),
    (matmul, dict(a=P + 8), "aligned"),
    (matmul, dict(b_scale=P + 1), "aligned"),
    (matmul, dict(b=0), "null"),
    (matmul, dict(out=0), "null"),
    (matmul, dict(a_fmt=5), "format"),
    (matmul, dict(b_block_rows=32), "block_rows"),
    (matmul, dict(status=P + 2), "aligned"),
    (orthogonalize, dict(steps=0), "steps"),
    (orthogonalize, dict(steps=17), "steps"),
    (orthogonalize, dict(workspace_bytes=1000), "workspace too small"),
    (orthogonalize, dict(workspace=0), "null"),
    (orthogonalize, dict(x=P + 2), "aligned"),
    (orthogonalize, dict(out_pitch=63), "pitch"),
    (orthogonalize, dict(out_type=3), "element type"),
    (muon, dict(lr=float("nan")), "finite"),
    (muon, dict(lr=-1.0), "hyper"),
    (muon, dict(momentum=1.0), "hyper"),
    (muon, dict(steps=0), "steps"),
    (muon, dict(precision=9), "precision"),
    (muon, dict(bytes=100), "workspace too small"),
    (muon, dict(workspace=0), "null"),
    (muon, dict(entry=(P, 0, P, 32, 64)), "null"),
    (muon, dict(entry=(P, P, P + 2, 32, 64)), "aligned"),
    (muon, dict(entry=(P, P, P, -1, 64)), "negative"),
])
def test_bad_arguments_are_refused(call, kw, match):
    with pytest.raises(sy.InvalidArgument, match=match):
        call(**kw)


def test_matrices_past_the_tile_counts_are_unsupported():
    with pytest.raises(sy.UnsupportedShape):
        orthogonalize(rows=1 << 21, cols=1 << 21, x_pitch=1 << 21, out_pitch=1 << 21, workspace_bytes=1 << 62)


@pytest.mark.parametrize("call, kw", [
    (quantize, dict(rows=(1 << 30) + 1, cols=1)),
    (quantize, dict(rows=1 << 28, cols=129)),
    (quantize, dict(rows=1, cols=(1 << 31) - 1, x_pitch=1 << 31)),
    (quantize, dict(rows=33, cols=3 << 28, x_pitch=3 << 28, block_rows=128, qt=P, scale_t=P)),
    (dequantize, dict(rows=(1 << 31) - 1)),
    (dequantize, dict(rows=1 << 28, cols=256)),
    (matmul, dict(k=(1 << 31) - 1)),
    (matmul, dict(m=(1 << 30) + 1, n=1)),
    (matmul, dict(m=1 << 20, k=1 << 16)),
    (matmul, dict(n=1 << 20, k=1 << 16, out_pitch=1 << 20)),
])
def test_8_bit_matrices_past_32_bit_counts_are_unsupported(call, kw):
    with pytest.raises(sy.UnsupportedShape, match="too large"):
        call(**kw)


def test_muon_tensors_that_share_memory_are_refused():
    n = 32 * 64 * 4

    def step(*entries):
        t = sy.muon_tensors([(w, m, g, 32, 64) for w, m, g in entries])
        sy.muon_update_device(t, sy.muon_options(0.02), P, 1 << 30)

    for entries in ([(P, P + n, P + 2 * n)] * 2,
                    [(P, P + n, P + 2 * n), (P + 3 * n, P + 4 * n, P + n - 4)],
                    [(P, P + n, P)], [(P, P, P + n)], [(P, P + n - 4, P + 4 * n)],
                    [(P + 9 * n, P + 8 * n, P + 7 * n), (P, P + n, P + 9 * n + 4)]):
        with pytest.raises(sy.InvalidArgument, match="share memory"):
            step(*entries)


def test_empty_calls_need_no_memory():
    quantize(rows=0, x=0, q=0, scale=0)
    dequantize(cols=0, q=0, scale=0, out=0)
    matmul(m=0, a=0, a_scale=0, out=0)
    orthogonalize(rows=0, x=0, out=0, workspace=0, workspace_bytes=0)
    muon(entry=(0, 0, 0, 0, 64), workspace=0, bytes=0)
    sy.muon_update_device(sy.muon_tensors([]), sy.muon_options(0.02), 0, 0)


def test_options_of_another_size_are_refused():
    o = sy.muon_options(0.02)
    o.struct_size -= 4
    with pytest.raises(sy.InvalidArgument, match="options"):
        sy.muon_update_device(sy.muon_tensors([]), o, 0, 0)
    assert sy.muon_workspace(sy.muon_tensors([(P, P, P, 8, 8)]), o) == 0


@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 16), (129, 17), (256, 4096), (5, 513)])
def test_layout_sizes(rows, cols):
    L = sy.lib()
    assert L.sy_cuda_fp8_bytes(rows, cols) == rows * sy.fp8_pitch(cols)
    assert sy.fp8_pitch(cols) % 16 == 0 and 0 <= sy.fp8_pitch(cols) - cols < 16
    for block in (1, 128):
        assert L.sy_cuda_fp8_scale_bytes(rows, cols, block) == -(-rows // block) * sy.fp8_scale_pitch(cols)
    assert L.sy_cuda_fp8_scale_bytes(rows, cols, 64) == 0


def test_workspaces_grow_with_the_matrix_and_with_the_precision():
    single = sy.orthogonalize_workspace(256, 512, sy.SY_TYPE_BF16)
    assert 0 < sy.orthogonalize_workspace(64, 576, sy.SY_TYPE_BF16) < single < sy.orthogonalize_workspace(256, 512, sy.SY_TYPE_F32)
    assert single == sy.orthogonalize_workspace(512, 256, sy.SY_TYPE_BF16)
    one = sy.muon_tensors([(P, P, P, 256, 512)])
    two = sy.muon_tensors([(P, P, P, 256, 512)] * 2)
    o = sy.muon_options(0.02)
    assert sy.muon_workspace(one, o) < sy.muon_workspace(two, o)
    assert sy.muon_workspace(one, sy.muon_options(0.02, precision=sy.SY_PRECISION_TF32)) < sy.muon_workspace(one, o)


def test_host_forms_refuse_bad_arguments():
    w = np.zeros((4, 4), np.float32)
    with pytest.raises(sy.InvalidArgument):
        sy.matmul_fp8(w, w, fmt=3)
    with pytest.raises(sy.InvalidArgument):
        sy.muon_update(w, w.copy(), w.copy(), sy.muon_options(0.02, steps=99))
    L = sy.lib()
    assert L.sy_cuda_muon_update(0, None, None, None, 4, 4, C.byref(sy.muon_options(0.02))) == sy.SY_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("rows, cols", [(1, 1 << 26), (1, 1 << 27), (16, 1 << 26), (128, 1 << 24), (128, (1 << 24) + 64),
                                        (1 << 26, 5), (1, 1 << 30)])
def test_workspaces_of_very_long_matrices_hold_their_operands(rows, cols):
    """Two X of fp16 pairs, 128 rows at least: such a matrix is too long to stay on chip, whatever its row count."""
    need = 2 * 128 * max(rows, cols) * 4
    for out in (sy.SY_TYPE_F32, sy.SY_TYPE_BF16):
        assert sy.orthogonalize_workspace(rows, cols, out) >= need
        with pytest.raises(sy.InvalidArgument, match="workspace too small"):
            orthogonalize(rows=rows, cols=cols, x_pitch=cols, out_pitch=cols, out_type=out, workspace_bytes=need - 1)
    t = sy.muon_tensors([(P, P, P, rows, cols)])
    assert sy.muon_workspace(t, sy.muon_options(0.02)) >= need
    assert sy.muon_workspace(t, sy.muon_options(0.02, precision=sy.SY_PRECISION_TF32)) >= need // 2


@pytest.mark.parametrize("rows, cols", [(1, (1 << 31) - 1), ((1 << 31) - 64, 1), (3, (1 << 30) + 1)])
def test_matrices_past_32_bit_columns_are_unsupported(rows, cols):
    with pytest.raises(sy.UnsupportedShape):
        orthogonalize(rows=rows, cols=cols, x_pitch=cols, out_pitch=cols, workspace_bytes=1 << 62)
    with pytest.raises(sy.UnsupportedShape):
        muon(entry=(P, P, P, rows, cols), bytes=1 << 62)
    assert sy.orthogonalize_workspace(rows, cols, sy.SY_TYPE_F32) == 0
    assert sy.muon_workspace(sy.muon_tensors([(P, P, P, rows, cols)]), sy.muon_options(0.02)) == 0


def test_host_forms_refuse_arrays_that_the_library_would_misread():
    """Nothing reaches the library, which sees addresses and sizes only."""
    w = np.zeros((4, 6), np.float32)
    for a, b in ((w, w), (w, np.zeros((5, 4), np.float32)), (w[0], w), (w, w[0])):
        with pytest.raises(sy.InvalidArgument, match="multiply"):
            sy.matmul_fp8(a, b)
    o = sy.muon_options(0.02)
    for bad in (w.astype(np.float64), w[:, ::2], w.T, w[:2].copy(), w.ravel(), np.zeros((8, 6), np.float32)[::2]):
        for args in ((bad, w, w), (w, bad, w), (w, w, bad)):
            with pytest.raises(sy.InvalidArgument, match="contiguous"):
                sy.muon_update(*args, o)
