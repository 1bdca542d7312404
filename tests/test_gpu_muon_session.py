"""SY_OPT_MUON: sessions whose dense conv weights step by Muon and whose other parameters step by AdamW.

The step's own gradients are taken as given (their parity is other tests' subject) and both update rules applied to
them in 64 bits.  These gradients have steep spectra, whose weak directions the iteration raises up to 3.4445^5 = 485
times, so the orthogonalisation is held to its worst-case bound (device_ops.orthogonal_bound) at half a step of
fp16 (2^-11) per operand, or 2^-21 for pairs of fp16 values; weights also differ by a few FP32 roundings.
"""
import numpy as np
import pytest
import torch

import simdyolo_b200 as sy
from simdyolo_b200 import data
from tests import device_ops as D

pytestmark = pytest.mark.gpu
LR, DECAY = 2e-3, 0.05


def session(model="yolov8n", batch=2, backbone=False, **kw):
    cfg = sy.make_config(model, image_size=128, max_batch=batch, max_boxes=20, backbone=backbone, lr=LR,
                         weight_decay=DECAY, optimizer=sy.SY_OPT_MUON, **kw)
    s = sy.Session(cfg)
    params, buffers = data.head_params(s, 2)
    s.set_flat_params(params)
    s.set_flat_buffers(buffers)
    return s, cfg


def features(cfg, batch, rng):
    sizes = [cfg.image_size >> (3 + l) for l in range(3)]
    return [(rng.standard_normal((batch, cfg.feature_channels[l], h, h)) * 0.7 + 0.2).astype(np.float32)
            for l, h in enumerate(sizes)]


def is_muon(t, dense):
    return len(t["shape"]) == 4 and dense(t)


@pytest.mark.parametrize("model", ["yolov8n", "yolo11s"])
@pytest.mark.parametrize("precision, unit", [(sy.SY_PRECISION_TF32, 2.0 ** -11), (sy.SY_PRECISION_3XTF32, 2.0 ** -21)])
def test_steps_follow_both_rules(model, precision, unit):
    rng = np.random.default_rng(7)
    s, cfg = session(model, precision=precision)
    dense = lambda t: t["shape"][1] > 1   # the depthwise weights are [channels, 1, 3, 3]
    steps = {0: 0, 1: 0}
    for k in range(3):
        truth = [[], []] if k == 1 else data.synthetic_batch(rng, 2, 128, cfg.num_classes, boxes=(1, 20), wh=(8.0, 64.0))[1]
        before = [s.get_tensor(t["index"]).astype(np.float64) for t in s.params]
        m1 = [s.get_optimizer_state(t["index"], 0).astype(np.float64) for t in s.params]
        m2 = [s.get_optimizer_state(t["index"], 1).astype(np.float64) for t in s.params]
        stats = s.step_features(features(cfg, 2, rng), truth)
        grad = s.last_gradients().astype(np.float64)
        assert stats.box_has_grad == (k != 1)
        for group in (0, 1):
            steps[group] += int(group == 0 or stats.box_has_grad)
        off = 0
        for t, w, a, b in zip(s.params, before, m1, m2):
            n = t["numel"]
            g = grad[off:off + n] / 2
            off += n
            now = s.get_tensor(t["index"]).astype(np.float64)
            moments = [s.get_optimizer_state(t["index"], m).astype(np.float64) for m in (0, 1)]
            group = sy.tensor_group(t["name"])
            if group == 1 and not stats.box_has_grad:
                assert np.array_equal(now, w) and np.array_equal(moments[0], a) and np.array_equal(moments[1], b)
                continue
            if is_muon(t, dense):
                mat = lambda v: torch.from_numpy(v.reshape(t["shape"][0], -1).copy())
                want, want_m = D.muon_reference(mat(w), mat(a), mat(g), LR, cfg.momentum, DECAY)
                want, want_m = want.numpy().ravel(), want_m.numpy().ravel()
                assert not moments[1].any()
                u = mat(g) + cfg.momentum * torch.from_numpy(want_m.reshape(t["shape"][0], -1))
                near = LR * 0.2 * max(u.shape) ** 0.5 * D.orthogonal_bound(u, unit)
            else:
                want_m = cfg.beta1 * a + (1 - cfg.beta1) * g
                want_v = cfg.beta2 * b + (1 - cfg.beta2) * g * g
                c1, c2 = 1 - cfg.beta1 ** steps[group], 1 - cfg.beta2 ** steps[group]
                decay = DECAY if len(t["shape"]) == 4 else 0.0
                want = w.ravel() * (1 - LR * decay) - LR / c1 * want_m / (np.sqrt(want_v) / np.sqrt(c2) + cfg.adam_eps)
                assert np.linalg.norm(moments[1] - want_v) <= 1e-6 * np.linalg.norm(want_v)
                # AdamW in FP32: bias corrections by powf, a quotient and a root
                near = 1e-5 * np.linalg.norm(want - w.ravel())
            assert np.linalg.norm(moments[0] - want_m) <= 1e-6 * np.linalg.norm(want_m)
            assert np.linalg.norm(now.ravel() - want) <= near + 4 * 2.0 ** -24 * np.linalg.norm(want), t["name"]
        assert s.optimizer_steps()[:2] == [steps[0], steps[1]]
    s.close()


def run(s, cfg, seed, count):
    rng = np.random.default_rng(seed)
    for _ in range(count):
        feats = features(cfg, 2, rng)
        s.step_features(feats, data.synthetic_batch(rng, 2, 128, cfg.num_classes, boxes=(1, 20), wh=(8.0, 64.0))[1])


def test_resume_continues_bit_identical():
    a, cfg = session()
    run(a, cfg, 1, 2)
    state = ([a.get_tensor(t["index"]) for t in a.tensors],
             [[a.get_optimizer_state(t["index"], m) for t in a.params] for m in (0, 1)], a.optimizer_steps())
    run(a, cfg, 2, 2)
    b, _ = session()
    for t, v in zip(b.tensors, state[0]):
        b.set_tensor(t["index"], v)
    for m in (0, 1):
        for t, v in zip(b.params, state[1][m]):
            b.set_optimizer_state(t["index"], m, v)
    b.set_optimizer_steps(state[2])
    run(b, cfg, 2, 2)
    assert np.array_equal(a.flat_params(), b.flat_params())
    for m in (0, 1):
        assert np.array_equal(a.flat_velocity(m), b.flat_velocity(m))
    a.close()
    b.close()


def test_image_steps_stay_finite():
    s, cfg = session(backbone=True)
    s.set_backbone(data.backbone_params("yolov8n", seed=0))
    rng = np.random.default_rng(3)
    images, truth = data.synthetic_batch(rng, 2, 128, cfg.num_classes, boxes=(1, 6), wh=(8.0, 64.0))
    for _ in range(4):
        stats = s.step(images, truth)
        assert np.isfinite([stats.box, stats.cls, stats.dfl]).all()
    assert np.isfinite(s.flat_params()).all()
    s.close()


@pytest.mark.parametrize("model", ["yolov8n", "yolo11s"])
@pytest.mark.parametrize("precision", [sy.SY_PRECISION_TF32, sy.SY_PRECISION_3XTF32], ids=["tf32", "3xtf32"])
def test_matrices_step_as_the_operator_steps_them(model, precision):
    """A session's matrices take the very step that muon_update_device gives the same weights, momenta and gradients."""
    rng = np.random.default_rng(11)
    s, cfg = session(model, precision=precision)
    o = sy.muon_options(LR, cfg.momentum, DECAY, grad_scale=0.5, precision=precision)
    for k in range(3):
        truth = [[], []] if k == 1 else data.synthetic_batch(rng, 2, 128, cfg.num_classes, boxes=(1, 20), wh=(8.0, 64.0))[1]
        mats = [t for t in s.params if is_muon(t, lambda t: t["shape"][1] > 1)]
        get = lambda read: [torch.from_numpy(np.asarray(read(t)).reshape(t["shape"][0], -1)).cuda() for t in mats]
        w, m = get(lambda t: s.get_tensor(t["index"])), get(lambda t: s.get_optimizer_state(t["index"], 0))
        stats = s.step_features(features(cfg, 2, rng), truth)
        grad, starts = s.last_gradients(), np.cumsum([0] + [t["numel"] for t in s.params])
        flat = {t["index"]: grad[a:a + t["numel"]] for t, a in zip(s.params, starts)}
        g = get(lambda t: flat[t["index"]])
        live = [i for i, t in enumerate(mats) if sy.tensor_group(t["name"]) == 0 or stats.box_has_grad]
        assert 0 < len(live) and (len(live) < len(mats)) == (k == 1)
        before = [x.clone() for x in w]
        keep = D.muon(*[[v[i] for i in live] for v in (w, m, g)], o)
        for i, t in enumerate(mats):
            assert torch.equal(get(lambda t: s.get_tensor(t["index"]))[i], w[i]), t["name"]
            assert torch.equal(get(lambda t: s.get_optimizer_state(t["index"], 0))[i], m[i]), t["name"]
            assert torch.equal(w[i], before[i]) == (i not in live)
        del keep
    s.close()


def test_a_step_that_is_not_finite_changes_nothing():
    s, cfg = session()
    run(s, cfg, 1, 1)
    rng = np.random.default_rng(4)
    feats, truth = features(cfg, 2, rng), data.synthetic_batch(rng, 2, 128, cfg.num_classes, boxes=(1, 5), wh=(8.0, 64.0))[1]
    index = next(t["index"] for t in s.tensors if t["name"] == "cv3.0.0.conv.weight")
    good = s.get_tensor(index)
    bad = good.copy()
    bad.flat[7] = np.nan
    s.set_tensor(index, bad)
    state = lambda: [a.tobytes() for a in (s.flat_params(), s.flat_buffers(), s.flat_velocity(0), s.flat_velocity(1))]
    before, steps = state(), s.optimizer_steps()
    for _ in range(2):
        with pytest.raises(sy.NonFinite):
            s.step_features(feats, truth)
        assert state() == before and s.optimizer_steps() == steps
    s.set_tensor(index, good)
    s.step_features(feats, truth)
    assert np.isfinite(s.flat_params()).all()
    s.close()

