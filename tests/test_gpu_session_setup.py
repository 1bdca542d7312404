"""What a session holds right after it was made: initial values and job lists are uploaded in its stream's order.

The memsets of a session's allocations are queued on its own stream, which does not wait for the legacy default stream
nor holds it up.  A larger capacity queues gigabytes of them ahead of the first calls.
"""
import numpy as np
import pytest

import simdyolo_b200 as sy
from simdyolo_b200 import data

pytestmark = pytest.mark.gpu


def make(precision, max_batch):
    return sy.Session(sy.make_config("yolov8n", image_size=640, max_batch=max_batch, max_boxes=8, backbone=False, lr=0.01,
                                     precision=precision))


@pytest.mark.parametrize("precision", [sy.SY_PRECISION_TF32, sy.SY_PRECISION_3XTF32], ids=["tf32", "3xtf32"])
@pytest.mark.parametrize("max_batch", [2, 48])
def test_a_fresh_session_steps_like_the_one_before(precision, max_batch):
    rng = np.random.default_rng(0)
    feats = truth = first = None
    for _ in range(6):
        with make(precision, max_batch) as s:
            variance = next(t for t in s.tensors if t["name"].endswith("running_var"))
            assert (s.get_tensor(variance["index"]) == 1).all()
            weight = next(t for t in s.params if t["name"] == "cv3.0.0.conv.weight")
            velocity = rng.standard_normal(weight["numel"]).astype(np.float32) * 1e-3
            s.set_optimizer_state(weight["index"], 0, velocity)
            assert np.array_equal(np.ravel(s.get_optimizer_state(weight["index"], 0)), velocity)
            s.set_optimizer_state(weight["index"], 0, velocity * 0)
            params, buffers = data.head_params(s, 0)
            s.set_flat_params(params)
            s.set_flat_buffers(buffers)
            if feats is None:
                feats = [rng.standard_normal((2, c, 640 >> (3 + l), 640 >> (3 + l))).astype(np.float32)
                         for l, c in enumerate(s.config.feature_channels)]
                truth = data.synthetic_batch(rng, 2, 640, 80, boxes=(1, 8), wh=(8.0, 320.0))[1]
            stats = s.step_features(feats, truth)
            grad, after, running = s.last_gradients(), s.flat_params(), s.flat_buffers()
            off = 0
            for t in s.params:      # head weights were laid out, and every parameter took its step
                part = slice(off, off + t["numel"])
                off += t["numel"]
                if t["name"].startswith("cv3.") and len(t["shape"]) == 4:   # (a level may be without a box to match)
                    assert grad[part].any() and not np.array_equal(after[part], params[part]), t["name"]
            assert not np.array_equal(running, buffers)
            now = (stats.box, stats.cls, stats.dfl, grad.tobytes(), after.tobytes(), running.tobytes())
            first = first or now
            assert now == first
