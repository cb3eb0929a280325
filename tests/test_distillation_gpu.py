"""The logit operators inside the LM: a teacher's record, the distillation step and
generation with tokens sampled on the device."""
import numpy as np
import pytest

import hexatrain_b200 as hx
from conftest import rel_err
from hexatrain_b200 import data, distillation
from hexatrain_b200.parallel import _device_view

pytestmark = pytest.mark.gpu

SMALL = hx.LmConfig(200, 16, 32, 48, 2, 4, learned_position=True)
WIDE = hx.LmConfig(200, 16, 64, 64, 2, 4, learned_position=True)


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def ready(cfg, batch, seed, std=0.2):
    rt = hx.Runtime()
    assert rt.initialize(0), rt.last_error
    assert rt.set_stream(1), rt.last_error
    assert rt.prepare_lm(cfg, batch), rt.last_error
    params = cfg.init_normal(seed, std)
    assert rt.lm_state_upload(params), rt.last_error
    return rt, params


def gradients(torch, rt):
    p, n = rt.lm_grad_buffer()
    assert rt.synchronize(), rt.last_error
    return _device_view(p, n).double().cpu().numpy()


def record(torch, rows, k):
    return (torch.empty(rows, k, device="cuda"), torch.empty(rows, k, device="cuda", dtype=torch.int32),
            torch.empty(rows, device="cuda"))


def device_tokens(torch, ids):
    return torch.from_numpy(np.ascontiguousarray(ids, np.uint32).view(np.int32)).cuda()


def test_record_is_the_forwards_top_logits(torch):
    rt, params = ready(WIDE, 3, 5)
    ids = data.lm_tokens(1, 3, 16, 200)
    tok = device_tokens(torch, ids)
    v, i, s = record(torch, 48, 12)
    for _ in range(4):  # eager, eager with a capture, replays
        assert rt.lm_top_logits_device(tok.data_ptr(), 12, v.data_ptr(), i.data_ptr(), s.data_ptr(), 2.0), rt.last_error
        assert rt.synchronize(), rt.last_error
        logits = rt.execute_tiny_transformer_forward_only_tokens(ids[:, :16])
        assert logits is not None, rt.last_error
        order = np.argsort(-logits, axis=1, kind="stable")[:, :12]
        assert np.array_equal(i.cpu().numpy(), order)
        assert np.array_equal(v.cpu().numpy(), np.take_along_axis(logits, order, 1))
        z = logits.astype(np.float64) / 2.0
        assert np.allclose(s.cpu().numpy(), np.log(np.exp(z - z.max(1, keepdims=True)).sum(1)) + z.max(1), atol=2e-5)
        v.zero_(), i.zero_()
    rt.close()


def test_hard_targets_alone_are_the_training_step(torch):
    """kd = 0, ce = 1 gives hx_lm_forward_backward_device's loss and gradients:
    both sum the same float32 terms, in other orders."""
    rt, _ = ready(SMALL, 5, 3)
    tok = device_tokens(torch, data.lm_tokens(2, 5, 16, 200))
    v, i, s = record(torch, 80, 4)
    v.zero_(), i.copy_(torch.arange(4).expand(80, 4))
    assert rt.lm_forward_backward_device(tok.data_ptr(), 0.2), rt.last_error
    want = gradients(torch, rt)
    for _ in range(4):
        assert rt.lm_distill_forward_backward_device(tok.data_ptr(), 0.2, 4, v.data_ptr(), i.data_ptr(), 0, 1.0, 0.0,
                                                     1.0), rt.last_error
        got = gradients(torch, rt)
        assert abs(got[-1] - want[-1]) <= 2e-5 * abs(want[-1])
        assert rel_err(got[:-1], want[:-1]) <= 5e-5
    rt.close()


@pytest.mark.parametrize("tail", [False, True])
def test_student_gradient_against_differences(torch, tail):
    """Along a random direction, (loss(w + h d) - loss(w - h d)) / 2h against
    g . d: with h |d| small against the curvature, float32 losses of about 5
    leave 2e-6 / 2h, and the ReLU kinks a little more."""
    teacher, _ = ready(WIDE, 4, 11)
    student, params = ready(SMALL, 4, 12)
    tok = device_tokens(torch, data.lm_tokens(3, 4, 16, 200))
    v, i, s = record(torch, 64, 20)
    assert teacher.lm_top_logits_device(tok.data_ptr(), 20, v.data_ptr(), i.data_ptr(), s.data_ptr(), 1.5), teacher.last_error
    assert teacher.synchronize(), teacher.last_error

    def run(w):
        assert student.lm_state_upload(w), student.last_error
        assert student.lm_distill_forward_backward_device(
            tok.data_ptr(), 0.25, 20, v.data_ptr(), i.data_ptr(), s.data_ptr() if tail else 0, 1.5, 0.7, 0.3), student.last_error
        return gradients(torch, student)

    g = run(params)
    rng = np.random.default_rng(4)
    for _ in range(3):
        d = rng.standard_normal(params.size)
        d *= 1.0 / np.linalg.norm(d)
        h = 0.02
        up = run((params + h * d).astype(np.float32))[-1]
        down = run((params - h * d).astype(np.float32))[-1]
        slope, want = (up - down) / (2 * h), float(g[:-1] @ d)
        assert abs(slope - want) <= 2e-3 * np.linalg.norm(g[:-1]) + 2e-4, (slope, want)
    teacher.close()
    student.close()


def test_students_own_record_leaves_little_to_learn(torch):
    """With itself as the teacher, every token in the record, the KL and its
    gradient vanish."""
    cfg = hx.LmConfig(64, 8, 16, 16, 1, 2)
    rt, _ = ready(cfg, 2, 9)
    tok = device_tokens(torch, data.lm_tokens(5, 2, 8, 64))
    v, i, s = record(torch, 16, 64)
    assert rt.lm_top_logits_device(tok.data_ptr(), 64, v.data_ptr(), i.data_ptr(), s.data_ptr(), 2.0), rt.last_error
    assert rt.lm_distill_forward_backward_device(tok.data_ptr(), 0.5, 64, v.data_ptr(), i.data_ptr(), 0, 2.0, 1.0, 0.0)
    g = gradients(torch, rt)
    assert abs(g[-1]) <= 1e-4 and np.abs(g[:-1]).max() <= 1e-5
    rt.close()


def test_device_generation_draws_the_hosts_tokens():
    rt, _ = ready(SMALL, 6, 21)
    prompts = data.lm_tokens(8, 6, 4, 200)[:, :5]
    for kw, dev in ((dict(greedy=True), dict(temperature=0.0)),
                    (dict(greedy=False, temperature=0.9, top_k=20, seed=77), dict(temperature=0.9, top_k=20, seed=77)),
                    (dict(greedy=False, temperature=1.1, seed=5), dict(temperature=1.1, seed=5))):
        want = rt.lm_generate(prompts, 20, **kw)
        got, logs = rt.lm_generate_device(prompts, 20, **dev)
        assert got is not None, rt.last_error
        assert np.array_equal(got, want)  # 15 tokens past the window: the windows slide alike
        assert np.all(logs <= 0) and np.all(np.isfinite(logs))
    u = np.random.default_rng(0).random((7, 6)).astype(np.float32)
    first = rt.lm_generate_device(prompts, 7, top_p=0.8, min_p=0.01, uniform=u)
    again = rt.lm_generate_device(prompts, 7, top_p=0.8, min_p=0.01, uniform=u)
    assert all(np.array_equal(x, y) for x, y in zip(first, again))
    rt.close()


def test_generation_refusals():
    rt, _ = ready(SMALL, 2, 1)
    assert rt.lm_generate_device(np.array([[200], [1]]), 2)[0] is None
    assert rt.last_error.startswith("INVALID_TINY_LM_TOKEN")
    assert rt.lm_generate_device(np.array([[1]]), 2)[0] is None  # not the prepared batch
    assert rt.lm_generate_device(np.zeros((2, 0)), 2)[0] is None
    assert "PROMPT_EMPTY" in rt.last_error
    assert not rt.lm_distill_forward_backward_device(0, 1.0, 4, 0, 0)
    assert not rt.lm_top_logits_device(0, 4, 0, 0)
    out, _ = rt.lm_generate_device(np.array([[1], [2]]), 0)
    assert out.shape == (2, 0)
    rt.close()


def test_example_trains_a_student(torch):
    report = distillation.main(["--steps", "30", "--batch", "8", "--vocab", "256"])
    assert report["last_loss"] < report["first_loss"]
    assert report["generated"].shape == (8, 8) and report["generated"].max() < 256
