"""The logit operators inside the LM where their input is not what it should be."""
import numpy as np
import pytest

from hexatrain_b200 import data
from hexatrain_b200.distillation import Distiller
from test_distillation_gpu import SMALL, WIDE, device_tokens, ready, record, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def test_token_ids_beyond_the_vocabulary_are_reported(torch):  # noqa: F811
    """As an input or as a target, in eager calls and in replayed graphs: the next
    synchronising call fails, once."""
    import hexatrain_b200 as hx
    rt = hx.Runtime()
    assert rt.initialize(0), rt.last_error  # its own stream, where steps become graphs
    assert rt.prepare_lm(SMALL, 3) and rt.lm_state_upload(SMALL.init_normal(1, 0.1)), rt.last_error
    good = data.lm_tokens(1, 3, 16, 200)
    v, i, s = record(torch, 48, 4)
    v.zero_(), i.copy_(torch.arange(4).expand(48, 4)), s.fill_(2.0)
    tok = device_tokens(torch, good)
    torch.cuda.synchronize()
    calls = (lambda: rt.lm_top_logits_device(tok.data_ptr(), 4, v.data_ptr(), i.data_ptr(), s.data_ptr(), 1.0),
             lambda: rt.lm_distill_forward_backward_device(tok.data_ptr(), 0.5, 4, v.data_ptr(), i.data_ptr(),
                                                           s.data_ptr(), 1.0, 0.5, 0.5))
    for call in calls:
        for turn in range(5):
            ids = good.copy()
            at = (turn % 3, (0, 16, 5, 16, 9)[turn])
            ids[at] = (200, 1 << 31, 0xffffffff, 201, 200)[turn]
            tok.copy_(device_tokens(torch, ids))
            torch.cuda.synchronize()
            assert call(), rt.last_error
            assert not rt.synchronize()
            assert rt.last_error.startswith("INVALID_TINY_LM_TOKEN"), rt.last_error
            tok.copy_(device_tokens(torch, good))
            torch.cuda.synchronize()
            assert call(), rt.last_error
            assert rt.synchronize(), rt.last_error
    rt.close()


def test_distiller_reports_the_teachers_errors(torch):  # noqa: F811
    teacher, _ = ready(WIDE, 2, 1)
    student, _ = ready(SMALL, 2, 2)
    from hexatrain_b200 import OptimizerConfig
    assert student.lm_set_optimizer(OptimizerConfig()), student.last_error
    d = Distiller(teacher, student, k=8)
    ids = data.lm_tokens(1, 2, 16, 200)
    d.step(ids, 1)
    assert np.isfinite(d.loss())
    ids[1, 3] = 200
    d.step(ids, 2)
    with pytest.raises(RuntimeError, match="INVALID_TINY_LM_TOKEN"):
        d.loss()
    teacher.close()
    student.close()


def test_generation_leaves_no_mark_on_the_next_step(torch):  # noqa: F811
    """A model whose logits are NaN: generation fails, and a training step afterwards is
    judged by its own tokens alone."""
    rt, params = ready(SMALL, 2, 3)
    from hexatrain_b200 import OptimizerConfig
    assert rt.lm_set_optimizer(OptimizerConfig()), rt.last_error
    assert rt.lm_state_upload(np.full_like(params, np.nan)), rt.last_error
    assert rt.lm_generate_device(np.array([[1], [2]]), 3)[0] is None
    assert "non-finite" in rt.last_error
    assert rt.lm_state_upload(params), rt.last_error
    ok, loss = rt.lm_train_step(data.lm_tokens(4, 2, 16, 200), 1)
    assert ok and np.isfinite(loss), rt.last_error
    out, logs = rt.lm_generate_device(np.array([[1], [2]]), 3)
    assert out is not None and np.all(np.isfinite(logs)), rt.last_error
    rt.close()
