"""The logit operators' host side: what fails closed without a device, and the host
sampler's random numbers."""
import ctypes as C

import numpy as np
import pytest

import hexatrain_b200 as hx
from hexatrain_b200 import _lib


def test_null_runtime_is_rejected():
    lib = _lib.load()
    assert lib.hx_top_logits_device(None, 0, 1, 4, None, 4, 1, 1.0, None, None, None) == _lib.HX_ERR_ARGUMENT
    assert lib.hx_sample_logits_device(None, 0, 1, 4, None, 4, None, None, None, None, None, None,
                                       None) == _lib.HX_ERR_ARGUMENT
    assert lib.hx_distill_forward_device(None, 0, 1, 4, None, 4, 1, None, None, None, None, 1.0, 1.0, 0.0, None,
                                         None) == _lib.HX_ERR_ARGUMENT
    assert lib.hx_lm_generate_device(None, None, 1, 1, None, None, None, None) == _lib.HX_ERR_ARGUMENT


def test_uninitialised_runtime_fails_closed():
    rt = hx.Runtime()
    assert not rt.top_logits_device(0, 1, 4, 0, 4, 1, 0, 0)
    assert rt.last_error == "runtime not initialized"
    assert not rt.sample_logits_device(0, 1, 4, 0, 4, 0, 0)
    assert not rt.distill_backward_device(0, 1, 4, 0, 4, 1, 0, 0, 0, 0, 1.0, 1.0, 0.0, 0, 0, 4)
    assert rt.lm_generate_device(np.zeros((1, 1)), 1) == (None, None)


def test_uniform_is_the_host_samplers_number():
    """The token of the host sampler is where its cumulative probability first
    reaches hx_sample_uniform."""
    lib = _lib.load()
    logits = np.random.default_rng(3).standard_normal(50).astype(np.float32)
    order = np.argsort(-logits, kind="stable")
    p = np.exp(logits[order].astype(np.float64) - logits.max())
    cum = np.cumsum(p / p.sum())
    for seed in range(40):
        u = lib.hx_sample_uniform(seed, 2)
        assert 0.0 <= u < 1.0
        tok, _ = hx.sample_next_token(logits, step=2, greedy=False, temperature=1.0, seed=seed)
        assert tok == order[np.searchsorted(cum, u)]


def test_device_sampling_layout():
    assert C.sizeof(_lib.DeviceSamplingC) == 24 and _lib.DeviceSamplingC.seed.offset == 16


def test_distiller_refuses_unprepared_runtimes():
    pytest.importorskip("torch")
    from hexatrain_b200.distillation import Distiller
    with pytest.raises(ValueError):
        Distiller(hx.Runtime(), hx.Runtime())


def test_pattern_tokens_stay_in_the_vocabulary():
    from hexatrain_b200.distillation import pattern_tokens
    for tokens in (1, 2, 63, 64):
        ids = pattern_tokens(1, 3, tokens, 200)
        assert ids.shape == (3, tokens + 1) and ids.max() < 200
        assert np.array_equal(ids[:, 1], (ids[:, 0].astype(np.int64) * 3 + 1) % 200)
