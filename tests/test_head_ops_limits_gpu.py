"""The operators on device logits at their limits: the shapes, masks and records that
leave a kernel little room.  Tolerances as in test_head_ops_gpu.py."""
import numpy as np
import pytest

from test_head_ops_gpu import CODES, REL, ULP, Distill, normal, record_of, rt, some_labels, torch  # noqa: F401

pytestmark = pytest.mark.gpu


# -- many rows to a block, wide records ----------------------------------------------

@pytest.mark.parametrize("rows,vocab,k,pad", [(2500, 2100, 255, 0), (2500, 4096, 256, 0), (1500, 4093, 256, 3),
                                              (40, 151936, 256, 0), (40, 140001, 213, 3), (30, 262144, 224, 1),
                                              (30, 262141, 5, 4)])
def test_top_wide_records_of_many_rows(rt, torch, rows, vocab, k, pad):  # noqa: F811
    """Float32 rows whose lists leave a block two row warps or one, several rows to
    every block (or cluster)."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows + vocab)
    view = (torch.randn(rows, vocab + pad, device="cuda", generator=gen) * 2)[:, :vocab]
    order = torch.sort(view, dim=1, descending=True, stable=True)
    want, lse = order.indices[:, :k].to(torch.int32), torch.logsumexp(view.double() / 2.0, 1)
    v, i = torch.empty(rows, k, device="cuda"), torch.empty(rows, k, device="cuda", dtype=torch.int32)
    s = torch.empty(rows, device="cuda")
    for _ in range(2):
        v.fill_(-7.0), i.fill_(-7)
        assert rt.top_logits_device(CODES["f32"], rows, vocab, view.data_ptr(), vocab + pad, k, v.data_ptr(),
                                    i.data_ptr(), s.data_ptr(), 2.0), rt.last_error
        assert rt.synchronize(), rt.last_error
        assert torch.equal(i, want) and torch.equal(v, order.values[:, :k])
        assert bool(((s.double() - lse).abs() <= REL + 4 * ULP * (lse.abs() + 12)).all())


# -- the gradient over the logits ------------------------------------------------------

@pytest.mark.parametrize("rows,vocab", [(3, 700), (5, 9001), (6, 40000), (300, 40001), (4, 262144)])
@pytest.mark.parametrize("tail", [False, True])
def test_backward_in_place(rt, torch, rows, vocab, tail):  # noqa: F811
    """The backward over the logits themselves is the one into a buffer of its own, in
    one block and in a cluster to a row."""
    x = normal(vocab, rows, vocab, 1.5)
    for dtype in ("f32", "bf16"):
        d = Distill(rt, torch, x, dtype, record_of(2, x, 40, 2.0, tail), some_labels(rows, vocab), 2.0, 0.5, 0.5, pad=3)
        d.forward()
        want = d.backward(None, 0.5)
        assert rt.distill_backward_device(*d.args, d.stats.data_ptr(), d.view.data_ptr(), vocab + 3, 0, 0.5), rt.last_error
        assert rt.synchronize(), rt.last_error
        assert np.array_equal(d.view.double().cpu().numpy(), want)
