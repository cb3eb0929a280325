"""The operators on device logits (top logits, distillation, sampling) against
their definitions in 64 bits.

Tolerances.  A float32 sum of n terms of one sign, added in parts of at most 64
and then pairwise, is off by less than 100 * 2^-24 of itself; ex2.approx adds
2^-22, and the argument (l - m) log2(e) / tau two roundings of at most
2^-24 |argument|, which the weight 2^argument keeps below 2^-23.  So a sum of
exponentials is within REL = 8e-6 of itself, its logarithm within 8e-6 plus the
rounding of the result, and a probability within 2 REL.
"""
import numpy as np
import pytest

import hexatrain_b200 as hx
from hexatrain_b200 import _lib

pytestmark = pytest.mark.gpu

REL = 8e-6
ULP = 2.0 ** -23
CODES = {"f32": _lib.HX_DTYPE_F32, "bf16": _lib.HX_DTYPE_BF16, "f16": _lib.HX_DTYPE_F16}
# the rounding of a result to the type: half a unit in the last place, relative
ROUND = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rt(torch):
    r = hx.Runtime()
    assert r.initialize(0), r.last_error
    assert r.set_stream(1), r.last_error  # the legacy default stream, where torch works
    yield r
    r.close()


def to_device(torch, x, dtype, pad=0, shift=0):
    """[rows, vocab] float array -> (a view with row stride vocab + pad whose
    first element lies `shift` elements into its buffer, the float64 values)."""
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    rows, vocab = x.shape
    buf = torch.full((rows * (vocab + pad) + shift,), 77.0, device="cuda", dtype=t)
    view = buf[shift:].as_strided((rows, vocab), (vocab + pad, 1))
    view.copy_(torch.from_numpy(np.ascontiguousarray(x, np.float32)).to("cuda"))
    return view, view.double().cpu().numpy()


def normal(seed, rows, vocab, spread=2.5):
    return np.random.default_rng(seed).standard_normal((rows, vocab)).astype(np.float32) * np.float32(spread)


def lse64(z):
    m = z.max(axis=1, keepdims=True)
    m = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore"):
        return m[:, 0] + np.log(np.exp(z - m).sum(axis=1))


# -- top logits -----------------------------------------------------------------

def top(rt, torch, x, dtype, k, tau=1.0, pad=0, shift=0):
    view, x64 = to_device(torch, x, dtype, pad, shift)
    rows, vocab = x.shape
    v = torch.full((rows, k), -7.0, device="cuda")
    i = torch.full((rows, k), -7, device="cuda", dtype=torch.int32)
    s = torch.full((rows,), -7.0, device="cuda")
    ok = rt.top_logits_device(CODES[dtype], rows, vocab, view.data_ptr(), vocab + pad, k, v.data_ptr(), i.data_ptr(),
                              s.data_ptr(), tau)
    assert ok, rt.last_error
    assert rt.synchronize(), rt.last_error
    return v.double().cpu().numpy(), i.cpu().numpy(), s.double().cpu().numpy(), x64


def check_top(rt, torch, x, dtype, k, tau=1.0, pad=0, shift=0):
    v, i, s, x64 = top(rt, torch, x, dtype, k, tau, pad, shift)
    order = np.argsort(-x64, axis=1, kind="stable")[:, :k]
    assert np.array_equal(i, order)
    assert np.array_equal(v, np.take_along_axis(x64, order, 1))
    want = lse64(x64 / tau)
    fine = np.isfinite(want)
    assert np.array_equal(s[~fine], want[~fine])
    assert np.all(np.abs(s - want)[fine] <= REL + 4 * ULP * (np.abs(want[fine]) + np.abs(x64).max(1, where=np.isfinite(x64), initial=0)[fine] / tau))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 33, 7), (4, 256, 256), (3, 1000, 100),
                                          (9, 1024, 32), (7, 1025, 256), (2, 4099, 64), (3, 16384, 1), (2, 16385, 256),
                                          (2, 50001, 200), (1, 131073, 256), (2, 262144, 17)])
def test_top_sizes(rt, torch, dtype, rows, vocab, k):
    check_top(rt, torch, normal(rows + vocab, rows, vocab), dtype, k)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (3, 3), (8, 5)])
@pytest.mark.parametrize("vocab", [37, 1024, 5001, 40000])
def test_top_strides(rt, torch, vocab, pad, shift):
    for dtype in ("f32", "bf16"):
        check_top(rt, torch, normal(vocab + pad, 5, vocab), dtype, 20, tau=1.7, pad=pad, shift=shift)


@pytest.mark.parametrize("vocab", [40, 1024, 3000, 40000])
@pytest.mark.parametrize("kind", ["equal", "two", "steps", "rising", "falling", "masked", "one", "none", "zeros", "far"])
def test_top_ties_and_masks(rt, torch, vocab, kind):
    rng = np.random.default_rng(vocab)
    x = np.zeros((3, vocab), np.float32)
    if kind == "equal":
        x[:] = 1.25
    elif kind == "two":
        x[:] = rng.integers(0, 2, x.shape)
    elif kind == "steps":
        x[:] = rng.integers(0, 9, x.shape) - 4
    elif kind == "rising":
        x[:] = np.arange(vocab, dtype=np.float32) / 64
    elif kind == "falling":
        x[:] = -np.arange(vocab, dtype=np.float32) / 64
    elif kind == "masked":  # fewer logits than the record has entries
        x[:] = -np.inf
        x[:, rng.integers(0, vocab, 5)] = rng.standard_normal(5)
    elif kind == "one":
        x[:] = -np.inf
        x[:, vocab - 1] = -3.0
    elif kind == "none":
        x[:] = -np.inf
    elif kind == "zeros":  # the two zeros are equal
        x[:, ::2] = -0.0
    else:  # the type's lowest value as a mask
        x[:] = np.finfo(np.float32).min
        x[:, ::3] = rng.standard_normal(x[:, ::3].shape)
    check_top(rt, torch, x, "f32", min(vocab, 37))
    if kind not in ("far", "rising", "falling"):
        check_top(rt, torch, x, "bf16", min(vocab, 37))


def test_largest_vocabulary_not_aligned(rt, torch):
    x = normal(7, 2, 262144)
    check_top(rt, torch, x, "f32", 224, pad=1)
    check_top(rt, torch, x, "bf16", 256, pad=3, shift=1)
    view, _ = to_device(torch, x, "f32", 1)
    out = torch.empty(2, 256, device="cuda")
    assert not rt.top_logits_device(0, 2, 262144, view.data_ptr(), 262145, 256, out.data_ptr(), out.data_ptr())
    assert "no room" in rt.last_error
    check_distill(rt, torch, x, "f32", 256, 1.0, 0.5, 0.5, True, some_labels(2, 262144), 1)
    check_sample(rt, torch, x, "f32", np.array([0.3, 0.8], np.float32), p=0.9, pad=1)


def test_top_not_finite(rt, torch):
    x = normal(3, 4, 2000)
    x[0, 100] = np.inf
    x[1, 5] = np.nan
    x[2, :] = np.nan
    v, i, s, _ = top(rt, torch, x, "f32", 3)
    assert i[0, 0] == 100 and v[0, 0] == np.inf and s[0] == np.inf
    assert 5 not in i[1] and np.all(np.isfinite(v[1])) and np.isnan(s[1])
    assert list(i[2]) == [0, 1, 2] and np.all(np.isnan(v[2]))
    assert np.isfinite(s[3])


# -- distillation -----------------------------------------------------------------

def loss64(x, record, labels, tau, kd, ce):
    """(loss, stats, gradient of every row's loss) in 64 bits."""
    tv, ti, tl = record
    rows, vocab = x.shape
    z = x / tau
    lt, l1 = lse64(z), lse64(x)
    loss, ratio, grad = np.zeros(rows), np.zeros(rows), np.zeros_like(x)
    for r in range(rows):
        on = [j for j in range(tv.shape[1]) if ti[r, j] >= 0]
        if tl is None:
            on = [j for j in on if tv[r, j] > -np.inf]
        ids = ti[r, on]
        logp = z[r] - lt[r]
        p = np.exp(logp)
        if on:
            t = tv[r, on].astype(np.float64) / tau
            logq = t - (lse64(t[None])[0] if tl is None else np.float64(tl[r]))
            q = np.exp(logq)
            kl = sum(q[j] * (logq[j] - logp[ids[j]]) for j in range(len(ids)) if q[j] > 0)
            c = np.ones(vocab)
            if tl is not None:
                out = np.ones(vocab, bool)
                out[ids] = False
                pt, qt = p[out].sum(), max(0.0, 1.0 - q.sum())
                if pt > 0 and qt > 0:
                    kl += qt * np.log(qt / pt)
                    ratio[r] = qt / pt
                c[out] -= ratio[r]
            loss[r] += kd * tau * tau * kl
            g = p * c
            g[ids] -= q
            grad[r] += kd * tau * g
        if labels is not None and labels[r] >= 0:
            loss[r] += ce * (l1[r] - x[r, labels[r]])
            g = np.exp(x[r] - l1[r])
            g[labels[r]] -= 1.0
            grad[r] += ce * g
    return loss, np.stack([lt, l1, ratio], 1), grad


def record_of(seed, x, k, tau, tail, short=True):
    """A teacher near the student, its k largest logits, some rows shorter and
    one empty."""
    rng = np.random.default_rng(seed)
    t = 0.7 * np.where(np.isfinite(x), x, 0.0) + rng.standard_normal(x.shape)
    ti = np.argsort(-t, axis=1, kind="stable")[:, :k].astype(np.int32)
    tv = np.take_along_axis(t, ti.astype(np.int64), 1).astype(np.float32)
    tl = lse64(t / tau).astype(np.float32) if tail else None
    if short and x.shape[0] >= 4:
        ti[1, k // 2:] = -1
        ti[3] = -1
    return tv, ti, tl


class Distill:
    def __init__(self, rt, torch, x, dtype, record, labels, tau, kd, ce, pad=0, shift=0):
        self.rt, self.torch, self.dtype = rt, torch, dtype
        self.view, self.x64 = to_device(torch, x, dtype, pad, shift)
        self.rows, self.vocab = x.shape
        self.pad = pad
        up = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to("cuda")  # noqa: E731
        self.record = [up(a) for a in record]
        self.labels = up(labels)
        self.args = (CODES[dtype], self.rows, self.vocab, self.view.data_ptr(), self.vocab + pad, record[0].shape[1],
                     *[0 if a is None else a.data_ptr() for a in (*self.record, self.labels)], tau, kd, ce)
        self.loss = torch.full((self.rows,), -7.0, device="cuda")
        self.stats = torch.full((self.rows, 3), -7.0, device="cuda")
        self.grad = torch.full((self.rows, self.vocab + 2), 55.0, device="cuda", dtype=self.view.dtype)

    def forward(self):
        assert self.rt.distill_forward_device(*self.args, self.loss.data_ptr(), self.stats.data_ptr()), self.rt.last_error
        assert self.rt.synchronize(), self.rt.last_error
        return self.loss.double().cpu().numpy(), self.stats.double().cpu().numpy()

    def backward(self, grad_loss=None, scale=1.0):
        g = 0 if grad_loss is None else grad_loss.data_ptr()
        assert self.rt.distill_backward_device(*self.args, self.stats.data_ptr(), self.grad.data_ptr(), self.vocab + 2,
                                               g, scale), self.rt.last_error
        return self._grad()

    def fused(self, grad_loss=None, scale=1.0, in_place=False):
        g = 0 if grad_loss is None else grad_loss.data_ptr()
        to, stride = (self.view.data_ptr(), self.vocab + self.pad) if in_place else (self.grad.data_ptr(), self.vocab + 2)
        assert self.rt.distill_forward_backward_device(*self.args, self.loss.data_ptr(), to, stride, g,
                                                       scale), self.rt.last_error
        if in_place:
            assert self.rt.synchronize(), self.rt.last_error
            return self.loss.double().cpu().numpy(), self.view.double().cpu().numpy()
        return self.loss.double().cpu().numpy(), self._grad()

    def _grad(self):
        assert self.rt.synchronize(), self.rt.last_error
        assert bool((self.grad[:, self.vocab:] == 55.0).all())  # nothing beyond the rows is written
        return self.grad[:, :self.vocab].double().cpu().numpy()


def check_distill(rt, torch, x, dtype, k, tau, kd, ce, tail, labels, pad=0, shift=0, record=None, seed=1):
    rec = record_of(seed, x, k, tau, tail) if record is None else record
    d = Distill(rt, torch, x, dtype, rec, labels, tau, kd, ce, pad, shift)
    want, stats, grad = loss64(d.x64, rec, labels, tau, kd, ce)
    rows = x.shape[0]
    with np.errstate(over="ignore"):  # a hard target at the type's lowest value: the loss itself overflows
        over = ~np.isfinite(want.astype(np.float32))

    def near(got, tol):
        assert np.array_equal(got[over], want.astype(np.float32)[over])
        assert np.all(np.abs(got - want)[~over] <= tol[~over]), np.abs(got - want)[~over].max()

    loss, got = d.forward()
    # log-probabilities are within REL + roundings of the logits' size; the
    # teacher's log q likewise, so a KL is off by that times tau^2, and the
    # tail's share by the error of 1 - sum q over its size; logits that are
    # masked with a low value have no part in it
    size = 4 * ULP * (np.abs(d.x64).max(where=d.x64 > -1e4, initial=0) + 30) * max(1.0, 1 / tau)
    slack = (2 * REL + size) * (kd * tau * tau + ce)
    near(loss, 4 * slack + 4 * ULP * np.abs(want))
    assert np.all(np.abs(got[:, :2] - stats[:, :2]) <= REL + size)
    assert np.all(np.abs(got[:, 2] - stats[:, 2]) <= 1e-4 * np.maximum(1.0, stats[:, 2]))
    weights = torch.linspace(0.25, 2.0, rows, device="cuda")
    w = weights.double().cpu().numpy()[:, None] * 0.5
    tol = lambda s: 4 * s * (2 * REL + size) * (kd * tau + ce) + ROUND[dtype] * np.abs(s * grad) + (6e-8 if dtype == "f16" else 0)  # noqa: E731
    g = d.backward(weights, 0.5)
    assert np.all(np.abs(g - w * grad) <= tol(w)), np.abs(g - w * grad).max()
    loss2, g2 = d.fused(weights, 0.5)
    near(loss2, 4 * slack + 4 * ULP * np.abs(want))
    assert np.all(np.abs(g2 - w * grad) <= tol(w)), np.abs(g2 - w * grad).max()
    loss3, g3 = d.fused(None, 1.0, in_place=True)
    assert np.array_equal(loss3, loss2)
    assert np.all(np.abs(g3 - grad) <= tol(1.0))


def some_labels(rows, vocab, seed=0):
    y = np.random.default_rng(seed).integers(0, vocab, rows).astype(np.int32)
    if rows >= 4:
        y[2] = -1
    return y


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (4, 2, 1), (5, 33, 33), (6, 300, 256), (9, 1000, 20), (5, 1024, 32),
                                          (4, 1025, 7), (4, 4097, 100), (3, 16384, 64), (4, 16385, 3), (2, 50001, 256),
                                          (1, 262144, 40)])
def test_distill_sizes(rt, torch, rows, vocab, k, tail):
    x = normal(vocab, rows, vocab, 1.5)
    for dtype, tau, kd, ce in (("f32", 2.0, 0.6, 0.4), ("f32", 1.0, 1.0, 0.0), ("bf16", 1.5, 0.5, 0.5), ("f16", 1.0, 0.3, 0.7)):
        check_distill(rt, torch, x, dtype, k, tau, kd, ce, tail, some_labels(rows, vocab) if ce else None)


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (5, 3)])
@pytest.mark.parametrize("vocab", [61, 1024, 3001, 33000])
def test_distill_strides(rt, torch, vocab, pad, shift):
    x = normal(vocab, 5, vocab, 1.5)
    for dtype in ("f32", "f16"):
        check_distill(rt, torch, x, dtype, 9, 1.3, 0.7, 0.3, True, some_labels(5, vocab), pad, shift)


@pytest.mark.parametrize("rows,vocab,dtype", [(1300, 9001, "f32"), (900, 20011, "f16"), (700, 60013, "f16"),
                                              (500, 40001, "f32"), (3000, 1500, "f32"), (5000, 700, "bf16")])
def test_distill_many_rows(rt, torch, rows, vocab, dtype):
    """Several rows to every block, in a padded buffer: the loss and statistics
    against 64 bits on the GPU, within the bounds of check_distill."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows)
    k, tau, kd, ce = 11, 1.5, 0.5, 0.5
    buf = torch.randn(rows, vocab + 29, device="cuda", generator=gen) * 2
    view = buf.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype])[:, :vocab]
    x = view.double()
    teacher = 0.7 * x.float() + torch.randn(rows, vocab, device="cuda", generator=gen)
    v, i = torch.topk(teacher, k, dim=1)
    i32, lse = i.to(torch.int32), torch.logsumexp(teacher / tau, 1)
    y = torch.randint(0, vocab, (rows,), device="cuda", generator=gen).to(torch.int32)
    loss, stats = torch.empty(rows, device="cuda"), torch.empty(rows, 3, device="cuda")
    logp, logq = torch.log_softmax(x / tau, 1), v.double() / tau - lse.double()[:, None]
    q = logq.exp()
    rest = logp.exp()
    rest.scatter_(1, i, 0.0)
    pt, qt = rest.sum(1), 1.0 - q.sum(1)
    kl = (q * (logq - logp.gather(1, i))).sum(1) + qt * (qt / pt).log()
    want = kd * tau ** 2 * kl + ce * (torch.logsumexp(x, 1) - x.gather(1, y.long()[:, None])[:, 0])
    size = 4 * ULP * (float(x.abs().max()) + 30)
    slack = (2 * REL + size) * (kd * tau * tau + ce)
    grad = torch.empty(rows, vocab, device="cuda", dtype=view.dtype)
    g64 = kd * tau * (logp.exp() * torch.where(rest == 0, 1.0, 1.0 - (qt / pt)[:, None]))
    g64.scatter_add_(1, i, -kd * tau * q)
    hard = torch.softmax(x, 1)
    hard.scatter_add_(1, y.long()[:, None], torch.full((rows, 1), -1.0, device="cuda", dtype=torch.float64))
    g64 += ce * hard
    args = (CODES[dtype], rows, vocab, view.data_ptr(), vocab + 29, k, v.data_ptr(), i32.data_ptr(), lse.data_ptr(),
            y.data_ptr(), tau, kd, ce)
    for _ in range(3):
        loss.fill_(-7.0)
        assert rt.distill_forward_device(*args, loss.data_ptr(), stats.data_ptr()), rt.last_error
        assert rt.synchronize(), rt.last_error
        assert bool(((loss.double() - want).abs() <= 4 * slack + 4 * ULP * want.abs()).all())
        assert bool(((stats[:, 2].double() - qt / pt).abs() <= 1e-4 * (qt / pt).clamp(min=1.0)).all())
        for fused in (True, False):
            grad.fill_(9.0)
            if fused:
                ok = rt.distill_forward_backward_device(*args, loss.data_ptr(), grad.data_ptr(), vocab)
            else:
                ok = rt.distill_backward_device(*args, stats.data_ptr(), grad.data_ptr(), vocab)
            assert ok and rt.synchronize(), rt.last_error
            tol = 4 * (2 * REL + size) * (kd * tau + ce) + ROUND[dtype] * g64.abs() + (6e-8 if dtype == "f16" else 0)
            assert bool(((grad.double() - g64).abs() <= tol).all())
            assert bool(((loss.double() - want).abs() <= 4 * slack + 4 * ULP * want.abs()).all())


@pytest.mark.parametrize("rows,vocab,k,dtype", [(1300, 9001, 30, "f32"), (700, 60013, 100, "f16"), (3000, 1500, 64, "bf16"),
                                                (9000, 700, 9, "f32"), (5000, 40, 17, "f32"), (400, 130001, 200, "bf16")])
def test_top_many_rows(rt, torch, rows, vocab, k, dtype):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows)
    buf = torch.randn(rows, vocab + 3, device="cuda", generator=gen) * 2
    view = buf.to({"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype])[:, :vocab]
    order = torch.sort(view.float(), dim=1, descending=True, stable=True)
    want, lse = order.indices[:, :k].to(torch.int32), torch.logsumexp(view.double(), 1)
    v, i = torch.empty(rows, k, device="cuda"), torch.empty(rows, k, device="cuda", dtype=torch.int32)
    s = torch.empty(rows, device="cuda")
    for _ in range(3):
        v.fill_(-7.0), i.fill_(-7)
        assert rt.top_logits_device(CODES[dtype], rows, vocab, view.data_ptr(), vocab + 3, k, v.data_ptr(), i.data_ptr(),
                                    s.data_ptr()), rt.last_error
        assert rt.synchronize(), rt.last_error
        assert torch.equal(i, want) and torch.equal(v, order.values[:, :k])
        assert bool(((s.double() - lse).abs() <= REL + 4 * ULP * (lse.abs() + 12)).all())


@pytest.mark.parametrize("vocab", [50, 1024, 9000])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_edges(rt, torch, vocab, tail):
    """Label inside and outside the record; hard targets only; rows with
    neither; masked student logits; teacher entries of -inf; a student that is
    sure."""
    rows, k = 8, 6
    x = normal(9, rows, vocab, 1.0)
    rec = record_of(4, x, k, 2.0, tail)
    named = {int(i) for i in rec[1][0]}
    y = np.array([rec[1][0][0], next(i for i in range(vocab) if i not in named), -1, -1, 0, 1, 2, 3], np.int32)
    masked = [i for i in range(vocab) if i not in set(rec[1][4].tolist()) | {0}][::2]
    x[4, masked] = -np.inf
    x[5, masked] = np.finfo(np.float32).min if vocab != 50 else -1e30
    rec[0][6, 1:3] = -np.inf
    x[7, rec[1][7][0]] = 25.0
    check_distill(rt, torch, x, "f32", k, 2.0, 0.5, 0.5, tail, y, record=rec)
    check_distill(rt, torch, x, "f32", k, 2.0, 0.0, 1.0, tail, y, record=rec)
    check_distill(rt, torch, x, "f32", k, 2.0, 1.0, 0.0, tail, None, record=rec)


def test_distill_empty_rows_are_zero(rt, torch):
    x = normal(1, 2, 700)
    rec = (np.zeros((2, 3), np.float32), np.full((2, 3), -1, np.int32), None)
    d = Distill(rt, torch, x, "f32", rec, np.array([-1, -5], np.int32), 1.0, 1.0, 1.0)
    loss, g = d.fused()
    assert not loss.any() and not g.any()
    tv = np.full((2, 3), -np.inf, np.float32)
    d = Distill(rt, torch, x, "f32", (tv, np.arange(6, dtype=np.int32).reshape(2, 3), None), None, 1.0, 1.0, 1.0)
    loss, g = d.fused()
    assert not loss.any() and not g.any()


def test_distill_whole_vocabulary_has_no_tail(rt, torch):
    """The record names every token: p_T = 0, and the tail bucket is left out."""
    x = normal(1, 3, 64)
    check_distill(rt, torch, x, "f32", 64, 1.0, 1.0, 0.0, True, None)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_against_differences(rt, torch, tail):
    """Central differences of the 64-bit loss at h = 1e-4: truncation h^2 / 6
    times a third derivative below 10, rounding 1e-15 / h."""
    x = normal(2, 4, 23, 1.0)
    y = some_labels(4, 23)
    tau, kd, ce, h = 1.6, 0.6, 0.4, 1e-4
    rec = record_of(3, x, 5, tau, tail)
    d = Distill(rt, torch, x, "f32", rec, y, tau, kd, ce)
    _, g = d.fused()
    num = np.zeros_like(g)
    for i in range(23):
        up, down = d.x64.copy(), d.x64.copy()
        up[:, i] += h
        down[:, i] -= h
        num[:, i] = (loss64(up, rec, y, tau, kd, ce)[0] - loss64(down, rec, y, tau, kd, ce)[0]) / (2 * h)
    assert np.all(np.abs(g - num) <= 4 * (2 * REL + 8 * ULP * 40) + 10 * h * h)


def test_distill_hard_targets_equal_cross_entropy(rt, torch):
    """kd = 0, ce = 1 is the LM step's cross-entropy and its gradient."""
    x = normal(5, 6, 1024)
    y = some_labels(6, 1024)
    y[2] = 7
    d = Distill(rt, torch, x, "f32", record_of(1, x, 2, 1.0, False), y, 1.0, 0.0, 1.0)
    loss, g = d.fused(scale=1 / 6)
    t = torch.from_numpy(d.x64).requires_grad_(True)
    ref = torch.nn.functional.cross_entropy(t, torch.from_numpy(y.astype(np.int64)))
    ref.backward()
    assert abs(loss.mean() - float(ref)) <= 4 * REL
    assert np.all(np.abs(g - t.grad.numpy()) <= 4 * REL / 6)


def test_distill_reports_bad_indices(rt, torch):
    x = normal(1, 2, 300)
    rec = list(record_of(1, x, 3, 1.0, False))
    rec[1][1, 1] = 300
    d = Distill(rt, torch, x, "f32", rec, None, 1.0, 1.0, 0.0)
    assert rt.distill_forward_device(*d.args, d.loss.data_ptr(), d.stats.data_ptr()), rt.last_error
    assert not rt.synchronize()
    assert rt.last_error.startswith("INVALID_DISTILL_INDEX")
    assert rt.synchronize(), rt.last_error  # reported once
    d = Distill(rt, torch, x, "f32", record_of(1, x, 3, 1.0, False), np.array([1, 300], np.int32), 1.0, 1.0, 1.0)
    assert rt.distill_forward_backward_device(*d.args, d.loss.data_ptr(), d.grad.data_ptr(), 302), rt.last_error
    assert not rt.synchronize()
    assert rt.last_error.startswith("INVALID_DISTILL_INDEX")


# -- sampling -------------------------------------------------------------------------

def sample(rt, torch, x, dtype, u, t=None, k=None, p=None, mp=None, pad=0, shift=0, log_probs=True):
    view, x64 = to_device(torch, x, dtype, pad, shift)
    rows, vocab = x.shape
    up = lambda a, d: None if a is None else torch.tensor(np.broadcast_to(np.asarray(a, d), rows).copy(), device="cuda")  # noqa: E731
    args = [up(u, np.float32), up(t, np.float32), up(k, np.int32), up(p, np.float32), up(mp, np.float32)]
    tok = torch.full((rows,), -7, device="cuda", dtype=torch.int32)
    lp = torch.full((rows,), -7.0, device="cuda")
    ptr = [0 if a is None else a.data_ptr() for a in args]
    ok = rt.sample_logits_device(CODES[dtype], rows, vocab, view.data_ptr(), vocab + pad, ptr[0], tok.data_ptr(),
                                 lp.data_ptr() if log_probs else 0, *ptr[1:])
    assert ok, rt.last_error
    assert rt.synchronize(), rt.last_error
    return tok.cpu().numpy(), lp.double().cpu().numpy(), view.float().cpu().numpy()


def check_sample(rt, torch, x, dtype, u, t=None, k=None, p=None, mp=None, pad=0, shift=0):
    """The token lies where the definition puts it, within the rounding of the
    masses: expf within 2 ulp and the floor of 2^31 times it, so a prefix mass
    (of the largest token's 1) is within 4 * 2^-23 of itself plus V 2^-31."""
    tok, lp, l = sample(rt, torch, x, dtype, u, t, k, p, mp, pad, shift)
    rows, vocab = x.shape
    full = lambda a, d: np.broadcast_to(np.asarray(d if a is None else a, np.float64), rows)  # noqa: E731
    U, T, K, P, M = full(np.float32(u) if np.isscalar(u) else u, 0), full(t, 1), full(k, 0), full(p, 1), full(mp, 0)
    for r in range(rows):
        m = l[r].max()
        if not (T[r] > 0 and np.isfinite(T[r])):
            assert tok[r] == int(np.argmax(l[r])) and lp[r] == 0.0
            continue
        y = (m - l[r]) * np.float32(np.float32(1) / np.float32(T[r]))
        order = np.argsort(y, kind="stable")
        mass = np.exp(-y.astype(np.float64))[order].cumsum()
        eps = lambda v: 4 * ULP * v + vocab * 2.0 ** -31 + 1e-12  # noqa: E731
        n = int(K[r]) if 0 < K[r] < vocab else vocab
        lo, hi = mass[n - 1] - eps(mass[n - 1]), mass[n - 1] + eps(mass[n - 1])
        if P[r] < 1:
            lo = mass[min(np.searchsorted(mass, P[r] * lo - eps(lo)), vocab - 1)] - eps(lo)
            hi = mass[min(np.searchsorted(mass, P[r] * hi + eps(hi)), vocab - 1)] + eps(hi)
        if M[r] > 0:
            w = np.exp(-y.astype(np.float64))[y <= max(0.0, -np.log(np.float32(M[r])) * (1 + 2 * ULP))].sum()
            lo, hi = min(lo, w - eps(w)), min(hi, w + eps(w))
        at = int(np.nonzero(order == tok[r])[0][0])
        before = mass[at - 1] if at else 0.0
        assert before <= U[r] * hi + eps(hi), (r, at, before, U[r], hi)
        assert mass[at] >= U[r] * lo - eps(hi), (r, at, mass[at], U[r], lo)
        assert before < hi
        want = -float(y[tok[r]])
        assert want - np.log(hi) - 4 * ULP * (1 - want) - 1e-6 <= lp[r] <= want - np.log(max(lo, 1e-300)) + 4 * ULP * (1 - want) + 1e-6


SETTINGS = [dict(), dict(t=0.7), dict(k=1), dict(k=40), dict(k=300), dict(p=0.9), dict(p=0.0), dict(mp=0.1), dict(mp=1.0),
            dict(t=1.4, k=100, p=0.95), dict(t=0.8, k=5000, p=0.8, mp=0.01), dict(t=0.0), dict(t=50.0, p=0.99)]


@pytest.mark.parametrize("setting", range(len(SETTINGS)))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (6, 33), (17, 1000), (16, 1024), (5, 1025), (6, 5000),
                                        (4, 16385), (3, 50001), (2, 131071), (1, 262144)])
def test_sample_sizes(rt, torch, rows, vocab, setting):
    rng = np.random.default_rng(vocab + setting)
    x = normal(vocab, rows, vocab)
    u = rng.random(rows, np.float32)
    check_sample(rt, torch, x, ("f32", "bf16", "f16")[setting % 3], u, **SETTINGS[setting])


@pytest.mark.parametrize("pad,shift", [(0, 1), (1, 0), (5, 3)])
@pytest.mark.parametrize("vocab", [61, 1024, 3001, 33000])
def test_sample_strides(rt, torch, vocab, pad, shift):
    u = np.random.default_rng(vocab).random(6, np.float32)
    for dtype in ("f32", "f16"):
        check_sample(rt, torch, normal(vocab, 6, vocab), dtype, u, t=[1, 0.5, 0, 2, 1, 1], k=[0, 5, 3, 0, 0, 600],
                     p=[0.9, 1, 1, 0.8, 1, 0.7], mp=[0, 0.1, 0, 0, 0.02, 0], pad=pad, shift=shift)


@pytest.mark.parametrize("vocab", [40, 1024, 3000, 40000])
@pytest.mark.parametrize("kind", ["equal", "near", "steps", "masked", "one", "sure"])
def test_sample_flat_tied_and_masked_rows(rt, torch, vocab, kind):
    rows = 6
    rng = np.random.default_rng(vocab)
    x = np.zeros((rows, vocab), np.float32)
    if kind == "near":  # an untrained model: every logit nearly the same
        x[:] = 0.01 * rng.standard_normal(x.shape)
    elif kind == "steps":
        x[:] = rng.integers(0, 9, x.shape) - 4
    elif kind == "masked":
        x[:] = -np.inf
        for r in range(rows):
            x[r, rng.integers(0, vocab, 7)] = rng.standard_normal(7)
    elif kind == "one":
        x[:] = -np.inf
        x[:, vocab - 2] = 3.0
    elif kind == "sure":
        x[:] = normal(1, rows, vocab, 1.0)
        x[:, 3] = 40.0
    u = np.array([0.0, 0.1, 0.37, 0.5, 0.93, 1 - 2.0 ** -24], np.float32)
    for s in (dict(), dict(p=0.9), dict(k=17), dict(k=700, p=0.5), dict(mp=0.3), dict(t=0.3)):
        check_sample(rt, torch, x, "f32", u, **s)


def test_sample_dead_rows(rt, torch):
    x = normal(2, 5, 3000)
    x[0] = -np.inf
    x[1, 9] = np.nan
    x[2, 7] = np.inf
    x[3] = np.nan
    tok, lp, _ = sample(rt, torch, x, "f32", 0.5)
    assert list(tok[:4]) == [-1, -1, -1, -1] and tok[4] >= 0
    assert lp[0] == -np.inf and np.all(np.isnan(lp[1:4])) and np.isfinite(lp[4])


def test_sample_follows_the_distribution(rt, torch):
    """Evenly spaced random numbers: every token is drawn n p times, within one
    at either end of its interval."""
    n, vocab = 4096, 50
    x = np.repeat(normal(8, 1, vocab, 1.0), n, 0)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    for s in (dict(), dict(k=7), dict(p=0.6), dict(mp=0.2), dict(t=2.0)):
        tok, lp, l = sample(rt, torch, x, "f32", u, **s)
        seen = np.bincount(tok, minlength=vocab)
        prob = np.zeros(vocab)
        prob[tok] = np.exp(lp)
        assert abs(prob.sum() - 1) < 1e-5 or (seen == 0).sum() > 0
        assert np.all(np.abs(seen - n * prob)[seen > 0] <= 2)


@pytest.mark.parametrize("vocab", [50, 1024, 20000])
def test_sample_agrees_with_the_host_sampler(rt, torch, vocab):
    """The same tokens as hx_sample_next_token for its own random numbers, but
    where one falls within rounding of a boundary (counted: at most one in the
    64 rows)."""
    rows = 64
    x = normal(vocab, rows, vocab, 2.0)
    mask = (1 << 64) - 1

    def u_of(seed, step):
        v = (seed + step * 0x9E3779B97F4A7C15 + 0x9E3779B97F4A7C15) & mask
        v = ((v ^ (v >> 30)) * 0xBF58476D1CE4E5B9) & mask
        v = ((v ^ (v >> 27)) * 0x94D049BB133111EB) & mask
        return ((v ^ (v >> 31)) >> 11) * 2.0 ** -53

    for t, k in ((1.0, 0), (0.7, 10), (1.3, 500)):
        want = [hx.sample_next_token(x[r], step=3, greedy=False, temperature=t, top_k=k, seed=r)[0] for r in range(rows)]
        u = np.array([u_of(r, 3) for r in range(rows)], np.float32)
        tok, _, _ = sample(rt, torch, x, "f32", u, t=t, k=k)
        assert (tok != np.array(want)).sum() <= 1
    tok, _, _ = sample(rt, torch, x, "f32", u, t=0.0)
    assert np.array_equal(tok, [hx.sample_next_token(x[r])[0] for r in range(rows)])


# -- all ---------------------------------------------------------------------------------

def test_same_results_on_every_call_and_stream(rt, torch):
    x = normal(4, 7, 40000)
    u = np.random.default_rng(1).random(7, np.float32)
    first = sample(rt, torch, x, "bf16", u, p=0.9), top(rt, torch, x, "bf16", 50)
    rec, y = record_of(1, x, 11, 2.0, True), some_labels(7, 40000)
    loss, grad = Distill(rt, torch, x, "bf16", rec, y, 2.0, 0.5, 0.5).fused()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    other = hx.Runtime()
    assert other.initialize(0), other.last_error
    with torch.cuda.stream(side):
        assert other.set_stream(side.cuda_stream), other.last_error
        again = sample(other, torch, x, "bf16", u, p=0.9), top(other, torch, x, "bf16", 50)
        loss2, grad2 = Distill(other, torch, x, "bf16", rec, y, 2.0, 0.5, 0.5).fused()
    side.synchronize()
    other.close()
    for a, b in zip(first, again):
        assert all(np.array_equal(p, q) for p, q in zip(a, b))
    assert np.array_equal(loss, loss2) and np.array_equal(grad, grad2)


def test_no_rows_and_no_log_probs(rt, torch):
    assert rt.top_logits_device(0, 0, 10, 0, 10, 2, 0, 0), rt.last_error
    assert rt.sample_logits_device(0, 0, 10, 0, 10, 0, 0), rt.last_error
    assert rt.distill_forward_device(0, 0, 10, 0, 10, 2, 0, 0, 0, 0, 1.0, 1.0, 0.0, 0, 0), rt.last_error
    tok, lp, _ = sample(rt, torch, normal(1, 3, 99), "f32", 0.5, log_probs=False)
    assert np.all(tok >= 0) and np.all(lp == -7.0)


def test_offsets_beyond_32_bits(rt, torch):
    """Rows that start more than 2^31 elements into the buffer."""
    vocab, rows, stride = 1500, 3, (1 << 30) + 12
    buf = torch.empty(2 * stride + vocab, device="cuda", dtype=torch.bfloat16)
    view = buf.as_strided((rows, vocab), (stride, 1))
    view.copy_(torch.from_numpy(normal(1, rows, vocab)).to("cuda"))
    x = view.float().cpu().numpy().astype(np.float64)
    v = torch.empty(rows, 5, device="cuda")
    i = torch.empty(rows, 5, device="cuda", dtype=torch.int32)
    assert rt.top_logits_device(1, rows, vocab, view.data_ptr(), stride, 5, v.data_ptr(), i.data_ptr()), rt.last_error
    u = torch.full((rows,), 0.5, device="cuda")
    tok = torch.empty(rows, device="cuda", dtype=torch.int32)
    assert rt.sample_logits_device(1, rows, vocab, view.data_ptr(), stride, u.data_ptr(), tok.data_ptr()), rt.last_error
    assert rt.synchronize(), rt.last_error
    order = np.argsort(-x, axis=1, kind="stable")
    assert np.array_equal(i.cpu().numpy(), order[:, :5])
    for r in range(rows):
        p = np.exp(x[r] - x[r].max())[order[r]].cumsum()
        at = int(np.nonzero(order[r] == int(tok[r]))[0][0])
        assert (p[at - 1] if at else 0) <= 0.5 * p[-1] * 1.00001 and p[at] >= 0.5 * p[-1] * 0.99999


def test_refusals(rt, torch):
    x = normal(1, 2, 64)
    view, _ = to_device(torch, x, "f32")
    out = torch.empty(4096, device="cuda")
    o, lp = out.data_ptr(), view.data_ptr()

    def refused(call, *a, has):
        assert not call(*a)
        assert has in rt.last_error, rt.last_error

    t = rt.top_logits_device
    refused(t, 3, 2, 64, lp, 64, 2, o, o, has="unknown logit type")
    refused(t, 0, 2, 0, lp, 64, 2, o, o, has="empty vocabulary")
    refused(t, 0, 2, 262145, lp, 262145, 2, o, o, has="not supported")
    refused(t, 0, 2, 64, lp, 63, 2, o, o, has="row stride")
    refused(t, 0, 2, 64, 0, 64, 2, o, o, has="null logits")
    refused(t, 0, 2, 64, lp + 2, 64, 2, o, o, has="not aligned")
    refused(t, 0, 2, 64, lp, 64, 0, o, o, has="k must be")
    refused(t, 0, 2, 64, lp, 64, 65, o, o, has="k must be")
    refused(t, 0, 2, 300, lp, 300, 257, o, o, has="k must be")
    refused(t, 0, 2, 64, lp, 64, 2, 0, o, has="null output")
    for tau in (0.0, -1.0, float("nan"), float("inf"), 1e-45):
        refused(t, 0, 2, 64, lp, 64, 2, o, o, o, tau, has="temperature")
    s = rt.sample_logits_device
    refused(s, 0, 2, 64, lp, 64, 0, o, has="null random numbers")
    refused(s, 0, 2, 64, lp, 64, o, 0, has="null random numbers")
    refused(s, 7, 2, 64, lp, 64, o, o, has="unknown logit type")
    f, b, fb = rt.distill_forward_device, rt.distill_backward_device, rt.distill_forward_backward_device
    refused(f, 0, 2, 64, lp, 64, 2, 0, o, 0, 0, 1.0, 1.0, 0.0, o, o, has="null teacher")
    refused(f, 0, 2, 64, lp, 64, 2, o, o, 0, 0, 1.0, 1.0, 0.0, o, 0, has="null output")
    refused(f, 0, 2, 64, lp, 64, 300, o, o, 0, 0, 1.0, 1.0, 0.0, o, o, has="record length")
    refused(f, 0, 2, 64, lp, 64, 2, o, o, 0, 0, 0.0, 1.0, 0.0, o, o, has="temperature")
    refused(f, 0, 2, 64, lp, 64, 2, o, o, 0, 0, 1.0, float("nan"), 0.0, o, o, has="weights")
    refused(b, 0, 2, 64, lp, 64, 2, o, o, 0, 0, 1.0, 1.0, 0.0, 0, o, 64, has="null statistics")
    refused(b, 0, 2, 64, lp, 64, 2, o, o, 0, 0, 1.0, 1.0, 0.0, o, o, 63, has="gradient row stride")
    refused(fb, 0, 2, 64, lp, 64, 2, o, o, 0, 0, 1.0, 1.0, 0.0, o, o + 2, 64, has="gradient not aligned")
    refused(fb, 0, 2, 64, lp, 64, 2, o, o, 0, 0, 1.0, 1.0, 0.0, o, lp, 65, has="in place")
    assert rt.synchronize(), rt.last_error


def test_uninitialised_runtime_fails_closed():
    r = hx.Runtime()
    assert not r.top_logits_device(0, 1, 4, 0, 4, 1, 0, 0)
    assert r.last_error == "runtime not initialized"
