"""The operators on device logits at their limits: the shapes, masks and records that
leave a kernel little room.  Tolerances as in test_head_ops_gpu.py."""
import numpy as np
import pytest

from test_head_ops_gpu import (CODES, REL, ROUND, ULP, Distill, check_sample, normal, record_of,  # noqa: F401
                               check_distill, check_top, loss64, lse64, rt,
                               sample, some_labels, to_device, top, torch)

pytestmark = pytest.mark.gpu


# -- many rows to a block, wide records ----------------------------------------------

@pytest.mark.parametrize("rows,vocab,k,pad", [(2500, 2100, 255, 0), (2500, 4096, 256, 0), (1500, 4093, 256, 3),
                                              (40, 150000, 256, 0), (40, 140001, 213, 3), (30, 262144, 224, 1),
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


# -- the tail bucket where the student has no mass for it --------------------------------

def soft64(x, record, tau, kd):
    """(loss, its derivative) of the record's part alone, from the definition: where
    p_T = 0 or q_T = 0 the bucket is left out, and sum q need not be 1."""
    tv, ti, tl = record
    rows = x.shape[0]
    z = x / tau
    logp = z - lse64(z)[:, None]
    p = np.exp(logp)
    loss, grad = np.zeros(rows), np.zeros_like(x)
    for r in range(rows):
        on = ti[r] >= 0
        ids = ti[r, on]
        logq = tv[r, on].astype(np.float64) / tau - np.float64(tl[r])
        q = np.exp(logq)
        loss[r] = (q * (logq - logp[r, ids]))[q > 0].sum()
        mass = q.sum()
        out = np.ones(x.shape[1], bool)
        out[ids] = False
        qt, pt = max(0.0, 1.0 - mass), p[r, out].sum()
        g = np.zeros(x.shape[1])
        if qt > 0 and pt >= 2.0 ** -126:  # (less is no mass in float32)
            loss[r] += qt * np.log(qt / pt)
            g[out] -= qt / pt * p[r, out]
            mass += qt
        g += mass * p[r]
        g[ids] -= q
        grad[r] = tau * g
    return kd * tau * tau * loss, kd * grad


NO_MASS = ["masked", "below", "sure", "whole"]


def no_mass_case(vocab, kind, k=9):
    """Rows whose tokens outside the record are masked, or too far below to have mass;
    a record whose entries add up to more than 1; one that names every token."""
    rows = 5
    x = normal(vocab + 1, rows, vocab, 1.0)
    if kind == "whole":
        k = min(vocab, 256)
    ti = np.stack([np.random.default_rng(r).permutation(vocab)[:k] for r in range(rows)]).astype(np.int32)
    tv = normal(k, rows, k, 1.0)
    tl = (lse64(tv.astype(np.float64) / 2.0) + (-0.3 if kind == "sure" else 0.4)).astype(np.float32)
    for r in range(rows - 1):  # the last row keeps its tail
        out = np.ones(vocab, bool)
        out[ti[r]] = False
        if kind in ("masked", "whole"):
            x[r, out] = -np.inf
        elif kind == "below":
            x[r, out] -= 2.0 * 120
    return x, (tv, ti, tl)


@pytest.mark.parametrize("kind", NO_MASS)
@pytest.mark.parametrize("vocab", [60, 1000, 1900, 9000, 40000])
def test_distill_gradient_without_a_tail(rt, torch, vocab, kind):  # noqa: F811
    """Loss and gradient, fused and from statistics, with and without labels.  The loss
    is a sum of q times log-probabilities, each off by REL and the roundings of its size;
    the gradient one of probabilities, each within 2 REL."""
    x, rec = no_mass_case(vocab, kind)
    tau, kd = 2.0, 0.7
    mass = np.exp(rec[0].astype(np.float64) / tau - rec[2][:, None]).sum(1).max()
    tol = 4 * (2 * REL + 8 * ULP * 30) * max(1.0, mass)
    for labels, ce in ((None, 0.0), (np.ascontiguousarray(rec[1][:, 0]), 0.3)):
        hard = loss64(x.astype(np.float64), rec, labels, tau, 0.0, ce)
        want, grad = soft64(x.astype(np.float64), rec, tau, kd)
        want, grad = want + hard[0], grad + hard[2]
        d = Distill(rt, torch, x, "f32", rec, labels, tau, kd, ce)
        loss, stats = d.forward()
        assert np.all(np.abs(loss - want) <= tol * (kd * tau * tau + ce) * 4)
        assert not stats[:-1, 2].any()
        for g in (d.backward(), d.fused()[1]):
            assert np.all(np.abs(g - grad) <= tol * (kd * tau + ce)), np.abs(g - grad).max()
            assert np.all(np.abs(g.sum(1)) <= tol * (kd * tau + ce) * 4)  # a softmax's gradient


@pytest.mark.parametrize("kind", ["masked", "sure"])
def test_distill_gradient_without_a_tail_against_differences(rt, torch, kind):  # noqa: F811
    """Central differences of the 64-bit loss, as for the rows with a tail."""
    x, rec = no_mass_case(40, kind)
    tau, kd, h = 2.0, 0.7, 1e-4
    d = Distill(rt, torch, x, "f32", rec, None, tau, kd, 0.0)
    _, g = d.fused()
    num = np.zeros_like(g)
    for i in range(40):
        up, down = d.x64.copy(), d.x64.copy()
        up[:, i] += h
        down[:, i] -= h
        num[:, i] = (loss64(up, rec, None, tau, kd, 0.0)[0] - loss64(down, rec, None, tau, kd, 0.0)[0]) / (2 * h)
    assert np.all(np.abs(g - num) <= 4 * (2 * REL + 8 * ULP * 40) * 2 + 10 * h * h)


# -- rows without targets ----------------------------------------------------------------

@pytest.mark.parametrize("value", [-np.inf, np.inf, np.nan, np.finfo(np.float32).min])
@pytest.mark.parametrize("rows,vocab", [(4, 50), (5, 1000), (5, 1900), (7, 9000), (300, 9001), (5, 40000)])
def test_distill_rows_without_targets_are_zero(rt, torch, rows, vocab, value):  # noqa: F811
    """Whatever their logits: one odd logit, or all of them."""
    x = normal(vocab, rows, vocab)
    x[0, vocab // 3] = value
    x[1] = value
    x[2, ::2] = value
    rec = list(record_of(1, normal(5, rows, vocab), 5, 1.0, True, short=False))
    y = some_labels(rows, vocab)
    rec[1][:3] = -1
    y[:3] = -1
    for tail in (False, True):
        for tau, kd, ce, labels in ((1.0, 1.0, 1.0, y), (2.0, 0.5, 0.5, y), (2.0, 1.0, 0.0, None), (1.0, 0.0, 1.0, y)):
            for dtype in ("f32", "bf16"):
                d = Distill(rt, torch, x, dtype, (rec[0], rec[1], rec[2] if tail else None), labels, tau, kd, ce)
                loss, _ = d.forward()
                back = d.backward()
                loss2, g = d.fused()
                for z in (loss[:3], loss2[:3], back[:3], g[:3]):
                    assert not z.any()
                assert np.all(np.isfinite(g[3:])) and g[3:].any() and np.all(np.isfinite(loss2[3:]))


# -- log-sum-exp of masked rows ------------------------------------------------------------

def far_masked(rows, vocab, low, rest, value=-np.inf, count=500):
    """Rows masked but for a few logits about `low`, none at the first token or at any of
    32 evenly spaced places: two at low, the others at rest."""
    rng = np.random.default_rng(vocab)
    places = set((np.arange(32) * vocab // 32).tolist())
    free = np.array([i for i in range(vocab) if i not in places])
    x = np.full((rows, vocab), value, np.float32)
    for r in range(rows):
        at = rng.permutation(free)[:min(count, len(free) // 2)]
        x[r, at] = rest
        x[r, at[:2]] = low
    return x


@pytest.mark.parametrize("value", [-np.inf, np.finfo(np.float32).min])
@pytest.mark.parametrize("rows,vocab", [(3, 100), (5, 1024), (5, 1030), (700, 2000), (5, 9000), (300, 9001), (4, 40000), (20, 140001)])
def test_log_sum_exp_of_far_masked_rows(rt, torch, rows, vocab, value):  # noqa: F811
    for low, rest, tau in ((-87.0, -87.6, 1.0), (-17.4, -17.52, 0.2), (-30.0, -31.0, 1.0), (-120.0, -121.0, 1.0),
                           (-87.0, -87.6, 2.0)):
        x = far_masked(rows, vocab, low, rest, value)
        check_top(rt, torch, x, "f32", 20, tau)
        tol = REL + 8 * ULP * 130 / min(tau, 1.0)
        assert np.all(np.abs(top(rt, torch, x, "f32", 20, tau)[2] - lse64(x.astype(np.float64) / tau)) <= tol)
        # the distillation's statistics, with no logit named but masked ones
        rec = (np.zeros((rows, 3), np.float32), np.full((rows, 3), -1, np.int32), None)
        rec[1][::2, 0] = 0
        d = Distill(rt, torch, x, "f32", rec, np.full(rows, -1, np.int32), tau, 0.5, 0.5)
        _, stats = d.forward()
        z = x.astype(np.float64)
        for got, want in ((stats[:, 0], lse64(z / tau)), (stats[:, 1], lse64(z))):
            assert np.all(np.abs(got - want) <= tol), np.abs(got - want).max()


# -- rows at the type's lowest value ----------------------------------------------------

LOWEST = [("f32", float(np.finfo(np.float32).min)), ("bf16", -float.fromhex("0x1.fep127")), ("f16", -65504.0),
          ("f32", -1e30), ("f32", -1e9), ("bf16", -1e9), ("f32", -1e7), ("f32", -1e4), ("f32", 3e38)]


@pytest.mark.parametrize("dtype,lowest", LOWEST)
@pytest.mark.parametrize("vocab", [40, 1000, 1024, 1900, 9000, 40000])
def test_rows_at_the_lowest_value(rt, torch, vocab, dtype, lowest):  # noqa: F811
    """Every logit masked by the type's lowest, or another low value: the softmax is uniform.  The same
    row less its maximum, in 64 bits, has the same loss and gradient."""
    rows = 5
    x = np.full((rows, vocab), lowest, np.float32)
    x[3, 1::2] = -np.inf
    x[4] = normal(2, 1, vocab)[0]
    for tau in (1.0, 2.0, 1.5):
        v, i, s, x64 = top(rt, torch, x, dtype, 7, tau)
        assert np.array_equal(i[:3], np.broadcast_to(np.arange(7), (3, 7))) and np.array_equal(i[3], np.arange(7) * 2)
        want = lse64(x64 / tau)
        assert np.all(np.abs(s - want) <= REL + 8 * ULP * np.abs(want))
        rec = record_of(3, normal(4, rows, vocab), 6, tau, False, short=False)
        rec[1][3] = rec[1][3] // 2 * 2
        rec[1][3, 1:] = -1
        y = np.array([rec[1][0, 2], 5, -1, 4, 3], np.int32)
        for kd, ce, labels in ((0.5, 0.5, y), (1.0, 0.0, None), (0.0, 1.0, y)):
            d = Distill(rt, torch, x, dtype, rec, labels, tau, kd, ce)
            want, _, grad = loss64(x64 - x64.max(1, keepdims=True), rec, labels, tau, kd, ce)
            size = (2 * REL + 8 * ULP * 40) * (kd * tau * max(tau, 1.0) + ce)
            for loss in (d.forward()[0], d.fused()[0]):
                assert np.all(np.abs(loss - want) <= 4 * size + 4 * ULP * np.abs(want)), (loss, want)
            g = d.fused()[1]
            assert np.all(np.abs(g - grad) <= 4 * size + ROUND[dtype] * np.abs(grad) + 6e-8), np.abs(g - grad).max()
            assert np.all(np.isfinite(d.backward()))


# -- infinity and NaN in one row -----------------------------------------------------------

@pytest.mark.parametrize("vocab", [50, 1024, 3000, 40000])
def test_top_nan_beside_infinity(rt, torch, vocab):  # noqa: F811
    """The largest logit is +inf, the log-sum-exp NaN: a NaN takes part in it."""
    x = normal(3, 4, vocab)
    x[0, 7] = x[1, 7] = np.inf
    x[1, vocab - 1] = np.nan
    x[2, 7] = np.nan
    for dtype in ("f32", "bf16", "f16"):
        v, i, s, _ = top(rt, torch, x, dtype, 3)
        assert i[0, 0] == 7 and i[1, 0] == 7 and np.all(np.isfinite(v[:2, 1:]))
        assert s[0] == np.inf and np.isnan(s[1]) and np.isnan(s[2]) and np.isfinite(s[3])


# -- a tail at the edge of float32 ---------------------------------------------------------

@pytest.mark.parametrize("vocab", [300, 1000, 1900, 9000, 40000])
def test_distill_tail_at_the_edge_of_float32(rt, torch, vocab):  # noqa: F811
    """200 equal named logits and one other token: its share is 2^-133 or 2^-132, below what
    a float32 quotient holds, then 2^-114."""
    k, tau, kd = 200, 1.0, 0.5
    x = np.full((3, vocab), -np.inf, np.float32)
    x[:, :k] = 0.0
    x[:, k] = (-87.0, -86.5, -74.0)
    rec = (np.zeros((3, k), np.float32), np.broadcast_to(np.arange(k, dtype=np.int32), (3, k)).copy(),
           np.full(3, np.log(k) + 0.5, np.float32))
    want, grad = soft64(x.astype(np.float64), rec, tau, kd)
    d = Distill(rt, torch, x, "f32", rec, None, tau, kd, 0.0)
    tol = 4 * (2 * REL + 8 * ULP * 100)
    for g in ((d.forward(), d.backward())[1], d.fused()[1]):
        assert np.all(np.abs(g - grad) <= tol * kd), np.abs(g - grad).max()
    assert np.all(np.abs(d.fused()[0] - want) <= tol * kd * 4)


# -- a teacher's row without logits ----------------------------------------------------------

@pytest.mark.parametrize("vocab", [50, 1000, 9000, 40000])
def test_distill_teacher_row_of_masked_logits(rt, torch, vocab):  # noqa: F811
    """The record of a row that the teacher masks as a whole: values and log-sum-exp -inf.
    There is no KL term, in either form of the record."""
    rows, k = 4, 6
    x = normal(vocab, rows, vocab)
    t = normal(8, rows, vocab)
    t[0] = t[1] = -np.inf
    v, i, s, _ = top(rt, torch, t, "f32", k, 2.0)
    assert np.all(v[:2] == -np.inf) and np.all(s[:2] == -np.inf)
    y = np.array([-1, 3, 5, -1], np.int32)
    for tail in (False, True):
        rec = (v.astype(np.float32), i, s.astype(np.float32) if tail else None)
        empty = (rec[0], np.where(np.arange(rows)[:, None] < 2, -1, i).astype(np.int32), rec[2])
        a = Distill(rt, torch, x, "f32", rec, y, 2.0, 0.5, 0.5)
        b = Distill(rt, torch, x, "f32", empty, y, 2.0, 0.5, 0.5)
        tol = 4 * (2 * REL + 8 * ULP * 40)  # (their exponentials are taken against other logits)
        assert np.all(np.abs(a.forward()[0] - b.forward()[0]) <= tol * 4)
        assert np.all(np.abs(a.backward() - b.backward()) <= tol)
        (la, ga), (lb, gb) = a.fused(), b.fused()
        assert np.all(np.abs(la - lb) <= tol * 4) and np.all(np.abs(ga - gb) <= tol)
        assert la[0] == 0 and not ga[0].any() and np.all(np.isfinite(ga))


# -- a reference far from the row's largest logit ---------------------------------------------

@pytest.mark.parametrize("above", [60.0, 200.0])
@pytest.mark.parametrize("rows,vocab", [(3, 60), (4, 1000), (4, 1900), (5, 9000), (300, 9001), (5, 40000), (20, 140001)])
def test_distill_student_far_from_the_teacher(rt, torch, rows, vocab, above):  # noqa: F811
    """A token that neither record nor label names lies far above all that they do: the
    sums against a named logit overflow, and are formed again against the maximum."""
    for tail in (False, True):
        for tau, kd, ce in ((1.0, 0.6, 0.4), (2.0, 0.5, 0.5), (2.0, 1.0, 0.0)):
            x = normal(vocab, rows, vocab, 1.0)
            rec = record_of(6, x, 7, tau, tail)
            y = some_labels(rows, vocab) if ce else None
            for r in range(0, rows, 2 if rows < 100 else 7):
                named = set(rec[1][r].tolist()) | ({int(y[r])} if ce else set())
                x[r, next(i for i in range(vocab // 2, vocab) if i not in named)] = above * tau
            check_distill(rt, torch, x, "f32", 7, tau, kd, ce, tail, y, record=rec)


@pytest.mark.parametrize("above", [45.0, 200.0])
@pytest.mark.parametrize("rows,vocab", [(4, 1500), (5, 9000), (300, 9001), (5, 40000), (20, 140001)])
def test_top_spike_away_from_the_sample(rt, torch, rows, vocab, above):  # noqa: F811
    x = normal(vocab, rows, vocab, 1.0)
    x[::2, vocab // 2 + 1] = above
    for tau in (1.0, 0.5):
        check_top(rt, torch, x, "f32", 9, tau)


# -- sampling: the probabilities of the kept tokens ----------------------------------------------

def test_sample_probabilities_of_the_kept_tokens(rt, torch):  # noqa: F811
    """Evenly spaced random numbers draw every kept token of more than one step's mass and
    no other, each with its probability among the kept."""
    n, vocab = 4096, 50
    x = np.repeat(normal(8, 1, vocab, 1.0), n, 0)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    for s in (dict(), dict(k=7), dict(p=0.6), dict(mp=0.2), dict(t=2.0)):
        tok, lp, l = sample(rt, torch, x, "f32", u, **s)
        y = (l[0].max() - l[0].astype(np.float64)) / s.get("t", 1.0)
        order = np.argsort(y, kind="stable")
        mass = np.exp(-y[order])
        keep = np.arange(vocab) < s.get("k", vocab)
        total = mass[keep].sum()
        keep &= mass.cumsum() - mass < s.get("p", 2.0) * total
        keep &= mass >= s.get("mp", 0.0)
        prob = np.zeros(vocab)
        prob[order[keep]] = mass[keep] / mass[keep].sum()
        seen = np.bincount(tok, minlength=vocab)
        assert np.all(prob[seen > 0] > 0) and np.all(prob[seen == 0] <= 1.01 / n)
        assert np.all(np.abs(lp - np.log(prob[tok])) <= 1e-5)


# -- sampling: the two zeros -------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab", [(40, 2), (40, 7), (20, 300), (9, 1024), (9, 4100), (5, 40000), (300, 9001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_sample_both_zeros_as_the_largest_logit(rt, torch, rows, vocab, dtype):  # noqa: F811
    """-0 and +0 are one logit: tokens of either are equally likely, in the order of their
    indices."""
    rng = np.random.default_rng(rows + vocab)
    x = -np.abs(normal(vocab, rows, vocab)) - np.float32(0.5)
    zeros = rng.random(x.shape) < 0.4
    zeros[:, vocab // 2] = True
    zeros[::5] = True
    x[zeros] = np.where(rng.random(x.shape) < 0.5, 0.0, -0.0)[zeros]
    u = rng.random(rows).astype(np.float32)
    for s in (dict(), dict(p=0.9), dict(k=17), dict(k=700, p=0.5), dict(mp=0.3), dict(t=0.3), dict(t=0.0)):
        check_sample(rt, torch, x, dtype, u, **s)
