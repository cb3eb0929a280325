"""Measured cases of the output-head operators: the largest logits of a row, the
distillation loss on them with its gradient, and sampling.

``run`` computes each operator in plain torch operations, or, where ``own`` is
true, through the framework's entry points.  ``exact`` gives the same outputs
from the definitions in 64-bit arithmetic.

  top      the k largest logits of every row, in order (value descending, index
           ascending), and log sum exp(l / tau): a teacher's record.
  fused    distillation loss and gradient in one pass: the training step.
  forward  the loss alone with the row statistics its backward needs.
  backward the gradient from those statistics and a gradient for every row's loss.
  sample   a token for every row from one given random number, with
           temperature, top-k, top-p and min-p of its own, and the token's
           log-probability among the kept ones.
"""
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one sequence of the small LM (64 tokens, vocabulary 1024): latency
        dict(name="fused_64x1024_f32", op="fused", rows=64, vocab=1024, dtype="f32", k=16, tau=2.0, kd=0.5, ce=0.5,
             tail=False, labels=True, pad=0),
        # the LM step of 512 sequences of 256 tokens, vocabulary 1024, soft targets only
        dict(name="fused_131072x1024_f32", op="fused", rows=131072, vocab=1024, dtype="f32", k=32, tau=1.0, kd=1.0,
             ce=0.0, tail=True, labels=False, pad=0),
        # a wide vocabulary in 16 bits, soft and hard targets at two temperatures
        dict(name="fused_4096x65536_bf16", op="fused", rows=4096, vocab=65536, dtype="bf16", k=64, tau=2.0, kd=0.9,
             ce=0.1, tail=True, labels=True, pad=0),
        # evaluation: the loss alone, an odd vocabulary in a padded buffer
        dict(name="forward_1000x50001_f32", op="forward", rows=1000, vocab=50001, dtype="f32", k=100, tau=1.5, kd=0.7,
             ce=0.3, tail=False, labels=True, pad=7),
        # the gradient where another program forms the rows' weights
        dict(name="backward_2048x32768_f16", op="backward", rows=2048, vocab=32768, dtype="f16", k=50, tau=1.0, kd=0.5,
             ce=0.5, tail=True, labels=True, pad=0),
        # a teacher answering one short sequence
        dict(name="top_16x1024_f32", op="top", rows=16, vocab=1024, dtype="f32", k=8, tau=1.0, pad=0),
        # the teacher's record of the LM step's batch
        dict(name="top_131072x1024_f32", op="top", rows=131072, vocab=1024, dtype="f32", k=32, tau=1.0, pad=0),
        # a wide teacher in 16 bits: many equal values
        dict(name="top_2048x131072_bf16", op="top", rows=2048, vocab=131072, dtype="bf16", k=128, tau=2.0, pad=0),
        # one stream of the small LM: latency
        dict(name="sample_1x1024_f32", op="sample", rows=1, vocab=1024, dtype="f32", kind="mixed", pad=0),
        # a serving batch, every request with settings of its own
        dict(name="sample_256x32768_f32", op="sample", rows=256, vocab=32768, dtype="f32", kind="mixed", pad=0),
        # a small batch over an odd wide vocabulary, nucleus only
        dict(name="sample_48x131071_bf16", op="sample", rows=48, vocab=131071, dtype="bf16", kind="nucleus", pad=1),
        # many rollouts drawn from the whole distribution
        dict(name="sample_4096x4096_f16", op="sample", rows=4096, vocab=4096, dtype="f16", kind="plain", pad=0),
    ]


def draw(rng):
    op = rng.choice(["top", "fused", "forward", "backward", "sample", "sample"])
    vocab = int(round(2 ** rng.uniform(5, 18)))
    most = min(17.0, 27.0 - torch.tensor(float(vocab)).log2().item())
    if op == "sample":
        most = min(most, 13.0)
    rows = int(2 ** rng.uniform(0, most))
    case = dict(op=op, rows=max(1, rows), vocab=vocab, dtype=rng.choice(["f32", "f32", "bf16", "f16"]),
                pad=rng.choice([0, 0, 0, 1, 3, 8, 29]))
    if op == "sample":
        case["kind"] = rng.choice(["mixed", "mixed", "nucleus", "plain", "topk"])
        return case
    case["k"] = min(vocab, int(round(2 ** rng.uniform(0, 8))))
    case["tau"] = rng.choice([1.0, 1.0, 2.0, 1.5, 4.0, 0.7])
    if op != "top":
        case["labels"] = rng.random() < 0.6
        case["kd"], case["ce"] = rng.choice([(1.0, 0.0), (0.5, 0.5), (0.9, 0.1)]) if case["labels"] else (1.0, 0.0)
        case["tail"] = rng.random() < 0.5
    return case


def work(case):
    r, v, b = case["rows"], case["vocab"], BYTES[case["dtype"]]
    logits = r * v * b
    if case["op"] == "sample":
        return {"bytes": logits + r * 28, "flops": 4.0 * r * v}
    if case["op"] == "top":
        return {"bytes": logits + r * (8 * case["k"] + 4), "flops": 4.0 * r * v}
    side = r * (8 * case["k"] + (4 if case["tail"] else 0) + (4 if case["labels"] else 0))
    if case["op"] == "forward":
        return {"bytes": logits + side + 16 * r, "flops": 6.0 * r * v}
    if case["op"] == "backward":
        return {"bytes": 2 * logits + side + 16 * r, "flops": 6.0 * r * v}
    return {"bytes": 2 * logits + side + 4 * r, "flops": 10.0 * r * v}


# -- inputs ------------------------------------------------------------------

def _logits(rows, vocab, pad, dtype, gen, spread=2.5):
    """A [rows, vocab] view of a [rows, vocab + pad] buffer: normal logits with
    a few favoured tokens per row, as a trained head gives them."""
    buf = torch.empty(rows, vocab + pad, device="cuda", dtype=DTYPES[dtype])
    step = max(1, (1 << 27) // (vocab + pad))
    for r0 in range(0, rows, step):
        part = torch.randn(min(step, rows - r0), vocab + pad, device="cuda", generator=gen) * spread
        high = torch.randint(0, vocab, (part.shape[0], 4), device="cuda", generator=gen)
        part.scatter_add_(1, high, torch.rand(part.shape[0], 4, device="cuda", generator=gen) * 8.0)
        buf[r0:r0 + step] = part
    return buf[:, :vocab]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r, v, op = case["rows"], case["vocab"], case["op"]
    s = dict(case, logits=_logits(r, v, case["pad"], case["dtype"], gen))
    f32 = dict(device="cuda", dtype=torch.float32)
    i32 = dict(device="cuda", dtype=torch.int32)
    if op == "sample":
        s.update(_sample_settings(case["kind"], r, gen))
        if case["kind"] == "mixed" and r >= 8:
            # every eighth row allows a few tokens only, and one row none
            allowed = torch.rand(r, v, device="cuda", generator=gen) < 8.0 / v
            rows = torch.arange(r, device="cuda")
            allowed[:, 0] |= rows % 8 == 3
            allowed |= (rows % 8 != 3)[:, None]
            allowed[5] = False
            s["logits"].masked_fill_(~allowed, float("-inf"))
        s["tokens"], s["log_probs"] = torch.empty(r, **i32), torch.empty(r, **f32)
        return s
    k = case["k"]
    if op == "top":
        s["values"], s["indices"], s["lse"] = torch.empty(r, k, **f32), torch.empty(r, k, **i32), torch.empty(r, **f32)
        return s
    # the teacher agrees with the student in part
    step = max(1, (1 << 27) // v)
    tv, ti, tl = [], [], []
    for r0 in range(0, r, step):
        x = s["logits"][r0:r0 + step].float()
        x = x * 0.8 + torch.randn(x.shape, device="cuda", generator=gen)
        top = torch.topk(x, k, dim=1)
        tv.append(top.values)
        ti.append(top.indices.to(torch.int32))
        tl.append(torch.logsumexp(x / case["tau"], dim=1))
    s["teacher_values"], s["teacher_indices"] = torch.cat(tv).contiguous(), torch.cat(ti).contiguous()
    s["teacher_lse"] = torch.cat(tl).contiguous() if case["tail"] else None
    if k >= 2:  # some records are shorter
        s["teacher_indices"][1::7, k - k // 2:] = -1
    if r >= 4:  # and a row has none
        s["teacher_indices"][3] = -1
    s["labels"] = torch.randint(0, v, (r,), device="cuda", generator=gen).to(torch.int32) if case["labels"] else None
    if case["labels"] and r >= 4:  # padding rows carry no label
        s["labels"][2::5] = -1
    s["grad_scale"] = 1.0 / r
    s["loss"] = torch.empty(r, **f32)
    s["stats"] = torch.empty(r, 3, **f32)
    s["grad_loss"] = None
    if op == "backward":
        s["grad_loss"] = torch.rand(r, device="cuda", generator=gen) + 0.5
        s["grad_scale"] = 1.0
        s["stats"] = _statistics(s)
    if op != "forward":
        s["grad"] = torch.empty(r, v, device="cuda", dtype=DTYPES[case["dtype"]])
    return s


def _sample_settings(kind, r, gen):
    def pick(values, dtype=torch.float32):
        at = torch.randint(0, len(values), (r,), device="cuda", generator=gen)
        return torch.tensor(values, device="cuda", dtype=dtype)[at].contiguous()

    s = dict(uniform=torch.rand(r, device="cuda", generator=gen), temperature=None, top_k=None, top_p=None, min_p=None)
    if kind == "mixed":
        s.update(temperature=pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3]), top_k=pick([0, 0, 1, 20, 50, 200], torch.int32),
                 top_p=pick([1.0, 0.9, 0.95, 0.5]), min_p=pick([0.0, 0.0, 0.05, 0.2]))
    elif kind == "nucleus":
        s.update(temperature=pick([0.8, 1.0, 1.2]), top_p=pick([0.8, 0.9, 0.95, 0.99]))
    elif kind == "topk":
        s.update(temperature=pick([0.7, 1.0]), top_k=pick([1, 5, 40, 100, 256, 1000], torch.int32))
    else:
        s.update(temperature=pick([0.9, 1.0, 1.1]))
    return s


# -- one pass -----------------------------------------------------------------

_RUNTIME = None
_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _runtime():
    """The framework's runtime on torch's current stream (1 names the legacy
    default stream, which torch calls 0)."""
    global _RUNTIME
    if _RUNTIME is None:
        import hexatrain_b200 as hx
        rt = hx.Runtime()
        if not rt.initialize(torch.cuda.current_device()):
            raise RuntimeError(rt.last_error)
        if not rt.set_stream(torch.cuda.current_stream().cuda_stream or 1):
            raise RuntimeError(rt.last_error)
        _RUNTIME = rt
    return _RUNTIME


def _p(t):
    return 0 if t is None else t.data_ptr()


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    rt = _runtime()
    x = s["logits"]
    rows, vocab = x.shape
    code, stride = _CODES[x.dtype], x.stride(0)
    op = s["op"]
    if op == "sample":
        ok = rt.sample_logits_device(code, rows, vocab, x.data_ptr(), stride, _p(s["uniform"]), _p(s["tokens"]),
                                     log_probs=_p(s["log_probs"]), temperature=_p(s["temperature"]),
                                     top_k=_p(s["top_k"]), top_p=_p(s["top_p"]), min_p=_p(s["min_p"]))
        out = dict(tokens=s["tokens"], log_probs=s["log_probs"])
    elif op == "top":
        ok = rt.top_logits_device(code, rows, vocab, x.data_ptr(), stride, s["k"], _p(s["values"]), _p(s["indices"]),
                                  lse=_p(s["lse"]), temperature=s["tau"])
        out = dict(values=s["values"], indices=s["indices"], lse=s["lse"])
    else:
        target = (code, rows, vocab, x.data_ptr(), stride, s["k"], _p(s["teacher_values"]), _p(s["teacher_indices"]),
                  _p(s["teacher_lse"]), _p(s["labels"]), s["tau"], s["kd"], s["ce"])
        if op == "forward":
            ok = rt.distill_forward_device(*target, loss=_p(s["loss"]), stats=_p(s["stats"]))
            out = dict(loss=s["loss"], stats=s["stats"])
        elif op == "backward":
            ok = rt.distill_backward_device(*target, stats=_p(s["stats"]), grad_loss=_p(s["grad_loss"]),
                                            grad_scale=s["grad_scale"], d_logits=_p(s["grad"]), grad_stride=vocab)
            out = dict(grad=s["grad"])
        else:
            ok = rt.distill_forward_backward_device(*target, grad_loss=_p(s["grad_loss"]), grad_scale=s["grad_scale"],
                                                    loss=_p(s["loss"]), d_logits=_p(s["grad"]), grad_stride=vocab)
            out = dict(loss=s["loss"], grad=s["grad"])
    if not ok:
        raise RuntimeError(rt.last_error)
    return out


def _run_plain(s):
    op = s["op"]
    if op == "sample":
        return _plain_sample(s)
    if op == "top":
        return _plain_top(s)
    if op == "forward":
        d = _plain_loss(s)
        return dict(loss=d["loss"], stats=d["stats"])
    if op == "backward":
        return dict(grad=_plain_grad(s, s["stats"]))
    d = _plain_loss(s)
    return dict(loss=d["loss"], grad=_plain_grad(s, d["stats"]))


def _plain_top(s):
    x = s["logits"].float()
    order = torch.sort(x, dim=1, descending=True, stable=True)
    z = x / s["tau"]
    m = z.amax(1, keepdim=True)
    lse = m[:, 0] + torch.exp(z - m).sum(1).log()
    k = s["k"]
    return dict(values=order.values[:, :k].contiguous(), indices=order.indices[:, :k].to(torch.int32), lse=lse)


def _teacher(s):
    """(valid, indices, log q, q, rows that have a teacher)."""
    idx, tau = s["teacher_indices"], s["tau"]
    valid = idx >= 0
    t = torch.where(valid, s["teacher_values"] / tau, float("-inf"))
    if s["teacher_lse"] is not None:
        logq = t - s["teacher_lse"][:, None]
    else:
        m = t.amax(1, keepdim=True)
        logq = t - m - torch.exp(t - m).sum(1, keepdim=True).log()
    has = valid.any(1)
    q = torch.where(valid & has[:, None], torch.exp(logq), 0.0)
    return valid, idx.clamp(min=0).long(), logq, q, has


def _in_record(valid, idx, rows, vocab):
    """Which tokens of every row the teacher's record names."""
    named = torch.zeros(rows, vocab + 1, device=idx.device, dtype=torch.bool)
    return named.scatter_(1, torch.where(valid, idx, vocab), True)[:, :vocab]


def _statistics(s):
    return _plain_loss(s)["stats"]


def _plain_loss(s):
    x, tau = s["logits"].float(), s["tau"]
    rows, vocab = x.shape
    z = x / tau
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1)
    lse_tau = m[:, 0] + total.log()
    valid, idx, logq, q, has = _teacher(s)
    logp = z.gather(1, idx) - lse_tau[:, None]
    kl = torch.where(q > 0, q * (logq - logp), 0.0).sum(1)
    ratio = torch.zeros_like(kl)
    if s["teacher_lse"] is not None:
        p_tail = e.masked_fill_(_in_record(valid, idx, rows, vocab), 0.0).sum(1) / total
        q_tail = torch.where(has & (p_tail > 0), (1.0 - q.sum(1)).clamp(min=0.0), 0.0)
        kl = kl + torch.where(q_tail > 0, q_tail * (q_tail.log() - p_tail.log()), 0.0)
        ratio = torch.where(q_tail > 0, q_tail / p_tail, 0.0)
    m1 = x.amax(1, keepdim=True)
    lse_1 = m1[:, 0] + torch.exp(x - m1).sum(1).log()
    loss = s["kd"] * tau * tau * kl
    if s["labels"] is not None:
        y = s["labels"].clamp(min=0).long()[:, None]
        loss = loss + s["ce"] * torch.where(s["labels"] >= 0, lse_1 - x.gather(1, y)[:, 0], 0.0)
    return dict(loss=loss, stats=torch.stack([lse_tau, lse_1, ratio], 1))


def _plain_grad(s, stats):
    x, tau = s["logits"].float(), s["tau"]
    rows, vocab = x.shape
    valid, idx, _, q, has = _teacher(s)
    g = torch.exp(x / tau - stats[:, 0:1])
    g *= has[:, None]
    if s["teacher_lse"] is not None:
        g *= torch.where(_in_record(valid, idx, rows, vocab), 1.0, 1.0 - stats[:, 2:3])
    g.scatter_add_(1, idx, -q)
    g *= s["kd"] * tau
    if s["labels"] is not None and s["ce"] != 0.0:
        on = (s["labels"] >= 0).float()[:, None]
        p = torch.exp(x - stats[:, 1:2]) * on
        p.scatter_add_(1, s["labels"].clamp(min=0).long()[:, None], -on)
        g += s["ce"] * p
    scale = s["grad_scale"] if s["grad_loss"] is None else s["grad_scale"] * s["grad_loss"][:, None]
    return (g * scale).to(s["logits"].dtype)


def _plain_sample(s):
    """Masses are whole numbers, floor(2^31 exp(-y)), so that their sums do not
    depend on an order; y = (max - l) / T orders the tokens, the lowest index
    first among equals.  Every filter keeps the head of that order."""
    x = s["logits"].float()
    rows, vocab = x.shape
    dev = x.device
    t = torch.ones(rows, device=dev) if s["temperature"] is None else s["temperature"]
    greedy = ~((t > 0) & torch.isfinite(t))
    m = x.amax(1, keepdim=True)
    y = (m - x) * (1.0 / torch.where(greedy, 1.0, t))[:, None]
    w = (torch.exp(-y) * 2.0 ** 31).nan_to_num_(0.0).to(torch.int64)
    order = torch.sort(y, dim=1, stable=True)
    mass = w.gather(1, order.indices).cumsum(1)
    k = torch.zeros(rows, device=dev, dtype=torch.int64) if s["top_k"] is None else s["top_k"].long()
    k = torch.where((k <= 0) | (k > vocab), vocab, k)
    k = torch.where(greedy, 1, k)
    kept = mass.gather(1, k[:, None] - 1)
    if s["top_p"] is not None:
        p = (s["top_p"].clamp(0.0, 1.0).double() * 2.0 ** 32).to(torch.int64)[:, None]
        need = torch.where(s["top_p"][:, None] < 1.0, _scaled(kept, p).clamp(min=1), kept)
        kept = mass.gather(1, torch.searchsorted(mass, need).clamp(max=vocab - 1))
    if s["min_p"] is not None:
        within = y <= -s["min_p"].log()[:, None]
        kept = torch.minimum(kept, torch.where(within, w, 0).sum(1, keepdim=True))
    u = (s["uniform"].clamp(0.0, 1.0).double() * 2.0 ** 32).to(torch.int64).clamp(max=2 ** 32 - 1)[:, None]
    at = torch.searchsorted(mass, _scaled(kept, u), right=True).clamp(max=vocab - 1)
    token = order.indices.gather(1, at)[:, 0]
    log_p = -order.values.gather(1, at)[:, 0] - (kept[:, 0].float() * 2.0 ** -31).log()
    alive = torch.isfinite(m[:, 0])
    return dict(tokens=torch.where(alive, token, -1).to(torch.int32),
                log_probs=torch.where(alive, torch.where(greedy, 0.0, log_p), float("-inf")))


def _scaled(mass, fraction):
    """floor(mass * fraction / 2^32) for masses below 2^50, in 64 bits."""
    high, low = (mass >> 25) * fraction, (mass & (2 ** 25 - 1)) * fraction
    return (high >> 7) + ((((high & 127) << 25) + low) >> 32)


# -- the definitions in 64 bits -------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    x = s["logits"].double()
    if op == "sample":
        return dict(tokens=None, log_probs=_exact_log_probs(s, x))
    if op == "top":
        return dict(values=torch.topk(x, case["k"], dim=1).values, indices=None,
                    lse=torch.logsumexp(x / case["tau"], dim=1))
    rows, vocab = x.shape
    tau = case["tau"]
    log_p = torch.log_softmax(x / tau, dim=1)
    idx = s["teacher_indices"].long()
    q_full = torch.zeros(rows, vocab, device=x.device, dtype=torch.float64)
    t = s["teacher_values"].double() / tau
    t = t.masked_fill(idx < 0, float("-inf"))
    with_teacher = (idx >= 0).any(1)
    log_z = torch.logsumexp(t, dim=1) if s["teacher_lse"] is None else s["teacher_lse"].double()
    q = torch.exp(t - log_z[:, None]).nan_to_num(0.0)
    q_full.scatter_add_(1, idx.clamp(min=0), q)
    kl = (torch.special.xlogy(q, q) - q * log_p.gather(1, idx.clamp(min=0))).sum(1)
    ratio = torch.zeros_like(kl)
    if s["teacher_lse"] is not None:
        outside = torch.ones_like(q_full)
        outside.scatter_reduce_(1, idx.clamp(min=0), (idx < 0).double(), reduce="amin")
        p_tail = (torch.exp(log_p) * outside).sum(1)
        q_tail = (1.0 - q.sum(1)).clamp(min=0.0) * with_teacher * (p_tail > 0)
        kl = kl + torch.where(q_tail > 0, q_tail * (q_tail / p_tail).log(), 0.0)
        ratio = torch.where(q_tail > 0, q_tail / p_tail, 0.0)
        if op == "backward":
            ratio = s["stats"][:, 2].double()
    hard = torch.log_softmax(x, dim=1)
    loss = case["kd"] * tau ** 2 * kl
    on = torch.zeros(rows, device=x.device, dtype=torch.float64)
    if s["labels"] is not None:
        label = s["labels"].clamp(min=0).long()[:, None]
        on = (s["labels"] >= 0).double()
        loss = loss - case["ce"] * on * hard.gather(1, label)[:, 0]
    if op == "forward":
        return dict(loss=loss, stats=torch.stack([torch.logsumexp(x / tau, 1), torch.logsumexp(x, 1), ratio], 1))
    if op == "backward":
        log_p, hard = x / tau - s["stats"][:, :1].double(), x - s["stats"][:, 1:2].double()
    g = torch.exp(log_p) * with_teacher[:, None]
    if s["teacher_lse"] is not None:
        g *= 1.0 - outside * ratio[:, None]
    g = case["kd"] * tau * (g - q_full)
    if s["labels"] is not None:
        p = torch.exp(hard).scatter_add_(1, label, torch.full_like(on, -1.0)[:, None])
        g += case["ce"] * on[:, None] * p
    if s["grad_loss"] is not None:
        g *= s["grad_loss"].double()[:, None]
    g *= s["grad_scale"]
    return dict(grad=g) if op == "backward" else dict(loss=loss, grad=g)


def _exact_log_probs(s, x):
    rows, vocab = x.shape
    ones = torch.ones(rows, device=x.device, dtype=torch.float64)
    t = ones if s["temperature"] is None else s["temperature"].double()
    greedy = ~(t > 0)
    z = (x - x.amax(1, keepdim=True)) / torch.where(greedy, 1.0, t)[:, None]
    z, _ = torch.sort(z, dim=1, descending=True)
    cum = torch.exp(z).cumsum(1)
    rank = torch.arange(vocab, device=x.device)[None, :]
    keep = torch.ones(rows, vocab, device=x.device, dtype=torch.bool)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
        keep &= rank < k
    mass = torch.where(keep, torch.exp(z), 0.0).sum(1, keepdim=True)
    head = keep.clone()
    if s["top_p"] is not None:
        head &= cum - torch.exp(z) < s["top_p"].double()[:, None] * mass
    if s["min_p"] is not None:
        head &= torch.exp(z) >= s["min_p"].double()[:, None]
    total = torch.where(head, torch.exp(z), 0.0).sum(1, keepdim=True)
    at = (cum <= s["uniform"].double()[:, None] * total).sum(1, keepdim=True).clamp(max=vocab - 1)
    log_p = torch.where(greedy, 0.0, (z.gather(1, at) - total.log())[:, 0])
    return torch.where(torch.isfinite(x.amax(1)), log_p, float("-inf"))
