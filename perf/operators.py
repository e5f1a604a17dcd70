"""Performance cases of the losses over a wide output layer: log-probabilities of labels, distillation from a teacher's
top logits, the clipped policy loss and the preference loss, each with the gradient of its logits.

A case is a dict:
  kind         "logprob" (forward), "logprob_grad" (its backward pass), "distill", "policy" or "preference" (loss and gradient)
  rows         rows of logits (tokens, samples)
  classes      classes of a row; pad: further columns of the matrix that are no classes
  dtype        f32, f16 or bf16: type of the logits and of their gradient
  temperature  the logits are divided by it
  entropy      logprob: the rows' entropies too; policy: coefficient of the entropy bonus
  k, tail      distill: entries of the teacher's list, and whether its mass outside the list is matched as one more class
  kl           policy: coefficient of the term that keeps the policy near a reference
  pairs, loss, average   preference: pairs of sequences; sigmoid, hinge or squared; sums or means over a sequence
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_CLIP = (0.2, 0.28)        # below and above 1
_BETA, _SMOOTH, _MARGIN = 0.1, 0.1, 0.25
_SCALE = 32.0              # loss scale of 16-bit gradients
_LEAST_TAIL = 1e-6         # a teacher's mass outside its list that counts


def _case(kind, rows, classes, dtype, pad=0, temperature=1.0, entropy=0.0, k=0, tail=False, kl=0.0, pairs=0, loss="", average=False, **name):
    return dict(name, kind=kind, rows=rows, classes=classes, pad=pad, dtype=dtype, temperature=temperature, entropy=entropy, k=k,
                tail=tail, kl=kl, pairs=pairs, loss=loss, average=average)


def listed():
    return [
        # an agent with ten actions records its log-probabilities for a minibatch: launch and latency
        _case("logprob", 64, 10, "f32", entropy=1.0, name="logprob_f32_64x10"),
        # old and reference log-probabilities of a batch of tokens over a large vocabulary: one read of a gigabyte
        _case("logprob", 4096, 131072, "bf16", name="logprob_bf16_4096x131072"),
        # gradient of a loss that the user wrote on the log-probabilities, vocabulary padded to whole tiles
        _case("logprob_grad", 2048, 32003, "f16", pad=61, temperature=0.7, name="logprob_grad_f16_2048x32003"),
        # image classifier that learns from a larger one's sixteen likeliest classes at a high temperature
        _case("distill", 512, 1000, "f16", temperature=4.0, k=16, name="distill_f16_512x1000"),
        # language model that learns from stored top logits with their tail: the largest pass
        _case("distill", 4096, 131072, "bf16", k=64, tail=True, name="distill_bf16_4096x131072"),
        # f32 training with a class count that fits no vector
        _case("distill", 777, 10007, "f32", temperature=2.0, k=20, tail=True, name="distill_f32_777x10007"),
        # one update of a small agent
        _case("policy", 64, 10, "f32", entropy=0.01, name="policy_f32_64x10"),
        # one update of a language model's policy with a reference term and an entropy bonus
        _case("policy", 8192, 32768, "bf16", entropy=0.005, kl=0.04, name="policy_bf16_8192x32768"),
        # odd action count, sampled at a low temperature
        _case("policy", 1001, 777, "f16", temperature=0.8, kl=0.1, name="policy_f16_1001x777"),
        # a few short answers
        _case("preference", 60, 1000, "f16", pairs=4, loss="sigmoid", name="preference_f16_4_pairs_1000"),
        # a batch of pairs of answers of a few hundred tokens each
        _case("preference", 8192, 32768, "bf16", pairs=8, loss="sigmoid", name="preference_bf16_8_pairs_32768"),
        # means over long sequences, squared loss, f32, odd class count
        _case("preference", 1500, 50021, "f32", pairs=3, loss="squared", average=True, name="preference_f32_3_pairs_50021"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(work(c)["bytes"] for c in listed())
    while True:
        kind = rng.choice(["logprob", "logprob_grad", "distill", "distill", "policy", "policy", "preference", "preference"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        rows, classes = _log(rng, 1, 16384), _log(rng, 2, 200000)
        if rng.random() < 0.4:
            classes = max(2, classes - classes % 8)
        pad = rng.choice([0, 0, 0, -classes % 64])
        c = _case(kind, rows, classes, dtype, pad, rng.choice([1.0, 1.0, 0.7, 1.3, 2.0]))
        if kind == "logprob":
            c["entropy"] = rng.choice([0.0, 1.0])
        elif kind == "logprob_grad":
            c["entropy"] = rng.choice([0.0, 0.02])
        elif kind == "distill":
            c.update(k=min(classes - 1, _log(rng, 1, 256)), tail=rng.random() < 0.5)
        elif kind == "policy":
            c.update(kl=rng.choice([0.0, 0.05]), entropy=rng.choice([0.0, 0.01]))
        else:
            c.update(pairs=_log(rng, 1, 64), loss=rng.choice(["sigmoid", "sigmoid", "hinge", "squared"]), average=rng.random() < 0.3)
        if work(c)["bytes"] <= most and rows * classes >= 64:
            return c


def work(case):
    """Each logit read once, each gradient written once, the rows' vectors and the teacher's lists once."""
    rows, one = case["rows"], _BYTES[case["dtype"]]
    read = rows * case["classes"] * one + 4 * rows
    written = 0 if case["kind"] == "logprob" else rows * (case["classes"] + case["pad"]) * one
    per_row = {"logprob": 8, "logprob_grad": 8, "distill": 8 * case["k"] + 12, "policy": 28, "preference": 4}[case["kind"]]
    return {"bytes": read + written + rows * per_row + 40 * case["pairs"], "flops": rows * case["classes"] * (4 if case["kind"] == "logprob" else 8)}


def _chunks(rows, classes, most=1 << 25):
    step = max(1, most // classes)
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def _label_logprob(x, labels, classes, t):
    """Log-probabilities of the labels in 64 bits, for the inputs that a program has stored from earlier passes."""
    got = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    for a, b in _chunks(x.shape[0], classes):
        z = x[a:b, :classes].double() / t
        got[a:b] = z.gather(1, labels[a:b, None].long().clamp(min=0))[:, 0] - torch.logsumexp(z, 1)
    return torch.where(labels >= 0, got, 0.0)


def _inputs(case, seed):
    dev, rows, c, t = torch.device("cuda", 0), case["rows"], case["classes"], case["temperature"]
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    rand = lambda *s: torch.rand(s, generator=gen, device=dev)  # noqa: E731
    x = torch.empty(rows, c + case["pad"], dtype=_DTYPE[case["dtype"]], device=dev)
    for a, b in _chunks(rows, c + case["pad"], 1 << 27):
        x[a:b] = randn(b - a, c + case["pad"]).mul_(2.0)
    x[:, c:] = 100.0                                        # no classes: larger than any of them
    # labels that the model likes more or less: a few of them nearly certain
    labels = torch.randint(0, c, (rows,), generator=gen, device=dev)
    at = torch.arange(rows, device=dev)
    x[at, labels] = (x[at, labels].float() + 2.0 + 12.0 * rand(rows)).to(x.dtype)
    labels = labels.int()
    s = {"x": x, "labels": labels, "case": case}
    kind = case["kind"]
    if kind in ("logprob", "logprob_grad"):
        labels[rand(rows) < 0.05] = -1                      # positions without a label
        if kind == "logprob_grad":
            s["d_logp"], s["d_entropy"] = randn(rows), case["entropy"] * randn(rows) if case["entropy"] else None
    elif kind == "distill":
        k = case["k"]
        lo = torch.arange(k, device=dev) * c // k
        hi = torch.arange(1, k + 1, device=dev) * c // k
        idx = lo + (rand(rows, k) * (hi - lo)).long().minimum(hi - lo - 1)
        idx = idx.gather(1, rand(rows, k).argsort(1))
        values = (randn(rows, k) * 2.0 + 8.0).sort(1, descending=True).values
        x.scatter_(1, idx, (values + randn(rows, k)).to(x.dtype))
        idx[(rand(rows) < 0.1)[:, None] & (torch.arange(k, device=dev) >= max(1, k // 2))] = -1   # some lists are shorter
        kept = torch.where(idx >= 0, values.double() / t, -math.inf)
        s["indices"], s["values"] = idx.int(), values
        s["lse"] = (torch.logsumexp(kept, 1) - torch.log1p(-(0.01 + 0.3 * rand(rows).double()))).float() if case["tail"] else None
        s["weights"] = torch.where(rand(rows) < 0.05, 0.0, 0.5 + rand(rows))
    elif kind == "policy":
        logp = _label_logprob(x, labels, c, t)
        step = 0.25 * randn(rows).double()
        near = ((step.exp() - 1.0 + _CLIP[0]).abs() < 0.01) | ((step.exp() - 1.0 - _CLIP[1]).abs() < 0.01)
        s["old"] = (logp - torch.where(near, 0.0, step)).float()   # the policy has moved since: ratios around 1, some clipped
        s["ref"] = (logp + 0.3 * randn(rows)).float() if case["kl"] else None
        s["advantages"], s["weights"] = randn(rows), torch.where(rand(rows) < 0.05, 0.0, 0.5 + rand(rows))
    else:
        p, used = case["pairs"], rows - rows // 32          # a few rows behind the last sequence
        cuts = torch.randint(0, used + 1, (2 * p - 1,), generator=gen, device=dev).sort().values
        off = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), cuts, torch.full((1,), used, dtype=torch.long, device=dev)])
        seq = torch.bucketize(at, off[1:], right=True)
        start, length = torch.cat([off, off[-1:]])[seq], torch.cat([off[1:] - off[:-1], off.new_ones(1)])[seq]
        labels[(at - start) * 4 < length] = -1              # the first quarter is the prompt
        sums, _ = _sequences(_label_logprob(x, labels, c, t), labels, off, case["average"])
        ref = sums + (3.0 if not case["average"] else 0.5) * randn(2 * p)
        if case["loss"] == "hinge":                         # not next to the corner
            m = _BETA * ((sums[0::2] - ref[0::2]) - (sums[1::2] - ref[1::2])) - _MARGIN
            ref[0::2] += torch.where((m - 1.0).abs() < 0.02, 0.6 / _BETA, 0.0)
        s["offsets"], s["ref"] = off.int(), ref.float()
        s["weights"] = 0.5 + rand(p)
    return s


def prepare(case, seed):
    return _inputs(case, seed)


def _sequences(row, labels, off, average):
    """Sums or means of `row` over the labelled rows of each sequence, and how many those are, in 64 bits."""
    total = torch.cat([row.new_zeros(1), row.double().cumsum(0)])
    count = torch.cat([off.new_zeros(1), (labels >= 0).long().cumsum(0)])
    off = off.long()
    n = (count[off[1:]] - count[off[:-1]]).double()
    sums = total[off[1:]] - total[off[:-1]]
    return (sums / n.clamp(min=1.0) if average else sums), n


def _rows(s):
    """t = (x - max) / temperature, e = exp(t) and their sum over the classes, in 32 bits."""
    case = s["case"]
    t = s["x"][:, :case["classes"]].float()
    t = (t - t.amax(1, keepdim=True)) / case["temperature"]
    e = t.exp()
    return t, e, e.sum(1, keepdim=True)


def _out(s, g):
    """The gradient in the logits' type, zero in the columns that are no classes."""
    x = s["x"]
    if s["case"]["pad"] == 0:
        return g.to(x.dtype)
    out = torch.zeros_like(x)
    out[:, :g.shape[1]] = g
    return out


def _plain_logprob(s):
    case, labels = s["case"], s["labels"]
    live = labels >= 0
    t, e, z = _rows(s)
    logp = t.gather(1, labels.long().clamp(min=0)[:, None])[:, 0].double() - z[:, 0].double().log()
    logp = torch.where(live, logp, 0.0).float()
    if not case["entropy"]:
        return [logp]
    h = z[:, 0].log() - (e * t).sum(1) / z[:, 0]
    return [logp, torch.where(live, h, 0.0)]


def _plain_logprob_grad(s):
    case, labels = s["case"], s["labels"]
    t, e, z = _rows(s)
    p = e / z
    g = torch.where(labels >= 0, s["d_logp"], 0.0)[:, None]
    d = -g * p
    if s["d_entropy"] is not None:
        logp = t - z.log()
        h = -(p * logp).sum(1, keepdim=True)
        d -= torch.where(labels >= 0, s["d_entropy"], 0.0)[:, None] * p * (logp + h)
    d.scatter_add_(1, labels.long().clamp(min=0)[:, None], g)
    return [_out(s, d * (_SCALE / case["temperature"]))]


def _plain_distill(s):
    case, c, tau = s["case"], s["case"]["classes"], s["case"]["temperature"]
    t, e, z = _rows(s)
    none = torch.zeros_like(z)                              # one more column, which unused entries of the list point at
    t, e = torch.cat([t, none], 1), torch.cat([e, none], 1)
    valid = s["indices"] >= 0
    at = torch.where(valid, s["indices"].long(), c)
    logp = t.gather(1, at).double() - z.double().log()
    if case["tail"]:
        q = torch.where(valid, (s["values"].double() / tau - s["lse"].double()[:, None]).exp(), 0.0)
    else:
        v = torch.where(valid, s["values"].double() / tau, -math.inf)
        q = (v - v.amax(1, keepdim=True)).exp()
        q = q / q.sum(1, keepdim=True)
    each = torch.where(q > 0, q * (torch.where(q > 0, q, 1.0).log() - logp), 0.0).sum(1)
    d = e / z
    if case["tail"]:
        rest = 1.0 - q.sum(1)
        rest = torch.where(rest > _LEAST_TAIL, rest, 0.0)
        outside = e.scatter(1, at, 0.0).sum(1).double() / z[:, 0]
        each += torch.where(rest > 0, rest * (torch.where(rest > 0, rest, 1.0) / outside).log(), 0.0)
        listed_p = d.gather(1, at)
        d = (d * (1.0 - rest / outside).float()[:, None]).scatter_(1, at, listed_p)
    d.scatter_add_(1, at, -q.float())
    w = s["weights"]
    return [(w.double() * tau * tau * each).float(), _out(s, d[:, :c] * (w * (tau * _SCALE))[:, None])]


def _plain_policy(s):
    case, labels, w = s["case"], s["labels"].long()[:, None], s["weights"].double()
    t, e, z = _rows(s)
    log_z = z.double().log()
    logp = t.gather(1, labels).double() - log_z
    ratio = (logp[:, 0] - s["old"].double()).exp()
    a = s["advantages"].double()
    loss = -torch.minimum(ratio * a, ratio.clamp(1.0 - _CLIP[0], 1.0 + _CLIP[1]) * a)
    clipped = ((a > 0) & (ratio > 1.0 + _CLIP[1])) | ((a < 0) & (ratio < 1.0 - _CLIP[0]))
    g = torch.where(clipped, 0.0, -a * ratio)
    kl = torch.zeros_like(ratio)
    if case["kl"]:
        d = s["ref"].double() - logp[:, 0]
        kl = d.exp() - d - 1.0
        loss += case["kl"] * kl
        g += case["kl"] * (1.0 - d.exp())
    p = e / z
    entropy = (log_z - (e * t).sum(1, keepdim=True) / z)[:, 0]
    d = -p * (g * w)[:, None].float()
    if case["entropy"]:
        loss -= case["entropy"] * entropy
        d += (w * case["entropy"])[:, None].float() * p * (t - log_z.float() + entropy[:, None].float())
    d.scatter_add_(1, labels, (g * w)[:, None].float())
    live = w > 0
    return [torch.where(live, v, 0.0).float() for v in (w * loss, logp[:, 0], kl, entropy)] + [_out(s, d * (_SCALE / case["temperature"]))]


def _plain_preference(s):
    case, labels, off, w = s["case"], s["labels"], s["offsets"], s["weights"].double()
    t, e, z = _rows(s)
    inside = (labels >= 0) & (torch.arange(labels.shape[0], device=labels.device) < off[-1]) & (torch.arange(labels.shape[0], device=labels.device) >= off[0])
    logp = t.gather(1, labels.long().clamp(min=0)[:, None])[:, 0].double() - z[:, 0].double().log()
    logp = torch.where(inside, logp, 0.0)
    sums, n = _sequences(logp, labels, off, case["average"])
    h = sums - s["ref"].double()
    h = h[0::2] - h[1::2]
    m = _BETA * h - _MARGIN
    if case["loss"] == "sigmoid":
        up, down = torch.log1p((-m.abs()).exp()) + (-m).clamp(min=0.0), torch.log1p((-m.abs()).exp()) + m.clamp(min=0.0)
        loss = (1.0 - _SMOOTH) * up + _SMOOTH * down
        dm = _SMOOTH - 1.0 / (1.0 + m.exp())
    elif case["loss"] == "hinge":
        loss, dm = (1.0 - m).clamp(min=0.0), torch.where(m < 1.0, -1.0, 0.0).double()
    else:
        loss, dm = (m - 0.5).square(), 2.0 * (m - 0.5)
    g = torch.stack([w * dm * _BETA, -w * dm * _BETA], 1).reshape(-1)
    if case["average"]:
        g = g / n.clamp(min=1.0)
    seq = torch.bucketize(torch.arange(labels.shape[0], device=labels.device), off[1:].long(), right=True)
    g = torch.where(inside, torch.cat([g, g.new_zeros(1)])[seq], 0.0).float()[:, None]
    d = (e / z) * -g
    d.scatter_add_(1, labels.long().clamp(min=0)[:, None], g)
    return [(w * loss).float(), m.float(), sums.float(), logp.float(), _out(s, d * (_SCALE / case["temperature"]))]


_PLAIN = {"logprob": _plain_logprob, "logprob_grad": _plain_logprob_grad, "distill": _plain_distill, "policy": _plain_policy,
          "preference": _plain_preference}
_context = []


def _own(s):
    import soklyn_b200 as sk
    from soklyn_b200 import losses
    if not _context:
        _context.append(sk.GpuContext(16, 0))
    ctx, case = _context[0], s["case"]
    precision = {"f32": sk.Precision.FP32, "f16": sk.Precision.FP16, "bf16": sk.Precision.BF16}[case["dtype"]]
    logits, tau = sk.Tensor(s["x"], precision, take_id=False), case["temperature"]
    kind, c = case["kind"], case["classes"]
    if kind == "logprob":
        got = losses.label_logprob(ctx, logits, s["labels"], temperature=tau, classes=c, entropy=case["entropy"] > 0)
        return [got.logp, got.entropy] if case["entropy"] else [got.logp]
    if kind == "logprob_grad":
        return [losses.label_logprob_backward(ctx, logits, s["labels"], s["d_logp"], s["d_entropy"], temperature=tau, classes=c, grad_scale=_SCALE).data]
    if kind == "distill":
        got = losses.distill_loss(ctx, logits, s["indices"], s["values"], losses.DistillLossConfig(temperature=tau), teacher_lse=s["lse"],
                                  weights=s["weights"], classes=c, grad_scale=_SCALE)
        return [got.loss, got.d_logits.data]
    if kind == "policy":
        config = losses.PolicyLossConfig(clip_low=_CLIP[0], clip_high=_CLIP[1], kl_coeff=case["kl"], entropy_coeff=case["entropy"], temperature=tau)
        got = losses.policy_loss(ctx, logits, s["labels"], s["old"], s["advantages"], config, logp_ref=s["ref"], weights=s["weights"],
                                 classes=c, grad_scale=_SCALE)
        return [got.loss, got.logp, got.kl, got.entropy, got.d_logits.data]
    form = {"sigmoid": losses.PreferenceForm.Sigmoid, "hinge": losses.PreferenceForm.Hinge, "squared": losses.PreferenceForm.Squared}[case["loss"]]
    config = losses.PreferenceLossConfig(form=form, beta=_BETA, label_smoothing=_SMOOTH if case["loss"] == "sigmoid" else 0.0,
                                         target_margin=_MARGIN, average=case["average"], temperature=tau)
    got = losses.preference_loss(ctx, logits, s["labels"], s["offsets"], config, logp_ref=s["ref"], weights=s["weights"], classes=c, grad_scale=_SCALE)
    return [got.loss, got.margin, got.logp, got.row_logp, got.d_logits.data]


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


def exact(case, seed):
    """The definitions in 64 bits, their gradients by differentiation."""
    s = _inputs(case, seed)
    x, labels, c, tau, dev = s["x"], s["labels"].long(), case["classes"], case["temperature"], s["x"].device
    rows, kind = case["rows"], case["kind"]

    def piece(a, b):
        """Differentiable logits of rows a to b and their log-probabilities over the classes."""
        leaf = x[a:b].double().requires_grad_(kind != "logprob")
        return leaf, torch.log_softmax(leaf[:, :c] / tau, 1)

    def picked(lp, a, b):
        got = lp.gather(1, labels[a:b].clamp(min=0)[:, None])[:, 0]
        return torch.where(labels[a:b] >= 0, got, 0.0)

    def slope(total, leaf):
        return torch.autograd.grad(total * _SCALE, leaf)[0]

    parts = _chunks(rows, c, 1 << 26)
    grad = None if kind == "logprob" else torch.empty(x.shape, dtype=torch.float64, device=dev)
    if kind in ("logprob", "logprob_grad"):
        logp, ent = torch.zeros(rows, dtype=torch.float64, device=dev), torch.zeros(rows, dtype=torch.float64, device=dev)
        for a, b in parts:
            leaf, lp = piece(a, b)
            one, h = picked(lp, a, b), torch.where(labels[a:b] >= 0, -(lp.exp() * lp).sum(1), 0.0)
            if grad is not None:
                total = (one * s["d_logp"][a:b].double()).sum()
                if s["d_entropy"] is not None:
                    total = total + (h * s["d_entropy"][a:b].double()).sum()
                grad[a:b] = slope(total, leaf)
            else:
                logp[a:b], ent[a:b] = one, h
        return [grad] if grad is not None else [logp, ent] if case["entropy"] else [logp]
    if kind == "distill":
        loss = torch.zeros(rows, dtype=torch.float64, device=dev)
        for a, b in parts:
            leaf, lp = piece(a, b)
            idx, v = s["indices"][a:b].long(), s["values"][a:b].double() / tau
            v = torch.where(idx >= 0, v, -math.inf)
            logq = v - s["lse"][a:b].double()[:, None] if case["tail"] else torch.log_softmax(v, 1)
            q = logq.exp()
            each = torch.xlogy(q, q).sum(1) - (q * lp.gather(1, idx.clamp(min=0))).sum(1)
            if case["tail"]:
                r = 1.0 - q.sum(1)
                r = torch.where(r > _LEAST_TAIL, r, 0.0)
                out = torch.ones(b - a, c + 1, dtype=torch.bool, device=dev).scatter_(1, torch.where(idx >= 0, idx, c), False)[:, :c]
                outside = torch.logsumexp(torch.where(out, lp, -math.inf), 1)
                each = each + torch.xlogy(r, r) - torch.where(r > 0, r * outside, 0.0)
            each = each * (tau * tau) * s["weights"][a:b].double()
            grad[a:b] = slope(each.sum(), leaf)
            loss[a:b] = each.detach()
        return [loss, grad]
    if kind == "policy":
        got = torch.zeros(4, rows, dtype=torch.float64, device=dev)
        for a, b in parts:
            leaf, lp = piece(a, b)
            one, h, w, adv = picked(lp, a, b), -(lp.exp() * lp).sum(1), s["weights"][a:b].double(), s["advantages"][a:b].double()
            ratio = torch.exp(one - s["old"][a:b].double())
            kl = torch.zeros_like(one)
            if case["kl"]:
                d = s["ref"][a:b].double() - one
                kl = torch.expm1(d) - d
            each = w * (torch.maximum(-ratio * adv, -ratio.clamp(1.0 - _CLIP[0], 1.0 + _CLIP[1]) * adv) + case["kl"] * kl - case["entropy"] * h)
            grad[a:b] = slope(each.sum(), leaf)
            got[:, a:b] = torch.stack([each, one, kl, h]).detach() * (w > 0)
        return [*got, grad]
    # preference: the rows' log-probabilities, then the losses as a function of them, then both through the chain rule
    off = [int(v) for v in s["offsets"]]
    one = torch.zeros(rows, dtype=torch.float64, device=dev)
    for a, b in parts:
        with torch.no_grad():
            one[a:b] = picked(piece(a, b)[1], a, b)
    one[off[-1]:] = 0.0
    one.requires_grad_(True)
    sums = []
    for a, b in zip(off[:-1], off[1:]):
        n = int((labels[a:b] >= 0).sum())
        sums.append(one[a:b].sum() / (max(1, n) if case["average"] else 1))
    sums = torch.stack(sums)
    h = sums - s["ref"].double()
    m = _BETA * (h[0::2] - h[1::2]) - _MARGIN
    if case["loss"] == "sigmoid":
        each = -(1.0 - _SMOOTH) * torch.nn.functional.logsigmoid(m) - _SMOOTH * torch.nn.functional.logsigmoid(-m)
    else:
        each = torch.relu(1.0 - m) if case["loss"] == "hinge" else (m - 0.5) ** 2
    each = each * s["weights"].double()
    pull = torch.autograd.grad(each.sum(), one)[0]
    pull[off[-1]:] = 0.0
    for a, b in parts:
        leaf, lp = piece(a, b)
        grad[a:b] = slope((picked(lp, a, b) * pull[a:b]).sum(), leaf)
    return [each.detach(), m.detach(), sums.detach(), one.detach(), grad]
