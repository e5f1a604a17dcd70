"""Losses over rows of logits (soklyn_b200/losses.py) against their formulas in 64 bits, at the sizes, alignments and
masks where they can go wrong.

Tolerances. A result of T is rounded by at most eps(T) / 2 of its value. Below that stands the f32 arithmetic: an exponential
ex2.approx(t) is off by 2^-22 and by the rounding of its argument, 2^-23 |t| in f32 and, with one product instead of
two, 2^-22 |t| for 16-bit gradients; sums of n terms are added in chains of at most n / 256 + 40, 2^-24 each.
"""
import math

import numpy as np
import pytest
import torch

import soklyn_b200 as sk
from soklyn_b200 import log, losses

pytestmark = pytest.mark.gpu

DT = {"f32": (torch.float32, sk.Precision.FP32), "f16": (torch.float16, sk.Precision.FP16), "bf16": (torch.bfloat16, sk.Precision.BF16)}
INF = math.inf
LOG2E = 1.4426950408889634
# classes: one, fewer than a unit, around warps, blocks and units, odd, wide
SIZES = [(3, 1), (5, 2), (4, 7), (64, 10), (9, 33), (3, 255), (2, 256), (7, 1000), (5, 1023), (3, 1025), (3, 4099), (2, 10007), (2, 32768), (1, 50021), (2, 131072), (1, 250001), (1, 950001)]


def _rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _logits(rows, classes, pad, kind, offset=0, seed=0, scale=3.0):
    """Tensor [rows x (classes + pad)] whose first element lies `offset` elements behind a 256-byte boundary; NaN in the padding."""
    dt, prec = DT[kind]
    g = _rng(seed * 1000003 + rows * 1009 + classes)
    flat = torch.full((rows * (classes + pad) + offset,), math.nan, dtype=dt, device="cuda")
    x = flat[offset:].view(rows, classes + pad)
    x[:, :classes] = (torch.randn(rows, classes, generator=g, device="cuda") * scale).to(dt)
    return sk.Tensor(x, prec, take_id=False), g


class Ref:
    """Statistics of rows in 64 bits. A row without a class above -inf is dead."""

    def __init__(self, x, classes, tau):
        self.tau, self.kind = tau, x.dtype
        z = x[:, :classes].double() / tau
        self.dead = (z == -INF).all(1)
        z = torch.where(self.dead[:, None], 0.0, z)
        z = z - z.amax(1, keepdim=True)        # first: beside 3e38 a logarithm of ten would be lost
        self.lse = torch.logsumexp(z, 1)
        self.lp = z - self.lse[:, None]
        self.p = self.lp.exp()
        self.plogp = torch.where(self.p > 0, self.p * self.lp.clamp(min=-1e5), 0.0)
        self.h = -self.plogp.sum(1)
        t2 = ((z - z.amax(1, keepdim=True)) * LOG2E).clamp(min=-200.0).abs()
        mean_t = (self.p * t2).sum(1, keepdim=True)
        chain = (classes / 256 + 40) * 2.0 ** -24
        self.sum_rel = (2.0 ** -22 + 2.0 ** -23 * mean_t + chain)[:, 0]                       # of s, so absolute of log s
        self.rel = self.sum_rel[:, None] + 2.0 ** -21 + 2.0 ** -22 * t2                        # of a term of the gradient
        self.h_tol = 4.0 * self.sum_rel * (1.0 + mean_t[:, 0]) + 2.0 ** -23 * self.h.abs()

    def pick(self, labels):
        return self.lp.gather(1, labels.long().clamp(min=0)[:, None])[:, 0]


def _close(got, want, tol, what):
    got = got.double()
    bad = ~((got - want).abs() <= tol) & ~(got.isnan() & want.isnan()) & ~(got == want)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; at {i} got {float(got[i])!r}, want {float(want[i])!r}, "
                             f"tolerance {float(torch.as_tensor(tol).expand_as(want)[i]):.3g}")


def _gradient(d, want, base, ref, classes, extra=0.0):
    """`base`: the sum of the magnitudes of the terms of each element, before they cancel."""
    x = d.data
    assert (x[:, classes:] == 0).all(), "columns that are no classes"
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[x.dtype]
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + ref.rel * base + tiny + extra
    _close(x[:, :classes], want, tol, "gradient")


def _label_rows(rows, classes, g):
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda").int()
    if rows > 2:
        labels[1] = -1
    return labels


# ---- log-probabilities ------------------------------------------------------------------------------------

def check_logprob(ctx, x, labels, classes, tau=1.0, with_entropy=True):
    got = losses.label_logprob(ctx, x, labels, temperature=tau, classes=classes, entropy=with_entropy)
    ctx.synchronize()
    r = Ref(x.data, classes, tau)
    live = (labels >= 0) & ~r.dead
    want = torch.where(live, r.pick(labels), 0.0)
    _close(got.logp, want, r.sum_rel + 2.0 ** -24 * want.abs().nan_to_num(posinf=0.0), "logp")
    if with_entropy:
        _close(got.entropy, torch.where(live, r.h, 0.0), r.h_tol, "entropy")
    else:
        assert got.entropy is None


def check_logprob_backward(ctx, x, labels, classes, g, tau=1.0, scale=1.0, with_entropy=True, out=None):
    d_logp = torch.randn(labels.shape[0], generator=g, device="cuda")
    d_ent = torch.randn(labels.shape[0], generator=g, device="cuda") if with_entropy else None
    r = Ref(x.data, classes, tau)
    d = losses.label_logprob_backward(ctx, x, labels, d_logp, d_ent, temperature=tau, classes=classes, grad_scale=scale, out=out)
    ctx.synchronize()
    live = ((labels >= 0) & ~r.dead)[:, None]
    k = scale / tau
    a = d_logp.double()[:, None]
    hit = torch.zeros_like(r.p).scatter_(1, labels.long().clamp(min=0)[:, None], 1.0)
    want = k * a * (hit - r.p)
    base = k * a.abs() * (hit + r.p)
    if with_entropy:
        b = d_ent.double()[:, None]
        want -= k * b * (r.plogp + r.p * r.h[:, None])
        base += k * b.abs() * (r.plogp.abs() + r.p * r.h[:, None] + r.p) * 2.0
    _gradient(d, torch.where(live, want, 0.0), torch.where(live, base, 0.0), r, classes)
    return d


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("rows,classes", SIZES)
def test_logprob_and_its_backward(gpu_ctx, rows, classes, kind):
    for pad, offset, tau in ((0, 0, 1.0), (5, 3, 0.7), (-classes % 64, 1, 2.5)):
        x, g = _logits(rows, classes, pad, kind, offset)
        labels = _label_rows(rows, classes, g)
        check_logprob(gpu_ctx, x, labels, classes, tau, with_entropy=offset != 1)
        check_logprob_backward(gpu_ctx, x, labels, classes, g, tau, 32.0, with_entropy=offset != 1)


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes", [10, 1000, 1027, 40009])
def test_masked_classes_and_odd_values(gpu_ctx, classes, kind):
    """-inf, the type's lowest and largest values, rows of nothing else, NaN and +inf: each row for itself."""
    x, g = _logits(9, classes, 3, kind, 1)
    v, low = x.data, torch.finfo(x.data.dtype).min
    labels = torch.randint(0, classes, (9,), generator=g, device="cuda").int()
    v[0, :classes:2] = -INF
    v[0, labels[0].long()] = 1.0
    v[1, :classes] = -INF                      # no class left
    v[2, :classes] = low                       # every class masked with the lowest value: equal shares
    v[3, :classes // 2] = low
    labels[3] = classes - 1
    v[4, :classes] = -INF                      # one class left
    v[4, labels[4].long()] = low
    v[5, labels[5].long()] = -INF              # the label itself masked
    v[6, :classes] = -1000.0                   # far below zero
    check_logprob(gpu_ctx, x, labels, classes)
    check_logprob_backward(gpu_ctx, x, labels, classes, g)
    v[7, classes // 3] = math.nan
    v[8, classes // 2] = INF
    labels[0] = -1
    v[0, :classes] = math.nan                  # does not count, whatever it holds
    d = losses.label_logprob_backward(gpu_ctx, x, labels, torch.ones(9, device="cuda"), classes=classes).data
    got = losses.label_logprob(gpu_ctx, x, labels, classes=classes, entropy=True)
    assert d[7:, :classes].isnan().all() and got.logp[7:].isnan().all() and got.entropy[7:].isnan().all()
    assert (d[:2] == 0).all() and (got.logp[:2] == 0).all() and (got.entropy[:2] == 0).all() and not d[:7].isnan().any()
    assert float(got.logp[5]) == -INF and float(got.logp[4]) == 0.0
    assert abs(float(got.logp[2]) + math.log(classes)) < 1e-5


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes", [9, 1000, 3001, 33003])
def test_gradient_over_the_logits_and_at_other_alignments(gpu_ctx, classes, kind):
    dt, prec = DT[kind]
    x, g = _logits(4, classes, 1, kind)
    labels = _label_rows(4, classes, g)
    want = check_logprob_backward(gpu_ctx, x, labels, classes, _rng(5)).data.clone()
    flat = torch.full((4 * (classes + 1) + 8,), 7.0, dtype=dt, device="cuda")
    for offset in (1, 3, 8):                   # other offsets within 16 bytes than the logits'; nothing else is written
        flat.fill_(7.0)
        out = sk.Tensor(flat[offset:offset + 4 * (classes + 1)].view(4, classes + 1), prec, take_id=False)
        assert check_logprob_backward(gpu_ctx, x, labels, classes, _rng(5), out=out) is out
        assert torch.equal(out.data, want) and (flat[:offset] == 7.0).all() and (flat[offset + out.len():] == 7.0).all()
    check = sk.Tensor(x.data.clone(), prec, take_id=False)
    d_logp = torch.randn(4, generator=_rng(5), device="cuda")
    d_ent = torch.randn(4, generator=(r := _rng(5)), device="cuda")
    d_ent = torch.randn(4, generator=r, device="cuda")
    losses.label_logprob_backward(gpu_ctx, check, labels, d_logp, d_ent, classes=classes, out=check)
    assert torch.equal(check.data, want)


def test_labels_out_of_range_are_reported_and_do_not_count(gpu_ctx):
    x, g = _logits(4, 50, 14, "f16")
    labels = torch.tensor([3, 50, 63, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    d = losses.label_logprob_backward(gpu_ctx, x, labels, torch.ones(4, device="cuda"), classes=50)
    with pytest.raises(log.IndexOutOfRange, match="a label"):
        gpu_ctx.synchronize()
    assert (d.data[1:] == 0).all() and (d.data[0, :50] != 0).any()
    gpu_ctx.synchronize()                      # reported once


# ---- distillation ----------------------------------------------------------------------------------------------

def distill_reference(x, classes, tau, idx, values, lse, weights, scale):
    """loss, gradient and their tolerances."""
    r = Ref(x, classes, tau)
    rows, k = idx.shape
    valid = (idx >= 0) & (idx < classes)
    at = torch.where(valid, idx.long(), classes)
    v = torch.where(valid, values.double() / tau, -INF)
    if lse is None:
        empty = (v == -INF).all(1)
        logq = torch.where(empty[:, None], -INF, v - torch.logsumexp(torch.where(empty[:, None], 0.0, v), 1)[:, None])
    else:
        empty = torch.zeros(rows, dtype=torch.bool, device=x.device)
        logq = v - lse.double()[:, None]
    q = logq.exp()
    w = torch.ones(rows, dtype=torch.float64, device=x.device) if weights is None else weights.double()
    lp = torch.cat([r.lp, torch.zeros(rows, 1, device=x.device, dtype=torch.float64)], 1)
    lpk = lp.gather(1, at)
    rest = (1.0 - q.sum(1)) if lse is not None else torch.zeros(rows, dtype=torch.float64, device=x.device)
    rest = torch.where(rest > 1e-6, rest, 0.0)
    inside = torch.zeros(rows, classes + 1, dtype=torch.bool, device=x.device).scatter_(1, at, True)[:, :classes]
    out_p = torch.where(inside, 0.0, r.p)
    s_out = out_p.sum(1)
    log_out = torch.logsumexp(torch.where(inside, -INF, r.lp), 1)
    each = torch.where(q > 0, q * (logq - lpk), 0.0).sum(1) + torch.where(rest > 0, rest * (rest.clamp(min=1e-300).log() - log_out), 0.0)
    total = (q.sum(1) + rest)[:, None] if lse is not None else 1.0
    share = torch.where(s_out > 0, rest / s_out.clamp(min=1e-300), 0.0)[:, None]
    target = torch.zeros(rows, classes + 1, dtype=torch.float64, device=x.device).scatter_add_(1, at, q)[:, :classes]
    f = (w * tau * scale)[:, None]
    want = f * (total * r.p - share * out_p - target)
    base = f.abs() * (total * r.p + share * out_p + target * 4.0)
    live = ((w != 0) & ~empty & ~r.dead)
    q_rel = 2.0 ** -22 * (1.0 + torch.where(q > 0, (v - v.amax(1, keepdim=True)).abs().clamp(max=200.0), 0.0))
    q_abs = (q * q_rel).sum(1)
    gap = torch.where(q > 0, (logq - lpk).abs() + 1.0, 0.0)
    gap = torch.where(gap.isinf(), 0.0, gap)
    tol = tau * tau * w.abs() * ((q * q_rel * gap).sum(1) + 2.0 * r.sum_rel * (1.0 + r.lse.abs() * 0.0) + 3.0 * q_abs *
                                 (1.0 + torch.where(rest > 0, rest.clamp(min=1e-300).log().abs() + log_out.abs(), 0.0))) + 2.0 ** -23 * (w * tau * tau * each).abs().nan_to_num(posinf=0.0)
    extra = torch.where(inside, 0.0, f.abs() * 3.0 * q_abs[:, None] * out_p / s_out.clamp(min=1e-300)[:, None]) if lse is not None else 0.0
    each = torch.where(live, w * tau * tau * each, 0.0)
    return each, tol, torch.where(live[:, None], want, 0.0), torch.where(live[:, None], base, 0.0), extra, r


def _teacher(rows, classes, k, g, spread=2.0):
    lo = torch.arange(k, device="cuda") * classes // k
    hi = torch.arange(1, k + 1, device="cuda") * classes // k
    idx = lo + (torch.rand(rows, k, generator=g, device="cuda") * (hi - lo)).long().minimum(hi - lo - 1)
    idx = idx.gather(1, torch.rand(rows, k, generator=g, device="cuda").argsort(1))
    return idx.int(), torch.randn(rows, k, generator=g, device="cuda") * spread + 3.0


def check_distill(ctx, x, classes, idx, values, lse=None, weights=None, tau=1.0, scale=1.0, out=None):
    each, tol, want, base, extra, r = distill_reference(x.data, classes, tau, idx, values, lse, weights, scale)
    got = losses.distill_loss(ctx, x, idx, values, sk.DistillLossConfig(tau), teacher_lse=lse, weights=weights, classes=classes, grad_scale=scale, out=out)
    _close(got.loss, each, tol, "loss")
    _gradient(got.d_logits, want, base, r, classes, extra)
    return got


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("rows,classes", SIZES)
def test_distillation(gpu_ctx, rows, classes, kind):
    for n, (pad, offset, tau, k, tail, weighted) in enumerate(((0, 0, 1.0, 1, False, False), (3, 1, 2.0, 20, True, True), (-classes % 64, 5, 4.0, 64, False, True),
                                                               (1, 2, 1.0, 300, True, False))):
        k = min(k, classes)
        if classes > losses.MAX_LIST_CLASSES:
            continue
        x, g = _logits(rows, classes, pad, kind, offset, seed=n)
        idx, values = _teacher(rows, classes, k, g)
        idx[:, k - k // 3:] = -1                                     # unused entries
        values = values.to(DT[["f32", "f16", "bf16", "f32"][n]][0])
        lse = torch.logsumexp(torch.where(idx >= 0, values.double() / tau, -INF), 1).float() + 0.2 if tail else None
        weights = torch.rand(rows, generator=g, device="cuda") + 0.5 if weighted else None
        if weighted and rows > 2:
            weights[0] = 0.0
        check_distill(gpu_ctx, x, classes, idx, values, lse, weights, tau, 16.0)
    gpu_ctx.synchronize()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [12, 700, 5003])
def test_distillation_lists_that_are_empty_double_or_the_whole_row(gpu_ctx, classes, kind):
    x, g = _logits(8, classes, 4, kind, 1)
    k = 12
    idx, values = _teacher(8, classes, k, g)
    idx[0] = -1                                                       # nothing to learn from
    idx[1, 3:9] = idx[1, 2]                                           # one class seven times
    idx[2] = idx[2, 0]
    values[3, 4:] = -INF                                              # probability zero
    values[4] = -INF                                                  # a list of zeros
    x.data[5, :classes] = -INF                                        # the student has no class
    x.data[6, idx[6].long()] = -INF                                   # the student rules the list out: infinite loss, finite gradient
    for lse in (None, torch.logsumexp(values.double(), 1).float().nan_to_num(neginf=0.0) + 0.3):
        got = check_distill(gpu_ctx, x, classes, idx, values, lse)
        # with every class listed row 6 has none left and does not count, else its list has probability zero
        assert float(got.loss[6]) == (0.0 if classes == k else INF) and not got.d_logits.data[:, :classes].isnan().any()
        assert (got.d_logits.data[5] == 0).all() and float(got.loss[5]) == 0.0
        again = losses.distill_loss(gpu_ctx, x, idx, values, teacher_lse=lse, classes=classes)
        assert torch.equal(again.loss, got.loss) and torch.equal(again.d_logits.data, got.d_logits.data)
    if classes == k:                                                  # every class listed: no tail is left
        idx = torch.arange(k, device="cuda").int().expand(8, k).contiguous()
        check_distill(gpu_ctx, x, classes, idx, values, torch.logsumexp(values.double(), 1).float().nan_to_num(neginf=0.0))
    gpu_ctx.synchronize()


def test_distillation_index_out_of_range_and_over_the_logits(gpu_ctx):
    x, g = _logits(5, 3333, 3, "bf16", 1)
    idx, values = _teacher(5, 3333, 512, g)
    bad = idx.clone()
    bad[2, 7], bad[4, 0] = 3333, 2 ** 31 - 1
    idx[2, 7] = idx[4, 0] = -1
    want = check_distill(gpu_ctx, x, 3333, idx, values)
    gpu_ctx.synchronize()
    got = losses.distill_loss(gpu_ctx, x, bad, values, classes=3333, out=x)
    with pytest.raises(log.IndexOutOfRange, match="teacher"):
        gpu_ctx.synchronize()
    assert got.d_logits is x and torch.equal(x.data, want.d_logits.data) and torch.equal(got.loss, want.loss)


def test_distillation_at_the_most_classes(gpu_ctx):
    classes = losses.MAX_LIST_CLASSES
    x, g = _logits(1, classes, 1, "f16", 7)
    idx, values = _teacher(1, classes, 512, g)
    idx[0, :2] = torch.tensor([0, classes - 1])
    check_distill(gpu_ctx, x, classes, idx, values, torch.logsumexp(values.double(), 1).float() + 0.1, None, 1.0, 64.0)


# ---- policy -----------------------------------------------------------------------------------------------------

def _policy_inputs(x, classes, tau, g, with_ref):
    rows = x.data.shape[0]
    actions = torch.randint(0, classes, (rows,), generator=g, device="cuda").int()
    lp = Ref(x.data, classes, tau).pick(actions)
    step = 0.3 * torch.randn(rows, generator=g, device="cuda").double()
    ratio = step.exp()
    step = torch.where(((ratio - 0.8).abs() < 0.01) | ((ratio - 1.3).abs() < 0.01), 0.0, step)   # not next to the borders
    old = (lp - step).nan_to_num(neginf=-5.0, posinf=5.0).float()
    ref = (lp + 0.3 * torch.randn(rows, generator=g, device="cuda")).nan_to_num(neginf=-5.0, posinf=5.0).float() if with_ref else None
    return actions, old, torch.randn(rows, generator=g, device="cuda"), ref


def check_policy(ctx, x, classes, actions, old, adv, ref, weights, tau=1.0, beta=0.0, eta=0.0, scale=1.0, out=None):
    r = Ref(x.data, classes, tau)
    lo, hi = float(np.float32(1) - np.float32(0.2)), float(np.float32(1) + np.float32(0.3))
    cfg = sk.PolicyLossConfig(0.2, 0.3, beta, eta, tau)
    got = losses.policy_loss(ctx, x, actions, old, adv, cfg, logp_ref=ref, weights=weights, classes=classes, grad_scale=scale, out=out)
    ctx.synchronize()
    w = torch.ones_like(r.lse) if weights is None else weights.double()
    live = (w != 0) & (actions >= 0) & ~r.dead
    lp, a = r.pick(actions), adv.double()
    rho = (lp - old.double()).exp()
    clipped = ((a > 0) & (rho > hi)) | ((a < 0) & (rho < lo))
    d = ref.double() - lp if ref is not None else torch.zeros_like(lp)
    kl = torch.expm1(d) - d
    loss = torch.maximum(-rho * a, -rho.clamp(lo, hi) * a) + beta * kl - eta * r.h
    g = torch.where(clipped, 0.0, -a * rho) + beta * (1.0 - d.exp())
    zero = lambda v: torch.where(live, v, 0.0)  # noqa: E731
    dl = r.sum_rel + 2.0 ** -24 * lp.abs() * 0.0
    kl_tol = torch.expm1(d).abs() * dl + 2.0 ** -22 * (kl.abs() + d.abs() * (d.abs() > 0.5))
    _close(got.logp, zero(lp), dl + 2.0 ** -24 * lp.abs(), "logp")
    _close(got.kl, zero(kl), zero(kl_tol), "kl")
    _close(got.entropy, zero(r.h), zero(r.h_tol), "entropy")
    g_tol = a.abs() * rho * (dl + 2.0 ** -22 + 2.0 ** -24 * (lp - old.double()).abs()) + beta * d.exp() * (dl + 2.0 ** -22)
    _close(got.loss, zero(w * loss), zero(w.abs() * (g_tol + beta * kl_tol + eta * r.h_tol) + 2.0 ** -22 * (w * loss).abs()), "loss")
    k = scale / tau
    hit = torch.zeros_like(r.p).scatter_(1, actions.long().clamp(min=0)[:, None], 1.0)
    gw, ew = (k * g * w)[:, None], k * eta * w[:, None]
    want = gw * (hit - r.p) + ew * (r.plogp + r.p * r.h[:, None])
    base = gw.abs() * (hit + r.p) + ew.abs() * (r.plogp.abs() + r.p * r.h[:, None] + r.p) * 2.0
    extra = (k * w.abs() * g_tol)[:, None] * (hit + r.p)
    z2 = lambda v: torch.where(live[:, None], v, 0.0)  # noqa: E731
    _gradient(got.d_logits, z2(want), z2(base), r, classes, z2(extra))
    return got


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("rows,classes", SIZES)
def test_policy(gpu_ctx, rows, classes, kind):
    for n, (pad, offset, tau, beta, eta, weighted) in enumerate(((0, 0, 1.0, 0.0, 0.0, False), (6, 3, 0.7, 0.1, 0.0, True), (-classes % 64, 1, 1.5, 0.05, 0.02, True))):
        x, g = _logits(rows, classes, pad, kind, offset, seed=n + 10)
        actions, old, adv, ref = _policy_inputs(x, classes, tau, g, beta > 0)
        weights = torch.rand(rows, generator=g, device="cuda") + 0.5 if weighted else None
        if rows > 2:
            actions[1] = -1
            if weighted:
                weights[0] = 0.0
                adv[0] = math.nan
                x.data[0, 0] = math.nan
        if weighted and rows > 2:      # the row that does not count holds NaN: the reference gets a clean copy
            check = x.data.clone()
            got = losses.policy_loss(gpu_ctx, x, actions, old, adv, sk.PolicyLossConfig(0.2, 0.3, beta, eta, tau), logp_ref=ref, weights=weights,
                                     classes=classes, grad_scale=32.0)
            for t in got[:4]:
                assert float(t[0]) == 0.0
            assert (got.d_logits.data[0] == 0).all()
            check[0, 0], adv[0] = 0.0, 1.0
            x = sk.Tensor(check, DT[kind][1], take_id=False)
        check_policy(gpu_ctx, x, classes, actions, old, adv, ref, weights, tau, beta, eta, 32.0)


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes", [10, 2049])
def test_policy_clips_on_the_side_of_the_advantage(gpu_ctx, classes, kind):
    x, g = _logits(6, classes, 0, kind)
    actions = torch.randint(0, classes, (6,), generator=g, device="cuda").int()
    lp = Ref(x.data, classes, 1.0).pick(actions)
    ratio = torch.tensor([0.5, 0.5, 1.0, 1.0, 2.0, 2.0], device="cuda", dtype=torch.float64)
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0], device="cuda")
    got = check_policy(gpu_ctx, x, classes, actions, (lp - ratio.log()).float(), adv, None, None)
    assert [bool((row != 0).any()) for row in got.d_logits.data] == [True, False, True, True, False, True]


# ---- preference ------------------------------------------------------------------------------------------------

def check_preference(ctx, x, classes, labels, offsets, cfg, ref=None, weights=None, scale=1.0, out=None):
    r = Ref(x.data, classes, cfg.temperature)
    off = [int(v) for v in offsets]
    rows, pairs = labels.shape[0], len(off) // 2
    got = losses.preference_loss(ctx, x, labels, offsets, cfg, logp_ref=ref, weights=weights, classes=classes, grad_scale=scale, out=out)
    ctx.synchronize()
    at = torch.arange(rows, device="cuda")
    live = (labels >= 0) & ~r.dead & (at >= off[0]) & (at < off[-1])
    lp = torch.where(live, r.pick(labels), 0.0)
    _close(got.row_logp, lp, r.sum_rel + 2.0 ** -24 * lp.abs(), "row_logp")
    sums, tols, counts = [], [], []
    for a, b in zip(off[:-1], off[1:]):
        n = int(live[a:b].sum())
        by = max(1, n) if cfg.average else 1
        counts.append(by)
        sums.append(lp[a:b].sum() / by)
        tols.append((r.sum_rel[a:b] * live[a:b]).sum() / by)
    if pairs == 0:
        assert (got.d_logits.data == 0).all()
        return got
    s, t = torch.stack(sums), torch.stack(tols) + 2.0 ** -40 * torch.stack(sums).abs()
    _close(got.logp, s, t + 2.0 ** -24 * s.abs(), "logp")
    h = s - (ref.double() if ref is not None else 0.0)
    beta, eps = float(np.float32(cfg.beta)), float(np.float32(cfg.label_smoothing))
    m = beta * (h[0::2] - h[1::2]) - float(np.float32(cfg.target_margin))
    m_tol = abs(beta) * (t[0::2] + t[1::2]) + 1e-14 * beta * (s.abs().sum())
    _close(got.margin, m, m_tol + 2.0 ** -24 * m.abs(), "margin")
    if cfg.form == sk.PreferenceForm.Sigmoid:
        ls = torch.nn.functional.logsigmoid
        loss, dm, bend = -(1 - eps) * ls(m) - eps * ls(-m), eps - torch.sigmoid(-m), 0.25
    elif cfg.form == sk.PreferenceForm.Hinge:
        loss, dm, bend = torch.relu(1 - m), -(m < 1).double(), 0.0
    else:
        loss, dm, bend = (m - 0.5) ** 2, 2 * (m - 0.5), 2.0
    w = torch.ones_like(m) if weights is None else weights.double()
    _close(got.loss, w * loss, w.abs() * (dm.abs() + m_tol * bend) * m_tol + 2.0 ** -23 * (w * loss).abs() + 1e-14, "loss")
    g, g_tol = torch.zeros(rows, dtype=torch.float64, device="cuda"), torch.zeros(rows, dtype=torch.float64, device="cuda")
    for i, (a, b) in enumerate(zip(off[:-1], off[1:])):
        sign = -beta if i % 2 else beta
        g[a:b], g_tol[a:b] = w[i // 2] * dm[i // 2] * sign / counts[i], (w[i // 2] * bend * m_tol[i // 2] * beta).abs() / counts[i]
    k = scale / cfg.temperature
    g, g_tol = torch.where(live, g, 0.0)[:, None] * k, torch.where(live, g_tol, 0.0)[:, None] * k
    hit = torch.zeros_like(r.p).scatter_(1, labels.long().clamp(min=0)[:, None], 1.0)
    _gradient(got.d_logits, g * (hit - r.p), g.abs() * (hit + r.p), r, classes, g_tol * (hit + r.p))
    return got


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes", [1, 7, 1000, 1026, 4099, 32768, 100003])
def test_preference(gpu_ctx, classes, kind):
    rows = 40 if classes < 5000 else 12
    cuts = [2, 9, 9, 10, 30, 31, 38] if rows == 40 else [1, 3, 3, 4, 8, 9, 11]    # an empty sequence, sequences of one row, rows before and behind
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    for n, (form, eps, margin, average, tau, pad, offset) in enumerate((
            (sk.PreferenceForm.Sigmoid, 0.0, 0.0, False, 1.0, 0, 0), (sk.PreferenceForm.Sigmoid, 0.1, 0.5, True, 0.7, 3, 1),
            (sk.PreferenceForm.Hinge, 0.0, 0.0, False, 1.0, -classes % 64, 0), (sk.PreferenceForm.Squared, 0.0, 0.2, True, 2.0, 1, 5))):
        x, g = _logits(rows, classes, pad, kind, offset, seed=n + 30)
        labels = torch.randint(0, classes, (rows,), generator=g, device="cuda").int()
        labels[::5] = -1
        cfg = sk.PreferenceLossConfig(form, 0.05, eps, margin, average, tau)
        ref = torch.randn(6, generator=g, device="cuda") * 3.0 - 10.0 if n else None
        weights = torch.tensor([0.5, 2.0, 1.0], device="cuda") if n == 1 else None
        check_preference(gpu_ctx, x, classes, labels, offsets, cfg, ref, weights, 32.0)


def test_preference_extremes(gpu_ctx):
    x, g = _logits(10, 100, 4, "f32", 1)
    labels = torch.randint(0, 100, (10,), generator=g, device="cuda").int()
    one = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    cfg = sk.PreferenceLossConfig(beta=0.1)
    check_preference(gpu_ctx, x, 100, labels, one(0), cfg)                       # no pair
    check_preference(gpu_ctx, x, 100, labels, one(4, 4, 4), cfg)                 # two empty sequences
    check_preference(gpu_ctx, x, 100, labels, one(0, 5, 10), cfg, torch.tensor([3000.0, -3000.0], device="cuda"))    # margins where exp overflows
    check_preference(gpu_ctx, x, 100, labels, one(0, 5, 10), cfg, torch.tensor([-30000.0, 30000.0], device="cuda"))
    x.data[2, :100] = -INF                                                       # a row without classes does not count
    check_preference(gpu_ctx, x, 100, labels, one(0, 5, 10), sk.PreferenceLossConfig(beta=0.1, average=True))
    x.data[7, labels[7].long()] = -INF                                           # the rejected one is impossible: nothing left to learn
    got = losses.preference_loss(gpu_ctx, x, labels, one(0, 5, 10), cfg, classes=100)
    assert float(got.margin) == INF and float(got.loss) == 0.0 and (got.d_logits.data == 0).all()
    got = losses.preference_loss(gpu_ctx, x, labels, one(0, 5, 10), cfg, weights=torch.zeros(1, device="cuda"), classes=100)
    assert float(got.loss) == 0.0 and (got.d_logits.data == 0).all()
    none = sk.Tensor(x.data[:0], sk.Precision.FP32, take_id=False)
    got = losses.preference_loss(gpu_ctx, none, labels[:0], one(0, 0, 0), cfg, classes=100)
    assert abs(float(got.loss) - math.log(2.0)) < 1e-6 and got.d_logits.data.shape == (0, 104)
    gpu_ctx.synchronize()


def test_preference_offsets_out_of_range_are_reported(gpu_ctx):
    x, g = _logits(10, 100, 0, "bf16")
    labels = torch.randint(0, 100, (10,), generator=g, device="cuda").int()
    for cuts in ([0, 5, 11], [0, 7, 4], [-1, 5, 10], [0, 2 ** 31 - 1, -2 ** 31]):
        got = losses.preference_loss(gpu_ctx, x, labels, torch.tensor(cuts, dtype=torch.int32, device="cuda"))
        with pytest.raises(log.IndexOutOfRange, match="offset"):
            gpu_ctx.synchronize()
        assert got.loss.isfinite().all()


def test_long_sequences_keep_their_margin(gpu_ctx):
    """The sums of a thousand rows are two orders above their difference: 64 bits hold them."""
    x, g = _logits(3000, 500, 0, "bf16")
    labels = torch.randint(0, 500, (3000,), generator=g, device="cuda").int()
    lp = Ref(x.data, 500, 1.0).pick(labels)
    ref = torch.stack([lp[:2600].sum(), lp[2600:].sum()]).float() - 1.0
    got = losses.preference_loss(gpu_ctx, x, labels, torch.tensor([0, 2600, 3000], dtype=torch.int32, device="cuda"), logp_ref=ref)
    h = lp[:2600].sum() - ref[0].double() - lp[2600:].sum() + ref[1].double()
    # 3000 rows: each log s off by a part of 2^-22 of either sign, the mean of ex2's error taken out (below 1e-8)
    assert abs(float(got.margin) - 0.1 * float(h)) < 0.1 * (2200 * 2e-8 + 2.0 ** -22 * math.sqrt(3000) + 2.0 ** -24 * 3000 ** 0.5 * 8)


# ---- all of them ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes,tau", [(20, 0.7), (20, 1.0), (3000, 0.7), (3000, 1.0), (20000, 0.7)])
def test_a_sequence_adds_no_bias_of_its_rows(gpu_ctx, classes, tau, kind):
    """4000 rows in one sequence. A row's error is a few roundings of 2^-24 and averages out (3e-7 a row makes 2e-5 of the
    sum, five times that is allowed), but for the part that has one sign in all of them: 5e-8 a row is allowed."""
    rows = 4000
    x, g = _logits(rows, classes, 0, kind, scale=1.0)
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda").int()
    at = torch.tensor([0, rows, rows], dtype=torch.int32, device="cuda")
    t = float(np.float32(tau))
    want = sum(float(torch.log_softmax(a.double() / t, 1).gather(1, b[:, None].long()).sum())
               for a, b in zip(x.data.split(500), labels.split(500)))
    ref = torch.tensor([want, 0.0], device="cuda")          # in f32: what it lacks is the margin's
    got = losses.preference_loss(gpu_ctx, x, labels, at, sk.PreferenceLossConfig(beta=1.0, temperature=tau), logp_ref=ref, gradient=False)
    assert abs(float(got.margin) - (want - float(ref[0].double()))) <= rows * 5e-8 + 5 * 3e-7 * rows ** 0.5


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("classes", [8, 64, 1000])
def test_labels_that_are_nearly_certain(gpu_ctx, classes, kind):
    """log p = -log1p(the rest's sum) keeps relative places where the label's own thread adds few classes: at most 4 chains
    of 8 sums with 1 in them (one unit of it up to 64 classes), 2^-24 each, beside the f32 terms of the rest and the label's own rounding of the difference."""
    rows = 256
    for rest in (0.3, 1e-2, 1e-4):
        x, g = _logits(rows, classes, 0, kind, seed=5, scale=2.0)
        labels = torch.randint(0, classes, (rows,), generator=g, device="cuda")
        x.data.scatter_(1, labels[:, None], -INF)
        top = torch.logsumexp(x.data.float(), 1, keepdim=True) - math.log(rest)
        x.data.scatter_(1, labels[:, None], top.to(x.data.dtype))
        want = torch.log_softmax(x.data.double(), 1).gather(1, labels[:, None])[:, 0]
        got = losses.label_logprob(gpu_ctx, x, labels.int()).logp.double()
        adds = 6 if classes <= 64 else 32
        assert ((got - want).abs() <= adds * 2.0 ** -24 + want.abs() * (2.0 ** -24 + 2.0 ** -22 + 2.0 ** -23 * 32)).all()


def _calls(x, g, classes):
    rows = x.data.shape[0]
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda").int()
    vec = [torch.randn(rows, generator=g, device="cuda") for _ in range(3)]
    idx, values = _teacher(rows, classes, min(5, classes), g)
    offsets = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
    cfg = sk.PolicyLossConfig(kl_coeff=0.1, entropy_coeff=0.02)
    return {
        "logprob": lambda ctx, **o: [losses.label_logprob(ctx, x, labels, entropy=True).logp],
        "logprob_backward": lambda ctx, **o: [losses.label_logprob_backward(ctx, x, labels, vec[0], vec[1], **o).data],
        "distill": lambda ctx, **o: [(r := losses.distill_loss(ctx, x, idx, values, teacher_lse=vec[0].abs() + 9.0, **o)).loss, r.d_logits.data],
        "policy": lambda ctx, **o: [(r := losses.policy_loss(ctx, x, labels, vec[0] - 5, vec[1], cfg, logp_ref=vec[2] - 5, **o)).loss, r.kl, r.entropy, r.d_logits.data],
        "preference": lambda ctx, **o: [(r := losses.preference_loss(ctx, x, labels, offsets, **o)).loss, r.row_logp, r.d_logits.data],
    }


@pytest.mark.parametrize("name", ["logprob_backward", "policy", "distill", "preference"])
def test_gradients_against_differences(gpu_ctx, name):
    """f32 losses at x +- h in one class of each row: f32 noise 2^-21 |L| / h, curvature h^2. The sum of the row losses that a
    row's logits enter."""
    rows, classes, h = 6, 11, 2.0 ** -6
    x, g = _logits(rows, classes, 0, "f32", scale=1.0)
    calls = _calls(x, g, classes)
    # as functions of the logits
    if name == "logprob_backward":
        labels, w, v = torch.randint(0, classes, (rows,), generator=g, device="cuda").int(), *[torch.randn(rows, generator=g, device="cuda") for _ in range(2)]
        value = lambda: (lambda r: float((r.logp.double() * w + r.entropy.double() * v).sum()))(losses.label_logprob(gpu_ctx, x, labels, entropy=True))  # noqa: E731
        d = losses.label_logprob_backward(gpu_ctx, x, labels, w, v).data
    else:
        value = lambda: float(calls[name](gpu_ctx)[0].double().sum())  # noqa: E731
        d = calls[name](gpu_ctx)[-1]
    d = d.clone()
    for row, c in ((0, 0), (1, 10), (2, 5), (3, 3), (4, 7), (5, 1)):
        kept = float(x.data[row, c])
        x.data[row, c] = kept + h
        up = value()
        x.data[row, c] = kept - h
        down = value()
        x.data[row, c] = kept
        slope = (up - down) / (2 * h)
        size = max(abs(up), abs(down), 10.0)
        assert abs(slope - float(d[row, c])) < 2.0 ** -21 * size * 4 / h + 4 * h * h * max(1.0, float(d[row].abs().max())), (row, c)


@pytest.mark.parametrize("classes", [10, 700, 5001, 70001])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_same_bits_again_on_another_stream_and_recorded(gpu_ctx, classes, kind):
    x, g = _logits(8, classes, 0, kind)
    calls = _calls(x, g, classes)
    want = {n: [t.clone() for t in f(gpu_ctx)] for n, f in calls.items()}
    for n, f in calls.items():
        for a, b in zip(f(gpu_ctx), want[n]):
            assert torch.equal(a, b), n
    side = torch.cuda.Stream()
    other = sk.GpuContext(16, 0, stream=side)
    torch.cuda.synchronize()
    got = {n: f(other) for n, f in calls.items()}
    other.synchronize()
    for n in calls:
        for a, b in zip(got[n], want[n]):
            assert torch.equal(a, b), n
    for _ in range(3):                         # a step's first round runs as it is, the later ones as one graph
        with gpu_ctx.step_graph(3):
            got = {n: f(gpu_ctx) for n, f in calls.items()}
        gpu_ctx.synchronize()
        for n in calls:
            for a, b in zip(got[n], want[n]):
                assert torch.equal(a, b), n
    # the caller's own graph, replayed on new values at the same place
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = {n: f(other) for n, f in calls.items()}
        before = x.data.clone()
        x.data.zero_()
        graph.replay()
        side.synchronize()
        assert not torch.equal(got["policy"][0], want["policy"][0])
        x.data.copy_(before)
        graph.replay()
    side.synchronize()
    for n in calls:
        for a, b in zip(got[n], want[n]):
            assert torch.equal(a, b), n
    del graph
    other.close()


def test_a_step_slot_takes_rows_of_any_width(gpu_ctx):
    """Wide rows are shared by the blocks of a cluster, narrow ones are not: one slot, one sequence of kernels, other clusters."""
    made = []
    for classes in (10, 70001, 700, 131072, 33, 40009, 250001):
        x, g = _logits(5, classes, 0, "f32")
        calls = _calls(x, g, classes)
        made.append((calls, {n: [t.clone() for t in f(gpu_ctx)] for n, f in calls.items()}))
    for _ in range(2):
        for calls, want in made:
            with gpu_ctx.step_graph(2):
                got = {n: f(gpu_ctx) for n, f in calls.items()}
            gpu_ctx.synchronize()
            for n in calls:
                for a, b in zip(got[n], want[n]):
                    assert torch.equal(a, b), n


def test_two_graphs_of_preference_losses_at_once(gpu_ctx):
    """Nothing is shared between calls: two recorded passes of one context replay beside each other."""
    side = torch.cuda.Stream()
    ctx = sk.GpuContext(16, 0, stream=side)
    made = []
    for seed in (1, 2):
        x, g = _logits(64, 20001, 0, "bf16", seed=seed)
        call = _calls(x, g, 20001)["preference"]
        want = [t.clone() for t in call(gpu_ctx)]
        gpu_ctx.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = call(ctx)
        made.append((graph, got, want, x, call))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, *_), s in zip(made, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, got, want, *_ in made:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    del made
    ctx.close()


def test_rows_behind_32_bits(gpu_ctx):
    """The last rows of a matrix of more than 2^32 elements."""
    rows, classes = 33000, 131072
    x = sk.Tensor(torch.zeros(rows, classes, dtype=torch.float16, device="cuda"), sk.Precision.FP16, take_id=False)
    g = _rng(3)
    labels = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    labels[-2:] = torch.tensor([5, 131071], dtype=torch.int32)
    x.data[-2:] = torch.randn(2, classes, generator=g, device="cuda").half()
    tail = sk.Tensor(x.data[-2:].clone(), sk.Precision.FP16, take_id=False)
    ones = torch.ones(rows, device="cuda")
    want = losses.label_logprob_backward(gpu_ctx, tail, labels[-2:].clone(), ones[:2])
    got = losses.label_logprob_backward(gpu_ctx, x, labels, ones, out=x)
    # The two calls share their rows among different numbers of blocks, so the sums are added in another order: chains of
    # at most 131072 / 1024 + 40 terms of 2^-24 each, below 2^-16 of the sum. Two values that near round to the same f16
    # or to neighbours, which are at most 2^-10 of the value (2^-24 where it is subnormal) apart.
    a, b = got.data[-2:].double(), want.data.double()
    assert ((a - b).abs() <= (b.abs() * 2.0 ** -10).clamp(min=2.0 ** -24) + 2.0 ** -16 * b.abs()).all()
    assert float(got.data[:64].abs().max()) == 0.0 and float(got.data[32800:-2].abs().max()) == 0.0
    del got, x
    torch.cuda.empty_cache()


def test_no_rows(gpu_ctx):
    x = sk.Tensor(torch.empty(0, 40, dtype=torch.float16, device="cuda"), sk.Precision.FP16, take_id=False)
    i, f = torch.empty(0, dtype=torch.int32, device="cuda"), torch.empty(0, device="cuda")
    assert losses.label_logprob(gpu_ctx, x, i).logp.shape == (0,)
    assert losses.label_logprob_backward(gpu_ctx, x, i, f).data.shape == (0, 40)
    assert losses.policy_loss(gpu_ctx, x, i, f, f).loss.shape == (0,)
    assert losses.distill_loss(gpu_ctx, x, i.view(0, 4), f.view(0, 4)).loss.shape == (0,)
    gpu_ctx.synchronize()


def test_losses_without_gradients(gpu_ctx):
    x, g = _logits(6, 1500, 0, "bf16")
    calls = _calls(x, g, 1500)
    labels = torch.randint(0, 1500, (6,), generator=g, device="cuda").int()
    v = torch.randn(6, generator=g, device="cuda") - 5
    a, b = (losses.policy_loss(gpu_ctx, x, labels, v, v, gradient=w) for w in (True, False))
    assert b.d_logits is None and all(torch.equal(s, t) for s, t in zip(a[:4], b[:4]))
    idx, values = _teacher(6, 1500, 7, g)
    a, b = (losses.distill_loss(gpu_ctx, x, idx, values, gradient=w) for w in (True, False))
    assert b.d_logits is None and torch.equal(a.loss, b.loss)
    off = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    a, b = (losses.preference_loss(gpu_ctx, x, labels, off, gradient=w) for w in (True, False))
    assert b.d_logits is None and torch.equal(a.loss, b.loss) and torch.equal(a.row_logp, b.row_logp)
    del calls


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,classes", [(300, 40009), (7, 131072), (200, 131075), (40, 3001), (700, 90)])
def test_gradients_over_the_logits_they_come_from(gpu_ctx, rows, classes, kind):
    """Blocks that share a row write their part while others may still be at theirs."""
    x, g = _logits(rows, classes, 3, kind, 1, scale=2.0)
    labels = _label_rows(rows, classes, g)
    vec = [torch.randn(rows, generator=g, device="cuda") for _ in range(3)]
    idx, values = _teacher(rows, classes, 40, g)
    offsets = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
    cfg = sk.PolicyLossConfig(kl_coeff=0.1, entropy_coeff=0.02)
    for call in (lambda t, o: losses.label_logprob_backward(gpu_ctx, t, labels, vec[0], vec[1], classes=classes, out=o),
                 lambda t, o: losses.policy_loss(gpu_ctx, t, labels, vec[0] - 9, vec[1], cfg, logp_ref=vec[2] - 9, classes=classes, out=o).d_logits,
                 lambda t, o: losses.distill_loss(gpu_ctx, t, idx, values, teacher_lse=vec[0].abs() + 8.0, classes=classes, out=o).d_logits,
                 lambda t, o: losses.preference_loss(gpu_ctx, t, labels, offsets, classes=classes, out=o).d_logits):
        want = call(x, None).data
        flat = torch.empty(x.len() + 1, dtype=x.data.dtype, device="cuda")        # at the same offset within 16 bytes, on which sums depend
        over = sk.Tensor(flat[1:].view(x.data.shape).copy_(x.data), x.precision, take_id=False)
        assert call(over, over) is over
        gpu_ctx.synchronize()
        assert torch.equal(over.data, want)


def test_inputs_of_another_stream_are_kept(gpu_ctx):
    """A context on a stream of its own: memory of inputs that are dropped right after the call is not handed out while
    the call still reads it."""
    side = torch.cuda.Stream()
    ctx = sk.GpuContext(16, 0, stream=side)
    rows, classes = 512, 32768
    x, g = _logits(rows, classes, 0, "bf16")
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda").int()
    want = losses.label_logprob_backward(gpu_ctx, x, labels, torch.full((rows,), 2.0, device="cuda")).data.clone()
    out = sk.Tensor(torch.empty_like(x.data), sk.Precision.BF16, take_id=False)
    for _ in range(5):
        scale = torch.full((rows,), 2.0, device="cuda")
        torch.cuda.synchronize()
        for _ in range(8):                     # several passes queue up
            losses.label_logprob_backward(ctx, x, labels, scale, out=out)
        del scale
        for _ in range(4):
            torch.full((rows,), 7.0, device="cuda")
        ctx.synchronize()
        assert torch.equal(out.data, want)
    ctx.close()


# ---- networks ----------------------------------------------------------------------------------------------------

def _network(ctx, prec, dims=(40, 64, 30), batch=24, seed=7, norm=sk.Normalisation.Disabled):
    sk.reset_tensor_ids(0)
    init = sk.InitXavierNormalFunc(seed)
    cfgs = [sk.LayerInitConfig(sk.Normalisation.RMSNorm, sk.Activation.SiLU)] * (len(dims) - 2) + [sk.LayerInitConfig(norm)]
    layers = [sk.DenseBlock(ctx, True, a, b, batch, init, c, prec) for a, b, c in zip(dims[:-1], dims[1:], cfgs)]
    return sk.FeedForwardNetwork(layers, dims[0])


def _state(net):
    return [t.data.clone() for l in net.get_layers() for t in (l.get_weights(), l.get_biases(), l.get_dv_weights(), l.get_norm_weights())]


@pytest.mark.parametrize("prec", [sk.Precision.FP32, sk.Precision.FP16, sk.Precision.BF16])
@pytest.mark.parametrize("graph", [False, True])
def test_log_probabilities_train_a_network_as_cross_entropy_does(gpu_ctx, prec, graph):
    """The gradient of -log p is softmax minus one-hot, what CrossEntropyLoss sends back: the same steps up to one
    rounding of the gradient to the storage type (half a step of eps) per step."""
    batch, steps = 24, 3
    g = _rng(11)
    xs = torch.randn(batch, 40, generator=g, device="cuda")
    labels = torch.randint(0, 30, (batch,), generator=g, device="cuda").int()
    dt = sk.core.TORCH_DTYPE[prec]
    x = sk.Tensor(xs.to(dt), prec)
    target = sk.Tensor(torch.nn.functional.one_hot(labels.long(), 30).to(dt), prec)
    opt = [sk.Optimiser.SGD(0.9, True)] * 2
    train = sk.MultiLayerTrainContext(opt, opt, batch, 0.05)
    minus = torch.full((batch,), -1.0, device="cuda")
    states = []
    for own in (False, True):
        net = _network(gpu_ctx, prec)
        for step in range(1, steps + 1):
            def one():
                outs = net.forward(gpu_ctx, x, batch, False, step)
                if own:
                    d = losses.label_logprob_backward(gpu_ctx, outs[-1], labels, minus, grad_scale=32.0)
                    net.backward_gradient(gpu_ctx, outs, d, x, train, step, grad_scale=32.0)
                else:
                    net.backward(gpu_ctx, outs, target, x, sk.LossConfig(sk.LossFunc.CrossEntropyLoss, sk.Activation.Softmax), train, step)
            if graph:
                with gpu_ctx.step_graph(4):
                    one()
            else:
                one()
        gpu_ctx.synchronize()
        states.append(_state(net))
    eps = {sk.Precision.FP32: 2.0 ** -20, sk.Precision.FP16: 2.0 ** -9, sk.Precision.BF16: 2.0 ** -6}[prec]
    for a, b in zip(*states):
        assert float((a.double() - b.double()).abs().max()) <= 2 * steps * eps * max(float(b.double().abs().max()), 1e-3)


@pytest.mark.parametrize("prec", [sk.Precision.FP32, sk.Precision.BF16])
def test_a_policy_is_recorded_stepped_and_distilled(gpu_ctx, prec):
    """The calls together, as they are used: log-probabilities of the old policy, policy and preference steps, and a second
    network that learns from the first one's top logits. The first block's weights after one SGD step are the formula's."""
    batch, actions_n = 24, 30
    g = _rng(12)
    dt = sk.core.TORCH_DTYPE[prec]
    x = sk.Tensor(torch.randn(batch, 40, generator=g, device="cuda").to(dt), prec)
    net = _network(gpu_ctx, prec, dims=(40, actions_n))
    opt = [sk.Optimiser.SGD(0.0, False)]
    train = sk.MultiLayerTrainContext(opt, opt, batch, 0.5)
    actions = torch.randint(0, actions_n, (batch,), generator=g, device="cuda").int()
    outs = net.forward(gpu_ctx, x, batch, False, 1)
    old = losses.label_logprob(gpu_ctx, outs[-1], actions).logp
    adv = torch.randn(batch, generator=g, device="cuda")
    w0 = net.get_layers()[0].get_weights().data.double().clone()
    z = x.data.double() @ w0
    got = losses.policy_loss(gpu_ctx, outs[-1], actions, old, adv, sk.PolicyLossConfig(kl_coeff=0.1), logp_ref=old, grad_scale=32.0)
    net.backward_gradient(gpu_ctx, outs, got.d_logits, x, train, 1, grad_scale=32.0)
    gpu_ctx.synchronize()
    # at ratio 1 and d = 0 the gradient is -A (onehot - p)
    p = torch.softmax(z, 1)
    dz = -adv.double()[:, None] * (torch.nn.functional.one_hot(actions.long(), actions_n) - p)
    want = w0 - 0.5 * (x.data.double().T @ dz) / batch
    got_w = net.get_layers()[0].get_weights().data.double()
    eps = torch.finfo(dt).eps
    # logits rounded to T (absolute error eps / 2 |z|, in p at most that), the gradient rounded to T twice, the weights once
    bound = 0.5 / batch * (x.data.double().abs().T @ ((eps * z.abs().max() + 2 * eps) * adv.double().abs()[:, None].expand(-1, actions_n))) + eps * w0.abs() + 1e-5 * (dt == torch.float32)
    assert ((got_w - want).abs() <= bound).all()
    assert float(got.kl.abs().max()) < 1e-6 and torch.allclose(got.loss, -adv, atol=1e-5)
    outs = net.forward(gpu_ctx, x, batch, False, 2)
    pref = losses.preference_loss(gpu_ctx, outs[-1], actions, torch.tensor([0, 6, 12, 18, 24], dtype=torch.int32, device="cuda"), grad_scale=32.0)
    net.backward_gradient(gpu_ctx, outs, pref.d_logits, x, train, 2, grad_scale=32.0)
    teacher = net.forward(gpu_ctx, x, batch, False, 3)[-1].data.float()
    top = teacher.topk(8, 1)
    student = _network(gpu_ctx, prec, dims=(40, 64, actions_n), seed=8)
    two = sk.MultiLayerTrainContext(opt * 2, opt * 2, batch, 0.5)
    outs = student.forward(gpu_ctx, x, batch, False, 1)
    kd = losses.distill_loss(gpu_ctx, outs[-1], top.indices.int(), top.values, teacher_lse=torch.logsumexp(teacher, 1), grad_scale=32.0)
    before = _state(student)
    student.backward_gradient(gpu_ctx, outs, kd.d_logits, x, two, 1, grad_scale=32.0)
    gpu_ctx.synchronize()
    assert (kd.loss > 0).all() and not any(torch.equal(a, b) for a, b in zip(before[:2], _state(student)[:2]))
    # the same gradient by hand: KL of all classes when the whole row is the list
    full = losses.distill_loss(gpu_ctx, outs[-1], torch.arange(actions_n, device="cuda").int().expand(batch, -1).contiguous(), teacher)
    q, lp = torch.softmax(teacher.double(), 1), torch.log_softmax(outs[-1].data.double(), 1)
    assert torch.allclose(full.loss.double(), (q * (q.log() - lp)).sum(1), atol=1e-5)


@pytest.mark.parametrize("prec", [sk.Precision.FP32, sk.Precision.FP16])
@pytest.mark.parametrize("norm,act", [(0, 0), (1, 6), (2, 7), (3, 4), (0, 1)])
def test_output_gradient_is_the_hidden_blocks_backward(gpu_ctx, prec, norm, act):
    """A block whose gradient arrives through an identity product and one that is given it take the same steps."""
    n, batch = 32, 16
    g = _rng(norm * 10 + act)
    dt = sk.core.TORCH_DTYPE[prec]
    cfg = sk.LayerInitConfig(sk.Normalisation(norm), sk.Activation(act))
    opt = sk.Optimiser.SGD(0.0, False)
    train = sk.TrainContext(opt, opt, batch, 0.1)
    x = sk.Tensor(torch.randn(batch, 24, generator=g, device="cuda").to(dt), prec)
    d = (torch.randn(batch, n, generator=g, device="cuda") / 8).to(dt)
    states = []
    for hidden in (True, False):
        sk.reset_tensor_ids(0)
        blk = sk.DenseBlock(gpu_ctx, True, 24, n, batch, sk.InitXavierNormalFunc(3), cfg, prec)
        blk.forward(gpu_ctx, x, batch, False, 1)
        if hidden:                             # the block behind it: unit weights, delta d
            nxt = sk.DenseBlock(gpu_ctx, True, n, n, batch, sk.InitZeroFunc(), None, prec)
            nxt.get_weights().data.copy_(torch.eye(n, device="cuda"))
            nxt.get_delta_prenorm_out().data.copy_(d.float() * 512.0)
            if nxt.d_prenorm_lp is not None:
                nxt.d_prenorm_lp.data.copy_(d.float() * 32.0)
            blk.backward_hidden(gpu_ctx, nxt, x, train, 1)
        else:
            blk.output_gradient(gpu_ctx, sk.Tensor(d * 4.0, prec), batch, grad_scale=4.0)
            blk.backward_output(gpu_ctx, x, train, 1)
        gpu_ctx.synchronize()
        states.append([t.data.double().clone() for t in (blk.get_grads(), blk.get_delta_prenorm_out(), blk.get_norm_weights_grad(), blk.get_weights(), blk.get_biases(),
                                                         blk.get_norm_weights())])
    for a, b in zip(*states):
        assert float((a - b).abs().max()) <= 2.0 ** -20 * max(float(a.abs().max()), 1e-6)


# ---- refusals -----------------------------------------------------------------------------------------------------

def test_native_refusals(gpu_ctx):
    """Wrong calls of the C ABI come back with their status and launch nothing."""
    import ctypes as C
    from soklyn_b200 import _native as N
    lib, h = gpu_ctx.lib, gpu_ctx.handle
    x, g = _logits(4, 50, 6, "f16")
    y = torch.zeros(4 * 56 + 64, dtype=torch.float16, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    f = torch.zeros(256, device="cuda")
    good = dict(dtype=1, rows=4, cols=56, classes=50, logits=x.ptr(), d_logits=y.data_ptr(), temperature=1.0, grad_scale=1.0)
    rows = lambda **o: C.byref(N.SkLogits(**{**good, **o}))  # noqa: E731
    blk = sk.DenseBlock(gpu_ctx, True, 8, 56, 4, sk.InitZeroFunc(), None, sk.Precision.FP16)
    before = gpu_ctx.launch_count()
    ip, fp = i.data_ptr(), f.data_ptr()
    for want, o in ((4, dict(dtype=3)), (4, dict(cols=0, classes=0)), (2, dict(classes=57)), (3, dict(cols=2 ** 30 + 1)), (3, dict(rows=2 ** 30 + 1)),
                    (4, dict(temperature=0.0)), (4, dict(temperature=math.nan)), (4, dict(temperature=INF)), (4, dict(grad_scale=INF)), (9, dict(logits=None)),
                    (9, dict(d_logits=None)), (4, dict(logits=x.ptr() + 1)), (4, dict(d_logits=y.data_ptr() + 1)), (4, dict(d_logits=x.ptr() + 16)),
                    (4, dict(d_logits=x.ptr() - 16))):
        assert lib.sk_label_logprob_backward(h, rows(**o), ip, fp, None) == want, o
    assert lib.sk_label_logprob(h, rows(), None, fp, None) == 9 and lib.sk_label_logprob(h, rows(), ip, None, None) == 9
    assert lib.sk_label_logprob_backward(h, rows(), ip, None, None) == 9 and lib.sk_label_logprob(h, None, ip, fp, None) == 9
    t = dict(indices=ip, values=fp, values_dtype=0, k=4, loss=fp)
    for want, o in ((4, dict(k=0)), (4, dict(k=513)), (4, dict(values_dtype=7)), (9, dict(indices=None)), (9, dict(values=None)), (9, dict(loss=None)), (4, dict(values=fp + 2))):
        assert lib.sk_distill_loss(h, rows(), C.byref(N.SkDistill(**{**t, **o}))) == want, o
    assert lib.sk_distill_loss(h, rows(), None) == 9
    assert lib.sk_distill_loss(h, rows(cols=2 ** 20 + 8, classes=2 ** 20 + 1, d_logits=None, rows=1), C.byref(N.SkDistill(**t))) == 3
    p = dict(actions=ip, logp_old=fp, advantages=fp, clip_low=0.2, clip_high=0.2, loss=fp, logp=fp, kl=fp)
    for want, o in ((4, dict(clip_low=1.5)), (4, dict(clip_low=-0.1)), (4, dict(clip_high=-0.1)), (4, dict(clip_high=math.nan)), (4, dict(kl_coeff=INF)), (9, dict(kl_coeff=0.1)),
                    (9, dict(actions=None)), (9, dict(logp_old=None)), (9, dict(advantages=None)), (9, dict(loss=None)), (9, dict(logp=None)), (9, dict(kl=None))):
        assert lib.sk_policy_loss(h, rows(), C.byref(N.SkPolicy(**{**p, **o}))) == want, o
    q = dict(labels=ip, offsets=ip, pairs=1, beta=0.1, loss=fp, margin=fp, logp=fp, row_logp=fp, scratch=fp)
    for want, o in ((4, dict(form=3)), (4, dict(beta=INF)), (4, dict(target_margin=math.nan)), (4, dict(label_smoothing=1.5)), (4, dict(form=1, label_smoothing=0.1)),
                    (3, dict(pairs=2 ** 29 + 1)), (9, dict(labels=None)), (9, dict(offsets=None)), (9, dict(loss=None)), (9, dict(margin=None)), (9, dict(logp=None)),
                    (9, dict(row_logp=None)), (9, dict(scratch=None)), (4, dict(scratch=fp + 4))):
        assert lib.sk_preference_loss(h, rows(), C.byref(N.SkPreference(**{**q, **o}))) == want, o
    d = C.byref(blk.desc())
    for want, a in ((9, (None, 4, 4, 4, 1.0)), (3, (y.data_ptr(), 5, 4, 4, 1.0)), (5, (y.data_ptr(), 4, 0, 4, 1.0)), (5, (y.data_ptr(), 4, 4, 0, 1.0)),
                    (2, (y.data_ptr(), 3, 4, 4, 1.0)), (4, (y.data_ptr(), 4, 4, 4, 0.0)), (4, (y.data_ptr(), 4, 4, 4, math.nan))):
        assert lib.sk_output_gradient(h, d, *a) == want, a
    gone = gpu_ctx.launch_count()
    assert gone == before
