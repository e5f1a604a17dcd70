"""Losses over rows of logits at the edges of their ranges: terms that are switched off beside infinities, NaN, classes far
below the listed ones, the most classes, offsets that fall, and what the context reports and leaves behind.

Tolerances as in test_losses_gpu.py: half a step of the result's type, and the f32 terms of a row's sum (`Ref.sum_rel`)
and of an exponential (`Ref.rel`).
"""
import ctypes as C
import math

import pytest
import torch

import soklyn_b200 as sk
from soklyn_b200 import log, losses
from test_losses_gpu import DT, INF, Ref, _close, _logits, _rng, _teacher, distill_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,classes", [(1, 1 << 20), (60, 1 << 20), (200, 1 << 20), (80, 1 << 20), (200, 323001), (200, 330001), (40, 700001)])
def test_distillation_without_a_gradient_takes_every_width(gpu_ctx, rows, classes):
    """The bits of a row's classes fit the shared memory of the blocks that work on it, however many rows there are."""
    x, g = _logits(rows, classes, 0, "bf16", seed=9)
    idx, values = _teacher(rows, classes, 40, g)
    lse = torch.logsumexp(values.double(), 1).float() + 0.2
    got = losses.distill_loss(gpu_ctx, x, idx, values, teacher_lse=lse, gradient=False)
    gpu_ctx.synchronize()
    assert got.d_logits is None
    for a in range(0, rows, 20):
        s = slice(a, a + 20)
        each, tol, *_ = distill_reference(x.data[s], classes, 1.0, idx[s], values[s], lse[s], None, 1.0)
        _close(got.loss[s], each, tol, "loss")


def _tail_reference(x, classes, tau, idx, values, lse, scale):
    """Loss and gradient of a distillation with its tail, in 64 bits and in logarithms: classes however far below the listed
    ones count. Tolerances: the list's and the tail's masses are 64 bits and add a rounding to f32; the rest is the two sums."""
    at = idx.long()
    logq = values.double() / tau - lse.double()[:, None]
    q = logq.exp()
    rest = 1.0 - q.sum(1)
    assert (rest > 1e-6).all()
    inside = torch.zeros(x.shape[0], classes, dtype=torch.bool, device=x.device).scatter_(1, at, True)
    z = x[:, :classes].double() / tau
    others = torch.where(inside, -INF, x[:, :classes])
    r, o = Ref(x, classes, tau), Ref(others, classes, tau)
    log_out = o.lse + (others.double() / tau).amax(1) - r.lse - z.amax(1)
    loss = (q * (logq - r.lp.gather(1, at))).sum(1) + rest * (rest.log() - log_out)
    tol = q.sum(1) * r.sum_rel + rest * (r.sum_rel + o.sum_rel) + 2.0 ** -23 * loss.abs()
    target = torch.zeros_like(r.p).scatter_add_(1, at, q)
    total, back, f = (q.sum(1) + rest)[:, None], rest[:, None] * o.p, tau * scale
    want = f * (total * r.p - back - target)
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}[x.dtype]
    d_tol = (torch.finfo(x.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + tiny
             + f * ((r.rel + torch.where(inside, 0.0, o.rel)) * total * r.p + o.rel * back + 2.0 ** -22 * target + 1e-36))
    return loss * tau * tau, tol * tau * tau, want, d_tol


def check_tail(ctx, x, classes, tau, idx, values, lse, scale, **kw):
    loss, tol, want, d_tol = _tail_reference(x.data, classes, tau, idx, values, lse, scale)
    got = losses.distill_loss(ctx, x, idx, values, sk.DistillLossConfig(tau), teacher_lse=lse, classes=classes, grad_scale=scale, **kw)
    ctx.synchronize()
    _close(got.loss, loss, tol, "loss")
    _close(got.d_logits.data[:, :classes], want, d_tol, "gradient")
    alone = losses.distill_loss(ctx, x, idx, values, sk.DistillLossConfig(tau), teacher_lse=lse, classes=classes, gradient=False)
    _close(alone.loss, loss, tol, "loss without a gradient")


def _with_tail(values, tau, tail):
    return (torch.logsumexp(values.double() / tau, 1) - math.log1p(-tail)).float()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("classes,k", [(13, 12), (1000, 64), (40009, 300), (131072, 512)])
def test_a_small_tail_keeps_its_places(gpu_ctx, classes, k, kind):
    """1 minus the sum of the list's masses: with those in f32 a tail of 1e-5 would be off by a hundredth, and with it the
    gradient of every class outside the list."""
    for tail in (0.2, 1e-3, 1e-5):
        x, g = _logits(40, classes, 3, kind, 1, scale=1.0)
        idx, values = _teacher(40, classes, k, g)
        lse = _with_tail(values, 1.0, tail)
        check_tail(gpu_ctx, x, classes, 1.0, idx, values, lse, 1.0)


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes,pad,offset", [(10, 3, 1), (1000, 0, 0), (5003, 0, 2), (70001, 7, 1)])
def test_a_tail_far_below_the_listed_classes(gpu_ctx, classes, pad, offset, kind):
    """The student's mass outside the list from e^-40 to far below what f32 holds: the loss grows with its logarithm and the
    gradient still moves the tail's whole mass to the classes outside."""
    for tau in (1.0, 0.25, 2.0 ** -6):
        for gap, tail in ((40.0, 0.2), (86.0, 0.2), (87.5, 1e-3), (88.5, 0.2), (104.0, 1e-3), (200.0, 0.2), (4000.0, 0.2)):
            x, g = _logits(5, classes, pad, kind, offset, scale=3.0 * tau)
            idx, values = _teacher(5, classes, 4, g, spread=tau)
            x.data.scatter_add_(1, idx.long(), torch.full((5, 4), gap * tau, device="cuda").to(x.data.dtype))
            check_tail(gpu_ctx, x, classes, tau, idx, values, _with_tail(values, tau, tail), 32.0)


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes", [12, 5003, 70001])
def test_a_listed_nan_beside_masked_classes_is_not_an_empty_row(gpu_ctx, classes, kind):
    x, g = _logits(4, classes, 1, kind, 1)
    idx, values = _teacher(4, classes, 4, g)
    x.data[:2, :classes] = -INF
    x.data[0, idx[0, 2].long()] = math.nan
    kept = x.data[3, idx[3].long()].clone()
    x.data[3, :classes] = -INF
    outside = min(set(range(5)) - set(idx[3].tolist()))
    x.data[3, idx[3].long()], x.data[3, outside] = kept, math.nan      # a class outside is NaN, the others there are masked
    for lse in (None, _with_tail(values, 1.0, 0.2)):
        got = losses.distill_loss(gpu_ctx, x, idx, values, teacher_lse=lse, classes=classes)
        assert got.loss[0].isnan() and got.d_logits.data[0, :classes].isnan().all()
        assert float(got.loss[1]) == 0.0 and (got.d_logits.data[1] == 0).all()       # no class at all: does not count
        assert got.loss[2].isfinite() and got.d_logits.data[2].isfinite().all()
        assert got.loss[3].isnan() and got.d_logits.data[3, :classes].isnan().all()


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes", [10, 5000])
@pytest.mark.parametrize("eta", [0.0, 0.02])
def test_a_kl_that_is_only_watched_changes_nothing(gpu_ctx, eta, classes, kind):
    """kl_coeff = 0 with a reference given: the KL is reported, infinite or not, and is no term of the loss."""
    x, g = _logits(4, classes, 0, kind)
    actions = torch.randint(0, classes, (4,), generator=g, device="cuda").int()
    x.data[0, actions[0].long()] = -INF                    # a masked action
    r = Ref(x.data, classes, 1.0)
    lp = r.pick(actions)
    ref = lp.nan_to_num(neginf=-3.0) + torch.tensor([0.0, 200.0, -200.0, 0.5], device="cuda")
    ref, old, adv = ref.float(), lp.nan_to_num(neginf=-5.0).float(), torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")
    cfg = sk.PolicyLossConfig(entropy_coeff=eta)
    want = losses.policy_loss(gpu_ctx, x, actions, old, adv, cfg)
    got = losses.policy_loss(gpu_ctx, x, actions, old, adv, cfg, logp_ref=ref)
    for name in ("loss", "logp", "entropy"):
        assert torch.equal(getattr(got, name), getattr(want, name)), name
    assert torch.equal(got.d_logits.data, want.d_logits.data)
    assert got.loss.isfinite().all() and got.d_logits.data.isfinite().all()
    d = ref.double() - lp
    assert float(got.kl[0]) == INF and float(got.kl[1]) == INF       # exp(200) is beyond f32
    tol = torch.expm1(d).abs() * r.sum_rel + r.sum_rel + 2.0 ** -22 * d.abs()
    _close(got.kl[2:], (torch.expm1(d) - d)[2:], tol[2:], "kl")


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes", [10, 5000])
def test_an_advantage_of_zero_pulls_nowhere(gpu_ctx, classes, kind):
    """However unlikely the action was: a ratio beyond f32 times no advantage is no loss."""
    x, g = _logits(3, classes, 0, kind)
    actions = torch.randint(0, classes, (3,), generator=g, device="cuda").int()
    old, adv = torch.full((3,), -200.0, device="cuda"), torch.tensor([0.0, -0.0, 0.0], device="cuda")
    got = losses.policy_loss(gpu_ctx, x, actions, old, adv)
    assert (got.loss == 0).all() and (got.d_logits.data == 0).all()
    got = losses.policy_loss(gpu_ctx, x, actions, old, adv, sk.PolicyLossConfig(entropy_coeff=0.5))
    near = losses.policy_loss(gpu_ctx, x, actions, got.logp, adv, sk.PolicyLossConfig(entropy_coeff=0.5))
    assert torch.equal(got.loss, near.loss) and torch.equal(got.d_logits.data, near.d_logits.data) and got.d_logits.data.isfinite().all()


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("classes", [10, 5000])
def test_nan_reaches_the_policy_loss(gpu_ctx, classes, kind):
    """NaN or +inf among a row's logits, or NaN in its inputs, makes NaN of its loss and gradient on either side of the clip."""
    x, g = _logits(7, classes, 0, kind)
    actions = torch.zeros(7, dtype=torch.int32, device="cuda")
    adv = torch.tensor([1.0, -1.0, 0.0, 1.0, -1.0, math.nan, 1.0], device="cuda")
    old = torch.full((7,), -3.0, device="cuda")
    x.data[0:3, 4] = math.nan
    x.data[3, 5] = INF
    old[4] = math.nan
    for eta in (0.0, 0.1):
        got = losses.policy_loss(gpu_ctx, x, actions, old, adv, sk.PolicyLossConfig(entropy_coeff=eta))
        assert got.loss[:6].isnan().all() and got.logp[:4].isnan().all() and got.d_logits.data[:6].isnan().all()
        assert got.loss[6].isfinite() and got.d_logits.data[6].isfinite().all()


@pytest.mark.parametrize("form", sk.PreferenceForm)
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_nan_reaches_the_preference_loss(gpu_ctx, kind, form):
    """A pair with a NaN in one of its rows has no margin, in any form of the loss; the other pair keeps its results."""
    x, g = _logits(12, 700, 0, kind)
    labels = torch.randint(0, 700, (12,), generator=g, device="cuda").int()
    labels[1] = -1
    offsets = torch.tensor([0, 3, 6, 9, 12], dtype=torch.int32, device="cuda")
    cfg = sk.PreferenceLossConfig(form)
    want = losses.preference_loss(gpu_ctx, x, labels, offsets, cfg)
    clean = [t.clone() for t in (want.loss[1], want.margin[1], want.d_logits.data[6:])]
    x.data[4, 9] = math.nan
    got = losses.preference_loss(gpu_ctx, x, labels, offsets, cfg)
    assert got.margin[0].isnan() and got.loss[0].isnan() and got.row_logp[4].isnan()
    counted = [r for r in range(6) if r != 1]
    assert got.d_logits.data[counted].isnan().all() and (got.d_logits.data[1] == 0).all()
    assert all(torch.equal(a, b) for a, b in zip((got.loss[1], got.margin[1], got.d_logits.data[6:]), clean))


def test_an_index_out_of_range_is_reported_beside_a_timeout(gpu_ctx):
    """A wait that ran out and a label out of range since the last synchronize: one report each."""
    x, _ = _logits(2, 50, 0, "f32")
    flags = torch.zeros(4, dtype=torch.int32, device=gpu_ctx.device)
    losses.label_logprob(gpu_ctx, x, torch.tensor([3, 50], dtype=torch.int32, device="cuda"))
    gpu_ctx.wait_flags(flags.data_ptr(), 2, 1)              # nobody sets them: gives up after about two seconds
    with pytest.raises(log.NativeError, match="status 11"):
        gpu_ctx.synchronize()
    with pytest.raises(log.IndexOutOfRange, match="a label"):
        gpu_ctx.synchronize()
    gpu_ctx.synchronize()


def test_the_threads_capture_mode_is_put_back(gpu_ctx):
    """Outputs that are allocated while a step is recorded change the thread's capture mode for the allocation alone."""
    exchange = C.CDLL("libcuda.so.1").cuThreadExchangeStreamCaptureMode

    def swap(mode):
        m = C.c_int(mode)
        assert exchange(C.byref(m)) == 0
        return m.value

    x, _ = _logits(3, 50, 0, "f32")
    labels = torch.zeros(3, dtype=torch.int32, device="cuda")
    before = swap(1)                                        # thread-local
    try:
        for _ in range(3):                                  # the slot's first step may run unrecorded
            with gpu_ctx.step_graph(6):
                losses.label_logprob(gpu_ctx, x, labels)
                inside = swap(1)
            gpu_ctx.synchronize()
            assert inside == 1
        assert swap(1) == 1
    finally:
        swap(before)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_offsets_that_fall_give_shared_rows_both_gradients(gpu_ctx, kind):
    """Offsets that fall leave an empty sequence, and the next one may begin inside the one before it: a row of two pairs
    gets the gradient of both losses, in every run."""
    rows, classes = 600, 40
    x, g = _logits(rows, classes, 0, kind)
    labels = torch.randint(0, classes, (rows,), generator=g, device="cuda").int()
    cuts = [0, 400, 200, 500, 600]                          # pair 0: [0, 400) and none; pair 1: [200, 500) and [500, 600)
    ref = torch.tensor([-900.0, 0.0, -700.0, -250.0], device="cuda")
    beta = 2.0 ** -7
    r = Ref(x.data, classes, 1.0)
    lp = r.pick(labels)
    pull = torch.zeros(rows, dtype=torch.float64, device="cuda")
    off = torch.zeros(rows, dtype=torch.float64, device="cuda")
    for chosen, rejected, i in ((slice(0, 400), slice(0, 0), 0), (slice(200, 500), slice(500, 600), 2)):
        m = beta * (lp[chosen].sum() - ref[i].double() - lp[rejected].sum() + ref[i + 1].double())
        slope, m_tol = -torch.sigmoid(-m) * beta, beta * (r.sum_rel[chosen].sum() + r.sum_rel[rejected].sum())
        pull[chosen] += slope
        pull[rejected] -= slope
        off[chosen] += 0.25 * beta * m_tol
        off[rejected] += 0.25 * beta * m_tol
    hit = torch.zeros_like(r.p).scatter_(1, labels.long()[:, None], 1.0)
    want, size = pull[:, None] * (hit - r.p), pull.abs()[:, None] * (hit + r.p)
    tiny = 2.0 ** -25 if kind == "f16" else 0.0
    tol = torch.finfo(x.data.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + (r.rel + 2.0 ** -22) * size + off[:, None] * (hit + r.p) + tiny
    for _ in range(4):
        got = losses.preference_loss(gpu_ctx, x, labels, torch.tensor(cuts, dtype=torch.int32, device="cuda"), sk.PreferenceLossConfig(beta=beta), logp_ref=ref)
        with pytest.raises(log.IndexOutOfRange, match="offset"):
            gpu_ctx.synchronize()
        _close(got.d_logits.data, want, tol, "gradient")
