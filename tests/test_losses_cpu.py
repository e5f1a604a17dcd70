"""What the losses refuse before anything reaches a GPU."""
import math
from types import SimpleNamespace

import pytest
import torch

import soklyn_b200 as sk
from soklyn_b200 import _native, log, losses


class Never:
    """A context none of whose calls may be reached."""
    device = torch.device("cpu")
    step_keeps = None

    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


def _tensor(t, prec):
    x = sk.Tensor.__new__(sk.Tensor)
    x.data, x.precision, x.id = t, prec, -1
    return x


@pytest.fixture
def given():
    x = _tensor(torch.zeros(4, 16), sk.Precision.FP32)
    return SimpleNamespace(x=x, i=torch.zeros(4, dtype=torch.int32), f=torch.zeros(4), idx=torch.zeros(4, 3, dtype=torch.int32), val=torch.zeros(4, 3),
                           off=torch.zeros(3, dtype=torch.int32))


def test_logits(given):
    for x, err in ((_tensor(torch.zeros(4), sk.Precision.FP32), log.InvalidConfiguration), (_tensor(torch.zeros(4, 0), sk.Precision.FP32), log.InvalidConfiguration),
                   (_tensor(torch.zeros(16, 4).T, sk.Precision.FP32), log.InvalidConfiguration), (_tensor(torch.zeros(4, 16, device="meta"), sk.Precision.FP32), log.InvalidConfiguration)):
        with pytest.raises(err):
            losses.label_logprob(Never(), x, given.i)
    for kw, err in ((dict(classes=17), log.MismatchedDimensions), (dict(classes=0), log.InvalidConfiguration), (dict(temperature=0.0), log.InvalidConfiguration),
                    (dict(temperature=math.nan), log.InvalidConfiguration), (dict(temperature=-1.0), log.InvalidConfiguration)):
        with pytest.raises(err):
            losses.label_logprob(Never(), given.x, given.i, **kw)


def test_vectors(given):
    for labels, err in ((given.i[:3], log.MismatchedDimensions), (given.i.long(), log.InvalidConfiguration), (torch.zeros(8, dtype=torch.int32)[::2], log.InvalidConfiguration)):
        with pytest.raises(err):
            losses.label_logprob(Never(), given.x, labels)
    with pytest.raises(log.InvalidConfiguration):
        losses.label_logprob_backward(Never(), given.x, given.i, None)
    with pytest.raises(log.MismatchedDimensions):
        losses.label_logprob_backward(Never(), given.x, given.i, given.f, given.f[:2])
    with pytest.raises(log.InvalidConfiguration):
        losses.label_logprob_backward(Never(), given.x, given.i, given.f.double())
    with pytest.raises(log.InvalidConfiguration):
        losses.label_logprob_backward(Never(), given.x, given.i, given.f, grad_scale=math.inf)


def test_gradient_tensors(given):
    for out, err in ((_tensor(torch.zeros(4, 15), sk.Precision.FP32), log.MismatchedDimensions), (_tensor(torch.zeros(4, 16).half(), sk.Precision.FP16), log.UnsupportedTypeCast),
                     (_tensor(torch.zeros(16, 4).T, sk.Precision.FP32), log.InvalidConfiguration)):
        with pytest.raises(err):
            losses.label_logprob_backward(Never(), given.x, given.i, given.f, out=out)


def test_distillation(given):
    for idx, val, err in ((given.idx[0], given.val[0], log.InvalidConfiguration), (given.idx, given.val[:, :2], log.InvalidConfiguration),
                          (torch.zeros(4, 0, dtype=torch.int32), torch.zeros(4, 0), log.InvalidConfiguration),
                          (torch.zeros(4, 513, dtype=torch.int32), torch.zeros(4, 513), log.InvalidConfiguration),
                          (given.idx.long(), given.val, log.InvalidConfiguration), (given.idx, given.val.double(), log.InvalidConfiguration),
                          (torch.zeros(3, 3, dtype=torch.int32), torch.zeros(3, 3), log.MismatchedDimensions)):
        with pytest.raises(err):
            losses.distill_loss(Never(), given.x, idx, val)
    with pytest.raises(log.MismatchedDimensions):
        losses.distill_loss(Never(), given.x, given.idx, given.val, teacher_lse=given.f[:1])
    wide = _tensor(torch.zeros(1, losses.MAX_LIST_CLASSES + 1, dtype=torch.bfloat16), sk.Precision.BF16)
    with pytest.raises(log.AllocationLimitExceeded):
        losses.distill_loss(Never(), wide, given.idx[:1], given.val[:1])


def test_policy(given):
    for cfg in (sk.PolicyLossConfig(clip_low=-0.1), sk.PolicyLossConfig(clip_low=1.1), sk.PolicyLossConfig(clip_high=-0.1), sk.PolicyLossConfig(kl_coeff=0.1),
                sk.PolicyLossConfig(kl_coeff=math.nan), sk.PolicyLossConfig(entropy_coeff=math.inf), sk.PolicyLossConfig(temperature=0.0)):
        with pytest.raises(log.InvalidConfiguration):
            losses.policy_loss(Never(), given.x, given.i, given.f, given.f, cfg)
    with pytest.raises(log.InvalidConfiguration):
        losses.policy_loss(Never(), given.x, given.i, given.f, None)


def test_preference(given):
    for cfg in (sk.PreferenceLossConfig(beta=math.inf), sk.PreferenceLossConfig(label_smoothing=-0.1), sk.PreferenceLossConfig(label_smoothing=1.1),
                sk.PreferenceLossConfig(sk.PreferenceForm.Hinge, label_smoothing=0.1), sk.PreferenceLossConfig(target_margin=math.nan)):
        with pytest.raises(log.InvalidConfiguration):
            losses.preference_loss(Never(), given.x, given.i, given.off, cfg)
    with pytest.raises(log.InvalidConfiguration):
        losses.preference_loss(Never(), given.x, given.i, given.off[:2])
    with pytest.raises(log.MismatchedDimensions):
        losses.preference_loss(Never(), given.x, given.i, given.off, logp_ref=given.f[:1])
    with pytest.raises(log.MismatchedDimensions):
        losses.preference_loss(Never(), given.x, given.i, given.off, weights=given.f)


def test_null_contexts_and_statuses():
    lib = _native.lib()
    assert lib.sk_label_logprob(None, None, None, None, None) == 9 and lib.sk_label_logprob_backward(None, None, None, None, None) == 9
    assert lib.sk_distill_loss(None, None, None) == 9 and lib.sk_policy_loss(None, None, None) == 9 and lib.sk_preference_loss(None, None, None) == 9
    assert lib.sk_output_gradient(None, None, None, 0, 0, 0, 1.0) == 9
    assert lib.sk_ffn_backward_gradient(None, None, 0, None, 0, 1.0, None, 0, None, None, 0, 0.1, 1.0, 1) == 9
    assert lib.sk_status_string(13) == b"Index out of range"
    with pytest.raises(log.IndexOutOfRange):
        log.raise_status(13, "a label")


def test_descriptor_layouts_match_the_header():
    import ctypes as C
    assert C.sizeof(_native.SkLogits) == 40 and C.sizeof(_native.SkDistill) == 48
    assert C.sizeof(_native.SkPolicy) == 88 and C.sizeof(_native.SkPreference) == 104
    # the packed forms, up to the padding behind the last field
    assert losses._LOGITS.size == 40 and losses._DISTILL.size == 48 and losses._POLICY.size == 88 and losses._PREFERENCE.size == 104
