"""Numbers that the losses refuse before anything reaches a GPU, at the edges of what their descriptors hold."""
import pytest

import soklyn_b200 as sk
from soklyn_b200 import log, losses
from test_losses_cpu import Never, given  # noqa: F401


def test_numbers_beyond_f32(given):  # noqa: F811
    """The descriptors hold f32: what does not fit is refused like other numbers out of range."""
    big = 1e39
    for call in (lambda: losses.label_logprob_backward(Never(), given.x, given.i, given.f, grad_scale=big),
                 lambda: losses.label_logprob_backward(Never(), given.x, given.i, given.f, grad_scale=-big),
                 lambda: losses.policy_loss(Never(), given.x, given.i, given.f, given.f, sk.PolicyLossConfig(clip_high=big)),
                 lambda: losses.policy_loss(Never(), given.x, given.i, given.f, given.f, sk.PolicyLossConfig(kl_coeff=big), logp_ref=given.f),
                 lambda: losses.policy_loss(Never(), given.x, given.i, given.f, given.f, sk.PolicyLossConfig(entropy_coeff=-big)),
                 lambda: losses.preference_loss(Never(), given.x, given.i, given.off, sk.PreferenceLossConfig(beta=big)),
                 lambda: losses.preference_loss(Never(), given.x, given.i, given.off, sk.PreferenceLossConfig(target_margin=-big))):
        with pytest.raises(log.InvalidConfiguration):
            call()
