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
