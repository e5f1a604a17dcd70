"""Losses over rows of logits with the gradient of the logits: log-probabilities of labels, distillation from a
teacher's top logits, the clipped policy loss and the preference loss (include/soklyn_b200.h states the formulas). The
reference has none of them; its own losses compare an output block with target rows (`DenseBlock.compute_loss`).

`logits` is a 2-D `Tensor`, typically the output of a network whose last block has neither normalisation nor activation
nor dropout. Labels, class indices and offsets are int32 torch tensors on the context's device, per-row f32 vectors
torch tensors or f32 `Tensor`s, all contiguous. The returned gradient `d_logits` (a `Tensor` of the logits' type, times
`grad_scale`) goes into `FeedForwardNetwork.backward_gradient`.

Calls are ordered on the context's stream and do not wait for it. Outputs belong to that stream; inputs that another
stream wrote have to be complete before the call. An index out of range makes its row count as unlabelled and is
reported by the next `GpuContext.synchronize()` as `log.IndexOutOfRange`.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from enum import Enum
from typing import NamedTuple, Optional

import torch

from . import log
from ._native import SkDistill, SkLogits, SkPolicy, SkPreference
from .core import SK_DTYPE, Tensor

MAX_LIST = 512                # entries of a teacher's list
MAX_LIST_CLASSES = 1 << 20    # classes that distillation takes


@dataclass(frozen=True)
class DistillLossConfig:
    temperature: float = 1.0


@dataclass(frozen=True)
class PolicyLossConfig:
    clip_low: float = 0.2
    clip_high: float = 0.2
    kl_coeff: float = 0.0
    entropy_coeff: float = 0.0
    temperature: float = 1.0


class PreferenceForm(Enum):
    Sigmoid = 0
    Hinge = 1
    Squared = 2


@dataclass(frozen=True)
class PreferenceLossConfig:
    form: PreferenceForm = PreferenceForm.Sigmoid
    beta: float = 0.1
    label_smoothing: float = 0.0
    target_margin: float = 0.0
    average: bool = False
    temperature: float = 1.0


class LabelLogprob(NamedTuple):
    logp: torch.Tensor                  # [rows]
    entropy: Optional[torch.Tensor]     # [rows]


class DistillLoss(NamedTuple):
    loss: torch.Tensor                  # [rows]
    d_logits: Optional[Tensor]


class PolicyLoss(NamedTuple):
    loss: torch.Tensor                  # [rows], as are the next three
    logp: torch.Tensor
    kl: torch.Tensor
    entropy: torch.Tensor
    d_logits: Optional[Tensor]


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor                  # [pairs]
    margin: torch.Tensor                # [pairs]
    logp: torch.Tensor                  # [2 pairs]: sums or means of the sequences
    row_logp: torch.Tensor              # [rows]
    d_logits: Optional[Tensor]


class _Call:
    """Checked logits of one call, the tensors it reads, and its outputs, allocated on the context's stream."""

    def __init__(self, context, logits: Tensor, classes, temperature, grad_scale=1.0):
        if logits.data.dim() != 2:
            raise log.InvalidConfiguration(f"Logits must have two dimensions, not {logits.data.dim()}.")
        self.context, self.device = context, context.device
        self.rows, self.cols = logits.data.shape
        classes = self.cols if classes is None else classes
        if self.cols == 0 or classes < 1:
            raise log.InvalidConfiguration("Input or output size cannot be 0.")
        if classes > self.cols:
            raise log.MismatchedDimensions("classes vs logit columns", self.cols, classes)
        if not 1e-4 <= temperature <= 1e4:
            raise log.InvalidConfiguration(f"Temperature {temperature} must lie between 1e-4 and 1e4.")
        if not math.isfinite(grad_scale):
            raise log.InvalidConfiguration("The gradient scale must be finite.")
        self.logits, self.classes = logits, classes
        self.used = [self._here(logits.data, "logits")]
        self.desc = SkLogits(SK_DTYPE[logits.precision], self.rows, self.cols, classes, logits.data.data_ptr(), None,
                             temperature, grad_scale)

    def _here(self, t: torch.Tensor, name: str) -> torch.Tensor:
        if t.device != self.device:
            raise log.InvalidConfiguration(f"{name} lives on {t.device}, the context on {self.device}.")
        if not t.is_contiguous():
            raise log.InvalidConfiguration(f"{name} must be contiguous.")
        return t

    def vector(self, t, name: str, length, dtype=torch.float32):
        """Address of a vector (or matrix) that the call reads; None stays None."""
        if t is None:
            return None
        t = self._here(t.data if isinstance(t, Tensor) else t, name)
        if t.dtype != dtype:
            raise log.InvalidConfiguration(f"{name} must be {dtype}, not {t.dtype}.")
        if t.numel() != length:
            raise log.MismatchedDimensions(name, length, t.numel())
        self.used.append(t)
        return t.data_ptr()

    def new(self, *shape, dtype=torch.float32) -> torch.Tensor:
        return self.context.new_buffer(shape, dtype)

    def gradient(self, wanted: bool, out: "Tensor | None") -> "Tensor | None":
        """The Tensor the gradient goes to: a new one, or `out`, which may be the logits themselves."""
        if not wanted:
            if out is not None:
                raise log.InvalidConfiguration("A gradient tensor was given, but no gradient asked for.")
            return None
        if out is None:
            out = Tensor(self.new(self.rows, self.cols, dtype=self.logits.data.dtype), self.logits.precision, take_id=False)
        else:
            self._here(out.data, "out")
            if out.precision != self.logits.precision:
                raise log.UnsupportedTypeCast(out.precision, self.logits.precision)
            if tuple(out.data.shape) != (self.rows, self.cols):
                raise log.MismatchedDimensions("gradient elements", self.rows * self.cols, out.len())
            self.used.append(out.data)
        self.desc.d_logits = out.data.data_ptr()
        return out

    def done(self):
        self.context.uses(self.used)


def label_logprob(context, logits: Tensor, labels: torch.Tensor, *, temperature: float = 1.0, classes: "int | None" = None,
                  entropy: bool = False) -> LabelLogprob:
    """Log-probability of each row's label (0 for labels below 0) and, if asked for, the rows' entropies."""
    call = _Call(context, logits, classes, temperature)
    at = call.vector(labels, "labels", call.rows, torch.int32)
    logp, ent = call.new(call.rows), call.new(call.rows) if entropy else None
    context.gpu_label_logprob(call.desc, at, logp.data_ptr(), ent.data_ptr() if entropy else None)
    call.done()
    return LabelLogprob(logp, ent)


def label_logprob_backward(context, logits: Tensor, labels: torch.Tensor, d_logp, d_entropy=None, *, temperature: float = 1.0,
                           classes: "int | None" = None, grad_scale: float = 1.0, out: "Tensor | None" = None) -> Tensor:
    """Gradient of the logits from the gradients of label_logprob's outputs."""
    call = _Call(context, logits, classes, temperature, grad_scale)
    at = call.vector(labels, "labels", call.rows, torch.int32)
    d_logp, d_entropy = call.vector(d_logp, "d_logp", call.rows), call.vector(d_entropy, "d_entropy", call.rows)
    if d_logp is None:
        raise log.InvalidConfiguration("The gradient of the log-probabilities is missing.")
    d = call.gradient(True, out)
    context.gpu_label_logprob_backward(call.desc, at, d_logp, d_entropy)
    call.done()
    return d


_VALUES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def distill_loss(context, logits: Tensor, indices: torch.Tensor, values, config: DistillLossConfig = DistillLossConfig(), *,
                 teacher_lse=None, weights=None, classes: "int | None" = None, gradient: bool = True, grad_scale: float = 1.0,
                 out: "Tensor | None" = None) -> DistillLoss:
    """Distillation from a teacher's top logits: `indices` int32 [rows x k], `values` [rows x k] (f32 or 16 bits) its
    logits there, `teacher_lse` the log-sum-exp of all its logits / temperature where the mass outside the list counts."""
    call = _Call(context, logits, classes, config.temperature, grad_scale)
    values = values.data if isinstance(values, Tensor) else values
    if indices.dim() != 2 or tuple(values.shape) != tuple(indices.shape):
        raise log.InvalidConfiguration(f"Indices {tuple(indices.shape)} and values {tuple(values.shape)} of a teacher must both be [rows x k].")
    k = indices.shape[1]
    if not 1 <= k <= MAX_LIST:
        raise log.InvalidConfiguration(f"A teacher's list has 1 to {MAX_LIST} entries, not {k}.")
    if call.classes > MAX_LIST_CLASSES:
        raise log.AllocationLimitExceeded(call.classes, MAX_LIST_CLASSES, "classes of a distillation")
    if values.dtype not in _VALUES:
        raise log.InvalidConfiguration(f"Teacher values must be f32, f16 or bf16, not {values.dtype}.")
    t = SkDistill(call.vector(indices, "teacher indices", call.rows * k, torch.int32),
                  call.vector(values, "teacher values", call.rows * k, values.dtype), _VALUES[values.dtype], k,
                  call.vector(teacher_lse, "teacher_lse", call.rows), call.vector(weights, "weights", call.rows))
    loss, d = call.new(call.rows), call.gradient(gradient, out)
    t.loss = loss.data_ptr()
    context.gpu_distill_loss(call.desc, t)
    call.done()
    return DistillLoss(loss, d)


def policy_loss(context, logits: Tensor, actions: torch.Tensor, logp_old, advantages, config: PolicyLossConfig = PolicyLossConfig(), *,
                logp_ref=None, weights=None, classes: "int | None" = None, gradient: bool = True, grad_scale: float = 1.0,
                out: "Tensor | None" = None) -> PolicyLoss:
    """Clipped policy loss of each row's action, with a KL term to a reference policy and an entropy bonus."""
    call = _Call(context, logits, classes, config.temperature, grad_scale)
    if not (0.0 <= config.clip_low <= 1.0 and config.clip_high >= 0.0):
        raise log.InvalidConfiguration(f"Clip range {config.clip_low} below and {config.clip_high} above 1.")
    if not (math.isfinite(config.kl_coeff) and math.isfinite(config.entropy_coeff)):
        raise log.InvalidConfiguration("Policy coefficients must be finite.")
    if config.kl_coeff != 0.0 and logp_ref is None:
        raise log.InvalidConfiguration("A KL term needs the reference's log-probabilities.")
    if logp_old is None or advantages is None:
        raise log.InvalidConfiguration("Old log-probabilities or advantages are missing.")
    n = call.rows
    p = SkPolicy(call.vector(actions, "actions", n, torch.int32), call.vector(logp_old, "logp_old", n),
                 call.vector(advantages, "advantages", n), call.vector(logp_ref, "logp_ref", n), call.vector(weights, "weights", n),
                 config.clip_low, config.clip_high, config.kl_coeff, config.entropy_coeff)
    loss, logp, kl, entropy = call.new(4, n).unbind()
    p.loss, p.logp, p.kl, p.entropy = loss.data_ptr(), logp.data_ptr(), kl.data_ptr(), entropy.data_ptr()
    d = call.gradient(gradient, out)
    context.gpu_policy_loss(call.desc, p)
    call.done()
    return PolicyLoss(loss, logp, kl, entropy, d)


def preference_loss(context, logits: Tensor, labels: torch.Tensor, offsets: torch.Tensor,
                    config: PreferenceLossConfig = PreferenceLossConfig(), *, logp_ref=None, weights=None,
                    classes: "int | None" = None, gradient: bool = True, grad_scale: float = 1.0,
                    out: "Tensor | None" = None) -> PreferenceLoss:
    """Preference loss over pairs of packed sequences: rows [offsets[s], offsets[s + 1]) are sequence s, of which 2i is the
    preferred one of pair i and 2i + 1 the other; `logp_ref` [2 pairs] holds the reference's sums (or means)."""
    call = _Call(context, logits, classes, config.temperature, grad_scale)
    if not (math.isfinite(config.beta) and math.isfinite(config.target_margin)):
        raise log.InvalidConfiguration("Beta and target margin must be finite.")
    if not 0.0 <= config.label_smoothing <= 1.0:
        raise log.InvalidConfiguration(f"Label smoothing {config.label_smoothing} must lie between 0 and 1.")
    if config.label_smoothing != 0.0 and config.form != PreferenceForm.Sigmoid:
        raise log.InvalidConfiguration("Only the sigmoid form takes label smoothing.")
    if offsets.numel() % 2 != 1:
        raise log.InvalidConfiguration(f"Pairs of sequences have an odd number of offsets, not {offsets.numel()}.")
    n, pairs = call.rows, offsets.numel() // 2
    p = SkPreference(call.vector(labels, "labels", n, torch.int32), call.vector(offsets, "offsets", 2 * pairs + 1, torch.int32),
                     pairs, config.form.value, int(config.average), call.vector(logp_ref, "logp_ref", 2 * pairs),
                     call.vector(weights, "weights", pairs), config.beta, config.label_smoothing, config.target_margin)
    of_pairs, of_rows = call.new(4 * pairs), call.new(5 * n)
    loss, margin, logp = of_pairs.split((pairs, pairs, 2 * pairs))
    scratch, row_logp = of_rows.split((4 * n, n))
    p.loss, p.margin, p.logp = loss.data_ptr(), margin.data_ptr(), logp.data_ptr()
    p.row_logp, p.scratch = row_logp.data_ptr(), scratch.data_ptr()
    d = call.gradient(gradient, out)
    context.gpu_preference_loss(call.desc, p)
    call.done()
    return PreferenceLoss(loss, margin, logp, row_logp, d)
