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

import math
import struct
from dataclasses import dataclass
from enum import Enum
from typing import NamedTuple, Optional

import torch

from . import log
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


# The descriptors of include/soklyn_b200.h, packed (a third of the time that ctypes structures of so many fields take)
_LOGITS = struct.Struct("@IIIIPPff")
_DISTILL = struct.Struct("@PPIIPPP")
_POLICY = struct.Struct("@PPPPPffffPPPP")
_PREFERENCE = struct.Struct("@PPIIIPPfffPPPPP")


_MAX_F32 = torch.finfo(torch.float32).max


def _in_f32(v: float) -> bool:
    return abs(v) <= _MAX_F32               # finite in the descriptors, too


class _Call:
    """Checked logits of one call, the tensors it reads, and its outputs, allocated on the context's stream."""

    __slots__ = ("context", "device", "rows", "cols", "classes", "data", "precision", "temperature", "grad_scale", "used", "_foreign")

    def __init__(self, context, logits: Tensor, classes, temperature, grad_scale=1.0):
        data = logits.data
        if data.dim() != 2:
            raise log.InvalidConfiguration(f"Logits must have two dimensions, not {data.dim()}.")
        self.context, self.device = context, context.device
        self.rows, self.cols = rows, cols = data.shape
        if classes is None:
            classes = cols
        if cols == 0 or classes < 1:
            raise log.InvalidConfiguration("Input or output size cannot be 0.")
        if classes > cols:
            raise log.MismatchedDimensions("classes vs logit columns", cols, classes)
        if max(rows, cols) > 1 << 30:
            raise log.AllocationLimitExceeded(max(rows, cols), 1 << 30, "rows or columns of logits")
        if not 1e-4 <= temperature <= 1e4:
            raise log.InvalidConfiguration(f"Temperature {temperature} must lie between 1e-4 and 1e4.")
        if not _in_f32(grad_scale):
            raise log.InvalidConfiguration("The gradient scale must be finite.")
        self.data, self.precision, self.classes, self.temperature, self.grad_scale = data, logits.precision, classes, temperature, grad_scale
        self.used = []
        self._use(data, "logits")
        self._foreign = None

    def _use(self, t: torch.Tensor, name: str) -> int:
        if t.device != self.device:
            raise log.InvalidConfiguration(f"{name} lives on {t.device}, the context on {self.device}.")
        if not t.is_contiguous():
            raise log.InvalidConfiguration(f"{name} must be contiguous.")
        self.used.append(t)
        return t.data_ptr()

    def vector(self, t, name: str, length, dtype=torch.float32) -> int:
        """Address of a vector (or matrix) that the call reads; 0 for None."""
        if t is None:
            return 0
        if isinstance(t, Tensor):
            t = t.data
        if t.dtype is not dtype:
            raise log.InvalidConfiguration(f"{name} must be {dtype}, not {t.dtype}.")
        if t.numel() != length:
            raise log.MismatchedDimensions(name, length, t.numel())
        return self._use(t, name)

    def foreign(self) -> bool:
        if self._foreign is None:
            self._foreign = self.context.is_foreign()
        return self._foreign

    def new(self, *shape, dtype=torch.float32) -> torch.Tensor:
        return self.context.new_buffer(shape, dtype, self.foreign())

    def gradient(self, wanted: bool, out: "Tensor | None") -> "Tensor | None":
        """The Tensor the gradient goes to: a new one, or `out`, which may be the logits themselves."""
        if not wanted:
            if out is not None:
                raise log.InvalidConfiguration("A gradient tensor was given, but no gradient asked for.")
            return None
        if out is None:
            return Tensor(self.new(self.rows, self.cols, dtype=self.data.dtype), self.precision, False)
        if out.precision != self.precision:
            raise log.UnsupportedTypeCast(out.precision, self.precision)
        if tuple(out.data.shape) != (self.rows, self.cols):
            raise log.MismatchedDimensions("gradient elements", self.rows * self.cols, out.len())
        self._use(out.data, "out")
        return out

    def logits(self, d: "Tensor | None") -> bytes:
        return _LOGITS.pack(SK_DTYPE[self.precision], self.rows, self.cols, self.classes, self.data.data_ptr(),
                            0 if d is None else d.data.data_ptr(), self.temperature, self.grad_scale)

    def done(self):
        self.context.uses(self.used, self.foreign())


def label_logprob(context, logits: Tensor, labels: torch.Tensor, *, temperature: float = 1.0, classes: "int | None" = None,
                  entropy: bool = False) -> LabelLogprob:
    """Log-probability of each row's label (0 for labels below 0) and, if asked for, the rows' entropies."""
    call = _Call(context, logits, classes, temperature)
    at = call.vector(labels, "labels", call.rows, torch.int32)
    logp, ent = call.new(call.rows), call.new(call.rows) if entropy else None
    context.gpu_label_logprob(call.logits(None), at, logp.data_ptr(), ent.data_ptr() if entropy else 0)
    call.done()
    return LabelLogprob(logp, ent)


def label_logprob_backward(context, logits: Tensor, labels: torch.Tensor, d_logp, d_entropy=None, *, temperature: float = 1.0,
                           classes: "int | None" = None, grad_scale: float = 1.0, out: "Tensor | None" = None) -> Tensor:
    """Gradient of the logits from the gradients of label_logprob's outputs."""
    call = _Call(context, logits, classes, temperature, grad_scale)
    if d_logp is None:
        raise log.InvalidConfiguration("The gradient of the log-probabilities is missing.")
    at = call.vector(labels, "labels", call.rows, torch.int32)
    d_logp, d_entropy = call.vector(d_logp, "d_logp", call.rows), call.vector(d_entropy, "d_entropy", call.rows)
    d = call.gradient(True, out)
    context.gpu_label_logprob_backward(call.logits(d), at, d_logp, d_entropy)
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
    if indices.dim() != 2 or values.shape != indices.shape:
        raise log.InvalidConfiguration(f"Indices {tuple(indices.shape)} and values {tuple(values.shape)} of a teacher must both be [rows x k].")
    k = indices.shape[1]
    if not 1 <= k <= MAX_LIST:
        raise log.InvalidConfiguration(f"A teacher's list has 1 to {MAX_LIST} entries, not {k}.")
    if call.classes > MAX_LIST_CLASSES:
        raise log.AllocationLimitExceeded(call.classes, MAX_LIST_CLASSES, "classes of a distillation")
    if values.dtype not in _VALUES:
        raise log.InvalidConfiguration(f"Teacher values must be f32, f16 or bf16, not {values.dtype}.")
    n = call.rows
    read = (call.vector(indices, "teacher indices", n * k, torch.int32), call.vector(values, "teacher values", n * k, values.dtype),
            _VALUES[values.dtype], k, call.vector(teacher_lse, "teacher_lse", n), call.vector(weights, "weights", n))
    loss, d = call.new(n), call.gradient(gradient, out)
    context.gpu_distill_loss(call.logits(d), _DISTILL.pack(*read, loss.data_ptr()))
    call.done()
    return DistillLoss(loss, d)


def policy_loss(context, logits: Tensor, actions: torch.Tensor, logp_old, advantages, config: PolicyLossConfig = PolicyLossConfig(), *,
                logp_ref=None, weights=None, classes: "int | None" = None, gradient: bool = True, grad_scale: float = 1.0,
                out: "Tensor | None" = None) -> PolicyLoss:
    """Clipped policy loss of each row's action, with a KL term to a reference policy and an entropy bonus."""
    call = _Call(context, logits, classes, config.temperature, grad_scale)
    low, high, beta, eta = config.clip_low, config.clip_high, config.kl_coeff, config.entropy_coeff
    if not (0.0 <= low <= 1.0 and (0.0 <= high <= _MAX_F32 or high == math.inf)):
        raise log.InvalidConfiguration(f"Clip range {low} below and {high} above 1.")
    if not (_in_f32(beta) and _in_f32(eta)):
        raise log.InvalidConfiguration("Policy coefficients must be finite.")
    if beta != 0.0 and logp_ref is None:
        raise log.InvalidConfiguration("A KL term needs the reference's log-probabilities.")
    if logp_old is None or advantages is None:
        raise log.InvalidConfiguration("Old log-probabilities or advantages are missing.")
    n = call.rows
    read = (call.vector(actions, "actions", n, torch.int32), call.vector(logp_old, "logp_old", n), call.vector(advantages, "advantages", n),
            call.vector(logp_ref, "logp_ref", n), call.vector(weights, "weights", n))
    of_rows = call.new(4, n)
    d = call.gradient(gradient, out)
    at = of_rows.data_ptr()
    context.gpu_policy_loss(call.logits(d), _POLICY.pack(*read, low, high, beta, eta, at, at + 4 * n, at + 8 * n, at + 12 * n))
    call.done()
    return PolicyLoss(*of_rows.unbind(), d)


def preference_loss(context, logits: Tensor, labels: torch.Tensor, offsets: torch.Tensor,
                    config: PreferenceLossConfig = PreferenceLossConfig(), *, logp_ref=None, weights=None,
                    classes: "int | None" = None, gradient: bool = True, grad_scale: float = 1.0,
                    out: "Tensor | None" = None) -> PreferenceLoss:
    """Preference loss over pairs of packed sequences: rows [offsets[s], offsets[s + 1]) are sequence s, of which 2i is the
    preferred one of pair i and 2i + 1 the other; `logp_ref` [2 pairs] holds the reference's sums (or means)."""
    call = _Call(context, logits, classes, config.temperature, grad_scale)
    if not (_in_f32(config.beta) and _in_f32(config.target_margin)):
        raise log.InvalidConfiguration("Beta and target margin must be finite.")
    if not 0.0 <= config.label_smoothing <= 1.0:
        raise log.InvalidConfiguration(f"Label smoothing {config.label_smoothing} must lie between 0 and 1.")
    if config.label_smoothing != 0.0 and config.form is not PreferenceForm.Sigmoid:
        raise log.InvalidConfiguration("Only the sigmoid form takes label smoothing.")
    if offsets.numel() % 2 != 1:
        raise log.InvalidConfiguration(f"Pairs of sequences have an odd number of offsets, not {offsets.numel()}.")
    n, pairs = call.rows, offsets.numel() // 2
    read = (call.vector(labels, "labels", n, torch.int32), call.vector(offsets, "offsets", 2 * pairs + 1, torch.int32), pairs,
            config.form.value, bool(config.average), call.vector(logp_ref, "logp_ref", 2 * pairs), call.vector(weights, "weights", pairs),
            config.beta, config.label_smoothing, config.target_margin)
    own = call.new(5 * n + 4 * pairs)       # scratch [4 n], row_logp [n], loss, margin [pairs], logp [2 pairs]
    d = call.gradient(gradient, out)
    at = own.data_ptr()
    of_pairs = at + 20 * n
    context.gpu_preference_loss(call.logits(d), _PREFERENCE.pack(*read, of_pairs, of_pairs + 4 * pairs, of_pairs + 8 * pairs, at + 16 * n, at))
    call.done()
    _, row_logp, loss, margin, logp = own.split_with_sizes((4 * n, n, pairs, pairs, 2 * pairs))
    return PreferenceLoss(loss, margin, logp, row_logp, d)
