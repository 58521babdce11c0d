"""Preference losses on interleaved (chosen, rejected) batches.

Parity: reference ``src/twinkle/loss/dpo.py:20-569`` — DPO with sigmoid /
hinge / ipo / kto_pair forms, label smoothing, ``sft_weight``,
``reference_free``; SimPO, CPO, ORPO.  Rows ``0::2`` are chosen and ``1::2``
rejected, so a contiguous data-parallel slice of even length keeps pairs whole.
On a GPU fp32 log-probs go through ``ops.preference_loss``; classes derived from
these, methods that were replaced on a class or an object, and functional transforms
keep to the PyTorch forms.
"""
from __future__ import annotations

from typing import Any, Dict, Optional

import torch
import torch.nn.functional as F

from .. import ops
from ..data_format import LossOutput
from .base import Loss, as_2d_labels, replaced, token_logps


class PreferenceLoss(Loss):

    def __init__(self, ignore_index: int = -100):
        self.ignore_index = ignore_index

    def _seq_logps(self, inputs, outputs):
        labels = as_2d_labels(inputs)
        logps = token_logps(outputs, labels, self.ignore_index)
        mask = (labels != self.ignore_index).to(logps.device)
        if logps.shape[0] % 2 != 0:
            raise AssertionError('preference batches interleave chosen/rejected rows; got an odd number of rows')
        seq = (logps * mask).sum(-1)
        return logps, mask, seq

    def _rows(self, inputs, outputs):
        """Mask (the labels may be written again before the backward pass) and log-probs where the kernel takes them, else None."""
        labels = as_2d_labels(inputs)
        logps = outputs.get('logps')
        if logps is not None and logps.dim() == 1:
            logps = logps.unsqueeze(0)
        if (type(self) not in _ON_KERNEL or replaced(self, _METHODS, _DEFINED) or ops.transformed() or logps is None or not logps.is_cuda or logps.dtype != torch.float32 or logps.shape != labels.shape or logps.numel() == 0
                or logps.shape[0] % 2):
            return None
        return (labels != self.ignore_index).to(logps.device), logps

    @staticmethod
    def _nll(chosen_seq_logps: torch.Tensor, mask: torch.Tensor) -> torch.Tensor:
        """Negative log-likelihood of the chosen rows per chosen *token* over the whole batch (total divided by the
        number of chosen tokens, reference ``loss/dpo.py:64-71``), not a mean of per-sequence means."""
        return -chosen_seq_logps.sum() / mask[0::2].sum().clamp_min(1)

    @staticmethod
    def _align_ref(ref, logps, mask):
        """Reference logps may be per-token ``[B, S']`` (S' ≥ or ≤ S), or
        already per-sequence ``[B]``."""
        if ref is None:
            return None
        if isinstance(ref, dict):
            ref = ref.get('logps')
        ref = torch.as_tensor(ref) if not torch.is_tensor(ref) else ref
        ref = ref.to(logps.device, logps.dtype)
        if ref.dim() == 1:
            return ref
        S = mask.shape[1]
        if ref.shape[1] < S:
            ref = F.pad(ref, (0, S - ref.shape[1]))
        return (ref[:, :S] * mask).sum(-1)


class DPOLoss(PreferenceLoss):

    def __init__(self, beta: float = 0.1, label_smoothing: float = 0.0, ignore_index: int = -100,
                 loss_type: str = 'sigmoid', reference_free: bool = False, sft_weight: float = 0.0, **kwargs):
        super().__init__(ignore_index)
        if loss_type not in ('sigmoid', 'hinge', 'ipo', 'kto_pair'):
            raise ValueError(f'Unknown loss_type: {loss_type}')
        if label_smoothing > 0 and loss_type != 'sigmoid':
            raise ValueError('label_smoothing is only defined for loss_type="sigmoid"')
        self.beta, self.label_smoothing, self.loss_type = beta, label_smoothing, loss_type
        self.reference_free, self.sft_weight = reference_free, sft_weight

    def __call__(self, inputs: Dict[str, Any], outputs: Dict[str, Any], *, ref_outputs=None, ref_logps=None,
                 ref_chosen_logps=None, ref_rejected_logps=None, **kwargs) -> LossOutput:
        """The reference policy comes as ``ref_outputs`` / ``ref_logps`` (per token or per sequence, rows interleaved
        like the batch) or as the two sequence-level vectors ``ref_chosen_logps`` / ``ref_rejected_logps``
        (reference ``src/twinkle/loss/dpo.py:257-320``)."""
        rows = self._rows(inputs, outputs)
        given = ref_outputs if ref_outputs is not None else ref_logps
        if rows is not None and ((ref_chosen_logps is not None and ref_rejected_logps is not None) or self._row_by_row(given, rows[1])):
            return self._kernel_loss(*rows, given, ref_chosen_logps, ref_rejected_logps)
        logps, mask, seq = self._seq_logps(inputs, outputs)
        pc, pr = seq[0::2], seq[1::2]
        ref = None
        if ref_chosen_logps is not None and ref_rejected_logps is not None:
            rc = torch.as_tensor(ref_chosen_logps).to(pc.device, pc.dtype).reshape(-1)
            rr = torch.as_tensor(ref_rejected_logps).to(pc.device, pc.dtype).reshape(-1)
            if rc.numel() != pc.numel() or rr.numel() != pr.numel():
                raise ValueError(f'ref_chosen_logps / ref_rejected_logps must hold one value per pair ({pc.numel()}), got {rc.numel()} / {rr.numel()}')
        else:
            ref = self._align_ref(given, logps, mask)
            if ref is None and not self.reference_free:
                return LossOutput(loss=logps.sum() * 0.0, num_tokens=0)
            if ref is None:
                rc = rr = torch.zeros_like(pc)
            else:
                rc, rr = ref[0::2], ref[1::2]
        dc, dr = pc - rc, pr - rr
        z = self.beta * (dc - dr)
        if self.loss_type == 'sigmoid':
            ls = self.label_smoothing
            per_pair = -F.logsigmoid(z) * (1 - ls) - F.logsigmoid(-z) * ls
        elif self.loss_type == 'hinge':
            per_pair = torch.relu(1 - z)
        elif self.loss_type == 'ipo':
            per_pair = (z - 1 / (2 * self.beta))**2  # on the β-scaled margin, as the reference (dpo.py:234-237)
        else:  # kto_pair
            per_pair = 1 - torch.sigmoid(self.beta * dc) + torch.sigmoid(self.beta * dr)
        loss = per_pair.mean()
        if self.sft_weight > 0:
            loss = loss + self.sft_weight * self._nll(pc, mask)
        self.last_stats = {
            'rewards/chosen': float((self.beta * dc).mean().detach()), 'rewards/rejected': float((self.beta * dr).mean().detach()),
            'rewards/margins': float((self.beta * (dc - dr)).mean().detach()), 'rewards/accuracies': float((dc > dr).float().mean()),
            'logps/chosen': float(pc.mean().detach()), 'logps/rejected': float(pr.mean().detach()),
        }
        return LossOutput(loss=loss, num_tokens=0)

    @staticmethod
    def _row_by_row(ref, logps) -> bool:
        """Whether the reference has an entry per row (one that stands for several rows, or for all pairs, is spread by the PyTorch form)."""
        if isinstance(ref, dict):
            ref = ref.get('logps')
        return ref is None or (torch.as_tensor(ref).dim() in (1, 2) and torch.as_tensor(ref).shape[0] == logps.shape[0])

    def _kernel_loss(self, mask, logps, ref, ref_chosen, ref_rejected) -> LossOutput:
        if ref_chosen is not None and ref_rejected is not None:
            rc, rr = (torch.as_tensor(r).to(logps.device, logps.dtype).reshape(-1) for r in (ref_chosen, ref_rejected))
            pairs = logps.shape[0] // 2
            if rc.numel() != pairs or rr.numel() != pairs:
                raise ValueError(f'ref_chosen_logps / ref_rejected_logps must hold one value per pair ({pairs}), got {rc.numel()} / {rr.numel()}')
            ref = torch.stack([rc, rr], -1).reshape(-1)
        else:
            if isinstance(ref, dict):
                ref = ref.get('logps')
            if ref is not None:
                ref = (ref if torch.is_tensor(ref) else torch.as_tensor(ref)).to(logps.device, logps.dtype)
                if ref.dim() == 2 and ref.shape[1] != logps.shape[1]:      # shorter rows end in nothing, longer ones are cut
                    ref = F.pad(ref, (0, logps.shape[1] - ref.shape[1]))
            elif not self.reference_free:
                return LossOutput(loss=logps.sum() * 0.0, num_tokens=0)
        loss, stats = ops.preference_loss(logps, mask, ref, self.loss_type, self.beta, label_smoothing=self.label_smoothing, nll_weight=max(self.sft_weight, 0.0),
                                          twice=True)
        self.last_stats = dict(zip(('rewards/chosen', 'rewards/rejected', 'rewards/margins', 'rewards/accuracies', 'logps/chosen', 'logps/rejected'), stats.tolist()))
        return LossOutput(loss=loss, num_tokens=0)


class SimPOLoss(PreferenceLoss):
    """Length-normalised, reference-free: ``−logσ(β(avg_c − avg_r) − γ)``."""

    def __init__(self, beta: float = 2.5, gamma: float = 0.5, ignore_index: int = -100, **kwargs):
        super().__init__(ignore_index)
        self.beta, self.gamma = beta, gamma

    def __call__(self, inputs, outputs, **kwargs) -> LossOutput:
        rows = self._rows(inputs, outputs)
        if rows is not None:
            return LossOutput(loss=ops.preference_loss(rows[1], rows[0], form='simpo', beta=self.beta, gamma=self.gamma, twice=True)[0], num_tokens=0)
        logps, mask, seq = self._seq_logps(inputs, outputs)
        avg = seq / mask.sum(-1).clamp_min(1)
        z = self.beta * (avg[0::2] - avg[1::2]) - self.gamma
        return LossOutput(loss=(-F.logsigmoid(z)).mean(), num_tokens=0)


class CPOLoss(PreferenceLoss):
    """``−logσ(β(π_c − π_r)) + bc_coef · NLL(chosen)``."""

    def __init__(self, beta: float = 0.1, bc_coef: float = 1.0, ignore_index: int = -100, **kwargs):
        super().__init__(ignore_index)
        self.beta, self.bc_coef = beta, bc_coef

    def __call__(self, inputs, outputs, **kwargs) -> LossOutput:
        rows = self._rows(inputs, outputs)
        if rows is not None:
            return LossOutput(loss=ops.preference_loss(rows[1], rows[0], beta=self.beta, nll_weight=self.bc_coef, twice=True)[0], num_tokens=0)
        logps, mask, seq = self._seq_logps(inputs, outputs)
        pref = -F.logsigmoid(self.beta * (seq[0::2] - seq[1::2])).mean()
        return LossOutput(loss=pref + self.bc_coef * self._nll(seq[0::2], mask), num_tokens=0)


class ORPOLoss(PreferenceLoss):
    """NLL(chosen) − λ·logσ(log odds ratio) on length-averaged logps."""

    def __init__(self, lambda_orpo: float = 0.1, ignore_index: int = -100, **kwargs):
        super().__init__(ignore_index)
        self.lambda_orpo = lambda_orpo

    def __call__(self, inputs, outputs, **kwargs) -> LossOutput:
        rows = self._rows(inputs, outputs)
        if rows is not None:
            return LossOutput(loss=ops.preference_loss(rows[1], rows[0], form='orpo', beta=self.lambda_orpo, nll_weight=1.0, twice=True)[0], num_tokens=0)
        logps, mask, seq = self._seq_logps(inputs, outputs)
        avg = seq / mask.sum(-1).clamp_min(1)
        c, r = avg[0::2], avg[1::2]
        log_odds = (c - r) - (torch.log1p(-torch.exp(c).clamp(max=1 - 1e-6)) - torch.log1p(-torch.exp(r).clamp(max=1 - 1e-6)))
        loss = self._nll(seq[0::2], mask) - self.lambda_orpo * F.logsigmoid(log_odds).mean()
        return LossOutput(loss=loss, num_tokens=0)


_ON_KERNEL = (DPOLoss, SimPOLoss, CPOLoss, ORPOLoss)
_METHODS = ('_seq_logps', '_nll', '_align_ref')
_DEFINED = tuple(getattr(PreferenceLoss, n) for n in _METHODS)
