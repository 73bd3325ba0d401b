"""Losses that tune a caption model on its own samples or on preferred / rejected captions, next to LabelSmoothing: modules around
bmt_amd.ops.policy_loss and bmt_amd.ops.preference_loss.  ``pred``: a Generator's log-probabilities or any logits (B, S, V)."""
import torch.nn as nn

from .. import ops


class PolicyLoss(nn.Module):

    def __init__(self, pad_idx=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, reduction="token"):
        super(PolicyLoss, self).__init__()
        self.pad_idx = pad_idx
        self.clip_low, self.clip_high = clip_low, clip_high
        self.kl_coef = kl_coef
        self.reduction = reduction

    def forward(self, pred, target, old_logp, advantages, ref_logp=None, mask=None):  # -> (loss, ops.PolicyStats)
        return ops.policy_loss(pred, target, old_logp, advantages, ref_logp, mask, self.pad_idx, self.clip_low, self.clip_high, self.kl_coef,
                               self.reduction)


class PreferenceLoss(nn.Module):

    def __init__(self, pad_idx=None, beta=0.1, label_smoothing=0.0, mean_logp=False):
        super(PreferenceLoss, self).__init__()
        self.pad_idx = pad_idx
        self.beta = beta
        self.label_smoothing = label_smoothing
        self.mean_logp = mean_logp

    def forward(self, pred, target, ref_logp, mask=None):  # first half of the batch preferred to the second; -> (loss, rewards (B,))
        return ops.preference_loss(pred, target, ref_logp, mask, self.pad_idx, self.beta, self.label_smoothing, self.mean_logp)
