"""Training losses on (logits, worst-case margins, targets), the reference's `--loss` choices (main.py:329-379).

`outputs` are the logits of the clean input, `worst_outputs` the worst-case margins of every class against the
target (0 in the target column) that the models return beside the logits (ell_inf_models.py:45-50).  Each loss is
a plain function; the classes below carry the reference's names, constructor arguments and the
`loss.update(ratio)` / `loss(outputs, worst_outputs, targets)` protocol of main.py:85-92, so a loss spec such as
`mixture(lam0=0.05,lam_end=0.0005)` maps onto them unchanged.

Beside them stand losses for heads that learn from answers, preferences and rewards instead of one right label
(no counterpart in the reference): `label_log_probs`, `preference_loss` and `policy_loss`, as HIP kernels.  They take
logits in fp32, bf16 or fp16 on the GPU; of `worst_outputs` in the place of `outputs` they take the certified lower bounds of the
log probabilities, as the cross entropies above do.  They are differentiated once: a derivative of their gradients raises an error.
"""
import math

import torch
import torch.nn.functional as TF

from . import ext


def lam_schedule(lam0, lam_end, ratio):
    """Weight of the clean cross-entropy term: lam0 (lam_end / lam0)^ratio, ratio = training progress in [0, 1]
    (main.py:338-347); 0 stays 0."""
    return 0.0 if lam0 == 0 else lam0 * math.exp(math.log(lam_end / lam0) * ratio)


def hinge_loss(worst_outputs, mix=0.25):
    """main.py:329-335: largest positive margin per sample, mixed with the mean over all classes."""
    res = worst_outputs.clamp(min=0)
    return (1 - mix) * res.max(dim=1)[0].mean() + mix * res.mean()


def crossentropy_loss(outputs, worst_outputs, targets, lam):
    """main.py:353-355."""
    return TF.cross_entropy(worst_outputs, targets) + lam * TF.cross_entropy(outputs, targets)


def mixture_loss(outputs, worst_outputs, targets, lam, clip=1.0):
    """main.py:358-365: clipped hinge on the worst margin plus the decaying clean cross entropy."""
    res = worst_outputs.clamp(min=0, max=clip)
    return res.max(dim=1)[0].mean() + lam * TF.cross_entropy(outputs, targets)


def ce_hinge_loss(outputs, worst_outputs, targets, lam):
    """main.py:368-373: unit-margin hinge between the worst margins, counted only for samples the clean logits
    classify correctly."""
    correct = (outputs.argmax(dim=1) == targets).to(outputs.dtype)
    col = targets.view(-1, 1)
    margin = (worst_outputs - worst_outputs.gather(1, col) + 1).scatter(1, col, 0)
    return (correct * margin.max(dim=1)[0]).mean() + lam * TF.cross_entropy(outputs, targets)


def ce_mixture_loss(outputs, worst_outputs, targets, lam):
    """main.py:376-379: cross entropy of the worst margins on correctly classified samples."""
    correct = (outputs.argmax(dim=1) == targets).to(outputs.dtype)
    return (correct * TF.cross_entropy(worst_outputs, targets, reduction="none")).mean() + \
        lam * TF.cross_entropy(outputs, targets)


def label_log_probs(outputs, targets, ignore_index=-100):
    """log softmax(outputs)[..., target], fp32, with gradients to `outputs`.

    outputs (..., classes); targets int64 or int32 with the sizes before the classes.  Rows whose target is `ignore_index` are not
    read: 0, with a gradient of zeros, whatever they hold.  A target that names no class gives NaN.  Rows may be strided (a padded vocabulary, a
    part of a batch); logits of -inf are classes that cannot be chosen.  A batch of no rows gives no values."""
    return ext.host().label_log_probs(outputs, targets, ignore_index)


def preference_loss(outputs, targets, ref_log_probs, offsets=None, beta=0.1, label_smoothing=0.0, ignore_index=-100):
    """Loss on pairs of answers, the chosen one against the rejected: (loss, rewards).

    The answers are the rows of `outputs` (answers, tokens, classes) or (answers, classes), or packed ones behind each other: outputs
    (rows, classes) and `offsets` (answers + 1, int32 or int64, not decreasing, on the GPU), the rows behind the last answer belonging to none.
    The first half of the answers is chosen over the second, each over the one half the answers further on.  `targets` are
    the tokens (`ignore_index` for prompts and padding), `ref_log_probs` what label_log_probs gives for the reference model.

    rewards[a] = beta sum over the rows of a of (log prob - ref), without a gradient; x = chosen's - rejected's reward;
    loss = mean of -(1 - s) log sigma(x) - s log sigma(-x) with s = label_smoothing below 1/2.  A batch of no pairs, or of no rows, is refused."""
    return ext.host().preference_loss(outputs, targets, ref_log_probs, offsets, beta, label_smoothing, ignore_index)


def policy_loss(outputs, targets, old_log_probs, advantages, ref_log_probs=None, clip=0.2, clip_high=None, kl_coef=0.0, ignore_index=-100):
    """Clipped policy loss with a KL term: (loss, stats).

    Per row, with ratio = exp(log prob - old) of the action `targets` and advantage A:
        -min(ratio A, clip(ratio, 1 - clip, 1 + clip_high) A) + kl_coef (exp(ref - log prob) - (ref - log prob) - 1)
    and the mean over the rows that are not ignored (0 where all are; a batch of no rows is refused).  clip_high defaults to clip.  `old_log_probs`, `advantages` and
    `ref_log_probs` have the sizes of `targets` and get no gradient; one advantage per answer is given as `a[:, None].expand(...)`, which is
    not copied.  From 32 MiB of logits on the gradient is made with the loss, for an upstream gradient of 1: a positive factor on the loss is cheaper
    as one on `advantages` and `kl_coef`.  stats: the first term, the divergence (without kl_coef; 0 where that is 0) and the share of clipped rows."""
    return ext.host().policy_loss(outputs, targets, old_log_probs, advantages, ref_log_probs, clip, clip if clip_high is None else clip_high,
                                  kl_coef, ignore_index)


class hinge:
    def __init__(self, mix=0.25):
        self.mix = mix

    def update(self, ratio):
        pass

    def __call__(self, outputs, worst_outputs, targets):
        return hinge_loss(worst_outputs, self.mix)


class _Decaying:
    fn = None

    def __init__(self, lam0=1.0, lam_end=0.01, **extra):
        self.lam_start, self.lam_end, self.lam, self.extra = lam0, lam_end, lam0, extra

    def update(self, ratio):
        self.lam = lam_schedule(self.lam_start, self.lam_end, ratio)

    def __call__(self, outputs, worst_outputs, targets):
        return type(self).fn(outputs, worst_outputs, targets, self.lam, **self.extra)


class crossentropy(_Decaying):
    fn = staticmethod(crossentropy_loss)


class mixture(_Decaying):
    fn = staticmethod(mixture_loss)

    def __init__(self, lam0=1.0, lam_end=0.01, clip=1):
        super().__init__(lam0, lam_end, clip=clip)


class ce_hinge(_Decaying):
    fn = staticmethod(ce_hinge_loss)


class ce_mixture(_Decaying):
    fn = staticmethod(ce_mixture_loss)


LOSSES = {c.__name__: c for c in (hinge, crossentropy, mixture, ce_hinge, ce_mixture)}
