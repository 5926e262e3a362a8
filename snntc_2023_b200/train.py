"""What surrounds the SNN-TC layers in a training step of the reference's example trainers, on this
library's own kernels (csrc/snntc_train.cu) instead of framework glue:

    encode(p)                       exp(1 - p) / exp(p) input encoding            snntc-mnist.py:75
    loss_func(logit, label)         softmax cross-entropy on -logit, batch mean   SNN_TC_Modules.py:286-288
    accuracy_count(logit, label)    number of samples whose earliest spike is the label   snntc-mnist.py:82
    label_log_probs(logit, label)   log softmax(-logit)[label], a number per row
    policy_loss(...)                clipped policy loss with a KL term            } losses on choices; the
    preference_loss(...)            paired log ratios of preferred and rejected texts }  reference has none
    constraint_cost(weights, K, K2) K*sum_w mean_j max(0,1-sum_i w_ij) + K2*sum_w mean(w^2)   snntc-mnist.py:55-59
    Adam / SGDM                     Keras-formulation optimisers over one flat parameter buffer and the
                                    flat gradient buffer the backward kernels (and the all-reduce) write

Everything here needs the CUDA library; there is no CPU path.
"""

import torch

from . import _lib
from .ops import _as_cuda_f32, _stream, _tensor


def encode(p, scale=1.0, one_minus=True):
    """x = exp(scale*(1-p)) (pixel intensities -> spike times, the reference's encoding) or exp(scale*p)."""
    return _lib.native().encode(_tensor(p, "p"), scale, one_minus)


def loss_func(logit=None, label=None, with_hits=False):
    """Mean softmax cross-entropy on the negated spike times. `label`: integer classes [B] or one-hot [B,C].
    with_hits=True also returns the number of samples whose arg-min output equals the label (a 0-d tensor)."""
    loss, hits = _lib.native().loss(_tensor(logit, "logit"), label)
    return (loss, hits) if with_hits else loss


def accuracy_count(logit, label):
    with torch.no_grad():
        return loss_func(logit, label, with_hits=True)[1]


def constraint_cost(weights, K, K2):
    """K * sum over tensors of mean_j max(0, 1 - sum_i w_ij) + K2 * sum over tensors of mean(w^2); each tensor is
    a layer's whole [fan_in(+1), fan_out] weight, bias row included, as in the reference's trainable_variables."""
    return _lib.native().constraint_cost(list(weights), K, K2)


def label_log_probs(logit, label):
    """log softmax(-logit)[label] of every row: logit [..., classes] spike values, label [...] integers; [...]. A row whose label
    is outside the classes (-1, say) does not count: 0, and no gradient. The gradient cannot be differentiated again. Under no_grad
    this is what policy_loss and preference_loss take as the old and the reference network's log-probabilities."""
    return _lib.native().label_log_probs(_tensor(logit, "logit"), _tensor(label, "label"))


def policy_loss(logit, label, old_logp, advantage, ref_logp=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, with_stats=False):
    """Clipped policy loss, the mean over the rows whose label is one of the classes (0 where there is none):

        -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef * k
        r = exp(lp - old_logp), A = advantage, k = exp(ref_logp - lp) - (ref_logp - lp) - 1, lp = label_log_probs(logit, label)

    logit [..., classes]; label, old_logp, advantage, ref_logp [...], one value per row, the last three constants. with_stats=True
    also returns [mean k, share of rows whose ratio was clipped]; with kl_coef = 0 k has no part in loss and gradient. Where k
    overflows -- a label that does not spike, lp near -1e5, beside a reference of -3 -- the mean k is infinite, and with kl_coef > 0
    the loss is, too, and that row's gradient (already from ref_logp - lp = 88 on, float32's range) infinite or NaN; a ratio that
    overflows beside a negative advantage does the same. The gradient is formed with the loss, in the pass that reads the
    logits; it cannot be differentiated again."""
    loss, stats = _lib.native().policy_loss(_tensor(logit, "logit"), _tensor(label, "label"), _tensor(old_logp, "old_logp"),
                                            _tensor(advantage, "advantage"),
                                            None if ref_logp is None else _tensor(ref_logp, "ref_logp"), float(clip_low),
                                            float(clip_high), float(kl_coef))
    return (loss, stats) if with_stats else loss


def preference_loss(logit, label, starts=None, ref_logp=None, beta=0.1, label_smoothing=0.0, with_margins=False):
    """Preference loss on P pairs of texts, text k preferred to text P + k:

        mean_k of -(1 - label_smoothing) log sigma(m_k) - label_smoothing log sigma(-m_k)
        m_k = beta * ((S_k - ref_logp[k]) - (S_{P+k} - ref_logp[P+k])),   S_s the sum of label_log_probs over text s

    Texts one behind the other: logit [rows, classes], label [rows], `starts` 2P+1 ascending offsets on the GPU, text s being
    rows starts[s] to starts[s+1] (rows behind the last are of no text). Padded texts: logit [2P, rows, classes], label
    [2P, rows], no starts. Rows whose label is outside the classes (prompts, padding) do not count. ref_logp [2P]: the
    reference network's sums (none: 0), a constant. with_margins=True also returns the m_k. The gradient cannot be differentiated
    again."""
    loss, margins = _lib.native().preference_loss(_tensor(logit, "logit"), _tensor(label, "label"),
                                                  None if starts is None else _tensor(starts, "starts"),
                                                  None if ref_logp is None else _tensor(ref_logp, "ref_logp"), float(beta),
                                                  float(label_smoothing))
    return (loss, margins) if with_margins else loss


class _FlatOptimizer:
    def __init__(self, param, grad):
        self.param = _as_cuda_f32(param.detach() if isinstance(param, torch.nn.Parameter) else param, "param")
        self.grad = _as_cuda_f32(grad, "grad")
        if self.param.numel() != self.grad.numel():
            raise ValueError("parameter and gradient buffers differ in size")

    def zero_grad(self):
        self.grad.zero_()


class Adam(_FlatOptimizer):
    """tf.keras.optimizers.Adam over one flat fp32 buffer; the step count lives on the device, so step() can be
    captured into a CUDA graph and replayed. grad_scale multiplies the gradient first (1/world for a summed
    all-reduce)."""

    def __init__(self, param, grad, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-7):
        super().__init__(param, grad)
        self.lr, self.beta1, self.beta2, self.eps = lr, beta1, beta2, eps
        self.m = torch.zeros_like(self.param)
        self.v = torch.zeros_like(self.param)
        self.steps = torch.zeros(1, dtype=torch.int32, device=self.param.device)

    def step(self, grad_scale=1.0):
        _lib.native().adam_step(self.param, self.grad, self.m, self.v, self.lr, self.beta1, self.beta2, self.eps,
                                grad_scale, self.steps)


class SGDM(_FlatOptimizer):
    """tf.keras.optimizers.SGD(momentum=...): vel = momentum*vel - lr*g; w += vel."""

    def __init__(self, param, grad, lr=1e-2, momentum=0.9):
        super().__init__(param, grad)
        self.lr, self.momentum = lr, momentum
        self.vel = torch.zeros_like(self.param)

    def step(self, grad_scale=1.0):
        lib = _lib.load()
        with torch.cuda.device(self.param.device):
            rc = lib.snntc_sgdm_step(self.param.data_ptr(), self.grad.data_ptr(), self.vel.data_ptr(),
                                     self.param.numel(), float(self.lr), float(self.momentum), float(grad_scale),
                                     _stream(self.param))
        _lib.check(rc, "SGDM.step")
