"""Log probabilities of given prototypes with entropy and best prototypes, differentiable with respect to the logits
(one pass over the logits forward, one backward; the kernels behind ops.logprob_fwd / logprob_bwd)."""
from typing import NamedTuple, Optional

import torch

from .. import ops


class PrototypeLogProbs(NamedTuple):
    log_prob: Optional[torch.Tensor]      # fp32, the targets' shape
    entropy: torch.Tensor                 # fp32 [R], natural logarithm
    top_log_prob: Optional[torch.Tensor]  # fp32 [R, topk]
    top_index: Optional[torch.Tensor]     # int64 [R, topk]


class _LogProbFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, center, temp, topk):
        ctx.set_materialize_grads(False)
        r = ops.logprob_fwd(logits, targets, center=center, temp=temp, topk=topk)
        ctx.save_for_backward(logits, targets, center, *[t for t in r if t is not None])
        ctx.temp, ctx.topk = temp, topk
        if topk:
            ctx.mark_non_differentiable(r.top_index)
            return r.log_prob, r.entropy, r.top_log_prob, r.top_index
        return r.log_prob, r.entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlp, dent, dtop=None, _=None):
        logits, targets, center, *saved = ctx.saved_tensors
        fwd = ops.LogProbs(*saved) if ctx.topk else ops.LogProbs(*saved, None, None)

        if dlp is None and dent is None and dtop is None:
            return (None,) * 5

        def dense(g):
            return None if g is None else g.to(torch.float32).contiguous()
        dx = ops.logprob_bwd(logits, fwd, targets=targets, center=center, temp=ctx.temp,
                             dlog_prob=dense(dlp) if targets is not None else None, dentropy=dense(dent),
                             dtop_log_prob=dense(dtop))
        return dx, None, None, None, None


def prototype_log_probs(logits, targets=None, *, center=None, temperature=1.0, topk=0) -> PrototypeLogProbs:
    """softmax((logits - center) / temperature) seen from outside: log probabilities at targets (int64 [R] or [R, T];
    -1: none, gives 0), entropy of each row, and the topk best prototypes with their log probabilities.

    logits: bf16 / fp32 [R, K]; -inf logits have probability 0, and a row of nothing else has entropy 0, log probabilities
    of -inf and no gradient.  center: fp32 [K] or [1, K] (DINOLoss.center), a constant.  The gradient reaches the logits
    from log_prob, entropy and top_log_prob (not under stream capture: ops.logprob_fwd / logprob_bwd there)."""
    if center is not None:
        if center.requires_grad:
            raise ValueError("prototype_log_probs: center is a constant, it gets no gradient")
        center = center.reshape(-1)
    if logits.is_cuda and logits.requires_grad and torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing():
        # a backward pass captured while another graph of the same leaf is alive ends the process inside torch
        raise RuntimeError("prototype_log_probs: under stream capture call ops.logprob_fwd and ops.logprob_bwd")
    flat = targets is not None and targets.dim() == 1
    tgt = targets.reshape(-1, 1) if flat else targets
    out = _LogProbFn.apply(logits, None if tgt is None else tgt.contiguous(), center, float(temperature), topk)
    lp = None if targets is None else (out[0].reshape(-1) if flat else out[0])
    return PrototypeLogProbs(lp, out[1], out[2] if topk else None, out[3] if topk else None)
