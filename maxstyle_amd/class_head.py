"""`class_cross_entropy`: a classification head and its cross entropy over many classes as one differentiable operator that never keeps the logits - cross_entropy_2D
(custom_loss.py:1043-1078) of `F.conv2d(h, weight, bias)` where head_ce's four classes are not enough."""
import torch

from . import ops


class _ClassCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, bias, labels):
        nll, lse = ops.class_ce_fwd(h, weight, bias, labels)
        ctx.save_for_backward(h, weight, bias, labels, lse)
        return nll

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("class_cross_entropy: its backward cannot be captured into a graph; capture ops.class_ce or ops.class_ce_bwd")
        h, weight, bias, labels, lse = ctx.saved_tensors
        dh, dw, db = ops.class_ce_bwd(h, weight, bias, labels, lse, grad.float().contiguous(), *ctx.needs_input_grad[:3])
        return dh, dw, db, None


def class_cross_entropy(h, weight, bias, labels, reduction="mean"):
    """Cross entropy of the logits `weight @ h + bias` against `labels`; differentiable in h, weight and bias, the logits never kept (recomputed in the backward).

    h [N,C,*spatial] or rows [T,C], fp32 or bf16; weight [V,C] or [V,C,1,1], fp32 or bf16; bias [V] fp32 or None; labels [N,*spatial] int64.  A label outside [0,V) takes
    its row out of the loss and of the gradients.  reduction: "mean" over all rows (what cross_entropy_2D does), "valid" over the rows that take part (0 if there are
    none), "sum", or "none" ([N,*spatial]).  Inside a graph capture use ops.class_ce or ops.class_ce_fwd / class_ce_bwd: a captured autograd backward of leaves that an
    eager graph still holds ends the process, so a call that would record one raises."""
    if reduction not in ("mean", "valid", "sum", "none"):
        raise ValueError("class_cross_entropy: reduction is 'mean', 'valid', 'sum' or 'none'")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (h, weight, bias)):
        if h.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("class_cross_entropy: not under graph capture with gradients; capture ops.class_ce (loss and gradients in one call)")
    elif reduction != "none":            # value only: summed by the operator's own kernels (a library sum over many blocks would put a memset into a captured graph)
        return ops.class_ce(h, weight, bias, labels, loss_sign=float(labels.numel()) if reduction == "sum" else 1.0, mean_over="valid" if reduction == "valid" else "all",
                            need_dh=False, need_dw=False)[0]
    nll = _ClassCrossEntropy.apply(h, weight, bias, labels)
    if reduction == "none":
        return nll
    if reduction == "sum":
        return nll.sum()
    if reduction == "mean":
        return nll.sum() / nll.numel()
    valid = ((labels >= 0) & (labels < weight.shape[0])).sum().clamp(min=1)
    return nll.sum() / valid
