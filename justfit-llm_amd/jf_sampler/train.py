"""Distillation of a draft model as a torch loss: the losses and gradients are
jf_distill's and jf_distill_backward's (no fallback)."""
import torch

from . import JF_TEACHER_TOKENS


class _DistillLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, scorer, teacher_ids, teacher_values, temperature, normalize):
        rows, k = teacher_ids.shape
        loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
        saved = torch.empty((rows, 2 + k), dtype=torch.float32, device=logits.device)
        args = scorer.distill_args(
            logits, teacher_ids, teacher_values, temperature=temperature, normalize=normalize,
            loss=loss, saved=saved)
        if rows:
            scorer.launch_distill(args)
        # The probabilities in `saved` are by slot: the ids as they are now, since a
        # trainer's list buffers may hold the next batch's by the backward pass, and
        # what the library writes into a tensor torch does not see.
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(logits, teacher_ids.clone(), saved)
        ctx.scorer, ctx.temperature, ctx.normalize = scorer, temperature, normalize
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, teacher_ids, saved = ctx.saved_tensors
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
        if grad_loss.numel():
            ctx.scorer.launch_distill_backward(ctx.scorer.distill_args(
                logits, teacher_ids, None, temperature=ctx.temperature, normalize=ctx.normalize,
                saved=saved, grad_loss=grad_loss, grad=grad))
        return grad, None, None, None, None, None


def distill_loss(scorer, logits, teacher_ids, teacher_values, temperature=1.0, normalize=True):
    """Each row's loss against a teacher's list (jf_distill) on torch's
    current stream, with gradients for `logits` ([rows, vocabulary], f32 or
    bf16, contiguous rows; an empty batch has no losses). teacher_ids: int32
    [rows, k], -1 for absent slots; teacher_values: f32 [rows, k], logits with
    `normalize`, otherwise log-probabilities at the temperature. The lists may be
    filled anew once the loss is taken; the logits have to stay as they are until
    its backward pass."""
    if not 1 <= teacher_ids.shape[1] <= JF_TEACHER_TOKENS:
        raise ValueError(f"a teacher's list holds 1..{JF_TEACHER_TOKENS} tokens")
    return _DistillLoss.apply(logits, scorer, teacher_ids, teacher_values, float(temperature),
                              bool(normalize))
