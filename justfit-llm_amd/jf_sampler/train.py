"""Losses over rows of logits as torch functions, and what a training step ends
with: distillation of a draft model, the clipped policy loss, the preference loss
over pairs of sequences, and clipping by the global gradient norm. Losses and
gradients are the library's passes (no fallback)."""
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


def _count_writes(tensors):
    """Counts what the library has written through addresses as torch counts its own writes
    in place, so that a graph that has saved one of the tensors refuses its backward pass.
    Inference tensors have no such count."""
    torch.autograd.graph.increment_version(
        [t for t in tensors if t is not None and not t.is_inference()])


def _rows_saved(logits):
    return torch.empty((logits.shape[0], 4), dtype=torch.float32, device=logits.device)


class _ClippedLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, scorer, tokens, advantages, options):
        loss = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
        saved = _rows_saved(logits)
        args = scorer.clipped_args(logits, tokens, advantages, loss=loss, saved=saved, **options)
        if advantages is None:
            raise ValueError("advantages are missing")
        if loss.numel():
            scorer.launch_clipped(args)
            _count_writes(options[k] for k in ("logprobs", "kl", "entropy"))
        # The tokens as they are now: a trainer's buffers may hold the next batch's by
        # the backward pass.
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(logits, tokens.clone(), saved)
        ctx.scorer = scorer
        ctx.options = {k: options[k] for k in ("entropy_weight", "temperature")}
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, tokens, saved = ctx.saved_tensors
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
        if grad.numel():
            ctx.scorer.launch_clipped_backward(ctx.scorer.clipped_args(
                logits, tokens, None, saved=saved, grad_loss=grad_loss, grad=grad, **ctx.options))
        return grad, None, None, None, None


def clipped_loss(scorer, logits, tokens, advantages, old_logprobs=None, reference_logprobs=None,
                 *, clip_low=0.2, clip_high=0.2, kl_weight=0.0, entropy_weight=0.0,
                 temperature=1.0, logprobs=None, kl=None, entropy=None):
    """Each row's clipped policy loss (jf_clipped_loss) on torch's current stream,
    with gradients for `logits` ([rows, vocabulary], f32 or bf16, contiguous rows; an
    empty batch has no losses). tokens: int32 [rows], -1 for rows that are not
    trained on, whose loss is 0; the others f32 [rows]. logprobs, kl, entropy: f32
    [rows] to be filled for a trainer's records, without gradients. All but the
    logits may be filled anew once the loss is taken; the logits have to stay as they
    are until its backward pass."""
    return _ClippedLoss.apply(logits, scorer, tokens, advantages, dict(
        old_logprobs=old_logprobs, reference_logprobs=reference_logprobs,
        clip_low=float(clip_low), clip_high=float(clip_high), kl_weight=float(kl_weight),
        entropy_weight=float(entropy_weight), temperature=float(temperature), logprobs=logprobs,
        kl=kl, entropy=entropy))


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, scorer, tokens, offsets, options):
        pairs = (offsets.shape[0] - 1) // 2 if torch.is_tensor(offsets) and offsets.dim() == 1 \
            else 0
        loss = torch.empty(max(0, pairs), dtype=torch.float32, device=logits.device)
        saved = _rows_saved(logits)
        args = scorer.preference_args(logits, tokens, offsets, loss=loss, saved=saved, **options)
        if saved.numel():
            scorer.launch_preference(args)
            _count_writes(options[k] for k in ("scores", "logprobs"))
        else:
            # Pairs without any token.
            for t in (loss, options["scores"]):
                if t is not None:
                    t.zero_()
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(logits, tokens.clone(), offsets.clone(), saved)
        ctx.scorer, ctx.temperature = scorer, options["temperature"]
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, tokens, offsets, saved = ctx.saved_tensors
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
        if grad.numel():
            ctx.scorer.launch_preference_backward(ctx.scorer.preference_args(
                logits, tokens, offsets, temperature=ctx.temperature, saved=saved,
                grad_loss=grad_loss, grad=grad))
        return grad, None, None, None, None


def preference_loss(scorer, logits, tokens, offsets, reference_logprobs=None, *, beta=0.1,
                    margin=0.0, smoothing=0.0, kind="sigmoid", mean=False, temperature=1.0,
                    scores=None, logprobs=None):
    """Each pair's preference loss (jf_preference_loss) on torch's current stream,
    with gradients for `logits` (as clipped_loss's). offsets: int32 [2 * pairs + 1],
    sequence q is rows offsets[q] .. offsets[q + 1] - 1, and pair p prefers sequence
    2p to 2p + 1. tokens: int32 [rows], -1 for rows that are not scored (a prompt's);
    reference_logprobs: f32 [rows]. scores (f32 [2 * pairs]) and logprobs (f32 [rows])
    are filled for a trainer's records, without gradients. All but the logits may be
    filled anew once the loss is taken; the logits have to stay as they are until its
    backward pass."""
    return _PreferenceLoss.apply(logits, scorer, tokens, offsets, dict(
        reference_logprobs=reference_logprobs, beta=float(beta), margin=float(margin),
        smoothing=float(smoothing), kind=kind, mean=bool(mean), temperature=float(temperature),
        scores=scores, logprobs=logprobs))


def clip_gradients(clipper, parameters, max_norm, order=2.0):
    """Scales the gradients of `parameters` (those that have one), in place, to a
    global norm of at most max_norm (jf_gradient_clip) on torch's current stream, and
    returns the norm that they had, a device scalar: nothing waits for the GPU.
    Gradients are f32 or bf16, at most clipper.max_tensors of them."""
    parameters = [parameters] if torch.is_tensor(parameters) else parameters
    gradients = [p.grad for p in parameters if p.grad is not None]
    norm = torch.empty((), dtype=torch.float32, device=torch.device("cuda", clipper.device))
    clipper.launch_clip(clipper.args(gradients, norm=norm, max_norm=float(max_norm),
                                     order=float(order)))
    _count_writes(gradients)
    return norm
