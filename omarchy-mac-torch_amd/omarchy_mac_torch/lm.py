"""Both ends of a language model's training step on the omarchy_mac_torch device, beside its feed-forward sublayers (ffn):

    embedding        scale * weight[tokens], its gradient summed in the order of positions
    token_logps      log softmax(logits)[label]: a reference's log-probabilities, or those that tokens were sampled with
    preference_loss  training on pairs of sequences: one chosen, one rejected
    policy_loss      training on rewards: clipped probability ratios times advantages, with a KL term to a reference

Differentiable functions, and Embedding as a module, over torch.ops.omt's operators. The two losses compute the logits' gradient with the loss, where
one can be asked for, and hand it on in the backward pass, which therefore runs once; scaled by what arrives there, a gradient in
bfloat16 is rounded a second time, unless that is a power of two. optim.AdamW is the step at the end.

No counterpart in the reference. hip_ops has the same operators as plain functions, for torch.cuda tensors too.
"""

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from omarchy_mac_torch import hip_ops
from omarchy_mac_torch.native import DEVICE

__all__ = ["Embedding", "embedding", "policy_loss", "preference_loss", "token_logps"]

_transforms_active = torch._C._are_functorch_transforms_active  # whether one of torch.func's is on


def _each(apply, size, in_dims, args):
    """apply on each of `size` samples of those arguments that have a dimension of them, stacked."""
    return torch.stack([apply(*(a if d is None else a.select(d, i) for a, d in zip(args, in_dims))) for i in range(size)]), 0


class _Embedding(torch.autograd.Function):
    """Linear in the weight, as _EmbeddingGradient is in gy: each is what the other's derivatives are made of, in either mode and of
    any order."""

    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx):
        ctx.save_for_backward(tokens)
        ctx.save_for_forward(tokens)
        ctx.vocab, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return hip_ops.embedding(tokens, weight, scale)

    @staticmethod
    def backward(ctx, gy):
        tokens, = ctx.saved_tensors
        gradient = _EmbeddingGradient.apply if torch.is_grad_enabled() or _transforms_active() else hip_ops.embedding_backward
        return None, gradient(gy, tokens, ctx.vocab, ctx.scale, ctx.padding_idx), None, None

    @staticmethod
    def jvp(ctx, _, tangent, *__):
        tokens, = ctx.saved_tensors
        return embedding(tokens, tangent, ctx.scale, ctx.padding_idx)


class _TransformedEmbedding(_Embedding):
    """The same in the form that torch.func's transforms take, which costs twice the host's time (forward 15 us for 7.5)."""

    @staticmethod
    def forward(tokens, weight, scale, padding_idx):
        return hip_ops.embedding(tokens, weight, scale)

    @staticmethod
    def setup_context(ctx, inputs, output):
        tokens, weight, ctx.scale, ctx.padding_idx = inputs
        ctx.vocab = weight.shape[0]
        ctx.save_for_backward(tokens)
        ctx.save_for_forward(tokens)

    @staticmethod
    def backward(ctx, gy):
        tokens, = ctx.saved_tensors
        return None, _EmbeddingGradient.apply(gy, tokens, ctx.vocab, ctx.scale, ctx.padding_idx), None, None

    @staticmethod
    def vmap(info, in_dims, tokens, weight, scale, padding_idx):
        if in_dims[1] is None:
            return embedding(tokens.movedim(in_dims[0], 0), weight, scale, padding_idx), 0
        return _each(lambda t, w: embedding(t, w, scale, padding_idx), info.batch_size, in_dims, (tokens, weight))


class _EmbeddingGradient(torch.autograd.Function):
    @staticmethod
    def forward(gy, tokens, vocab, scale, padding_idx):
        return hip_ops.embedding_backward(gy, tokens, vocab, scale, padding_idx)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, tokens, ctx.vocab, ctx.scale, ctx.padding_idx = inputs
        ctx.save_for_backward(tokens)
        ctx.save_for_forward(tokens)

    @staticmethod
    def backward(ctx, ggw):
        tokens, = ctx.saved_tensors
        took_part = (tokens >= 0) & (tokens < ctx.vocab)
        if ctx.padding_idx is not None:
            took_part &= tokens != ctx.padding_idx % ctx.vocab
        rows = embedding(tokens, ggw, ctx.scale, ctx.padding_idx)
        return torch.where(took_part[..., None], rows, 0.0), None, None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        tokens, = ctx.saved_tensors
        return _EmbeddingGradient.apply(tangent, tokens, ctx.vocab, ctx.scale, ctx.padding_idx)

    @staticmethod
    def vmap(info, in_dims, gy, tokens, vocab, scale, padding_idx):
        return _each(lambda g, t: _EmbeddingGradient.apply(g, t, vocab, scale, padding_idx), info.batch_size, in_dims, (gy, tokens))


class _TokenLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ignore_index):
        logps, lse = hip_ops.token_logps(logits, labels, ignore_index, lse_dtype=torch.float64)
        ctx.save_for_backward(logits, labels, lse)
        ctx.ignore_index = ignore_index
        return logps

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        return hip_ops.token_logps_backward(g, *ctx.saved_tensors, ctx.ignore_index), None, None


class _Loss(torch.autograd.Function):
    """A loss whose operator, op(logits, **arguments), gives (loss, others..., the logits' gradient)."""

    @staticmethod
    def forward(ctx, logits, op, arguments):
        loss, *others, ctx.gradient = op(logits, **arguments)
        ctx.mark_non_differentiable(*others)
        ctx.set_materialize_grads(False)
        return loss, *others

    @staticmethod
    @once_differentiable
    def backward(ctx, gloss, *_):
        if gloss is None:
            return None, None, None
        if ctx.gradient is None:
            raise RuntimeError("the loss's gradient has been handed on already: its backward pass runs once")
        gradient, ctx.gradient = ctx.gradient, None
        return hip_ops.scale_by_(gradient, gloss), None, None


def _loss(op, logits, arguments):
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Loss.apply(logits, op, arguments)
    return op(logits, **arguments, grad=False)[:-1]


@torch.compiler.disable  # one operator each way: nothing for a compiler to fuse
def embedding(tokens, weight, scale=1.0, padding_idx=None):
    """hip_ops.embedding, differentiable in the weight; the row padding_idx gets no gradient."""
    if padding_idx is not None and not -weight.shape[0] <= padding_idx < weight.shape[0]:
        raise ValueError(f"padding_idx: expected a row of {weight.shape[0]}, got {padding_idx}")
    apply = _TransformedEmbedding.apply if _transforms_active() else _Embedding.apply
    return apply(tokens, weight, scale, padding_idx)


class Embedding(nn.Embedding):
    """nn.Embedding whose rows are multiplied by `scale`, with nn.Embedding's other arguments by keyword: embedding's forward and
    gradient on the HIP device; elsewhere, in other types and with those options that embedding lacks (max_norm,
    scale_grad_by_freq, sparse), torch's."""

    def __init__(self, num_embeddings, embedding_dim, padding_idx=None, scale=1.0, **options):
        super().__init__(num_embeddings, embedding_dim, padding_idx, **options)
        self.scale = scale

    @classmethod
    def from_pretrained(cls, *args, scale=1.0, **options):
        """nn.Embedding.from_pretrained, with a scale."""
        module = super().from_pretrained(*args, **options)
        module.scale = scale
        return module

    def forward(self, tokens):
        w = self.weight
        if (w.device.type in (DEVICE, "cuda") and w.dtype in (torch.float32, torch.bfloat16) and self.max_norm is None
                and not self.scale_grad_by_freq and not self.sparse):
            return embedding(tokens, w, self.scale, self.padding_idx)
        return super().forward(tokens) * self.scale

    def extra_repr(self):
        return super().extra_repr() + f", scale={self.scale}"


@torch.compiler.disable
def token_logps(logits, labels, ignore_index=-100):
    """hip_ops.token_logps' logps, differentiable in the logits."""
    return _TokenLogps.apply(logits, labels, ignore_index)


@torch.compiler.disable
def preference_loss(logits, labels, reference, beta=0.1, kind="sigmoid", smoothing=0.0, average=False, ignore_index=-100):
    """hip_ops.preference_loss, differentiable in the logits: (loss, rewards), the rewards without a gradient."""
    return _loss(hip_ops.preference_loss, logits,
                 dict(labels=labels, reference=reference, beta=beta, kind=kind, smoothing=smoothing, average=average,
                      ignore_index=ignore_index))


@torch.compiler.disable
def policy_loss(logits, labels, old_logps, advantages, reference=None, clip=(0.2, 0.2), kl=0.0, reduction="token",
                ignore_index=-100):
    """hip_ops.policy_loss, differentiable in the logits: (loss, the KL term's mean, logps), the latter two without a
    gradient (the loss holds the KL term's)."""
    return _loss(hip_ops.policy_loss, logits,
                 dict(labels=labels, old_logps=old_logps, advantages=advantages, reference=reference, clip=clip, kl=kl,
                      reduction=reduction, ignore_index=ignore_index))
