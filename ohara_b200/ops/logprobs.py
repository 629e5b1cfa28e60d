"""Log-probabilities over the vocabulary and distillation from a teacher's top tokens.

``token_logprobs(logits, tokens)`` gives the log-probability of one token per row, and with
``entropy=True`` / ``top=K`` the entropy of each row and its ``K`` most likely tokens, all from one
read of the logits and with gradients for every floating-point result. ``distillation_loss(logits,
teacher_logprobs, teacher_tokens)`` is the per-row divergence from such a list of a teacher: what
``token_logprobs(teacher_logits, top=K, temperature=T)`` returns as ``top_logprobs`` and
``top_tokens`` can be stored and fed to it. The ``linear_*`` forms take the final hidden states and the
output projection instead and never keep the (tokens x vocab) logits, like
:func:`ohara_b200.ops.linear_cross_entropy`.

CUDA tensors run the kernels of ``csrc/vocab_rows.cu`` (statistics in fp32 whatever the type of the
logits; results are fp32, gradients have the type of the logits); CPU tensors run the reference
expressions below, which are also the kernels' oracle.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch import Tensor

from ._ext import ext

IGNORE_INDEX = -100
MAX_ALTERNATIVES = 128  # longest list of alternatives per row (csrc/api.h: kMaxAlternatives)

# A teacher's mass outside its list of up to this much is the rounding of the list's fp32 sum and
# counts as none (csrc/vocab_rows.cu: kLeastRest).
LEAST_REST = 1e-6

_LOGIT_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_TOKEN_TYPES = (torch.int64, torch.int32, torch.int16, torch.uint8, torch.int8)


class TokenLogprobs(NamedTuple):
    """Results of :func:`token_logprobs`; fields that were not asked for are ``None``."""

    logprobs: Tensor | None      # (...,) of the given tokens
    entropy: Tensor | None       # (...,)
    top_logprobs: Tensor | None  # (..., K) descending
    top_tokens: Tensor | None    # (..., K) int64


# --------------------------------------------------------------------------------------------------
# Reference expressions
# --------------------------------------------------------------------------------------------------
def _scaled(logits: Tensor, temperature: float) -> Tensor:
    return (logits if logits.dtype == torch.float64 else logits.float()) / temperature


def _nan_where(bad: Tensor, like: Tensor) -> Tensor:
    """A factor that turns values, and gradients, into NaN where ``bad``."""
    return torch.ones_like(bad, dtype=like.dtype).masked_fill(bad, math.nan)


def token_logprobs_reference(logits: Tensor, tokens: Tensor | None = None, *,
                             temperature: float = 1.0, entropy: bool = False, top: int = 0,
                             ignore_index: int = IGNORE_INDEX) -> TokenLogprobs:
    logq = torch.log_softmax(_scaled(logits, temperature), dim=-1)
    keep = torch.ones(logits.shape[:-1], dtype=torch.bool, device=logits.device)
    picked = h = top_logprobs = top_tokens = None
    if tokens is not None:
        tokens = tokens.long()
        keep = tokens != ignore_index
        inside = (tokens >= 0) & (tokens < logits.shape[-1])
        picked = logq.gather(-1, tokens.masked_fill(~inside, 0).unsqueeze(-1)).squeeze(-1)
        picked = (picked * _nan_where(keep & ~inside, picked)).masked_fill(~keep, 0.0)
    if entropy:
        h = -(logq.exp() * logq.masked_fill(logq == -math.inf, 0.0)).sum(dim=-1)
        h = h.masked_fill(~keep, 0.0)
    if top:
        order = torch.sort(logits.detach(), dim=-1, descending=True, stable=True).indices[..., :top]
        top_logprobs = logq.gather(-1, order).masked_fill(~keep.unsqueeze(-1), -math.inf)
        top_tokens = order.masked_fill(~keep.unsqueeze(-1), -1)
    return TokenLogprobs(picked, h, top_logprobs, top_tokens)


def distillation_loss_reference(logits: Tensor, teacher_logprobs: Tensor, teacher_tokens: Tensor, *,
                                temperature: float = 1.0, tail: bool = False) -> Tensor:
    z = _scaled(logits, temperature)
    logq = torch.log_softmax(z, dim=-1)
    tokens = teacher_tokens.long()
    present = tokens >= 0
    inside = present & (tokens < logits.shape[-1])
    at = tokens.masked_fill(~inside, 0)
    logp = teacher_logprobs.to(logq.dtype).masked_fill(~present, -math.inf)
    taught = present if tail else logp != -math.inf
    some = taught.any(dim=-1)
    if not tail:  # rows without any entry are replaced below; keep them finite on the way
        logp = torch.log_softmax(logp.masked_fill(~some.unsqueeze(-1), 0.0), dim=-1)
    p = logp.exp().masked_fill(~present, 0.0)
    used = p != 0
    picked = logq.gather(-1, at) * _nan_where(used & ~inside, logq)
    zero = torch.zeros((), dtype=logq.dtype, device=logq.device)
    loss = torch.where(used, p * (torch.where(used, logp, zero) - torch.where(used, picked, zero)),
                       zero).sum(dim=-1)
    if tail:
        listed = torch.zeros(logits.shape, dtype=torch.int32, device=logits.device)
        listed.scatter_add_(-1, at, inside.int())
        rest = 1.0 - p.sum(dim=-1)
        some_rest = (rest > LEAST_REST) | rest.isnan()
        # (from z, so that the denominator keeps its gradient where nothing is outside)
        outside = torch.logsumexp(z.masked_fill(listed > 0, -math.inf), dim=-1)
        outside = outside - torch.logsumexp(z, dim=-1)
        outside = torch.where(some_rest, outside, zero)
        rest = torch.where(some_rest, rest, zero + 1.0)
        loss = loss + torch.where(some_rest, rest * (rest.log() - outside), zero)
    return torch.where(some, loss, zero)


# --------------------------------------------------------------------------------------------------
# Argument checks
# --------------------------------------------------------------------------------------------------
def _check_temperature(temperature: float) -> float:
    temperature = float(temperature)
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must lie between 1e-6 and 1e6, got {temperature}")
    return temperature


def _check_token_query(shape, vocab: int, device, tokens: Tensor | None, entropy: bool, top: int) -> None:
    if vocab < 1:
        raise ValueError("the vocabulary is empty")
    if tokens is None and not entropy and top == 0:
        raise ValueError("nothing to compute: give tokens, entropy=True or top > 0")
    if not 0 <= top <= min(MAX_ALTERNATIVES, vocab):
        raise ValueError(f"top must be between 0 and {min(MAX_ALTERNATIVES, vocab)}, got {top}")
    if tokens is not None:
        if tokens.dtype not in _TOKEN_TYPES:
            raise TypeError(f"tokens must be integers, got {tokens.dtype}")
        if tokens.shape != shape:
            raise ValueError(f"tokens {tuple(tokens.shape)} must have one entry per row of the logits, "
                             f"{tuple(shape)}")
        if tokens.device != device:
            raise ValueError("tokens must be on the device of the logits")


def _check_teacher(shape, device, teacher_logprobs: Tensor, teacher_tokens: Tensor) -> None:
    if teacher_tokens.dtype not in _TOKEN_TYPES:
        raise TypeError(f"teacher_tokens must be integers, got {teacher_tokens.dtype}")
    if not teacher_logprobs.is_floating_point():
        raise TypeError("teacher_logprobs must be floating point")
    if teacher_logprobs.shape != teacher_tokens.shape or teacher_tokens.shape[:-1] != shape \
            or teacher_tokens.dim() != len(shape) + 1:
        raise ValueError(
            f"teacher_logprobs {tuple(teacher_logprobs.shape)} and teacher_tokens "
            f"{tuple(teacher_tokens.shape)} must both be {tuple(shape)} + (entries,)")
    if not 1 <= teacher_tokens.shape[-1] <= MAX_ALTERNATIVES:
        raise ValueError(f"a teacher's list has 1 to {MAX_ALTERNATIVES} entries, got "
                         f"{teacher_tokens.shape[-1]}")
    if teacher_logprobs.requires_grad:
        raise ValueError("the teacher's log-probabilities are constants here: detach them")
    if teacher_logprobs.device != device or teacher_tokens.device != device:
        raise ValueError("the teacher's list must be on the device of the logits")


def _check_logits(logits: Tensor) -> None:
    if logits.dim() < 1:
        raise ValueError("logits need a vocabulary dimension")
    if logits.is_cuda and logits.dtype not in _LOGIT_TYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if not logits.is_floating_point():
        raise TypeError(f"logits must be floating point, got {logits.dtype}")


def _results(found: list, tokens: Tensor | None, entropy: bool, top: int) -> TokenLogprobs:
    """The extension returns what was asked for, in order."""
    each = iter(found)
    return TokenLogprobs(None if tokens is None else next(each), next(each) if entropy else None,
                         next(each) if top else None, next(each) if top else None)


# --------------------------------------------------------------------------------------------------
# On given logits
# --------------------------------------------------------------------------------------------------
def token_logprobs(logits: Tensor, tokens: Tensor | None = None, *, temperature: float = 1.0,
                   entropy: bool = False, top: int = 0,
                   ignore_index: int = IGNORE_INDEX) -> TokenLogprobs:
    """Log-probabilities under ``softmax(logits / temperature)`` of ``tokens`` (one per row of
    ``logits (..., V)``), and on demand the entropy of every row and its ``top`` most likely tokens
    in order (equal logits by their index; NaN counts as largest).

    Rows whose token is ``ignore_index`` are padding: they are not read, their log-probability and
    entropy are 0, their list is empty (token -1, log-probability -inf) and their gradient is 0.
    A token outside the vocabulary gets NaN, and so does a row that holds NaN, +inf or nothing but
    -inf; a logit of -inf in any other row is a token of probability 0. Everything floating point is
    differentiable (once) with respect to the logits; a row whose incoming gradients are all 0 gets
    a gradient of 0."""
    _check_logits(logits)
    temperature = _check_temperature(temperature)
    _check_token_query(logits.shape[:-1], logits.shape[-1], logits.device, tokens, entropy, top)
    if not logits.is_cuda:
        return token_logprobs_reference(logits, tokens, temperature=temperature, entropy=entropy,
                                        top=top, ignore_index=ignore_index)
    found = ext().token_logprobs(logits, tokens, 1.0 / temperature, bool(entropy), top, ignore_index)
    return _results(found, tokens, entropy, top)


def distillation_loss(logits: Tensor, teacher_logprobs: Tensor, teacher_tokens: Tensor, *,
                      temperature: float = 1.0, tail: bool = False) -> Tensor:
    """Per-row divergence ``sum_k p_k (log p_k - log q[token_k])`` of the student's
    ``q = softmax(logits / temperature)`` from a teacher that is known by a list of tokens
    (``teacher_logprobs`` and ``teacher_tokens`` are ``(..., K)``); fp32, shape ``(...)``, not
    multiplied by ``temperature ** 2``.

    ``tail=False`` renormalises the list (``p = softmax(teacher_logprobs)``, so logits divided by the
    temperature serve as well); ``tail=True`` takes ``p = exp(teacher_logprobs)`` as it is and compares
    the mass outside the list, ``1 - sum p``, with the student's mass outside it as one more token
    (up to 1e-6 of it is taken for rounding and dropped). ``teacher_logprobs`` belong to the same
    temperature.

    Entries with a negative token are left out, and a row without any entry (with ``tail=False``:
    none above -inf) is not read: loss 0, gradient 0. A token that is listed twice counts with both
    of its probabilities. A listed token outside the vocabulary, or a row of logits without a
    distribution, gives NaN; a listed token that the student rules out (-inf) gives +inf."""
    _check_logits(logits)
    temperature = _check_temperature(temperature)
    _check_teacher(logits.shape[:-1], logits.device, teacher_logprobs, teacher_tokens)
    if not logits.is_cuda:
        return distillation_loss_reference(logits, teacher_logprobs, teacher_tokens,
                                           temperature=temperature, tail=tail)
    return ext().distillation_loss(logits, teacher_logprobs, teacher_tokens, 1.0 / temperature,
                                   bool(tail))


# --------------------------------------------------------------------------------------------------
# From hidden states
# --------------------------------------------------------------------------------------------------
# The gradient with respect to the logits (bf16), and with a top list the fp32 logits, exist for as many
# rows at a time as fill this: enough for the products to run at full rate, small next to a training
# step's activations.
_CHUNK_BYTES = 1024 * 1024 * 1024


def _check_head(hidden: Tensor, weight: Tensor) -> None:
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden {tuple(hidden.shape)} and weight {tuple(weight.shape)} must be "
                         "(..., width) and (vocab, width)")
    if hidden.device != weight.device:
        raise ValueError("hidden and weight must be on the same device")
    if not hidden.is_floating_point() or not weight.is_floating_point():
        raise TypeError("hidden and weight must be floating point")


def _fused_head(hidden: Tensor) -> bool:
    from . import fast_path

    return fast_path(hidden) and hidden.shape[-1] % 8 == 0 and hidden.shape[-1] > 0


def linear_token_logprobs(hidden: Tensor, weight: Tensor, tokens: Tensor | None = None, *,
                          temperature: float = 1.0, entropy: bool = False, top: int = 0,
                          ignore_index: int = IGNORE_INDEX) -> TokenLogprobs:
    """:func:`token_logprobs` of the logits ``hidden @ weight.T`` (``hidden (..., width)``, ``weight
    (V, width)``), which are not kept; the backward pass makes them again. On the bf16 path (CUDA, bf16
    inputs or bf16 autocast, a width that is a multiple of 8) the statistics are taken from the fp32
    accumulators of the tensor-core product, and with ``top`` from a gigabyte of fp32 logits at a time;
    otherwise the logits come from one ``F.linear``."""
    _check_head(hidden, weight)
    temperature = _check_temperature(temperature)
    _check_token_query(hidden.shape[:-1], weight.shape[0], hidden.device, tokens, entropy, top)
    if not _fused_head(hidden):
        return token_logprobs(torch.nn.functional.linear(hidden, weight), tokens,
                              temperature=temperature, entropy=entropy, top=top,
                              ignore_index=ignore_index)
    from . import bf16_weight

    found = ext().linear_token_logprobs(hidden, weight, bf16_weight(weight), tokens, 1.0 / temperature,
                                        bool(entropy), top, ignore_index, _CHUNK_BYTES)
    return _results(found, tokens, entropy, top)


def linear_distillation_loss(hidden: Tensor, weight: Tensor, teacher_logprobs: Tensor,
                             teacher_tokens: Tensor, *, temperature: float = 1.0,
                             tail: bool = False) -> Tensor:
    """:func:`distillation_loss` of the logits ``hidden @ weight.T``, which are not kept (see
    :func:`linear_token_logprobs`)."""
    _check_head(hidden, weight)
    temperature = _check_temperature(temperature)
    _check_teacher(hidden.shape[:-1], hidden.device, teacher_logprobs, teacher_tokens)
    if weight.shape[0] < 1:
        raise ValueError("the vocabulary is empty")
    if not _fused_head(hidden):
        return distillation_loss(torch.nn.functional.linear(hidden, weight), teacher_logprobs,
                                 teacher_tokens, temperature=temperature, tail=tail)
    from . import bf16_weight

    return ext().linear_distillation_loss(hidden, weight, bf16_weight(weight), teacher_logprobs,
                                          teacher_tokens, 1.0 / temperature, bool(tail), _CHUNK_BYTES)
