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
from torch.autograd.function import once_differentiable

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
def _scaled_log_softmax(logits: Tensor, temperature: float) -> Tensor:
    wide = logits if logits.dtype == torch.float64 else logits.float()
    return torch.log_softmax(wide / temperature, dim=-1)


def _nan_where(bad: Tensor, like: Tensor) -> Tensor:
    """A factor that turns values, and gradients, into NaN where ``bad``."""
    return torch.ones_like(bad, dtype=like.dtype).masked_fill(bad, math.nan)


def token_logprobs_reference(logits: Tensor, tokens: Tensor | None = None, *,
                             temperature: float = 1.0, entropy: bool = False, top: int = 0,
                             ignore_index: int = IGNORE_INDEX) -> TokenLogprobs:
    logq = _scaled_log_softmax(logits, temperature)
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
    logq = _scaled_log_softmax(logits, temperature)
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
        outside = torch.logsumexp(logq.masked_fill(listed > 0, -math.inf), dim=-1)
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


def _as_tokens(tokens: Tensor) -> Tensor:
    return (tokens if tokens.dtype == torch.int64 else tokens.long()).contiguous()


def _as_f32(t: Tensor | None) -> Tensor | None:
    return None if t is None else (t if t.dtype == torch.float32 else t.float()).contiguous()


# --------------------------------------------------------------------------------------------------
# On given logits
# --------------------------------------------------------------------------------------------------
def _empty_results(lead, device, tokens, entropy: bool, top: int):
    f32 = dict(device=device, dtype=torch.float32)
    rows = math.prod(lead)
    return (torch.empty(lead, **f32) if tokens is not None else None,
            torch.empty(lead, **f32) if entropy else None,
            torch.empty((*lead, top), **f32) if top else None,
            torch.empty((*lead, top), device=device, dtype=torch.int64) if top else None,
            torch.empty((rows, 4), **f32))


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, tokens: Tensor | None, inv_temperature: float, entropy: bool,
                top: int, ignore_index: int):
        out = _empty_results(logits.shape[:-1], logits.device, tokens, entropy, top)
        logprobs, h, top_logprobs, top_tokens, stats = out
        ext().token_logprobs_fwd(logits, tokens, inv_temperature, top, ignore_index, *out)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_tokens)
        ctx.save_for_backward(logits, tokens, top_tokens, stats)
        ctx.inv_temperature = inv_temperature
        return logprobs, h, top_logprobs, top_tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprobs, d_entropy, d_top, _):
        logits, tokens, top_tokens, stats = ctx.saved_tensors
        if d_logprobs is None and d_entropy is None and d_top is None:
            return (None,) * 6
        d = ext().token_logprobs_bwd(logits, stats, tokens, top_tokens, _as_f32(d_logprobs),
                                     _as_f32(d_entropy), _as_f32(d_top), ctx.inv_temperature)
        return (d, None, None, None, None, None)


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
    tokens = None if tokens is None else _as_tokens(tokens)
    return TokenLogprobs(*_TokenLogprobsFn.apply(logits, tokens, 1.0 / temperature, bool(entropy),
                                                 int(top), int(ignore_index)))


class _DistillationFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, teacher: Tensor, tokens: Tensor, inv_temperature: float,
                tail: bool):
        loss = torch.empty(logits.shape[:-1], device=logits.device, dtype=torch.float32)
        stats = torch.empty((loss.numel(), 4), device=logits.device, dtype=torch.float32)
        ext().distillation_fwd(logits, teacher, tokens, inv_temperature, tail, loss, stats)
        ctx.save_for_backward(logits, teacher, tokens, stats)
        ctx.inv_temperature = inv_temperature
        ctx.tail = tail
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss: Tensor):
        logits, teacher, tokens, stats = ctx.saved_tensors
        d = ext().distillation_bwd(logits, stats, teacher, tokens, _as_f32(d_loss),
                                   ctx.inv_temperature, ctx.tail)
        return d, None, None, None, None


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
    return _DistillationFn.apply(logits, _as_f32(teacher_logprobs), _as_tokens(teacher_tokens),
                                 1.0 / temperature, bool(tail))


# --------------------------------------------------------------------------------------------------
# From hidden states
# --------------------------------------------------------------------------------------------------
def _chunk_rows(tokens: int, vocab: int) -> int:
    budget = 1024 * 1024 * 1024 // (4 * max(vocab, 1))
    rows = max(128, (budget // 128) * 128)
    return min(rows, max(128, ((tokens + 127) // 128) * 128))


class _HeadChunks:
    """The logits of ``hidden @ weight.T`` chunk by chunk: fp32, because the log-probabilities of a
    bf16 logit of size 10 would be off by 0.03, in one buffer of a gigabyte that every chunk reuses."""

    def __init__(self, hidden: Tensor, weight: Tensor):
        from . import bf16_weight

        h2 = hidden.reshape(-1, hidden.shape[-1])
        self.h2 = (h2 if h2.dtype == torch.bfloat16 else h2.to(torch.bfloat16)).contiguous()
        self.w16 = bf16_weight(weight)
        self.tokens, self.vocab = self.h2.shape[0], weight.shape[0]
        self.rows = _chunk_rows(self.tokens, self.vocab)
        self.pitch = (self.vocab + 7) // 8 * 8
        n = min(self.rows, max(self.tokens, 1))
        self.buffer = torch.empty(n, self.pitch, device=self.h2.device, dtype=torch.float32)

    def __iter__(self):
        from . import matmul_nt

        for start in range(0, self.tokens, self.rows):
            stop = min(start + self.rows, self.tokens)
            logits = self.buffer[:stop - start, :self.vocab]
            matmul_nt(self.h2[start:stop], self.w16, out=logits)
            yield slice(start, stop), logits


def _head_backward(ctx, hidden: Tensor, weight: Tensor, gradient_of):
    """Gradients of ``hidden`` and ``weight`` from ``gradient_of(rows, logits, out)``, which writes
    d(loss) / d(logits) of a chunk. The chunk's gradient is rounded to bf16, the operand type of the
    two products; both accumulate in fp32, the weight's over all chunks."""
    from . import matmul_nn

    chunks = _HeadChunks(hidden, weight)
    need_dh, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
    device = chunks.h2.device
    dh = torch.empty_like(chunks.h2) if need_dh else None
    dw = torch.zeros(weight.shape, device=device, dtype=torch.float32) if need_dw else None
    grads = torch.empty(chunks.buffer.shape, device=device, dtype=torch.bfloat16)
    for rows, logits in chunks:
        d = grads[:logits.shape[0], :chunks.vocab]
        gradient_of(rows, logits, d)
        if need_dh:
            matmul_nn(d, chunks.w16, out=dh[rows])
        if need_dw:
            # one split of the token dimension: the order of the sum is fixed
            ext().gemm(d, chunks.h2[rows], dw, chunks.vocab, dw.shape[1], d.shape[0], True, True, 1,
                       True, 1.0, None, None)
    if need_dh:
        dh = dh.view(hidden.shape)
        dh = dh if dh.dtype == hidden.dtype else dh.to(hidden.dtype)
    if need_dw and dw.dtype != weight.dtype:
        dw = dw.to(weight.dtype)
    return dh, dw


def _rows_of(t: Tensor | None, rows: slice) -> Tensor | None:
    return None if t is None else t[rows]


class _LinearTokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden: Tensor, weight: Tensor, tokens: Tensor | None, inv_temperature: float,
                entropy: bool, top: int, ignore_index: int):
        lead = hidden.shape[:-1]
        out = _empty_results(lead, hidden.device, tokens, entropy, top)
        logprobs, h, top_logprobs, top_tokens, stats = out
        n = stats.shape[0]
        flat = [None if t is None else t.view(n, *t.shape[len(lead):]) for t in out[:4]] + [stats]
        t1 = None if tokens is None else tokens.view(-1)
        for rows, logits in _HeadChunks(hidden, weight):
            ext().token_logprobs_fwd(logits, _rows_of(t1, rows), inv_temperature, top, ignore_index,
                                     *(_rows_of(t, rows) for t in flat))
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_tokens)
        ctx.save_for_backward(hidden, weight, tokens, top_tokens, stats)
        ctx.inv_temperature = inv_temperature
        return logprobs, h, top_logprobs, top_tokens

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprobs, d_entropy, d_top, _):
        hidden, weight, tokens, top_tokens, stats = ctx.saved_tensors
        if d_logprobs is None and d_entropy is None and d_top is None:
            return (None,) * 7
        n = stats.shape[0]
        g = [None if t is None else _as_f32(t).view(n) for t in (d_logprobs, d_entropy)]
        g_top = None if d_top is None else _as_f32(d_top).view(n, -1)
        t1 = None if tokens is None else tokens.view(-1)
        listed = None if top_tokens is None else top_tokens.view(n, -1)

        def gradient_of(rows, logits, out):
            ext().token_logprobs_bwd(logits, stats[rows], _rows_of(t1, rows), _rows_of(listed, rows),
                                     _rows_of(g[0], rows), _rows_of(g[1], rows),
                                     _rows_of(g_top, rows), ctx.inv_temperature, out)

        dh, dw = _head_backward(ctx, hidden, weight, gradient_of)
        return dh, dw, None, None, None, None, None


class _LinearDistillationFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden: Tensor, weight: Tensor, teacher: Tensor, tokens: Tensor,
                inv_temperature: float, tail: bool):
        loss = torch.empty(hidden.shape[:-1], device=hidden.device, dtype=torch.float32)
        n = loss.numel()
        stats = torch.empty((n, 4), device=hidden.device, dtype=torch.float32)
        l1, p1, t1 = loss.view(-1), teacher.view(n, teacher.shape[-1]), tokens.view(n, tokens.shape[-1])
        for rows, logits in _HeadChunks(hidden, weight):
            ext().distillation_fwd(logits, p1[rows], t1[rows], inv_temperature, tail, l1[rows],
                                   stats[rows])
        ctx.save_for_backward(hidden, weight, p1, t1, stats)
        ctx.inv_temperature = inv_temperature
        ctx.tail = tail
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss: Tensor):
        hidden, weight, teacher, tokens, stats = ctx.saved_tensors
        g = _as_f32(d_loss).view(-1)

        def gradient_of(rows, logits, out):
            ext().distillation_bwd(logits, stats[rows], teacher[rows], tokens[rows], g[rows],
                                   ctx.inv_temperature, ctx.tail, out)

        dh, dw = _head_backward(ctx, hidden, weight, gradient_of)
        return dh, dw, None, None, None, None


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
    (V, width)``), which are made chunk by chunk and not kept; the backward pass makes them again.
    On the bf16 path (CUDA, bf16 inputs or bf16 autocast) the products run on the tensor cores with
    fp32 logits; otherwise the logits come from one ``F.linear``."""
    _check_head(hidden, weight)
    temperature = _check_temperature(temperature)
    _check_token_query(hidden.shape[:-1], weight.shape[0], hidden.device, tokens, entropy, top)
    if not _fused_head(hidden):
        return token_logprobs(torch.nn.functional.linear(hidden, weight), tokens,
                              temperature=temperature, entropy=entropy, top=top,
                              ignore_index=ignore_index)
    tokens = None if tokens is None else _as_tokens(tokens)
    return TokenLogprobs(*_LinearTokenLogprobsFn.apply(
        hidden, weight, tokens, 1.0 / temperature, bool(entropy), int(top), int(ignore_index)))


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
    return _LinearDistillationFn.apply(hidden, weight, _as_f32(teacher_logprobs),
                                       _as_tokens(teacher_tokens), 1.0 / temperature, bool(tail))
