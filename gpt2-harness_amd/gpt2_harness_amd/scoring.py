"""Scores of given tokens under a model's logits, on the GPU.

:func:`token_logprobs` reads each row of logits once and returns the log
probability of the row's token, the entropy of the row and its most probable
alternatives; where autograd follows the logits, one more pass gives their
gradient. The reference computes the first of these inside ``F.cross_entropy``
(``src/transformer_internals/model.py:593-598``, ``quantization.py:262-319``),
which writes the whole ``log_softmax`` to memory on the way; entropy and
alternatives are an extension. :func:`score_tokens` applies it to a model and
token windows. :func:`~gpt2_harness_amd.sampling.generate` (``scores=``) and
:func:`~gpt2_harness_amd.quantization.perplexity_with_error_bars`
(``token_scores=``) use it as well.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["MAX_TOP", "TokenScores", "score_tokens", "token_logprobs"]

#: the most alternatives :func:`token_logprobs` returns
MAX_TOP = 64


class TokenScores(NamedTuple):
    """What :func:`token_logprobs` returns, one entry a row of logits."""

    logprob: torch.Tensor  #: fp32 log probability of the given token
    entropy: torch.Tensor  #: fp32 entropy of the row, in nats
    top_ids: torch.Tensor | None  #: int64 ``(..., top)`` most probable tokens, best first
    top_logprobs: torch.Tensor | None  #: fp32 ``(..., top)`` their log probabilities


def _rows_of(logits: torch.Tensor) -> tuple[torch.Tensor, int, int, int, int]:
    """``logits`` as ``batch`` times ``rows`` rows at two strides, copied only
    where its layout has no such form (or the vocabulary is not consecutive)."""
    shape, stride = logits.shape, logits.stride()
    if shape[-1] > 1 and stride[-1] != 1:
        logits = logits.contiguous()
        stride = logits.stride()
    n = len(shape)
    if n == 2:
        return logits, 1, shape[0], 0, stride[0]
    if n == 3:
        return logits, shape[0], shape[1], stride[0], stride[1]
    if n == 1:
        return logits, 1, 1, 0, shape[0]
    flat = logits.reshape(-1, shape[-1])
    return flat, 1, flat.shape[0], 0, flat.stride(0)


def _forward(logits, tokens, top, ignore_index, stats):
    """The library call; ``stats``: whether the gradient's two floats a row are wanted."""
    dev = logits.get_device()
    if dev != torch._C._cuda_getDevice():  # launches go to the current device
        with torch.cuda.device(dev):
            return _forward(logits, tokens, top, ignore_index, stats)
    x, batch, rows, sb, sr = _rows_of(logits)
    lead, V, n, f32 = tokens.shape, x.shape[-1], batch * rows, torch.float32
    L = _lib.lib()
    code = _lib.F32 if x.dtype is f32 else _lib.BF16
    logprob, entropy = x.new_empty(lead, dtype=f32), x.new_empty(lead, dtype=f32)
    st = x.new_empty((n, 2), dtype=f32) if stats else None
    ids = values = ws = None
    if top:
        ids, values = tokens.new_empty((*lead, top)), x.new_empty((*lead, top), dtype=f32)
    ws_bytes = L.tiq_token_logprobs_workspace(code, n, V, top)
    if ws_bytes:
        ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    rc = L.tiq_token_logprobs(x.data_ptr(), code, batch, rows, sb, sr, V, tokens.data_ptr(), ignore_index, top,
                              logprob.data_ptr(), entropy.data_ptr(), None if st is None else st.data_ptr(),
                              None if ids is None else ids.data_ptr(), None if values is None else values.data_ptr(),
                              None if ws is None else ws.data_ptr(), ws_bytes, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc, f"token_logprobs ({n} rows of {V}, top={top})")
    return logprob, entropy, st, ids, values


def _as_weight(t: torch.Tensor | None) -> torch.Tensor | None:
    """A gradient as contiguous fp32."""
    if t is None or (t.dtype is torch.float32 and t.is_contiguous()):
        return t
    return t.to(torch.float32).contiguous()


class _TokenLogprobs(torch.autograd.Function):
    # An eager step waits for this class's Python and autograd's own, not for the kernels
    # (96 rows of 50257: 18 us of kernels, 116 us a step with the usual helpers around
    # forward and backward): no device guards (autograd sets the device of a node's
    # thread), the refusal of a second order by the grad mode it would run under.
    @staticmethod
    def forward(ctx, logits, tokens, top, ignore_index):
        logprob, entropy, stats, ids, values = _forward(logits, tokens, top, ignore_index, True)
        ctx.set_materialize_grads(False)
        ctx.stats, ctx.options = stats, (top, ignore_index)
        if top:
            ctx.mark_non_differentiable(ids)
            ctx.save_for_backward(logits, tokens, entropy, ids)
            return logprob, entropy, ids, values
        ctx.save_for_backward(logits, tokens, entropy)
        return logprob, entropy

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, _=None, g_top=None):
        if torch.is_grad_enabled():
            raise RuntimeError("token_logprobs has no second derivative: call backward without create_graph")
        if g_logprob is None and g_entropy is None and g_top is None:
            return None, None, None, None
        logits, tokens, entropy, *ids = ctx.saved_tensors
        top, ignore_index = ctx.options
        gl, gh, gt = _as_weight(g_logprob), _as_weight(g_entropy), _as_weight(g_top)
        x, batch, rows, sb, sr = _rows_of(logits)
        grad = logits.new_empty(logits.shape)
        rc = _lib.lib().tiq_token_logprobs_grad(
            x.data_ptr(), _lib.F32 if x.dtype is torch.float32 else _lib.BF16, batch, rows, sb, sr, x.shape[-1],
            tokens.data_ptr(), ignore_index, ctx.stats.data_ptr(), entropy.data_ptr(),
            None if gl is None else gl.data_ptr(), None if gh is None else gh.data_ptr(), top,
            ids[0].data_ptr() if ids else None, None if gt is None else gt.data_ptr(), grad.data_ptr(),
            _lib.stream_of(x))
        if rc:
            _lib.check(rc, "token_logprobs gradient")
        return grad, None, None, None


def token_logprobs(
    logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, ignore_index: int = -100
) -> TokenScores:
    """Log probabilities of given tokens, with entropy and top alternatives.

    Args:
        logits: ``(..., V)`` fp32 or bf16 on the GPU; a slice such as
            ``logits[:, :-1]`` is read in place through its strides.
        tokens: ``(...)`` integer token ids on the same device. A token equal to
            ``ignore_index`` has log probability 0 and sends no gradient; any other
            outside ``[0, V)`` has log probability NaN.
        top: how many alternatives to return, at most ``min(V, 64)``; they are the
            largest logits in falling order, of equal ones the lower id first.
        ignore_index: as in ``F.cross_entropy``.

    Returns:
        :class:`TokenScores`: ``logprob`` and ``entropy`` of shape ``(...)``, and
        with ``top`` the alternatives ``(..., top)`` (else ``None``), all fp32 but
        the ids. ``logprob``, ``entropy`` and ``top_logprobs`` carry gradients to
        ``logits`` (first order; ``top_ids`` is a choice and carries none).

    ``-inf`` logits are probabilities of 0. A row that holds NaN or ``+inf``, or
    nothing above ``-inf``, has NaN scores. A training step captured into a graph takes
    its gradients with ``torch.autograd.grad``, or lets no eager step's results of the
    same leaves live meanwhile: autograd would accumulate into them on the eager
    step's stream, which a capture does not survive.
    """
    if not (isinstance(logits, torch.Tensor) and isinstance(tokens, torch.Tensor) and logits.is_cuda
            and tokens.is_cuda):
        _lib.require_gpu(logits, "logits")
        _lib.require_gpu(tokens, "tokens")
    if logits.dtype is not torch.float32 and logits.dtype is not torch.bfloat16:
        raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    if tokens.dtype is not torch.int64:
        if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype is torch.bool:
            raise TypeError(f"tokens must be integers, got {tokens.dtype}")
        tokens = tokens.to(torch.int64)
    shape = logits.shape
    if not shape or shape[:-1] != tokens.shape:
        raise ValueError(f"logits {tuple(shape)} and tokens {tuple(tokens.shape)} do not match")
    if logits.get_device() != tokens.get_device():
        raise RuntimeError(f"logits are on {logits.device}, tokens on {tokens.device}")
    V = shape[-1]
    if V < 1:
        raise ValueError("logits hold no vocabulary")
    if not 0 <= top <= min(V, MAX_TOP):
        raise ValueError(f"top must be in [0, {min(V, MAX_TOP)}], got {top}")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(logits).tangent is not None:
        raise RuntimeError("token_logprobs has no forward-mode derivative")
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        out = _TokenLogprobs.apply(logits, tokens, top, ignore_index)
        return TokenScores(*out) if top else TokenScores(*out, None, None)
    logprob, entropy, _, ids, values = _forward(logits, tokens, top, ignore_index, False)
    return TokenScores(logprob, entropy, ids, values)


@torch.no_grad()
def score_tokens(model, idx: torch.Tensor, targets: torch.Tensor | None = None, *, top: int = 0) -> TokenScores:
    """:func:`token_logprobs` of token windows under ``model``.

    Without ``targets`` every token of ``idx`` ``(B, T)`` after the first is scored
    given those before it: ``(B, T - 1)`` scores. With ``targets`` ``(B, T)`` (as
    ``GPT.forward`` takes them, ``-100`` ignored) each position's target is:
    ``(B, T)`` scores.
    """
    if targets is not None and targets.shape != idx.shape:
        raise ValueError(f"idx {tuple(idx.shape)} and targets {tuple(targets.shape)} do not match")
    was_training = model.training
    model.eval()
    try:
        logits = model(idx)["logits"]
    finally:
        model.train(was_training)
    if targets is None:
        return token_logprobs(logits[:, :-1], idx[:, 1:], top=top)
    return token_logprobs(logits, targets, top=top)
