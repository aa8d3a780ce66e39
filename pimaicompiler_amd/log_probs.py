"""What a decoder's or a scorer's logits say about tokens: log probabilities, entropy, and the most likely alternatives.

The reference's decoding loops end in an argmax over the logits (aten_ops_executor.cpp:520-560); beam search, sampling and scoring of given
texts need the probabilities themselves."""
import torch

from . import _lib as L
from .mx4 import _CODES, _require, _rows_of
from .ops import NNRuntimeException, _check, _ensure_init, _Launch, _native, _require_no_gradient, _result

TOP_MOST = 32


def token_log_probs(logits, tokens=None, top=0, stream=None):
    """logits [.., V] in fp16, bf16 or fp32, tokens [..] int64 or int32 (or None) ->

        logp [..] fp32       log softmax(logits)[token]; 0 where the token is negative (padding), NaN where it is V or more; None without tokens
        entropy [..] fp32    -sum p log p, masked entries (-inf) counting nothing

    and, where `top` (at most 32) is not 0,

        top_logp [.., top] fp32, top_ids [.., top] int32    the most likely tokens, equal ones by their index

    One pass over the logits, statistics in fp32.  A row of -inf alone leaves every token impossible: log probabilities -inf, entropy 0.  A row
    with a NaN or +inf has no distribution: NaN throughout, and -1 for its alternatives."""
    out = _native().fast_log_probs(logits, tokens, top) if stream is None else None
    if out is not None:
        return _result(out)
    _require("logits", logits, tuple(_CODES))
    _require_no_gradient(logits)
    if logits.dim() < 1 or logits.size(-1) < 1:
        raise NNRuntimeException("logits must have at least one dimension, the last of at least one value")
    V, lead = logits.size(-1), logits.shape[:-1]
    if not isinstance(top, int) or not 0 <= top <= min(TOP_MOST, V):
        raise NNRuntimeException(f"top={top!r} must be a whole number in [0, {min(TOP_MOST, V)}]")
    if tokens is not None:
        _require("tokens", tokens, (torch.int64, torch.int32))
        if tokens.shape != lead or tokens.device != logits.device:
            raise NNRuntimeException(f"tokens must be {tuple(lead)} on {logits.device}, got {tuple(tokens.shape)} on {tokens.device}")
    _ensure_init(logits)
    with _Launch(logits.device, stream, logits, tokens) as handle:
        x, ld = _rows_of(logits)
        if tokens is not None:
            tokens = tokens.contiguous()
        new = lambda *shape, dtype=torch.float32: torch.empty((*lead, *shape), dtype=dtype, device=logits.device)  # noqa: E731
        logp, entropy = new() if tokens is not None else None, new()
        top_logp, top_ids = (new(top), new(top, dtype=torch.int32)) if top else (None, None)
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        _check(L.load().pimhip_token_log_probs(x.data_ptr(), _CODES[x.dtype], ld, x.size(0), V, ptr(tokens),
                                               int(tokens is not None and tokens.dtype == torch.int64), top, ptr(logp), ptr(entropy), ptr(top_logp),
                                               ptr(top_ids), handle))
    return (logp, entropy, top_logp, top_ids) if top else (logp, entropy)
