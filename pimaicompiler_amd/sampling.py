"""The next token drawn from a decoder's logits, by a random number that the caller gives.

The reference's decoding loops end in an argmax over the logits (aten_ops_executor.cpp:520-560); a served request sets a temperature and how much
of the distribution may be drawn from."""
import ctypes
import math

import torch

from . import _lib as L
from .mx4 import _CODES, _require, _rows_of
from .ops import NNRuntimeException, _check, _ensure_init, _Launch, _native, _require_no_gradient, _result

VOCAB_MOST = 1 << 21


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, stream=None):
    """logits [.., V] in fp16, bf16 or fp32 and uniform [..] fp32, a number in [0, 1) for each row ->

        tokens [..] int64    the token drawn
        logp [..] fp32       the logarithm of its probability among those that could have been drawn

    w = exp((x - max x) / temperature).  Of a row's tokens in falling order, equal ones by their index: the first top_k stay (0: all); of them those before
    which less than top_p of their sum has been reached (1: all), the first always; of them those with w >= min_p, that is min_p times the largest
    probability (0: all).  The token is the first, in the order of indices, at which the running sum of w over what stayed exceeds uniform times
    the whole.  temperature 0: the most likely token.

    temperature, top_p and min_p are numbers or fp32 tensors [..], top_k a whole number or an int32 tensor [..].  Weights are worked out and summed in
    64 bits, as whole numbers of 2^-45 of the largest for up to 2^17 tokens, of 2^-41 for 2^21: shares are good to 2^-36 and half such a number for each token,
    and one that meets a border to within 2^-36 is taken to meet it.  Equal calls give equal results.
    A row of -inf alone gives token -1 and logp -inf; one with a NaN or +inf -1 and NaN, and so does a tensor's temperature that is negative,
    infinite or NaN, or a NaN in its other settings or its number.  Numbers outside of [0, 1) count as the nearest in it, 0 or 1 - 2^-24."""
    out = _native().fast_sample_tokens(logits, uniform, temperature, top_k, top_p, min_p) if stream is None else None
    if out is not None:
        return _result(out)
    _require("logits", logits, tuple(_CODES))
    _require("uniform", uniform, (torch.float32,))
    _require_no_gradient(logits, uniform)
    if logits.dim() < 1 or not 1 <= logits.size(-1) <= VOCAB_MOST:
        raise NNRuntimeException(f"logits must have at least one dimension, the last of 1 to {VOCAB_MOST} values")
    V, lead = logits.size(-1), logits.shape[:-1]
    if uniform.shape != lead or uniform.device != logits.device:
        raise NNRuntimeException(f"uniform must be {tuple(lead)} on {logits.device}, got {tuple(uniform.shape)} on {uniform.device}")
    settings, each = L.SampleSettings(), []
    for name, v, dtype, plural in (("temperature", temperature, torch.float32, "temperatures"), ("top_k", top_k, torch.int32, "top_ks"),
                                   ("top_p", top_p, torch.float32, "top_ps"), ("min_p", min_p, torch.float32, "min_ps")):
        if isinstance(v, torch.Tensor):
            _require(name, v, (dtype,))
            _require_no_gradient(v)
            if v.shape != lead or v.device != logits.device:
                raise NNRuntimeException(f"{name} must be {tuple(lead)} on {logits.device}, got {tuple(v.shape)} on {v.device}")
            each.append((plural, v))
        elif dtype == torch.int32:
            if not isinstance(v, int) or not 0 <= v <= 2**31 - 1:
                raise NNRuntimeException(f"{name}={v!r} must be a whole number from 0 on")
            settings.top_k = v
        else:
            if not isinstance(v, (int, float)) or not math.isfinite(v) or v < 0 or name == "temperature" and v > 3.4e38 or name != "temperature" and v > 1:
                raise NNRuntimeException(f"{name}={v!r} must be {'0 or more' if name == 'temperature' else 'in [0, 1]'}")
            setattr(settings, name, v)
    _ensure_init(logits)
    with _Launch(logits.device, stream, logits, uniform, *(v for _, v in each)) as handle:
        x, ld = _rows_of(logits)
        uniform = uniform.contiguous()
        each = [(name, v.contiguous()) for name, v in each]
        for name, v in each:
            setattr(settings, name, v.data_ptr())
        tokens = torch.empty(lead, dtype=torch.int64, device=logits.device)
        logp = torch.empty(lead, dtype=torch.float32, device=logits.device)
        lib, n = L.load(), ctypes.c_uint64()
        _check(lib.pimhip_sample_workspace_bytes(_CODES[x.dtype], x.size(0), V, ctypes.byref(settings), ctypes.byref(n)))
        workspace = torch.empty(n.value, dtype=torch.uint8, device=logits.device) if n.value else None
        _check(lib.pimhip_sample_tokens(x.data_ptr(), _CODES[x.dtype], ld, x.size(0), V, uniform.data_ptr(), ctypes.byref(settings), tokens.data_ptr(),
                                        logp.data_ptr(), workspace.data_ptr() if workspace is not None else None, handle))
    return tokens, logp
