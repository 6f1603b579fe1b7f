"""What a serving or scoring program asks of logits: log probabilities of given
tokens, the entropy, the likeliest alternatives. Batch-invariant: a row's results
have the same bits whatever other rows are beside it (csrc/bi_logprobs.hip). There
is no backward pass."""

import collections

import torch

from . import _lib
from ._paged import _call, _no_grad, _on_one_gpu

MAX_TOP = 64
_INTS = (torch.int64, torch.int32)

TokenLogprobs = collections.namedtuple("TokenLogprobs",
                                       ("logprobs", "entropy", "top_ids", "top_logprobs"))


def token_logprobs(logits, tokens, top=0):
    """Log probabilities of ``tokens`` (...) under ``logits`` (..., vocab).

    ``logits`` are float32, float16 or bfloat16, ``tokens`` int64 or int32.
    Returns a :class:`TokenLogprobs`, all but the ids float32:

    - ``logprobs`` (...): ln softmax(logits)[token]; NaN for a token that is not
      in the vocabulary;
    - ``entropy`` (...): -sum p ln p in nats; logits of -inf count for nothing;
    - ``top_ids`` (..., top) int64 and ``top_logprobs`` (..., top): the largest
      logits in descending order, ties by ascending id (a NaN counts as the
      largest). ``top`` is at most 64 and at most the vocabulary.

    Log probabilities and entropy of a row that holds a NaN or +inf, or nothing
    but -inf, are NaN.
    """
    shape = logits.shape
    if not len(shape) or logits.dtype not in _lib.DTYPE_CODES:
        raise ValueError("logits must be float32, float16 or bfloat16 of one dimension or more, got "
                         "%s of shape %s" % (logits.dtype, tuple(shape)))
    if tokens.dtype not in _INTS or tokens.shape != shape[:-1]:
        raise ValueError("tokens must be int64 or int32 of shape %s, got %s of shape %s"
                         % (tuple(shape[:-1]), tokens.dtype, tuple(tokens.shape)))
    if not 0 <= top <= MAX_TOP or top > shape[-1]:
        raise ValueError("top must be between 0 and %d and at most the vocabulary of %d, got %r"
                         % (MAX_TOP, shape[-1], top))
    if not shape[-1]:
        raise ValueError("logits of no vocabulary")
    _no_grad("token_logprobs", logits)
    if torch.compiler.is_compiling():
        from . import _ops  # noqa: F401  (registers the ops)

        return TokenLogprobs(*torch.ops.mlx_bi.token_logprobs(logits, tokens, int(top)))
    return TokenLogprobs(*_logprobs_eager(logits, tokens, int(top)))


def _logprobs_eager(logits, tokens, top):
    dev = logits.device
    _on_one_gpu("token_logprobs", dev, (tokens,))
    lead, V = tokens.shape, logits.shape[-1]
    rows = tokens.numel()
    f32 = dict(dtype=torch.float32, device=dev)
    logprobs, entropy = torch.empty(lead, **f32), torch.empty(lead, **f32)
    tops = torch.empty((*lead, top), **f32)
    ids = torch.empty((*lead, top), dtype=torch.int64, device=dev)
    if rows:
        x = logits
        if x.ndim != 2 or (x.stride(1) != 1 and V > 1):
            x = x.reshape(rows, V)
            if V > 1 and x.stride(1) != 1:
                x = x.contiguous()
        tokens = tokens.contiguous()
        _call(dev, "bi_token_logprobs", _lib.lib().bi_token_logprobs, x.data_ptr(), tokens.data_ptr(),
              logprobs.data_ptr(), entropy.data_ptr(), ids.data_ptr(), tops.data_ptr(), rows, V,
              x.stride(0), top, tokens.element_size(), _lib.DTYPE_CODES[x.dtype])
    return logprobs, entropy, ids, tops
