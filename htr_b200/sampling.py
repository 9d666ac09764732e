"""Sampling of tokens from logits: temperature, top-k, top-p and min-p, from random numbers that the caller gives.

The logits are what `ops.linear` gives for an LM head (bf16, fp16 or float32); the sampler reads them once, on the GPU, and returns the
tokens there, so that a decode step with its sampling is one chain of launches and can be captured in a CUDA graph.
"""
import torch

from . import _lib, ops

_SETTINGS = (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32))


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """One token per row of logits [rows, vocab] from uniform numbers u [rows] in [0, 1).  Returns (tokens int64 [rows], logprobs float32 [rows]).

    Tokens are ordered by logit, ties by index, and weigh w = exp((logit - largest) / temperature).  Kept is the shortest of three beginnings of
    that order: the first `top_k` (0: all); the shortest one with at least `top_p` of the weight of those (1: all); all with w >= `min_p` (0: all);
    at least one token.  The token is the first, in the order of the vocabulary, at which the running weight of the kept ones exceeds u times
    their sum; its logprob is the logarithm of its share of that sum.  temperature 0 takes the largest logit (logprob 0).  Logits of -inf or NaN
    are never chosen; a row that has no other gives token -1 and logprob NaN.

    Settings are None, one number for all rows, or a CUDA tensor of one value per row (float32; int32 for top_k).  Rows may be strided.
    The choice is reproducible to the bit: weights are added as 64-bit integers, multiples of 2^-42 of the largest weight.  Borders are those of real
    numbers to within vocab * 2^-42 of it, and a token below 2^-43 of it (29.8 temperatures) is never chosen.  No gradients."""
    both = _lib.host.sample(logits, u, temperature, top_k, top_p, min_p)     # the usual case; None: whatever it does not take
    if both is not None:
        return both
    if not logits.is_cuda:
        raise _lib.HTRError("sample has no CPU path: tensors must live on a CUDA device")
    if logits.dtype not in ops._DTYPES or logits.dim() != 2:
        raise _lib.HTRError("sample: logits must be a bf16, fp16 or float32 matrix [rows, vocab]")
    rows, vocab = logits.shape
    dev = logits.device
    if vocab < 1:
        raise _lib.HTRError("sample: the vocabulary is empty")
    if vocab > 1 and logits.stride(1) != 1 or rows > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    if u.dtype != torch.float32 or u.device != dev or tuple(u.shape) != (rows,):
        raise _lib.HTRError(f"sample: u must be a float32 tensor of {rows} values on {dev}")
    settings = []
    for (name, dtype), value in zip(_SETTINGS, (temperature, top_k, top_p, min_p)):
        if value is None:
            settings.append(None)
        elif isinstance(value, torch.Tensor):
            if value.dtype != dtype or value.device != dev or tuple(value.shape) != (rows,):
                raise _lib.HTRError(f"sample: {name} must be a number or a {dtype} tensor of {rows} values on {dev}")
            settings.append(value.contiguous())
        else:
            settings.append(torch.full((rows,), value, dtype=dtype, device=dev))
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev)
    if rows == 0:
        return tokens, logprobs
    u = u.contiguous()
    with torch.cuda.device(dev):
        rc = _lib.lib.htr_sample(logits.data_ptr(), ops._DTYPES[logits.dtype], max(logits.stride(0), vocab), rows, vocab, u.data_ptr(),
                                 *[None if s is None else s.data_ptr() for s in settings], tokens.data_ptr(), logprobs.data_ptr(),
                                 torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(rc, "htr_sample")
    return tokens, logprobs
