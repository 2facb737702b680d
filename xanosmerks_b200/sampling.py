"""Sampling tokens from logits (the reference's ``sample``, sampling.py:94-158) from given random numbers.

``sample(logits, u, ...)`` chooses one token per row by temperature, top-k, top-p and min-p; the random
numbers are an input (one uniform number in [0, 1) per row), so that the same call gives the same tokens.
"""

from __future__ import annotations

import torch

from ._lib import DT_BF16, DT_F16, DT_F32, call_on, check, lib

__all__ = ["sample"]

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16}


def _per_row(v, name, dtype, rows, dev):
    """(scalar, device pointer or None) of a parameter given as a number or as a tensor with one entry per row."""
    if not isinstance(v, torch.Tensor):
        return v, None
    if v.dtype != dtype or v.dim() != 1 or v.shape[0] != rows or v.device != dev or not v.is_contiguous():
        raise ValueError(f"sample: {name} must be a number or a contiguous {dtype} tensor [{rows}] on {dev}")
    return 0, v.data_ptr()


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
           out: torch.Tensor | None = None):
    """(ids int32 [B], logprobs fp32 [B]) of ``logits`` [B, V] (fp32, fp16 or bf16, on a CUDA device; V <= 2^20).

    Tokens weigh exp((x - max) / temperature).  In descending order of x (equal logits by ascending index)
    the first ``top_k`` are kept (0: all), of those the ones before which less than ``top_p`` of their mass
    lies, of those the ones with at least ``min_p`` times the largest weight; the first is always kept.  The
    token is the first, by index, at which the kept mass exceeds ``u`` [B] (fp32 in [0, 1)) times the whole
    kept mass; the log-probability is that of its share.  Temperature 0: the first maximum.  NaN logits
    count as -inf; a row of nothing else gives token 0 with log-probability -inf.

    Each parameter is a number or a tensor with one entry per row (``top_k`` int32, the others fp32).
    ``out``: an int32 tensor [B] for the ids."""
    dt = _DT.get(logits.dtype) if isinstance(logits, torch.Tensor) else None
    if dt is None or logits.dim() != 2 or not logits.is_cuda or logits.shape[1] < 1:
        raise ValueError("sample: logits must be a 2-D fp32, fp16 or bf16 CUDA tensor")
    b, v = logits.shape
    dev = logits.device
    pitch, one = logits.stride()
    if v > 1 and one != 1:
        raise ValueError("sample: logits must have unit stride in the last dimension")
    if not isinstance(u, torch.Tensor):
        raise ValueError(f"sample: u must be a contiguous fp32 tensor [{b}] on {dev}")
    _, up = _per_row(u, "u", torch.float32, b, dev)
    t, tp = _per_row(temperature, "temperature", torch.float32, b, dev)
    k, kp = _per_row(top_k, "top_k", torch.int32, b, dev)
    if kp is None:
        k = min(max(k, 0), v)                            # (a number that C's int need not hold)
    p, pp = _per_row(top_p, "top_p", torch.float32, b, dev)
    m, mp = _per_row(min_p, "min_p", torch.float32, b, dev)
    if out is None:
        out = u.new_empty(b, dtype=torch.int32)
    else:
        _per_row(out, "out", torch.int32, b, dev)
    logp = torch.empty_like(u)
    check(call_on(dev, lib.xm_sample, logits.data_ptr(), dt, b, v, pitch if b > 1 else v, up, t, tp, k, kp, p, pp, m,
                  mp, out.data_ptr(), logp.data_ptr()), "sample")
    return out, logp
