"""Sampling tokens from logits (the reference's ``sample``, sampling.py:94-158) from given random numbers, and
the log-probabilities of given tokens.

``sample(logits, u, ...)`` chooses one token per row by temperature, top-k, top-p and min-p; the random
numbers are an input (one uniform number in [0, 1) per row), so that the same call gives the same tokens.
``logprobs(logits, tokens, ...)`` scores tokens: their log-probability and rank, the entropy of each row and
its largest alternatives.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from ._lib import DT_BF16, DT_F16, DT_F32, call_on, check, lib

__all__ = ["sample", "logprobs", "TokenLogprobs", "MAX_TOP"]

MAX_TOP = 64   # alternatives of a row

_DT = {torch.float32: DT_F32, torch.bfloat16: DT_BF16, torch.float16: DT_F16}


def _per_row(v, name, dtype, rows, dev, what="sample"):
    """(scalar, device pointer or None) of a parameter given as a number or as a tensor with one entry per row."""
    if not isinstance(v, torch.Tensor):
        return v, None
    if v.dtype != dtype or v.dim() != 1 or v.shape[0] != rows or v.device != dev or not v.is_contiguous():
        raise ValueError(f"{what}: {name} must be a number or a contiguous {dtype} tensor [{rows}] on {dev}")
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


@functools.lru_cache(maxsize=64)
def _empty_on(dev):
    """What makes new fp32 and int32 tensors on a device (new_empty of one that is there takes half the time of empty)."""
    return (torch.empty(0, dtype=torch.float32, device=dev).new_empty, torch.empty(0, dtype=torch.int32, device=dev).new_empty)


class TokenLogprobs(NamedTuple):
    """What :func:`logprobs` gives of B rows (on the logits' device)."""

    logprob: torch.Tensor                    # fp32 [B]: of the given tokens
    entropy: torch.Tensor                    # fp32 [B], in nats
    rank: torch.Tensor                       # int32 [B]: tokens before the given one in descending order
    top_ids: torch.Tensor | None             # int32 [B, top], in descending order
    top_logprobs: torch.Tensor | None        # fp32 [B, top]


def logprobs(logits: torch.Tensor, tokens: torch.Tensor, temperature=1.0, top: int = 0) -> TokenLogprobs:
    """Log-probabilities of ``tokens`` [B] (int32 or int64) under softmax(``logits`` / temperature), ``logits`` [B, V]
    (fp32, fp16 or bf16, on a CUDA device; V <= 2^20), with the entropy of each row, the rank of each token (how many
    have a larger logit, or the same one at a lower index) and the ``top`` (up to 64) largest logits (equal ones by
    ascending index).

    ``temperature``: a number, or an fp32 tensor [B]; 0: the first maximum has log-probability 0, the others -inf.  A token
    outside the vocabulary (-1 for padding, say) gives NaN and rank -1.  NaN logits count as -inf, which have
    log-probability -inf; a row of nothing else has entropy 0.  Logits of +inf share the mass.  Results are good to 2^-16 of
    themselves, those of confident rows too.  Rows that lie on one another (``row.expand(B, -1)``: tokens under one row) are
    copied.  With alternatives, rows of equal or rising logits throughout are read once for each of them."""
    dt = _DT.get(logits.dtype) if isinstance(logits, torch.Tensor) else None
    if dt is None or logits.dim() != 2 or not logits.is_cuda or logits.shape[1] < 1:
        raise ValueError("logprobs: logits must be a 2-D fp32, fp16 or bf16 CUDA tensor")
    b, v = logits.shape
    dev = logits.device
    pitch, one = logits.stride()
    if v > 1 and one != 1:
        raise ValueError("logprobs: logits must have unit stride in the last dimension")
    if b > 1 and pitch < v:                            # rows that lie on one another (expanded: tokens under one row)
        logits, pitch = logits.contiguous(), v
    if (not isinstance(tokens, torch.Tensor) or tokens.dtype not in (torch.int32, torch.int64) or tokens.dim() != 1
            or tokens.shape[0] != b or tokens.device != dev or not tokens.is_contiguous()):
        raise ValueError(f"logprobs: tokens must be a contiguous int32 or int64 tensor [{b}] on {dev}")
    if not 0 <= top <= min(MAX_TOP, v):
        raise ValueError(f"logprobs: {top} alternatives (0 to {min(MAX_TOP, v)})")
    t, tp = _per_row(temperature, "temperature", torch.float32, b, dev, "logprobs")
    reals, ints = _empty_on(dev)
    lp, ent, rank = reals(b), reals(b), ints(b)
    ids = tops = None
    if top:
        ids, tops = ints((b, top)), reals((b, top))
    check(call_on(dev, lib.xm_logprobs, logits.data_ptr(), dt, b, v, pitch if b > 1 else v, tokens.data_ptr(),
                  4 if tokens.dtype is torch.int32 else 8, t, tp, top, lp.data_ptr(), ent.data_ptr(), rank.data_ptr(),
                  ids.data_ptr() if top else None, tops.data_ptr() if top else None), "logprobs")
    return TokenLogprobs(lp, ent, rank, ids, tops)
