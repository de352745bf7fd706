"""Beam search: the selection over beams and vocabulary (``csrc/beam.cu``; the cache follows with ``ops.kv4_reorder``)."""
from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _count
from ._lib import lib
from .kv4 import _call, _ints, _name

BEAM_MAX = 64
_SELECT = struct.Struct("@7Pq6i")            # BeamSelectArgs of csrc/beam.cu


def _meets_rows(at: int, size: int, rows: int, pitch: int, width: int) -> bool:
    """Whether the bytes at .. at + size meet one of the rows r pitch .. r pitch + width."""
    first = max(0, (at - width) // pitch + 1) if pitch else 0          # the first row that ends behind ``at``
    return first < rows and first * pitch < at + size and first * pitch + width > at


def beam_select(scores_out: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, logits: torch.Tensor, scores: torch.Tensor,
                vocab_size: int, finished_out: Optional[torch.Tensor] = None, finished: Optional[torch.Tensor] = None, eos: int = -1) -> None:
    """One step of a beam search for B items of K beams.

    The candidates of an item are its beams' continuations, scores[b, k] + log softmax(logits[b K + k, :vocab_size])[v]; the K best go to
    ``scores_out`` (fp32), ``tokens`` and ``parents`` (int32; the beam that is continued), all [B, K], best first, ties to the lowest
    k vocab_size + v.  ``logits`` [B K, >= vocab_size] bf16 or fp32, rows dense, any row pitch; ``scores`` fp32 [B, K].

    With ``eos``, a beam that ``finished`` (bool [B, K]) has one continuation: ``eos`` at the same score; its other candidates count -inf.
    ``finished_out`` says which of the new beams are finished: those that continue a finished one or end in ``eos``.  A beam that is not
    alive is given the score -inf (all but one of an item at the start); a beam whose score is not finite, or whose logits have no finite
    log-sum-exp (a NaN or +inf among them, or nothing but -inf), offers -inf throughout.  Outputs may not share memory with inputs (columns of
    ``logits`` behind ``vocab_size`` are no input).

    The order within a beam is that of its logits, between beams that of the sums in 64 bits, with each log-sum-exp from fp32 exponentials."""
    shape, dev = scores.shape, scores.get_device()
    if len(shape) != 2 or scores.dtype is not torch.float32 or not scores.is_contiguous():
        raise ValueError(f"scores must be a contiguous fp32 [B, K], not {scores.dtype} {tuple(shape)}")
    B, K = shape
    rows, dtype = logits.shape, logits.dtype
    if len(rows) != 2 or rows[0] != B * K or logits.get_device() != dev or (logits.stride()[1] != 1 and logits.numel()):
        raise ValueError(f"logits must be [{B * K}, at least {vocab_size}] on {_name(dev)} with dense rows, not {tuple(rows)} on {logits.device}")
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise TypeError(f"logits must be bf16 or fp32, not {dtype}")
    if not 1 <= K <= BEAM_MAX:
        raise ValueError(f"1 to {BEAM_MAX} beams, not {K}")
    if not K <= vocab_size <= rows[1] or K * vocab_size >= 2 ** 31:
        raise ValueError(f"vocabulary of {vocab_size}: at least {K} beams, at most the {rows[1]} columns, and K x V below 2^31")
    if B * K > 65535 or K * -(-vocab_size // 8192) > 2944:
        raise ValueError(f"{B} items of {K} beams over {vocab_size} tokens are too many: at most 65535 rows, and K x V up to 24 million")
    if not -1 <= eos < vocab_size:
        raise ValueError(f"eos {eos} is no token of a vocabulary of {vocab_size}")
    if finished is not None and eos < 0:
        raise ValueError("finished beams go on with eos: it is needed")
    if scores_out.dtype is not torch.float32 or scores_out.shape != shape or scores_out.get_device() != dev or not scores_out.is_contiguous():
        raise ValueError(f"scores_out must be a contiguous fp32 {tuple(shape)} on {_name(dev)}")
    so, si = scores_out.data_ptr(), scores.data_ptr()
    tk, pa = _ints(tokens, "tokens", shape, dev), _ints(parents, "parents", shape, dev)
    if tokens is None or parents is None:
        raise ValueError("tokens and parents are outputs that every call needs")
    n = B * K
    spans = [(so, 4 * n), (tk, 4 * n), (pa, 4 * n), (si, 4 * n)]
    fi = fo = 0
    for name, t in (("finished", finished), ("finished_out", finished_out)):
        if t is None:
            continue
        if t.dtype is not torch.bool or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous bool {tuple(shape)} on {_name(dev)}")
        at = t.data_ptr()
        spans.append((at, n))
        fi, fo = (at, fo) if t is finished else (fi, at)
    if n == 0:
        return
    spans.sort()
    end = 0
    for at, size in spans:
        if at < end:
            raise ValueError("outputs must not share memory with each other or with inputs")
        end = at + size
    xi, pitch, elt = logits.data_ptr(), logits.stride()[0], 2 if dtype is torch.bfloat16 else 4
    if spans[0][0] < xi + ((n - 1) * pitch + vocab_size) * elt and end > xi:
        for at, size in ((so, 4 * n), (tk, 4 * n), (pa, 4 * n), (fo, n if fo else 0)):
            if size and _meets_rows(at - xi, size, n, pitch * elt, vocab_size * elt):
                raise ValueError("outputs must not share memory with the columns of logits that are read")
    if dev >= 0:
        L = lib()
        # one call's own workspace: it lives as long as the work on this stream, and captured graphs do not share it
        work = scores.new_empty(n * -(-vocab_size // 8192) * (2 + 2 * K))
        _call(L.llmb_beam_select, "beam_select", dev,
              _SELECT.pack(so, tk, pa, fo, xi, si, fi, pitch, B, K, vocab_size, eos, 1 if dtype is torch.bfloat16 else 0, 0), work.data_ptr())
        _count(2)
        return
    x = logits[:, :vocab_size].double().view(B, K, vocab_size)
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    base = scores.double().unsqueeze(-1)
    cand = torch.where(torch.isfinite(base) & torch.isfinite(lse), base + (x - lse), torch.full_like(x, float("-inf")))
    if finished is not None:
        done = torch.full_like(x, float("-inf"))
        done[:, :, eos] = torch.where(torch.isfinite(base), base, torch.full_like(base, float("-inf"))).squeeze(-1)
        cand = torch.where(finished.unsqueeze(-1), done, cand)
    best, at = torch.sort(cand.view(B, K * vocab_size), dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    scores_out.copy_(best)
    tokens.copy_(at % vocab_size)
    parents.copy_(at // vocab_size)
    if finished_out is not None:
        f = (at % vocab_size) == eos
        finished_out.copy_(f | finished.gather(1, at // vocab_size) if finished is not None else f)
