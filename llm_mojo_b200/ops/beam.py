"""Beam search: the selection over beams and vocabulary (``csrc/beam.cu``; the cache follows with ``ops.kv4_reorder``)."""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import check, dtype_code, lib, ptr
from .kv4 import _count, _ints, _on

BEAM_MAX = 64


def beam_select(scores_out: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, logits: torch.Tensor, scores: torch.Tensor,
                vocab_size: int, finished_out: Optional[torch.Tensor] = None, finished: Optional[torch.Tensor] = None, eos: int = -1) -> None:
    """One step of a beam search for B items of K beams.

    The candidates of an item are its beams' continuations, scores[b, k] + log softmax(logits[b K + k, :vocab_size])[v]; the K best go to
    ``scores_out`` (fp32), ``tokens`` and ``parents`` (int32; the beam that is continued), all [B, K], best first, ties to the lowest
    k vocab_size + v.  ``logits`` [B K, >= vocab_size] bf16 or fp32, rows dense, any row pitch; ``scores`` fp32 [B, K].

    With ``eos``, a beam that ``finished`` (bool [B, K]) has one continuation: ``eos`` at the same score; its other candidates count -inf.
    ``finished_out`` says which of the new beams are finished: those that continue a finished one or end in ``eos``.  A beam that is not
    alive is given the score -inf (all but one of an item at the start); a beam whose score is not finite, or whose logits have no finite
    log-sum-exp (a NaN or +inf among them, or nothing but -inf), offers -inf throughout.  Outputs may not share memory with inputs.

    The order within a beam is that of its logits, between beams that of the sums in 64 bits, with each log-sum-exp from fp32 exponentials."""
    if scores.dim() != 2 or scores.dtype != torch.float32 or not scores.is_contiguous():
        raise ValueError(f"scores must be a contiguous fp32 [B, K], not {scores.dtype} {tuple(scores.shape)}")
    B, K = scores.shape
    dev = scores.device
    if logits.dim() != 2 or logits.shape[0] != B * K or logits.device != dev or (logits.numel() and logits.stride(1) != 1):
        raise ValueError(f"logits must be [{B * K}, at least {vocab_size}] on {dev} with dense rows, not {tuple(logits.shape)} on {logits.device}")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"logits must be bf16 or fp32, not {logits.dtype}")
    if not 1 <= K <= BEAM_MAX:
        raise ValueError(f"1 to {BEAM_MAX} beams, not {K}")
    if not K <= vocab_size <= logits.shape[1] or K * vocab_size >= 2 ** 31:
        raise ValueError(f"vocabulary of {vocab_size}: at least {K} beams, at most the {logits.shape[1]} columns, and K x V below 2^31")
    if B * K > 65535 or K * -(-vocab_size // 4096) > 10240:
        raise ValueError(f"{B} items of {K} beams over {vocab_size} tokens are too many: at most 65535 rows, and K x V up to 40 million")
    if not -1 <= eos < vocab_size:
        raise ValueError(f"eos {eos} is no token of a vocabulary of {vocab_size}")
    if finished is not None and eos < 0:
        raise ValueError("finished beams go on with eos: it is needed")
    if scores_out.dtype != torch.float32 or tuple(scores_out.shape) != (B, K) or scores_out.device != dev or not scores_out.is_contiguous():
        raise ValueError(f"scores_out must be a contiguous fp32 {(B, K)} on {dev}")
    _ints(tokens, "tokens", (B, K), dev)
    _ints(parents, "parents", (B, K), dev)
    for name, t in (("finished", finished), ("finished_out", finished_out)):
        if t is not None and (t.dtype != torch.bool or tuple(t.shape) != (B, K) or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous bool {(B, K)} on {dev}")
    outs = [t for t in (scores_out, tokens, parents, finished_out) if t is not None]
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in (*outs, scores, *([finished] if finished is not None else []))]
    if B and any(a[0] < b[1] and b[0] < a[1] for i, a in enumerate(spans[:len(outs)]) for b in spans[i + 1:]):
        raise ValueError("outputs must not share memory with each other or with inputs")
    if B == 0:
        return
    if scores.is_cuda:
        L = lib()
        with _on(dev) as stream:
            # one call's own workspace: it lives as long as the work on this stream, and captured graphs do not share it
            work = torch.empty(L.llmb_beam_select_work_bytes(B, K, vocab_size), dtype=torch.uint8, device=dev)
            check(L.llmb_beam_select(ptr(scores_out), ptr(tokens), ptr(parents), ptr(finished_out), ptr(logits), ptr(scores), ptr(finished),
                                     B, K, vocab_size, logits.stride(0), eos, dtype_code(logits), ptr(work), stream), "beam_select")
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
