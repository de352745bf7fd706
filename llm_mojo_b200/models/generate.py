"""Generation with a key/value cache: one pass over the prompt, then one token at a time; and beam search.

The reference generates by a whole forward pass for every token (``infer_gpt2.mojo:56-144``); ``infer_gpt2.py`` does so too unless it is asked
for a cache.  Here the keys and values of earlier tokens are kept in 4 bits (``ops.KV4Cache``), so a token costs one row of each linear
layer and a read of the cache.  Keys and values are rounded before anything attends to them, the prompt's among themselves as well: what a text
answers does not depend on how it was cut into calls.  Linear layers run in the model's storage type whatever its training precision.
"""
from __future__ import annotations

import contextlib
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from .. import ops
from ..ops import _lib


def on_device(device: torch.device):
    """Makes ``device`` the current one: the linear and normalisation operators launch to the current device's stream, whatever their tensors'."""
    return torch.cuda.device(device) if device.type == "cuda" else contextlib.nullcontext()


class CachedDecoder:
    """``slots`` texts (times ``beams``) of one model, up to ``max_len`` tokens each (the model's maximum by default).

    ``prefill`` takes the prompts, ``step`` one more token of every text; both return the logits behind the newest token.  On a GPU the steps are
    replayed from a CUDA graph after the first one (``graph=False``: launched one by one).  Both only launch; ``check`` waits and says whether
    what they answered is valid."""

    def __init__(self, model, slots: int, max_len: Optional[int] = None, beams: int = 1, graph: bool = True):
        cfg = model.config
        if model.zero is not None:
            raise ValueError("cached generation runs on a whole model, not on a ZeRO engine's shards")
        if cfg.channels % cfg.num_heads or cfg.head_size not in ops.kv4.KV4_HEAD_SIZES:
            raise ValueError(f"head size {cfg.head_size}: the cache takes {ops.kv4.KV4_HEAD_SIZES}")
        max_len = cfg.max_seq_len if max_len is None else max_len
        if not 1 <= max_len <= cfg.max_seq_len:
            raise ValueError(f"max_len {max_len}: the model has {cfg.max_seq_len} positions")
        if slots < 1 or beams < 1:
            raise ValueError(f"at least one text and one beam, not {slots} and {beams}")
        self.model, self.items, self.beams, self.max_len = model, slots, beams, max_len
        self.slots = slots * beams
        self.device = model.params.device                              # with its index, whichever is current later
        self.cache = ops.KV4Cache.empty(cfg.num_layer, self.slots, cfg.num_heads, max_len, cfg.head_size, self.device)
        self.first = self.cache.select(slice(0, None, beams))          # each item's first beam: where its prompt is read
        self.lens = torch.zeros(self.slots, dtype=torch.int32, device=self.device)
        self.pages = self.cache.own_pages() if beams > 1 else None
        self.longest = 0                                               # of any text, known on the host
        self.token = torch.zeros(self.slots, 1, dtype=torch.int32, device=self.device)
        self.graph = graph and self.device.type == "cuda"
        self._captured: Optional[Tuple[torch.cuda.CUDAGraph, torch.Tensor]] = None
        self._steps = 0

    # ------------------------------------------------------------------ one pass
    def _forward(self, tokens: torch.Tensor, cache, lens: torch.Tensor, counts: Optional[torch.Tensor], pages) -> torch.Tensor:
        """Logits [slots of ``cache``, padded vocabulary] behind the last of each row's tokens; ``lens`` moves on."""
        m, p, cfg = self.model, self.model.p, self.model.config
        S, n = tokens.shape
        C, NH, hd, rows = cfg.channels, cfg.num_heads, cfg.head_size, S * n
        e = lambda *shape, dtype=m.dtype: torch.empty(*shape, dtype=dtype, device=self.device)  # noqa: E731
        before = lens.clone()
        lens += n if counts is None else counts
        pos = (before.long().view(S, 1) + torch.arange(n, device=self.device)).clamp_(max=cfg.max_seq_len - 1)
        x = p["wte"][tokens.long().view(-1).clamp(0, cfg.vocab_size - 1)] + p["wpe"][pos.view(-1)]        # an index from outside addresses nothing
        ln, mean, rstd, qkv, att, pre, act = e(rows, C), e(rows, dtype=torch.float32), e(rows, dtype=torch.float32), e(rows, 3 * C), e(rows, C), e(rows, 4 * C), e(rows, 4 * C)
        heads = qkv.view(S, n, 3, NH, hd)
        q, k, v = heads[:, :, 0], heads[:, :, 1], heads[:, :, 2]
        mid, nxt = e(rows, C), e(rows, C)
        for l in range(cfg.num_layer):
            ops.layernorm_fwd(ln, mean, rstd, x, p["ln1w"][l], p["ln1b"][l])
            ops.matmul_fwd(qkv, ln, p["qkvw"][l], p["qkvb"][l])
            ops.kv4_append(cache, l, k, v, before, counts=counts)
            if counts is not None:
                att.zero_()                                            # rows behind a prompt's end: numbers, whatever they are
            ops.attention_kv4(att.view(S, n, NH, hd), q, cache, l, lens, counts=counts, pages=pages)
            ops.matmul_fwd(mid, att, p["attprojw"][l], p["attprojb"][l], residual=x)
            ops.layernorm_fwd(ln, mean, rstd, mid, p["ln2w"][l], p["ln2b"][l])
            ops.matmul_fwd(act, ln, p["fcw"][l], p["fcb"][l], pre_gelu=pre)
            ops.matmul_fwd(nxt, act, p["fcprojw"][l], p["fcprojb"][l], residual=mid)
            x, nxt = nxt, (x if l else e(rows, C))
        if n > 1:
            last = (counts.long() - 1 if counts is not None else torch.full((S,), n - 1, device=self.device)) + torch.arange(S, device=self.device) * n
            x = x[last]
        out, logits = e(S, C), e(S, cfg.padded_vocab_size)
        ops.layernorm_fwd(out, mean[:S], rstd[:S], x, p["lnfw"], p["lnfb"])
        ops.matmul_fwd(logits, out, p["wte"])
        return logits

    def _grow(self, n: int) -> None:
        if self.longest + n > self.max_len:
            raise ValueError(f"{self.longest} + {n} tokens: the cache has {self.max_len} places")
        self.longest += n

    @torch.no_grad()
    def prefill(self, prompts: Sequence[Sequence[int]]) -> torch.Tensor:
        """Reads one prompt per item into empty texts; returns the logits [items, padded vocabulary] behind each."""
        if self.longest:
            raise ValueError("the texts have been begun already")
        if len(prompts) != self.items or any(len(t) == 0 for t in prompts):
            raise ValueError(f"{self.items} prompts of at least one token each, not {[len(t) for t in prompts]}")
        V = self.model.config.vocab_size
        if any(not 0 <= int(t) < V for row in prompts for t in row):
            raise ValueError(f"a token is none of the {V}")
        n = max(len(t) for t in prompts)
        self._grow(n)
        toks = torch.zeros(self.items, n, dtype=torch.int32)
        for b, t in enumerate(prompts):
            toks[b, :len(t)] = torch.tensor(list(t), dtype=torch.int32)
        counts = torch.tensor([len(t) for t in prompts], dtype=torch.int32, device=self.device)
        lens = torch.zeros(self.items, dtype=torch.int32, device=self.device)
        with on_device(self.device):
            logits = self._forward(toks.to(self.device), self.first, lens, None if n * self.items == sum(len(t) for t in prompts) else counts, None)
        self.lens[::self.beams] = lens
        if self.beams > 1:                                             # every beam continues its item's prompt
            self.reorder(torch.zeros(self.items, self.beams, dtype=torch.int32, device=self.device))
        return logits

    @torch.no_grad()
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """Appends ``tokens`` (int32 [slots] or [slots, 1] on the model's device), one to every text; returns the logits behind them.  The
        result is overwritten by the next step.  Tokens outside the vocabulary, which only the device knows, count as the nearest in it."""
        if tokens.numel() != self.slots:
            raise ValueError(f"one token for each of {self.slots} texts, not {tuple(tokens.shape)}")
        self._grow(1)
        with on_device(self.device):
            return self._step(tokens)

    def _step(self, tokens: torch.Tensor) -> torch.Tensor:
        self.token.copy_(tokens.reshape(self.slots, 1))
        self._steps += 1
        if not self.graph or self._steps == 1:                         # the first step loads kernels, which a capture may not
            return self._forward(self.token, self.cache, self.lens, None, self.pages)
        if self._captured is None:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = self._forward(self.token, self.cache, self.lens, None, self.pages)
            self._captured = (g, out)
        self._captured[0].replay()
        return self._captured[1]

    def check(self) -> None:
        """Raises ``KernelError`` if a kernel's bounded wait has run out since the last look: logits made since then are not valid.  Synchronises;
        meant for places where the host waits for the device anyway."""
        dev = self.device
        if dev.type != "cuda":
            return
        status = _lib.read_status(dev)
        if status:
            _lib.status_word(dev).zero_()
            raise _lib.KernelError(f"a bounded device wait ran out while generating (status {status}): what was generated is not valid")

    def reorder(self, parents: torch.Tensor) -> None:
        """Beam j of item b becomes what beam ``parents[b, j]`` was (int32 [items, beams])."""
        if self.pages is None:
            raise ValueError("a decoder without beams has no order to change")
        ops.kv4_reorder(self.cache, self.pages, self.lens, parents)


@torch.no_grad()
def beam_search(model, prompts: Sequence[Sequence[int]], beams: int, new_tokens: int, eos: int = -1, length_penalty: float = 0.0,
                max_len: Optional[int] = None, graph: bool = True) -> List[List[Tuple[List[int], float]]]:
    """The ``beams`` best continuations of each prompt by up to ``new_tokens`` tokens: per prompt a list of (tokens, log probability), best first.
    A beam that draws ``eos`` is finished (the token is its last); beams are compared by log probability while they grow, and in the end
    by log probability / length ** ``length_penalty``."""
    if new_tokens < 1:
        raise ValueError(f"at least one new token, not {new_tokens}")
    dec = CachedDecoder(model, len(prompts), max_len, beams, graph)
    if max(len(t) for t in prompts) + new_tokens - 1 > dec.max_len:
        raise ValueError(f"prompts of {max(len(t) for t in prompts)} tokens and {new_tokens} new ones: the cache has {dec.max_len} places")
    cfg, dev, B, K = model.config, dec.device, len(prompts), beams
    if K > cfg.vocab_size:
        raise ValueError(f"{K} beams over {cfg.vocab_size} tokens")
    logits = dec.prefill(prompts).repeat_interleave(K, 0)
    scores = torch.full((B, K), float("-inf"), device=dev)
    scores[:, 0] = 0.0                                                 # the beams of an item are one text so far
    finished = torch.zeros(B, K, dtype=torch.bool, device=dev)
    new_scores, new_finished = torch.empty_like(scores), torch.empty_like(finished)
    tokens, parents = (torch.empty(B, K, dtype=torch.int32, device=dev) for _ in range(2))
    history = torch.zeros(B, K, new_tokens, dtype=torch.int32, device=dev)
    lengths = torch.zeros(B, K, dtype=torch.int32, device=dev)
    for t in range(new_tokens):
        done = finished if eos >= 0 else None
        ops.beam_select(new_scores, tokens, parents, logits, scores, cfg.vocab_size, finished_out=new_finished, finished=done, eos=eos)
        at = parents.long()
        history = history.gather(1, at.unsqueeze(-1).expand(B, K, new_tokens))
        history[:, :, t] = tokens
        lengths = lengths.gather(1, at) + (~finished.gather(1, at)).int()
        scores, new_scores, finished, new_finished = new_scores, scores, new_finished, finished
        last = t == new_tokens - 1
        if not last and eos >= 0 and t % 8 == 7:
            last = bool(finished.all())
            dec.check()
        if last:
            break
        if K > 1:
            dec.reorder(parents)
        logits = dec.step(tokens)
    dec.check()
    out = []
    for row, n, s in zip(history.tolist(), lengths.tolist(), scores.double().tolist()):
        texts = [(h[:k], v) for h, k, v in zip(row, n, s)]
        out.append(sorted(texts, key=lambda tv: -tv[1] / max(len(tv[0]), 1) ** length_penalty) if length_penalty else texts)
    return out
