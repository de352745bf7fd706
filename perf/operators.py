"""Generation with a key/value cache in 4 bits, and beam search over it: the operators, their plain forms and the sizes that count.

A cache holds the keys and values of S sequences ("slots") for L layers in the NVFP4 form of this framework's low-precision products:
e2m1 values, two to a byte (the first in the low nibble), and one e4m3 scale for every 16 of them along the head, times one power of two
for all keys and one for all values (``UNIT`` here).  Four uint8 tensors: codes [L, S, H, T, head / 2] and scales [L, S, H, T, head / 16] of keys
and of values; T is a multiple of the 64 tokens of a page.  ``pages`` [S, T / 64] names for each slot and page the slot in whose place the
page lies (beams share the pages that they have in common); without it every page lies in its own slot.

* ``append``   new keys and values are rounded to that form and written behind the tokens that a slot has; what they stand for is read back
* ``attend``   attention of a slot's newest tokens (one while generating, many for a prompt) over the cache, causal among themselves
* ``select``   beam search: the K best of the K x V continuations of each prompt, ties to the lowest beam and token
* ``reorder``  the cache follows the selection: page tables and lengths are permuted, the page that is being filled is copied

Sizes are those of the models of ``config.py``: heads of 64 (GPT-2 ladder and GPT-3 ladder up to c1024), 80, 96 and 128, 6 to 32 of them,
up to 48 layers and a vocabulary of 50257 in rows of 50304; caches go on to 32768 tokens and to heads that share keys, as generic sizes.
"""
import math
import random

import torch

own = False

PAGE = 64
UNIT = 2.0 ** -4
VOCAB, VOCAB_ROW = 50257, 50304
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _attend(name, B, heads, kv_heads, head, longest, new=1, dtype="bf16", pages=False):
    return {"name": name, "kind": "attend", "B": B, "heads": heads, "kv_heads": kv_heads, "head": head, "longest": longest, "new": new,
            "dtype": dtype, "pages": pages}


def _append(name, B, kv_heads, head, longest, new, dtype="bf16"):
    return {"name": name, "kind": "append", "B": B, "kv_heads": kv_heads, "head": head, "longest": longest, "new": new, "dtype": dtype}


def _select(name, B, beams, vocab, row, dtype="bf16"):
    return {"name": name, "kind": "select", "B": B, "beams": beams, "vocab": vocab, "row": row, "dtype": dtype}


def _reorder(name, layers, B, beams, kv_heads, head, longest):
    return {"name": name, "kind": "reorder", "layers": layers, "B": B, "beams": beams, "kv_heads": kv_heads, "head": head, "longest": longest}


def listed():
    return [
        # one text on the smallest model that people use, early on: a launch and a few loads, latency is all
        _attend("attend_1x12_len40", 1, 12, 12, 64, 40),
        # eight prompts with four beams each in the middle of a text: ragged lengths, pages shared between beams
        _attend("attend_32x12_beams_len777", 32, 12, 12, 64, 777, pages=True),
        # a full batch of d24 late in its context
        _attend("attend_256x16_len1024", 256, 16, 16, 64, 1024),
        # heads of 128 of which four share keys and values, long documents: few rows, a long axis
        _attend("attend_4x32_shared_len32001", 4, 32, 8, 128, 32001),
        # prompts of uneven length on d12, padded to one shape, behind nothing but themselves
        _attend("attend_prompt_16x12_len1000", 16, 12, 12, 64, 1000, new=1000),
        # fp32 storage, heads of 96 (the GPT-3 ladder's c1536), generation
        _attend("attend_fp32_16x16_len1500", 16, 16, 16, 96, 1500, dtype="fp32"),
        # the new token of every sequence of a batch
        _append("append_32x12_new1", 32, 12, 64, 777, 1),
        # the prompts of a batch on d48
        _append("append_16x25_new1000", 16, 25, 64, 1000, 1000),
        # one prompt, four beams
        _select("select_1x4", 1, 4, VOCAB, VOCAB_ROW),
        # a batch of prompts, eight beams each, logits in fp32 in rows that no vector divides
        _select("select_48x8_fp32", 48, 8, VOCAB, VOCAB, dtype="fp32"),
        # the four beams of one prompt on d12
        _reorder("reorder_d12_1x4_len100", 12, 1, 4, 12, 64, 100),
        # a batch of beams on d24
        _reorder("reorder_d24_8x8_len800", 24, 8, 8, 16, 64, 800),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["attend", "attend", "attend", "append", "select", "reorder"])
        head = rng.choice([64, 64, 64, 80, 96, 128])
        kv_heads = _log_int(rng, 1, 32)
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        if kind == "attend":
            new = 1 if rng.random() < 0.6 else _log_int(rng, 2, 1024)
            longest = new + _log_int(rng, 1, 2048 if rng.random() < 0.8 else 32000)
            case = _attend("", _log_int(rng, 1, 256), kv_heads * rng.choice([1, 1, 1, 2, 3, 4, 8]), kv_heads, head, longest, new, dtype,
                           rng.random() < 0.3)
        elif kind == "append":
            new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048)
            case = _append("", _log_int(rng, 1, 256), kv_heads, head, new + rng.randint(0, 1000), new, dtype)
        elif kind == "select":
            vocab = rng.choice([VOCAB, VOCAB, _log_int(rng, 256, VOCAB)])
            case = _select("", _log_int(rng, 1, 64), rng.randint(1, 16), vocab, vocab + rng.choice([0, 0, 7, 47]), dtype)
        else:
            case = _reorder("", rng.randint(6, 48), _log_int(rng, 1, 16), rng.randint(2, 16), kv_heads, head, _log_int(rng, 1, 2048))
        del case["name"]
        if _cost(case) <= most:
            return case


def _cost(case):
    """What one plain pass costs, roughly: elements that it makes in 32 bits."""
    k = case["kind"]
    if k == "attend":
        keys = case["B"] * (case["longest"] + 2 * PAGE)
        return keys * (2 * case["kv_heads"] * case["head"] + 3 * case["heads"] * case["new"])
    if k == "append":
        return 8 * case["B"] * case["new"] * case["kv_heads"] * case["head"]
    if k == "select":
        return 12 * case["B"] * case["beams"] * case["row"]
    return case["layers"] * case["B"] * case["beams"] * case["kv_heads"] * case["head"] * (4 * PAGE + case["longest"] / 4)


def _capacity(case):
    return -(-case["longest"] // PAGE) * PAGE


def _lens(case):
    """Tokens of each sequence (new ones included) and how many of them are new: the same whatever the seed."""
    r = random.Random(case["longest"] * 1000 + case["B"])
    new = case.get("new", 1)
    lens = [case["longest"]] + [r.randint(max(1, case["longest"] // 2), case["longest"]) for _ in range(case["B"] - 1)]
    return lens, [min(n, new if b == 0 else r.randint(max(1, new // 2), new)) for b, n in enumerate(lens)]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(7000 + seed)

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    if case["kind"] == "select":
        rows = case["B"] * case["beams"]
        finished = torch.rand(case["B"], case["beams"], generator=gen, device="cuda") < 0.1
        return {"kind": "select", "vocab": case["vocab"], "eos": case["vocab"] - 1, "finished": finished,
                "logits": normal(rows, case["row"], dtype=DTYPES[case["dtype"]], scale=2.5),
                "scores": torch.rand(case["B"], case["beams"], generator=gen, device="cuda") * -30.0 - 1.0,
                "out": (torch.empty(case["B"], case["beams"], device="cuda"),
                        torch.empty(case["B"], case["beams"], dtype=torch.int32, device="cuda"),
                        torch.empty(case["B"], case["beams"], dtype=torch.int32, device="cuda"),
                        torch.empty(case["B"], case["beams"], dtype=torch.bool, device="cuda"))}
    beams = case.get("beams", 1)
    H, hd, T, S, L = case["kv_heads"], case["head"], _capacity(case), case["B"] * beams, case.get("layers", 1)
    lens, new = _lens(case)

    def cached():
        """Codes and scales of keys or values with a few channels that are larger than the others, as models have them."""
        codes = torch.empty(L, S, H, T, hd // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(L, S, H, T, hd // 16, dtype=torch.uint8, device="cuda")
        channel = 1.0 + 4.0 * (torch.rand(H, 1, hd, generator=gen, device="cuda") < 0.04)
        step = max(1, (1 << 25) // (S * H * hd * L))
        for t in range(0, T, step):
            x = normal(L, S, H, min(step, T - t), hd) * channel
            codes[:, :, :, t:t + step], scales[:, :, :, t:t + step] = _quantize(x)
        return codes, scales

    keys, values = cached(), cached()
    state = {"kind": case["kind"], "cache": (*keys, *values), "head": hd}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["kind"] == "append":
        dt = DTYPES[case["dtype"]]
        qkv = normal(S, case["new"], 3, H, hd, dtype=dt)                   # as a linear layer leaves them: one row per token
        state |= {"k": qkv[:, :, 1], "v": qkv[:, :, 2], "start": ints([a - n for a, n in zip(lens, new)]), "counts": ints(new),
                  "out": tuple(torch.zeros(S, case["new"], H, hd, dtype=dt, device="cuda") for _ in range(2))}
    elif case["kind"] == "attend":
        dt = DTYPES[case["dtype"]]
        pages = None
        if case["pages"]:                                                  # groups of four beams whose full pages were permuted
            own_slot = torch.arange(S, device="cuda").view(S, 1).expand(S, T // PAGE)
            other = own_slot // 4 * 4 + torch.randint(0, 4, (S, T // PAGE), generator=gen, device="cuda")
            full = torch.arange(T // PAGE, device="cuda") < (ints(lens) - ints(new)).view(S, 1) // PAGE
            pages = torch.where(full & (other < S), other, own_slot).to(torch.int32).contiguous()
        q = normal(S, case["new"], case["heads"], hd, dtype=dt, scale=0.7)
        state |= {"q": q, "lens": ints(lens), "counts": ints(new), "pages": pages, "out": torch.zeros_like(q)}
    else:
        parents = torch.randint(0, beams, (case["B"], beams), generator=gen, device="cuda", dtype=torch.int32)
        each = ints(lens).repeat_interleave(beams)
        slot = torch.arange(S, device="cuda").view(S, 1).expand(S, T // PAGE)
        other = slot // beams * beams + torch.randint(0, beams, (S, T // PAGE), generator=gen, device="cuda")
        full = torch.arange(T // PAGE, device="cuda") < each.view(S, 1) // PAGE
        state |= {"beams": beams, "parents": parents, "lens": each, "pages": torch.where(full, other, slot).to(torch.int32).contiguous(),
                  "start": each // PAGE * PAGE,
                  "out": tuple(torch.zeros(L, S, PAGE, H, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))}
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _quantize(x):
    """(codes, scales) as uint8.  A block's scale is its largest magnitude / 6 in e4m3, its values are rounded to the nearest level, ties to
    the even code.  A quotient in 32 bits that is not a tie is never rounded to one: scales have 4 bits and levels' midpoints 3."""
    b = x.float().unflatten(-1, (-1, 16))
    scale = (b.abs().amax(-1, keepdim=True) / (6.0 * UNIT)).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float() * UNIT
    t = torch.where(s > 0, b.abs() / s, torch.zeros_like(b))
    code = ((t > 0.25).to(torch.uint8) + (t >= 0.75) + (t > 1.25) + (t >= 1.75) + (t > 2.5) + (t >= 3.5) + (t > 5.0)) | torch.signbit(b).to(torch.uint8) << 3
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.view(torch.uint8).squeeze(-1)


def _values(codes, scales):
    """fp32 values of codes [..., head / 2] and scales [..., head / 16]."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)[code]
    return (level.unflatten(-1, (-1, 16)) * (scales.view(torch.float8_e4m3fn).float() * UNIT).unsqueeze(-1)).flatten(-2)


def _at(start, n, T):
    """Positions [S, n] behind ``start``, and whether they lie in the cache."""
    pos = start.long().view(-1, 1) + torch.arange(n, device=start.device)
    return pos.clamp(max=T - 1), pos < T


def _read(cache, start, n, dtype):
    """Keys and values [L, S, n, H, head] at the positions behind ``start``; zeros outside the cache."""
    S, T = cache[0].shape[1], cache[0].shape[3]
    pos, inside = _at(start, n, T)
    slot = torch.arange(S, device=pos.device).view(S, 1)
    pick = lambda t: t[:, slot, :, pos].movedim(2, 0)  # noqa: E731          # [S, n, L, H, c] -> [L, S, n, H, c]
    out = [_values(pick(cache[i]), pick(cache[i + 1])) for i in (0, 2)]
    return [torch.where(inside[..., None, None], v, torch.zeros_like(v)).to(dtype) for v in out]


def _plain_append(s):
    S, n = s["k"].shape[:2]
    T = s["cache"][0].shape[3]
    pos, inside = _at(s["start"], n, T)
    keep = (inside & (torch.arange(n, device=pos.device) < s["counts"].view(S, 1))).flatten()
    slot = torch.arange(S, device=pos.device).view(S, 1).expand(S, n).flatten()[keep]
    pos = pos.flatten()[keep]
    for codes, scales, x in ((*s["cache"][:2], s["k"]), (*s["cache"][2:], s["v"])):
        c, f = _quantize(x)
        codes[0, slot, :, pos] = c.flatten(0, 1)[keep]
        scales[0, slot, :, pos] = f.flatten(0, 1)[keep]
    k, v = _read(s["cache"], s["start"], n, s["k"].dtype)
    return {"k": k[0], "v": v[0]}


def _plain_attend(s):
    q = s["q"]
    B, n, heads, hd = q.shape
    kc, ks, vc, vs = (t[0] for t in s["cache"])
    H, T = kc.shape[1:3]
    if s["pages"] is not None:
        src = s["pages"].long().repeat_interleave(PAGE, 1)                 # [S, T]
        kc, ks, vc, vs = (t[src, :, torch.arange(T, device=q.device)].transpose(1, 2) for t in (kc, ks, vc, vs))
    k, v = _values(kc, ks), _values(vc, vs)                                # [B, H, T, head]
    qf = q.float().view(B, n, H, heads // H, hd).permute(0, 2, 3, 1, 4).reshape(B, H, heads // H * n, hd)
    score = (qf @ k.transpose(-1, -2)).view(B, H, heads // H, n, T) / math.sqrt(hd)
    i = torch.arange(n, device=q.device)
    seen = (s["lens"] - s["counts"]).view(B, 1) + i + 1                    # keys that new token i sees
    hidden = torch.arange(T, device=q.device) >= seen.view(B, 1, 1, n, 1)
    score = score.masked_fill_(hidden, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)))
    total = p.sum(-1, keepdim=True)
    o = (p.view(B, H, -1, T) @ v).view(B, H, heads // H, n, hd) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(B, n, heads, hd).to(q.dtype)
    return torch.where((i < s["counts"].view(B, 1))[..., None, None], o, s["out"])


def _plain_select(s):
    B, K = s["scores"].shape
    V, eos = s["vocab"], s["eos"]
    x = s["logits"][:, :V].double().view(B, K, V)                          # candidates of two beams may differ in the last bits alone
    top = x.amax(-1, keepdim=True)
    logp = x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    done = torch.full((V,), float("-inf"), dtype=torch.float64, device=x.device)
    done[eos] = 0.0
    logp = torch.where(s["finished"].unsqueeze(-1), done, logp)
    best, at = torch.sort((s["scores"].double().unsqueeze(-1) + logp).view(B, K * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :K], at[:, :K]
    parents, tokens = at // V, at % V
    finished = s["finished"].gather(1, parents) | (tokens == eos)
    return {"scores": best.float(), "tokens": tokens.int(), "parents": parents.int(), "finished": finished}


def _plain_reorder(s):
    S, K, T = s["lens"].numel(), s["beams"], s["cache"][0].shape[3]
    slot = torch.arange(S, device=s["lens"].device)
    src = slot // K * K + s["parents"].flatten().long()
    lens = s["lens"][src]
    pos, inside = _at(lens // PAGE * PAGE, PAGE, T)
    mine = inside & (pos < lens.view(S, 1))
    at, to, of = pos[mine], slot.view(S, 1).expand(S, PAGE)[mine], src.view(S, 1).expand(S, PAGE)[mine]
    for t in s["cache"]:
        t[:, to, :, at] = t[:, of, :, at]
    full = torch.arange(T // PAGE, device=slot.device) < (lens // PAGE).view(S, 1)
    s["pages"].copy_(torch.where(full, s["pages"][src], slot.view(S, 1).int()))
    s["lens"].copy_(lens)
    k, v = _read(s["cache"], s["start"], PAGE, torch.bfloat16)
    return {"pages": s["pages"], "lens": s["lens"], "k": k, "v": v}


def run(state):
    kind = state["kind"]
    if own:
        from llm_mojo_b200 import ops

        if kind == "select":
            scores, tokens, parents, finished = state["out"]
            ops.beam_select(scores, tokens, parents, state["logits"], state["scores"], state["vocab"], finished_out=finished,
                            finished=state["finished"], eos=state["eos"])
            return {"scores": scores, "tokens": tokens, "parents": parents, "finished": finished}
        cache = ops.KV4Cache(*state["cache"])
        if kind == "attend":
            ops.attention_kv4(state["out"], state["q"], cache, 0, state["lens"], counts=state["counts"], pages=state["pages"])
            return state["out"]
        k, v = state["out"]
        if kind == "append":
            ops.kv4_append(cache, 0, state["k"], state["v"], state["start"], counts=state["counts"])
            ops.kv4_values(k, v, cache, 0, state["start"])
            return {"k": k, "v": v}
        ops.kv4_reorder(cache, state["pages"], state["lens"], state["parents"])
        ops.kv4_values(k, v, cache, None, state["start"])
        return {"pages": state["pages"], "lens": state["lens"], "k": k, "v": v}
    return {"append": _plain_append, "attend": _plain_attend, "select": _plain_select, "reorder": _plain_reorder}[kind](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "select":
        rows = case["B"] * case["beams"]
        e = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": rows * (case["vocab"] * e + 5 + 13), "flops": 3 * rows * case["vocab"]}
    lens, new = _lens(case)
    H, hd = case["kv_heads"], case["head"]
    token = 2 * H * (hd // 2 + hd // 16)                                   # bytes of a token's key and value in one layer
    if case["kind"] == "append":
        e = 4 if case["dtype"] == "fp32" else 2
        back = 2 * case["B"] * case["new"] * H * hd * e                    # the values read back, behind the last new token too
        return {"bytes": sum(new) * (2 * H * hd * e + token) + back + 8 * case["B"], "flops": 8 * sum(new) * H * hd}
    if case["kind"] == "attend":
        e = 4 if case["dtype"] == "fp32" else 2
        pairs = sum(n * (a - n) + n * (n + 1) // 2 for a, n in zip(lens, new))
        return {"bytes": sum(lens) * token + 2 * sum(new) * case["heads"] * hd * e + 8 * case["B"], "flops": 4 * pairs * case["heads"] * hd}
    # every slot's newest page is written once and, where beams share a parent, read once for all of them (1 - 1/e of the slots)
    K, L = case["beams"], case["layers"]
    kept = 1.0 - (1.0 - 1.0 / K) ** K
    moved = L * sum(a % PAGE for a in lens) * K * token * (1 - 1.0 / K + kept)
    back = 2 * L * case["B"] * K * PAGE * H * hd * 2
    tables = case["B"] * K * (8 * (_capacity(case) // PAGE) + 12)
    return {"bytes": moved + back + tables, "flops": back / 2}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _e4m3(x):
    """x >= 0 in float64, rounded to e4m3 (ties to even, the largest is 448)."""
    exponent = torch.floor(torch.log2(x.clamp(min=2.0 ** -6))).clamp(min=-6.0)
    exponent = torch.where(x >= torch.exp2(exponent + 1), exponent + 1, exponent)
    exponent = torch.where((x < torch.exp2(exponent)) & (exponent > -6), exponent - 1, exponent)
    ulp = torch.exp2(exponent - 3)
    return (torch.round(x / ulp) * ulp).clamp(max=448.0)


def _rounded(x):
    """What x stands for once it has been in the cache, in float64."""
    b = x.double().unflatten(-1, (-1, 16))
    s = _e4m3(b.abs().amax(-1, keepdim=True) / 6.0 / UNIT) * UNIT
    r = b.abs() / torch.where(s > 0, s, torch.ones_like(s))
    level = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    low = torch.bucketize(r, level, right=True).sub(1).clamp(0, 6)         # level[low] <= r
    a, c = r - level[low], level[low + 1] - r
    up = (a > c) | ((a == c) & (low % 2 == 1))
    out = level[torch.where(up, low + 1, low)] * s
    return torch.copysign(torch.where(s > 0, out, torch.zeros_like(out)), b).flatten(-2)


def _decoded(codes, scales):
    """float64 values from the bits of codes and scales."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    e, m = (code >> 1 & 3).double(), (code & 1).double()
    mag = torch.where(e > 0, torch.exp2(e - 1) * (1 + m / 2), m / 2)
    f = scales.long()
    fe, fm = (f >> 3 & 15).double(), (f & 7).double()
    scale = torch.where(fe > 0, torch.exp2(fe - 7) * (1 + fm / 8), torch.exp2(torch.full_like(fm, -6.0)) * fm / 8) * UNIT
    return torch.where(code >= 8, -mag, mag) * scale.repeat_interleave(16, -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "select":
        return _exact_select(s)
    kc, ks, vc, vs = s["cache"]
    T = kc.shape[3]
    if case["kind"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lens, new = _lens(case)
        group = case["heads"] // case["kv_heads"]
        for b in range(case["B"]):
            places = list(range(-(-lens[b] // PAGE)))
            slots = [b] * len(places) if s["pages"] is None else s["pages"][b].tolist()
            whole = lambda t: torch.cat([t[0, slots[p], :, p * PAGE:(p + 1) * PAGE] for p in places], 1)[:, :lens[b]]  # noqa: E731
            k, v = _decoded(whole(kc), whole(ks)), _decoded(whole(vc), whole(vs))
            k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
            for h in range(case["heads"]):
                w = s["q"][b, :new[b], h].double() @ k[h].t() * hd_scale(case)
                order = torch.arange(lens[b], device="cuda").view(1, -1) - torch.arange(new[b], device="cuda").view(-1, 1)
                out[b, :new[b], h] = torch.softmax(w.masked_fill(order > lens[b] - new[b], float("-inf")), -1) @ v[h]
        return out
    if case["kind"] == "append":
        lens, new = _lens(case)
        n = case["new"]
        k, v = (torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2))
        for b in range(case["B"]):
            first = lens[b] - new[b]
            have = min(n, T - first)
            for out, codes, scales, x in ((k, kc, ks, s["k"]), (v, vc, vs, s["v"])):
                out[b, :have] = _decoded(codes[0, b, :, first:first + have], scales[0, b, :, first:first + have]).transpose(0, 1)
                out[b, :new[b]] = _rounded(x[b, :new[b]])
        return {"k": k, "v": v}
    parents, K = s["parents"].tolist(), case["beams"]
    lens = s["lens"].tolist()
    pages, k, v = s["pages"].clone(), [], []
    for slot in range(case["B"] * K):
        of = slot // K * K + parents[slot // K][slot % K]
        full, rest = lens[of] // PAGE, lens[of] % PAGE
        pages[slot, :full], pages[slot, full:] = s["pages"][of, :full], slot
        for out, codes, scales in ((k, kc, ks), (v, vc, vs)):
            place = slice(full * PAGE, full * PAGE + PAGE)
            page = torch.cat([_decoded(codes[:, i, :, place], scales[:, i, :, place])[:, :, a:z] for i, a, z in ((of, 0, rest), (slot, rest, PAGE))], 2)
            out.append(page.transpose(1, 2) if page.shape[2] else torch.zeros(page.shape[0], PAGE, page.shape[1], page.shape[3], dtype=torch.float64, device="cuda"))
    src = [b * K + p for b, row in enumerate(parents) for p in row]
    return {"pages": pages, "lens": s["lens"][src], "k": torch.stack(k, 1), "v": torch.stack(v, 1)}


def hd_scale(case):
    return case["head"] ** -0.5


def _exact_select(s):
    B, K = s["scores"].shape
    V = s["vocab"]
    scores, tokens, parents, finished = (torch.zeros(B, K, dtype=t, device="cuda") for t in (torch.float64, torch.int32, torch.int32, torch.bool))
    for b in range(B):
        c = torch.log_softmax(s["logits"][b * K:(b + 1) * K, :V].double(), -1)
        c[s["finished"][b]] = float("-inf")
        c[s["finished"][b], s["eos"]] = 0.0
        c = (c + s["scores"][b].double().unsqueeze(-1)).flatten()
        for i in range(K):
            at = int(torch.argmax(c))
            scores[b, i], tokens[b, i], parents[b, i] = c[at], at % V, at // V
            finished[b, i] = bool(s["finished"][b, at // V]) or at % V == s["eos"]
            c[at] = float("-inf")
    return {"scores": scores, "tokens": tokens, "parents": parents, "finished": finished}
