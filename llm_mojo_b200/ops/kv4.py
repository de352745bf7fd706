"""Key/value cache in 4 bits: write, read back, attention of new tokens over it, and its reordering by a beam search.

The cache keeps keys and values in the form of the NVFP4 operands (``csrc/quant.cu``): e2m1 values, two to a byte with the first in the low
nibble, and an e4m3 scale for every 16 values along the head; instead of a tensor scale, which would have to be known before the text is,
there is one power of two for all keys and one for all values.  Every value that the cache can hold is then a bf16 number.

    k_codes, v_codes    uint8 [layers, slots, kv_heads, capacity, head_size / 2]
    k_scales, v_scales  uint8 [layers, slots, kv_heads, capacity, head_size / 16]

A slot is one sequence.  ``capacity`` is a multiple of the ``KV4_PAGE`` = 64 tokens of a page; ``pages`` (int32 [slots, capacity / 64], optional)
names for each slot and page the slot in whose place that page is kept, so that beams share the pages they have in common.  The page that a
slot is filling, and those behind it, are always its own.

CUDA tensors run ``csrc/kv4.cu`` and ``csrc/attention_kv4.cu``; CPU tensors run the fp32 PyTorch statement of the same definitions.
"""
from __future__ import annotations

import itertools
import math
import struct
from typing import Optional

import torch

from . import _count
from ._lib import check, lib, status_word

KV4_PAGE = 64
KV4_UNIT = 2.0 ** -4          # largest value 2688 / 16 = 168; scales of 2^-6 and more (values of 0.006 and more) have all their bits
KV4_HEAD_SIZES = (32, 64, 80, 96, 128)
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# Arguments travel as packed structures, one pointer a call: a ctypes call that converts twenty arguments takes longer than a launch.
_DESC = struct.Struct("@4P4q8i")             # Kv4Desc of csrc/kv4.cuh
_APPEND = struct.Struct("@4P6q4i")           # Kv4AppendArgs of csrc/kv4.cu
_VALUES = struct.Struct("@4P7q4i")           # Kv4ValuesArgs
_REORDER = struct.Struct("@3P2i")            # Kv4ReorderArgs
_ATTEND = struct.Struct("@6P6qf5i")          # Kv4AttendArgs of csrc/attention_kv4.cu


def _exponent(unit: float, name: str) -> int:
    m, e = math.frexp(unit) if isinstance(unit, (int, float)) and math.isfinite(unit) else (0.0, 0)
    if m != 0.5 or not -32 <= e - 1 <= 32:
        raise ValueError(f"{name} must be a power of two between 2^-32 and 2^32, not {unit!r}")
    return e - 1


_STATUS_AT = {}


def _status_at(device: torch.device, index: int) -> int:
    at = _STATUS_AT[index] = status_word(device).data_ptr()      # the word lives as long as the process
    return at


class KV4Cache:
    """The four tensors of a cache (see the module), checked once.  Layers and slots may be strided views of larger caches (every third
    slot, some of the layers); heads, tokens and values lie densely, every row 16-byte aligned.  No two of the four share memory."""

    __slots__ = ("k_codes", "k_scales", "v_codes", "v_scales", "k_unit", "v_unit", "layers", "slots", "kv_heads", "capacity", "head_size",
                 "device", "index", "_desc", "_status")

    def __init__(self, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
                 k_unit: float = KV4_UNIT, v_unit: float = KV4_UNIT):
        codes, scales = k_codes.shape, k_scales.shape
        if len(codes) != 5:
            raise ValueError(f"codes are [layers, slots, kv_heads, capacity, head_size / 2], not {tuple(codes)}")
        L, S, H, T, half = codes
        if 2 * half not in KV4_HEAD_SIZES:
            raise ValueError(f"head size {2 * half}: the cache takes {KV4_HEAD_SIZES}")
        if T % KV4_PAGE or T == 0 or L == 0 or S == 0 or H == 0:
            raise ValueError(f"capacity {T} must be a multiple of {KV4_PAGE}, and no dimension of {tuple(codes)} empty")
        if H > 65535 or S > 65535 or L > 65535 or T > 2 ** 30:
            raise ValueError(f"at most 65535 layers, slots and heads and 2^30 tokens, not {L}, {S}, {H} and {T}")
        dev, at = k_codes.device, k_codes.get_device()
        p = (k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr())
        u8 = torch.uint8
        if p[0] == p[2] or p[1] == p[3]:
            raise ValueError("keys and values must not be the same memory")
        if (scales != (L, S, H, T, half // 8) or v_codes.shape != codes or v_scales.shape != scales or k_scales.get_device() != at
                or v_codes.get_device() != at or v_scales.get_device() != at or k_codes.dtype is not u8 or k_scales.dtype is not u8
                or v_codes.dtype is not u8 or v_scales.dtype is not u8):
            for name, t, shape in (("k_codes", k_codes, tuple(codes)), ("k_scales", k_scales, (L, S, H, T, half // 8)),
                                   ("v_codes", v_codes, tuple(codes)), ("v_scales", v_scales, (L, S, H, T, half // 8))):
                if t.dtype != u8 or t.shape != shape or t.device != dev:
                    raise ValueError(f"{name} must be uint8 {shape} on {dev}, not {t.dtype} {tuple(t.shape)} on {t.device}")
        if (p[0] | p[1] | p[2] | p[3]) % 16 == 0 and k_codes.is_contiguous() and k_scales.is_contiguous() and v_codes.is_contiguous() and v_scales.is_contiguous():
            cs1, ss1 = H * T * half, H * T * (half // 8)
            cs0, ss0 = S * cs1, S * ss1
            c, s, dense = L * cs0, L * ss0, True
        else:
            cs, ss = k_codes.stride(), k_scales.stride()
            cs0, cs1, ss0, ss1 = cs[0], cs[1], ss[0], ss[1]
            for name, t, st, ptr in (("k_codes", k_codes, cs, p[0]), ("k_scales", k_scales, ss, p[1]), ("v_codes", v_codes, cs, p[2]),
                                     ("v_scales", v_scales, ss, p[3])):
                if t.stride() != st:
                    raise ValueError(f"{name}: keys and values must have the same strides, not {t.stride()} and {st}")
                c = t.shape[4]
                if st[4] != 1 or st[3] != c or (H > 1 and st[2] != T * c) or (ptr | (st[1] if S > 1 else 0) | (st[0] if L > 1 else 0)) % 16:
                    raise ValueError(f"{name}: heads, tokens and values must lie densely, slots and layers 16-byte aligned (strides {st})")
                row = H * T * c
                if (S > 1 and st[1] < row) or (L > 1 and st[0] < row) or (L > 1 and S > 1 and (S - 1) * st[1] + row > st[0] and (L - 1) * st[0] + row > st[1]):
                    raise ValueError(f"{name}: slots and layers must not overlap (strides {st})")
            c, s, dense = (L - 1) * cs0 + (S - 1) * cs1 + H * T * half, (L - 1) * ss0 + (S - 1) * ss1 + H * T * (half // 8), False
        kc, ks, vc, vs = p                                   # c, s: from the first byte of codes and of scales to their last
        if (-c < kc - vc < c or -s < ks - vs < s or -s < ks - kc < c or -s < vs - kc < c or -s < ks - vc < c or -s < vs - vc < c) and (
                dense or any(_meet(a, b) for a, b in itertools.combinations((k_codes, k_scales, v_codes, v_scales), 2))):
            raise ValueError("codes and scales of keys and of values are four tensors: they must not share memory")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.k_unit, self.v_unit = k_unit, v_unit
        self.layers, self.slots, self.kv_heads, self.capacity, self.head_size, self.device, self.index = L, S, H, T, 2 * half, dev, at
        self._desc = _DESC.pack(*p, cs0, cs1, ss0, ss1, L, S, H, T, 2 * half, -4 if k_unit == KV4_UNIT else _exponent(k_unit, "k_unit"),
                                -4 if v_unit == KV4_UNIT else _exponent(v_unit, "v_unit"), 0)
        # made with the cache: in a call that a graph captures, the word's zeros would become a step of the graph
        self._status = 0 if at < 0 else _STATUS_AT.get(at) or _status_at(dev, at)

    @classmethod
    def empty(cls, layers: int, slots: int, kv_heads: int, max_len: int, head_size: int, device="cuda", k_unit: float = KV4_UNIT,
              v_unit: float = KV4_UNIT) -> "KV4Cache":
        """A cache for ``slots`` sequences of up to ``max_len`` tokens, all zeros."""
        if head_size not in KV4_HEAD_SIZES:
            raise ValueError(f"head size {head_size}: the cache takes {KV4_HEAD_SIZES}")
        T = max(1, -(-max_len // KV4_PAGE)) * KV4_PAGE
        z = lambda c: torch.zeros(layers, slots, kv_heads, T, c, dtype=torch.uint8, device=device)  # noqa: E731
        return cls(z(head_size // 2), z(head_size // 16), z(head_size // 2), z(head_size // 16), k_unit, v_unit)

    def own_pages(self) -> torch.Tensor:
        """The page table in which every page lies in its own slot."""
        return torch.arange(self.slots, dtype=torch.int32, device=self.device).view(-1, 1).repeat(1, self.capacity // KV4_PAGE)

    def select(self, slots: slice) -> "KV4Cache":
        """The same cache restricted to some of its slots (a slice): a view."""
        return KV4Cache(self.k_codes[:, slots], self.k_scales[:, slots], self.v_codes[:, slots], self.v_scales[:, slots], self.k_unit, self.v_unit)

    def nbytes(self) -> int:
        return self.layers * self.slots * self.kv_heads * self.capacity * (self.head_size // 2 + self.head_size // 16) * 2


# ------------------------------------------------------------------ arguments
# private names of torch, each with the public form beside it: the public forms take as long as a launch
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    lambda index: torch.cuda.current_stream(index).cuda_stream


_current = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


def _call(fn, name: str, index: int, first, second) -> None:
    """Launches go to the current stream of the tensors' device, whichever device is current."""
    if index == _current():
        rc = fn(first, second, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(first, second, _raw_stream(index))
    if rc:
        check(rc, name)


def _ints(t: Optional[torch.Tensor], name: str, shape: tuple, index: int) -> int:
    """The address of an optional tensor of integers."""
    if t is None:
        return 0
    if t.dtype is not torch.int32 or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 {tuple(shape)} on {_name(index)}, not {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _name(index: int) -> str:
    return f"cuda:{index}" if index >= 0 else "cpu"


def _layer(cache: KV4Cache, layer: int) -> None:
    if not isinstance(layer, int) or not 0 <= layer < cache.layers:
        raise ValueError(f"layer {layer!r} of a cache of {cache.layers} layers")


def _rows(t: torch.Tensor, name: str, shape: tuple, dtype, index: int, known: bool = False) -> tuple:
    """The strides of a tensor of rows (``known``: the shape and the type are the tensor's own)."""
    if (not known and (t.dtype is not dtype or t.shape != shape)) or t.get_device() != index:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} on {_name(index)}, not {t.dtype} {tuple(t.shape)} on {t.device}")
    st = t.stride()
    if st[-1] != 1 and t.numel():
        raise ValueError(f"{name}: the values of a head must lie densely (strides {st})")
    return st


def _spread(t: torch.Tensor, name: str) -> None:
    """An output whose elements share memory would be written by several threads."""
    if t.is_contiguous():
        return
    span = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda p: p[1]):
        if s < span:
            raise ValueError(f"{name}: elements of an output must not overlap (shape {tuple(t.shape)}, strides {t.stride()})")
        span += s * (n - 1)


def _places(t: torch.Tensor) -> list:
    """(extent, stride in bytes) of the dimensions that have more than one index, the widest stride first."""
    e = t.element_size()
    return sorted(((n, s * e) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda p: -p[1])


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one device have a byte in common; the elements of each by themselves do not overlap (see ``_spread``)."""
    if not a.numel() or not b.numel():
        return False
    (da, db), e = (_places(a), _places(b)), a.element_size()
    pa, pb = a.data_ptr(), b.data_ptr()
    last = lambda d, t: sum((n - 1) * s for n, s in d) + t.element_size()  # noqa: E731
    if pa >= pb + last(db, b) or pb >= pa + last(da, a):
        return False
    if da == db and e == b.element_size():                   # as slices of one tensor have them: a distance that indices make up, or none
        def makes(d, far):
            if not d:
                return -e < far < e
            (n, s), rest = d[0], d[1:]
            if not s:
                return makes(rest, far)
            return any(makes(rest, far - i * s) for i in (far // s, far // s + 1) if -n < i < n)
        return makes(da, pb - pa)
    starts, width = [], []
    for p, d, t in ((pa, da, a), (pb, db, b)):               # runs of bytes that lie densely
        w, d = t.element_size(), list(d)
        while d and d[-1][1] == w:
            w *= d.pop()[0]
        at = torch.tensor([p], device="cpu")
        for n, s in d:
            at = (at.view(-1, 1) + torch.arange(n, device="cpu") * s).view(-1)
        starts.append(at)
        width.append(w)
    at = starts[0].sort().values
    i = torch.searchsorted(at, starts[1] + width[1]) - 1     # the last run of a that begins before a run of b ends
    return bool(((i >= 0) & (at[i.clamp(min=0)] + width[0] > starts[1])).any())


# ------------------------------------------------------------------ the definitions, on any device, in fp32
def _encode(x: torch.Tensor, unit: float):
    """(codes, scales) of x [..., head_size]: a block's scale is e4m3(amax / 6 / unit), its values e2m1(x / (scale unit)), ties to even."""
    b = x.float().unflatten(-1, (-1, 16))
    scale = (b.abs().amax(-1, keepdim=True) / unit / 6.0).nan_to_num(0.0, 448.0, 448.0).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float() * unit
    t = torch.where(s > 0, b.abs() / s, torch.zeros_like(b))
    code = sum(((t > e) if i % 2 == 0 else (t >= e)).to(torch.uint8) for i, e in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code = torch.where(s > 0, code | torch.signbit(b).to(torch.uint8) << 3, torch.zeros_like(code)).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, scale.view(torch.uint8).squeeze(-1)


def _decode(codes: torch.Tensor, scales: torch.Tensor, unit: float) -> torch.Tensor:
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    level = torch.tensor(_LEVELS + tuple(-v for v in _LEVELS), device=codes.device)[code]
    return (level.unflatten(-1, (-1, 16)) * (scales.view(torch.float8_e4m3fn).float() * unit).unsqueeze(-1)).flatten(-2)


# ------------------------------------------------------------------ operators
def kv4_append(cache: KV4Cache, layer: int, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor,
               counts: Optional[torch.Tensor] = None) -> None:
    """Writes keys and values ``k``, ``v`` [slots, n, kv_heads, head_size] (bf16 or fp32; strided views of a packed qkv, for instance) of
    ``n`` new tokens to the positions ``start[s] + i`` of one layer.  ``counts`` [slots]: the first ``counts[s]`` of them only (prompts padded
    to one shape).  Positions outside the cache are not written.  ``start`` and ``counts`` are int32 on the device.

    A value beyond the largest one (2688 units) becomes that one.  A token and head with a non-finite key or value has no 4-bit form: its
    key and its value are kept as NaN, and every query that sees it answers NaN."""
    shape = k.shape
    if len(shape) != 4 or shape[0] != cache.slots or shape[2] != cache.kv_heads or shape[3] != cache.head_size:
        raise ValueError(f"k must be [{cache.slots}, n, {cache.kv_heads}, {cache.head_size}], not {tuple(shape)}")
    S, n, H, hd = shape
    dtype, dev = k.dtype, cache.index
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise TypeError(f"k and v must be bf16 or fp32, not {dtype}")
    _layer(cache, layer)
    ks, vs = _rows(k, "k", shape, dtype, dev, True), _rows(v, "v", shape, dtype, dev)
    at, cnt = _ints(start, "start", (S,), dev), _ints(counts, "counts", (S,), dev)
    if n == 0:
        return
    if dev >= 0:
        _call(lib().llmb_kv4_append, "kv4_append", dev, cache._desc,
              _APPEND.pack(k.data_ptr(), v.data_ptr(), at, cnt, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], layer, n, 1 if dtype is torch.bfloat16 else 0, 0))
        _count()
        return
    kf, vf = k.float(), v.float()
    bad = ~(torch.isfinite(kf).all(-1, keepdim=True) & torch.isfinite(vf).all(-1, keepdim=True))
    for s in range(S):
        p0 = int(start[s])
        lo, hi = max(0, -p0), min(n if counts is None else min(n, int(counts[s])), cache.capacity - p0)
        if lo >= hi:
            continue
        for x, codes, scales, unit in ((kf, cache.k_codes, cache.k_scales, cache.k_unit), (vf, cache.v_codes, cache.v_scales, cache.v_unit)):
            c, f = _encode(x[s, lo:hi].nan_to_num(0.0, 0.0, 0.0), unit)
            f = torch.where(bad[s, lo:hi], torch.full_like(f, 0x7f), f)
            codes[layer, s, :, p0 + lo:p0 + hi] = c.transpose(0, 1)
            scales[layer, s, :, p0 + lo:p0 + hi] = f.transpose(0, 1)


def kv4_values(k_out: torch.Tensor, v_out: torch.Tensor, cache: KV4Cache, layer: Optional[int], start: torch.Tensor,
               pages: Optional[torch.Tensor] = None) -> None:
    """Reads back what the cache holds: ``k_out``, ``v_out`` [slots, n, kv_heads, head_size] (bf16, in which every value is exact, or fp32) of
    the positions ``start[s] + i`` of one layer, or [layers, slots, ...] of all layers (``layer`` None).  Positions outside the cache read as
    zeros, pages whose entry in ``pages`` names no slot as NaN.  The outputs share no memory."""
    dtype, dev, shape = k_out.dtype, cache.index, k_out.shape
    lead = (cache.slots,) if layer is not None else (cache.layers, cache.slots)
    if len(shape) != len(lead) + 3 or shape[:-3] != lead or shape[-2] != cache.kv_heads or shape[-1] != cache.head_size:
        raise ValueError(f"k_out must be {[*lead, 'n', cache.kv_heads, cache.head_size]}, not {tuple(shape)}")
    n = shape[-3]
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise TypeError(f"k_out and v_out must be bf16 or fp32, not {dtype}")
    if layer is not None:
        _layer(cache, layer)
    ks, vs = _rows(k_out, "k_out", shape, dtype, dev, True), _rows(v_out, "v_out", shape, dtype, dev)
    _spread(k_out, "k_out")
    _spread(v_out, "v_out")
    kp, vp = k_out.data_ptr(), v_out.data_ptr()
    if (abs(kp - vp) < k_out.numel() * (2 if dtype is torch.bfloat16 else 4) or not (k_out.is_contiguous() and v_out.is_contiguous())) and _meet(k_out, v_out):
        raise ValueError("k_out and v_out are two outputs: they must not be the same memory")
    if layer is None and n and ks != vs:
        raise ValueError(f"k_out and v_out must have the same strides, not {ks} and {vs}")
    at, pg = _ints(start, "start", (cache.slots,), dev), _ints(pages, "pages", (cache.slots, cache.capacity // KV4_PAGE), dev)
    if n == 0:
        return
    if dev >= 0:
        _call(lib().llmb_kv4_values, "kv4_values", dev, cache._desc,
              _VALUES.pack(kp, vp, at, pg, ks[0] if layer is None else 0, ks[-4], ks[-3], ks[-2], vs[-4], vs[-3], vs[-2],
                           -1 if layer is None else layer, n, 1 if dtype is torch.bfloat16 else 0, 0))
        _count()
        return
    T, i = cache.capacity, torch.arange(n)
    for s in range(cache.slots):
        pos = int(start[s]) + i
        inside = (pos >= 0) & (pos < T)
        pos = pos.clamp(0, T - 1)
        slot = torch.full_like(pos, s) if pages is None else pages[s].long()[pos // KV4_PAGE]
        wrong = (slot < 0) | (slot >= cache.slots)
        slot = slot.clamp(0, cache.slots - 1)
        for l in range(cache.layers) if layer is None else (layer,):
            for out, codes, scales, unit in ((k_out, cache.k_codes, cache.k_scales, cache.k_unit), (v_out, cache.v_codes, cache.v_scales, cache.v_unit)):
                x = _decode(codes[l, slot, :, pos], scales[l, slot, :, pos], unit)
                x[wrong] = float("nan")
                x[~inside] = 0.0
                (out[l] if layer is None else out)[s] = x.to(out.dtype)


def attention_kv4(out: torch.Tensor, q: torch.Tensor, cache: KV4Cache, layer: int, lens: torch.Tensor, counts: Optional[torch.Tensor] = None,
                  pages: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> None:
    """Attention of the newest tokens of each slot over one layer of the cache (their own keys and values are in it already).

    ``q``, ``out`` [slots, n, heads, head_size], bf16 or fp32, strided views allowed, ``heads`` a multiple of the cache's; head h reads key head
    h // (heads / kv_heads).  ``lens`` [slots]: tokens in the cache; ``counts`` [slots]: how many of the n rows of a slot are queries (n without
    it).  Row i < counts[s] is the token at position lens[s] - counts[s] + i and sees the positions up to its own; a row that sees none (an
    empty slot) gives zeros; rows behind counts[s] are left as they are.  ``scale``: of the scores, 1 / sqrt(head_size) by default.
    ``out`` may be ``q`` itself, and otherwise has no memory in common with it.  A page whose entry in ``pages`` names no slot gives NaN to every row that sees it.

    Scores, statistics and sums are in fp32.  lens above the capacity count as the capacity."""
    shape, dtype, dev = q.shape, q.dtype, cache.index
    if len(shape) != 4 or shape[0] != cache.slots or shape[3] != cache.head_size or shape[2] % cache.kv_heads or shape[2] == 0:
        raise ValueError(f"q must be [{cache.slots}, n, a multiple of {cache.kv_heads}, {cache.head_size}], not {tuple(shape)}")
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise TypeError(f"q must be bf16 or fp32, not {dtype}")
    S, n, heads, hd = shape
    if not isinstance(layer, int) or not 0 <= layer < cache.layers:
        _layer(cache, layer)
    qs, os_ = q.stride(), out.stride()
    if out.shape != shape or out.dtype is not dtype or q.get_device() != dev or out.get_device() != dev or qs[3] != 1 or os_[3] != 1:
        _rows(q, "q", shape, dtype, dev, True), _rows(out, "out", shape, dtype, dev)          # says what is wrong, or that nothing is (no element)
    flat = out.is_contiguous()
    if not flat:
        _spread(out, "out")
    qp, op = q.data_ptr(), out.data_ptr()
    if qp != op or qs != os_:                                # rows that are written while others are still to be read
        far, e = op - qp, 2 if dtype is torch.bfloat16 else 4
        if flat and qs == os_:
            near = abs(far) < q.numel() * e
        else:
            a, z, w = S - 1, n - 1, heads - 1
            near = -(a * os_[0] + z * os_[1] + w * os_[2] + hd) * e < far < (a * qs[0] + z * qs[1] + w * qs[2] + hd) * e
        if near and (far or _places(q) != _places(out)) and _meet(q, out):
            raise ValueError(f"out must be q itself or share no memory with it (strides {qs} and {os_})")
    ln, cnt = _ints(lens, "lens", (S,), dev), _ints(counts, "counts", (S,), dev)
    pg = _ints(pages, "pages", (S, cache.capacity // KV4_PAGE), dev)
    if scale is None:
        scale = hd ** -0.5
    elif not math.isfinite(scale):
        raise ValueError(f"scale must be finite, not {scale}")
    if n * heads > 2 ** 30:
        raise ValueError(f"{n} rows of {heads} heads are too many")
    if n == 0:
        return
    if dev >= 0:
        _call(lib().llmb_attention_kv4, "attention_kv4", dev, cache._desc,
              _ATTEND.pack(op, qp, ln, cnt, pg, cache._status, qs[0], qs[1], qs[2], os_[0], os_[1], os_[2], scale, layer, n,
                           heads, 1 if dtype is torch.bfloat16 else 0, 0))
        _count()
        return
    group, T = heads // cache.kv_heads, cache.capacity
    for s in range(S):
        L = min(max(int(lens[s]), 0), T)
        c = n if counts is None else min(max(int(counts[s]), 0), n)
        if c == 0:
            continue
        pos = torch.arange(L)
        slot = torch.full_like(pos, s) if pages is None else pages[s].long()[pos // KV4_PAGE]
        wrong = (slot < 0) | (slot >= cache.slots)
        slot = slot.clamp(0, cache.slots - 1)
        k = _decode(cache.k_codes[layer, slot, :, pos], cache.k_scales[layer, slot, :, pos], cache.k_unit)      # [L, H, hd]
        v = _decode(cache.v_codes[layer, slot, :, pos], cache.v_scales[layer, slot, :, pos], cache.v_unit)
        k[wrong] = float("nan")
        v = v.nan_to_num(0.0)                    # such a token's key is NaN as well: its weight says so to the rows that see it
        x = q[s, :c].float().view(c, cache.kv_heads, group, hd)
        w = torch.einsum("chgd,lhd->hgcl", x, k) * scale
        w = w.masked_fill(pos.view(1, -1) >= (L - c + 1 + torch.arange(c)).view(-1, 1), float("-inf"))
        m = w.amax(-1, keepdim=True) if L else torch.zeros(*w.shape[:-1], 1)
        p = torch.exp(w - torch.where(torch.isneginf(m), torch.zeros_like(m), m))
        total = p.sum(-1, keepdim=True)
        o = torch.einsum("hgcl,lhd->chgd", p / torch.where(total == 0, torch.ones_like(total), total), v)
        out[s, :c] = o.reshape(c, heads, hd).to(out.dtype)


def kv4_reorder(cache: KV4Cache, pages: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor) -> None:
    """The cache follows a beam search: slot b K + j of item b becomes what slot b K + ``parents[b, j]`` was (``parents`` int32 [items, K],
    items x K = slots), in place and in every layer.  Entries of ``pages`` for whole pages and ``lens`` are permuted; of the keys and values
    only the page that is being filled is copied, at most 63 tokens.  Entries for pages that are not full name the slot itself.  A parent
    outside 0 .. K - 1 counts as j itself; lengths beyond the capacity count as the capacity.  The three tables share no memory.

    The parents that one item names have one length, as beams that grew together have: the page in which a shorter one ends may be a full
    page of a longer one, shared by that one's other children, and the shorter one's child goes on writing into it.

    A full page is never written again, so any number of slots may share it; the tokens appended next go to the slot's own place."""
    if parents.dim() != 2 or parents.numel() != cache.slots or parents.shape[1] == 0:
        raise ValueError(f"parents must be [items, K] with items x K = {cache.slots}, not {tuple(parents.shape)}")
    B, K = parents.shape
    if K > 64:
        raise ValueError(f"at most 64 beams, not {K}")
    dev = cache.index
    if pages is None or lens is None:
        raise ValueError("kv4_reorder permutes pages and lens: both are needed")
    par, ln = _ints(parents, "parents", (B, K), dev), _ints(lens, "lens", (cache.slots,), dev)
    pg = _ints(pages, "pages", (cache.slots, cache.capacity // KV4_PAGE), dev)
    tables, each = 4 * pages.numel(), 4 * cache.slots        # bytes, of lens and of parents alike
    if -each < ln - par < each or -tables < pg - par < each or -tables < pg - ln < each:
        raise ValueError("pages, lens and parents must not share memory")
    if dev >= 0:
        _call(lib().llmb_kv4_reorder, "kv4_reorder", dev, cache._desc, _REORDER.pack(pg, ln, par, K, 0))
        _count(2)
        return
    slot = torch.arange(cache.slots)
    j = parents.flatten().long()
    src = torch.where((j < 0) | (j >= K), slot, slot // K * K + j)
    new = lens[src].clamp(0, cache.capacity)
    full = new // KV4_PAGE
    old = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    for s in range(cache.slots):
        a, z = int(full[s]) * KV4_PAGE, int(new[s])
        for t, o in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), old):
            t[:, s, :, a:z] = o[:, src[s], :, a:z]
    whole = torch.arange(pages.shape[1]) < full.view(-1, 1)
    pages.copy_(torch.where(whole, pages[src], slot.view(-1, 1).int()))
    lens.copy_(new)
