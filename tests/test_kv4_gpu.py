"""The 4-bit key/value cache on the GPU against 64-bit statements: where tiles, pages, masks, strides and types can go wrong."""
import math

import pytest
import torch

from kv4_oracle import Dense, attention64, rounded64
from llm_mojo_b200 import ops
from llm_mojo_b200.ops import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float32
UNIT = ops.kv4.KV4_UNIT


def rnd(*shape, dtype=FP, scale=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 13 * sum(shape))
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def assert_attention(got, q, dense, lens, counts, scale=None, what=""):
    """|error| against the 64-bit statement on the values that the cache holds.  Scores: products of the exact inputs, summed in fp32: an
    error of at most (head + 8) 2^-24 of sum |q k|, twice that in a weight relative to the others.  Weights in f16 on the tensor path
    (2^-11 of each, 2^-25 below f16's normals, and the sum of the rounded ones is not what they are divided by), sums over the keys in
    fp32 (at most one unit in the last place of the partial sums for each 16 keys, and one for each of up to 64 partial results).
    The result is rounded once."""
    want, mag = attention64(q, dense, lens, counts, scale)
    S, n, heads, hd = q.shape
    sc = 1 / math.sqrt(hd) if scale is None else abs(scale)
    group = heads // dense.k.shape[2]
    for s in range(S):
        c, L = counts[s], min(lens[s], dense.T)
        w, g, m = want[s, :c], got[s, :c].double(), mag[s, :c]
        assert torch.equal(torch.isnan(g), torch.isnan(w)), (what, s)
        if c == 0 or L == 0:
            assert not g.numel() or (g == 0).all(), (what, s)
            continue
        k = dense.k[s, :L].nan_to_num(0.0).abs().amax(0).repeat_interleave(group, 0)                       # [heads, hd]
        qk = (q[s, :c].double().abs().nan_to_num(0.0) * k).sum(-1) * sc                                    # >= |score| of any key
        delta = 2 * (hd + 8) * 2.0 ** -24 * qk + 2.0 ** -22 * qk + (L / 16 + 80) * 2.0 ** -23
        low = got.dtype == BF
        rel = 2.0 ** -8 if low else 2.0 ** -24
        tol = rel * w.abs() + ((2.0 ** -10 if low else 0.0) + delta).unsqueeze(-1) * m + L * 2.0 ** -24 * (2.0 ** -14 if low else 0.0) + 1e-30
        off = ((g - w).abs() - tol).nan_to_num(-1.0)
        assert off.max().item() <= 0, (what, s, off.max().item(), (g - w).abs().nan_to_num(0.0).max().item())


def filled(S, H, hd, lens, T, dtype=BF, seed=0, layers=1, layer=0, scale=1.0):
    c, d = ops.KV4Cache.empty(layers, S, H, T, hd, DEV), Dense(S, H, -(-T // 64) * 64, hd, device=DEV)
    n = max(max(lens), 1)
    k, v = rnd(S, n, H, hd, dtype=dtype, scale=scale, seed=seed), rnd(S, n, H, hd, dtype=dtype, seed=seed + 1)
    ops.kv4_append(c, layer, k, v, i32([0] * S), counts=i32(lens))
    d.append(k, v, [0] * S, lens)
    return c, d


# ------------------------------------------------------------------ write and read back
@pytest.mark.parametrize("hd", ops.kv4.KV4_HEAD_SIZES)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n", [1, 7, 130])
def test_append_then_values(hd, dtype, n):
    S, H, T = 3, 5, 192
    c = ops.KV4Cache.empty(2, S, H, T, hd, DEV)
    qkv = rnd(S, n, 3, H, hd, dtype=dtype, scale=2.0)
    k, v = qkv[:, :, 1], qkv[:, :, 2]
    start = [0, 61, T - 1]                                   # the last one runs out of the cache
    cnt = [n, max(0, n - 2), n]
    before = c.k_codes.clone()
    ops.kv4_append(c, 1, k, v, i32(start), counts=i32(cnt))
    assert torch.equal(c.k_codes[0], before[0])
    for out_dtype in (BF, FP):
        ko, vo = torch.full((S, n, H, hd), 9.0, dtype=out_dtype, device=DEV), torch.full((S, n, H, hd), 9.0, dtype=out_dtype, device=DEV)
        ops.kv4_values(ko, vo, c, 1, i32(start))
        for got, x in ((ko, k), (vo, v)):
            want = rounded64(x, UNIT)
            want[1, cnt[1]:] = 0.0                           # never written
            want[2, 1:] = 0.0                                # outside the cache
            assert torch.equal(got.double(), want)           # every value of the cache is exact in bf16
    # the same bytes as the statement in PyTorch writes
    cpu = ops.KV4Cache.empty(2, S, H, T, hd, "cpu")
    ops.kv4_append(cpu, 1, k.cpu(), v.cpu(), torch.tensor(start, dtype=torch.int32), counts=torch.tensor(cnt, dtype=torch.int32))
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(getattr(c, name).cpu(), getattr(cpu, name)), name


def test_append_of_midpoints_extremes_and_odd_addresses():
    hd, H = 64, 2
    level = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 0.0], device=DEV)
    rows = torch.stack([level.repeat(4) * s for s in (1.0, 448 * UNIT, 2.0 ** -9 * UNIT, 1.875 * 2.0 ** -6 * UNIT)] +
                       [level.repeat(4) * 1e30, level.repeat(4) * 1e-30, torch.zeros(hd, device=DEV), -level.repeat(4) * 7 * 2.0 ** -9 * UNIT])
    up, down = (torch.nextafter(rows, torch.full_like(rows, e)) for e in (math.inf, -math.inf))      # next to the midpoints
    x = torch.stack([rows, up, down]).view(1, -1, 1, hd).expand(1, -1, H, hd)
    n = x.shape[1]
    for shift in (0, 1):                                     # an address that no vector load takes
        buf = torch.zeros(n * H * hd + 1, device=DEV)
        k = buf[shift:shift + n * H * hd].view(1, n, H, hd)
        k.copy_(x)
        c = ops.KV4Cache.empty(1, 1, H, n, hd, DEV)
        ops.kv4_append(c, 0, k, -k, i32([0]))
        ko, vo = torch.empty_like(k), torch.empty(n * H * hd + 1, device=DEV)[shift:shift + n * H * hd].view(1, n, H, hd)
        ops.kv4_values(ko, vo, c, 0, i32([0]))
        want = rounded64(k, UNIT)
        assert torch.equal(ko.double(), want) and torch.equal(vo.double(), -want)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("unit", [2.0 ** -32, UNIT, 1.0, 2.0 ** 20])
def test_append_with_every_scale(dtype, unit):
    """Every scale with every midpoint between two levels, exact and (fp32) with its neighbours; rows that are not finite."""
    level = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0], dtype=torch.float64, device=DEV)
    scale = torch.arange(1, 127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()
    exact = (scale.view(-1, 1) * level).mul(unit).float()                    # [126, 16]: three bits times four
    x = torch.stack([exact, exact if dtype == BF else torch.nextafter(exact, exact * 2), exact if dtype == BF else torch.nextafter(exact, exact * 0)], 1)
    x = torch.cat([x.reshape(1, -1, 1, 16), torch.full((1, 6, 1, 16), 1e38, device=DEV) * level.float()], 1).to(dtype)
    x = x.reshape(1, -1, 1, 64)
    c = ops.KV4Cache(*(torch.zeros(1, 1, 1, 128, w, dtype=torch.uint8, device=DEV) for w in (32, 4, 32, 4)), k_unit=unit, v_unit=unit * 2)
    ops.kv4_append(c, 0, x, x * 2 if unit < 1e6 else x, i32([0]))
    ko, vo = (torch.empty(x.shape, device=DEV) for _ in range(2))
    ops.kv4_values(ko, vo, c, 0, i32([0]))
    want = rounded64(x.nan_to_num(0.0, 0.0, 0.0), unit)
    want[~torch.isfinite(x).all(-1)] = math.nan              # 6e38 is infinite
    assert torch.equal(ko.double().nan_to_num(7e7), want.nan_to_num(7e7))


def test_positions_before_the_cache_and_bad_pages():
    c, d = filled(2, 2, 64, [64, 64], 128)
    x = rnd(2, 4, 2, 64, dtype=BF, seed=9)
    ops.kv4_append(c, 0, x, x, i32([-2, 126]))
    d.k[0, :2], d.k[1, 126:128] = rounded64(x[0, 2:], UNIT), rounded64(x[1, :2], UNIT)
    pages = c.own_pages()
    pages[0, 1], pages[1, 0] = 1, 2                          # slot 2 is none
    ko, vo = (torch.empty(2, 132, 2, 64, device=DEV) for _ in range(2))
    ops.kv4_values(ko, vo, c, 0, i32([-2, -2]), pages=pages)
    assert (ko[:, :2] == 0).all() and (vo[:, 130:] == 0).all()
    assert torch.equal(ko[0, 2:66].double(), d.k[0, :64]) and torch.equal(ko[0, 66:130].double(), d.k[1, 64:128])
    assert torch.isnan(ko[1, 2:66]).all() and torch.isnan(vo[1, 2:66]).all() and torch.equal(ko[1, 66:130].double(), d.k[1, 64:128])


# ------------------------------------------------------------------ attention
LENS = [0, 1, 63, 64, 65, 777, 1000]


@pytest.mark.parametrize("hd", ops.kv4.KV4_HEAD_SIZES)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (6, 2), (8, 1), (9, 1), (20, 1)])
def test_attention_of_single_tokens(hd, dtype, heads, kv_heads):
    S = len(LENS)
    c, d = filled(S, kv_heads, hd, LENS, 1000, dtype)
    q = rnd(S, 1, heads, hd, dtype=dtype, seed=5)
    out = torch.full_like(q, 3.0)
    ops.attention_kv4(out, q, c, 0, i32(LENS))
    assert_attention(out, q, d, LENS, [1] * S)


@pytest.mark.parametrize("hd,heads,kv_heads", [(64, 3, 3), (64, 8, 2), (96, 2, 2), (128, 5, 1), (80, 2, 1), (32, 4, 4)])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n", [2, 5, 33, 130, 300])
def test_attention_of_many_tokens(hd, heads, kv_heads, dtype, n):
    """Prompts behind a cache, behind nothing, shorter than the rows, of no token at all, and with more rows than tokens."""
    lens = [n + 200, n, 700, 65, 0, max(1, n // 2)]
    counts = [n, n, max(1, n - 3), min(n, 65), 0, n]
    c, d = filled(len(lens), kv_heads, hd, lens, 700, dtype)
    q = rnd(len(lens), n, heads, hd, dtype=dtype, seed=5)
    out = torch.full_like(q, 3.0)
    ops.attention_kv4(out, q, c, 0, i32(lens), counts=i32(counts))
    assert_attention(out, q, d, lens, counts)
    for s, k in enumerate(counts):
        assert (out[s, k:] == 3.0).all()


@pytest.mark.parametrize("n", [1, 40, 200])
def test_attention_through_pages_strides_and_in_place(n):
    S, H, hd = 6, 4, 64
    lens = [300, 512, 448, 230, 512, 320]
    c, d = filled(S, H, hd, lens, 512, layers=3, layer=2)
    g = torch.Generator().manual_seed(2)
    pages = torch.randint(0, S, (S, 8), generator=g).to(torch.int32)
    for s in range(S):
        for p in range(8):
            if (p + 1) * 64 > lens[s] - n or lens[int(pages[s, p])] < (p + 1) * 64:
                pages[s, p] = s
    e = Dense(S, H, 512, hd, device=DEV)
    for s in range(S):
        for p in range(8):
            e.k[s, p * 64:p * 64 + 64], e.v[s, p * 64:p * 64 + 64] = d.k[pages[s, p], p * 64:p * 64 + 64], d.v[pages[s, p], p * 64:p * 64 + 64]
    qkv = rnd(S, n, 3, H, hd, dtype=BF, seed=5)
    q = qkv[:, :, 0]
    want_rest = qkv[:, :, 1:].clone()
    ref = q.clone()
    ops.attention_kv4(q, q, c, 2, i32(lens), pages=pages.to(DEV), scale=0.2)
    assert_attention(q, ref, e, lens, [n] * S, scale=0.2)
    assert torch.equal(qkv[:, :, 1:], want_rest)
    # every second slot of the cache; an output in another order, at an address that no vector store takes
    sub = c.select(slice(0, None, 2))
    f = Dense(3, H, 512, hd, device=DEV)
    f.k, f.v = d.k[::2], d.v[::2]
    buf = torch.zeros(H * 3 * n * (hd + 3) + 1, dtype=BF, device=DEV)[1:].view(H, 3, n, hd + 3)
    out = buf[..., :hd].permute(1, 2, 0, 3)
    ops.attention_kv4(out, ref[::2], sub, 2, i32(lens[::2]))
    assert_attention(out, ref[::2], f, lens[::2], [n] * 3)
    assert (buf[..., hd:] == 0).all()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n", [1, 6, 100])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, n):
    S, H, hd = 3, 2, 64
    lens = [200, 130, 320]
    c, d = filled(S, H, hd, lens, 512, dtype)
    q = rnd(S, n, 4, hd, dtype=dtype, seed=5)
    out = torch.empty_like(q)
    # the bytes behind the last token: all scales NaN, negative ones, the largest
    for byte in (0xff, 0x7f, 0x7e):
        for s in range(S):
            for t in (c.k_scales, c.v_scales, c.k_codes, c.v_codes):
                t[:, s, :, lens[s]:] = byte
        ops.attention_kv4(out, q, c, 0, i32(lens))
        assert_attention(out, q, d, lens, [n] * S, what=hex(byte))
    # a token with an infinite value: NaN for those who see it, nothing for those before it
    x, y = rnd(S, 1, H, hd, dtype=dtype, seed=7), rnd(S, 1, H, hd, dtype=dtype, seed=8)
    y[:, :, 1, 17] = math.inf
    x[:, :, 0, 3] = math.nan
    at = [n_ - max(1, n // 2) for n_ in lens]
    ops.kv4_append(c, 0, x, y, i32(at))
    d.append(x, y, at, [1] * S)
    ops.attention_kv4(out, q, c, 0, i32(lens))
    assert_attention(out, q, d, lens, [n] * S)
    assert torch.isnan(out[:, -1]).all() and (n < 4 or torch.isfinite(out[:, 0]).all())
    # a query with a NaN spoils its own row and head alone
    c, d = filled(S, H, hd, lens, 512, dtype)
    q[1, n // 2, 1, 5], q[2, n - 1, 0, 0] = math.nan, math.inf
    ops.attention_kv4(out, q, c, 0, i32(lens))
    bad = ~torch.isfinite(out).all(-1)
    want = torch.zeros_like(bad)
    want[1, n // 2, 1] = want[2, n - 1, 0] = True
    assert torch.equal(bad, want)


def test_attention_with_a_page_that_names_no_slot():
    c, d = filled(2, 2, 64, [300, 300], 320)
    q = rnd(2, 240, 2, 64, dtype=BF, seed=5)
    pages = c.own_pages()
    pages[0, 2], pages[1, 1] = -1, 7                         # tokens 128 .. 191 of slot 0, 64 .. 127 of slot 1
    out = torch.empty_like(q)
    ops.attention_kv4(out, q, c, 0, i32([300, 300]), pages=pages)
    pos = torch.arange(60, 300, device=DEV)
    assert torch.equal(torch.isnan(out).any(-1).any(-1), torch.stack([pos >= 128, pos >= 64]))
    assert torch.equal(torch.isnan(out).all(-1).all(-1), torch.stack([pos >= 128, pos >= 64]))
    one = torch.empty_like(q[:, :1])
    ops.attention_kv4(one, q[:, :1], c, 0, i32([128, 64]), pages=pages)      # the pages are there but not seen
    assert torch.isfinite(one).all()


def test_attention_with_extreme_scores_and_scales():
    """Scores that overflow an unshifted exponential, queries beyond f16's range, negative and zero scales, a flat row."""
    c, d = filled(2, 2, 64, [257, 100], 320, scale=20.0)
    for mul, scale in ((1.0, None), (1e4, 1e-3), (1e-6, 1e3), (3.0, -0.5), (1.0, 0.0)):
        q = rnd(2, 3, 2, 64, dtype=BF, scale=mul, seed=5)
        out = torch.empty_like(q)
        ops.attention_kv4(out, q, c, 0, i32([257, 100]), scale=scale)
        assert_attention(out, q, d, [257, 100], [3, 3], scale=scale, what=(mul, scale))
    q = torch.zeros(2, 1, 2, 64, dtype=BF, device=DEV)
    out = torch.empty_like(q)
    ops.attention_kv4(out, q, c, 0, i32([257, 100]))
    assert_attention(out, q, d, [257, 100], [1, 1])


def test_lens_and_counts_out_of_range_are_clamped():
    c, d = filled(4, 2, 64, [128] * 4, 128)
    q = rnd(4, 3, 2, 64, dtype=BF, seed=5)
    out = torch.full_like(q, 3.0)
    ops.attention_kv4(out, q, c, 0, i32([500, -4, 128, 2]), counts=i32([9, 3, -1, 3]))
    assert_attention(out, q, d, [128, 0, 128, 2], [3, 3, 0, 3])
    assert (out[2] == 3.0).all() and (out[1] == 0).all() and (out[3, 0] == 0).all()


def test_offsets_beyond_32_bits():
    """Slots that lie further apart than 32 bits reach, and a slot whose own rows do."""
    hd, H, T = 64, 2, 128
    gap = (1 << 32) + 4096
    size = gap + H * T * hd // 2
    big = [torch.empty(size, dtype=torch.uint8, device=DEV) for _ in range(2)]
    sgap = gap // 4
    small = [torch.empty(sgap + H * T * hd // 16, dtype=torch.uint8, device=DEV) for _ in range(2)]
    view = lambda t, c, s: t.as_strided((1, 2, H, T, c), (2 * s, s, T * c, c, 1))  # noqa: E731
    c = ops.KV4Cache(view(big[0], hd // 2, gap), view(small[0], hd // 16, sgap), view(big[1], hd // 2, gap), view(small[1], hd // 16, sgap))
    d = Dense(2, H, T, hd, device=DEV)
    k, v = rnd(2, 100, H, hd, dtype=BF), rnd(2, 100, H, hd, dtype=BF, seed=1)
    ops.kv4_append(c, 0, k, v, i32([0, 0]))
    d.append(k, v, [0, 0], [100, 100])
    for n in (1, 70):
        q = rnd(2, n, H, hd, dtype=BF, seed=5)
        out = torch.empty_like(q)
        ops.attention_kv4(out, q, c, 0, i32([100, 100]))
        assert_attention(out, q, d, [100, 100], [n, n])
    pages, lens = c.own_pages(), i32([100, 100])
    ops.kv4_reorder(c, pages, lens, i32([[1, 1]]))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.kv4_values(ko, vo, c, 0, i32([0, 0]), pages=pages)
    assert torch.equal(ko[0].double(), d.k[1, :100]) and torch.equal(vo[1].double(), d.v[1, :100])
    del big, small, c
    T = 1 << 20                                              # a cache row of 2^20 tokens x 48 heads x 64 bytes: 3.2 GB in one slot
    c = ops.KV4Cache(*(torch.zeros(1, 1, 72, T, w, dtype=torch.uint8, device=DEV) for w in (64, 8, 64, 8)))
    k = rnd(1, 3, 72, 128, dtype=BF)
    ops.kv4_append(c, 0, k, k, i32([T - 3]))
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    ops.kv4_values(ko, vo, c, 0, i32([T - 3]))
    assert torch.equal(ko.double(), rounded64(k, UNIT)) and torch.equal(vo, ko)
    d = Dense(1, 72, 3, 128, device=DEV)
    c3 = ops.KV4Cache.empty(1, 1, 72, 64, 128, DEV)
    ops.kv4_append(c3, 0, k, k, i32([0]))
    d.append(k, k, [0], [3])
    q = rnd(1, 1, 72, 128, dtype=BF, seed=5)
    out = torch.empty_like(q)
    ops.attention_kv4(out, q, c, 0, i32([T]))               # 2^20 - 3 keys of zeros beside the three
    w = torch.softmax(torch.cat([torch.zeros(72, 1, dtype=torch.float64, device=DEV) + math.log(T - 3),
                                 torch.einsum("hd,lhd->hl", q[0, 0].double(), d.k[0]) / math.sqrt(128)], -1), -1)
    want = torch.einsum("hl,lhd->hd", w[:, 1:], d.v[0])
    mag = torch.einsum("hl,lhd->hd", w[:, 1:], d.v[0].abs())
    # a million equal weights: their sum in fp32 is exact to 2^-24 for each of the partial sums that it is taken in
    assert ((out[0, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -8 * mag + T * 2.0 ** -24 * 1e-3 * mag + 1e-12).all()


# ------------------------------------------------------------------ reorder
@pytest.mark.parametrize("hd,layers,items,K,H", [(64, 2, 3, 4, 3), (80, 1, 2, 16, 2), (128, 3, 1, 64, 1), (32, 1, 5, 1, 2), (96, 2, 1, 5, 7)])
def test_reorder_is_the_statement_in_pytorch(hd, layers, items, K, H):
    S, T = items * K, 256
    g = torch.Generator().manual_seed(hd)
    cpu = ops.KV4Cache(*(torch.randint(0, 256, (layers, S, H, T, w), generator=g, dtype=torch.uint8) for w in (hd // 2, hd // 16, hd // 2, hd // 16)))
    gpu = ops.KV4Cache(*(getattr(cpu, n).to(DEV) for n in ("k_codes", "k_scales", "v_codes", "v_scales")))
    for trial in range(4):
        lens = torch.randint(0, T + 1, (S,), generator=g, dtype=torch.int32)
        lens[0] = (0, 64, T, T + 9)[trial]
        lens[-1] = (-1, 63, 65, 128)[trial]
        pages = torch.randint(0, S, (S, T // 64), generator=g, dtype=torch.int32)
        parents = torch.randint(0, K, (items, K), generator=g, dtype=torch.int32)
        if trial == 2:
            parents[0, 0], parents[-1, -1] = -1, K           # no parents: they stay what they are
        lg, pg = lens.to(DEV), pages.to(DEV)
        ops.kv4_reorder(cpu, pages, lens, parents)
        ops.kv4_reorder(gpu, pg, lg, parents.to(DEV))
        assert torch.equal(lg.cpu(), lens) and torch.equal(pg.cpu(), pages)
        for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
            assert torch.equal(getattr(gpu, name).cpu(), getattr(cpu, name)), (trial, name)


def test_a_run_of_appends_attentions_and_reorders():
    """As a beam search uses them: the cache in pages stays what dense copies of the beams are."""
    items, K, H, hd, T = 2, 4, 3, 64, 256
    S = items * K
    c, d = ops.KV4Cache.empty(2, S, H, T, hd, DEV), Dense(S, H, T, hd, device=DEV)
    pages, lens = c.own_pages(), i32([0] * S)
    g = torch.Generator().manual_seed(3)
    for step, n in enumerate((50, 14, 1, 1, 60, 1, 3, 70, 1)):
        k, v, q = (rnd(S, n, H, hd, dtype=BF, seed=10 * step + i) for i in range(3))
        before = lens.clone()
        lens += n
        for l in range(2):
            ops.kv4_append(c, l, k, v, before)
            out = torch.empty_like(q)
            if l == 0:
                d.append(k, v, before.tolist(), [n] * S)
            ops.attention_kv4(out, q, c, l, lens, pages=pages)
            assert_attention(out, q, d, lens.tolist(), [n] * S, what=(step, l))
        parents = torch.randint(0, K, (items, K), generator=g, dtype=torch.int32)
        ops.kv4_reorder(c, pages, lens, parents.to(DEV))
        d.reorder([b * K + p for b, row in enumerate(parents.tolist()) for p in row])


# ------------------------------------------------------------------ streams and graphs
def test_operators_follow_the_current_stream_and_replay_in_graphs():
    S, H, hd = 4, 3, 64
    c, d = filled(S, H, hd, [100] * S, 512)
    lens, start = i32([100] * S), i32([0] * S)
    k, v, q = (torch.empty(S, 1, H, hd, dtype=BF, device=DEV) for _ in range(3))
    outs = [torch.empty_like(q) for _ in range(2)]

    def step(out):
        start.copy_(lens)
        lens.add_(1)
        ops.kv4_append(c, 0, k, v, start)
        ops.attention_kv4(out, q, c, 0, lens)

    def fill(i):
        for j, t in enumerate((k, v, q)):
            t.copy_(rnd(S, 1, H, hd, dtype=BF, seed=100 * i + j))

    side = torch.cuda.Stream()
    fill(0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(outs[0])
    side.synchronize()
    d.append(k, v, [100] * S, [1] * S)
    assert_attention(outs[0], q, d, [101] * S, [1] * S)
    graphs = []
    for out in outs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(out)
        graphs.append(gr)
    assert lens.tolist() == [101] * S                        # capture runs nothing
    for i in range(1, 7):
        fill(i)
        graphs[i % 2].replay()
        d.append(k, v, [100 + i] * S, [1] * S)
        assert_attention(outs[i % 2], q, d, [101 + i] * S, [1] * S, what=i)
    assert _lib.read_status() == 0


def test_the_same_inputs_give_the_same_bits():
    c, _ = filled(3, 4, 64, [700, 33, 512], 768)
    for n in (1, 50):
        q = rnd(3, n, 8, 64, dtype=BF, seed=5)
        outs = [torch.empty_like(q) for _ in range(3)]
        for o in outs:
            ops.attention_kv4(o, q, c, 0, i32([700, 33, 512]), counts=i32([n, min(n, 33), n]))
        torch.cuda.synchronize()
        assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[1][2], outs[2][2])


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_blocks_around_the_smallest_scale_are_the_statement_in_pytorch(dtype):
    """To the byte, signs of zeros too: amounts on both sides of the ties between no scale, the smallest and the next."""
    S, H, hd = 4, 2, 64
    x = rnd(S, 3, H, hd, dtype=torch.float32, seed=5)
    x = (x / x.abs().unflatten(-1, (-1, 16)).amax(-1, keepdim=True).expand(S, 3, H, 4, 16).flatten(-2)).float()
    top = torch.tensor([2.0 ** -10 * f for f in (0.5, 0.99, 1.0, 1.01, 1.5, 2.0, 2.99, 3.0, 3.01, 4.0, 5.0, 7.0)], device=DEV).view(S, 3, 1, 1)
    x = (x * top * 6 * 2.0 ** -4).to(dtype)
    start = [0, 5, 61, 100]
    gpu, cpu = ops.KV4Cache.empty(1, S, H, 128, hd, DEV), ops.KV4Cache.empty(1, S, H, 128, hd, "cpu")
    ops.kv4_append(gpu, 0, x, -x, i32(start))
    ops.kv4_append(cpu, 0, x.cpu(), -x.cpu(), torch.tensor(start, dtype=torch.int32))
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(getattr(gpu, name).cpu(), getattr(cpu, name)), name


@pytest.mark.parametrize("hd", ops.kv4.KV4_HEAD_SIZES)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("cap,lens", [(2048, [2048, 1]), (2560, [1300, 2499]), (8192, [8192, 0]), (8192, [65, 4097])])
def test_few_long_texts_over_many_blocks(hd, dtype, cap, lens):
    """Capacities at which one, two and up to sixteen blocks join; lengths that leave all but one of them, or part of a tile, without keys."""
    c, d = filled(2, 1, hd, lens, cap, dtype, seed=cap)
    q = rnd(2, 1, 3, hd, dtype=dtype, seed=hd)
    out = torch.empty_like(q)
    ops.attention_kv4(out, q, c, 0, i32(lens))
    assert_attention(out, q, d, lens, [1, 1], what=(hd, cap, lens))


def test_calls_on_two_streams_at_once_over_views_of_one_cache():
    """Two halves of a larger cache's slots (every other one), the second of its layers, appended to and attended to on a stream each."""
    S, H, hd, n = 6, 2, 64, 90
    whole = ops.KV4Cache.empty(3, S, H, 192, hd, DEV)
    views = [ops.KV4Cache(*(getattr(whole, name)[1:, i::2] for name in ("k_codes", "k_scales", "v_codes", "v_scales"))) for i in range(2)]
    k, v = rnd(S, n, H, hd, dtype=BF, seed=1), rnd(S, n, H, hd, dtype=BF, seed=2)
    q = rnd(S, 1, H, hd, dtype=BF, seed=3)
    d = Dense(S, H, 192, hd, device=DEV)
    d.append(k, v, [20] * S, [n] * S)
    out = torch.full_like(q, 3.0)
    lens, start = i32([110] * 3), i32([20] * 3)
    streams = [torch.cuda.Stream() for _ in views]
    torch.cuda.synchronize()
    for i, (view, stream) in enumerate(zip(views, streams)):
        with torch.cuda.stream(stream):
            for _ in range(5):
                ops.kv4_append(view, 0, k[i::2], v[i::2], start)
                ops.attention_kv4(out[i::2], q[i::2], view, 0, lens)
    torch.cuda.synchronize()
    assert_attention(out, q, d, [110] * S, [1] * S)
    assert not whole.k_codes[0].any() and not whole.k_codes[2].any() and bool(whole.k_codes[1].any())


@pytest.mark.parametrize("dtype", [BF, FP])
def test_zeros_keep_their_signs(dtype):
    """Zeros of both signs among other values, and values so small that they round to one: the code of a negative one is 8, as in the statement
    in PyTorch, to the byte; only a block without a scale keeps no signs."""
    S, n, H, hd = 2, 5, 3, 64
    x = rnd(S, n, H, hd, dtype=dtype, seed=3)
    x[..., 0::5], x[..., 1::5] = 0.0, -0.0
    x[..., 2::5] = -1e-30
    x[0, 0, 0] = -0.0
    x[1, 4, 2, :16], x[1, 4, 2, 16] = -0.0, 7.0
    start = [0, 61]
    gpu, cpu = ops.KV4Cache.empty(1, S, H, 128, hd, DEV), ops.KV4Cache.empty(1, S, H, 128, hd, "cpu")
    ops.kv4_append(gpu, 0, x, -x, i32(start))
    ops.kv4_append(cpu, 0, x.cpu(), -x.cpu(), torch.tensor(start, dtype=torch.int32))
    for name in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(getattr(gpu, name).cpu(), getattr(cpu, name)), name
    ko, vo = torch.empty_like(x), torch.empty_like(x)
    ops.kv4_values(ko, vo, gpu, 0, i32(start))
    scaled = (x.unflatten(-1, (-1, 16)).abs().amax(-1, keepdim=True) > 0.01).expand(S, n, H, 4, 16).flatten(-2)
    assert torch.equal(torch.signbit(ko), torch.signbit(x) & scaled) and torch.equal(torch.signbit(vo), ~torch.signbit(x) & scaled)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("unit", [2.0 ** -32, UNIT, 2.0 ** 20])
def test_scales_around_every_midpoint(dtype, unit):
    """The largest value of a block on every midpoint between two scales (five bits times six: exact in both types) and, for fp32, next to it on
    both sides: the scale's byte, and the values, by the definition in 64 bits.  A quotient by 6 that is rounded more than once would reach the midpoint."""
    scale = torch.arange(0, 127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()
    top = ((scale[1:] + scale[:-1]) / 2 * 6 * unit).float()
    top = torch.stack([top, top if dtype == BF else torch.nextafter(top, top * 2), top if dtype == BF else torch.nextafter(top, top * 0)], 1).to(dtype)
    want = torch.bucketize(top.double() / 6 / unit, (scale[1:] + scale[:-1]) / 2)          # of equals the lower place: a tie, then
    tie = top.double() / 6 / unit == ((scale[1:] + scale[:-1]) / 2).view(-1, 1)
    want = torch.where(tie & (want % 2 == 1), want + 1, want)
    x = (rnd(126, 3, 64, dtype=FP, seed=11).clamp(-1, 1) * top.unsqueeze(-1).float()).to(dtype)
    x[..., 5::16] = -top.unsqueeze(-1)
    x = x.view(1, -1, 1, 64)
    c = ops.KV4Cache(*(torch.zeros(1, 1, 1, 384, w, dtype=torch.uint8, device=DEV) for w in (32, 4, 32, 4)), k_unit=unit, v_unit=unit)
    ops.kv4_append(c, 0, x, -x, i32([0]))
    assert torch.equal(c.k_scales[0, 0, 0, :378].long(), want.view(-1, 1).expand(378, 4)) and torch.equal(c.v_scales, c.k_scales)
    ko, vo = (torch.empty(x.shape, device=DEV) for _ in range(2))
    ops.kv4_values(ko, vo, c, 0, i32([0]))
    assert torch.equal(ko.double(), rounded64(x, unit)) and torch.equal(vo, -ko)


@pytest.mark.parametrize("S,heads,kv_heads,n,ragged,paged", [
    (16, 12, 12, 320, True, False),                          # three tiles: two that share a stream of keys, and one beside an empty one
    (16, 12, 12, 320, True, True),
    (40, 12, 3, 100, True, False),                           # rows of four heads over one
    (160, 2, 2, 300, True, True),                            # more pairs of tiles than are sorted by their cost
    (160, 2, 2, 300, False, False),
    (9, 20, 20, 384, False, True),
])
def test_prompts_of_more_items_than_the_chip_has_places(S, heads, kv_heads, n, ragged, paged):
    """Each block of the kernel for prompts takes several items in turn: texts that see nothing, have no rows, rows in one tile of two or one row in
    the second, fewer keys than rows; a capacity that ends inside a block of 128 keys.  The same bits every time."""
    hd, T = 64, 832
    tiles = -(-n * heads // kv_heads // 128)
    assert -(-tiles // 2) * kv_heads * S > torch.cuda.get_device_properties(0).multi_processor_count      # or a block has no second item
    kinds = [(n + 400, n), (0, n), (n // 2, n), (n + 7, 0), (T, 1), (T, n), (n + 130, 129 * kv_heads // heads + 1), (n, 128 * kv_heads // heads), (n, n)]
    lens, counts = zip(*(kinds[(5 * s + s // 9) % 9] for s in range(S)))
    lens, counts = [min(x, T) for x in lens], list(counts) if ragged else [n] * S
    c, d = filled(S, kv_heads, hd, lens, T)
    pages = None
    if paged:                                                # any page of any text: what lies there is read as it is
        pages = torch.randint(0, S, (S, T // 64), generator=torch.Generator().manual_seed(4)).to(torch.int32)
        e = Dense(S, kv_heads, T, hd, device=DEV)
        at = pages.to(DEV).long().repeat_interleave(64, 1), torch.arange(T, device=DEV)
        e.k, e.v = d.k[at], d.v[at]
        d, pages = e, pages.to(DEV)
    q = rnd(S, n, heads, hd, dtype=BF, seed=5)
    outs = [torch.full_like(q, 3.0) for _ in range(3)]
    for out in outs:
        ops.attention_kv4(out, q, c, 0, i32(lens), counts=i32(counts) if ragged else None, pages=pages)
    assert_attention(outs[0], q, d, lens, counts)
    assert all((outs[0][s, k:] == 3.0).all() for s, k in enumerate(counts))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and _lib.read_status() == 0


def test_many_query_heads_over_a_long_text_share_its_keys():
    """Sixty and sixty-four query heads over one key head are the same work: no form of the operator may leave a long text to a single block.
    (It took sixteen times as long; four is far from both.)"""
    c = ops.KV4Cache.empty(1, 1, 1, 30016, 64, DEV)
    d = Dense(1, 1, 30016, 64, device=DEV)
    k, v = rnd(1, 3000, 1, 64, dtype=BF), rnd(1, 3000, 1, 64, dtype=BF, seed=1)
    for at in range(0, 30000, 3000):
        ops.kv4_append(c, 0, k.roll(at // 3000, 1), v, i32([at]))
        d.append(k.roll(at // 3000, 1), v, [at], [3000])
    took = {}
    for heads in (60, 64):
        q = rnd(1, 1, heads, 64, dtype=BF, seed=heads)
        out = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        ops.attention_kv4(out, q, c, 0, i32([30000]))
        lens = i32([30000])
        with torch.cuda.graph(graph):
            for _ in range(20):
                ops.attention_kv4(out, q, c, 0, lens)
        graph.replay()
        a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        z.record()
        z.synchronize()
        took[heads] = a.elapsed_time(z)
        assert_attention(out, q, d, [30000], [1])
    assert took[64] < 4 * took[60], took


def assert_lagging_attention(got, q, dense, lens, counts, scale=None, what=""):
    """``assert_attention`` for bf16 and a maximum that may lag.  A row's weights are 2^(7 + s - m) for the largest score m of some keys that the row
    has seen, so that the weight of that key is 2^7 and the sum of all at least as much.  A weight is rounded to f16: by 2^-11 of itself, or, below
    f16's smallest normal number, by half of 2^-24.  That is 2^-25 / 2^7 = 2^-32 of the sum for each key, whatever the other weights: 2^-32 sum |v|
    beside the terms of ``assert_attention``, which takes the largest weight for 2^13 and more."""
    want, mag = attention64(q, dense, lens, counts, scale)
    S, n, heads, hd = q.shape
    group, sc = heads // dense.k.shape[2], 1 / math.sqrt(hd) if scale is None else abs(scale)
    for s in range(S):
        c, L = counts[s], min(lens[s], dense.T)
        w, g = want[s, :c], got[s, :c].double()
        assert torch.equal(torch.isnan(g), torch.isnan(w)), (what, s)
        k, v = (x[s, :L].nan_to_num(0.0).abs().repeat_interleave(group, 1) for x in (dense.k, dense.v))
        qk = (q[s, :c].double().abs().nan_to_num(0.0) * (k.amax(0) if L else 0.0)).sum(-1) * sc
        delta = 2.0 ** -10 + 2 * (hd + 8) * 2.0 ** -24 * qk + 2.0 ** -22 * qk + (L / 16 + 80) * 2.0 ** -23
        tol = 2.0 ** -8 * w.abs() + delta.unsqueeze(-1) * mag[s, :c] + 2.0 ** -32 * v.sum(0) + 1e-30
        off = ((g - w).abs() - tol).nan_to_num(-1.0)
        assert not off.numel() or off.max().item() <= 0, (what, s, off.max().item())


@pytest.mark.parametrize("T", [320, 832])
def test_prompts_on_the_tensor_memory_kernel(T):
    """Sixteen texts of twelve heads, 200 rows: in place among packed values, through strides at odd addresses, with extreme scales, queries, values
    and pages that are not finite, and bytes behind the last token."""
    S, H, hd, n = 16, 12, 64, 200
    lens = [T - 17 * (s % 4) if s % 3 else n + s for s in range(S)]
    c, d = filled(S, H, hd, lens, T)
    for byte in (0xff, 0x7e):                                # behind the last token: NaN, the largest
        for s in range(S):
            for t in (c.k_scales, c.v_scales, c.k_codes, c.v_codes):
                t[:, s, :, lens[s]:] = byte
    qkv = rnd(S, n, 3, H, hd, dtype=BF, seed=5)
    q, rest = qkv[:, :, 0], qkv[:, :, 1:].clone()
    ref = q.clone()
    for scale in (None, -0.3, 0.0, 1e3):
        q.copy_(ref if scale != 1e3 else ref * 1e-3)
        want = q.clone()
        ops.attention_kv4(q, q, c, 0, i32(lens), scale=scale)
        assert_lagging_attention(q, want, d, lens, [n] * S, scale=scale, what=scale)
        assert torch.equal(qkv[:, :, 1:], rest)
    buf = torch.zeros(H * S * n * (hd + 3) + 1, dtype=BF, device=DEV)[1:].view(H, S, n, hd + 3)
    odd = torch.empty(S * n * H * hd + 1, dtype=BF, device=DEV)[1:].view(S, n, H, hd)
    odd.copy_(ref)
    out = buf[..., :hd].permute(1, 2, 0, 3)
    ops.attention_kv4(out, odd, c, 0, i32(lens))
    assert_lagging_attention(out, odd, d, lens, [n] * S)
    assert (buf[..., hd:] == 0).all()
    # a query that is not finite spoils its own row; a key or value its token and head, for those that see it
    odd[3, 7, 2, 5], odd[9, 199, 11, 0] = math.nan, math.inf
    ops.attention_kv4(out, odd, c, 0, i32(lens))
    bad = torch.zeros(S, n, H, dtype=torch.bool, device=DEV)
    bad[3, 7, 2] = bad[9, 199, 11] = True
    assert torch.equal(~torch.isfinite(out).all(-1), bad)
    x, y = rnd(S, 1, H, hd, dtype=BF, seed=7), rnd(S, 1, H, hd, dtype=BF, seed=8)
    x[:, :, 1, 3], y[:, :, 4, 17] = math.nan, math.inf
    at = [L - n // 2 for L in lens]
    ops.kv4_append(c, 0, x, y, i32(at))
    d.append(x, y, at, [1] * S)
    ops.attention_kv4(out, ref, c, 0, i32(lens))
    assert_lagging_attention(out, ref, d, lens, [n] * S)
    assert torch.isnan(out[:, -1, 1]).all() and torch.isnan(out[:, -1, 4]).all() and torch.isfinite(out[:, :n // 2]).all()
    pages = c.own_pages()
    pages[2, 1], pages[5, 4] = -1, S                         # tokens 64 .. 127 of one text, 256 .. 319 of another
    c, d = filled(S, H, hd, lens, T, seed=3)
    ops.attention_kv4(out, ref, c, 0, i32(lens), pages=pages)
    pos = i32(lens).view(S, 1) - n + torch.arange(n, device=DEV)
    bad = torch.zeros(S, n, dtype=torch.bool, device=DEV)
    bad[2], bad[5] = pos[2] >= 64, pos[5] >= 256
    assert torch.equal(torch.isnan(out).all(-1).all(-1), bad) and torch.equal(torch.isnan(out).any(-1).any(-1), bad)
    assert _lib.read_status() == 0
