"""The 4-bit key/value cache and the beam selection on CPU tensors: definitions against 64-bit statements, and what is refused."""
import math

import pytest
import torch

from kv4_oracle import Dense, attention64, rounded64, select64
from llm_mojo_b200 import ops


def rnd(*shape, dtype=torch.float32, scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed + 13 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("hd", ops.kv4.KV4_HEAD_SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_then_values_is_the_rounding(hd, dtype):
    c = ops.KV4Cache.empty(2, 3, 2, 100, hd, "cpu")
    k, v = rnd(3, 5, 2, hd, dtype=dtype, scale=3.0), rnd(3, 5, 2, hd, dtype=dtype, scale=0.01, seed=1)
    ops.kv4_append(c, 1, k, v, i32(0, 60, 125), counts=i32(5, 5, 5))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.kv4_values(ko, vo, c, 1, i32(0, 60, 125))
    for got, x in ((ko, k), (vo, v)):
        want = rounded64(x, ops.kv4.KV4_UNIT)
        want[2, 3:] = 0.0                                    # positions 128, 129 of a capacity of 128
        assert torch.equal(got.double(), want)
    assert not c.k_codes[0].any() and not c.v_scales[0].any()


def test_attention_is_causal_and_rows_behind_the_counts_stay():
    c = ops.KV4Cache.empty(1, 2, 2, 64, 32, "cpu")
    d = Dense(2, 2, 64, 32)
    k, v = rnd(2, 9, 2, 32), rnd(2, 9, 2, 32, seed=1)
    ops.kv4_append(c, 0, k, v, i32(0, 0), counts=i32(9, 4))
    d.append(k, v, [0, 0], [9, 4])
    q = rnd(2, 5, 6, 32, seed=2)
    out = torch.full_like(q, 7.0)
    ops.attention_kv4(out, q, c, 0, i32(9, 4), counts=i32(5, 3))
    want, _ = attention64(q, d, [9, 4], [5, 3])
    assert torch.allclose(out[0].double(), want[0], atol=1e-5) and torch.allclose(out[1, :3].double(), want[1, :3], atol=1e-5)
    assert (out[1, 3:] == 7.0).all()


def test_reorder_follows_dense_copies_of_the_beams():
    items, K, H, hd, T = 2, 3, 2, 32, 192
    S = items * K
    c, d = ops.KV4Cache.empty(2, S, H, T, hd, "cpu"), Dense(S, H, T, hd)
    pages, lens = c.own_pages(), torch.zeros(S, dtype=torch.int32)
    g = torch.Generator().manual_seed(3)
    for step, n in enumerate((50, 14, 1, 63, 2, 30)):
        k, v = rnd(S, n, H, hd, seed=step), rnd(S, n, H, hd, seed=100 + step)
        for l in range(2):
            ops.kv4_append(c, l, k, v, lens)
        d.append(k, v, lens.tolist(), [n] * S)
        lens += n
        parents = torch.randint(0, K, (items, K), generator=g, dtype=torch.int32)
        ops.kv4_reorder(c, pages, lens, parents)
        d.reorder([b * K + p for b, row in enumerate(parents.tolist()) for p in row])
        L = int(lens[0])
        ko, vo = torch.empty(2, S, L, H, hd), torch.empty(2, S, L, H, hd)
        ops.kv4_values(ko, vo, c, None, torch.zeros(S, dtype=torch.int32), pages)
        assert torch.equal(ko[1].double(), d.k[:, :L]) and torch.equal(vo[0].double(), d.v[:, :L])


@pytest.mark.parametrize("K,V", [(1, 5), (4, 4), (3, 50), (8, 5000)])
def test_beam_select_is_the_definition(K, V):
    B = 3
    logits = rnd(B * K, V + 3, dtype=torch.bfloat16, scale=2.0)
    scores = -rnd(B, K).abs()
    finished = torch.rand(B, K, generator=torch.Generator().manual_seed(1)) < 0.3
    so, t, p, f = torch.empty(B, K), torch.empty(B, K, dtype=torch.int32), torch.empty(B, K, dtype=torch.int32), torch.empty(B, K, dtype=torch.bool)
    ops.beam_select(so, t, p, logits, scores, V, finished_out=f, finished=finished, eos=2)
    w = select64(logits, scores, V, finished, 2)
    assert torch.equal(t.long(), w[1]) and torch.equal(p.long(), w[2]) and torch.equal(f, w[3])
    assert torch.allclose(so.double(), w[0], rtol=1e-6)


def _cache(**kw):
    a = dict(layers=1, slots=2, kv_heads=2, max_len=64, head_size=64, device="cpu")
    return ops.KV4Cache.empty(**{**a, **kw})


def test_cache_refusals():
    c = _cache()
    t = (c.k_codes, c.k_scales, c.v_codes, c.v_scales)
    with pytest.raises(ValueError, match="head size"):
        _cache(head_size=72)
    with pytest.raises(ValueError, match="power of two"):
        ops.KV4Cache(*t, k_unit=0.1)
    with pytest.raises(ValueError, match="power of two"):
        ops.KV4Cache(*t, v_unit=float("nan"))
    with pytest.raises(ValueError, match="k_scales"):
        ops.KV4Cache(t[0], t[1][..., :2], t[2], t[3])
    with pytest.raises(ValueError, match="v_codes"):
        ops.KV4Cache(t[0], t[1], t[2].to(torch.int8), t[3])
    with pytest.raises(ValueError, match="capacity"):
        ops.KV4Cache(*(x[:, :, :, :32] for x in t))
    with pytest.raises(ValueError, match="densely"):
        ops.KV4Cache(*(x.transpose(1, 2).contiguous().transpose(1, 2) for x in t))
    with pytest.raises(ValueError, match="overlap"):
        ops.KV4Cache(*(x[:, :1].expand(1, 2, *x.shape[2:]) for x in t))
    with pytest.raises(ValueError, match="layers"):
        ops.KV4Cache(*(x[0] for x in t))
    with pytest.raises(ValueError, match="2\\^30"):
        ops.KV4Cache(*(torch.empty(1, 1, 1, 2 ** 31, c, dtype=torch.uint8, device="meta") for c in (32, 4, 32, 4)))
    assert c.select(slice(0, None, 2)).slots == 1
    assert _cache(layers=2, slots=6).select(slice(0, None, 4)).slots == 2
    with pytest.raises(ValueError, match="overlap"):
        ops.KV4Cache(*(x.as_strided((2, 2, *x.shape[2:]), (x.stride(1) * 3 // 2 // 16 * 16, x.stride(1), *x.stride()[2:]))
                       for x in (lambda y: (y.k_codes, y.k_scales, y.v_codes, y.v_scales))(_cache(slots=4))))


def test_append_and_values_refusals():
    c, x, z = _cache(), torch.zeros(2, 3, 2, 64), i32(0, 0)
    for bad in (torch.zeros(2, 3, 2, 32), torch.zeros(1, 3, 2, 64), torch.zeros(2, 3, 64)):
        with pytest.raises(ValueError):
            ops.kv4_append(c, 0, bad, bad, z)
    with pytest.raises(TypeError):
        ops.kv4_append(c, 0, x.half(), x.half(), z)
    with pytest.raises(ValueError, match="v must be"):
        ops.kv4_append(c, 0, x, x.bfloat16(), z)
    with pytest.raises(ValueError, match="densely"):
        ops.kv4_append(c, 0, torch.zeros(2, 3, 2, 128)[..., ::2], x, z)
    with pytest.raises(ValueError, match="layer"):
        ops.kv4_append(c, 1, x, x, z)
    with pytest.raises(ValueError, match="start"):
        ops.kv4_append(c, 0, x, x, z.long())
    with pytest.raises(ValueError, match="counts"):
        ops.kv4_append(c, 0, x, x, z, counts=i32(1))
    with pytest.raises(ValueError, match="overlap"):
        ops.kv4_values(torch.zeros(2, 1, 2, 64).expand(2, 3, 2, 64), x, c, 0, z)
    with pytest.raises(ValueError, match="k_out"):
        ops.kv4_values(x, x.clone(), c, None, z)
    with pytest.raises(ValueError, match="same memory"):
        ops.kv4_values(x, x, c, 0, z)
    with pytest.raises(ValueError, match="pages"):
        ops.kv4_values(x, x.clone(), c, 0, z, pages=torch.zeros(2, 2, dtype=torch.int32))
    ops.kv4_append(c, 0, x[:, :0], x[:, :0], z)              # nothing to do is no error


def test_attention_refusals():
    c, q, n = _cache(), torch.zeros(2, 1, 4, 64), i32(1, 1)
    for bad in (torch.zeros(2, 1, 3, 64), torch.zeros(2, 1, 4, 32), torch.zeros(3, 1, 4, 64), torch.zeros(2, 4, 64), torch.zeros(2, 1, 0, 64)):
        with pytest.raises(ValueError, match="q must be"):
            ops.attention_kv4(bad.clone(), bad, c, 0, n)
    with pytest.raises(TypeError):
        ops.attention_kv4(q.half(), q.half(), c, 0, n)
    with pytest.raises(ValueError, match="out must be"):
        ops.attention_kv4(q.bfloat16(), q, c, 0, n)
    with pytest.raises(ValueError, match="overlap"):
        ops.attention_kv4(torch.zeros(1, 1, 4, 64).expand(2, 1, 4, 64), q, c, 0, n)
    with pytest.raises(ValueError, match="lens"):
        ops.attention_kv4(q.clone(), q, c, 0, torch.ones(2, 2, dtype=torch.int32)[:, 0])
    with pytest.raises(ValueError, match="scale"):
        ops.attention_kv4(q.clone(), q, c, 0, n, scale=float("inf"))
    with pytest.raises(ValueError, match="layer"):
        ops.attention_kv4(q.clone(), q, c, -1, n)


def test_reorder_and_select_refusals():
    c = _cache(slots=6)
    pages, lens, par = c.own_pages(), torch.zeros(6, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="parents"):
        ops.kv4_reorder(c, pages, lens, par[:1])
    with pytest.raises(ValueError, match="parents"):
        ops.kv4_reorder(c, pages, lens, par.long())
    with pytest.raises(ValueError, match="pages"):
        ops.kv4_reorder(c, pages[:, :0], lens, par)
    with pytest.raises(ValueError, match="needed"):
        ops.kv4_reorder(c, None, lens, par)
    so, t, p = torch.empty(2, 3), par.clone(), par.clone()
    x, s = torch.zeros(6, 10), torch.zeros(2, 3)
    with pytest.raises(ValueError, match="logits"):
        ops.beam_select(so, t, p, x[:5], s, 10)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.beam_select(so, t, p, x, s, 11)
    with pytest.raises(ValueError, match="vocabulary"):
        ops.beam_select(so, t, p, x, s, 2)                   # fewer tokens than beams
    with pytest.raises(ValueError, match="eos"):
        ops.beam_select(so, t, p, x, s, 10, eos=10)
    with pytest.raises(ValueError, match="eos"):
        ops.beam_select(so, t, p, x, s, 10, finished=torch.zeros(2, 3, dtype=torch.bool))
    with pytest.raises(ValueError, match="share"):
        ops.beam_select(s, t, p, x, s, 10)
    with pytest.raises(ValueError, match="share"):
        ops.beam_select(so, t, t, x, s, 10)
    with pytest.raises(ValueError, match="tokens"):
        ops.beam_select(so, t.long(), p, x, s, 10)
    with pytest.raises(TypeError):
        ops.beam_select(so, t, p, x.half(), s, 10)
    with pytest.raises(ValueError, match="beams"):
        ops.beam_select(torch.empty(1, 65), torch.empty(1, 65, dtype=torch.int32), torch.empty(1, 65, dtype=torch.int32), torch.zeros(65, 100),
                        torch.zeros(1, 65), 100)


def test_a_row_that_is_not_finite_is_kept_as_nan_and_seen_by_no_one_else():
    c = ops.KV4Cache.empty(1, 1, 1, 64, 32, "cpu")
    k, v = rnd(1, 6, 1, 32), rnd(1, 6, 1, 32, seed=1)
    v[0, 4, 0, 20] = float("inf")
    ops.kv4_append(c, 0, k, v, i32(0))
    q = rnd(1, 6, 1, 32, seed=2)
    out = torch.empty_like(q)
    ops.attention_kv4(out, q, c, 0, i32(6))
    assert torch.isfinite(out[0, :4]).all() and torch.isnan(out[0, 4:]).all()


def test_keys_and_values_are_two_memories():
    c = _cache()
    with pytest.raises(ValueError, match="same memory"):
        ops.KV4Cache(c.k_codes, c.k_scales, c.k_codes, c.v_scales)
    with pytest.raises(ValueError, match="same memory"):
        ops.KV4Cache(c.k_codes, c.k_scales, c.v_codes, c.k_scales)


def test_a_block_too_small_for_a_scale_is_all_zeros():
    """2^-10 is half the smallest e4m3 number, a tie that goes to zero: values of up to 6 x 2^-10 units leave neither a code nor a sign."""
    c = _cache()
    x = torch.full((2, 1, 2, 64), -6 * 2.0 ** -10 * c.k_unit)
    c.k_codes.fill_(0x55)
    ops.kv4_append(c, 0, x, x, i32(0, 3))
    assert not c.k_codes[0, 0, :, 0].any() and not c.k_scales[0, 0, :, 0].any()
    assert not c.k_codes[0, 1, :, 3].any() and bool((c.k_codes[0, 1, :, 4] == 0x55).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scales_around_every_midpoint(dtype):
    """A block's largest value on the midpoints between scales (exact in both types) and, for fp32, next to them, by the definition in 64 bits."""
    scale = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    top = ((scale[1:] + scale[:-1]) / 2 * 6 * ops.kv4.KV4_UNIT).float()
    top = torch.cat([top, torch.nextafter(top, top * 2), torch.nextafter(top, top * 0)] if dtype == torch.float32 else [top]).to(dtype)
    x = (rnd(top.numel(), 32, seed=11).clamp(-1, 1) * top.view(-1, 1).float()).to(dtype)
    x[:, 5::16] = -top.view(-1, 1)
    x = x.view(1, -1, 1, 32)
    c = ops.KV4Cache.empty(1, 1, 1, 384, 32, "cpu")
    ops.kv4_append(c, 0, x, -x, i32(0))
    ko, vo = torch.empty(x.shape), torch.empty(x.shape)
    ops.kv4_values(ko, vo, c, 0, i32(0))
    assert torch.equal(ko.double(), rounded64(x, ops.kv4.KV4_UNIT)) and torch.equal(vo, -ko)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_outputs_of_the_selection_are_not_among_its_logits(dtype):
    """Each output in the columns that are read, in the last of them, across two rows; columns behind the vocabulary may hold one."""
    B, K, V, row = 2, 3, 40, 64
    n = B * K
    memory = torch.zeros(n * row, dtype=dtype)
    logits = memory.view(n, row)
    bytes_ = memory.view(torch.uint8)
    size = dtype.itemsize

    def place(at, d):                                        # an output that starts at a byte of the logits
        return bytes_[at:at + n * d.itemsize].view(d).view(B, K)

    def call(**out):
        o = {"scores_out": torch.empty(B, K), "tokens": torch.empty(B, K, dtype=torch.int32), "parents": torch.empty(B, K, dtype=torch.int32),
             "finished_out": torch.empty(B, K, dtype=torch.bool), **out}
        ops.beam_select(o.pop("scores_out"), o.pop("tokens"), o.pop("parents"), logits, torch.zeros(B, K), V, **o)
    for name, d in (("scores_out", torch.float32), ("tokens", torch.int32), ("parents", torch.int32), ("finished_out", torch.bool)):
        used = n * d.itemsize
        for at in (0, 4, V * size - 4, 2 * row * size - 4, 3 * row * size - (used - 4) // 4 * 4, ((n - 1) * row + V) * size - 4):
            with pytest.raises(ValueError, match="columns of logits"):
                call(**{name: place(at, d)})
        if used <= (row - V) * size:
            call(**{name: place(V * size, d)})
            call(**{name: place(row * size - used // 4 * 4 - (4 if used % 4 else 0), d)})
    logits = torch.zeros(1, V, dtype=dtype).expand(n, V)     # one row for all
    call()


def test_an_output_of_attention_is_q_itself_or_apart_from_it():
    c = _cache(max_len=64)
    S, n, H, hd = 2, 3, 2, 64
    k = rnd(S, 5, H, hd)
    ops.kv4_append(c, 0, k, k, i32(0, 0))
    lens = i32(5, 5)
    memory = rnd(2 * S * n * 3 * H * hd, seed=2)
    qkv = memory[:S * n * 3 * H * hd].view(S, n, 3, H, hd)
    q = qkv[:, :, 0]
    want = torch.empty(S, n, H, hd)
    ops.attention_kv4(want, q, c, 0, lens)
    size = (S, n, H, hd)
    one = (n * 3 * H * hd, 3 * H * hd, hd, 1)
    for out in (memory.as_strided(size, one, 1),             # shifted by a value, a head, a token; in another order
                memory.as_strided(size, one, hd), memory.as_strided(size, one, 3 * H * hd), memory.as_strided(size, one, n * 3 * H * hd),
                memory.as_strided(size, (n * H * hd, H * hd, hd, 1), 0), memory.as_strided(size, (hd, S * H * hd, S * hd, 1), 64),
                memory.as_strided(size, (3 * H * hd, S * 3 * H * hd, hd, 1), 0)):
        with pytest.raises(ValueError, match="q itself"):
            ops.attention_kv4(out, q, c, 0, lens)
    with pytest.raises(ValueError, match="q itself"):        # rows of q that are one
        x = memory[:S * n * H * hd].view(size)
        ops.attention_kv4(x, x[:, :1].expand(size), c, 0, lens)
    kept = q.clone()
    for out in (qkv[:, :, 1], qkv[:, :, 2]):                 # the places of the keys and values, which are in the cache by now
        ops.attention_kv4(out, q, c, 0, lens)
        assert torch.equal(out, want) and torch.equal(q, kept)
    wide = torch.zeros(S, n, H, 2 * hd)                      # halves of one row, with other strides from token to token
    wide[..., :hd] = kept
    ops.attention_kv4(wide[..., hd:], wide[..., :hd], c, 0, lens)
    assert torch.equal(wide[..., hd:], want)
    row = torch.zeros(S, n, 2 * H * hd)
    row[..., :H * hd] = kept.flatten(-2)
    out = row.as_strided(size, (n * 2 * H * hd, 2 * H * hd, hd, 1), H * hd)
    ops.attention_kv4(out, row[..., :H * hd].view(size), c, 0, lens)
    assert torch.equal(out, want)
    ops.attention_kv4(q, q, c, 0, lens)
    assert torch.equal(q, want)


def test_the_two_read_backs_share_no_memory():
    c = _cache()
    memory, size = torch.zeros(2 * 3 * 2 * 2 * 64), (2, 3, 2, 64)
    pair = memory.view(2, 3, 2, 2, 64)
    k, v = rnd(2, 3, 2, 64), rnd(2, 3, 2, 64, seed=1)
    ops.kv4_append(c, 0, k, v, i32(0, 0))
    ops.kv4_values(pair[:, :, 0], pair[:, :, 1], c, 0, i32(0, 0))            # side by side in one tensor
    assert torch.equal(pair[:, :, 0].double(), rounded64(k, c.k_unit)) and torch.equal(pair[:, :, 1].double(), rounded64(v, c.v_unit))
    flat = memory[:2 * 3 * 2 * 64].view(size)
    for shift in (1, 64, 2 * 64, 3 * 2 * 64):
        for a, b in ((flat, memory[shift:shift + flat.numel()].view(size)), (memory[shift:shift + flat.numel()].view(size), flat),
                     (pair[:, :, 0], memory[shift:shift + flat.numel()].view(size))):
            with pytest.raises(ValueError, match="same memory"):
                ops.kv4_values(a, b, c, 0, i32(0, 0))
    ops.kv4_values(flat[:, :0], flat[:, :0], c, 0, i32(0, 0))                # nothing to write is no error


def test_the_four_tensors_of_a_cache_share_no_memory():
    L, S, H, T, half = 2, 3, 2, 64, 32
    nc, ns = L * S * H * T * half, L * S * H * T * half // 8
    memory = torch.zeros(8 * nc, dtype=torch.uint8)
    codes = lambda at: memory[at:at + nc].view(L, S, H, T, half)  # noqa: E731
    scales = lambda at: memory[at:at + ns].view(L, S, H, T, half // 8)  # noqa: E731
    ops.KV4Cache(codes(0), scales(2 * nc), codes(nc), scales(2 * nc + ns))               # one behind the other
    for at in ((0, 4 * nc, 16, 5 * nc), (nc, 4 * nc, 16, 5 * nc), (0, 4 * nc, nc - 16, 5 * nc), (0, nc - 16, 2 * nc, 5 * nc), (0, 4 * nc, 2 * nc, nc - 16),
               (0, 4 * nc, 2 * nc, 3 * nc - 16), (ns - 16, 0, 2 * nc, 5 * nc), (0, 4 * nc, 2 * nc, 4 * nc + ns - 16), (0, 2 * nc + 64, 2 * nc, 5 * nc)):
        with pytest.raises(ValueError, match="share memory"):
            ops.KV4Cache(codes(at[0]), scales(at[1]), codes(at[2]), scales(at[3]))
    # keys and values of each layer, and of each slot, side by side in one tensor: no byte in common
    x, y = torch.zeros(L, 2, S, H, T, half, dtype=torch.uint8), torch.zeros(L, S, 2, H, T, half // 8, dtype=torch.uint8)
    c = ops.KV4Cache(x[:, 0], y[:, :, 0], x[:, 1], y[:, :, 1])
    k, v = rnd(S, 5, H, 2 * half), rnd(S, 5, H, 2 * half, seed=1)
    ops.kv4_append(c, 1, k, v, i32(0, 3, 60))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.kv4_values(ko, vo, c, 1, i32(0, 3, 60))
    assert torch.equal(ko[:2].double(), rounded64(k, c.k_unit)[:2]) and torch.equal(vo[:2].double(), rounded64(v, c.v_unit)[:2])
    with pytest.raises(ValueError, match="share memory"):
        ops.KV4Cache(x[:, 0], y[:, :, 0], x[:, 0, :].as_strided((L, S, H, T, half), x[:, 0].stride(), 64), y[:, :, 1])
    with pytest.raises(ValueError, match="share memory"):
        ops.KV4Cache(x[:, 0], y[:, :, 0], x[:, 1], y.as_strided(y[:, :, 0].shape, y[:, :, 0].stride(), 16))


def test_tables_of_a_reorder_share_no_memory():
    c = _cache(slots=6, max_len=128)
    memory = torch.zeros(40, dtype=torch.int32)
    at = lambda i, *shape: memory[i:i + math.prod(shape)].view(shape)  # noqa: E731
    ops.kv4_reorder(c, at(6, 6, 2), at(0, 6), at(18, 2, 3))                  # side by side
    ops.kv4_reorder(c, at(12, 6, 2), at(24, 6), at(6, 2, 3))
    for pages, lens, parents in ((0, 11, 20), (5, 0, 20), (0, 20, 11), (9, 20, 4), (20, 0, 5), (20, 5, 0), (20, 0, 0)):
        with pytest.raises(ValueError, match="share memory"):
            ops.kv4_reorder(c, at(pages, 6, 2), at(lens, 6), at(parents, 2, 3))


def test_memory_in_common_is_decided_exactly():
    """Against sets of addresses: nested strides in any order, shifted copies of one layout and two layouts, types of other sizes; on the host
    whatever the default device is."""
    import random
    r, memory, seen = random.Random(0), torch.zeros(4000, dtype=torch.uint8), set()

    def layout():
        shape = [r.randint(1, 4) for _ in range(r.randint(1, 4))]
        strides, span = [0] * len(shape), 1
        for i in r.sample(range(len(shape)), len(shape)):
            strides[i] = span + r.choice([0, 0, 1, 4])
            span += strides[i] * (shape[i] - 1)
        return shape, strides, span

    def addresses(t):
        at = [t.data_ptr()]
        for n, s in zip(t.shape, t.stride()):
            at = [a + i * s * t.element_size() for a in at for i in range(n)]
        return {a + b for a in at for b in range(t.element_size())}
    with torch.device("meta"):
        for _ in range(4000):
            one, d1 = layout(), r.choice([torch.uint8, torch.bfloat16, torch.float32])
            two, d2 = (one, d1) if r.random() < 0.5 else (layout(), r.choice([torch.uint8, torch.bfloat16]))
            if max(one[2] * d1.itemsize, two[2] * d2.itemsize) > 1500:
                continue
            first = r.randint(0, 300)
            a = memory.view(d1).as_strided(*one[:2], first)
            b = memory.view(d2).as_strided(*two[:2], max(0, first * d1.itemsize // d2.itemsize + r.randint(-60, 60)))
            want = bool(addresses(a) & addresses(b))
            seen.add((one is two, want))
            assert ops.kv4._meet(a, b) == want, (a.shape, a.stride(), b.shape, b.stride(), b.data_ptr() - a.data_ptr())
    assert len(seen) == 4
