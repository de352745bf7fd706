"""Generation over the 4-bit cache on CPU tensors: the decoder and the beam search against a whole forward pass whose keys and values are rounded."""
import io
import math
import os
import subprocess
import sys

import pytest
import torch
import torch.nn.functional as F

from kv4_oracle import rounded64, select64
from llm_mojo_b200.config import GPT2Config
from llm_mojo_b200.models import GPT2, CachedDecoder, beam_search

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CFG = GPT2Config(max_seq_len=96, vocab_size=210, num_layer=3, num_heads=2, channels=64, padded_vocab_size=256)


def make(device="cpu", precision="fp32", cfg=CFG, sharp=4.0):
    m = GPT2(cfg, precision, device)
    for n in ("qkvw", "fcw", "attprojw", "fcprojw", "wpe"):       # larger than the initialisation: attention that is not flat
        m.p[n].mul_(sharp)
    return m


def logits64(m, tokens):
    """Logits [n, Vp] behind every token of one text, in float64, with the keys and values rounded as the cache rounds them."""
    p = {k: v.detach().cpu().double() for k, v in m.p.items()}
    C, NH = m.config.channels, m.config.num_heads
    n, hd = len(tokens), C // NH
    x = p["wte"][torch.tensor(tokens)] + p["wpe"][:n]
    for l in range(m.config.num_layer):
        h = F.layer_norm(x, (C,), p["ln1w"][l], p["ln1b"][l], 1e-5)
        q, k, v = (t.view(n, NH, hd) for t in (h @ p["qkvw"][l].t() + p["qkvb"][l]).split(C, dim=1))
        k, v = rounded64(k.float(), 2.0 ** -4), rounded64(v.float(), 2.0 ** -4)
        s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), float("-inf"))
        x = x + torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(n, C) @ p["attprojw"][l].t() + p["attprojb"][l]
        h = F.layer_norm(x, (C,), p["ln2w"][l], p["ln2b"][l], 1e-5)
        x = x + F.gelu(h @ p["fcw"][l].t() + p["fcb"][l], approximate="tanh") @ p["fcprojw"][l].t() + p["fcprojb"][l]
    return F.layer_norm(x, (C,), p["lnfw"], p["lnfb"], 1e-5) @ p["wte"].t()


def search64(m, prompt, K, new, eos):
    """Beam search by whole forward passes."""
    beams = [(list(prompt), 0.0 if i == 0 else float("-inf"), False) for i in range(K)]
    V = m.config.vocab_size
    for _ in range(new):
        logits = torch.stack([logits64(m, b[0])[-1] for b in beams])
        fin = torch.tensor([[b[2] for b in beams]])
        best, tok, par, nf = select64(logits, torch.tensor([[b[1] for b in beams]], dtype=torch.float64), V, fin if eos >= 0 else None, eos)
        beams = [(beams[p][0] + ([] if beams[p][2] else [t]), s, f) for p, t, s, f in zip(par[0].tolist(), tok[0].tolist(), best[0].tolist(), nf[0].tolist())]
    return [(b[0][len(prompt):], b[1]) for b in beams]


def close(a, b, what=""):
    # fp32 against float64: sums of up to 256 terms in three layers, 2^-24 each; a rounding of a key that goes the other way would show as 1e-2
    assert (a.double() - b).abs().max().item() <= 2e-4 * b.abs().max().item(), what


def test_prefill_and_steps_are_a_whole_forward_pass():
    m = make()
    g = torch.Generator().manual_seed(0)
    texts = [torch.randint(0, 210, (n,), generator=g).tolist() for n in (70, 1, 33)]
    dec = CachedDecoder(m, 3)
    heads = [t[:max(1, len(t) - 6)] for t in texts]
    got = dec.prefill(heads)
    for b in range(3):
        close(got[b], logits64(m, heads[b])[-1], b)
    extra = torch.randint(0, 210, (6, 3), generator=g, dtype=torch.int32)
    for i in range(6):
        got = dec.step(extra[i])
        for b in range(3):
            close(got[b], logits64(m, heads[b] + extra[:i + 1, b].tolist())[-1], (i, b))
    assert dec.lens.tolist() == [len(h) + 6 for h in heads]


@pytest.mark.parametrize("eos", [-1, 7])
def test_beam_search_is_the_search_by_whole_passes(eos):
    m = make()
    prompts = [[5, 6, 7, 8], [100], list(range(60, 124))]
    if eos >= 0:
        m.p["wte"][eos] *= 3.0                                    # a token that comes up
    got = beam_search(m, prompts, 4, 9, eos=eos)
    for row, prompt in zip(got, prompts):
        want = search64(m, prompt, 4, 9, eos)
        assert [t for t, _ in row] == [t for t, _ in want]
        assert all(abs(a - b) < 1e-3 for (_, a), (_, b) in zip(row, want))
        if eos >= 0:
            assert all(eos not in t[:-1] for t, _ in row)
    if eos >= 0:
        assert any(t[-1] == eos for row in got for t, _ in row)
        ranked = beam_search(m, prompts, 4, 9, eos=eos, length_penalty=1.0)
        for row, ref in zip(ranked, got):
            assert sorted(map(str, row)) == sorted(map(str, ref))
            assert [v / len(t) for t, v in row] == sorted((v / len(t) for t, v in row), reverse=True)


def test_one_beam_is_greedy():
    m = make()
    toks = [3, 1, 4]
    for _ in range(5):
        toks.append(int(logits64(m, toks)[-1, :210].argmax()))
    assert beam_search(m, [[3, 1, 4]], 1, 5)[0][0][0] == toks[3:]


def test_refusals():
    m = make()
    with pytest.raises(ValueError, match="head size"):
        CachedDecoder(make(cfg=GPT2Config(96, 210, 1, 4, 64, 256)), 1)
    with pytest.raises(ValueError, match="positions"):
        CachedDecoder(m, 1, 97)
    with pytest.raises(ValueError, match="at least one"):
        CachedDecoder(m, 0)
    dec = CachedDecoder(m, 2, 10)
    with pytest.raises(ValueError, match="prompts"):
        dec.prefill([[1]])
    with pytest.raises(ValueError, match="prompts"):
        dec.prefill([[1], []])
    with pytest.raises(ValueError, match="none of the"):
        dec.prefill([[1], [210]])
    with pytest.raises(ValueError, match="places"):
        dec.prefill([[1], [1] * 11])
    dec.prefill([[1], [1] * 9])
    with pytest.raises(ValueError, match="begun"):
        dec.prefill([[1], [1]])
    with pytest.raises(ValueError, match="one token"):
        dec.step(torch.zeros(3, dtype=torch.int32))
    dec.step(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="places"):
        dec.step(torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="order"):
        dec.reorder(torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="new token"):
        beam_search(m, [[1]], 2, 0)
    with pytest.raises(ValueError, match="places"):
        beam_search(m, [[1] * 90], 2, 8)


def test_a_token_from_outside_counts_as_the_nearest():
    m = make()
    a, b = CachedDecoder(m, 2), CachedDecoder(m, 2)
    a.prefill([[1, 2], [3]]), b.prefill([[1, 2], [3]])
    assert torch.equal(a.step(torch.tensor([-5, 10 ** 6], dtype=torch.int32)), b.step(torch.tensor([0, 209], dtype=torch.int32)))


def test_command_line(tmp_path):
    from llm_mojo_b200.utils import checkpointing as ckpt
    m = make()
    ck = str(tmp_path / "tiny.bin")
    ckpt.write_model_checkpoint(ck, m.config, m.full_params(), m.precision.checkpoint_version)

    def run(*more):
        r = subprocess.run([sys.executable, os.path.join(ROOT, "infer_gpt2.py"), ck, "--tokens", "8", "--device", "cpu", "--seed", "7",
                            "--prompt-tokens", "5,6,7", *more], capture_output=True, text=True, timeout=300, cwd=str(tmp_path))
        assert r.returncode == 0, r.stderr
        return r.stdout

    ids = run("--kv-cache", "4bit").split("---")[-2].split()
    assert len(ids) == 8 and all(0 <= int(t) < 210 for t in ids)
    want = beam_search(m, [[5, 6, 7]], 3, 8)[0]
    rows = [line.split() for line in run("--beams", "3").strip().splitlines()[-3:]]
    assert [[int(t) for t in r[1:]] for r in rows] == [t for t, _ in want]


def test_generation_asks_whether_what_it_answers_is_valid(monkeypatch):
    """Before anything is answered, and in a long search on the way."""
    import infer_gpt2
    from llm_mojo_b200.ops._lib import KernelError
    m, asked = make(), []

    class Tok:
        has_initialized, eot_token = False, 0
    monkeypatch.setattr(CachedDecoder, "check", lambda self: asked.append(self.longest))
    beam_search(m, [[1, 2]], 2, 20, eos=7)
    assert asked[:2] == [2 + 7, 2 + 15] and len(asked) == 3
    asked.clear()
    infer_gpt2.run_infer_cached(m, Tok(), [1, 2], 3, seed=1, out=io.StringIO())
    assert asked == [2, 3, 4]

    def expired(self):
        raise KernelError("a bounded device wait ran out")
    monkeypatch.setattr(CachedDecoder, "check", expired)
    out = io.StringIO()
    with pytest.raises(KernelError):
        beam_search(m, [[1, 2]], 2, 3)
    with pytest.raises(KernelError):
        infer_gpt2.run_infer_cached(m, Tok(), [1, 2], 3, seed=1, out=out)
    assert out.getvalue() == ""


def test_every_launch_is_made_with_the_models_device_current(monkeypatch):
    """The operators without a cache among their arguments launch to the current device's stream."""
    import contextlib

    import infer_gpt2
    from llm_mojo_b200 import ops
    from llm_mojo_b200.models import generate
    m, inside, launched = make(), [], []

    @contextlib.contextmanager
    def on_device(device):
        inside.append(device)
        yield
        inside.pop()

    def watched(fn):
        def call(*a, **kw):
            assert inside == [m.params.device], fn.__name__
            launched.append(fn.__name__)
            return fn(*a, **kw)
        return call

    class Tok:
        has_initialized, eot_token = False, 0
    for module in (generate, infer_gpt2):
        monkeypatch.setattr(module, "on_device", on_device)
    for name in ("layernorm_fwd", "matmul_fwd", "softmax_rows"):
        monkeypatch.setattr(ops, name, watched(getattr(ops, name)))
    dec = CachedDecoder(m, 2, beams=2)
    dec.prefill([[1, 2], [3]])
    dec.step(torch.zeros(4, dtype=torch.int32))
    beam_search(m, [[1, 2]], 2, 3)
    infer_gpt2.run_infer_cached(m, Tok(), [1, 2], 3, seed=1, out=io.StringIO())
    assert set(launched) == {"layernorm_fwd", "matmul_fwd", "softmax_rows"} and not inside
