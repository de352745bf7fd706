"""Generation over the 4-bit cache on the GPU."""
import io

import pytest
import torch

from llm_mojo_b200 import ops
from llm_mojo_b200.config import GPT2Config
from llm_mojo_b200.models import GPT2, CachedDecoder, beam_search
from llm_mojo_b200.ops import _lib
from test_generate import CFG, logits64, make, search64

pytestmark = pytest.mark.gpu
WIDE = GPT2Config(max_seq_len=512, vocab_size=5000, num_layer=3, num_heads=4, channels=256, padded_vocab_size=5056)


def near(a, b, tol, what=""):
    a, b = a.double().cpu(), b.double().cpu()
    assert torch.isfinite(a).all(), what
    assert ((a - b).norm() / b.norm()).item() <= tol, (what, ((a - b).norm() / b.norm()).item())


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("precision", ["bf16", "tf32", "fp32"])
def test_prefill_and_steps(precision, graph, monkeypatch):
    """Against float64 passes on the same weights.

    The 4-bit rounding makes much of little: an error of eps moves a value across a midpoint, by a step of about a third of its size, with
    probability 3 eps, an rms error of sqrt(eps / 3): 4 % for the 2^-8 of bf16, 1.3 % for the 2^-11 of TF32, in the first layer, and the next
    starts from that.  The bound is what the two roundings can differ by at all: each is off by some 10 % rms, |Q(v + d) - Q(v)| by at most
    twice that and d, of the keys, the values and what attention makes of them; 25 % of the logits with the rest of the layers unchanged.
    fp32 products: eps 2^-22 in 10^5 values a layer, 0.1 values expected to move; without one 2^-24 for sums of up to 1024 terms in three layers,
    with one a third of one of 256 elements of a token among 300."""
    if precision == "fp32":
        monkeypatch.setenv("LLMM_NO_TF32", "1")
    m = make("cuda", precision, WIDE, 2.0)
    g = torch.Generator().manual_seed(0)
    texts = [torch.randint(0, 5000, (n,), generator=g).tolist() for n in (300, 1, 129)]
    dec = CachedDecoder(m, 3, graph=graph)
    got = dec.prefill(texts)
    tol = 2e-3 if precision == "fp32" else 0.25
    for b in range(3):
        near(got[b], logits64(m, texts[b])[-1], tol, b)
    extra = torch.randint(0, 5000, (5, 3), generator=g, dtype=torch.int32)
    for i in range(5):
        got = dec.step(extra[i].cuda())
    for b in range(3):
        near(got[b], logits64(m, texts[b] + extra[:, b].tolist())[-1], tol, b)
    assert dec.lens.tolist() == [305, 6, 134] and _lib.read_status() == 0


def test_steps_of_a_graph_are_those_of_launches_to_the_bit():
    m = make("cuda", "bf16", WIDE, 2.0)
    outs = []
    for graph in (False, True):
        dec = CachedDecoder(m, 2, beams=3, graph=graph)
        dec.prefill([[1, 2, 3] * 40, [4]])
        seen = []
        for i in range(70):                                       # across the end of a page
            seen.append(dec.step(torch.full((6,), 10 + i, dtype=torch.int32, device="cuda")).clone())
            dec.reorder(torch.tensor([[0, 0, 2], [(i + 1) % 3, 1, 0]], dtype=torch.int32, device="cuda"))
        outs.append(torch.stack(seen))
    assert torch.equal(*outs)


def test_beam_search_in_fp32_is_the_search_by_whole_passes(monkeypatch):
    monkeypatch.setenv("LLMM_NO_TF32", "1")                       # library products in fp32: the selections have to be the same
    m = make("cuda", "fp32", CFG)
    m.p["wte"][7] *= 3.0
    prompts = [[5, 6, 7, 8], [100], list(range(60, 124))]
    for eos in (-1, 7):
        got = beam_search(m, prompts, 4, 9, eos=eos)
        for row, prompt in zip(got, prompts):
            want = search64(m, prompt, 4, 9, eos)
            assert [t for t, _ in row] == [t for t, _ in want]
            assert all(abs(a - b) < 1e-3 for (_, a), (_, b) in zip(row, want))


def test_scores_of_a_beam_search_are_those_of_its_texts(monkeypatch):
    monkeypatch.setenv("LLMM_NO_TF32", "1")
    m = make("cuda", "fp32", WIDE, 2.0)
    prompt = list(range(100, 230))
    best = beam_search(m, [prompt, [9]], 5, 20)[0]
    assert [v for _, v in best] == sorted((v for _, v in best), reverse=True) and len({tuple(t) for t, _ in best}) == 5
    # read again one by one: the same keys and values in another cut; an error of 2e-3 of logits of size 1 in each of twenty log probabilities
    text, score = best[0]
    dec = CachedDecoder(m, 1)
    logits, total = dec.prefill([prompt]), 0.0
    for t in text:
        total += float(torch.log_softmax(logits[0, :5000].double(), -1)[t])
        logits = dec.step(torch.tensor([t], dtype=torch.int32, device="cuda"))
    assert abs(total - score) < 20 * 2e-3


def test_infer_writes_tokens(tmp_path):
    import infer_gpt2
    m = GPT2("d6", "bf16", "cuda")

    class Tok:
        has_initialized, eot_token = False, 50256
    a, b = io.StringIO(), io.StringIO()
    ids = infer_gpt2.run_infer_cached(m, Tok(), [50256, 11, 12], 12, seed=3, out=a)
    again = infer_gpt2.run_infer_cached(m, Tok(), [50256, 11, 12], 12, seed=3, out=b)
    assert len(ids) == 12 and ids == again and all(0 <= t < 50257 for t in ids)
    best = infer_gpt2.run_beams(m, Tok(), [50256], 6, 3, out=a)
    assert len(best) == 3 and all(len(t) == 6 for t, _ in best)


def test_a_wait_that_ran_out_is_an_error():
    """The word that kernels set where a bounded wait ends without its event is set from the host here."""
    import infer_gpt2
    m = make("cuda", "bf16", WIDE, 2.0)
    word = _lib.status_word(torch.device("cuda", torch.cuda.current_device()))

    class Tok:
        has_initialized, eot_token = False, 0
    dec, out = CachedDecoder(m, 1), io.StringIO()
    dec.prefill([[1, 2, 3]])
    for call in (dec.check, lambda: beam_search(m, [[1, 2, 3], [4]], 3, 5), lambda: beam_search(m, [[1]], 2, 20, eos=7),
                 lambda: infer_gpt2.run_infer_cached(m, Tok(), [1, 2, 3], 4, seed=3, out=out)):
        word.fill_(1)
        with pytest.raises(_lib.KernelError, match="wait ran out"):
            call()
        assert _lib.read_status() == 0                            # said once
        assert out.getvalue() == ""                               # no token of it was written
        call()
