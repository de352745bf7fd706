"""The beam selection on the GPU against its 64-bit statement."""
import math

import pytest
import torch

from kv4_oracle import select64
from llm_mojo_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float32


def run(logits, scores, V, finished=None, eos=-1, exact_order=True):
    B, K = scores.shape
    so = torch.empty(B, K, device=DEV)
    t, p = (torch.empty(B, K, dtype=torch.int32, device=DEV) for _ in range(2))
    f = torch.empty(B, K, dtype=torch.bool, device=DEV)
    ops.beam_select(so, t, p, logits, scores, V, finished_out=f, finished=finished, eos=eos)
    w = select64(logits, scores, V, finished, eos)
    assert torch.equal(t.long(), w[1]) and torch.equal(p.long(), w[2]) and torch.equal(f, w[3])
    # one rounding to fp32, and a log-sum-exp whose exponentials and partial sums are fp32: 2^-22 of it covers 4096 terms a chunk
    fin = torch.isfinite(w[0])
    assert torch.equal(so[~fin].double(), w[0][~fin])
    assert ((so.double() - w[0])[fin].abs() <= 2.0 ** -23 * w[0][fin].abs() + 2.0 ** -12 * 2.0 ** -8).all()
    return so, t, p, f


def rnd(*shape, dtype=FP, scale=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 13 * sum(shape))
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


@pytest.mark.parametrize("B,K,V,pad", [(1, 1, 1, 0), (1, 4, 50257, 47), (5, 3, 255, 1), (2, 8, 4096, 0), (3, 5, 4097, 7), (7, 16, 9001, 3), (2, 64, 5000, 0), (1, 64, 64, 0)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_selection(B, K, V, pad, dtype):
    logits = rnd(B * K, V + pad, dtype=dtype, scale=2.5)
    logits[:, V:] = 1e4                                      # columns behind the vocabulary are not read
    scores = -rnd(B, K, seed=1).abs() * 5
    run(logits, scores, V)
    finished = torch.rand(B, K, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV) < 0.4
    run(logits, scores, V, finished, V - 1)
    run(logits, scores, V, torch.ones_like(finished), V // 2)
    run(logits, scores, V, eos=0)


def test_first_step_and_dead_beams():
    B, K, V = 3, 4, 6000
    logits = rnd(B * K, V, dtype=BF, scale=2.5)
    scores = torch.full((B, K), -math.inf, device=DEV)
    scores[:, 0] = 0.0                                       # the first step: one beam of each item is alive
    _, _, p, _ = run(logits, scores, V)
    assert (p == 0).all()
    run(logits, torch.full((B, K), -math.inf, device=DEV), V)          # none is: the lowest places
    scores = -rnd(B, K, seed=1).abs()
    scores[0, 1], scores[1, 2] = math.nan, math.inf
    run(logits, scores, V)
    fin = torch.zeros(B, K, dtype=torch.bool, device=DEV)
    fin[0, 1] = fin[2, 0] = True
    scores[2, 0] = -math.inf
    run(logits, scores, V, fin, 5)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_logits_that_are_not_finite(dtype):
    B, K, V = 2, 4, 5000
    logits = rnd(B * K, V, dtype=dtype, scale=2.5)
    scores = -rnd(B, K, seed=1).abs()
    logits[1, 4097] = math.nan                               # a beam without a log-sum-exp offers nothing
    logits[2, 17] = math.inf
    logits[4] = -math.inf
    logits[5, 100:] = -math.inf                              # tokens that are ruled out
    logits[6, 3:] = -math.inf                                # fewer than K are left
    run(logits, scores, V)
    logits[:] = -math.inf
    logits[:, 4500] = 1.0                                    # one token each, in the second chunk: the others tie at -inf
    run(logits, scores, V)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_ties_go_to_the_lowest_beam_and_token(dtype):
    B, K, V = 2, 8, 9000
    run(torch.zeros(B * K, V, dtype=dtype, device=DEV), torch.zeros(B, K, device=DEV), V)
    logits = torch.zeros(B * K, V, dtype=dtype, device=DEV)
    logits[:, 1::2] = -0.0                                   # the two zeros are one number
    run(logits, torch.zeros(B, K, device=DEV), V)
    base = rnd(1, V, dtype=dtype, scale=2.0)
    base[0, 8000] = base[0, 30] = base[0, 4095] = base[0, 4096] = 9.0
    # the same beam K times, in rows of odd length whose addresses differ
    logits = torch.zeros(B * K, V + 1, dtype=dtype, device=DEV)
    logits[:, :V] = base
    run(logits, torch.full((B, K), -1.25, device=DEV), V)


def test_large_values_and_the_call_in_a_graph():
    B, K, V = 4, 4, 50257
    logits = rnd(B * K, V, dtype=FP, scale=50.0) + 3e4       # a log-sum-exp that needs its maximum
    scores = -rnd(B, K, seed=1).abs() * 100
    so, t, p, f = run(logits, scores, V, eos=1)
    side = torch.cuda.Stream()
    keep = [x.clone() for x in (so, t, p, f)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.beam_select(so, t, p, logits, scores, V, finished_out=f, eos=1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(keep, (so, t, p, f)))
    graphs = []
    for _ in range(2):                                       # two graphs, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.beam_select(so, t, p, logits, scores, V, finished_out=f, eos=1)
        graphs.append(g)
    for i, g in enumerate(graphs * 2):
        logits.copy_(rnd(B * K, V, scale=3.0, seed=i))
        g.replay()
        w = select64(logits, scores, V, None, 1)
        assert torch.equal(t.long(), w[1]) and torch.equal(p.long(), w[2])


@pytest.mark.parametrize("B,K,V", [(3, 33, 8193), (2, 32, 40000), (9, 16, 20000), (1, 9, 130), (1, 64, 46 * 8192)])
def test_many_beams_and_the_largest_merge(B, K, V):
    """More lists than the merge stages, more beams than a warp has lanes, chunks whose last warps have no columns."""
    logits = rnd(B * K, V, scale=2.5)
    run(logits, -rnd(B, K, seed=1).abs() * 5, V)


def test_the_same_logits_in_every_column():
    """Every candidate of a beam ties: columns in order, however many chunks and candidates there are."""
    B, K, V = 2, 12, 9000
    logits = torch.full((B * K, V), 1.5, dtype=BF, device=DEV)
    scores = -torch.arange(1, K + 1, device=DEV, dtype=FP).repeat(B, 1) * 0.25
    so, t, p, _ = run(logits, scores, V)
    assert torch.equal(t, torch.arange(K, device=DEV, dtype=torch.int32).repeat(B, 1)) and not p.any()


def test_more_lists_than_the_merge_holds_are_refused():
    K, V = 64, 46 * 8192 + 1
    so, t, p = torch.empty(1, K, device=DEV), torch.empty(1, K, dtype=torch.int32, device=DEV), torch.empty(1, K, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="too many"):
        ops.beam_select(so, t, p, torch.zeros(K, V, dtype=BF, device=DEV), torch.zeros(1, K, device=DEV), V)


# ------------------------------------------------------------------ where chunks of 8192 columns meet
LONG = 17000                                                 # two whole chunks and a short one


@pytest.mark.parametrize("dtype", [BF, FP])
def test_logits_that_are_not_finite_in_any_chunk(dtype):
    B, K = 2, 6
    logits = rnd(B * K, LONG + 1, dtype=dtype, scale=2.5)
    scores = -rnd(B, K, seed=1).abs()
    logits[0, 8192], logits[1, 16383], logits[2, 16999] = math.nan, math.inf, math.nan      # beams that offer nothing
    logits[3, :8192] = -math.inf                             # a whole chunk ruled out: the first,
    logits[4, 8192:16384] = -math.inf                        # the middle one,
    logits[5, 16384:] = -math.inf                            # the last
    logits[6, :16384] = -math.inf                            # all but the last
    logits[7] = -math.inf
    logits[8, 1:] = -math.inf                                # one token each, in the first, the second and the third chunk
    logits[9], logits[9, 8192] = -math.inf, 1.0
    logits[10], logits[10, 16999] = -math.inf, 1.0
    run(logits, scores, LONG)
    run(logits[6:].contiguous(), scores[:1], LONG, eos=9)
    for at in (8191, 8192, 16384):                           # nothing but these: the others tie at -inf
        x = torch.full((B * K, LONG), -math.inf, dtype=dtype, device=DEV)
        x[:, at] = 1.0
        run(x, scores, LONG)


def test_dead_and_finished_beams_of_many_chunks():
    B, K = 3, 4
    logits = rnd(B * K, LONG, dtype=BF, scale=2.5)
    scores = torch.full((B, K), -math.inf, device=DEV)
    run(logits, scores, LONG)                                # none is alive: the lowest places
    scores[:, 2] = 0.0                                       # one is
    _, _, p, _ = run(logits, scores, LONG)
    assert (p == 2).all()
    scores = -rnd(B, K, seed=1).abs()
    scores[0, 1], scores[1, 2] = math.nan, math.inf
    run(logits, scores, LONG)
    fin = torch.zeros(B, K, dtype=torch.bool, device=DEV)
    fin[0, 1] = fin[1, 0] = fin[2, 0] = fin[2, 3] = True
    scores[2, 0] = -math.inf
    for eos in (0, 8191, 8192, 16999):
        run(logits, scores, LONG, fin, eos)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_ties_across_chunks(dtype):
    B, K = 2, 8
    logits = rnd(B * K, LONG, dtype=dtype, scale=2.0)
    logits[:] = logits[0]
    logits[:, [8191, 8192, 16383, 16384, 16999, 30]] = 12.0  # of each beam, and between the beams
    _, t, p, _ = run(logits, torch.full((B, K), -1.25, device=DEV), LONG)
    assert t[0].tolist() == [30, 8191, 8192, 16383, 16384, 16999, 30, 8191] and p[0].tolist() == [0] * 6 + [1] * 2
    run(torch.zeros(B * K, LONG, dtype=dtype, device=DEV), torch.zeros(B, K, device=DEV), LONG)
