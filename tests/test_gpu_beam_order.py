"""
nn_ops.beam_select at the ends of the logits' range: infinities, masks of the type's lowest value, against the definition
in 64 bits (the difference from the row's largest logit is formed before anything else, so nothing is lost beside a
logit of 1e38).

Scores: the total is formed in 64 bits from sums of up to 2^15 terms, off by less than 1e-11 of its size or of 1; rounded
to f32 it is off by 2^-24 of its size more.
"""
import math

import pytest
import torch

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda:0"
INF = float("inf")


def randn(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def definition(logits, scores, K):
    """the K best of score + log_softmax(logits): ties of hypotheses to the lowest, of one hypothesis' continuations
    to the larger logit, then to the lower token"""
    n, b = scores.shape
    x = torch.nan_to_num(logits.double().view(n, b, -1), nan=-INF, neginf=-INF, posinf=torch.finfo(torch.float32).max)
    out = []
    for i in range(n):
        found = []
        for j in range(b):
            row = x[i, j]
            top = row.max()
            if top == -INF or not scores[i, j] > -INF:
                found += [(INF, j, INF, t) for t in range(K)]
                continue
            d = row - top
            log = math.log(math.fsum(torch.exp(d).tolist()))  # (the same for equal rows)
            total = scores[i, j].double() + (d - log)
            found += [(-t, j, -r, at) for at, (t, r) in enumerate(zip(total.tolist(), row.tolist()))]
        out.append(sorted(found)[:K])
    best = torch.tensor([[-f[0] for f in o] for o in out], dtype=torch.float64)
    return best, *(torch.tensor([[f[at] for f in o] for o in out]) for at in (1, 3))


def check(logits, scores, K):
    from aps_amd import nn_ops
    got = [t.cpu() for t in nn_ops.beam_select(logits.to(DEV), scores.to(DEV), 1, beam=K)]
    best, parent, token = definition(logits.cpu(), scores, K)
    assert torch.equal(got[1], parent), (got[1], parent)
    assert torch.equal(got[2], token), (got[2], token)
    assert torch.equal(got[3], token == 1)
    bound = 2**-24 * best.abs() + 1e-11 * best.abs().clamp_min(1.0)
    assert ((got[0].double() == best) | ((got[0].double() - best).abs() <= bound)).all(), (got[0], best)


SCORES = torch.tensor([[-1.0, -1.5, -2.0], [-3.0, -0.5, -0.75]])


@gpu
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("v", [70, 3001, 20000])
@pytest.mark.parametrize("largest", [INF, None])
def test_infinite_and_largest_logits_win_their_row(kind, v, largest):
    dtype = TYPES[kind]
    value = torch.finfo(dtype).max if largest is None else largest
    for row, at in ((0, [v - 1]), (2, [7]), (3, [v // 2, 9]), (5, [0, 1, v - 2])):
        x = randn(6, v, dtype=dtype, seed=v)
        x[row, at] = value
        check(x, SCORES, 5)
        x[row, 3] = -INF
        x[row, 4] = float("nan")
        check(x, SCORES, 5)


@gpu
@pytest.mark.parametrize("kind,low", [("f32", None), ("f32", -1e30), ("f32", -1e15), ("f32", -1e9), ("bf16", None), ("bf16", -1e30),
                                      ("f16", None)])
@pytest.mark.parametrize("v", [70, 4233, 20000])
def test_masks_of_large_finite_values(kind, low, v):
    """whole rows, the first part, the last part and all but one token at the mask's value: no other hypothesis
    changes, and a row that is masked throughout spreads over its vocabulary"""
    dtype = TYPES[kind]
    low = torch.finfo(dtype).min if low is None else low
    for cut in (slice(0, v), slice(0, v - v // 8), slice(v // 8, v), slice(1, v), slice(0, v - 1)):
        x = randn(6, v, dtype=dtype, seed=v + 1)
        x[1, cut] = low
        x[3, cut] = low
        check(x, SCORES, 6)
        x[4:] = low
        check(x, SCORES, 6)


@gpu
def test_rows_of_one_large_value():
    """every logit the same: each continuation has 1 / V, whatever the value"""
    for value in (1e38, -1e38, 3e15, -7e20, torch.finfo(torch.float32).max, torch.finfo(torch.float32).min):
        for v in (33, 9000):
            check(torch.full((6, v), value), SCORES, 7)


@gpu
@pytest.mark.parametrize("kind,v", [("f32", 501), ("f32", 4233), ("bf16", 10007), ("f16", 333), ("f32", 20011)])
def test_equal_hypotheses_tie_to_the_first(kind, v):
    """hypotheses with the same logits and the same score: every token of the first comes ahead of the second's,
    whatever address their rows begin at"""
    n, b = 12, 5
    x = randn(n, 1, v, dtype=TYPES[kind], seed=v, std=2.0).expand(n, b, v).reshape(n * b, v)
    scores = -randn(n, 1, seed=3).abs().expand(n, b).contiguous()
    for K in (b, 2 * b + 1):
        check(x, scores, K)
    wide = torch.zeros(n * b, v + 5, dtype=TYPES[kind], device=DEV)
    for first in (0, 1, 3):
        wide[:, first:first + v] = x.to(DEV)
        check(wide[:, first:first + v], scores, b)


@gpu
def test_logits_too_near_for_their_totals():
    """totals of one hypothesis that 64 bits round to the same number are taken by logit: a vocabulary of tiny logits, and
    one whose largest is the largest f32, which hides all differences of the others"""
    for v in (90, 5000):
        x = randn(4, v, seed=v) * 1e-25
        check(x, torch.zeros(4, 1), 11)
        check(x, torch.zeros(2, 2), 11)
        x = randn(4, v, seed=v)
        x[:, v // 3] = torch.finfo(torch.float32).max
        check(x, torch.zeros(4, 1), 9)
        x[:, 5] = INF
        check(x, torch.zeros(4, 1), 9)
    # more equal totals than the candidate list holds
    x = randn(24, 60, seed=9) * 1e-25
    check(x, torch.zeros(1, 24), 50)
