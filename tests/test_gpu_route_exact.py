"""The choice of experts where fp32, or 64 bits, cannot tell scores apart: against the
definition with scores of 60 decimal digits and exact sums."""
import decimal
from fractions import Fraction

import numpy as np
import pytest

import llambda_b200 as LB

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

D = decimal.Decimal
CTX = decimal.Context(prec=60)
U32 = 2.0 ** -24  # half a step of fp32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def route_reference(logits, k, score, bias=None, groups=1, top_groups=1, group_top=1, renorm=True,
                    scale=1.0):
    """(selected, weights as Python floats, gap between the sums of the last group kept and the
    first one left out), logits and biases finite."""
    l = logits.double().cpu().tolist()
    b = bias.double().cpu().tolist() if bias is not None else [0.0] * logits.shape[1]
    sel, wts, gaps = [], [], []
    with decimal.localcontext(CTX):
        for row in l:
            if score == "softmax":
                p = [(D(v) - D(max(row))).exp() for v in row]
                s = [v / sum(p) for v in p]
            else:
                s = [1 / (1 + (-D(v)).exp()) for v in row]
            # (sums rounded to 60 digits would break ties of other pairs with the same sum)
            c = [Fraction(v) + Fraction(w) for v, w in zip(s, b)]
            size = len(row) // groups
            ranks = [sum(sorted(c[g * size:(g + 1) * size], reverse=True)[:group_top])
                     for g in range(groups)]
            order = sorted(range(groups), key=lambda g: (-ranks[g], g))
            kept = order[:top_groups]
            gaps.append(float(ranks[kept[-1]] - ranks[order[top_groups]])
                        if group_top == 2 and top_groups < groups else 0.0)
            cand = [e for g in kept for e in range(g * size, (g + 1) * size)]
            chosen = sorted(cand, key=lambda e: (-c[e], e))[:k]
            total = sum(s[e] for e in chosen) if renorm else 1
            sel.append(chosen)
            wts.append([float(s[e] / total * D(scale)) for e in chosen])
    return np.array(sel), np.array(wts), np.array(gaps)


def check_choice(logits, k, score, bias=None, least=0.0, **kw):
    """least: sums of two that are nearer to each other, and not equal, are not compared."""
    sel, _ = LB.route_experts(logits, k, score=score, bias=bias, **kw)
    want, _, gaps = route_reference(logits, k, score, bias, **kw)
    got = sel.cpu().numpy()
    told = (gaps == 0) | (gaps >= least)
    assert told.mean() >= 0.5
    bad = np.nonzero(told & (got != want).any(1))[0]
    assert bad.size == 0, (bad.size, bad[:4], got[bad[:4]], want[bad[:4]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("row,best", [([20.0, 20.0, 20.5, 0.0], 2), ([18.0, 18.0, 19.0, 1.0], 2),
                                      ([19.0, 18.0, 18.0, 18.0], 0), ([18.0, 18.0, 18.0, 1.0], 0)])
def test_a_tie_at_the_last_rank_hides_no_better_expert(dtype, row, best):
    """Scores that are all 1.0 in fp32: the two first are equal, a further one is larger."""
    logits = torch.tensor([row], device="cuda").to(dtype)
    sel, _ = LB.route_experts(logits, 1, score="sigmoid", bias=torch.zeros(4, device="cuda"))
    assert sel.tolist() == [[best]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups,top_groups,group_top", [
    (16, 3, 1, 1, 1), (64, 8, 1, 1, 1), (64, 8, 4, 2, 2), (33, 32, 1, 1, 1), (160, 6, 8, 3, 1),
    (512, 10, 1, 1, 1), (6, 6, 1, 1, 1)])
def test_ties_beside_scores_closer_than_fp32_tells_apart(score, E, k, groups, top_groups,
                                                         group_top):
    """A few values of logits, many times each, whose scores (or whose sums with the bias) are
    the same in fp32 and not in 64 bits."""
    g = gen(E + k)
    T = 40 if E < 200 else 12
    levels = torch.tensor([17.5, 18.0, 18.5, 19.0, 20.0, 21.0], device="cuda")
    if score == "softmax":  # a tail far below the largest, swallowed by the bias in fp32
        levels = levels - 36.0
    pick = torch.randint(0, 6, (T, E), generator=g, device="cuda")
    # the larger a value, the rarer: ties at every border
    pick = torch.minimum(pick, torch.randint(0, 6, (T, E), generator=g, device="cuda"))
    logits = levels[pick]
    if score == "softmax":
        logits[:, 0] = 0.0
    for bias in (torch.zeros(E, device="cuda"), torch.full((E,), 0.75, device="cuda")):
        for dtype in (torch.float32, torch.bfloat16):
            check_choice(logits.to(dtype), k, score, bias, groups=groups, top_groups=top_groups,
                         group_top=group_top)


@pytest.mark.parametrize("score,E,groups,top_groups,big,small", [
    ("sigmoid", 4, 2, 1, 100.0, 2e-5), ("sigmoid", 24, 8, 3, 100.0, 2e-5),
    ("sigmoid", 64, 32, 9, 1000.0, 2e-4), ("softmax", 256, 16, 5, 8.0, 1e-3),
    ("softmax", 16, 8, 2, 50.0, 2e-5)])
def test_sums_of_two_that_cancel(score, E, groups, top_groups, big, small):
    """Biases of opposite sign in every group: a sum is small and its rounding is not."""
    g = gen(E + groups)
    T = 600 if E < 100 else 60
    logits = small * randn(g, T, E)
    size = E // groups
    bias = torch.full((E,), -big, device="cuda")
    bias[::size] = big
    kw = dict(groups=groups, top_groups=top_groups, group_top=2)
    check_choice(logits, 1, score, bias, **kw)
    # groups whose sums are as large and whose addends are not
    bias[:size] = 0.0
    bias[0] = 1.0 / E if score == "softmax" else 0.0
    check_choice(logits, 1, score, bias, **kw)
    check_choice(logits, min(size * top_groups, 4), score, None, **kw)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups,top_groups", [(2, 1, 1, 1), (16, 4, 1, 1), (64, 8, 8, 3),
                                                   (60, 5, 5, 2), (1024, 32, 1, 1)])
@pytest.mark.parametrize("lo,hi", [(30.0, 60.0), (-60.0, -30.0), (-1e-8, 1e-8), (37.0, 38.0)])
def test_equal_biases_choose_as_none_does(score, E, k, groups, top_groups, lo, hi):
    """Logits whose scores 64 bits do not tell apart: the logits' order decides."""
    g = gen(E + k)
    logits = torch.rand(20, E, generator=g, device="cuda") * (hi - lo) + lo
    logits[:, ::5] = logits[:, 1:2]  # and true ties
    kw = dict(score=score, groups=groups, top_groups=top_groups)
    for dtype in (torch.float32, torch.bfloat16):
        l = logits.to(dtype)
        want, w = LB.route_experts(l, k, **kw)
        for b in (0.0, 0.3, -1.0, 1e6, -1e30):
            sel, _ = LB.route_experts(l, k, bias=torch.full((E,), b, device="cuda"), **kw)
            assert torch.equal(sel, want), b
        if groups == 1:  # without groups the order is the logits' by definition
            order = torch.sort(l.float(), dim=1, descending=True, stable=True).indices[:, :k]
            assert torch.equal(want.long(), order)


@pytest.mark.parametrize("E,k,groups,top_groups", [(8, 3, 1, 1), (32, 6, 4, 2), (96, 10, 1, 1),
                                                   (24, 2, 3, 1)])
def test_scores_near_one_with_small_biases(E, k, groups, top_groups):
    g = gen(E * k)
    logits = 38 + 22 * torch.rand(30, E, generator=g, device="cuda")
    bias = 1e-20 * randn(g, E)
    for top in (1, 2):
        kw = dict(groups=groups, top_groups=top_groups, group_top=top)
        check_choice(logits, k, "sigmoid", bias, **kw)
        check_choice(logits, k, "sigmoid", bias - 1.0, **kw)
        check_choice(logits, k, "sigmoid", torch.zeros_like(bias), **kw)
    # scores on both sides of one half, and a few far from it
    mixed = torch.where(torch.rand(30, E, generator=g, device="cuda") < 0.5, logits, -logits)
    check_choice(mixed, k, "sigmoid", torch.zeros_like(bias), groups=groups, top_groups=top_groups)


def test_masked_experts_and_unusual_biases_keep_their_order():
    """-inf logits after all others, NaN last, whatever sends a token to the 64-bit choice."""
    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[40.0, 50.0, -inf, nan, 41.0, -inf, 50.0, 30.0]], device="cuda")
    zero = torch.zeros(8, device="cuda")
    sel, _ = LB.route_experts(logits, 8, score="sigmoid", bias=zero)
    assert sel.tolist() == [[1, 6, 4, 0, 7, 2, 5, 3]]
    bias = zero.clone()
    bias[7], bias[0] = inf, -inf
    sel, _ = LB.route_experts(logits, 8, score="sigmoid", bias=bias)
    assert sel.tolist() == [[7, 1, 6, 4, 0, 2, 5, 3]]
    # groups of two: one with a masked expert and one with NaN come last
    sel, _ = LB.route_experts(logits, 4, score="sigmoid", bias=zero, groups=4, top_groups=2,
                              group_top=2)
    assert sel.tolist() == [[1, 6, 0, 7]]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,top_groups", [(64, 8, 3), (24, 8, 2), (256, 8, 4), (96, 32, 7)])
@pytest.mark.parametrize("levels", [[1.0, 1.5, 2.0, 2.5], [17.0, 17.5, 38.0, 40.0, 50.0],
                                    [0.0, 1e-9, 2e-9, 1.0]])
def test_groups_whose_sums_tie(score, E, groups, top_groups, levels):
    """Groups with the same two largest logits, and some that only look so."""
    g = gen(E + len(levels))
    lv = torch.tensor(levels, device="cuda")
    T = 40 if E < 200 else 12
    logits = lv[torch.randint(0, len(levels), (T, E), generator=g, device="cuda")]
    two = 0.25 * torch.randint(0, 2, (E,), generator=g, device="cuda")
    # Four scores of 64 bits, each within 2^-52 (exp a step, two operations half a step each, of a
    # value of at most 1), do not tell sums apart that differ by less than 2^-50 and are not
    # equal.  Logits 0 and 2e-9 against twice 1e-9 (fp32's 2e-9 is twice its 1e-9) give such:
    # 1 / (1 + exp(-l)) = 1/2 + l / 4 - l^3 / 48 + ..., sums 6e-27 / 48 = 1.25e-28 apart.
    least = 2.0 ** -50 if levels[0] == 0.0 else 0.0
    for bias in (None, torch.zeros(E, device="cuda"), two):
        for top in (1, 2):
            check_choice(logits, min(4, top_groups * (E // groups)), score, bias, least,
                         groups=groups, top_groups=top_groups, group_top=top)


# the argument of exp is off by 70 * U32 at most (scores below 2^-100 are computed in 64 bits),
# exp by two steps, the sum of exponentials by 37 adds, then the division, the sum of 32 weights, its
# division, the scale; a weight below fp32's smallest normal number by half of its smallest step
FAINT_RTOL, FAINT_ATOL = (70 + 4 + 37 + 1 + 32 + 1 + 1) * U32, 2.0 ** -150


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,k", [(8, 3), (64, 8), (40, 32)])
def test_weights_of_scores_below_what_fp32_holds(E, k, dtype, renorm):
    g = gen(E + k)
    noise = randn(g, 6, E)
    far = torch.tensor([-70.0, -95.0, -104.0, -200.0, -3000.0, -88.0], device="cuda")[:, None]
    logits = (noise + far).to(dtype)
    mixed = logits.clone()
    mixed[:, 1] = noise[:, 1].to(dtype)  # one ordinary score beside them
    # softmax: the bias keeps the choice off the experts that are not far below the largest
    keep_off = torch.zeros(E, device="cuda")
    keep_off[0] = -10.0
    below = logits.clone()
    below[:, 0] = noise[:, 0].to(dtype)
    for l, score, bias in ((logits, "sigmoid", None), (mixed, "sigmoid", None),
                           (logits, "sigmoid", keep_off), (mixed, "softmax", None),
                           (below, "softmax", keep_off)):
        sel, w = LB.route_experts(l, k, score=score, bias=bias, renormalise=renorm,
                                  weight_scale=2.5)
        rs, rw, _ = route_reference(l, k, score, bias, renorm=renorm, scale=2.5)
        assert np.array_equal(sel.cpu().numpy(), rs)
        np.testing.assert_allclose(w.double().cpu().numpy(), rw, rtol=FAINT_RTOL, atol=FAINT_ATOL)


def test_weights_of_the_farthest_logits():
    for v in (-3e38, -1e30, -800.0):
        logits = torch.full((3, 16), v, device="cuda")
        logits[1, 5], logits[2] = -float("inf"), -float("inf")
        logits[2, 3] = v
        _, w = LB.route_experts(logits, 4, score="sigmoid")
        assert w[:2].tolist() == [[0.25] * 4] * 2 and w[2].tolist() == [1.0, 0.0, 0.0, 0.0]
        bias = torch.zeros(16, device="cuda")
        bias[15], logits[:2, 15] = -5.0, 0.0
        sel, w = LB.route_experts(logits, 4, score="softmax", bias=bias)
        assert w[0].tolist() == [0.25] * 4 and 15 not in sel[0].tolist()


@pytest.mark.parametrize("big", [1.0, 100.0, 1e6])
def test_sums_of_the_same_terms_in_other_pairs_tie(big):
    """(l + B) + (l' - B) and (l' + B) + (l - B): a true tie, whatever each choice rounds."""
    g = gen(int(big))
    T, E = 60, 64
    for levels in ([18.0, 18.5, 19.0, 19.5], [40.0, 40.5, 45.0, 50.0], [-20.0, -3.0, 0.5, 2.0]):
        lv = torch.tensor(levels, device="cuda")
        logits = lv[torch.randint(0, 4, (T, E), generator=g, device="cuda")]
        bias = big * (2.0 * torch.randint(0, 2, (E,), generator=g, device="cuda") - 1.0)
        for groups, top_groups in ((32, 13), (16, 5)):
            check_choice(logits, 8, "sigmoid", bias, groups=groups, top_groups=top_groups,
                         group_top=2)
