"""The choice of experts where fp32, or 64 bits, cannot tell scores apart: against the
definition in 60 decimal digits."""
import decimal

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
    """(selected, weights as Python floats), logits and biases finite."""
    l = logits.double().cpu().tolist()
    b = bias.double().cpu().tolist() if bias is not None else [0.0] * logits.shape[1]
    sel, wts = [], []
    with decimal.localcontext(CTX):
        for row in l:
            if score == "softmax":
                p = [(D(v) - D(max(row))).exp() for v in row]
                s = [v / sum(p) for v in p]
            else:
                s = [1 / (1 + (-D(v)).exp()) for v in row]
            c = [v + D(w) for v, w in zip(s, b)]
            size = len(row) // groups
            ranks = [sum(sorted(c[g * size:(g + 1) * size], reverse=True)[:group_top])
                     for g in range(groups)]
            kept = sorted(range(groups), key=lambda g: (-ranks[g], g))[:top_groups]
            cand = [e for g in kept for e in range(g * size, (g + 1) * size)]
            chosen = sorted(cand, key=lambda e: (-c[e], e))[:k]
            total = sum(s[e] for e in chosen) if renorm else 1
            sel.append(chosen)
            wts.append([float(s[e] / total * D(scale)) for e in chosen])
    return np.array(sel), np.array(wts)


def check_choice(logits, k, score, bias=None, **kw):
    sel, _ = LB.route_experts(logits, k, score=score, bias=bias, **kw)
    want, _ = route_reference(logits, k, score, bias, **kw)
    got = sel.cpu().numpy()
    bad = np.nonzero((got != want).any(1))[0]
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
