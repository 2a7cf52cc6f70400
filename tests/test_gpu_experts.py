"""Routing, 8-bit quantisation, the block-scaled 8-bit product and the routed
experts against their definitions in 64 bits."""
import numpy as np
import pytest

import llambda_b200 as LB

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
U32 = 2.0 ** -24  # half a step of fp32
HALF_STEP = {torch.float32: U32, torch.bfloat16: 2.0 ** -8}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


# ------------------------------------------------------------------ routing


def route_reference(logits, k, score, bias, groups, top_groups, group_top, renorm, scale):
    """The definition, token by token, in Python floats (64 bits)."""
    l = logits.double().cpu().numpy()
    b = bias.double().cpu().numpy() if bias is not None else np.zeros(l.shape[1])
    sel, wts = [], []
    for row in l:
        masked = np.isneginf(row)
        if score == "softmax":
            top = row.max() if not masked.all() else 0.0
            p = np.where(masked, 0.0, np.exp(np.where(masked, 0.0, row) - top))
            s = p / p.sum() if p.sum() else p
        else:
            s = np.where(masked, 0.0, 1.0 / (1.0 + np.exp(-np.where(masked, 0.0, row))))
        c = np.where(masked, -np.inf, s + b)
        size = len(row) // groups
        ranks = [sum(sorted(c[g * size:(g + 1) * size], reverse=True)[:group_top])
                 for g in range(groups)]
        kept = sorted(range(groups), key=lambda g: (-ranks[g], g))[:top_groups]
        cand = [e for g in kept for e in range(g * size, (g + 1) * size)]
        chosen = sorted(cand, key=lambda e: (-c[e], e))[:k]
        w = s[chosen]
        if renorm:
            w = w / w.sum() if w.sum() else w * 0.0
        sel.append(chosen)
        wts.append(w * scale)
    return np.array(sel), np.array(wts)


# the score's error is at most: the argument's rounding (20 * U32), exp (2 steps), the sum of
# exponentials (37 adds), the division; then the sum of 32 weights, its division, the scale
WEIGHT_RTOL = (20 + 4 + 37 + 1 + 32 + 1 + 1) * U32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k,groups,top_groups,group_top", [
    (1, 1, 1, 1, 1, 1), (3, 7, 7, 1, 1, 1), (5, 33, 32, 1, 1, 1), (130, 64, 6, 1, 1, 1),
    (9, 128, 6, 4, 2, 1), (257, 256, 8, 8, 4, 2), (33, 160, 6, 8, 3, 1), (6, 512, 10, 1, 1, 1),
    (4, 1024, 32, 32, 31, 2), (8, 64, 2, 32, 1, 2), (7, 96, 3, 3, 3, 2),
])
@pytest.mark.parametrize("biased", [False, True])
def test_route(dtype, score, T, E, k, groups, top_groups, group_top, biased):
    g = gen(T * 1000 + E)
    logits = (2 * randn(g, T, E)).to(dtype)
    bias = 0.1 * randn(g, E) if biased else None
    sel, w = LB.route_experts(logits, k, score=score, bias=bias, groups=groups,
                              top_groups=top_groups, group_top=group_top, weight_scale=1.5)
    rs, rw = route_reference(logits, k, score, bias, groups, top_groups, group_top, True, 1.5)
    assert np.array_equal(sel.cpu().numpy(), rs)
    np.testing.assert_allclose(w.cpu().numpy(), rw, rtol=WEIGHT_RTOL)
    _, w = LB.route_experts(logits, k, score=score, bias=bias, groups=groups,
                            top_groups=top_groups, group_top=group_top, renormalise=False)
    _, rw = route_reference(logits, k, score, bias, groups, top_groups, group_top, False, 1.0)
    np.testing.assert_allclose(w.cpu().numpy(), rw, rtol=WEIGHT_RTOL)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_route_scores_closer_than_fp32_tells_apart(score, groups, top_groups):
    """Choices (score + bias) that fp32 rounds to the same or the wrong order."""
    g = gen(7)
    T, E, k = 64, 64, 8
    logits = randn(g, T, E)
    l = logits.double()
    s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    # a bias that levels the first row's choices to within fp32's rounding of it
    bias = (1.0 - s[0]).float()
    logits[1:32] = logits[0]
    kw = dict(groups=groups, top_groups=top_groups, group_top=2)
    sel, _ = LB.route_experts(logits, k, score=score, bias=bias, **kw)
    rs, _ = route_reference(logits, k, score, bias, groups, top_groups, 2, True, 1.0)
    assert np.array_equal(sel.cpu().numpy(), rs)


def test_route_ties_and_masks():
    inf = float("inf")
    E = 48
    logits = torch.zeros(6, E, device="cuda")
    logits[1] = -inf                       # nothing left
    logits[2, 3:] = -inf                   # fewer experts left than are chosen
    logits[3, ::2] = 1.0                   # ties
    logits[4, 5] = float("nan")
    logits[5, :] = -0.0
    logits[5, 40] = 0.0                    # equal to -0
    for score in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(E, device="cuda")):
            sel, w = (v.cpu().numpy() for v in LB.route_experts(logits, 5, score=score, bias=bias))
            assert list(sel[0]) == [0, 1, 2, 3, 4] and np.allclose(w[0], 0.2, rtol=1e-6)
            assert list(sel[1]) == [0, 1, 2, 3, 4] and not w[1].any()
            assert list(sel[2]) == [0, 1, 2, 3, 4]
            assert np.allclose(w[2], [1 / 3] * 3 + [0, 0], rtol=1e-6)
            assert list(sel[3]) == [0, 2, 4, 6, 8]
            if score == "sigmoid":  # an expert with NaN comes after all others
                assert list(sel[4]) == [0, 1, 2, 3, 4] and np.allclose(w[4], 0.2, rtol=1e-6)
            else:                   # every score of the row is NaN
                assert np.isnan(w[4]).all()
            assert list(sel[5]) == [0, 1, 2, 3, 4]


def test_route_host_form_strides_and_refusals():
    g = gen(3)
    wide = randn(g, 9, 70)
    logits = wide[:, 3:67]
    sel, w = LB.route_experts(logits, 4)
    want = LB.route_experts(logits.contiguous(), 4)
    assert torch.equal(sel, want[0]) and torch.equal(w, want[1])
    hs, hw = LB.route_experts(logits.cpu().numpy(), 4)
    assert np.array_equal(hs, sel.cpu().numpy()) and np.array_equal(hw, w.cpu().numpy())
    with pytest.raises(ValueError, match="unit stride"):
        LB.route_experts(wide.t(), 2)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        LB.route_experts(logits.half(), 2)
    with pytest.raises(ValueError, match="bias"):
        LB.route_experts(logits, 2, bias=torch.zeros(8, device="cuda"))
    with pytest.raises(LB.LlambdaCudaError, match="equal groups"):
        LB.route_experts(logits, 2, groups=5)
    with pytest.raises(LB.LlambdaCudaError, match="top_k"):
        LB.route_experts(logits, 33)
    with pytest.raises(ValueError, match="positive token count"):
        LB.route_experts(logits[:0], 2)
    with pytest.raises(ValueError, match="no backward"):
        LB.route_experts(logits.clone().requires_grad_(), 2)


# ------------------------------------------------------------------ quantiser


def e4m3(v):
    """v (double, |v| <= 448) rounded to e4m3, ties to even; and the step there."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(v / step) * step, step


def blocks_of(x):
    T, K = x.shape
    KB = -(-K // 128)
    p = torch.zeros(T, KB * 128, dtype=torch.float64, device=x.device)
    p[:, :K] = x.double()
    return p.view(T, KB, 128)


def quantize_reference(x):
    """(q [T][KB][128], scales [T][KB]): each fp32 quantity rounded once."""
    p = blocks_of(x)
    s = (p.abs().amax(2) / 448).float().double().clamp(min=2.0 ** -126)
    return e4m3((p / s[:, :, None]).float().double())[0], s


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 128), (3, 16), (5, 130), (17, 400), (33, 2688),
                                 (129, 1040), (1000, 257)])
def test_quantize(dtype, T, K):
    g = gen(T + K)
    x = (randn(g, T, K) * torch.exp2(6 * randn(g, T, 1))).to(dtype)
    x[0] = 0
    q, s = LB.fp8_quantize(x)
    rq, rs = quantize_reference(x)
    KB, TP = -(-K // 128), -(-T // 4) * 4
    assert q.shape == (T, -(-K // 16) * 16) and s.shape == (KB, TP)
    assert torch.equal(q[:, :K].double(), rq.flatten(1)[:, :K])
    assert torch.equal(s[:, :T].double(), rs.t())
    assert not q[:, K:].float().any() and not s[:, T:].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_every_magnitude(dtype):
    """Blocks from below the smallest scale to the largest number, and values that are exact
    ties of the type at their scale: the quotient has to be the correctly rounded one."""
    g = gen(6)
    e = torch.arange(-149, 128, device="cuda", dtype=torch.float64)
    x = torch.rand(e.numel(), 384, generator=g, device="cuda").double() * 2 - 1
    x = (x * torch.exp2(e)[:, None]).clamp(-3e38, 3e38)
    # a power of two times 448 as the block's largest: every quotient is exact, many are ties
    ties = torch.randint(0, 449 * 16, (e.numel(), 128), generator=g, device="cuda").double() / 16
    ties[:, 0] = 448
    x[:, 128:256] = (ties * torch.exp2(e)[:, None]).clamp(-3e38, 3e38)
    x = x.float().to(dtype)
    q, s = LB.fp8_quantize(x)
    rq, rs = quantize_reference(x)
    assert torch.equal(s[:, :x.shape[0]].double(), rs.t())
    assert torch.equal(q.double(), rq.flatten(1))


def test_quantize_strides_and_special_values():
    g = gen(5)
    wide = randn(g, 40, 300)
    for x in (wide[:, 1:258], wide[:, 4:132], wide[::2, :200], wide[3:4, 7:8]):
        q, s = LB.fp8_quantize(x)
        q2, s2 = LB.fp8_quantize(x.contiguous())
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    x = torch.zeros(4, 256, device="cuda")
    x[0, 0], x[0, 1], x[0, 128] = float("inf"), 3.0, 5.0
    x[1, 7], x[1, 130] = float("nan"), 5.0
    x[2] = 1e-44
    x[3] = torch.finfo(torch.float32).max
    q, s = LB.fp8_quantize(x)
    f = q.float()
    assert s[0, 0].isinf() and f[0, 0].isnan() and f[0, 1] == 0 and f[0, 128] == 448
    assert s[0, 1].isnan() and f[1, :128].isnan().all() and f[1, 130] == 448
    assert s[0, 2] == 2.0 ** -126 and not f[2].any()
    assert (f[3] == 448).all() and torch.isfinite(s[:, 3]).all()


# ------------------------------------------------------------------ products


def matrices(g, *shape):
    """e4m3 weights over the whole range of the type, with block scales of either sign."""
    w = (randn(g, *shape) * 40).clamp(-448, 448).to(E4M3)
    s = randn(g, *shape[:-2], -(-shape[-2] // 128), -(-shape[-1] // 128)) * 0.01
    return w, s


def product_reference(q, sx, w, s):
    """(y, bound): the product of quantised rows with one matrix, and how far fp32 may be off:
    a block's sum of 128 products by 127 steps of 2^-23 (adders that cut), the scale product,
    the FMA over the blocks and its own sum by a step each, relative to the sum of magnitudes."""
    T, KB, _ = q.shape
    N, K = w.shape
    y = torch.zeros(T, N, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(y)
    for b in range(KB):
        wb = w[:, 128 * b:128 * b + 128].double()
        f = sx[:, b:b + 1] * s[:, b].double().repeat_interleave(128)[:N]
        qb = q[:, b, :wb.shape[1]]
        y += (qb @ wb.t()) * f
        mag += (qb.abs() @ wb.abs().t()) * f.abs()
    return y, mag * (127 * 2 + KB + 2) * U32


def check(out, y, bound):
    t = out.dtype
    err = (out.double() - y).abs()
    lim = bound + HALF_STEP[t] * (y.abs() + bound)
    assert torch.isfinite(out).all() and bool((err <= lim).all()), float((err / lim).max())


SIZES = [(1, 1, 16), (1, 300, 400), (2, 128, 128), (5, 64, 112), (16, 130, 1040), (17, 257, 144),
         (33, 2688, 1856), (64, 128, 2064), (65, 96, 256), (129, 384, 384), (300, 200, 640),
         (513, 1030, 272), (1, 4096, 4096), (31, 4096, 8192), (48, 200, 4112), (100, 128, 4096),
         (127, 2700, 528), (300, 20000, 272), (257, 19000, 144), (1025, 5000, 400),
         (1, 20000, 8192), (4, 300, 4096), (3, 128, 8208), (2, 20000, 8208), (16, 640, 1024),
         (7, 130, 16), (1, 1000, 16400),
         (24, 4096, 4096), (32, 2688, 512), (17, 130, 1536), (31, 256, 144)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,N,K", SIZES)
def test_projection(dtype, T, N, K):
    g = gen(T + N + K)
    x = randn(g, T, K).to(dtype)
    w, s = matrices(g, N, K)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    out = p.run_device(x)
    q, sx = quantize_reference(x)
    y, bound = product_reference(q, sx, w, s)
    assert out.dtype == dtype and out.shape == (T, N)
    check(out, y, bound)
    other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16
    check(p.run_device(x, out_dtype=other), y, bound)
    # the same bits from rows that were quantised before, and from a second call
    assert torch.equal(p.run_quantized(*LB.fp8_quantize(x), T, out_dtype=dtype), out)
    assert torch.equal(p.run_device(x), out)
    assert p.status() == 0
    p.close()


@pytest.mark.parametrize("N,K", [(5, 7), (130, 100), (257, 401), (128, 1)])
def test_projection_from_host(N, K):
    """Host tensors have any width; host and device calls agree."""
    g = gen(N * K)
    w, s = matrices(g, N, K)
    p = LB.Fp8ProjectionSession.from_tensor(w.view(torch.uint8).cpu().numpy(), s.cpu().numpy())
    x = randn(g, 19, K)
    out = p.run_device(x)
    y, bound = product_reference(*quantize_reference(x), w, s)
    check(out, y, bound)
    assert np.array_equal(p.run(x.cpu().numpy()), out.cpu().numpy())
    assert np.array_equal(p.run(x[3].cpu().numpy()), p.run_device(x[3:4]).cpu().numpy()[0])


@pytest.mark.parametrize("T,N,K", [(3, 128, 8192), (16, 300, 4096), (50, 128, 4112),
                                   (300, 128, 2064), (600, 5000, 400)])
def test_rows_do_not_depend_on_their_place(T, N, K):
    """The same rows in another order give the same bits, long K shared by CTAs too."""
    g = gen(T + K)
    w, s = matrices(g, N, K)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    x = randn(g, T, K)
    order = torch.randperm(T, generator=g, device="cuda")
    assert torch.equal(p.run_device(x[order].contiguous()), p.run_device(x)[order])


def test_experts_rows_do_not_depend_on_their_place():
    g = gen(27)
    E, k, H, I = 3, 2, 2048, 1552
    up, down, gate = matrices(g, E, I, H), matrices(g, E, 400, I), matrices(g, E, I, H)
    for gated in (gate, None):
        m = LB.Fp8MoeSession.from_device(up=up, down=down, gate=gated)
        for T in (2, 20, 140):
            x, wt = randn(g, T, H), randn(g, T, k)
            sel = torch.randint(0, E, (T, k), generator=g, device="cuda").int()
            order = torch.randperm(T, generator=g, device="cuda")
            want = m.run_device(x, sel, wt)
            got = m.run_device(x[order].contiguous(), sel[order].contiguous(),
                               wt[order].contiguous())
            assert torch.equal(got, want[order])
            assert torch.equal(m.run_device(x, sel, wt), want)


def test_projection_views_leave_the_rest_alone():
    g = gen(11)
    w, s = matrices(g, 200, 160)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    wide = randn(g, 50, 400)
    for T in (1, 7, 40):
        x = wide[2:2 + T, 5:165]
        want = p.run_device(x.contiguous())
        big = torch.full((60, 333), 7.0, device="cuda")
        p.run_device(x, out=big[4:4 + T, 9:209])
        assert torch.equal(big[4:4 + T, 9:209], want)
        big[4:4 + T, 9:209] = 7.0
        assert bool((big == 7.0).all())


def test_projection_special_values():
    g = gen(12)
    w, s = matrices(g, 64, 256)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    x = randn(g, 20, 256)
    want = p.run_device(x)
    x[3, 17], x[4, 200], x[5] = float("nan"), float("inf"), 0.0
    out = p.run_device(x)
    assert out[3].isnan().all() and out[4].isnan().any() and not out[5].any()
    rest = [i for i in range(20) if i not in (3, 4, 5)]
    assert torch.equal(out[rest], want[rest])


def test_product_refusals():
    g = gen(13)
    w, s = matrices(g, 64, 64)
    with pytest.raises(LB.LlambdaCudaError, match="multiple of 16"):
        LB.Fp8ProjectionSession.from_device(w[:, :40].contiguous(), s)
    with pytest.raises(ValueError, match="contiguous"):
        LB.Fp8ProjectionSession.from_device(w[:, :32], s)
    with pytest.raises(ValueError, match="scales"):
        LB.Fp8ProjectionSession.from_device(w, s[:0])
    with pytest.raises(LB.LlambdaCudaError, match="not finite"):
        LB.Fp8ProjectionSession.from_device(w, s * float("inf"))
    with pytest.raises(LB.LlambdaCudaError, match="not finite"):
        LB.Fp8ProjectionSession.from_tensor(np.zeros((4, 4), np.uint8), np.full((1, 1), np.nan))
    p = LB.Fp8ProjectionSession.from_device(w, s)
    x = randn(g, 3, 64)
    for bad, match in ((x[:, :63], "shape"), (x.double(), "float32"), (x[:0], "positive"),
                       (x.t(), "shape"), (x.cpu(), "CUDA"), (x[0], "shape")):
        with pytest.raises(ValueError, match=match):
            p.run_device(bad)
    with pytest.raises(ValueError, match="shape"):
        p.run_device(x, out=torch.empty(3, 63, device="cuda"))
    q, sc = LB.fp8_quantize(x)
    with pytest.raises(ValueError, match="shape"):
        p.run_quantized(q, sc[:, :3], 3)
    # C calls: a workspace that is too small, host memory, a short row stride
    from llambda_b200 import _native as N
    x = randn(g, 40, 64)
    L, out = N.lib(), torch.empty(40, 64, device="cuda")
    work = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    assert 0 < L.llambda_cuda_fp8_session_workspace(p._h, 40) <= work.numel()
    args = [p._h, 0, x.data_ptr(), 64, 40, 0, out.data_ptr(), 64, work.data_ptr(), work.numel(),
            None]

    def call(i, v):
        return L.llambda_cuda_fp8_session_run_device(*(args[:i] + [v] + args[i + 1:]))

    assert call(9, 8) == -1 and "workspace" in N.last_error()
    assert call(8, None) == -1 and "workspace" in N.last_error()
    assert call(8, work.data_ptr() + 16) == -1 and "256-byte" in N.last_error()
    assert call(3, 63) == -1 and "row stride" in N.last_error()
    assert call(1, 1) == -1 and "element type" in N.last_error()
    assert call(4, 0) == -1 and "token count" in N.last_error()
    host = np.zeros((40, 64), np.float32)
    assert call(2, host.ctypes.data) == -1 and "device memory" in N.last_error()
    assert call(3, 64) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, p.run_device(x))
    # a few rows need none
    assert L.llambda_cuda_fp8_session_workspace(p._h, 1) == 0
    args[4:5], args[8:10] = [1], [None, 0]
    assert call(3, 64) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[:1], p.run_device(x[:1]))


def test_an_output_over_an_input_is_refused():
    g = gen(31)
    w, s = matrices(g, 128, 128)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    up, down = matrices(g, 4, 256, 128), matrices(g, 4, 128, 256)
    m = LB.Fp8MoeSession.from_device(up=up, down=down)
    for T in (1, 3, 70):
        buf = randn(g, T + 1, 272)
        sel = torch.randint(0, 4, (T, 2), generator=g, device="cuda").int()
        wt = randn(g, T, 2)
        x = buf[:T, :128]
        want, keep = p.run_device(x.clone()), x.clone()
        # the same place, a shared column, a row further on, an unequal stride
        bad = [x, buf[:T, 127:255], torch.as_strided(buf, (T, 128), (136, 1), 0)]
        if T > 1:
            bad.append(buf[1:T + 1, :128])
        for out in bad:
            with pytest.raises(LB.LlambdaCudaError, match="overlaps the input"):
                p.run_device(x, out=out)
            with pytest.raises(LB.LlambdaCudaError, match="overlaps the input"):
                m.run_device(x, sel, wt, out=out)
        assert torch.equal(x, keep)
        # columns next to each other, on either side
        assert torch.equal(p.run_device(x, out=buf[:T, 128:256]), want)
        buf[:T, 144:272] = keep
        assert torch.equal(p.run_device(buf[:T, 144:272], out=buf[:T, 16:144]), want)
        big = torch.randn(T * 128, generator=g, device="cuda")
        with pytest.raises(LB.LlambdaCudaError, match="overlaps the weights"):
            m.run_device(keep, sel, big[:2 * T].view(T, 2), out=big.view(T, 128))


# ------------------------------------------------------------------ routed experts


def experts_reference(x, sel, wt, up, down, gate):
    """(out, bound): 64 bits, and how far fp32 may be off.  The intermediate h is rounded to
    e4m3: where its exact quotient lies within its own error of a rounding border, the other
    neighbour (a whole step away) is as right."""
    T, O = x.shape[0], down[0].shape[1]
    q, sx = quantize_reference(x)
    out = torch.zeros(T, O, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    for t in range(T):
        for j in range(sel.shape[1]):
            e = int(sel[t, j])
            if not 0 <= e < up[0].shape[0]:
                continue
            u, du = product_reference(q[t:t + 1], sx[t:t + 1], up[0][e], up[1][e])
            if gate is None:
                h, dh = torch.relu(u) ** 2, 2.0 * torch.relu(u) * du + du * du
            else:
                v, dv = product_reference(q[t:t + 1], sx[t:t + 1], gate[0][e], gate[1][e])
                a = v * torch.sigmoid(v)  # |silu'| <= 1.1
                h, dh = a * u, (1.1 * dv + 8 * U32 * a.abs()) * (u.abs() + du) + a.abs() * du
            dh = dh + 8 * U32 * h.abs()
            p, dp = blocks_of(h), blocks_of(dh)
            s = (p.abs().amax(2) / 448).clamp(min=2.0 ** -126)
            ds = dp.amax(2) / 448 / s + 2 * U32  # relative
            v = p / s[:, :, None]
            dv = dp / s[:, :, None] + v.abs() * (ds[:, :, None] + 2 * U32)
            hq, step = e4m3(v)
            lo, _ = e4m3(v - dv)
            hi, _ = e4m3(v + dv)
            slack = torch.maximum((hq - lo).abs(), (hi - hq).abs()) + hq.abs() * ds[:, :, None]
            y, dy = product_reference(hq, s, down[0][e], down[1][e])
            mag, _ = product_reference(slack, s, down[0][e].float().abs(), down[1][e].abs())
            w = float(wt[t, j])
            out[t] += w * y[0]
            bound[t] += abs(w) * ((dy + mag)[0] + 4 * U32 * y[0].abs())
    return out, bound + sel.shape[1] * U32 * bound


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("T,E,k,H,I,O", [
    (1, 1, 1, 16, 16, 16), (1, 8, 4, 256, 128, 256), (3, 5, 5, 144, 80, 100),
    (9, 16, 3, 128, 192, 128), (40, 4, 2, 160, 144, 160), (70, 2, 2, 64, 272, 65),
    (200, 1, 1, 128, 128, 130), (1, 4, 2, 2688, 1856, 2688), (60, 4, 2, 96, 144, 128),
    (40, 2, 1, 1024, 640, 512), (60, 2, 1, 1040, 528, 528), (2, 64, 40, 64, 128, 64),
    (10, 64, 40, 128, 64, 80), (300, 2, 1, 256, 256, 1000)])
def test_experts(dtype, gated, T, E, k, H, I, O):
    g = gen(T * 7 + H)
    x = randn(g, T, H).to(dtype)
    up, down = matrices(g, E, I, H), matrices(g, E, O, I)
    gate = matrices(g, E, I, H) if gated else None
    sel = torch.rand(T, E, generator=g, device="cuda").topk(k, dim=1).indices.int()
    sel[torch.rand(T, k, generator=g, device="cuda") < 0.1] = -1
    wt = randn(g, T, k)
    m = LB.Fp8MoeSession.from_device(up=up, down=down, gate=gate)
    out = m.run_device(x, sel, wt)
    y, bound = experts_reference(x, sel, wt, up, down, gate)
    assert out.dtype == dtype and out.shape == (T, O)
    check(out, y, bound)
    assert torch.equal(m.run_device(x, sel, wt), out)
    if dtype == torch.float32:
        host = LB.Fp8MoeSession.from_tensor(*[
            None if p is None else (p[0].view(torch.uint8).cpu().numpy(), p[1].cpu().numpy())
            for p in (up, down, gate)])
        got = host.run(x.cpu().numpy(), sel.cpu().numpy(), wt.cpu().numpy())
        assert np.array_equal(got, out.cpu().numpy())
    assert m.status() == 0


def test_experts_do_not_depend_on_the_batch():
    """A token's result has the same bits alone, in a batch, and beside skipped entries (at
    widths too small for CTAs to share them out, which another number of tiles may change)."""
    g = gen(21)
    E, k, H, I, T = 12, 3, 192, 160, 150
    up, down, gate = matrices(g, E, I, H), matrices(g, E, H, I), matrices(g, E, I, H)
    m = LB.Fp8MoeSession.from_device(up=up, down=down, gate=gate)
    x, wt = randn(g, T, H), randn(g, T, k)
    sel = torch.randint(0, E, (T, k), generator=g, device="cuda").int()  # repeated experts too
    out = m.run_device(x, sel, wt)
    for t in (0, 77, 149):
        assert torch.equal(m.run_device(x[t:t + 1], sel[t:t + 1], wt[t:t + 1])[0], out[t])
    part = sel.clone()
    part[::2] = torch.tensor([-1, E, 1 << 30], device="cuda", dtype=torch.int32)
    got = m.run_device(x, part, wt)
    assert torch.equal(got[1::2], out[1::2]) and not got[::2].any()
    one = torch.full_like(sel, 5)  # every token to one expert
    got = m.run_device(x, one, wt)
    for t in (0, 149):
        assert torch.equal(m.run_device(x[t:t + 1], one[t:t + 1], wt[t:t + 1])[0], got[t])


def test_experts_keep_special_values_to_their_token():
    g = gen(23)
    E, k, H, I, T = 4, 2, 160, 144, 30
    up, down, gate = matrices(g, E, I, H), matrices(g, E, H, I), matrices(g, E, I, H)
    sel = torch.randint(0, E, (T, k), generator=g, device="cuda").int()
    x, wt = randn(g, T, H), randn(g, T, k)
    for gated in (gate, None):
        m = LB.Fp8MoeSession.from_device(up=up, down=down, gate=gated)
        want = m.run_device(x, sel, wt)
        bad = x.clone()
        bad[3, 5], bad[7, 100], bad[11] = float("nan"), float("inf"), 0.0
        out = m.run_device(bad, sel, wt)
        assert out[3].isnan().all() and out[7].isnan().any() and not out[11].any()
        rest = [t for t in range(T) if t not in (3, 7, 11)]
        assert torch.equal(out[rest], want[rest])


def test_experts_without_any_entry_give_zeros():
    g = gen(24)
    up, down = matrices(g, 3, 64, 32), matrices(g, 3, 40, 64)
    m = LB.Fp8MoeSession.from_device(up=up, down=down)
    for T, k in ((1, 1), (5, 2), (300, 4)):
        x, wt = randn(g, T, 32), randn(g, T, k)
        sel = torch.full((T, k), -7, dtype=torch.int32, device="cuda")
        big = torch.full((T + 2, 50), 9.0, device="cuda")
        m.run_device(x, sel, wt, out=big[1:1 + T, 3:43])
        assert not big[1:1 + T, 3:43].any()
        big[1:1 + T, 3:43] = 9.0
        assert bool((big == 9.0).all())
        sel[T - 1, 0] = 2  # one entry only: the last token's
        out = m.run_device(x, sel, wt)
        y, bound = experts_reference(x, sel, wt, up, down, None)
        check(out, y, bound)


def test_experts_views_leave_the_rest_alone():
    g = gen(25)
    up, down = matrices(g, 6, 128, 96), matrices(g, 6, 112, 128)
    m = LB.Fp8MoeSession.from_device(up=up, down=down)
    wide = randn(g, 400, 200)
    for T in (1, 30, 390):
        x = wide[3:3 + T, 7:103]
        sel = torch.randint(0, 6, (T, 2), generator=g, device="cuda").int()
        wt = randn(g, T, 2)
        want = m.run_device(x.contiguous(), sel, wt)
        big = torch.full((T + 5, 301), 4.0, device="cuda")
        m.run_device(x, sel, wt, out=big[2:2 + T, 5:117])
        assert torch.equal(big[2:2 + T, 5:117], want)
        big[2:2 + T, 5:117] = 4.0
        assert bool((big == 4.0).all())


def test_offsets_past_32_bits():
    """Rows of x and of out that start more than 2^31 elements in."""
    g = gen(26)
    N, K, T = 65536, 128, 40000
    w, s = matrices(g, N, K)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    x = randn(g, T, K).to(torch.bfloat16)
    out = p.run_device(x)
    assert out.numel() > 2 ** 31
    rows = torch.tensor([0, 32767, 32768, 39999], device="cuda")
    y, bound = product_reference(*quantize_reference(x[rows]), w, s)
    check(out[rows], y, bound)
    del out
    wide = torch.empty(9000, 262144, dtype=torch.bfloat16, device="cuda")
    assert wide.numel() > 2 ** 31
    wide[:, 70:70 + K] = x[:9000]
    view = wide[:, 70:70 + K]
    assert torch.equal(p.run_device(view[8900:]), p.run_device(x[8900:9000].contiguous()))
    q, sc = LB.fp8_quantize(view)
    q2, sc2 = LB.fp8_quantize(x[:9000].contiguous())
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(sc, sc2)
    wide[:, 70:70 + K] = randn(g, 9000, K).to(torch.bfloat16)
    sel, wt = LB.route_experts(view, 4)
    sel2, wt2 = LB.route_experts(view.contiguous(), 4)
    assert torch.equal(sel, sel2) and torch.equal(wt, wt2)


def test_experts_refusals():
    g = gen(22)
    up, down = matrices(g, 2, 64, 32), matrices(g, 2, 32, 64)
    m = LB.Fp8MoeSession.from_device(up=up, down=down)
    x, sel, wt = randn(g, 4, 32), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), randn(g, 4, 2)
    with pytest.raises(LB.LlambdaCudaError, match="down tensor"):
        LB.Fp8MoeSession.from_device(up=up, down=up)
    with pytest.raises(LB.LlambdaCudaError, match="gate tensor"):
        LB.Fp8MoeSession.from_device(up=up, down=down, gate=down)
    for args in ((x[:, :16], sel, wt), (x, sel.long(), wt), (x, sel[:3], wt), (x, sel, wt[:, :1]),
                 (x, sel, wt.double()), (x[:0], sel[:0], wt[:0]), (x, sel[:, :0], wt[:, :0]),
                 (x, sel.t().contiguous().t(), wt)):
        with pytest.raises(ValueError):
            m.run_device(*args)
    m.close()
    with pytest.raises(ValueError, match="closed"):
        m.run_device(x, sel, wt)


# ------------------------------------------------------------------ as they are used


def layer(g, T, E=16, k=4, H=256, I=192):
    router = randn(g, E, H) / 16
    up, down, gate = matrices(g, E, I, H), matrices(g, E, H, I), matrices(g, E, I, H)
    proj = matrices(g, H, H)
    bias = 0.05 * randn(g, E)
    keep = (router, up, down, gate, proj, bias)
    rs = LB.ProjectionSession.from_device(LB.TYPE_F32, H, E, router)
    ps = LB.Fp8ProjectionSession.from_device(*proj)
    ms = LB.Fp8MoeSession.from_device(up=up, down=down, gate=gate)

    def run(x, stream=None):
        stream = stream or torch.cuda.current_stream()
        with torch.cuda.stream(stream):
            h = ps.run_device(x)
            logits = torch.empty(x.shape[0], E, device="cuda")
            rs.run_device(h, logits, x.shape[0], stream)
            sel, wt = LB.route_experts(logits, k, score="sigmoid", bias=bias, groups=4,
                                       top_groups=2, group_top=2, weight_scale=2.0)
            return h, logits, sel, wt, ms.run_device(h, sel, wt)

    return run, keep


def test_a_layer_of_them():
    """Projection, router, choice, experts: each step against its definition on what the step
    before gave."""
    g = gen(31)
    run, (router, up, down, gate, proj, bias) = layer(g, 23)
    x = randn(g, 23, 256)
    h, logits, sel, wt, out = run(x)
    check(h, *product_reference(*quantize_reference(x), *proj))
    rs, rw = route_reference(logits, 4, "sigmoid", bias, 4, 2, 2, True, 2.0)
    assert np.array_equal(sel.cpu().numpy(), rs)
    np.testing.assert_allclose(wt.cpu().numpy(), rw, rtol=WEIGHT_RTOL)
    check(out, *experts_reference(h, sel, wt, up, down, gate))


def test_a_captured_layer_replays_on_new_inputs():
    g = gen(32)
    run, _keep = layer(g, 9)
    x = randn(g, 9, 256)
    run(x)
    graphs = []
    for _ in range(2):  # two graphs of the same sessions, replayed side by side
        xin = x.clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = run(xin)
        graphs.append((gr, xin, res))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    new = [randn(g, 9, 256) for _ in range(2)]
    want = [run(v) for v in new]
    torch.cuda.synchronize()
    for (gr, xin, _), st, v in zip(graphs, streams, new):
        xin.copy_(v)
    torch.cuda.synchronize()
    for _ in range(20):
        for (gr, _, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for (_, _, res), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(res, w))


def test_two_streams_share_the_sessions():
    g = gen(33)
    E, k, H, I = 8, 2, 256, 256
    up, down, gate = matrices(g, E, I, H), matrices(g, E, H, I), matrices(g, E, I, H)
    proj = matrices(g, 512, H)
    ms = LB.Fp8MoeSession.from_device(up=up, down=down, gate=gate)
    ps = LB.Fp8ProjectionSession.from_device(*proj)
    xs = [randn(g, T, H) for T in (5, 90)]
    sels = [torch.randint(0, E, (v.shape[0], k), generator=g, device="cuda").int() for v in xs]
    wts = [randn(g, v.shape[0], k) for v in xs]
    want = [(ps.run_device(x), ms.run_device(x, s, w)) for x, s, w in zip(xs, sels, wts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(30):
        for i, st in enumerate(streams):
            got[i].append((ps.run_device(xs[i], stream=st),
                           ms.run_device(xs[i], sels[i], wts[i], stream=st.cuda_stream)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


def test_the_status_waits_for_every_stream():
    g = gen(34)
    w, s = matrices(g, 4096, 4096)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    x = randn(g, 2048, 4096)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    for _ in range(50):
        out = p.run_device(x, stream=st)
    assert p.status() == 0 and st.query()
    assert torch.equal(out, p.run_device(x))
