"""Calls of the routing and 8-bit entry points that are refused, and how they deal with
streams and memory."""
import ctypes as C

import pytest

import llambda_b200 as LB
from llambda_b200 import _native as N

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_experts import (U32, blocks_of, check, e4m3, gen, matrices,  # noqa: E402
                              product_reference, quantize_reference, randn)


def refused(rc, match):
    assert rc == -1 and match in N.last_error(), (rc, N.last_error())


def test_routing_refuses_outputs_that_overlap():
    g = gen(1)
    T, E, k = 40, 16, 4
    logits, bias = randn(g, T, E), randn(g, E)
    sel = torch.empty(T, k, dtype=torch.int32, device="cuda")
    wts = torch.empty(T, k, device="cuda")
    d = N.RouteDesc(E, k, 0, 1, 1, 1, 1, 1.0)

    def call(s, w, b=bias.data_ptr()):
        return N.lib().llambda_cuda_route_device(C.byref(d), 0, logits.data_ptr(), E, b, T, s, w,
                                                 None)

    s, w, nb = sel.data_ptr(), wts.data_ptr(), T * k * 4
    buf = torch.zeros(2 * nb, dtype=torch.uint8, device="cuda")
    at = buf.data_ptr()
    refused(call(bias.data_ptr(), w), "overlaps the bias")
    refused(call(s, bias.data_ptr()), "overlaps the bias")
    refused(call(s, at, at + nb - 4), "overlaps the bias")
    refused(call(at, w, at + nb - 4), "overlaps the bias")
    refused(call(s, s), "overlaps the output of weights")
    refused(call(at, at + nb - 4), "overlaps the output of weights")
    refused(call(at + nb - 4, at), "overlaps the output of weights")
    # next to each other
    assert call(at, at + nb) == 0 and call(at + nb, at) == 0 and call(s, w) == 0
    torch.cuda.synchronize()
    assert torch.equal(buf[:nb].view(torch.float32).view(T, k), wts)
    assert torch.equal(buf[nb:].view(torch.int32).view(T, k), sel)


def test_the_quantiser_refuses_outputs_that_overlap():
    g = gen(2)
    T, K = 24, 256
    x = randn(g, T, K)
    nq, ns = T * K, 2 * T * 4
    buf = torch.zeros(nq + ns, dtype=torch.uint8, device="cuda")
    at = buf.data_ptr()

    def call(q, s):
        return N.lib().llambda_cuda_fp8_quantize_device(0, x.data_ptr(), K, T, K, q, s, None)

    refused(call(at, at), "overlaps the output of scales")
    refused(call(at, at + nq - 16), "overlaps the output of scales")
    refused(call(at + ns - 16, at), "overlaps the output of scales")
    assert call(at, at + nq) == 0
    torch.cuda.synchronize()
    q, s = LB.fp8_quantize(x)
    assert torch.equal(buf[:nq], q.view(torch.uint8).flatten())
    assert torch.equal(buf[nq:].view(torch.float32), s.flatten())


def test_products_refuse_outputs_and_workspaces_that_overlap():
    g = gen(3)
    H = 256
    whole = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")
    w = whole[:H * H].view(torch.float8_e4m3fn).view(H, H)
    src, s = matrices(g, H, H)
    w.copy_(src)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    for T in (3, 100):  # without and with a workspace
        x = randn(g, T, H)
        want = p.run_device(x)
        q, sc = LB.fp8_quantize(x)
        n = T * H * 4
        over_w = whole[:n].view(torch.float32).view(T, H)
        with pytest.raises(LB.LlambdaCudaError, match="overlaps the session's weights"):
            p.run_device(x, out=over_w)
        with pytest.raises(LB.LlambdaCudaError, match="overlaps the session's weights"):
            p.run_quantized(q, sc, T, out=over_w)
        assert torch.equal(w.view(torch.uint8), src.view(torch.uint8))
        # next to the weights
        out = whole[H * H:H * H + n].view(torch.float32).view(T, H)
        assert torch.equal(p.run_device(x, out=out), want)
    # a session whose scales lie in a buffer
    tail = torch.ones(1 + T * H, device="cuda")
    p2 = LB.Fp8ProjectionSession.from_device(src[:128, :128].contiguous(), tail[:1].view(1, 1))
    with pytest.raises(LB.LlambdaCudaError, match="overlaps the session's scales"):
        p2.run_device(x[:, :128], out=tail[:T * 128].view(T, 128))
    # workspaces, through the C call
    L, T = N.lib(), 100
    need = L.llambda_cuda_fp8_session_workspace(p._h, T)
    assert need
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    room = torch.zeros(need + T * H * 4 + 256, dtype=torch.uint8, device="cuda")
    out = torch.empty(T, H, device="cuda")

    def call(px, po, pw):
        return L.llambda_cuda_fp8_session_run_device(p._h, 0, px, H, T, 0, po, H, pw, need, None)

    last = room.data_ptr() + (need - 1) // 256 * 256
    refused(call(room.data_ptr(), out.data_ptr(), room.data_ptr()), "workspace overlaps the input")
    refused(call(last, out.data_ptr(), room.data_ptr()), "workspace overlaps the input")
    refused(call(x.data_ptr(), last, room.data_ptr()), "workspace overlaps the output")
    refused(call(x.data_ptr(), out.data_ptr(), whole.data_ptr()), "workspace overlaps the session")
    assert call(x.data_ptr(), out.data_ptr(), work.data_ptr()) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("T", [1, 70])
def test_experts_refuse_outputs_and_workspaces_that_overlap(T):
    g = gen(4)
    E, k, H, I = 4, 2, 128, 256
    up, down, gate = matrices(g, E, I, H), matrices(g, E, H, I), matrices(g, E, I, H)
    m = LB.Fp8MoeSession.from_device(up=up, down=down, gate=gate)
    x, wt = randn(g, T, H), randn(g, T, k)
    sel = torch.randint(0, E, (T, k), generator=g, device="cuda").int()
    want = m.run_device(x, sel, wt)
    for name in ("up", "down", "gate"):
        t = dict(up=up, down=down, gate=gate)[name]
        out = t[0].view(torch.uint8).flatten()[:T * H * 4].view(torch.float32).view(T, H)
        with pytest.raises(LB.LlambdaCudaError, match="overlaps the session's weights"):
            m.run_device(x, sel, wt, out=out)
    L = N.lib()
    need = L.llambda_cuda_fp8_moe_session_workspace(m._h, T, k)
    room = torch.zeros(need + T * H * 4 + 256, dtype=torch.uint8, device="cuda")
    out = torch.empty(T, H, device="cuda")
    names = ("input", "selection", "weights", "output")
    ptrs = [x.data_ptr(), sel.data_ptr(), wt.data_ptr(), out.data_ptr()]

    def call(a, work=room.data_ptr()):
        return L.llambda_cuda_fp8_moe_session_run_device(m._h, 0, a[0], H, T, k, a[1], a[2], 0, a[3],
                                                         H, work, need, None)

    for i, name in enumerate(names):
        for at in (room.data_ptr(), room.data_ptr() + (need - 1) // 256 * 256):
            refused(call(ptrs[:i] + [at] + ptrs[i + 1:]), "workspace overlaps the " + name)
    assert call(ptrs) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_inputs_dropped_after_a_call_on_another_stream_keep_their_memory():
    """The caller's allocator gives an input's memory out again only when the call's stream is
    done with it."""
    g = gen(5)
    E, k, H = 8, 2, 1024
    up, down = matrices(g, E, 256, H), matrices(g, E, H, 256)
    m = LB.Fp8MoeSession.from_device(up=up, down=down)
    p = LB.Fp8ProjectionSession.from_device(*matrices(g, 256, H))
    T = 300
    x = randn(g, T, H)
    q, sc = LB.fp8_quantize(x)
    sel = torch.randint(0, E, (T, k), generator=g, device="cuda").int()
    wt, logits, bias = randn(g, T, k), randn(g, T, 600), randn(g, 600)
    side = torch.cuda.Stream()

    def busy(call, want, *inputs):
        copies = [t.clone() for t in inputs]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)  # about a tenth of a second
        got = call(*copies)
        places = {t.data_ptr() for t in copies}
        del copies
        again = [torch.empty_like(t) for t in inputs]  # (nothing is written to them)
        assert not side.query(), "the side stream was done too soon to show anything"
        assert not places & {t.data_ptr() for t in again}
        torch.cuda.synchronize()
        for a, b in zip(got if isinstance(got, tuple) else (got,),
                        want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))

    busy(lambda a: p.run_device(a, stream=side), p.run_device(x), x)
    busy(lambda a, b: p.run_quantized(a, b, T, stream=side), p.run_quantized(q, sc, T), q, sc)
    busy(lambda a: LB.fp8_quantize(a, stream=side), (q, sc), x)
    busy(lambda a, b, c: m.run_device(a, b, c, stream=side), m.run_device(x, sel, wt), x, sel, wt)
    busy(lambda a, b: LB.route_experts(a, k, bias=b, stream=side),
         LB.route_experts(logits, k, bias=bias), logits, bias)


def test_a_session_waits_for_scales_that_another_stream_writes():
    g = gen(6)
    w, s = matrices(g, 64, 64)
    up, down = matrices(g, 2, 64, 64), matrices(g, 2, 64, 64)
    side = torch.cuda.Stream()

    def late(t):
        """t's values, not finite until the side stream has written them."""
        to = torch.full_like(t, float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)
            to.copy_(t)
        return to

    x = randn(g, 3, 64)
    want = LB.Fp8ProjectionSession.from_device(w, s).run_device(x)
    assert torch.equal(LB.Fp8ProjectionSession.from_device(w, late(s)).run_device(x), want)
    sel, wt = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), randn(g, 3, 1)
    want = LB.Fp8MoeSession.from_device(up=up, down=down).run_device(x, sel, wt)
    got = LB.Fp8MoeSession.from_device(up=up, down=(down[0], late(down[1])))
    assert torch.equal(got.run_device(x, sel, wt), want)


def test_tangents_of_forward_mode_are_refused():
    import torch.autograd.forward_ad as fwd
    g = gen(7)
    w, s = matrices(g, 64, 64)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    m = LB.Fp8MoeSession.from_device(up=matrices(g, 2, 64, 64), down=matrices(g, 2, 64, 64))
    x, sel, wt = randn(g, 3, 64), torch.zeros(3, 1, dtype=torch.int32, device="cuda"), randn(g, 3, 1)
    want = p.run_device(x), m.run_device(x, sel, wt)
    with fwd.dual_level():
        d, dw = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(wt, torch.ones_like(wt))
        for call in (lambda: LB.route_experts(d, 2), lambda: LB.fp8_quantize(d),
                     lambda: p.run_device(d), lambda: m.run_device(d, sel, wt),
                     lambda: m.run_device(x, sel, dw),
                     lambda: LB.route_experts(x, 2, bias=fwd.make_dual(x[0], x[1]))):
            with pytest.raises(ValueError, match="tangent"):
                call()
        # without one
        assert torch.equal(p.run_device(x), want[0])
        assert torch.equal(m.run_device(x, sel, wt), want[1])
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(p.run_device, (x,), (torch.ones_like(x),))
    assert torch.equal(p.run_device(x), want[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,at", [(5000 + 9, 4), (5003, 3), (5008, 8), (5002, 2), (5004, 1),
                                      (5001, 0), (5000, 0)])
def test_a_prompt_into_rows_of_any_stride_and_alignment(dtype, width, at):
    """Pairs of CTAs store rows by bulk copies where they start on 16 bytes, by words or values
    elsewhere; nothing beside them changes."""
    g = gen(width + at)
    T, N, K = 601, 5000, 272
    w, s = matrices(g, N, K)
    p = LB.Fp8ProjectionSession.from_device(w, s)
    x = randn(g, T, K).to(dtype)
    big = torch.full((T + 3, width), 7.0, dtype=dtype, device="cuda")
    view = big[2:2 + T, at:at + N]
    p.run_device(x, out=view)
    check(view, *product_reference(*quantize_reference(x), w, s))
    assert torch.equal(view, p.run_device(x))
    view.fill_(7.0)
    assert bool((big == 7.0).all())


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 8, 4096, 1536), (1, 16, 2, 7168, 256), (3, 8, 3, 4096, 1536),
                                       (40, 8, 2, 7168, 2048), (300, 4, 2, 4096, 1536)])
def test_experts_of_wide_layers(T, E, k, H, I, gated):
    g = gen(H + I + T)
    up, down, gate = matrices(g, E, I, H), matrices(g, E, H, I), matrices(g, E, I, H)
    x, wt = randn(g, T, H), randn(g, T, k)
    sel = torch.rand(T, E, generator=g, device="cuda").topk(k, dim=1).indices.int()
    m = LB.Fp8MoeSession.from_device(up=up, down=down, gate=gate if gated else None)
    out = m.run_device(x, sel, wt)
    assert torch.equal(m.run_device(x, sel, wt), out) and m.status() == 0
    q, sx = quantize_reference(x)
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(want)
    for e in range(E):  # an expert's entries together
        t, j = torch.nonzero(sel == e, as_tuple=True)
        if not t.numel():
            continue
        u, du = product_reference(q[t], sx[t], up[0][e], up[1][e])
        if gated:
            v, dv = product_reference(q[t], sx[t], gate[0][e], gate[1][e])
            a = v * torch.sigmoid(v)  # |silu'| <= 1.1; its own error 8 half steps
            h, dh = a * u, (1.1 * dv + 8 * U32 * a.abs()) * (u.abs() + du) + a.abs() * du
        else:
            h, dh = torch.relu(u) ** 2, 2.0 * torch.relu(u) * du + du * du
        p, dp = blocks_of(h), blocks_of(dh + 8 * U32 * h.abs())
        s = (p.abs().amax(2) / 448).clamp(min=2.0 ** -126)
        ds = dp.amax(2) / 448 / s + 2 * U32
        v = p / s[:, :, None]
        dv = dp / s[:, :, None] + v.abs() * (ds[:, :, None] + 2 * U32)
        # a quotient within its error of a border of e4m3 may go to the other neighbour
        hq, (lo, _), (hi, _) = e4m3(v)[0], e4m3(v - dv), e4m3(v + dv)
        slack = torch.maximum((hq - lo).abs(), (hi - hq).abs()) + hq.abs() * ds[:, :, None]
        y, dy = product_reference(hq, s, down[0][e], down[1][e])
        mag, _ = product_reference(slack, s, down[0][e].float().abs(), down[1][e].abs())
        w = wt[t, j][:, None].double()
        want.index_add_(0, t, w * y)
        bound.index_add_(0, t, w.abs() * (dy + mag + 4 * U32 * y.abs()))
    check(out, want, bound * (1 + k * U32))


def test_a_captured_call_on_a_forked_stream():
    """stream= inside a capture: inputs made and dropped in it, replayed on new values."""
    g = gen(8)
    E, k, H = 8, 2, 256
    m = LB.Fp8MoeSession.from_device(up=matrices(g, E, 128, H), down=matrices(g, E, H, 128))
    p = LB.Fp8ProjectionSession.from_device(*matrices(g, H, H))
    bias = 0.1 * randn(g, E)
    router = randn(g, H, E) / 16

    def run(x, side):
        here = torch.cuda.current_stream()
        h = p.run_device(x)
        logits, h2 = h @ router, h + 1.0
        side.wait_stream(here)
        sel, wt = LB.route_experts(logits, k, score="sigmoid", bias=bias, stream=side)
        del logits
        out = m.run_device(h, sel, wt, stream=side)
        del h
        q, s = LB.fp8_quantize(h2, stream=side)
        del h2
        junk = torch.full((4 * T, H), 9.0, device="cuda")  # beside them, in memory that is free
        here.wait_stream(side)
        del junk
        return sel, wt, out, q, s

    for T in (3, 130):
        x = randn(g, T, H)
        side = torch.cuda.Stream()
        run(x, side)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = run(x, side)
        for _ in range(3):
            new = randn(g, T, H)
            x.copy_(new)
            gr.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in res]
            want = run(new, side)
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
