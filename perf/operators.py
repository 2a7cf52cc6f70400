"""What the routed-expert operators are measured on: routing, 8-bit quantisation, the
block-scaled 8-bit product and the routed experts' feed-forward, each in a plain form
(`own` false: elementary torch operations) and through the framework (`own` true)."""
import math

import torch

own = False

BF16, F32 = "bf16", "f32"
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # one token of a decode step, 128 experts with sigmoid scores and a balance bias
        dict(name="route_step", op="route", T=1, E=128, k=6, score="sigmoid", bias=True, groups=1,
             top_groups=1, group_top=1, scale=1.0, type=F32),
        # a prefill batch over 512 experts, softmax scores
        dict(name="route_batch", op="route", T=2048, E=512, k=10, score="softmax", bias=False,
             groups=1, top_groups=1, group_top=1, scale=1.0, type=F32),
        # a long prompt, experts in groups, 16-bit logits
        dict(name="route_groups", op="route", T=8191, E=256, k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, group_top=2, scale=2.5, type=BF16),
        # a decode batch's activations, and a long prompt's
        dict(name="quantize_decode", op="quantize", T=64, K=2688, type=F32),
        dict(name="quantize_prompt", op="quantize", T=8192, K=4096, type=BF16),
        # one token through a feed-forward projection; a ragged small batch whose last blocks are
        # partial; a batch through a very tall matrix; a prompt
        dict(name="project_step", op="project", T=1, N=14336, K=4096, type=BF16),
        dict(name="project_ragged", op="project", T=33, N=2688, K=1856, type=F32),
        dict(name="project_tall", op="project", T=256, N=65536, K=2688, type=BF16),
        dict(name="project_prompt", op="project", T=2048, N=14336, K=4096, type=BF16),
        # one token through a layer of 512 small experts; a decode batch through 128 larger ones
        # without gate (the last 128-block of 1856 is half full); a prompt
        dict(name="experts_step", op="experts", T=1, E=512, k=10, H=2048, I=512, gate=True,
             skipped=0.0, type=BF16),
        dict(name="experts_decode", op="experts", T=32, E=128, k=6, H=2688, I=1856, gate=False,
             skipped=0.0, type=F32),
        dict(name="experts_prompt", op="experts", T=2048, E=512, k=10, H=2048, I=512, gate=True,
             skipped=0.0, type=BF16),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    op = rng.choice(["route", "quantize", "project", "experts"])
    typ = rng.choice([BF16, F32])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        size = _log(rng, 2, 512 // groups)
        E = groups * size
        top_groups = rng.randint(1, groups)
        return dict(op=op, T=_log(rng, 1, 8192), E=E, k=rng.randint(1, min(16, top_groups * size)),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    groups=groups, top_groups=top_groups, group_top=rng.choice([1, 2]),
                    scale=rng.choice([1.0, 2.5]), type=typ)
    if op == "quantize":
        return dict(op=op, T=_log(rng, 1, 8192), K=_log(rng, 16, 4096), type=typ)
    if op == "project":
        while True:
            T, N, K = _log(rng, 1, 4096), _log(rng, 64, 65536), _log(rng, 16, 8192, 16)
            if T * N * K <= 2048 * 14336 * 4096 and N * K <= 65536 * 2688 and T * N <= 1 << 25:
                return dict(op=op, T=T, N=N, K=K, type=typ)
    while True:
        E, H, I = _log(rng, 2, 512), _log(rng, 64, 4096, 16), _log(rng, 32, 2048, 16)
        T, k = _log(rng, 1, 2048), rng.randint(1, min(10, E))
        if E * H * I <= 512 * 2048 * 512 and T * k * H * I <= 2048 * 10 * 2048 * 512:
            return dict(op=op, T=T, E=E, k=k, H=H, I=I, gate=rng.random() < 0.5,
                        skipped=rng.choice([0.0, 0.25]), type=typ)


def _dtype(case):
    return torch.bfloat16 if case["type"] == BF16 else torch.float32


def _blocks(n):
    return (n + 127) // 128


def _weights(g, E, N, K):
    """E matrices [N][K] in e4m3 and their block scales, values about N(0, 1/sqrt(K))."""
    w = torch.empty(E, N, K, dtype=E4M3, device="cuda")
    step = max(1, (1 << 28) // (N * K))
    for e in range(0, E, step):
        v = torch.randn(min(step, E - e), N, K, generator=g, device="cuda")
        w[e:e + step] = v.mul_(64.0).clamp_(-448.0, 448.0).to(E4M3)
    s = torch.rand(E, _blocks(N), _blocks(K), generator=g, device="cuda")
    return w, (s + 0.5) * (1.0 / (64.0 * math.sqrt(K)))


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, op, dt = case["T"], case["op"], _dtype(case)
    if op == "route":
        st = {"logits": (1.5 * torch.randn(T, case["E"], generator=g, device="cuda")).to(dt)}
        b = 0.05 * torch.randn(case["E"], generator=g, device="cuda")
        st["bias"] = b if case["bias"] else None
        return st
    K = case["H"] if op == "experts" else case["K"]
    # activations of a residual stream: normal, with a few columns that are much larger
    x = torch.randn(T, K, generator=g, device="cuda")
    x *= 1.0 + 15.0 * (torch.rand(K, generator=g, device="cuda") > 0.99)
    st = {"x": x.to(dt)}
    if op == "project":
        st["w"], st["s"] = (t[0] for t in _weights(g, 1, case["N"], K))
    if op == "experts":
        E, I, k = case["E"], case["I"], case["k"]
        if case["gate"]:
            st["gate"] = _weights(g, E, I, K)
        st["up"], st["down"] = _weights(g, E, I, K), _weights(g, E, K, I)
        st["sel"] = torch.rand(T, E, generator=g, device="cuda").topk(k, dim=1).indices.int()
        wt = torch.rand(T, k, generator=g, device="cuda") + 0.1
        st["wt"] = wt / wt.sum(1, keepdim=True)
        # entries that belong to no expert of this process
        st["sel"][torch.rand(T, k, generator=g, device="cuda") < case["skipped"]] = -1
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if own:  # the session over the weights, which a program keeps as long as its weights
        import llambda_b200 as LB
        if case["op"] == "project":
            st["session"] = LB.Fp8ProjectionSession.from_device(st["w"], st["s"])
        if case["op"] == "experts":
            st["session"] = LB.Fp8MoeSession.from_device(up=st["up"], down=st["down"],
                                                         gate=st.get("gate"))
    return st


def run(state):
    case = state["case"]
    if own:
        import llambda_b200 as LB
        if case["op"] == "route":
            return LB.route_experts(state["logits"], case["k"], score=case["score"],
                                    bias=state["bias"], groups=case["groups"],
                                    top_groups=case["top_groups"], group_top=case["group_top"],
                                    weight_scale=case["scale"])
        if case["op"] == "quantize":
            q, s = LB.fp8_quantize(state["x"])
            return q[:, :case["K"]], s[:, :case["T"]]
        if case["op"] == "project":
            return state["session"].run_device(state["x"])
        return state["session"].run_device(state["x"], state["sel"], state["wt"],
                                           out_dtype=torch.bfloat16)
    if case["op"] == "route":
        return _route(state, case)
    if case["op"] == "quantize":
        q, s = _quantize(state["x"].float())
        return q.to(E4M3), s.t().contiguous()
    if case["op"] == "project":
        y = _dequantized(state["x"].float()) @ _matrices(state["w"], state["s"]).t()
        return y.to(state["x"].dtype)
    return _experts(state, case)


# ------------------------------------------------------------------ plain forms


def _route(st, case):
    """64 bits: two experts' scores may lie closer than 32 bits tell apart."""
    l = st["logits"].double()
    T, E, G = l.shape[0], l.shape[1], case["groups"]
    if case["score"] == "softmax":
        p = torch.exp(l - l.amax(1, keepdim=True))
        s = p / p.sum(1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-l))
    c = s if st["bias"] is None else s + st["bias"].double()
    if case["top_groups"] < G:
        cg = c.view(T, G, E // G)
        gs = cg.sort(dim=2, descending=True).values[:, :, :case["group_top"]].sum(2)
        best = gs.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=l.device).scatter_(1, best, True)
        c = torch.where(keep[:, :, None], cg, -math.inf).reshape(T, E)
    sel = c.sort(dim=1, descending=True, stable=True).indices[:, :case["k"]]
    w = s.gather(1, sel)
    w = w / w.sum(1, keepdim=True) * case["scale"]
    return sel.int(), w.float()


def _quantize(x):
    """(e4m3 values as floats, scales) of the rows of x, in blocks of 128 columns."""
    T, K = x.shape
    KB = _blocks(K)
    p = torch.nn.functional.pad(x, (0, KB * 128 - K)).view(T, KB, 128)
    top = p.abs().amax(2)
    # a tensor by a tensor: by a number it would be a product with the rounded reciprocal
    s = (top / torch.full_like(top, 448.0)).clamp(min=2.0 ** -126)
    q = (p / s[:, :, None]).to(E4M3).float()
    return q.view(T, KB * 128)[:, :K], s


def _dequantized(x):
    q, s = _quantize(x)
    return q * s.repeat_interleave(128, 1)[:, :x.shape[1]]


def _matrices(w, s):
    N, K = w.shape[-2:]
    return w.float() * s.repeat_interleave(128, -2)[..., :N, :].repeat_interleave(128, -1)[..., :K]


def _experts(st, case):
    """Entries grouped by expert, every group padded to the longest, one batched product."""
    T, k, E = case["T"], case["k"], case["E"]
    sel = st["sel"].long().view(-1)
    ids, slot, counts = torch.unique(torch.where(sel < 0, E, sel), return_inverse=True,
                                     return_counts=True)
    order = slot.argsort(stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device=sel.device) - (counts.cumsum(0) - counts)[slot[order]]
    live = ids.clamp(max=E - 1)  # the group of the skipped entries takes part and is not used
    x = _dequantized(st["x"].float())
    xg = torch.zeros(ids.numel(), int(counts.max()), x.shape[1], device=x.device)
    xg[slot, place] = x.repeat_interleave(k, 0)
    u = xg @ _matrices(st["up"][0][live], st["up"][1][live]).transpose(1, 2)
    if case["gate"]:
        v = xg @ _matrices(st["gate"][0][live], st["gate"][1][live]).transpose(1, 2)
        h = v / (1.0 + torch.exp(-v)) * u
    else:
        h = u.clamp(min=0.0) ** 2
    h = _dequantized(h.view(-1, h.shape[2])).view(h.shape)
    y = h @ _matrices(st["down"][0][live], st["down"][1][live]).transpose(1, 2)
    wt = torch.where(st["sel"] < 0, 0.0, st["wt"])
    out = (y[slot, place].view(T, k, -1) * wt[:, :, None]).sum(1)
    return out.to(torch.bfloat16)


# ------------------------------------------------------------------ work and exact values


def work(case):
    T, op, xb = case["T"], case["op"], 2 if case["type"] == BF16 else 4
    if op == "route":
        E, k = case["E"], case["k"]
        return {"bytes": T * (E * xb + 8 * k) + (4 * E if case["bias"] else 0), "flops": 4 * T * E}
    if op == "quantize":
        K = case["K"]
        return {"bytes": T * (K * (xb + 1) + 4 * _blocks(K)), "flops": 2 * T * K}
    if op == "project":
        N, K = case["N"], case["K"]
        return {"bytes": N * K + 4 * _blocks(N) * _blocks(K) + T * (K + N) * xb,
                "flops": 2 * T * N * K}
    E, k, H, I = case["E"], case["k"], case["H"], case["I"]
    mats = 3 if case["gate"] else 2
    live = T * k * (1.0 - case["skipped"])
    active = E * (1.0 - (1.0 - 1.0 / E) ** live)  # distinct experts expected
    return {"bytes": int(active * mats * (H * I + 4 * _blocks(H) * _blocks(I))
                         + T * (H * xb + H * 2 + 8 * k)),
            "flops": int(2 * live * mats * H * I)}


def _exact_rows(x):
    """Rows quantised by the definition: the scale and the quotient are 32-bit numbers, each
    rounded once from its exact value; the result in 64 bits."""
    T, K = x.shape
    KB = _blocks(K)
    p = torch.zeros(T, KB * 128, dtype=torch.float64, device=x.device)
    p[:, :K] = x
    p = p.view(T, KB, 128)
    s = torch.maximum((p.abs().amax(2) / 448.0).float().double(),
                      torch.tensor(2.0 ** -126, dtype=torch.float64, device=x.device))
    v = (p / s[:, :, None]).float().double()
    a = v.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(a)) - 3.0)  # e4m3: three bits after the leading one
    q = torch.round(v / step) * step
    return q, s


def _exact_product(x, w, s):
    """x [T][K] quantised, times one matrix, block column by block column."""
    q, sx = _exact_rows(x)
    N, K = w.shape
    y = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    for b in range(_blocks(K)):
        wb = w[:, 128 * b:128 * b + 128].double()
        part = q[:, b, :wb.shape[1]] @ wb.t()
        y += part * sx[:, b:b + 1] * s[:, b].double().repeat_interleave(128)[:N]
    return y


def exact(case, seed):
    st, op = _inputs(case, seed), case["op"]
    if op == "route":
        l = st["logits"].double().cpu().numpy()
        import numpy as np
        s = (1.0 / (1.0 + np.exp(-l)) if case["score"] == "sigmoid"
             else np.exp(l) / np.exp(l).sum(1, keepdims=True))
        c = s + (st["bias"].double().cpu().numpy() if st["bias"] is not None else 0.0)
        G = case["groups"]
        if case["top_groups"] < G:
            size = case["E"] // G
            best = -np.sort(-c.reshape(-1, G, size), axis=2)[:, :, :case["group_top"]].sum(2)
            out = np.argsort(-best, axis=1, kind="stable")[:, case["top_groups"]:]
            for t in range(c.shape[0]):
                for gi in out[t]:
                    c[t, gi * size:(gi + 1) * size] = -np.inf
        sel = np.argsort(-c, axis=1, kind="stable")[:, :case["k"]]
        w = np.take_along_axis(s, sel, 1)
        w = w / w.sum(1, keepdims=True) * case["scale"]
        return torch.from_numpy(sel.astype(np.int32)), torch.from_numpy(w)
    if op == "quantize":
        q, s = _exact_rows(st["x"].double())
        return q.flatten(1)[:, :case["K"]], s.t().contiguous()
    if op == "project":
        return _exact_product(st["x"].double(), st["w"], st["s"])
    x, sel, wt = st["x"].double(), st["sel"].cpu(), st["wt"].double()
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
    for e in sorted(set(sel.flatten().tolist()) - {-1}):
        t, j = (v.cuda() for v in torch.nonzero(sel == e, as_tuple=True))
        u = _exact_product(x[t], st["up"][0][e], st["up"][1][e])
        if case["gate"]:
            g = _exact_product(x[t], st["gate"][0][e], st["gate"][1][e])
            h = g * torch.sigmoid(g) * u
        else:
            h = torch.relu(u) ** 2
        y = _exact_product(h, st["down"][0][e], st["down"][1][e])
        out.index_add_(0, t, y * wt[t, j][:, None])
    return out
