"""Timing cases of the operators around a routed FP8 expert layer (``wanferenz_b200.ops``).

One transformer layer's way from the residual stream through its experts and back: the residual's addition with the
RMS norm and its E4M3 output (``rms_norm_quant``), routing with groups (``route_topk``), the router's choice turned
into rows sorted by expert (``expert_dispatch``), the experts' block-scaled FP8 product (``grouped_fp8_gemm``) and the
way back to token order (``expert_combine``).  Each has a plain form in elementary torch operations and an ``exact``
form in 64 bits.
"""

import math

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a decode step: latency alone
        dict(name="norm_1x4096", op="norm", T=1, D=4096, residual=True, norm_out=True, e8m0=True),
        # a short prompt's rows before an attention projection: no residual yet, float32 scales, no bf16 output wanted
        dict(name="norm_509x2048", op="norm", T=509, D=2048, residual=False, norm_out=False, e8m0=False),
        # a batch of prompts between two layers
        dict(name="norm_16384x4096", op="norm", T=16384, D=4096, residual=True, norm_out=True, e8m0=True),
        # a decode batch, sigmoid scores with a balance bias
        dict(name="route_16x256", op="route", T=16, E=256, k=6, score="sigmoid", bias=True, groups=1, keep=1, half=False),
        # a prompt batch, experts in 8 groups of which 4 stay
        dict(name="route_8191x256_g8", op="route", T=8191, E=256, k=8, score="sigmoid", bias=True, groups=8, keep=4,
             half=False),
        # speculative verification: 16 sequences x 4 draft tokens
        dict(name="dispatch_64x6", op="dispatch", T=64, k=6, E=256, skew=0.5),
        # a batch of prompts
        dict(name="dispatch_16384x8", op="dispatch", T=16384, k=8, E=256, skew=0.5),
        # a decode batch of 16 tokens through 64 experts: a few rows each, the weights' bytes count
        dict(name="gemm_16x6_2048x2048", op="gemm", T=16, k=6, E=64, N=2048, K=2048, e8m0=True, gather=True, skew=0.3),
        # the down projection of a 256-token chunk, float32 scales, rows already in expert order
        dict(name="gemm_256x6_2048x1024", op="gemm", T=256, k=6, E=64, N=2048, K=1024, e8m0=False, gather=False, skew=0.3),
        # a prompt batch through one rank's 32 experts of 256: tensor cores count
        dict(name="gemm_2731x6_4096x4096", op="gemm", T=2731, k=6, E=32, N=4096, K=4096, e8m0=True, gather=True, skew=0.3),
        # a decode batch back to token order, with the shared expert's rows
        dict(name="combine_16x6", op="combine", T=16, k=6, D=4096, E=256, weighted=True, shared=True, skew=0.5),
        # a batch of prompts
        dict(name="combine_8192x8", op="combine", T=8192, k=8, D=4096, E=256, weighted=True, shared=True, skew=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "route", "dispatch", "gemm", "gemm", "combine"])
    if op == "norm":
        D = BLOCK * rng.randint(4, 64)
        return dict(op=op, T=min(_log(rng, 1, 16384), 16384 * 4096 // D), D=D, residual=rng.random() < 0.6,
                    norm_out=rng.random() < 0.6, e8m0=rng.random() < 0.5)
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        E = groups * rng.randint(max(2, 16 // groups), 256 // groups)
        keep = rng.randint(max(1, groups // 2), groups)
        return dict(op=op, T=_log(rng, 1, 8191), E=E, k=rng.randint(1, min(8, keep * (E // groups))),
                    score=rng.choice(["sigmoid", "softmax", "sqrtsoftplus"]), bias=rng.random() < 0.6, groups=groups,
                    keep=keep, half=rng.random() < 0.3)
    if op == "dispatch":
        return dict(op=op, T=_log(rng, 1, 16384), k=rng.randint(1, 8), E=_log(rng, 8, 256), skew=rng.uniform(0, 1))
    if op == "combine":
        return dict(op=op, T=_log(rng, 1, 8192), k=rng.randint(1, 8), D=8 * rng.randint(64, 512), E=_log(rng, 8, 256),
                    weighted=rng.random() < 0.7, shared=rng.random() < 0.6, skew=rng.uniform(0, 1))
    # weights of at most 32 x 4096 x 4096, products of at most the largest listed case's
    N, K = 8 * rng.randint(64, 512), BLOCK * rng.randint(4, 32)
    E, k = _log(rng, 8, 32), rng.randint(1, 6)
    return dict(op=op, T=_log(rng, 1, 2731), k=k, E=E, N=N, K=K, e8m0=rng.random() < 0.5, gather=rng.random() < 0.6,
                skew=rng.uniform(0, 0.4))


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _choices(gen, T, k, E, skew):
    """``[T, k]`` distinct experts of each token, expert popularity falling as ``rank^-skew``."""
    pop = -skew * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    pop = pop[torch.randperm(E, generator=gen, device="cuda")]
    u = torch.rand(T, E, generator=gen, device="cuda").clamp_(1e-7, 1 - 1e-7)
    return (pop - torch.log(-torch.log(u))).topk(min(k, E), dim=-1).indices


def _sorted_rows(indices, E):
    """Offsets, token of each sorted row and sorted row of each pair, rows ordered by (expert, token, slot)."""
    k = indices.size(1)
    flat = indices.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum((flat[:, None] == torch.arange(E, device="cuda")).sum(0), 0)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device="cuda")
    return offsets, (order // k).int(), slots.view_as(indices).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    op, T = case["op"], case["T"]
    st = dict(case=case)
    if op == "norm":
        D = case["D"]
        # rows of different energy, a few channels that stand out
        chan = torch.where(uniform(D) < 0.01, 8.0, 1.0)
        st["x"] = (normal(T, D) * chan * (0.25 + uniform(T, 1))).bfloat16()
        st["residual"] = (normal(T, D) * 3 * chan).bfloat16() if case["residual"] else None
        st["weight"] = 0.5 + uniform(D)
    elif op == "route":
        E = case["E"]
        st["logits"] = normal(T, E) * 1.28
        if case["half"]:
            st["logits"] = st["logits"].bfloat16()
        st["bias"] = normal(E) * 0.01 if case["bias"] else None
    elif op == "dispatch":
        st["indices"] = _choices(gen, T, case["k"], case["E"], case["skew"])
    elif op == "combine":
        idx = _choices(gen, T, case["k"], case["E"], case["skew"])
        st["slots"] = _sorted_rows(idx, case["E"])[2]
        st["rows"] = normal(idx.numel(), case["D"]).bfloat16()
        w = uniform(*idx.shape) + 0.05
        st["weights"] = w / w.sum(-1, keepdim=True) * 1.5 if case["weighted"] else None
        st["shared"] = normal(T, case["D"]).bfloat16() if case["shared"] else None
    else:
        E, N, K = case["E"], case["N"], case["K"]
        st["offsets"], tokens, _ = _sorted_rows(_choices(gen, T, case["k"], E, case["skew"]), E)
        counts = st["offsets"][1:] - st["offsets"][:-1]
        st["most"] = int(counts.max())  # of the plain form's padded batch
        st["rows"] = tokens if case["gather"] else None
        M = T if case["gather"] else tokens.numel()
        a = normal(M, K // BLOCK, BLOCK)
        amax = a.abs().amax(-1, keepdim=True)
        nb = -(-N // BLOCK)
        if case["e8m0"]:
            a_s = torch.exp2(torch.ceil(torch.log2(amax / FP8_MAX)))
            w_s = torch.exp2(torch.randint(-14, -11, (E, nb, K // BLOCK), generator=gen, device="cuda").float())
        else:
            a_s = amax / FP8_MAX
            w_s = (0.5 + uniform(E, nb, K // BLOCK)) * 2e-4
        kind = torch.float8_e8m0fnu if case["e8m0"] else torch.float32
        st["a"] = (a / a_s).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(M, K)
        st["a_s"], st["w_s"] = a_s[..., 0].to(kind).contiguous(), w_s.to(kind)
        st["w"] = torch.empty(E, N, K, dtype=torch.float8_e4m3fn, device="cuda")
        for e in range(E):
            st["w"][e] = (normal(N, K) * 100).clamp(-FP8_MAX, FP8_MAX)
    return st


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if own:
        if c["op"] == "route":  # names the group score: the operator's default without a bias is the largest
            return _own_route_top2(c, st)
        return _OWN[c["op"]](c, st)
    return _PLAIN[c["op"]](c, st)


def _own_norm(c, st):
    from wanferenz_b200 import ops

    r = ops.rms_norm_quant(st["x"], st["weight"], 1e-6, residual=st["residual"], norm_out=c["norm_out"],
                           scale_fmt="ue8m0" if c["e8m0"] else None,
                           scale_dtype=torch.float8_e8m0fnu if c["e8m0"] else torch.float32)
    return dict(q=r.q, s=r.s, y=r.y, h=r.h)


def _own_route(c, st):
    from wanferenz_b200 import ops

    return ops.route_topk(st["logits"], c["k"], bias=st["bias"], score_func=c["score"], n_groups=c["groups"],
                          topk_groups=c["keep"], route_scale=1.5)


def _own_route_top2(c, st):
    from wanferenz_b200 import ops

    return ops.route_topk(st["logits"], c["k"], bias=st["bias"], score_func=c["score"], n_groups=c["groups"],
                          topk_groups=c["keep"], group_score="top2", route_scale=1.5)


def _own_dispatch(c, st):
    from wanferenz_b200 import ops

    return ops.expert_dispatch(st["indices"], c["E"])


def _own_gemm(c, st):
    from wanferenz_b200 import ops

    return ops.grouped_fp8_gemm(st["a"], st["a_s"], st["w"], st["w_s"], st["offsets"], rows=st["rows"])


def _own_combine(c, st):
    from wanferenz_b200 import ops

    return ops.expert_combine(st["rows"], st["slots"], weights=st["weights"], shared=st["shared"])


_OWN = dict(norm=_own_norm, route=_own_route, dispatch=_own_dispatch, gemm=_own_gemm, combine=_own_combine)


def _plain_norm(c, st):
    x = st["x"].float()
    h = None
    if st["residual"] is not None:
        h = (x + st["residual"].float()).bfloat16()
        x = h.float()
    n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * st["weight"]
    b = n.view(c["T"], -1, BLOCK)
    s = b.abs().amax(-1, keepdim=True).clamp(min=1e-4) * (1.0 / FP8_MAX)
    if c["e8m0"]:
        s = torch.exp2(torch.ceil(torch.log2(s)))
    q = (b / s).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view_as(x)
    s = s[..., 0].to(torch.float8_e8m0fnu) if c["e8m0"] else s[..., 0]
    return dict(q=q, s=s, y=n.bfloat16() if c["norm_out"] else None, h=h)


def _scores(logits, how):
    """In 64 bits: two experts whose scores lie within a 32-bit rounding of each other keep their order."""
    z = logits.double()
    if how == "softmax":
        e = torch.exp(z - z.amax(-1, keepdim=True))
        return e / e.sum(-1, keepdim=True)
    if how == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return torch.sqrt(torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs())))


def _plain_route(c, st):
    s = _scores(st["logits"], c["score"])
    sel = s if st["bias"] is None else s + st["bias"].double()
    T, E, G = c["T"], c["E"], c["groups"]
    if G > 1:
        g = torch.sort(sel.view(T, G, -1), dim=-1, descending=True).values[..., :2].sum(-1)
        rank = torch.sort(torch.sort(g, dim=-1, descending=True, stable=True).indices, dim=-1).indices
        sel = torch.where((rank < c["keep"])[..., None], sel.view(T, G, -1), -math.inf).view(T, E)
    idx = torch.sort(sel, dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    w = torch.gather(s, 1, idx)
    if c["score"] != "softmax":
        w = w / w.sum(-1, keepdim=True)
    return (w * 1.5).float(), idx


def _plain_dispatch(c, st):
    return _sorted_rows(st["indices"], c["E"])


def _plain_gemm(c, st):
    E, N, K = c["E"], c["N"], c["K"]
    off = st["offsets"].long()
    R = st["rows"].numel() if st["rows"] is not None else st["a"].size(0)
    a = (st["a"].float().view(-1, K // BLOCK, BLOCK) * st["a_s"].float()[..., None]).view(-1, K)
    if st["rows"] is not None:
        a = a[st["rows"].long()]
    w_s = st["w_s"].float().repeat_interleave(BLOCK, 1)[:, :N]
    w = (st["w"].float().view(E, N, -1, BLOCK) * w_s[..., None]).view(E, N, K)
    # every expert's rows padded to the longest list: one batched product
    at = (off[:-1, None] + torch.arange(st["most"], device="cuda")).clamp(max=R - 1)
    o = torch.bmm(a[at], w.transpose(1, 2)).bfloat16()
    r = torch.arange(R, device="cuda")
    e = (r[:, None] >= off[1:]).sum(-1)
    return o[e, r - off[e]]


def _plain_combine(c, st):
    # ascending slot is ascending expert; every slot of these cases is a row
    slots, order = torch.sort(st["slots"].long(), dim=-1)
    v = st["rows"][slots].float()
    if st["weights"] is not None:
        v = v * torch.gather(st["weights"], 1, order)[..., None]
    y = v.sum(1)
    if st["shared"] is not None:
        y = y + st["shared"].float()
    return y.bfloat16()


_PLAIN = dict(norm=_plain_norm, route=_plain_route, dispatch=_plain_dispatch, gemm=_plain_gemm, combine=_plain_combine)


# ---------------------------------------------------------------------------------------------------------------------
# bytes and operations of one pass
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    c, op, T = case, case["op"], case["T"]
    if op == "norm":
        D = c["D"]
        per = 2 + 1 + (4 if c["residual"] else 0) + (2 if c["norm_out"] else 0)
        return dict(bytes=T * D * per + T * (D // BLOCK) * (1 if c["e8m0"] else 4) + 4 * D, flops=8 * T * D)
    if op == "route":
        return dict(bytes=T * c["E"] * (2 if c["half"] else 4) + 12 * T * c["k"] + (4 * c["E"] if c["bias"] else 0),
                    flops=12 * T * c["E"])
    k = min(c["k"], c["E"])
    if op == "dispatch":
        return dict(bytes=16 * T * k + 4 * (c["E"] + 1), flops=0)
    if op == "combine":
        return dict(bytes=T * c["D"] * (2 * k + 2 + (2 if c["shared"] else 0)) + T * k * (8 if c["weighted"] else 4),
                    flops=2 * T * k * c["D"])
    E, N, K, R = c["E"], c["N"], c["K"], T * k
    sb = 1 if c["e8m0"] else 4
    touched = E * (1 - (1 - 1 / E) ** R)  # experts that any row goes to
    M = T if c["gather"] else R
    return dict(bytes=touched * N * (K + sb * K / BLOCK / BLOCK) + M * (K + sb * K / BLOCK) + 2 * R * N
                + (4 * R if c["gather"] else 0), flops=2 * R * N * K)


# ---------------------------------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return dict(norm=_exact_norm, route=_exact_route, dispatch=_exact_dispatch, gemm=_exact_gemm,
                combine=_exact_combine)[case["op"]](case, st)


def _exact_norm(c, st):
    v, h = st["x"].double(), None
    if st["residual"] is not None:
        h = (v + st["residual"].double()).float().bfloat16()  # the sum of two bf16 values, rounded to the stream's type
        v = h.double()
    n = v / torch.sqrt(v.pow(2).sum(-1, keepdim=True) / c["D"] + 1e-6) * st["weight"].double()
    top = n.view(c["T"], c["D"] // BLOCK, BLOCK).abs().max(-1).values.clamp(min=1e-4) / FP8_MAX
    s = torch.pow(2.0, torch.ceil(torch.log2(top))) if c["e8m0"] else top
    each = s.repeat_interleave(BLOCK, -1)
    q = (n / each).float().clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).double()
    return dict(q=q, s=s, y=n if c["norm_out"] else None, h=None if h is None else h.double())


def _exact_route(c, st):
    z, k, G = st["logits"].double(), c["k"], c["groups"]
    s = {"softmax": lambda: torch.softmax(z, -1), "sigmoid": lambda: torch.sigmoid(z),
         "sqrtsoftplus": lambda: torch.logaddexp(z, torch.zeros_like(z)).sqrt()}[c["score"]]()
    left = s.clone() if st["bias"] is None else s + st["bias"].double()
    if G > 1:
        m = left.view(c["T"], G, -1)
        best = m.topk(2, dim=-1).values.sum(-1)
        drop = torch.ones_like(best, dtype=torch.bool)
        for _ in range(c["keep"]):  # max() gives the lowest index of equal values here
            at = (best == best.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)
            drop.scatter_(1, at, False)
            best.scatter_(1, at, -math.inf)
        left = m.masked_fill(drop[..., None], -math.inf).reshape(c["T"], -1)
    picks = []
    for _ in range(k):
        at = (left == left.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)
        picks.append(at)
        left.scatter_(1, at, -math.inf)
    idx = torch.cat(picks, 1)
    w = s.gather(1, idx)
    if c["score"] != "softmax":
        w = w / w.sum(1, keepdim=True)
    return w * 1.5, None


def _exact_dispatch(c, st):
    return None


def _exact_gemm(c, st):
    E, N, K = c["E"], c["N"], c["K"]
    bounds = st["offsets"].tolist()
    R = bounds[-1]
    out = torch.empty(R, N, dtype=torch.float64, device="cuda")
    for e in range(E):
        lo, hi = bounds[e], bounds[e + 1]
        if lo == hi:
            continue
        at = st["rows"][lo:hi].long() if st["rows"] is not None else torch.arange(lo, hi, device="cuda")
        a = st["a"][at].float().double() * st["a_s"][at].float().double().repeat_interleave(BLOCK, 1)
        scale = st["w_s"][e].float().double().repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)
        out[lo:hi] = a @ (st["w"][e].float().double() * scale).T
    return out


def _exact_combine(c, st):
    y = torch.zeros(c["T"], c["D"], dtype=torch.float64, device="cuda")
    for j in range(st["slots"].size(1)):
        v = st["rows"][st["slots"][:, j].long()].double()
        y += v if st["weights"] is None else v * st["weights"][:, j:j + 1].double()
    return y if st["shared"] is None else y + st["shared"].double()
