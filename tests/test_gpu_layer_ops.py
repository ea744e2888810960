"""The operators around a routed expert layer against plain implementations in 64 bits.

Tolerances, derived before the first run.  A rounding is off by at most half a step relative to the value: fp32
2^-24, bf16 2^-8, e4m3 2^-4 (subnormals: 2^-10 absolute).  The norm's 32-bit value n carries the sum of squares (at
most 8 x 8 terms in a row and 8 + 5 tree levels: under 80 roundings, halved by the square root), the reciprocal square
root (2 ulp), and four products: N_REL = (80 / 2 + 8) x 2^-24 < 2^-18.  The scale adds two roundings to the largest n.
"""

import math
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

N_REL = 2.0 ** -18
BF16, E4M3, FP32 = 2.0 ** -8, 2.0 ** -4, 2.0 ** -24
E8 = torch.float8_e8m0fnu


def _ops():
    from wanferenz_b200 import ops
    return ops


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _within(got, want, rel, floor=0.0):
    err = (got.double() - want).abs()
    assert bool((err <= want.abs() * rel + floor).all()), float((err - want.abs() * rel - floor).max())


# ---- rms_norm_quant ---------------------------------------------------------------------------------------------
def _check_norm(x, weight, residual, r, ue8m0, eps=1e-6):
    h = x
    if residual is not None:
        h = (x.float() + residual.float()).bfloat16()
        assert torch.equal(r.h, h)
    else:
        assert r.h is None
    d = h.double()
    n = d / torch.sqrt(d.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    if r.y is not None:
        _within(r.y, n, BF16 + 2 * N_REL)
    blocks = n.unflatten(-1, (-1, 128))
    top = blocks.abs().amax(-1).clamp(min=1e-4) / 448
    s = r.s.float().double()
    if ue8m0:
        lo = torch.exp2(torch.ceil(torch.log2(top * (1 - 2 * N_REL))))
        hi = torch.exp2(torch.ceil(torch.log2(top * (1 + 2 * N_REL))))
        assert bool(((s == lo) | (s == hi)).all())
    else:
        _within(s, top, 2 * N_REL)
    v = (blocks / s[..., None])
    _within(r.q.float().unflatten(-1, (-1, 128)), v.clamp(-448, 448), E4M3 + 4 * N_REL, 2.0 ** -10)
    # the rounding is to nearest: where v is not within the error of a midpoint, q is the nearest e4m3 value
    near = v.float().clamp(-448, 448).to(torch.float8_e4m3fn).float().double()
    off = (r.q.float().unflatten(-1, (-1, 128)).double() != near)
    assert bool(((v - near).abs()[off] >= (near.abs()[off] * E4M3 / 2).clamp(max=2.0 ** -10) * (1 - 2.0 ** -6)).all())


@pytest.mark.parametrize("T,D", [(1, 128), (3, 256), (5, 2048), (2, 2176), (7, 4096), (4, 5248), (2, 8192), (3, 16384),
                                 (1000, 640)])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("scale", ["f32", "f32_pow2", "e8m0"])
def test_rms_norm_quant(T, D, residual, scale):
    g = _gen(1, T, D, residual)
    x = torch.randn(T, D, generator=g, device="cuda").mul(3).bfloat16()
    res = torch.randn(T, D, generator=g, device="cuda").bfloat16() if residual else None
    w = torch.rand(D, generator=g, device="cuda") + 0.5
    if D % 256 == 0:
        w = w.bfloat16()
    r = _ops().rms_norm_quant(x, w, residual=res, norm_out=scale != "f32", scale_fmt=None if scale == "f32" else "ue8m0",
                              scale_dtype=E8 if scale == "e8m0" else torch.float32)
    assert (r.y is None) == (scale == "f32") and r.s.dtype == (E8 if scale == "e8m0" else torch.float32)
    _check_norm(x, w, res, r, scale != "f32")


def test_rms_norm_quant_special_rows():
    """Zeros, tiny and huge rows, one NaN, one infinity: each row is its own, and a fault in a row shows in it."""
    D = 512
    g = _gen(2)
    x = torch.randn(7, D, generator=g, device="cuda")
    x[1] = 0
    x[2] *= 1e-20
    x[3] *= 1e15
    x[4, 200] = math.nan
    x[5, 300] = math.inf
    x = x.bfloat16()
    w = torch.ones(D, device="cuda")
    for fmt, kind in ((None, torch.float32), ("ue8m0", E8)):
        r = _ops().rms_norm_quant(x, w, 1e-6, scale_fmt=fmt, scale_dtype=kind)
        ok = [0, 1, 2, 3, 6]
        part = type(r)(r.q[ok], r.s[ok], r.y[ok], None)
        _check_norm(x[ok], w, None, part, fmt is not None)
        assert bool((r.q[1].float() == 0).all()) and bool((r.y[1] == 0).all())
        assert bool(r.y[4].isnan().all()) and bool(r.q[4].float().isnan().all()) and bool(r.s[4].float().isnan().all())
        # inf / inf is NaN in its own block; the other blocks of the row are 0
        assert bool(r.y[5, 300].isnan()) and bool(r.s[5, 2].float().isnan()) and bool((r.q[5, :256].float() == 0).all())


def test_rms_norm_quant_shapes_strides_and_zero_rows():
    ops = _ops()
    g = _gen(3)
    big = torch.randn(6, 4, 1024, generator=g, device="cuda").bfloat16()
    w = torch.rand(512, generator=g, device="cuda")
    x = big[:, :, 256:768]  # rows apart
    r = ops.rms_norm_quant(x, w, residual=x.transpose(0, 1).contiguous().transpose(0, 1))
    assert r.q.shape == x.shape and r.s.shape == (6, 4, 4) and r.h.shape == x.shape
    _check_norm(x.contiguous(), w, x.contiguous(), r, False)
    one = ops.rms_norm_quant(x[0, 0], w)
    assert torch.equal(one.y, ops.rms_norm_quant(x, w).y[0, 0])
    z = ops.rms_norm_quant(x[:0], w, residual=x[:0])
    assert z.q.shape == (0, 4, 512) and z.s.shape == (0, 4, 4) and z.h.shape == (0, 4, 512)


def test_rms_norm_quant_feeds_fp8_gemm():
    """The quantized rows are operands of the framework's FP8 product as they are."""
    ops = _ops()
    g = _gen(4)
    x = torch.randn(5, 512, generator=g, device="cuda").bfloat16()
    w = torch.rand(512, generator=g, device="cuda") + 0.5
    b = (torch.randn(256, 512, generator=g, device="cuda") * 40).to(torch.float8_e4m3fn)
    b_s = torch.full((2, 4), 2.0 ** -11, device="cuda")
    for fmt, kind in ((None, torch.float32), ("ue8m0", E8)):
        r = ops.rms_norm_quant(x, w, scale_fmt=fmt, scale_dtype=kind)
        c = ops.fp8_gemm(r.q, r.s, b, b_s.to(kind))
        a = r.q.float().double() * r.s.float().double().repeat_interleave(128, 1)
        bd = b.float().double() * 2.0 ** -11
        mag = a.abs() @ bd.abs().T
        _within(c, a @ bd.T, BF16, float((mag * 512 * FP32).max()))


# ---- route_topk ------------------------------------------------------------------------------------------------
def _route_ref(logits, k, bias, score, G, keep, top2, renorm, scale):
    z = logits.double()
    dead = z == -math.inf
    if score == "softmax":
        e = torch.where(dead, 0.0, torch.exp(z - z.amax(-1, keepdim=True)))
        s = e / e.sum(-1, keepdim=True)
        s = torch.where(dead, 0.0, s)
    elif score == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
    else:
        s = torch.sqrt(z.clamp(min=0) + torch.log1p(torch.exp(-z.abs())))
    sel = s if bias is None else s + bias.double()
    sel = torch.where(dead, -math.inf, sel)
    T, E = z.shape
    out_i = torch.full((T, k), -1, dtype=torch.int64)
    out_w = torch.zeros(T, k, dtype=torch.float64)
    key = lambda v: (math.inf if v != v else v)  # noqa: E731
    for t in range(T):
        row = [float(v) for v in sel[t]]
        if G > 1:
            per = E // G
            val = []
            for i in range(G):
                m = sorted((v for v in row[i * per:(i + 1) * per] if v != -math.inf), key=key, reverse=True)
                val.append(-math.inf if not m else m[0] + m[1] if top2 and len(m) > 1 else m[0])
            order = [i for i in sorted(range(G), key=lambda i: (-key(val[i]), i)) if val[i] != -math.inf][:keep]
            row = [v if e // per in order else -math.inf for e, v in enumerate(row)]
        pick = [e for e in sorted(range(E), key=lambda e: (-key(row[e]), e)) if row[e] != -math.inf][:k]
        w = torch.tensor([float(s[t, e]) for e in pick], dtype=torch.float64)
        if renorm and len(pick):
            w = w / w.sum() if float(w.sum()) != 0 else w * 0
        for j, e in enumerate(pick):
            out_i[t, j] = e
            out_w[t, j] = w[j] * scale
    return out_w, out_i


def _check_route(logits, k, bias=None, score="sigmoid", G=1, keep=1, top2=None, renorm=None, scale=1.0, **kw):
    w, i = _ops().route_topk(logits, k, bias=bias, score_func=score, n_groups=G, topk_groups=keep, route_scale=scale,
                             group_score=None if top2 is None else "top2" if top2 else "max", renormalize=renorm)
    top2 = bias is not None if top2 is None else top2
    renorm = score != "softmax" if renorm is None else renorm
    rw, ri = _route_ref(logits.cpu(), k, None if bias is None else bias.cpu(), score, G, keep, top2, renorm, scale)
    assert torch.equal(i.cpu(), ri)
    finite = rw.isfinite()
    assert torch.equal(finite, w.cpu().isfinite())
    _within(w.cpu()[finite], rw[finite], 2 * FP32, 2.0 ** -149)
    return w, i


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 8), (3, 64, 6), (9, 256, 8), (130, 256, 6), (5, 384, 16), (4, 512, 8),
                                   (6, 33, 3), (2, 100, 7)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax", "sqrtsoftplus"])
@pytest.mark.parametrize("bias", [False, True])
def test_route_topk(T, E, k, score, bias):
    g = _gen(11, T, E, k)
    logits = torch.randn(T, E, generator=g, device="cuda") * 1.3
    b = torch.randn(E, generator=g, device="cuda") * 0.01 if bias else None
    _check_route(logits, k, b, score, scale=1.5)


@pytest.mark.parametrize("E,G,keep,k", [(256, 8, 4, 8), (64, 4, 1, 6), (48, 16, 3, 9), (96, 32, 7, 8), (512, 2, 1, 8), (30, 5, 5, 4),
                                        (32, 32, 6, 6)])
@pytest.mark.parametrize("top2", [True, False])
@pytest.mark.parametrize("score,bias", [("sigmoid", True), ("softmax", False)])
def test_route_topk_groups(E, G, keep, k, top2, score, bias):
    g = _gen(12, E, G, keep)
    logits = torch.randn(37, E, generator=g, device="cuda")
    b = torch.randn(E, generator=g, device="cuda") * 0.05 if bias else None
    _check_route(logits, k, b, score, G, keep, top2)


def test_route_topk_ties_go_to_the_lower_index():
    g = _gen(13)
    logits = torch.randint(-2, 3, (64, 128), generator=g, device="cuda").float()
    for score in ("sigmoid", "softmax", "sqrtsoftplus"):
        _check_route(logits, 8, None, score)
        _check_route(logits.bfloat16(), 8, torch.zeros(128, device="cuda"), score, 8, 3)
    _check_route(torch.zeros(3, 64, device="cuda"), 6)
    z = torch.zeros(2, 64, device="cuda")
    z[:, 1::2] = -0.0
    _check_route(z, 6)


def test_route_topk_neighbouring_values():
    """Logits one fp32 step apart, whose 32-bit sigmoids are equal, come out in the logits' order."""
    base = torch.full((1, 64), 2.0, device="cuda")
    steps = torch.arange(64, device="cuda").flip(0) * 2.0 ** -22
    logits = (base + steps).expand(3, 64).contiguous()
    assert torch.sigmoid(logits[0]).unique().numel() < 64
    _, i = _check_route(logits, 8)
    assert i[0].tolist() == list(range(8))


@pytest.mark.parametrize("score", ["sigmoid", "softmax", "sqrtsoftplus"])
@pytest.mark.parametrize("G,keep", [(1, 1), (8, 4)])
def test_route_topk_masks(score, G, keep):
    """-inf masks an expert; rows with fewer experts than slots, and with none, fill up with -1 and weight 0."""
    g = _gen(14, score, G)
    logits = torch.randn(12, 64, generator=g, device="cuda")
    logits[0] = -math.inf
    logits[1, 3:] = -math.inf
    logits[2, :60] = -math.inf
    logits[3, ::2] = -math.inf
    logits[4, 8:16] = -math.inf
    logits[5, 17] = torch.finfo(torch.float32).min
    logits[6] = torch.finfo(torch.float32).min
    logits[7] = -200.0
    bias = torch.randn(64, generator=g, device="cuda") * 0.01
    for b in (None, bias):
        w, i = _check_route(logits, 6, b, score, G, keep)
        assert i[0].tolist() == [-1] * 6 and w[0].tolist() == [0.0] * 6
    bias[5] = -math.inf
    _, i = _check_route(logits, 6, bias, score, G, keep)
    assert 5 not in i.tolist()[8]


def test_route_topk_nan_shows():
    g = _gen(15)
    logits = torch.randn(4, 64, generator=g, device="cuda")
    logits[1, 40] = math.nan
    for score in ("sigmoid", "softmax", "sqrtsoftplus"):
        w, i = _ops().route_topk(logits, 6, score_func=score)
        clean = [0, 2, 3]
        assert bool(w[clean].isfinite().all())
        assert bool(w[1].isnan().any())
        if score != "softmax":
            assert int(i[1, 0]) == 40


def test_route_topk_bf16_strides_zero_rows_and_defaults():
    ops = _ops()
    g = _gen(16)
    big = torch.randn(20, 128, generator=g, device="cuda").bfloat16()
    view = big[::2, :64]
    _check_route(view, 6, score="softmax")
    w, i = ops.route_topk(view, 6, score_func="softmax", renormalize=True)
    _within(w.sum(-1), torch.ones(10, dtype=torch.float64, device="cuda"), 8 * FP32)
    w, i = ops.route_topk(view[:0], 6)
    assert w.shape == (0, 6) and i.shape == (0, 6) and i.dtype == torch.int64


# ---- expert_dispatch ----------------------------------------------------------------------------------------------
def _dispatch_ref(indices, E, base):
    k = indices.size(1)
    flat = (indices.cpu().long().reshape(-1) - base).tolist()
    rows = sorted((e, p) for p, e in enumerate(flat) if 0 <= e < E)
    off, tok, slots = [0] * (E + 1), [-1] * len(flat), [-1] * len(flat)
    for r, (e, p) in enumerate(rows):
        tok[r] = p // k
        slots[p] = r
        off[e + 1] += 1
    for e in range(E):
        off[e + 1] += off[e]
    return off, tok, slots


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 6, 256), (5, 6, 64), (64, 6, 256), (341, 6, 512), (342, 6, 511), (2048, 1, 3),
                                   (2049, 1, 7), (3000, 8, 256), (700, 16, 100)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_expert_dispatch(T, k, E, dtype):
    g = _gen(21, T, k, E)
    ind = torch.randint(0, E, (T, k), generator=g, device="cuda").to(dtype)
    off, tok, slots = _ops().expert_dispatch(ind, E)
    ro, rt, rs = _dispatch_ref(ind, E, 0)
    assert off.tolist() == ro and tok.tolist() == rt and slots.reshape(-1).tolist() == rs


@pytest.mark.parametrize("T", [7, 1500])
def test_expert_dispatch_local_range_and_masked(T):
    g = _gen(22, T)
    ind = torch.randint(-1, 300, (T, 6), generator=g, device="cuda")
    ind[0, 0], ind[0, 1] = 1 << 40, -(1 << 40)
    for base, E in ((0, 256), (64, 32), (250, 100), (400, 8)):
        off, tok, slots = _ops().expert_dispatch(ind, E, expert_offset=base)
        ro, rt, rs = _dispatch_ref(ind, E, base)
        assert off.tolist() == ro and tok.tolist() == rt and slots.reshape(-1).tolist() == rs
    off, tok, slots = _ops().expert_dispatch(torch.full((T, 6), -1, device="cuda"), 16)
    assert not off.any() and bool((tok == -1).all()) and bool((slots == -1).all())


@pytest.mark.parametrize("how", ["one", "sorted", "reversed", "repeated"])
def test_expert_dispatch_skewed(how):
    """All pairs at one expert; runs of equal experts; an expert named twice by a token."""
    T, k, E = 1111, 4, 128
    if how == "one":
        ind = torch.full((T, k), 77, device="cuda")
    else:
        ind = (torch.arange(T * k, device="cuda") * E // (T * k)).view(T, k)
        if how == "reversed":
            ind = ind.flip(0, 1)
        if how == "repeated":
            ind[:, 1] = ind[:, 0]
    off, tok, slots = _ops().expert_dispatch(ind, E)
    ro, rt, rs = _dispatch_ref(ind, E, 0)
    assert off.tolist() == ro and tok.tolist() == rt and slots.reshape(-1).tolist() == rs


def test_expert_dispatch_many_pairs():
    """More pairs than the chunk count allows at the usual chunk size: against a stable sort."""
    T, k, E = 150001, 8, 256
    g = _gen(23)
    ind = torch.randint(0, E, (T, k), generator=g, device="cuda")
    off, tok, slots = _ops().expert_dispatch(ind, E)
    order = torch.sort(ind.reshape(-1), stable=True).indices
    assert torch.equal(tok.long(), order // k)
    assert torch.equal(slots.reshape(-1)[order].long(), torch.arange(T * k, device="cuda"))
    assert torch.equal(off[1:].long(), torch.bincount(ind.reshape(-1), minlength=E).cumsum(0)) and int(off[0]) == 0
    e = _ops().expert_dispatch(ind[:0], E)
    assert e[0].tolist() == [0] * (E + 1) and e[1].numel() == 0 and e[2].shape == (0, k)


# ---- expert_combine ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,k,D", [(1, 1, 8), (3, 6, 264), (16, 6, 4096), (5, 16, 2056), (2, 8, 8192), (300, 4, 512)])
@pytest.mark.parametrize("weighted,shared", [(True, True), (False, False), (True, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_expert_combine(T, k, D, weighted, shared, dtype):
    g = _gen(31, T, k, D)
    R = T * k
    rows = torch.randn(R, D, generator=g, device="cuda").bfloat16()
    slots = torch.randperm(R, generator=g, device="cuda").view(T, k).int()
    slots[0, 0] = -1
    slots[-1, -1] = R  # outside: adds nothing
    w = torch.rand(T, k, generator=g, device="cuda") if weighted else None
    sh = torch.randn(T, D, generator=g, device="cuda").bfloat16() if shared else None
    y = _ops().expert_combine(rows, slots, weights=w, shared=sh, out_dtype=dtype)
    ok = ((slots >= 0) & (slots < R))
    v = rows[slots.clamp(0, R - 1).long()].double() * ok[..., None]
    if weighted:
        v = v * w.double()[..., None]
    want, mag = v.sum(1), v.abs().sum(1)
    if shared:
        want, mag = want + sh.double(), mag + sh.double().abs()
    tol = mag * (k + 2) * FP32 + (want.abs() * BF16 * (1 + 2.0 ** -12) if dtype == torch.bfloat16 else 0)
    assert y.dtype == dtype and bool(((y.double() - want).abs() <= tol).all())


def test_expert_combine_order_and_empty():
    """Ascending rows whatever the slots' order: the same bits; no rows at all: the shared rows, or zeros."""
    ops = _ops()
    g = _gen(32)
    rows = torch.randn(64, 256, generator=g, device="cuda").bfloat16()
    slots = torch.randperm(64, generator=g, device="cuda").view(8, 8).int()
    w = torch.rand(8, 8, generator=g, device="cuda")
    y = ops.expert_combine(rows, slots, weights=w, out_dtype=torch.float32)
    perm = torch.randperm(8, generator=g, device="cuda")
    assert torch.equal(y, ops.expert_combine(rows, slots[:, perm], weights=w[:, perm], out_dtype=torch.float32))
    acc = torch.zeros(8, 256, device="cuda", dtype=torch.float64)
    s, o = slots.sort(-1)
    for j in range(8):  # the fused multiply-add of each step, rounded to 32 bits
        acc = (acc + w.gather(1, o)[:, j:j + 1].double() * rows[s[:, j].long()].double()).float().double()
    assert torch.equal(y, acc.float())
    none = torch.full((8, 8), -1, dtype=torch.int32, device="cuda")
    assert not ops.expert_combine(rows, none).any()
    assert torch.equal(ops.expert_combine(rows[:0], none, shared=rows[:8]), rows[:8])
    assert ops.expert_combine(rows, slots[:0]).shape == (0, 256)


# ---- streams, graphs, refusals --------------------------------------------------------------------------------------
def _pass(x, res, w, gate, bias):
    ops = _ops()
    r = ops.rms_norm_quant(x, w, residual=res, scale_fmt="ue8m0", scale_dtype=E8)
    logits = r.y.float() @ gate
    rw, ri = ops.route_topk(logits, 6, bias=bias, n_groups=8, topk_groups=4)
    off, tok, slots = ops.expert_dispatch(ri, 64)
    y = ops.expert_combine(r.y[tok.long()], slots, weights=rw, shared=r.h)
    return [r.q.view(torch.uint8), r.s.view(torch.uint8), r.y, r.h, rw, ri, off, tok, slots, y]


def test_side_stream_and_graph_replay():
    g = _gen(41)
    mk = lambda: (torch.randn(48, 512, generator=g, device="cuda").bfloat16(),  # noqa: E731
                  torch.randn(48, 512, generator=g, device="cuda").bfloat16())
    w = torch.rand(512, generator=g, device="cuda") + 0.5
    gate = torch.randn(512, 64, generator=g, device="cuda") * 0.05
    bias = torch.randn(64, generator=g, device="cuda") * 0.01
    (x, res), (x2, res2) = mk(), mk()
    want, want2 = _pass(x, res, w, gate, bias), _pass(x2, res2, w, gate, bias)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _pass(x, res, w, gate, bias)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # two graphs captured after one another, replayed in turn with new inputs
    ins = [[x.clone(), res.clone()] for _ in range(2)]
    graphs, outs = [], []
    for a, b in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_pass(a, b, w, gate, bias))
        graphs.append(graph)
    for (a, b), src in zip(ins, ((x2, res2), (x, res))):
        a.copy_(src[0])
        b.copy_(src[1])
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want2, outs[0]))
    assert all(torch.equal(a, b) for a, b in zip(want, outs[1]))


def test_refusals():
    ops = _ops()
    c = dict(device="cuda")
    x = torch.zeros(2, 256, dtype=torch.bfloat16, **c)
    w = torch.ones(256, **c)
    i64 = torch.zeros(2, 6, dtype=torch.int64, **c)
    bad = [
        (TypeError, lambda: ops.rms_norm_quant(x.float(), w)),
        (TypeError, lambda: ops.rms_norm_quant(x, w.half())),
        (ValueError, lambda: ops.rms_norm_quant(x, w[:128])),
        (ValueError, lambda: ops.rms_norm_quant(x[:, :192], w[:192])),
        (ValueError, lambda: ops.rms_norm_quant(x, w.cpu())),
        (ValueError, lambda: ops.rms_norm_quant(x, w, residual=x[:1])),
        (TypeError, lambda: ops.rms_norm_quant(x, w, residual=x.float())),
        (ValueError, lambda: ops.rms_norm_quant(x, w, scale_dtype=E8)),
        (TypeError, lambda: ops.rms_norm_quant(x, w, scale_fmt="ue8m0", scale_dtype=torch.float16)),
        (TypeError, lambda: ops.route_topk(x.double(), 6)),
        (ValueError, lambda: ops.route_topk(x[0], 6)),
        (ValueError, lambda: ops.route_topk(x, 17)),
        (ValueError, lambda: ops.route_topk(x, 0)),
        (ValueError, lambda: ops.route_topk(x, 6, score_func="relu")),
        (ValueError, lambda: ops.route_topk(x, 6, n_groups=7)),
        (ValueError, lambda: ops.route_topk(x, 6, n_groups=64, topk_groups=1)),
        (ValueError, lambda: ops.route_topk(x, 6, n_groups=8, topk_groups=9)),
        (ValueError, lambda: ops.route_topk(x, 6, group_score="sum")),
        (ValueError, lambda: ops.route_topk(x, 6, bias=w[:64])),
        (TypeError, lambda: ops.route_topk(x, 6, bias=w.bfloat16())),
        (TypeError, lambda: ops.expert_dispatch(i64.float(), 8)),
        (ValueError, lambda: ops.expert_dispatch(i64[0], 8)),
        (ValueError, lambda: ops.expert_dispatch(i64, 513)),
        (ValueError, lambda: ops.expert_dispatch(i64, 8, expert_offset=-1)),
        (ValueError, lambda: ops.expert_dispatch(i64.repeat(1, 3), 8)),
        (TypeError, lambda: ops.expert_combine(x.float(), i64.int())),
        (TypeError, lambda: ops.expert_combine(x, i64)),
        (ValueError, lambda: ops.expert_combine(x[:, :12], i64.int())),
        (ValueError, lambda: ops.expert_combine(x, i64.int(), weights=w[:6])),
        (ValueError, lambda: ops.expert_combine(x, i64.int(), shared=x[:1])),
        (TypeError, lambda: ops.expert_combine(x, i64.int(), out_dtype=torch.float16)),
    ]
    for k, (err, call) in enumerate(bad):
        with pytest.raises(err):
            call()
            pytest.fail(f"call {k} was not refused")


@pytest.mark.parametrize("score", ["sigmoid", "sqrtsoftplus"])
@pytest.mark.parametrize("bits", [6, 12, 20])
def test_route_topk_close_calls(score, bits):
    """Logits on coarse grids and pairs one step apart: many slots and groups that 32 bits cannot tell apart."""
    g = _gen(17, bits)
    base = torch.randn(96, 64, generator=g, device="cuda")
    logits = (base * 2 ** bits).round() / 2 ** bits
    # every second expert of the first half a neighbour of the one before it
    up = torch.nextafter(logits[:48, ::2], torch.full_like(logits[:48, ::2], math.inf))
    logits[:48, 1::2] = torch.where(torch.rand(48, 32, generator=g, device="cuda") < 0.5, up, logits[:48, ::2])
    # groups that mirror one another up to a step
    logits[48:, 32:] = logits[48:, :32]
    logits[72:, 33] = torch.nextafter(logits[72:, 33], torch.full_like(logits[72:, 33], math.inf))
    bias = torch.randn(64, generator=g, device="cuda") * 0.01
    bias[32:] = bias[:32]
    for b in (None, bias):
        for G, keep, top2 in ((1, 1, True), (8, 3, True), (8, 5, False), (4, 2, True), (32, 9, True)):
            _check_route(logits, 6, b, score, G, keep, top2)


def test_route_topk_large_and_cancelling_biases():
    """Biases that dwarf the scores, and pairs that cancel in a group's sum, leave the choice exact."""
    g = _gen(18)
    logits = torch.randn(64, 64, generator=g, device="cuda")
    bias = torch.zeros(64, device="cuda")
    bias[::8] = 1000.0
    bias[1::8] = -1000.0
    _check_route(logits, 6, bias, "sigmoid", 8, 4)
    bias = torch.full((64,), -1e9, device="cuda")
    bias[:20] = 0
    _check_route(logits, 8, bias, "sigmoid", 8, 4)
    _check_route(logits - 100, 8, None, "sqrtsoftplus")
    _check_route(logits - 95, 8, None, "sigmoid")


def test_outputs_are_complete_before_the_next_product_reads_them():
    """A norm's q is the weight operand of the framework's FP8 product at once, which reads weights ahead of its wait."""
    ops = _ops()
    g = _gen(42)
    w = torch.ones(2048, device="cuda")
    a = (torch.randn(4, 2048, generator=g, device="cuda") * 60).to(torch.float8_e4m3fn)
    a_s = torch.ones(4, 16, device="cuda").to(E8)
    b_s = torch.ones(32, 16, device="cuda").to(E8)
    for k in range(20):
        x = torch.randn(4096, 2048, generator=g, device="cuda").bfloat16()
        res = torch.randn(4096, 2048, generator=g, device="cuda").bfloat16()
        torch.cuda.synchronize()
        r = ops.rms_norm_quant(x, w, residual=res, norm_out=False, scale_fmt="ue8m0", scale_dtype=E8)
        c = ops.fp8_gemm(a, a_s, r.q, b_s)
        torch.cuda.synchronize()
        assert torch.equal(c, ops.fp8_gemm(a, a_s, r.q, b_s)), k


def test_offsets_past_32_bits():
    """More than 2^31 elements: the last rows are as right as the first."""
    ops = _ops()
    T, D = 150000, 16384  # 2.46e9 elements
    x = torch.ones(T, D, dtype=torch.bfloat16, device="cuda")
    x[-1, ::2] = 3.0
    r = ops.rms_norm_quant(x, torch.ones(D, device="cuda"), norm_out=True)
    want = ops.rms_norm_quant(x[-1:].clone(), torch.ones(D, device="cuda"), norm_out=True)
    for i, ref in ((0, None), (-1, want), (T - 2, None)):
        if ref is None:
            ref = ops.rms_norm_quant(x[i:i + 1 or None].clone(), torch.ones(D, device="cuda"), norm_out=True)
        assert torch.equal(r.q[i].view(torch.uint8), ref.q[0].view(torch.uint8))
        assert torch.equal(r.s[i], ref.s[0]) and torch.equal(r.y[i], ref.y[0])
    slots = torch.tensor([[T - 1, 0], [T - 2, T - 1], [1, T]], device="cuda").int()
    y = ops.expert_combine(x, slots)
    assert torch.equal(y[0].float(), x[-1].float() + 1) and torch.equal(y[1], y[0]) and bool((y[2] == 1).all())
    del r, x, want
    T, E = 4300000, 512  # 2.2e9 logits
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device="cuda")
    logits[-1, 300] = logits[-1, 17] = 1.0
    logits[0, 5] = 2.0
    w, i = ops.route_topk(logits, 2)
    assert i[-1].tolist() == [17, 300] and i[0].tolist() == [5, 0] and i[T // 2].tolist() == [0, 1]
    assert bool((w[1:].sum(-1) - 1).abs().max() < 1e-6)


def test_rms_norm_quant_overflowing_block():
    """A norm past the largest float: its block's scale is infinite (e8m0: NaN), its finite values become 0 (NaN)."""
    x = torch.zeros(1, 256, dtype=torch.bfloat16, device="cuda")
    x[0, 0], x[0, 1], x[0, 130] = 16.0, 1.0, 1.0
    w = torch.ones(256, device="cuda")
    w[0] = 3e38
    r = _ops().rms_norm_quant(x, w)
    assert float(r.s[0, 0]) == float("inf") and bool(r.y[0, 0].isinf())
    assert bool(r.q[0, 0].float().isnan()) and bool((r.q[0, 1:128].float() == 0).all())
    assert float(r.q[0, 130].float()) == 448.0
    e = _ops().rms_norm_quant(x, w, scale_fmt="ue8m0", scale_dtype=E8)
    assert bool(e.s[0, 0].float().isnan()) and bool(e.q[0, :128].float().isnan().all()) and not bool(e.s[0, 1].float().isnan())


def test_small_outputs_are_tensors_of_their_own():
    """Outputs that share an allocation do not overlap, have their own versions, and survive one another."""
    ops = _ops()
    g = _gen(43)
    for T in (1, 5, 300, 4000):
        x = torch.randn(T, 256, generator=g, device="cuda").bfloat16()
        r = ops.rms_norm_quant(x, torch.ones(256, device="cuda"), residual=x, scale_fmt="ue8m0", scale_dtype=E8)
        _check_norm(x, torch.ones(256, device="cuda"), x, r, True)
        w, i = ops.route_topk(torch.randn(T, 64, generator=g, device="cuda"), 6)
        d = ops.expert_dispatch(i, 64)
        every = [r.q, r.s, r.y, r.h, w, i, *d]
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in every)
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
        for t in every:
            assert t.is_contiguous() and t.data_ptr() % 16 == 0 and not t._is_view() and t._version == 0
        y, keep = r.y, r.y.clone()
        r.q.view(torch.uint8).fill_(0)
        assert y._version == 0
        del r
        other = [torch.full((T, 256), 7.0, device="cuda") for _ in range(8)]
        assert torch.equal(y, keep) and len(other) == 8
        i2 = i.clone()
        i.add_(1)
        assert torch.equal(i - 1, i2) and torch.equal(d[1], ops.expert_dispatch(i2, 64)[1])


def test_rms_norm_quant_divides_like_a_division():
    """q is what e4m3 of the float32 quotient n / s gives, on random values and next to every e4m3 midpoint.

    A row of ones with eps 0 has the norm 1, so n is the weight.  The one dividend that differs by a step, a power of two
    over a scale whose significand is all ones, does not occur: no scale here has that significand."""
    mids = [(2 * m + 1) * 2.0 ** -10 for m in range(8)] + [(2 * m + 17) * 2.0 ** (e - 4) for e in range(-6, 9) for m in range(8)]
    mids = torch.tensor([m for m in mids if m < 448], dtype=torch.float64, device="cuda")
    g = _gen(5)
    D = 16384
    x = torch.ones(1, D, dtype=torch.bfloat16, device="cuda")
    for k in range(48):
        top = torch.rand(D // 128, 1, generator=g, device="cuda") + 1
        top = top * torch.exp2(torch.randint(-9, 12, top.shape, generator=g, device="cuda").float())
        s = top * torch.tensor(1.0 / 448, device="cuda")
        assert not bool(((s.view(torch.int32) & 0x7fffff) == 0x7fffff).any())
        if k % 3 == 0:
            n = top * torch.rand(D // 128, 128, generator=g, device="cuda")
        else:  # within three float32 steps of a midpoint times the scale
            m = mids[torch.randint(0, mids.numel(), (D // 128, 128), generator=g, device="cuda")]
            n = (m * s.double()).float()
            n = (n.view(torch.int32) + torch.randint(-3, 4, n.shape, generator=g, device="cuda").int()).view(torch.float32)
            n = torch.minimum(n, top)
        n = torch.where(torch.rand(n.shape, generator=g, device="cuda") < 0.5, n, -n)
        n[:, 7] = top[:, 0]
        r = _ops().rms_norm_quant(x, n.reshape(-1), 0.0)
        assert torch.equal(r.s[0], s[:, 0])
        assert torch.equal(r.q[0].float(), (n / s).clamp(-448, 448).to(torch.float8_e4m3fn).float().reshape(-1))


def test_outputs_have_memory_of_their_own():
    """An output may be grown, shrunk to nothing or saved as any tensor; the call's other outputs stay as they are."""
    ops = _ops()
    g = _gen(44)
    x = torch.randn(5, 256, generator=g, device="cuda").bfloat16()
    r = ops.rms_norm_quant(x, torch.ones(256, device="cuda"), residual=x)
    w, i = ops.route_topk(torch.randn(5, 64, generator=g, device="cuda"), 6)
    d = ops.expert_dispatch(i, 64)
    every = [r.q, r.s, r.y, r.h, w, i, *d]
    assert len({t.untyped_storage().data_ptr() for t in every}) == len(every)
    assert all(t.untyped_storage().nbytes() == t.numel() * t.element_size() and t.storage_offset() == 0 for t in every)
    keep = [t.clone() for t in every]
    w.resize_(64, 6).fill_(-5)
    d[0].resize_(512).fill_(-5)
    r.s.untyped_storage().resize_(0)
    for t, k in zip(every, keep):
        if t is not w and t is not d[0] and t is not r.s:
            assert torch.equal(t.view(torch.uint8), k.view(torch.uint8))


def test_lazily_negated_inputs():
    """The imaginary part of a conjugate is a float32 view whose memory holds the negatives."""
    ops = _ops()
    g = _gen(45)
    z = torch.randn(1, 1, generator=g, device="cuda") + 1j * (torch.rand(1, 1, generator=g, device="cuda") + 1)
    rows = torch.randn(1, 256, generator=g, device="cuda").bfloat16()
    slots = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    w = z.conj().imag
    assert w.is_neg() and w.is_contiguous()
    got = ops.expert_combine(rows, slots, weights=w, out_dtype=torch.float32)
    assert torch.equal(got, -z.imag.clone() * rows.float())
    logits = torch.randn(3, 64, generator=g, device="cuda")
    for a, b in zip(ops.route_topk(torch._neg_view(logits), 6), ops.route_topk(-logits, 6)):
        assert torch.equal(a, b)
