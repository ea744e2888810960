"""grouped_fp8_gemm against a 64-bit product, and the whole way of a routed FP8 expert layer.

Tolerance, derived before the first run.  Products of two e4m3 values are exact in 32 bits; a scale product and its
application round once each (2 x 2^-24), and the sum of K terms in 32 bits is off by at most K roundings of the sum of
magnitudes, a truncating adder counted twice: (K + 2) x 2^-23 of the magnitudes, then half a bf16 step, 2^-8, of the value.
"""

import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

E8 = torch.float8_e8m0fnu


def _ops():
    from wanferenz_b200 import ops
    return ops


def _gen(*key):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(key).encode()))


def _operands(g, M, E, N, K, a_kind, w_kind):
    def q(*shape):
        return (torch.randn(*shape, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn)

    def s(kind, *shape):
        if kind == E8:
            return torch.exp2(torch.randint(-14, -4, shape, generator=g, device="cuda").float()).to(E8)
        return torch.rand(*shape, generator=g, device="cuda") * 1e-2 + 1e-4

    return (q(M, K), s(a_kind, M, K // 128), q(E, N, K), s(w_kind, E, -(-N // 128), K // 128))


def _check(out, a, a_s, w, w_s, offsets, rows, lo=0):
    E, N, K = w.shape
    off = offsets.tolist()
    ad = a.float().double() * a_s.float().double().repeat_interleave(128, 1)
    for e in range(E):
        if off[e] >= off[e + 1]:
            continue
        r = torch.arange(off[e], off[e + 1], device="cuda")
        i = r if rows is None else rows[r].long()
        ok = (i >= 0) & (i < a.size(0))
        x = ad[i.clamp(0, a.size(0) - 1)] * ok[:, None]
        wd = w[e].float().double() * w_s[e].float().double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
        want, mag = x @ wd.T, x.abs() @ wd.abs().T
        err = (out[r].double() - want).abs()
        tol = mag * (K + 2) * 2.0 ** -23 + want.abs() * 2.0 ** -8 + 2.0 ** -130
        assert bool((err <= tol).all()), (e, float((err - tol).max()))


def _offsets(counts):
    return torch.tensor([0] + list(counts), device="cuda").cumsum(0).int()


KINDS = [(torch.float32, torch.float32), (E8, E8), (E8, torch.float32), (torch.float32, E8)]


@pytest.mark.parametrize("counts", [[1], [16], [17, 0, 1], [0, 0, 5], [127, 128, 129], [3, 300, 0, 40, 257], [513, 2]])
@pytest.mark.parametrize("N,K", [(128, 128), (8, 256), (136, 1152), (384, 1024), (1000, 640)])
@pytest.mark.parametrize("kinds", KINDS)
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_fp8_gemm(counts, N, K, kinds, gather):
    g = _gen(1, counts, N, K, gather)
    R = sum(counts)
    M = R if not gather else max(1, R // 3)
    a, a_s, w, w_s = _operands(g, M, len(counts), N, K, *kinds)
    rows = torch.randint(0, M, (R,), generator=g, device="cuda").int() if gather else None
    off = _offsets(counts)
    out = _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows)
    _check(out, a, a_s, w, w_s, off, rows)


@pytest.mark.parametrize("kind", [torch.float32, E8])
@pytest.mark.parametrize("E,R,N,K", [(32, 2000, 4096, 512), (256, 900, 512, 2048), (512, 700, 256, 256), (3, 5000, 512, 4096),
                                     (1, 1100, 2048, 1024)])
def test_grouped_fp8_gemm_many_tiles(kind, E, R, N, K):
    """More tiles than SMs, uneven experts, many of them empty: every role's rings go round many times."""
    g = _gen(2, E, R, N, K)
    a, a_s, w, w_s = _operands(g, 333, E, N, K, kind, kind)
    e = (torch.rand(R, generator=g, device="cuda") ** 2 * E).long()
    off = torch.cat([torch.zeros(1, device="cuda").int(), torch.bincount(e, minlength=E).cumsum(0).int()])
    rows = torch.randint(0, 333, (R,), generator=g, device="cuda").int()
    ops = _ops()
    out = ops.grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows)
    _check(out, a, a_s, w, w_s, off, rows)
    for _ in range(3):
        assert torch.equal(out, ops.grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows))
    ops.grouped_read_error()


@pytest.mark.parametrize("kind", [torch.float32, E8])
def test_rows_of_no_expert_stay(kind):
    """Rows before the first expert's, between and behind the experts' are left as they were."""
    g = _gen(3)
    a, a_s, w, w_s = _operands(g, 100, 3, 256, 512, kind, kind)
    off = torch.tensor([0, 20, 20, 70], device="cuda").int()
    out = torch.full((100, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    assert _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, out=out) is out
    _check(out, a, a_s, w, w_s, off, None)
    assert bool((out[70:] == 7).all())
    out.fill_(7.0)
    off = torch.tensor([30, 31, 60, 60], device="cuda").int()
    _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, out=out)
    _check(out, a, a_s, w, w_s, off, None)
    assert bool((out[:30] == 7).all()) and bool((out[60:] == 7).all())
    off = torch.zeros(4, device="cuda").int()
    out.fill_(7.0)
    _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, out=out)
    assert bool((out == 7).all())


@pytest.mark.parametrize("kind", [torch.float32, E8])
def test_bad_offsets_and_rows(kind):
    """Offsets outside [0, R] are clamped; a row list entry outside [0, M) gives zeros, even beside NaN rows."""
    g = _gen(4)
    M, N, K = 40, 256, 256
    a, a_s, w, w_s = _operands(g, M, 3, N, K, kind, kind)
    a.view(torch.uint8)[0] = 0x7f  # row 0 is NaN, and no valid entry names it
    a.view(torch.uint8)[M - 1] = 0x7f
    rows = torch.randint(1, M - 1, (60,), generator=g, device="cuda").int()
    rows[3], rows[20], rows[59] = -1, M, 2 ** 31 - 1
    off = torch.tensor([-5, 20, 45, 1000], device="cuda").int()
    out = _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows)
    assert not out[3].any() and not out[20].any() and not out[59].any()
    b = a.clone()
    b.view(torch.uint8)[0] = 0
    b.view(torch.uint8)[M - 1] = 0
    _check(out, b, a_s, w, w_s, off.clamp(0, 60), rows)
    off = torch.tensor([50, 10, 40, 20], device="cuda").int()  # falling: such an expert has no rows
    out = torch.full((60, N), 7.0, dtype=torch.bfloat16, device="cuda")
    _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows, out=out)
    _check(out, b, a_s, w, w_s, off, rows)
    assert bool((out[:10] == 7).all()) and bool((out[40:] == 7).all())


@pytest.mark.parametrize("kind", [torch.float32, E8])
def test_nan_and_wide_scales(kind):
    """A NaN value or scale stays in its row or column block; scales far apart keep their meaning."""
    g = _gen(5)
    a, a_s, w, w_s = _operands(g, 20, 2, 256, 512, kind, kind)
    off = _offsets([12, 8])
    a.view(torch.uint8)[3, 130] = 0x7f
    a_s[5, 2] = float("nan")
    if kind == E8:
        w_s.view(torch.uint8)[1, 1, 3] = 255
        a_s.view(torch.uint8)[7, :] = torch.tensor([40, 100, 127, 160], device="cuda").byte()
        w_s.view(torch.uint8)[0, 0, :] = torch.tensor([190, 127, 120, 60], device="cuda").byte()
    else:
        w_s[1, 1, 3] = float("nan")
        a_s[7] = torch.tensor([2.0 ** -80, 1e-8, 1.0, 2.0 ** 30], device="cuda")
        w_s[0, 0] = torch.tensor([2.0 ** 60, 1.0, 2e-3, 2.0 ** -60], device="cuda")
    out = _ops().grouped_fp8_gemm(a, a_s, w, w_s, off)
    nan = out.isnan()
    want = torch.zeros(20, 256, dtype=torch.bool, device="cuda")
    want[[3, 5]] = True
    want[12:, 128:] = True
    assert torch.equal(nan, want)
    keep = [r for r in range(20) if r not in (3, 5)]
    clean, cs = a[keep].clone(), a_s[keep].clone()
    ws = w_s.clone()
    ws.view(torch.uint8)[1, 1, 3] = 0 if kind == E8 else ws.view(torch.uint8)[1, 1, 3]
    if kind != E8:
        ws[1, 1, 3] = 0
    o = out[keep].clone()
    o[10:, 128:] = 0
    wz = w.clone()
    wz.view(torch.uint8)[1, 128:] = 0
    _check(o, clean, cs, wz, ws, _offsets([10, 8]), None)


def test_agrees_with_the_dense_product():
    """One expert: fp8_gemm's result up to the order of the sums."""
    ops = _ops()
    g = _gen(6)
    for kind in (torch.float32, E8):
        a, a_s, w, w_s = _operands(g, 33, 1, 512, 1024, kind, kind)
        x = ops.grouped_fp8_gemm(a, a_s, w, w_s, _offsets([33])).double()
        y = ops.fp8_gemm(a, a_s, w[0], w_s[0]).double()
        mag = (a.float().abs() * a_s.float().repeat_interleave(128, 1)) @ \
            (w[0].float().abs() * w_s[0].float().repeat_interleave(128, 0).repeat_interleave(128, 1)).T
        assert bool(((x - y).abs() <= 2 * (1026 * 2.0 ** -23 * mag.double() + 2.0 ** -8 * y.abs())).all())


def _layer(x, res, p, k, graph_safe=True):
    """A prompt's way through a layer of FP8 experts, as a user's program chains the operators."""
    ops = _ops()
    r = ops.rms_norm_quant(x, p["norm"], residual=res, scale_fmt="ue8m0", scale_dtype=E8)
    w, idx = ops.route_topk(r.y.float() @ p["gate"], k, bias=p["bias"], n_groups=4, topk_groups=2, route_scale=1.5)
    off, tok, slots = ops.expert_dispatch(idx, p["w13"].size(0))
    gu = ops.grouped_fp8_gemm(r.q, r.s, p["w13"], p["w13_s"], off, rows=tok)
    gate, up = gu.float().chunk(2, -1)
    hq, hs = ops.act_quant((torch.nn.functional.silu(gate) * up).bfloat16(), 128, "ue8m0", E8)
    o = ops.grouped_fp8_gemm(hq, hs, p["w2"], p["w2_s"], off)
    return ops.expert_combine(o, slots, weights=w, shared=r.h), dict(r=r, w=w, idx=idx, off=off, tok=tok, slots=slots,
                                                                     hq=hq, hs=hs, o=o)


def _layer_params(g, E, D, I):
    wd = lambda *s: (torch.randn(*s, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    sc = lambda *s: torch.exp2(torch.randint(-13, -11, s, generator=g, device="cuda").float()).to(E8)  # noqa: E731
    return dict(norm=torch.rand(D, generator=g, device="cuda") + 0.5, gate=torch.randn(D, E, generator=g, device="cuda") * 0.02,
                bias=torch.randn(E, generator=g, device="cuda") * 0.01, w13=wd(E, 2 * I, D), w13_s=sc(E, 2 * I // 128, D // 128),
                w2=wd(E, D, I), w2_s=sc(E, D // 128, I // 128))


@pytest.mark.parametrize("T", [1, 5, 64, 700])
def test_a_layer_of_fp8_experts(T):
    """norm -> route -> dispatch -> w1/w3 -> SwiGLU -> w2 -> combine, against 64 bits from the quantized rows on."""
    E, D, I, k = 16, 512, 256, 4
    g = _gen(7, T)
    p = _layer_params(g, E, D, I)
    x = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    res = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    y, s = _layer(x, res, p, k)
    a = s["r"].q.float().double() * s["r"].s.float().double().repeat_interleave(128, 1)
    h = s["hq"].float().double() * s["hs"].float().double().repeat_interleave(128, 1)
    want, mag = s["r"].h.double(), s["r"].h.double().abs()
    for t in range(T):
        for j in range(k):
            e, r, w = int(s["idx"][t, j]), int(s["slots"][t, j]), s["w"][t, j].double()
            assert int(s["tok"][r]) == t and int(s["off"][e]) <= r < int(s["off"][e + 1])
            if t < 8:
                deq = lambda q, z: q[e].float().double() * z[e].float().double().repeat_interleave(128, 0).repeat_interleave(128, 1)  # noqa: E731
                gu = (deq(p["w13"], p["w13_s"]) @ a[t]).bfloat16().double()
                ref = torch.nn.functional.silu(gu[:I]) * gu[I:]
                # the bf16 roundings of gate, up and their product, then half an e4m3 step of the block's scale
                step = s["hs"][r].float().double().repeat_interleave(128) * 2.0 ** -10
                assert bool(((h[r] - ref).abs() <= ref.abs() * (2.0 ** -4 + 2.0 ** -5) + step + 2.0 ** -6 * gu[:I].abs().clamp(min=1e-3)
                             * gu[I:].abs()).all())
            c = w * s["o"][r].double()
            want[t] += c
            mag[t] += c.abs()
    assert bool(((y.double() - want).abs() <= mag * (k + 2) * 2.0 ** -24 + want.abs() * 2.0 ** -8 * (1 + 2.0 ** -12)).all())
    _check(s["o"], s["hq"], s["hs"], p["w2"], p["w2_s"], s["off"], None)


def test_layer_graph_replay_and_split_over_ranks():
    """The chain captured once and replayed on new tokens; two ranks' halves of the experts add up to the whole."""
    E, D, I, k, T = 16, 512, 256, 4, 96
    g = _gen(8)
    ops = _ops()
    p = _layer_params(g, E, D, I)
    xs = [torch.randn(T, D, generator=g, device="cuda").bfloat16() for _ in range(3)]
    res = torch.randn(T, D, generator=g, device="cuda").bfloat16()
    want = [_layer(x, res, p, k)[0] for x in xs]
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = _layer(x, res, p, k)
    for src, ref in zip(xs, want):
        x.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)
    _, s = _layer(xs[0], res, p, k)
    total = torch.zeros(T, D, dtype=torch.float64, device="cuda")
    for base in (0, E // 2):
        half = slice(base, base + E // 2)
        off, tok, slots = ops.expert_dispatch(s["idx"], E // 2, expert_offset=base)
        gu = ops.grouped_fp8_gemm(s["r"].q, s["r"].s, p["w13"][half], p["w13_s"][half], off, rows=tok)
        n = int(off[-1])
        gate, up = gu[:n].float().chunk(2, -1)
        hq, hs = ops.act_quant((torch.nn.functional.silu(gate) * up).bfloat16(), 128, "ue8m0", E8)
        o = ops.grouped_fp8_gemm(hq, hs, p["w2"][half], p["w2_s"][half], off)
        total += ops.expert_combine(o, slots, weights=s["w"], out_dtype=torch.float32).double()
    whole = ops.expert_combine(s["o"], s["slots"], weights=s["w"], out_dtype=torch.float32).double()
    mag = (s["o"].double()[s["slots"].long()].abs() * s["w"].double()[..., None]).sum(1)
    assert bool(((total - whole).abs() <= mag * (2 * k + 2) * 2.0 ** -24).all())


def test_zero_rows_and_refusals():
    ops = _ops()
    g = _gen(9)
    a, a_s, w, w_s = _operands(g, 10, 2, 256, 256, torch.float32, torch.float32)
    off = _offsets([4, 6])
    none = ops.grouped_fp8_gemm(a, a_s, w, w_s, off, rows=torch.empty(0, dtype=torch.int32, device="cuda"))
    assert none.shape == (0, 256)
    bad = [
        (TypeError, lambda: ops.grouped_fp8_gemm(a.float(), a_s, w, w_s, off)),
        (TypeError, lambda: ops.grouped_fp8_gemm(a, a_s.half(), w, w_s, off)),
        (TypeError, lambda: ops.grouped_fp8_gemm(a, a_s, w, w_s, off.long())),
        (TypeError, lambda: ops.grouped_fp8_gemm(a, a_s, w, w_s, off, rows=torch.arange(10, device="cuda"))),
        (ValueError, lambda: ops.grouped_fp8_gemm(a, a_s[:5], w, w_s, off)),
        (ValueError, lambda: ops.grouped_fp8_gemm(a, a_s, w, w_s[:, :1], off)),
        (ValueError, lambda: ops.grouped_fp8_gemm(a, a_s, w, w_s, off[:2])),
        (ValueError, lambda: ops.grouped_fp8_gemm(a[:, :192], a_s, w[:, :, :192], w_s, off)),
        (ValueError, lambda: ops.grouped_fp8_gemm(a, a_s, w[:, :252], w_s, off)),
        (ValueError, lambda: ops.grouped_fp8_gemm(a, a_s, w[0], w_s, off)),
        (ValueError, lambda: ops.grouped_fp8_gemm(a, a_s, w.cpu(), w_s, off)),
        (ValueError, lambda: ops.grouped_fp8_gemm(a[:0], a_s[:0], w, w_s, off, rows=torch.zeros(4, device="cuda").int())),
        (ValueError, lambda: ops.grouped_fp8_gemm(a, a_s, w, w_s, off, out=torch.empty(9, 256, device="cuda").bfloat16())),
        (ValueError, lambda: ops.grouped_fp8_gemm(a, a_s, w, w_s, off, out=torch.empty(10, 512, device="cuda").bfloat16()[:, ::2])),
    ]
    for k, (err, call) in enumerate(bad):
        with pytest.raises(err):
            call()
            pytest.fail(f"call {k} was not refused")


@pytest.mark.parametrize("kind", [torch.float32, E8])
@pytest.mark.parametrize("per", [3, 200])
def test_a_wait_that_runs_out_is_reported(kind, per):
    """With the bound of device waits at 200 cycles a wait for a copy runs out: the call ends early and says so, and
    the next call is not affected."""
    from wanferenz_b200 import _lib as L
    ops = _ops()
    g = _gen(10, per)
    E, N, K = 4, 512, 2048
    a, a_s, w, w_s = _operands(g, E * per, E, N, K, kind, kind)
    off = _offsets([per] * E)
    want = ops.grouped_fp8_gemm(a, a_s, w, w_s, off)
    ops.grouped_read_error()
    try:
        L.check(L.load().wf_set_wait_limit(200), "wf_set_wait_limit")
        ops.grouped_fp8_gemm(a, a_s, w, w_s, off)
        with pytest.raises(L.WfError) as e:
            ops.grouped_read_error()
        assert e.value.code == L.WF_E_TIMEOUT
    finally:
        L.load().wf_set_wait_limit(0)
    assert torch.equal(want, ops.grouped_fp8_gemm(a, a_s, w, w_s, off))
    ops.grouped_read_error()


def test_views_off_a_16_byte_boundary():
    """Inputs that start inside a 16-byte line are copied, an output that does is refused."""
    ops = _ops()
    g = _gen(11)
    a, a_s, w, w_s = _operands(g, 24, 2, 256, 256, torch.float32, E8)
    off = _offsets([9, 15])
    want = ops.grouped_fp8_gemm(a, a_s, w, w_s, off)

    def shifted(t):
        s = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        s.copy_(t)
        return s

    got = ops.grouped_fp8_gemm(shifted(a), shifted(a_s), shifted(w), shifted(w_s), shifted(off))
    assert torch.equal(got, want)
    with pytest.raises(ValueError):
        ops.grouped_fp8_gemm(a, a_s, w, w_s, off, out=shifted(want))
    x = torch.randn(5, 256, generator=g, device="cuda").bfloat16()
    r, s = ops.rms_norm_quant(x, torch.ones(256, device="cuda"), residual=x), None
    s = ops.rms_norm_quant(shifted(x), shifted(torch.ones(256, device="cuda")), residual=shifted(x))
    assert torch.equal(r.q.view(torch.uint8), s.q.view(torch.uint8)) and torch.equal(r.s, s.s) and torch.equal(r.y, s.y)
    slots = torch.arange(5, device="cuda").int().view(5, 1)
    assert torch.equal(ops.expert_combine(shifted(x), shifted(slots), shared=shifted(x)), ops.expert_combine(x, slots, shared=x))


@pytest.mark.parametrize("kind", [torch.float32, E8])
def test_offsets_past_32_bits(kind):
    """An output of more than 2^31 elements, rows listed and packed: the last rows are as right as the first."""
    ops = _ops()
    g = _gen(12)
    R, N, K = 600000, 4096, 128
    a, a_s, w, w_s = _operands(g, 1000, 2, N, K, kind, kind)
    rows = (torch.arange(R, device="cuda") % 1000).int()
    off = torch.tensor([0, 599990, R], device="cuda").int()
    out = ops.grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows)
    few = ops.grouped_fp8_gemm(a, a_s, w[1:], w_s[1:], _offsets([10]), rows=rows[-10:].contiguous())
    assert torch.equal(out[-10:], few)
    part = torch.cat([torch.arange(40), torch.arange(599990 - 40, 599990)]).cuda()
    _check(out[part], a, a_s, w[:1], w_s[:1], _offsets([80]), rows[part])


@pytest.mark.parametrize("kind", [torch.float32, E8])
def test_offsets_that_give_every_expert_all_rows(kind):
    """Offsets that fall again and again: every second expert owns all rows; the call stays in bounds, and with equal
    weights it does not matter which expert writes last."""
    ops = _ops()
    g = _gen(13)
    a, a_s, w, w_s = _operands(g, 3000, 1, 128, 128, kind, kind)
    E = 512
    off = torch.tensor([0, 3000], device="cuda").repeat(E // 2 + 1)[:E + 1].int()
    out = ops.grouped_fp8_gemm(a, a_s, w.view(torch.uint8).expand(E, 128, 128).contiguous().view(w.dtype),
                               w_s.float().expand(E, 1, 1).contiguous().to(kind), off)
    _check(out, a, a_s, w, w_s, _offsets([3000]), None)


def test_two_streams_and_threads_at_once():
    """Layers running at the same time on two streams, from two host threads, do not touch one another."""
    import threading

    g = _gen(14)
    p = [_layer_params(g, 16, 512, 256) for _ in range(2)]
    x = [torch.randn(T, 512, generator=g, device="cuda").bfloat16() for T in (3, 900)]
    res = [torch.randn(T, 512, generator=g, device="cuda").bfloat16() for T in (3, 900)]
    want = [_layer(x[i], res[i], p[i], 4)[0] for i in range(2)]
    torch.cuda.synchronize()
    got, bad = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i].append(_layer(x[i], res[i], p[i], 4)[0])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001 (reported by the main thread)
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(y, want[i]) for y in got[i])


def test_inference_mode_and_parameters():
    """Weights that are parameters, and calls inside inference mode, are taken as they are."""
    g = _gen(15)
    ops = _ops()
    x = torch.randn(5, 256, generator=g, device="cuda").bfloat16()
    w = torch.nn.Parameter(torch.rand(256, generator=g, device="cuda"))
    want = ops.rms_norm_quant(x, w.detach())
    with torch.inference_mode():
        got = ops.rms_norm_quant(x, w)
    assert torch.equal(want.y, got.y) and torch.equal(want.s, got.s) and not want.y.requires_grad
    assert torch.equal(ops.rms_norm_quant(x, w).y, want.y)


@pytest.mark.parametrize("kind", [torch.float32, E8])
@pytest.mark.parametrize("per", [3, 200])
@pytest.mark.parametrize("K", [128, 512])
def test_a_short_product_whose_wait_runs_out(kind, per, K):
    """As few K steps as stages: the producer issues every copy without a wait of its own, and the CTA still leaves
    only when they have landed.  The next call, in the same shared memory, is not affected."""
    from wanferenz_b200 import _lib as L
    ops = _ops()
    g = _gen(16, per, K)
    E, N = 4, 512
    a, a_s, w, w_s = _operands(g, E * per, E, N, K, kind, kind)
    off = _offsets([per] * E)
    want = ops.grouped_fp8_gemm(a, a_s, w, w_s, off)
    ops.grouped_read_error()
    try:
        L.check(L.load().wf_set_wait_limit(200), "wf_set_wait_limit")
        ops.grouped_fp8_gemm(a, a_s, w, w_s, off)
        with pytest.raises(L.WfError) as e:
            ops.grouped_read_error()
        assert e.value.code == L.WF_E_TIMEOUT
    finally:
        L.load().wf_set_wait_limit(0)
    assert torch.equal(want, ops.grouped_fp8_gemm(a, a_s, w, w_s, off))
    ops.grouped_read_error()


# Every path of the product by rows per expert: lists gathered in place, narrow tiles (lists packed first), wide tiles of
# either kind of scales.  300 rows an expert are two wide tiles, so an entry may lie past columns 32, 64 and 128 of one.
PATHS = [("gather", True, 12), ("narrow", True, 40), ("narrow", False, 40), ("wide", True, 300), ("wide", False, 300)]


def _marked(t, at):
    """`t` with the e4m3 rows `at` NaN, and with them zero."""
    nan, zero = t.clone(), t.clone()
    nan.view(torch.uint8)[at] = 0x7f
    zero.view(torch.uint8)[at] = 0
    return nan, zero


@pytest.mark.parametrize("kind", [torch.float32, E8])
@pytest.mark.parametrize("path,listed,per", PATHS)
@pytest.mark.parametrize("N,K", [(264, 384), (128, 1024)])
def test_gaps_and_bad_rows_on_every_path(kind, path, listed, per, N, K):
    """Rows of no expert stay as they were, NaN rows right behind an expert's last row do not reach it, and entries
    outside [0, M) give zeros wherever in a tile they stand, though row 0 of a is NaN."""
    g = _gen(17, path, listed, N)
    E, R = 3, 3 * per
    M = 50 if listed else R
    a, a_s, w, w_s = _operands(g, M, E, N, K, kind, kind)
    ends = [3, per - 3, per + 2, 2 * per + 5, R - 4]
    off = torch.tensor([ends[0], ends[1], 2 * per + 5, ends[4]], device="cuda").int()  # rows before, none between, behind
    if listed:
        a, clean = _marked(a, [0, M - 1])
        rows = torch.randint(1, M - 1, (R,), generator=g, device="cuda").int()
        rows[:ends[0]] = 0
        rows[ends[4]:] = M - 1
        bad = [p for p in (3, 3 + 33, 3 + 66, 3 + 130, per - 4, per + 40, 2 * per + 4, R - 5) if 3 <= p < R - 4]
        for j, p in enumerate(bad):
            rows[p] = (-1, M, 2 ** 31 - 1, -2 ** 31)[j % 4]
    else:
        a, clean = _marked(a, list(range(ends[0])) + list(range(ends[4], R)))
        rows, bad = None, []
    out = torch.full((R, N), 7.0, dtype=torch.bfloat16, device="cuda")
    _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows, out=out)
    _check(out, clean, a_s, w, w_s, off, rows)
    assert bool((out[:ends[0]] == 7).all()) and bool((out[ends[4]:] == 7).all())
    assert not bad or not out[bad].any()
    # an expert without rows between two with rows, its neighbours' rows NaN to one another
    off = torch.tensor([0, ends[1], ends[1], ends[2]], device="cuda").int()
    out.fill_(7.0)
    _ops().grouped_fp8_gemm(clean, a_s, w, w_s, off, rows=rows, out=out)
    _check(out, clean, a_s, w, w_s, off, rows)
    assert bool((out[ends[2]:] == 7).all())
    _ops().grouped_read_error()


@pytest.mark.parametrize("kind", [torch.float32, E8])
@pytest.mark.parametrize("path,listed,per", PATHS)
def test_clamped_and_falling_offsets_on_every_path(kind, path, listed, per):
    """Offsets outside [0, R] are clamped to it; an expert whose end lies before its start has no rows."""
    g = _gen(18, path, listed)
    E, R, N, K = 3, 3 * per, 136, 256
    M = 40 if listed else R
    a, a_s, w, w_s = _operands(g, M, E, N, K, kind, kind)
    rows = torch.randint(0, M, (R,), generator=g, device="cuda").int() if listed else None
    for off in ([-2 ** 31, per, R - 1, 2 ** 31 - 1], [2 * per, per, 2 * per + 1, per + 1], [R, R, R + 5, 0], [R + 1, -1, 1, 0]):
        off = torch.tensor(off, device="cuda").int()
        out = torch.full((R, N), 7.0, dtype=torch.bfloat16, device="cuda")
        _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows, out=out)
        inside = off.clamp(0, R)
        _check(out, a, a_s, w, w_s, inside, rows)
        owned = torch.zeros(R, dtype=torch.bool, device="cuda")
        lo, hi = inside[:-1].tolist(), inside[1:].tolist()
        for x, y in zip(lo, hi):
            owned[x:max(x, y)] = True
        assert bool((out[~owned] == 7).all())
    _ops().grouped_read_error()


@pytest.mark.parametrize("kind", [torch.float32, E8])
@pytest.mark.parametrize("path,listed,per", PATHS)
def test_nan_stays_in_its_row_or_block_on_every_path(kind, path, listed, per):
    g = _gen(19, path, listed)
    E, R, N, K = 2, 2 * per, 264, 512
    a, a_s, w, w_s = _operands(g, R, E, N, K, kind, kind)
    off = _offsets([per, per])
    rows = torch.randperm(R, generator=g, device="cuda").int() if listed else None
    named = rows.long() if listed else torch.arange(R, device="cuda")
    at = [1, per // 2, per - 1, per + 2]  # rows of the product
    a.view(torch.uint8)[named[at[0]], 130] = 0x7f
    a.view(torch.uint8)[named[at[1]], 511] = 0xff
    a_s[named[at[2]], 2] = float("nan")
    a_s[named[at[3]], 0] = float("nan")
    if kind == E8:
        w_s.view(torch.uint8)[1, 1, 3] = 255
    else:
        w_s[1, 1, 3] = float("nan")
    w.view(torch.uint8)[0, 263, 5] = 0x7f
    out = _ops().grouped_fp8_gemm(a, a_s, w, w_s, off, rows=rows)
    want = torch.zeros(R, N, dtype=torch.bool, device="cuda")
    want[at] = True
    want[per:, 128:256] = True
    want[:per, 263] = True
    assert torch.equal(out.isnan(), want)
    _ops().grouped_read_error()


def test_a_given_output_counts_as_changed():
    """A graph that holds `out` from before the call says so in its backward pass, as for any write in place."""
    g = _gen(20)
    a, a_s, w, w_s = _operands(g, 10, 2, 128, 128, E8, E8)
    out = torch.zeros(10, 128, dtype=torch.bfloat16, device="cuda")
    factor = torch.ones(10, 128, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    held = (out * factor).sum()
    _ops().grouped_fp8_gemm(a, a_s, w, w_s, _offsets([4, 6]), out=out)
    assert out._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        held.backward()
    with torch.inference_mode():
        inner = torch.zeros_like(out)
        assert _ops().grouped_fp8_gemm(a, a_s, w, w_s, _offsets([4, 6]), out=inner) is inner
    assert torch.equal(_ops().grouped_fp8_gemm(a, a_s, w, w_s, _offsets([4, 6]), out=inner), out)


@pytest.mark.parametrize("kind", [torch.float32, E8])
def test_a_bounded_list_of_local_rows(kind):
    """A rank's experts with the list of all pairs, and with its first rows alone (narrower tiles): the same values up
    to the order of the sums, through to the rank's partial sums."""
    ops = _ops()
    g = _gen(21)
    T, k, ranks, E, N, K = 256, 4, 8, 4, 256, 512
    idx = torch.rand(T, ranks * E, generator=g, device="cuda").topk(k, dim=-1).indices
    a, a_s, w, w_s = _operands(g, T, E, N, K, kind, kind)
    off, tok, slots = ops.expert_dispatch(idx, E, expert_offset=2 * E)
    n = int(off[-1])
    bound = n + 5
    assert bound < 48 * E < T * k
    whole = ops.grouped_fp8_gemm(a, a_s, w, w_s, off, rows=tok)
    part = ops.grouped_fp8_gemm(a, a_s, w, w_s, off, rows=tok[:bound])
    assert part.shape == (bound, N)
    _check(whole, a, a_s, w, w_s, off, tok)
    _check(part, a, a_s, w, w_s, off, tok)
    y = ops.expert_combine(part, slots, out_dtype=torch.float32).double()
    local = slots.clamp(min=0).long()
    want = (part[local].double() * (slots >= 0)[..., None]).sum(1)
    mag = (part[local].double().abs() * (slots >= 0)[..., None]).sum(1)
    assert bool(((y - want).abs() <= mag * (k + 1) * 2.0 ** -24).all())
