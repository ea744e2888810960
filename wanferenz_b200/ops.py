"""Operator API of ``wanferenz.kernels.reference`` on the B200 kernels.

Same names, arguments and return values as the reference's operators
(wanferenz/kernels/reference.py and its CPU twin wanferenz/kernels/torch_ops.py),
so ``architecture.linear()`` can bind them unchanged:

* ``act_quant(x, block_size=128, scale_fmt=None, scale_dtype=torch.float32, inplace=False)``
* ``fp4_act_quant(x, block_size=32, inplace=False)``
* ``fp8_gemm(a, a_s, b, b_s, scale_dtype=torch.float32)``
* ``fp4_gemm(a, a_s, b, b_s, scale_dtype=torch.float32)``
* ``grouped_fp4_gemm(a, a_s, w, w_s, scale_dtype=torch.float32)`` (fp4_grouped.py:96-128)

and the operators around a layer of routed FP8 experts, for one token or many, on the
way from the residual stream through the experts' products and back:

* ``rms_norm_quant(x, weight, eps, residual)``  residual + RMS norm + E4M3 output with scales
* ``route_topk(logits, topk, ...)``             scores, bias, groups, top-k, renormalised weights
* ``expert_dispatch(indices, n_experts)``       the router's choice as rows in expert order
* ``grouped_fp8_gemm(a, a_s, w, w_s, offsets, rows)``  each expert's rows times its FP8 weights
* ``expert_combine(rows, slots, weights)``      the experts' rows back in token order

These run on their tensors' device (which need not be the current one) and on its
current stream, and keep nothing between calls.

All tensors must be CUDA tensors; there is no CPU path.  Outputs are bf16,
as the reference's are under the model's bf16 default dtype.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib as L

_GEMM_WS = {}


def _need_cuda(*ts):
    for t in ts:
        if not t.is_cuda:
            raise ValueError("wanferenz_b200 operators run on CUDA tensors only")


def _kind(s: torch.Tensor) -> int:
    if s.dtype == torch.float32:
        return L.WF_SCALE_F32
    if s.dtype == torch.float8_e8m0fnu:
        return L.WF_SCALE_E8M0
    raise TypeError(f"unsupported scale dtype {s.dtype}")


def _u8(t: torch.Tensor) -> torch.Tensor:
    return t.contiguous().view(torch.uint8)


def _gemm_ws(device, m, n, k) -> torch.Tensor:
    """Per-device workspace, grown to the largest (M, N, K) seen; zero-filled when allocated
    (its split-K counters return to zero after every call)."""
    need = L.load().wf_gemm_workspace_bytes(m, n, k)
    if need == 0:
        raise ValueError(f"unsupported GEMM shape M={m} N={n} K={k}")
    key = (device.type, device.index)
    ws = _GEMM_WS.get(key)
    if ws is None or ws.numel() < need:
        ws = _GEMM_WS[key] = torch.zeros(need, dtype=torch.uint8, device=device)
    return ws


def act_quant(x, block_size=128, scale_fmt=None, scale_dtype=torch.float32, inplace=False):
    """Per-``block_size`` E4M3 quantization (torch_ops.py:33-49; reference.py:117-146)."""
    _need_cuda(x)
    lib = L.load()
    z = x.contiguous()
    if z.dtype != torch.bfloat16:
        raise TypeError("act_quant expects bf16 input")
    n = z.size(-1)
    if n % block_size:
        raise ValueError(f"last dim {n} is not a multiple of {block_size}")
    m = z.numel() // n
    y = torch.empty(z.shape, dtype=torch.float8_e4m3fn, device=z.device)
    s = torch.empty(*z.shape[:-1], n // block_size, dtype=scale_dtype, device=z.device)
    L.check(lib.wf_act_quant(L.ptr(z), m, n, block_size, int(scale_fmt is not None), L.ptr(y),
                             L.ptr(s), _kind(s), L.stream_ptr()), "wf_act_quant")
    if inplace:
        deq = y.float() * s.float().repeat_interleave(block_size, -1)
        x.copy_(deq.to(x.dtype))
        return x
    return y, s


def fp4_act_quant(x, block_size=32, inplace=False):
    """Per-32 E2M1 quantization with UE8M0 scales (torch_ops.py:61-74; reference.py:212-232)."""
    _need_cuda(x)
    if block_size != 32:
        raise ValueError("fp4_act_quant supports block_size=32 only")
    lib = L.load()
    z = x.contiguous()
    n = z.size(-1)
    m = z.numel() // n
    q = torch.empty(*z.shape[:-1], n // 2, dtype=torch.uint8, device=z.device)
    s = torch.empty(*z.shape[:-1], n // 32, dtype=torch.uint8, device=z.device)
    L.check(lib.wf_fp4_act_quant(L.ptr(z), m, n, L.ptr(q), L.ptr(s), L.stream_ptr()),
            "wf_fp4_act_quant")
    q = q.view(torch.float4_e2m1fn_x2)
    s = s.view(torch.float8_e8m0fnu)
    if inplace:
        from . import moe as _moe

        x.copy_(_moe.dequant_fp4(q, s).to(x.dtype))
        return x
    return q, s


def _out(a, n):
    return torch.empty(*a.shape[:-1], n, dtype=torch.bfloat16, device=a.device)


def fp8_gemm(a, a_s, b, b_s, scale_dtype=torch.float32):
    """``C = (a*a_s) @ (b*b_s)^T`` for E4M3 ``a [.., K]``, ``b [N, K]`` with 128x128 weight blocks."""
    _need_cuda(a, a_s, b, b_s)
    lib = L.load()
    k, n = a.size(-1), b.size(0)
    m = a.numel() // k
    c = _out(a, n)
    ws = _gemm_ws(a.device, m, n, k)
    L.check(lib.wf_fp8_gemm(L.ptr(_u8(a)), L.ptr(a_s.contiguous()), _kind(a_s), L.ptr(_u8(b)),
                            L.ptr(b_s.contiguous()), _kind(b_s), m, n, k, L.ptr(c), L.ptr(ws),
                            ws.numel(), L.stream_ptr()), "wf_fp8_gemm")
    return c


def fp4_gemm(a, a_s, b, b_s, scale_dtype=torch.float32):
    """``C = (a*a_s) @ (unpack(b)*b_s)^T`` for E4M3 ``a [.., K]`` and packed E2M1 ``b [N, K/2]``."""
    _need_cuda(a, a_s, b, b_s)
    lib = L.load()
    k, n = a.size(-1), b.size(0)
    m = a.numel() // k
    c = _out(a, n)
    ws = _gemm_ws(a.device, m, n, k)
    L.check(lib.wf_fp4_gemm(L.ptr(_u8(a)), L.ptr(a_s.contiguous()), _kind(a_s), L.ptr(_u8(b)),
                            L.ptr(_u8(b_s)), m, n, k, L.ptr(c), L.ptr(ws), ws.numel(),
                            L.stream_ptr()), "wf_fp4_gemm")
    return c


def grouped_fp4_gemm(a, a_s, w, w_s, scale_dtype=torch.float32):
    """Slot ``g`` multiplies ``a[g]`` by its own FP4 weights ``w[g]`` (fp4_grouped.py:96-128)."""
    _need_cuda(a, a_s, w, w_s)
    lib = L.load()
    g, k = a.shape
    n = w.size(1)
    c = torch.empty(g, n, dtype=torch.bfloat16, device=a.device)
    ws = _gemm_ws(a.device, g, n, k)
    L.check(lib.wf_grouped_fp4_gemm(L.ptr(_u8(a)), L.ptr(a_s.contiguous()), _kind(a_s),
                                    L.ptr(_u8(w)), L.ptr(_u8(w_s)), g, n, k, L.ptr(c), L.ptr(ws),
                                    ws.numel(), L.stream_ptr()), "wf_grouped_fp4_gemm")
    return c


# ----------------------------------------------------------------------------
# the operators around a layer of routed FP8 experts
# ----------------------------------------------------------------------------
class NormQuant(NamedTuple):
    """What ``rms_norm_quant`` returns."""

    q: torch.Tensor             # [.., D] float8_e4m3fn
    s: torch.Tensor             # [.., D/128] scales
    y: Optional[torch.Tensor]   # [.., D] bf16 norm (norm_out=True)
    h: Optional[torch.Tensor]   # [.., D] bf16 residual stream (residual given)


def _check(name, t, dtypes, device=None, shape=None):
    """Argument checks shared by the operators below: a CUDA tensor of one of ``dtypes`` (on
    ``device``, of ``shape``); returns it contiguous."""
    if not t.is_cuda:
        raise ValueError("wanferenz_b200 operators run on CUDA tensors only")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t.contiguous()


def _run(device, name, *args):
    """Calls entry point ``name`` with ``args`` and the current stream of ``device``, with that device current."""
    fn = getattr(L.load(), name)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc:
        L.check(rc, name)


_F32, _BF16, _E4M3, _E8M0 = (torch.float32,), (torch.bfloat16,), (torch.float8_e4m3fn,), (torch.float8_e8m0fnu,)


def rms_norm_quant(x, weight, eps=1e-6, *, residual=None, norm_out=True, scale_fmt=None, scale_dtype=torch.float32):
    """RMS norm (with the residual's addition) and its E4M3 quantization, in one pass.

    ``x [.., D]`` bf16, ``weight [D]`` f32 or bf16, ``residual [.., D]`` bf16 or None; ``D`` a
    multiple of 128 up to 16384.  The reference's RMSNorm.forward followed by ``act_quant(.., 128, scale_fmt, scale_dtype)``, on ``h = bf16(x + residual)``::

        n = h * rsqrt(mean(h^2) + eps) * weight           (32 bits)
        s = max(amax|n|, 1e-4) / 448 per 128 columns      (scale_fmt: rounded up to a power of two)
        q = e4m3(n / s)

    Returns ``NormQuant(q, s, y, h)``: ``y = bf16(n)`` for readers of the bf16 norm (the router,
    ``MoELayer``) unless ``norm_out=False``, ``h`` when ``residual`` is given.  ``q`` is taken from
    the 32-bit ``n``, so it can differ from ``act_quant(y)`` by that one bf16 rounding.
    """
    x = _check("x", x, _BF16)
    dev = x.device
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    d = x.size(-1)
    if d == 0 or d % 128 or d > 16384:
        raise ValueError(f"last dim {d} must be a multiple of 128, at most 16384")
    weight = _check("weight", weight, _F32 + _BF16, dev, (d,))
    if scale_dtype not in _F32 + _E8M0:
        raise TypeError(f"unsupported scale dtype {scale_dtype}")
    if scale_fmt is None and scale_dtype == torch.float8_e8m0fnu:
        raise ValueError("e8m0 scales need scale_fmt (power-of-two rounding)")
    h = None
    if residual is not None:
        residual = _check("residual", residual, _BF16, dev, x.shape)
        h = torch.empty_like(x)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    s = torch.empty(*x.shape[:-1], d // 128, dtype=scale_dtype, device=dev)
    y = torch.empty_like(x) if norm_out else None
    if x.numel():
        _run(dev, "wf_rms_norm_quant", L.ptr(x), L.ptr(residual), L.ptr(weight), int(weight.dtype == torch.bfloat16),
             x.numel() // d, d, float(eps), int(scale_fmt is not None), L.ptr(q), L.ptr(s), _kind(s), L.ptr(y),
             L.ptr(h))
    return NormQuant(q, s, y, h)


def route_topk(logits, topk, *, bias=None, score_func="sigmoid", n_groups=1, topk_groups=None, group_score=None,
               renormalize=None, route_scale=1.0):
    """Expert choice from router logits ``[T, E]`` (f32 or bf16): ``(weights [T, topk] f32, indices [T, topk] int64)``.

    ``Gate.forward`` (architecture.py:699-718) for any number of tokens, with a choice limited
    to groups: ``s = score(logit)``, ``sel = s + bias``; of ``n_groups`` groups of neighbouring
    experts the ``topk_groups`` with the largest value stay (``group_score`` "top2": the sum of
    the group's two largest ``sel``, "max": its largest; by default "top2" with a bias and "max"
    without); the ``topk`` largest ``sel`` among them are chosen, in descending order, equal ones
    by ascending index.  ``weights = s / sum(s) * route_scale``, without the division for
    ``renormalize=False`` (the default for softmax, as in Gate).

    Scores are computed in 64 bits, so the order does not depend on how a 32-bit score rounds.  A
    logit (or ``sel``) of -inf masks its expert; a slot that finds no expert has index -1 and
    weight 0, which ``expert_dispatch`` leaves out.  NaN counts as the largest value and shows
    in the weights.  E up to 512, topk up to 16, n_groups up to 32.
    """
    logits = _check("logits", logits, _F32 + _BF16)
    dev = logits.device
    if logits.dim() != 2:
        raise ValueError("logits must be [T, E]")
    t, e = logits.shape
    if score_func not in L.WF_SCORE:
        raise ValueError(f"score_func {score_func!r} is not one of {sorted(L.WF_SCORE)}")
    if bias is not None:
        bias = _check("bias", bias, _F32, dev, (e,))
    if group_score is None:
        group_score = "top2" if bias is not None else "max"
    if group_score not in ("top2", "max"):
        raise ValueError(f"group_score {group_score!r} is not 'top2' or 'max'")
    if topk_groups is None:
        topk_groups = n_groups
    if renormalize is None:
        renormalize = score_func != "softmax"
    if not 1 <= e <= 512:
        raise ValueError(f"{e} experts: 1 to 512 are supported")
    if not 1 <= n_groups <= 32 or e % n_groups or not 1 <= topk_groups <= n_groups:
        raise ValueError(f"n_groups {n_groups} (1 to 32) must divide the {e} experts, topk_groups {topk_groups} lie in it")
    if not 1 <= topk <= min(16, topk_groups * (e // n_groups)):
        raise ValueError(f"topk {topk} must be in 1..min(16, experts of topk_groups groups)")
    w = torch.empty(t, topk, dtype=torch.float32, device=dev)
    i = torch.empty(t, topk, dtype=torch.int64, device=dev)
    if t:
        _run(dev, "wf_route_topk", L.ptr(logits), int(logits.dtype == torch.bfloat16), L.ptr(bias), t, e, topk,
             L.WF_SCORE[score_func], n_groups, topk_groups, int(group_score == "top2"), int(bool(renormalize)),
             float(route_scale), L.ptr(w), L.ptr(i))
    return w, i


def expert_dispatch(indices, n_experts, *, expert_offset=0):
    """The router's choice ``indices [T, k]`` (int64 or int32) as rows in expert order.

    Returns ``(offsets [n_experts + 1], tokens [T * k], slots [T, k])``, all int32: expert ``e``
    (of this rank's ``[expert_offset, expert_offset + n_experts)``) owns rows ``offsets[e]`` to
    ``offsets[e + 1]``, ``tokens`` is each row's token (-1 behind the last row) and ``slots`` each
    pair's row (-1 for an expert that is not this rank's, and for index -1).  Rows are ordered by
    (expert, token, slot).  No host synchronization: ``offsets`` and ``tokens`` are what
    ``grouped_fp8_gemm`` takes, ``slots`` what ``expert_combine`` takes.
    """
    indices = _check("indices", indices, (torch.int64, torch.int32))
    dev = indices.device
    if indices.dim() != 2:
        raise ValueError("indices must be [T, k]")
    t, k = indices.shape
    if not 1 <= k <= 16 or not 1 <= n_experts <= 512 or t * k > 1 << 30:
        raise ValueError(f"indices [{t}, {k}] over {n_experts} experts: k in 1..16, 1 to 512 experts, at most 2^30 pairs")
    if not 0 <= expert_offset <= 0x7fffffff - 512:
        raise ValueError(f"expert_offset {expert_offset} out of range")
    if not t:
        z = torch.zeros(n_experts + 1, dtype=torch.int32, device=dev)
        return z, torch.empty(0, dtype=torch.int32, device=dev), torch.empty(0, k, dtype=torch.int32, device=dev)
    offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=dev)
    tokens = torch.empty(t * k, dtype=torch.int32, device=dev)
    slots = torch.empty(t, k, dtype=torch.int32, device=dev)
    need = L.load().wf_expert_dispatch_workspace_bytes(t, k, n_experts)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _run(dev, "wf_expert_dispatch", L.ptr(indices), int(indices.dtype == torch.int64), t, k, n_experts, expert_offset,
         L.ptr(offsets), L.ptr(tokens), L.ptr(slots), L.ptr(ws), need)
    return offsets, tokens, slots


def grouped_fp8_gemm(a, a_s, w, w_s, offsets, *, rows=None, out=None):
    """Each expert's rows times its own FP8 weights, any number of rows per expert.

    For expert ``e`` and row ``r`` in ``[offsets[e], offsets[e + 1])``::

        out[r] = (a[i] * a_s[i]) @ (w[e] * w_s[e])^T,   i = rows[r] (r without a row list)

    ``a [M, K]`` e4m3 with ``a_s [M, K/128]``, ``w [E, N, K]`` e4m3 with ``w_s [E, ceil(N/128),
    K/128]``, scales f32 or e8m0 (as ``act_quant`` and ``rms_norm_quant`` give them); ``offsets
    [E + 1]`` and ``rows [R]`` int32 on the device, as ``expert_dispatch`` gives them (its
    ``tokens`` gather a token's row for each of its experts, so no permuted copy is made).
    Returns bf16 ``[R, N]`` (``out`` when given); rows behind ``offsets[E]`` are not written.  An
    entry of ``rows`` outside ``[0, M)`` gives a row of zeros.  N a multiple of 8, K of 128.
    """
    a = _check("a", a, _E4M3)
    dev = a.device
    if a.dim() != 2 or w.dim() != 3 or offsets.dim() != 1:
        raise ValueError("a must be [M, K], w [E, N, K] and offsets [E + 1]")
    m, k = a.shape
    e, n, _ = w.shape
    if k == 0 or k % 128 or k > 1 << 20 or n == 0 or n % 8 or n > 1 << 20 or not 1 <= e <= 512 or e * n > 1 << 30:
        raise ValueError(f"E {e}, N {n}, K {k}: E in 1..512, N a multiple of 8, K a multiple of 128 (at most 2^20 each)")
    w = _check("w", w, _E4M3, dev, (e, n, k))
    a_s = _check("a_s", a_s, _F32 + _E8M0, dev, (m, k // 128))
    w_s = _check("w_s", w_s, _F32 + _E8M0, dev, (e, (n + 127) // 128, k // 128))
    offsets = _check("offsets", offsets, (torch.int32,), dev, (e + 1,))
    r = m
    if rows is not None:
        rows = _check("rows", rows, (torch.int32,), dev)
        if rows.dim() != 1:
            raise ValueError("rows must be [R]")
        r = rows.size(0)
    if m > 1 << 30 or r > 1 << 30:
        raise ValueError(f"{m} rows of a, {r} rows: at most 2^30 are supported")
    if out is None:
        out = torch.empty(r, n, dtype=torch.bfloat16, device=dev)
    elif _check("out", out, _BF16, dev, (r, n)) is not out:
        raise ValueError("out must be contiguous")
    if r:
        if not m:
            raise ValueError("a has no rows to take")
        need = L.load().wf_grouped_fp8_workspace_bytes(int(rows is not None), r, e, k)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _run(dev, "wf_grouped_fp8_gemm", L.ptr(a), L.ptr(a_s), _kind(a_s), L.ptr(w), L.ptr(w_s), _kind(w_s),
             L.ptr(offsets), L.ptr(rows), m, r, e, n, k, L.ptr(out), L.ptr(ws), need)
    return out


def grouped_read_error(device=None):
    """Raises if a device wait of ``grouped_fp8_gemm`` on ``device`` ran out since the last read (synchronizes)."""
    with torch.cuda.device(device):
        L.check(L.load().wf_grouped_read_error(L.stream_ptr()), "wf_grouped_read_error")


def expert_combine(rows, slots, *, weights=None, shared=None, out_dtype=torch.bfloat16):
    """Back to token order: ``y[t] = sum_j weights[t, j] * rows[slots[t, j]] (+ shared[t])``.

    ``rows [R, D]`` bf16 (an expert product's output), ``slots [T, k]`` int32 from
    ``expert_dispatch`` (a slot outside ``[0, R)`` adds nothing), ``weights [T, k]`` f32 or None
    for 1, ``shared [T, D]`` bf16 or None.  The sum runs in 32 bits in ascending row order, which
    is ascending expert, as MoE.forward's does (architecture.py:785-794).  ``out_dtype``
    ``torch.float32`` gives a rank's partial sum (``MoELayer.sum_ranks`` adds those).
    """
    rows = _check("rows", rows, _BF16)
    dev = rows.device
    slots = _check("slots", slots, (torch.int32,), dev)
    if rows.dim() != 2 or slots.dim() != 2:
        raise ValueError("rows must be [R, D] and slots [T, k]")
    r, d = rows.shape
    t, k = slots.shape
    if d == 0 or d % 8 or d > 1 << 20 or not 1 <= k <= 16 or r > 0x7fffffff:
        raise ValueError(f"rows [{r}, {d}], slots [{t}, {k}]: D must be a multiple of 8 up to 2^20, k in 1..16")
    if weights is not None:
        weights = _check("weights", weights, _F32, dev, (t, k))
    if shared is not None:
        shared = _check("shared", shared, _BF16, dev, (t, d))
    if out_dtype not in _BF16 + _F32:
        raise TypeError(f"out_dtype {out_dtype} is not bfloat16 or float32")
    y = torch.empty(t, d, dtype=out_dtype, device=dev)
    if t:
        _run(dev, "wf_expert_combine", L.ptr(rows), r, L.ptr(slots), L.ptr(weights), L.ptr(shared), t, k, d, L.ptr(y),
             int(out_dtype == torch.float32))
    return y


OPERATORS = {
    "act_quant": act_quant,
    "fp4_act_quant": fp4_act_quant,
    "fp8_gemm": fp8_gemm,
    "fp4_gemm": fp4_gemm,
}
