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
current stream, keep nothing between calls, and have no gradients.  An input that is
not contiguous, or starts off a 16-byte boundary, is copied first, on every call: keep
weights contiguous.

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


_EXT = None


def _ext():
    global _EXT
    if _EXT is None:
        _EXT = L.load_ext()
    return _EXT


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
    return NormQuant._make(_ext().rms_norm_quant(x, weight, eps, residual, norm_out, scale_fmt is not None, scale_dtype))


def route_topk(logits, topk, *, bias=None, score_func="sigmoid", n_groups=1, topk_groups=None, group_score=None,
               renormalize=None, route_scale=1.0):
    """Expert choice from router logits ``[T, E]`` (f32 or bf16): ``(weights [T, topk] f32, indices [T, topk] int64)``.

    ``Gate.forward`` (architecture.py:699-718) for any number of tokens, with a choice limited
    to groups: ``s = score(logit)``, ``sel = s + bias``; of ``n_groups`` groups of neighbouring
    experts the ``topk_groups`` with the largest value stay (``group_score`` "top2": the sum of
    the group's two largest ``sel``, or the one that is not masked, "max": its largest; by default
    "top2" with a bias and "max" without); the ``topk`` largest ``sel`` among them are chosen, in descending order, equal ones
    by ascending index.  ``weights = s / sum(s) * route_scale``, without the division for
    ``renormalize=False`` (the default for softmax, as in Gate).

    Scores are computed in 64 bits, so the order does not depend on how a 32-bit score rounds.  A
    logit (or ``sel``) of -inf masks its expert; a slot that finds no expert has index -1 and
    weight 0, which ``expert_dispatch`` leaves out.  NaN counts as the largest value and shows
    in the weights.  E up to 512, topk up to 16, n_groups up to 32.
    """
    if score_func not in L.WF_SCORE:
        raise ValueError(f"score_func {score_func!r} is not one of {sorted(L.WF_SCORE)}")
    if group_score is None:
        group_score = "max" if bias is None else "top2"
    elif group_score not in ("top2", "max"):
        raise ValueError(f"group_score {group_score!r} is not 'top2' or 'max'")
    return _ext().route_topk(logits, topk, bias, L.WF_SCORE[score_func], n_groups,
                             n_groups if topk_groups is None else topk_groups, group_score == "top2",
                             score_func != "softmax" if renormalize is None else renormalize, route_scale)


def expert_dispatch(indices, n_experts, *, expert_offset=0):
    """The router's choice ``indices [T, k]`` (int64 or int32) as rows in expert order.

    Returns ``(offsets [n_experts + 1], tokens [T * k], slots [T, k])``, all int32: expert ``e``
    (of this rank's ``[expert_offset, expert_offset + n_experts)``) owns rows ``offsets[e]`` to
    ``offsets[e + 1]``, ``tokens`` is each row's token (-1 behind the last row) and ``slots`` each
    pair's row (-1 for an expert that is not this rank's, and for index -1).  Rows are ordered by
    (expert, token, slot).  No host synchronization: ``offsets`` and ``tokens`` are what
    ``grouped_fp8_gemm`` takes, ``slots`` what ``expert_combine`` takes.
    """
    return _ext().expert_dispatch(indices, n_experts, expert_offset)


def grouped_fp8_gemm(a, a_s, w, w_s, offsets, *, rows=None, out=None):
    """Each expert's rows times its own FP8 weights, any number of rows per expert.

    For expert ``e`` and row ``r`` in ``[offsets[e], offsets[e + 1])``::

        out[r] = (a[i] * a_s[i]) @ (w[e] * w_s[e])^T,   i = rows[r] (r without a row list)

    ``a [M, K]`` e4m3 with ``a_s [M, K/128]``, ``w [E, N, K]`` e4m3 with ``w_s [E, ceil(N/128),
    K/128]``, scales f32 or e8m0 (as ``act_quant`` and ``rms_norm_quant`` give them); ``offsets
    [E + 1]`` and ``rows [R]`` int32 on the device, as ``expert_dispatch`` gives them (its
    ``tokens`` gather a token's row for each of its experts, so no permuted copy is made).
    Returns bf16 ``[R, N]`` (``out`` when given, which must not overlap an input); rows behind
    ``offsets[E]`` are not written.  An entry of ``rows`` outside ``[0, M)`` gives a row of zeros.
    N a multiple of 8, K of 128.  With f32 scales the product of a row's and a block's scale is a
    32-bit value, and must not overflow or fall below the normal range.

    Tiles, workspace and output go by ``R``, all rows of the list.  With the experts split over
    ranks most of ``expert_dispatch``'s list belongs to no local expert: the result is right, the
    tiles are wider than the local rows need.  A program that knows a bound of at least
    ``offsets[E]`` passes ``rows=tokens[:bound]``.
    """
    return _ext().grouped_fp8_gemm(a, a_s, w, w_s, offsets, rows, out)


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
    return _ext().expert_combine(rows, slots, weights, shared, out_dtype)


OPERATORS = {
    "act_quant": act_quant,
    "fp4_act_quant": fp4_act_quant,
    "fp8_gemm": fp8_gemm,
    "fp4_gemm": fp4_gemm,
}
