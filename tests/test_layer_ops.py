"""Refusals of the operators around a routed expert layer: every check precedes any launch (no GPU needed)."""

import ctypes

import pytest
import torch

from wanferenz_b200 import _lib as L
from wanferenz_b200 import ops

P = ctypes.c_void_p(4096)  # never dereferenced
ODD = ctypes.c_void_p(4097)
F32, E8M0 = L.WF_SCALE_F32, L.WF_SCALE_E8M0


def _norm(x=P, res=None, w=P, wb=0, T=2, D=256, ue=0, q=P, s=P, kind=F32, y=None, h=None):
    return L.load().wf_rms_norm_quant(x, res, w, wb, T, D, 1e-6, ue, q, s, kind, y, h, None)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), L.WF_E_ARG), (dict(w=None), L.WF_E_ARG), (dict(q=None), L.WF_E_ARG), (dict(s=None), L.WF_E_ARG),
    (dict(res=P), L.WF_E_ARG), (dict(h=P), L.WF_E_ARG),
    (dict(T=0), L.WF_E_SHAPE), (dict(T=1 << 31), L.WF_E_SHAPE),
    (dict(D=0), L.WF_E_SHAPE), (dict(D=192), L.WF_E_SHAPE), (dict(D=16512), L.WF_E_SHAPE),
    (dict(kind=7), L.WF_E_DTYPE), (dict(kind=E8M0, ue=0), L.WF_E_DTYPE),
    (dict(x=ODD), L.WF_E_ARG), (dict(y=ODD), L.WF_E_ARG), (dict(w=ODD), L.WF_E_ARG)])
def test_rms_norm_quant_refuses(kw, code):
    assert _norm(**kw) == code
    assert L.load().wf_last_error()


def _route(l=P, bf16=0, bias=None, T=2, E=64, k=6, score=1, G=1, keep=1, top2=1, w=P, i=P):
    return L.load().wf_route_topk(l, bf16, bias, T, E, k, score, G, keep, top2, 1, 1.0, w, i, None)


@pytest.mark.parametrize("kw,code", [
    (dict(l=None), L.WF_E_ARG), (dict(w=None), L.WF_E_ARG), (dict(i=None), L.WF_E_ARG),
    (dict(T=0), L.WF_E_SHAPE), (dict(E=0), L.WF_E_SHAPE), (dict(E=513), L.WF_E_SHAPE),
    (dict(k=0), L.WF_E_SHAPE), (dict(k=17), L.WF_E_SHAPE), (dict(E=4, k=5), L.WF_E_SHAPE),
    (dict(score=3), L.WF_E_DTYPE), (dict(score=-1), L.WF_E_DTYPE),
    (dict(G=0), L.WF_E_SHAPE), (dict(G=7), L.WF_E_SHAPE), (dict(G=64, E=512), L.WF_E_SHAPE),
    (dict(G=8, keep=0), L.WF_E_SHAPE), (dict(G=8, keep=9), L.WF_E_SHAPE),
    (dict(G=16, keep=1, k=6), L.WF_E_SHAPE),  # 4 experts a group
    (dict(l=ODD), L.WF_E_ARG), (dict(i=ctypes.c_void_p(4100)), L.WF_E_ARG)])
def test_route_topk_refuses(kw, code):
    assert _route(**kw) == code


def _dispatch(ind=P, T=4, k=6, E=64, base=0, ws=P, n=1 << 20, off=P, tok=P, slots=P):
    return L.load().wf_expert_dispatch(ind, 1, T, k, E, base, off, tok, slots, ws, n, None)


@pytest.mark.parametrize("kw,code", [
    (dict(ind=None), L.WF_E_ARG), (dict(ws=None, T=4096), L.WF_E_ARG), (dict(off=None), L.WF_E_ARG),
    (dict(T=0), L.WF_E_SHAPE), (dict(k=0), L.WF_E_SHAPE), (dict(k=17), L.WF_E_SHAPE), (dict(E=0), L.WF_E_SHAPE),
    (dict(E=513), L.WF_E_SHAPE), (dict(T=1 << 30, k=2), L.WF_E_SHAPE), (dict(T=1 << 62, k=8), L.WF_E_SHAPE),
    (dict(base=-1), L.WF_E_SHAPE), (dict(base=1 << 31), L.WF_E_SHAPE),
    (dict(T=4096, n=64), L.WF_E_ARG), (dict(ind=ctypes.c_void_p(4100)), L.WF_E_ARG), (dict(tok=ODD), L.WF_E_ARG)])
def test_expert_dispatch_refuses(kw, code):
    assert _dispatch(**kw) == code


def test_expert_dispatch_workspace_is_bounded():
    f = L.load().wf_expert_dispatch_workspace_bytes
    assert 0 == f(1, 1, 1) < f(1 << 12, 8, 256) <= f(1 << 26, 16, 512) <= 512 * 512 * 4
    assert f(0, 1, 1) == 0 and f(1, 17, 1) == 0 and f(1, 1, 513) == 0


def _combine(rows=P, R=12, slots=P, w=None, sh=None, T=2, k=6, D=256, y=P):
    return L.load().wf_expert_combine(rows, R, slots, w, sh, T, k, D, y, 0, None)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=None), L.WF_E_ARG), (dict(slots=None), L.WF_E_ARG), (dict(y=None), L.WF_E_ARG),
    (dict(R=-1), L.WF_E_SHAPE), (dict(R=1 << 31), L.WF_E_SHAPE), (dict(T=0), L.WF_E_SHAPE),
    (dict(k=0), L.WF_E_SHAPE), (dict(k=17), L.WF_E_SHAPE), (dict(D=0), L.WF_E_SHAPE), (dict(D=12), L.WF_E_SHAPE),
    (dict(rows=ctypes.c_void_p(4104)), L.WF_E_ARG), (dict(sh=ctypes.c_void_p(4104)), L.WF_E_ARG),
    (dict(y=ODD), L.WF_E_ARG)])
def test_expert_combine_refuses(kw, code):
    assert _combine(**kw) == code


def test_operators_take_cuda_tensors_only():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rms_norm_quant(x, torch.ones(256))
    with pytest.raises(ValueError, match="CUDA"):
        ops.route_topk(torch.zeros(2, 64), 6)
    with pytest.raises(ValueError, match="CUDA"):
        ops.expert_dispatch(torch.zeros(2, 6, dtype=torch.int64), 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.expert_combine(x, torch.zeros(2, 1, dtype=torch.int32))


def _grouped(a=P, a_s=P, ak=F32, w=P, w_s=P, wk=F32, off=P, rows=P, M=8, R=12, E=4, N=256, K=256, out=P, ws=None, n=0):
    return L.load().wf_grouped_fp8_gemm(a, a_s, ak, w, w_s, wk, off, rows, M, R, E, N, K, out, ws, n, None)


@pytest.mark.parametrize("kw,code", [
    (dict(a=None), L.WF_E_ARG), (dict(a_s=None), L.WF_E_ARG), (dict(w=None), L.WF_E_ARG), (dict(w_s=None), L.WF_E_ARG),
    (dict(off=None), L.WF_E_ARG), (dict(out=None), L.WF_E_ARG), (dict(ak=2), L.WF_E_DTYPE), (dict(wk=-1), L.WF_E_DTYPE),
    (dict(M=0), L.WF_E_SHAPE), (dict(R=0), L.WF_E_SHAPE), (dict(R=1 << 31), L.WF_E_SHAPE), (dict(rows=None), L.WF_E_SHAPE),
    (dict(E=0), L.WF_E_SHAPE), (dict(E=513), L.WF_E_SHAPE), (dict(N=0), L.WF_E_SHAPE), (dict(N=12), L.WF_E_SHAPE),
    (dict(E=512, N=1 << 22), L.WF_E_SHAPE), (dict(K=0), L.WF_E_SHAPE), (dict(K=192), L.WF_E_SHAPE),
    (dict(R=1024), L.WF_E_ARG), (dict(R=1024, ws=P, n=1024 * 256 - 1), L.WF_E_ARG), (dict(R=1024, ws=ODD, n=1 << 20), L.WF_E_ARG),
    (dict(a=ctypes.c_void_p(4104)), L.WF_E_ARG), (dict(w=ctypes.c_void_p(4104)), L.WF_E_ARG),
    (dict(out=ctypes.c_void_p(4104)), L.WF_E_ARG), (dict(a_s=ODD), L.WF_E_ARG), (dict(rows=ODD), L.WF_E_ARG)])
def test_grouped_fp8_gemm_refuses(kw, code):
    assert _grouped(**kw) == code


AT = {"a": 1 << 40, "a_s": 2 << 40, "w": 3 << 40, "w_s": 4 << 40, "off": 5 << 40, "rows": 6 << 40, "ws": 7 << 40}


@pytest.mark.parametrize("name,size", [("a", 8 * 256), ("a_s", 8 * 2 * 4), ("w", 4 * 256 * 256), ("w_s", 4 * 2 * 2 * 4),
                                       ("off", 5 * 4), ("rows", 1024 * 4), ("ws", 1024 * 256)])
@pytest.mark.parametrize("side", ["front", "end"])
def test_grouped_fp8_gemm_refuses_an_output_over_an_input(name, size, side):
    """Other rows' results would be read as inputs; a workspace over an input is the same."""
    ptr = {k: ctypes.c_void_p(v) for k, v in AT.items()}
    out = AT[name] - 1024 * 256 * 2 + 16 if side == "front" else AT[name] + (size - 1) // 16 * 16
    kw = dict(R=1024, n=1024 * 256, **ptr)
    assert _grouped(out=ctypes.c_void_p(out), **kw) == L.WF_E_ARG
    assert b"overlap" in L.load().wf_last_error()
    if name != "ws":
        kw["ws"] = ctypes.c_void_p(AT[name] - 1024 * 256 + 16 if side == "front" else AT[name] + (size - 1) // 16 * 16)
        assert _grouped(out=ctypes.c_void_p(8 << 40), **kw) == L.WF_E_ARG
        assert b"overlap" in L.load().wf_last_error()
