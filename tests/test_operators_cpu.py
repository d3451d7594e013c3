"""Refusals of the feed-forward and optimiser entry points: they answer before any
CUDA call, so no GPU is needed (and none sees the bad arguments)."""
from __future__ import annotations

import ctypes as C
import math
import types

import pytest

import zengpu_b200 as zg
from zengpu_b200 import _lib as L

F32, F16, BF16, I32 = 0, 1, 2, 6
FAKE = 0x1000
DISPATCH = zg.api.Dispatch.code


def ff(dtype=BF16, mode=1, act=0, m=4, k=8, f=16, d=8, ptrs=None, pre=(None, None), ws=FAKE,
       nbytes=1 << 20):
    x, wg, wu, wd, y = ptrs or [FAKE] * 5
    return L.load().zg_gated_ff(dtype, mode, act, m, k, f, d, x, wg, wu, wd, y, *pre, ws, nbytes,
                                None)


def ff_backward(ptrs=None, ws=FAKE, nbytes=1 << 20, **kw):
    a = dict(dtype=BF16, mode=1, act=0, m=4, k=8, f=16, d=8) | kw
    return L.load().zg_gated_ff_backward(*a.values(), *(ptrs or [FAKE] * 11), ws, nbytes, None)


def test_gated_ff_refusals():
    for bad in (dict(dtype=I32), dict(act=4), dict(act=-1), dict(dtype=F32, mode=5), dict(m=-1),
                dict(k=0), dict(f=-3), dict(d=0), dict(f=(1 << 28) + 1), dict(ws=None), dict(nbytes=16), dict(ws=FAKE + 8),
                dict(pre=(FAKE, None)), dict(ptrs=[FAKE + 2] + [FAKE] * 4)):
        assert ff(**bad) == DISPATCH, bad
        assert L.last_error(), bad
    for i in range(5):
        assert ff(ptrs=[None if i == j else FAKE for j in range(5)]) == DISPATCH
    assert ff(m=0, ptrs=[None] * 5, ws=None, nbytes=0) == 0  # no rows: nothing to do


def test_gated_ff_backward_refusals():
    for bad in (dict(dtype=I32), dict(act=4), dict(dtype=F32, mode=-1), dict(m=-1), dict(k=0),
                dict(f=0), dict(d=0), dict(ws=None), dict(nbytes=16), dict(ws=FAKE + 8),
                dict(ptrs=[FAKE + 2] + [FAKE] * 10)):
        assert ff_backward(**bad) == DISPATCH, bad
    for i in range(11):
        assert ff_backward([None if i == j else FAKE for j in range(11)]) == DISPATCH


def test_gated_ff_workspace():
    size = L.load().zg_gated_ff_workspace_bytes
    assert size(BF16, 1, 4, 8, 16, 8, 0) > 0
    assert size(BF16, 1, 4, 8, 16, 8, 1) >= size(BF16, 1, 4, 8, 16, 8, 0)
    assert size(BF16, 1, 0, 8, 16, 8, 0) == 0 and size(I32, 1, 4, 8, 16, 8, 0) == 0


def adamw(param=F32, grad=F32, bits=32, count=1, tensors=None, hyper=None, **kw):
    t = (L.AdamWTensor * 1)()
    t[0].n = 8
    for name in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
        setattr(t[0], name, FAKE)
    for name, v in (tensors or {}).items():
        setattr(t[0], name, v)
    h = L.AdamWHyper(*((dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, step=1)
                        | (hyper or {})).values()))
    return L.load().zg_adamw(param, grad, bits, count, t, C.byref(h), None, None, None, None)


def test_adamw_refusals():
    for bad in (dict(param=I32), dict(grad=I32), dict(bits=16), dict(hyper=dict(beta1=1.0)),
                dict(hyper=dict(beta2=-0.5)), dict(hyper=dict(beta1=math.nan)),
                dict(hyper=dict(eps=-1.0)), dict(hyper=dict(lr=math.inf)), dict(hyper=dict(step=0)),
                dict(hyper=dict(weight_decay=math.nan)), dict(tensors=dict(param=None)),
                dict(tensors=dict(grad=None)), dict(tensors=dict(exp_avg=None)),
                dict(tensors=dict(exp_avg_sq=None)), dict(bits=8, tensors=dict(exp_avg_scale=None)),
                dict(tensors=dict(master=FAKE)), dict(tensors=dict(n=1 << 40)),
                dict(tensors=dict(param=FAKE + 2)), dict(tensors=dict(exp_avg=FAKE + 1))):
        assert adamw(**bad) == DISPATCH, bad
    assert adamw(count=0) == 0 and adamw(tensors=dict(n=0, param=None)) == 0


def test_grad_norm_refusals():
    lib = L.load()
    need = lib.zg_grad_norm_workspace_bytes(1)
    def call(dtype=F32, ptr=FAKE, n=8, most=1.0, out=FAKE, ws=FAKE, nbytes=need):
        return lib.zg_grad_norm(dtype, 1, (C.c_void_p * 1)(ptr), (C.c_uint64 * 1)(n), most, out, ws,
                                nbytes, None)
    for bad in (dict(dtype=I32), dict(ptr=None), dict(ptr=FAKE + 2), dict(n=1 << 40),
                dict(most=0.0), dict(most=math.nan), dict(out=None), dict(ws=None),
                dict(nbytes=need - 1), dict(ws=FAKE + 4)):
        assert call(**bad) == DISPATCH, bad


def test_python_refuses_cpu_tensors():
    import torch

    from zengpu_b200 import kernels as K
    x = torch.zeros(2, 4)
    with pytest.raises(ValueError):
        K.gated_ff(x, torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(6, 4))
    with pytest.raises(ValueError, match="exceed"):
        K._ff_sizes(types.SimpleNamespace(is_cuda=True, dtype=torch.bfloat16, shape=(1 << 33, 4),
                                          dim=lambda: 2), torch.zeros(4, 6), torch.zeros(6, 4))
    with pytest.raises(ValueError):
        K.AdamW([x], [x.clone()])
    with pytest.raises(ValueError):
        K.AdamW([], [])
    with pytest.raises(ValueError):
        K.GradNorm([x])
