"""Refusals of the transformer-block operators (layer norm, 8-bit linear
layers, rotary positions): every call here is turned down by the host's
checks, before any launch, so no GPU is needed.  The pointers are made up and
never read."""
import ctypes as C

import pytest
import torch

import ppdl

P = 1 << 20  # an aligned address that nothing dereferences


def L():
    return ppdl.lib()


def ln(**kw):
    a = dict(x=P, ldx=8, res=None, ldres=0, w=P, b=P, type=0, wt=0, rows=4, D=8, eps=1e-5, y=P,
             ldy=8, sum=None, lds=0, mean=None, rstd=None)
    a.update(kw)
    return L().ppdl_layernorm(*a.values(), None)


def ln_bwd(**kw):
    a = dict(dy=P, lddy=8, x=P, ldx=8, w=P, mean=P, rstd=P, dsum=None, ldds=0, type=0, wt=0, rows=4,
             D=8, dx=P, lddx=8, dw=P, db=P, work=P)
    a.update(kw)
    return L().ppdl_layernorm_backward(*a.values(), None)


def quant(**kw):
    a = dict(x=P, ldx=8, type=0, rows=4, K=8, q=P, ldq=16, scale=P)
    a.update(kw)
    return L().ppdl_quantize_rows_i8(*a.values(), None)


def linear(**kw):
    a = dict(q=P, ldq=16, qs=P, w=P, ldw=16, ws=P, bias=None, res=None, ldres=0, type=0, act=0, M=4,
             N=4, K=16, y=P, ldy=4)
    a.update(kw)
    return L().ppdl_linear_i8(*a.values(), None)


def dynamic(**kw):
    a = dict(x=P, ldx=16, xt=0, w=P, ldw=16, ws=P, bias=None, res=None, ldres=0, type=0, act=0, M=4,
             N=4, K=16, y=P, ldy=4, work=P)
    a.update(kw)
    return L().ppdl_linear_i8_dynamic(*a.values(), None)


def rotary(heads=None, sections=(4,), **kw):
    h = dict(in_=P, out=P, heads=2, in_batch=64, in_token=16, in_head=8, out_batch=64, out_token=16,
             out_head=8)
    h.update(heads or {})
    q = ppdl.RotaryHeads(*h.values())
    a = dict(q=C.byref(q), k=None, type=0, batch=1, length=4, dim=8, rotated=8, pos=P, pb=8, ps=4,
             pbs=4, pts=1, axes=len(sections), sections=(C.c_int32 * 8)(*sections), freq=P, il=0,
             inv=0)
    a.update(kw)
    return L().ppdl_rotary(*a.values(), None)


@pytest.mark.parametrize("call,bad", [
    (ln, dict(type=3)), (ln, dict(type=-1)), (ln, dict(type=1, wt=2)), (ln, dict(wt=1)),
    (ln, dict(rows=-1)), (ln, dict(D=0)), (ln, dict(D=-8)), (ln, dict(eps=-1e-5)),
    (ln, dict(eps=float("nan"))), (ln, dict(eps=float("inf"))), (ln, dict(x=None)),
    (ln, dict(y=None)), (ln, dict(ldx=7)), (ln, dict(ldy=0)), (ln, dict(sum=P, lds=8)),
    (ln, dict(res=P, ldres=4)), (ln, dict(x=P + 2)), (ln, dict(w=P + 1)), (ln, dict(mean=P + 2)),
    (ln_bwd, dict(type=5)), (ln_bwd, dict(mean=None)), (ln_bwd, dict(rstd=None)),
    (ln_bwd, dict(dx=None)), (ln_bwd, dict(work=None)), (ln_bwd, dict(work=P + 4)),
    (ln_bwd, dict(lddx=4)), (ln_bwd, dict(dsum=P, ldds=4)), (ln_bwd, dict(rows=-2)),
    (ln_bwd, dict(dw=P + 2)),
    (quant, dict(type=9)), (quant, dict(K=0)), (quant, dict(rows=-1)), (quant, dict(x=None)),
    (quant, dict(q=None)), (quant, dict(scale=None)), (quant, dict(q=P + 8)), (quant, dict(ldq=8)),
    (quant, dict(ldq=24)), (quant, dict(K=17, ldx=17, ldq=16)), (quant, dict(ldx=4)),
    (linear, dict(act=4)), (linear, dict(act=-1)), (linear, dict(type=3)), (linear, dict(K=0)),
    (linear, dict(K=131072, ldq=131072, ldw=131072)), (linear, dict(N=0)), (linear, dict(M=-1)),
    (linear, dict(q=None)), (linear, dict(w=None)), (linear, dict(qs=None)), (linear, dict(ws=None)),
    (linear, dict(y=None)), (linear, dict(ldq=8)), (linear, dict(ldw=20)), (linear, dict(q=P + 1)),
    (linear, dict(w=P + 8)), (linear, dict(ldy=3)), (linear, dict(res=P, ldres=3)),
    (linear, dict(bias=P + 2)), (linear, dict(K=17)),
    (dynamic, dict(x=None)), (dynamic, dict(xt=7)), (dynamic, dict(ldx=8)), (dynamic, dict(x=P + 2)),
    (dynamic, dict(work=None)), (dynamic, dict(work=P + 8)), (dynamic, dict(M=-1)), (dynamic, dict(K=0)),
    (dynamic, dict(w=None)), (dynamic, dict(act=9)), (dynamic, dict(ldy=2)), (dynamic, dict(type=5)),
    (rotary, dict(type=3)), (rotary, dict(dim=0)), (rotary, dict(dim=1025)), (rotary, dict(rotated=7)),
    (rotary, dict(rotated=0, sections=(0,))), (rotary, dict(rotated=10, sections=(5,))),
    (rotary, dict(sections=(3,))), (rotary, dict(sections=(5, -1))),
    (rotary, dict(sections=(1, 1, 1, 1, 0))), (rotary, dict(axes=0)), (rotary, dict(pb=2)),
    (rotary, dict(pos=None)), (rotary, dict(pos=P + 4)), (rotary, dict(freq=None)),
    (rotary, dict(freq=P + 4)), (rotary, dict(batch=-1)), (rotary, dict(length=-1)),
    (rotary, dict(heads=dict(heads=-1))), (rotary, dict(heads=dict(heads=65536))), (rotary, dict(heads=dict(in_=None))),
    (rotary, dict(heads=dict(out=None))), (rotary, dict(heads=dict(in_=P + 2))),
])
def test_refused(call, bad):
    assert call(**bad) == ppdl.PPDL_ERR_SHAPE
    assert ppdl.last_error()


@pytest.mark.parametrize("call,none", [(ln, dict(rows=0)), (quant, dict(rows=0)),
                                       (linear, dict(M=0)), (dynamic, dict(M=0, work=None)),
                                       (rotary, dict(batch=0)),
                                       (rotary, dict(length=0)),
                                       (ln_bwd, dict(rows=0, dw=None, db=None))])
def test_nothing_to_do(call, none):
    """No rows or tokens: nothing is launched and the call succeeds."""
    assert call(**none) == ppdl.PPDL_OK


def test_backward_workspace_size():
    f = L().ppdl_layernorm_backward_workspace
    assert f(0, 8) == 0 and f(8, 0) == 0 and f(-1, 8) == 0
    assert f(1, 8) >= 16 and f(1 << 20, 4096) >= 2 * 4096


def test_dynamic_workspace_size():
    f = L().ppdl_linear_i8_dynamic_workspace
    assert f(0, 8) == 0 and f(8, 0) == 0
    assert f(3, 17) == 3 * 32 + 12 and f(1 << 20, 131071) == (131072 + 4) << 20


def rejects(f, *args, **kw):
    with pytest.raises(ValueError):
        f(*args, **kw)


def test_python_refusals():
    x, w = torch.zeros(4, 8), torch.ones(8)
    rejects(ppdl.layernorm, x, w, w)                     # not on a GPU
    rejects(ppdl.layernorm, x.double(), w, w)
    rejects(ppdl.layernorm, x.t(), w, w)
    rejects(ppdl.layernorm, x, w[:4], w)
    rejects(ppdl.layernorm, x, w, w.bfloat16())
    rejects(ppdl.layernorm, x, w, w, residual=x[:2])
    rejects(ppdl.layernorm, x, w, w, residual=x.bfloat16())
    rejects(ppdl.layernorm, x, w, w, return_sum=True)
    s = torch.zeros(4)
    rejects(ppdl.layernorm_backward, x, x, w, s, s)      # not on a GPU
    rejects(ppdl.layernorm_backward, x.half(), x, w, s, s)
    rejects(ppdl.layernorm_backward, x, x, w, s[:3], s)
    rejects(ppdl.layernorm_backward, x, x, w, s, s.double())
    q, qs = torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)
    rejects(ppdl.quantize_rows, q)
    rejects(ppdl.linear_i8, q, q, qs)                    # int8 x without its scale
    rejects(ppdl.linear_i8, torch.zeros(4, 16), q, qs, x_scale=qs)
    rejects(ppdl.linear_i8, torch.zeros(4, 8), q, qs)
    rejects(ppdl.linear_i8, torch.zeros(4, 16), q.float(), qs)
    rejects(ppdl.linear_i8, torch.zeros(4, 16), q, qs, act="tanh")
    rejects(ppdl.linear_i8, torch.zeros(4, 16), q, qs, bias=torch.zeros(4, dtype=torch.float16))
    rejects(ppdl.linear_i8, torch.zeros(4, 16), q, qs, residual=torch.zeros(4, 5))
    h, pos, f = torch.zeros(2, 3, 2, 8), torch.zeros(2, 2, 3, dtype=torch.int64), torch.ones(4).double()
    rejects(ppdl.rotary, h, h, pos, f, (2, 2))           # not on a GPU
    rejects(ppdl.rotary, h, h, pos, f, (4,))
    rejects(ppdl.rotary, h, h, pos.float(), f, (2, 2))
    rejects(ppdl.rotary, h, h, pos, f.float(), (2, 2))
    rejects(ppdl.rotary, h, h.half(), pos, f, (2, 2))
    rejects(ppdl.rotary, h, h[:, :2], pos, f, (2, 2))
