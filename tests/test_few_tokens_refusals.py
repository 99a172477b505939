"""What the few-token NVFP4 entry points refuse, checked through the C ABI
without a GPU: every argument check comes before the first device call."""
from __future__ import annotations

import ctypes

import pytest

BAD_ARG, OK = 1, 0
PTR = 1 << 20  # never dereferenced: these calls end in an argument check


def _gemv(gplk, **kw):
    a = dict(X=PTR, W=PTR, SF=PTR, Y=2 * PTR, R=None, T=1, N=128, K=256, ldx=256, ldy=128, ldr=0, alpha=PTR, dtype=0, workspace=None,
             workspace_bytes=0)
    a.update(kw)
    return gplk.lib().gplk_gemv_nvfp4(*a.values(), None)


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(T=33), dict(N=-1), dict(K=-64), dict(K=0), dict(K=32), dict(K=100), dict(dtype=2), dict(dtype=-1),
    dict(ldx=255), dict(ldy=127), dict(R=PTR, ldr=127), dict(X=None), dict(W=None), dict(SF=None), dict(Y=None),
    dict(alpha=None), dict(W=PTR + 8), dict(SF=PTR + 4), dict(X=PTR + 1), dict(Y=PTR + 1), dict(X=PTR, Y=PTR), dict(R=PTR + 1, ldr=128),
    dict(alpha=PTR + 2), dict(workspace=PTR + 8)])
def test_gemv_refuses(kw, gplk):
    assert _gemv(gplk, **kw) == BAD_ARG


@pytest.mark.parametrize("kw", [dict(T=0), dict(N=0), dict(T=0, X=None, Y=None)])
def test_gemv_empty_is_ok(kw, gplk):
    assert _gemv(gplk, **kw) == OK


def _moe(gplk, **kw):
    c = gplk.MoeCfg()
    for name in ("x", "router", "gate", "up", "down", "sf_gate", "sf_up", "sf_down", "alpha_gate", "alpha_up",
                 "alpha_down", "y", "workspace"):
        setattr(c, name, PTR)
    c.T, c.E, c.top, c.D, c.F, c.ldx, c.ldy, c.renormalise, c.dtype = 2, 8, 2, 256, 128, 256, 256, 1, 0
    c.workspace_bytes = gplk.moe_nvfp4_workspace_bytes(2, 8, 2, 256, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return gplk.lib().gplk_moe_nvfp4(ctypes.byref(c), None)


@pytest.mark.parametrize("kw", [
    dict(T=-1), dict(T=33), dict(E=0), dict(E=513), dict(top=0), dict(top=9), dict(top=17, E=64), dict(D=0),
    dict(D=32), dict(D=257), dict(F=0), dict(F=96), dict(ldx=255), dict(ldy=255), dict(dtype=2),
    dict(workspace_bytes=0), dict(workspace=None), dict(workspace=PTR + 8), dict(E=512, F=1 << 23, T=1, top=1),
    *[{n: None} for n in ("x", "router", "gate", "up", "down", "sf_gate", "sf_up", "sf_down", "alpha_gate",
                          "alpha_up", "alpha_down", "y")],
    *[{n: PTR + 8} for n in ("gate", "up", "down", "sf_gate", "sf_up", "sf_down")],
    *[{n: PTR + 2} for n in ("alpha_gate", "alpha_up", "alpha_down", "ids", "weights")],
    dict(x=PTR + 1), dict(y=PTR + 1), dict(router=PTR + 1)])
def test_moe_refuses(kw, gplk):
    assert _moe(gplk, **kw) == BAD_ARG


def test_moe_refuses_a_workspace_one_byte_short(gplk):
    assert _moe(gplk, workspace_bytes=gplk.moe_nvfp4_workspace_bytes(2, 8, 2, 256, 128) - 1) == BAD_ARG


def test_moe_null_and_empty(gplk):
    assert gplk.lib().gplk_moe_nvfp4(None, None) == BAD_ARG
    assert _moe(gplk, T=0, x=None, y=None, workspace=None, workspace_bytes=0) == OK


def test_moe_workspace_bytes(gplk):
    ws = gplk.moe_nvfp4_workspace_bytes
    assert ws(2, 8, 2, 256, 128) > 0
    for bad in ((0, 8, 2, 256, 128), (33, 8, 2, 256, 128), (2, 0, 2, 256, 128), (2, 513, 2, 256, 128),
                (2, 8, 9, 256, 128), (2, 8, 0, 256, 128), (2, 8, 2, 0, 128), (2, 8, 2, 256, 0)):
        assert ws(*bad) == 0
    assert ws(32, 64, 8, 4096, 2048) >= 32 * 8 * 2048 * 4


@pytest.mark.parametrize("sizes", [
    (2, 8, 2, 100, 128), (2, 8, 2, 128, 100), (2, 8, 2, 32, 64), (2, 8, 2, 64, 32), (2, 512, 2, 1 << 20, 64),
    (2, 512, 2, 64, 1 << 20), (-1, 8, 2, 64, 64), (2, 8, 17, 64, 64)])
def test_moe_workspace_is_zero_where_the_call_refuses(sizes, gplk):
    T, E, top, D, F = sizes
    assert _moe(gplk, T=T, E=E, top=top, D=D, F=F, ldx=D, ldy=D, workspace_bytes=1 << 60) == BAD_ARG
    assert gplk.moe_nvfp4_workspace_bytes(*sizes) == 0


def test_python_wrappers_refuse_cpu_tensors(gplk):
    import torch

    x = torch.zeros(1, 64, dtype=torch.bfloat16)
    w, sf = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(512, dtype=torch.uint8)
    with pytest.raises(gplk.GplkError):
        gplk.gemv_nvfp4(x, w, sf, torch.zeros(1, 8, dtype=torch.bfloat16), torch.ones(1))
    m = (torch.zeros(4, 64, 32, dtype=torch.uint8), torch.zeros(4, 512, dtype=torch.uint8), torch.ones(4))
    with pytest.raises(gplk.GplkError):
        gplk.moe_nvfp4(x, torch.zeros(4, 64, dtype=torch.bfloat16), m, m, m, torch.zeros_like(x),
                       torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 2))
