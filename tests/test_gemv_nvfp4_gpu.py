"""gplk_gemv_nvfp4 (a few tokens against NVFP4 weights) against the product in
64 bits on the same codes, scale bytes and activations, within the bound that
nvfp4_reference.product_error derives plus half a step of the output type."""
from __future__ import annotations

import pytest

import nvfp4_reference as ref

pytestmark = pytest.mark.gpu


def _gen(cuda, seed):
    import torch

    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _check(gplk, cuda, t, n, k, dtype="bf16", residual=None, pad=0, seed=0, x=None, alpha=0.0123, pad_byte=0x7F,
           **kw):
    import torch

    gen = _gen(cuda, seed + 7 * t + 31 * n + k)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    w, sf, wd = ref.random_weights(n, k, gen, cuda, pad_byte)
    al = torch.tensor([alpha], dtype=torch.float32, device=cuda)
    if x is None:
        x = torch.randn(t, k + pad, device=cuda, generator=gen).to(dt)[:, :k]
    else:
        x = x.to(dt)
    buf = torch.full((t, n + pad), 7.0, dtype=dt, device=cuda)
    y, r = buf[:, :n], None
    want = float(al) * (x.double() @ wd.T)
    err = ref.product_error(wd, x, float(al)) + 2 * 2.0 ** -24 * want.abs()
    if residual == "apart":
        r = torch.randn(t, n + 3, device=cuda, generator=gen).to(dt)[:, :n]
    elif residual == "inplace":
        y.copy_(torch.randn(t, n, device=cuda, generator=gen))
        r = y
    if r is not None:
        want = want + r.double()
        err = err + 2.0 ** -24 * want.abs()
    gplk.gemv_nvfp4(x, w, sf, y, al, residual=r, **kw)
    torch.cuda.synchronize()
    got = y.double()
    assert torch.isfinite(got).all()
    # The computed value is within err of `want`; rounding it is off by half a step at that value.
    tol = err + ref.rounding(want.abs() + err, dt)
    off = (got - want).abs()
    assert bool((off <= tol).all()), (t, n, k, float((off / tol).max()))
    if pad:
        assert bool((buf[:, n:] == 7.0).all()), "columns beyond N were written"
    return y


@pytest.mark.parametrize("t", [1, 2, 3, 5, 8, 13, 16, 25, 26, 31, 32])
def test_tokens(t, gplk, cuda):
    _check(gplk, cuda, t, 300, 1088)


@pytest.mark.parametrize("n", [1, 7, 127, 128, 129, 255, 1000, 4097])
@pytest.mark.parametrize("t", [1, 4])
def test_odd_outputs(t, n, gplk, cuda):
    _check(gplk, cuda, t, n, 512, pad=5)


@pytest.mark.parametrize("k", [64, 128, 192, 256, 320, 576, 1024, 2112, 4160, 16384])
@pytest.mark.parametrize("t", [1, 9])
def test_depths(t, k, gplk, cuda):
    _check(gplk, cuda, t, 200, k)


@pytest.mark.parametrize("tnk", [(4, 700, 8192), (8, 129, 8256), (17, 1000, 4160), (25, 128, 16384), (26, 300, 8192),
                                 (32, 130, 16448), (32, 9000, 1088), (7, 20000, 1600)])
@pytest.mark.parametrize("workspace", ["auto", None])
def test_converted_ahead_or_by_every_block(tnk, workspace, gplk, cuda):
    """Sizes about and above where activations are converted ahead of the
    products, and the same without the workspace that this takes."""
    _check(gplk, cuda, *tnk, workspace=workspace, residual="apart", pad=3)


def test_workspace_of_any_content_and_size(gplk, cuda):
    """A workspace full of NaN serves; one a byte short is not used; both agree
    with the automatic one's product."""
    import torch

    t, n, k = 9, 500, 8192
    need = gplk.gemv_nvfp4_workspace_bytes(t, n, k)
    auto = _check(gplk, cuda, t, n, k)
    full = _check(gplk, cuda, t, n, k, workspace=torch.full((need,), 0xFF, dtype=torch.uint8, device=cuda))
    short = torch.full((need,), 0xFF, dtype=torch.uint8, device=cuda)
    without = _check(gplk, cuda, t, n, k, workspace=short[: need - 1])
    none = _check(gplk, cuda, t, n, k, workspace=None)
    assert bool((short == 0xFF).all())
    assert torch.equal(auto.view(torch.int16), full.view(torch.int16))
    assert torch.equal(without.view(torch.int16), none.view(torch.int16))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("residual", [None, "apart", "inplace"])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_types_residual_strides(dtype, residual, pad, gplk, cuda):
    _check(gplk, cuda, 6, 515, 704, dtype=dtype, residual=residual, pad=pad)


@pytest.mark.parametrize("tnk", [(1, 4096, 4096), (8, 8192, 2048), (32, 2048, 8192), (17, 20000, 512), (1, 40000, 1024)])
def test_larger(tnk, gplk, cuda):
    _check(gplk, cuda, *tnk)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_magnitudes(dtype, gplk, cuda):
    """Rows of zeros, of one value, with one channel far above the rest, with
    groups spread over 2^24, near the type's ends."""
    import torch

    k = 1024
    gen = _gen(cuda, 5)
    x = torch.randn(8, k, device=cuda, generator=gen)
    x[0] = 0
    x[1] = 0
    x[1, 77] = -3.5
    x[2, 100] = 3000.0
    x[3] *= torch.pow(2.0, torch.arange(k, device=cuda) // 16 % 25 - 12)
    top = 2.0 ** 100 if dtype == "bf16" else 30000.0
    x[4] = x[4].clamp(-1, 1) * top
    x[5] *= 2.0 ** -100 if dtype == "bf16" else 2.0 ** -12
    x[6] = 1.0
    x[7] = -1.0 / 3
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    gen2 = _gen(cuda, 6)
    w, sf, wd = ref.random_weights(260, k, gen2, cuda)
    al = torch.tensor([1e-7 if dtype == "f16" else 1e-3], device=cuda)
    xs = x.to(dt)
    y = torch.empty(8, 260, dtype=dt, device=cuda)
    gplk.gemv_nvfp4(xs, w, sf, y, al)
    want = float(al) * (xs.double() @ wd.T)
    err = ref.product_error(wd, xs, float(al)) + 2 * 2.0 ** -24 * want.abs()
    tol = err + ref.rounding(want.abs() + err, dt)
    assert bool((y[0] == 0).all())
    assert bool(((y.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("bad", ["inf", "-inf", "nan"])
def test_nonfinite_token_stays_in_its_row(bad, gplk, cuda):
    import torch

    gen = _gen(cuda, 9)
    w, sf, wd = ref.random_weights(300, 512, gen, cuda)
    al = torch.ones(1, device=cuda)
    x = torch.randn(4, 512, device=cuda, generator=gen).to(torch.bfloat16)
    clean, y = (torch.empty(4, 300, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    gplk.gemv_nvfp4(x, w, sf, clean, al)
    x[2, 511] = float(bad)
    gplk.gemv_nvfp4(x, w, sf, y, al)
    torch.cuda.synchronize()
    keep = [0, 1, 3]
    assert torch.equal(y[keep].view(torch.int16), clean[keep].view(torch.int16))
    assert not bool(torch.isfinite(y[2][wd[:, 511] != 0]).any())


def test_same_inputs_same_bits_on_any_stream(gplk, cuda):
    import torch

    gen = _gen(cuda, 11)
    w, sf, _ = ref.random_weights(3000, 2048, gen, cuda)
    al = torch.ones(1, device=cuda)
    x = torch.randn(3, 2048, device=cuda, generator=gen).to(torch.bfloat16)
    first = torch.empty(3, 3000, dtype=torch.bfloat16, device=cuda)
    gplk.gemv_nvfp4(x, w, sf, first, al)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=cuda) for _ in range(3)]
    outs = [torch.empty_like(first) for _ in range(12)]
    for i, o in enumerate(outs):
        gplk.gemv_nvfp4(x, w, sf, o, al, stream=streams[i % 3])
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.view(torch.int16), first.view(torch.int16))


def test_captured_and_replayed_on_new_inputs(gplk, cuda):
    import torch

    gen = _gen(cuda, 12)
    w, sf, _ = ref.random_weights(1030, 1024, gen, cuda)
    al = torch.ones(1, device=cuda)
    x = torch.zeros(5, 1024, dtype=torch.bfloat16, device=cuda)
    y = torch.empty(5, 1030, dtype=torch.bfloat16, device=cuda)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gplk.gemv_nvfp4(x, w, sf, y, al)
        gplk.gemv_nvfp4(x, w, sf, y, al, residual=y)
    for seed in (1, 2):
        x.copy_(torch.randn(5, 1024, device=cuda, generator=gen))
        g.replay()
        eager = torch.empty_like(y)
        gplk.gemv_nvfp4(x, w, sf, eager, al)
        gplk.gemv_nvfp4(x, w, sf, eager, al, residual=eager)
        torch.cuda.synchronize()
        assert torch.equal(y.view(torch.int16), eager.view(torch.int16))


def test_reads_what_the_previous_kernel_wrote(gplk, cuda):
    """A chain on one stream: each product's output is the next one's input."""
    import torch

    gen = _gen(cuda, 13)
    w, sf, wd = ref.random_weights(1024, 1024, gen, cuda)
    al = torch.tensor([2e-3], device=cuda)
    x0 = torch.randn(2, 1024, device=cuda, generator=gen).to(torch.bfloat16)
    steps = [x0] + [torch.empty_like(x0) for _ in range(6)]
    for a, b in zip(steps, steps[1:]):
        gplk.gemv_nvfp4(a, w, sf, b, al)
    torch.cuda.synchronize()
    for a, b in zip(steps, steps[1:]):
        want = float(al) * (a.double() @ wd.T)
        err = ref.product_error(wd, a, float(al)) + 2 * 2.0 ** -24 * want.abs()
        assert bool(((b.double() - want).abs() <= err + ref.rounding(want.abs() + err, torch.bfloat16)).all())


def test_agrees_with_the_gemm_on_its_own_operands(gplk, cuda):
    """Prefill and decode on the same weights: activations that NVFP4 holds
    exactly go through gplk_gemm_nvfp4_tn and through the few-token product."""
    import torch
    from gplk import operands

    n, k, t = 384, 512, 16
    wf = operands.normal(n, k, 3, cuda)
    w, sf, g = operands.quantize_nvfp4(wf)
    xf = operands.normal(t, k, 4, cuda)
    xq, xsf, xg = operands.quantize_nvfp4(xf)
    xg = 2.0 ** round(torch.tensor(xg).log2().item())
    r, c = torch.arange(t, device=cuda).view(-1, 1), torch.arange(k // 16, device=cuda).view(1, -1)
    s = xsf[(r // 128 * (k // 64) + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4]
    x = (ref.decode(xq, s) * xg).to(torch.bfloat16)  # 2 bits times 4 bits times a power of two: exact
    D = torch.empty(t, n, dtype=torch.bfloat16, device=cuda)
    gplk.gemm_nvfp4_tn(w, xq, sf, xsf, D, k, torch.tensor([g * xg], dtype=torch.float32, device=cuda))
    y = torch.empty(t, n, dtype=torch.bfloat16, device=cuda)
    gplk.gemv_nvfp4(x, w, sf, y, torch.tensor([g], dtype=torch.float32, device=cuda))
    torch.cuda.synchronize()
    rows, cols = torch.arange(n, device=cuda).view(-1, 1), torch.arange(k // 16, device=cuda).view(1, -1)
    ws = sf[(rows // 128 * (k // 64) + cols // 4) * 512 + rows % 32 * 16 + rows % 128 // 32 * 4 + cols % 4]
    wd = ref.decode(w, ws)
    want = g * (x.double() @ wd.T)
    err = ref.product_error(wd, x, g) + 4 * 2.0 ** -24 * want.abs()
    tol = err + ref.rounding(want.abs() + err, torch.bfloat16)
    assert bool(((y.double() - want).abs() <= tol).all())
    assert bool(((D.double() - want).abs() <= tol).all())


def test_empty(gplk, cuda):
    import torch

    w, sf = torch.empty(0, 32, dtype=torch.uint8, device=cuda), torch.empty(0, dtype=torch.uint8, device=cuda)
    al = torch.ones(1, device=cuda)
    gplk.gemv_nvfp4(torch.empty(3, 64, dtype=torch.bfloat16, device=cuda), w, sf,
                    torch.empty(3, 0, dtype=torch.bfloat16, device=cuda), al)
    w, sf, _ = ref.random_weights(8, 64, _gen(cuda, 1), cuda)
    gplk.gemv_nvfp4(torch.empty(0, 64, dtype=torch.bfloat16, device=cuda), w, sf,
                    torch.empty(0, 8, dtype=torch.bfloat16, device=cuda), al)
    torch.cuda.synchronize()


def test_two_calls_at_once_converting_ahead(gplk, cuda):
    """Products of many tokens on two streams, replayed from two graphs that
    were captured with automatic workspaces."""
    import torch

    gen = _gen(cuda, 21)
    w, sf, _ = ref.random_weights(2000, 4096, gen, cuda)
    al = torch.ones(1, device=cuda)
    xs = [torch.zeros(16, 4096, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    ys = [torch.empty(16, 2000, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, x, y in zip(graphs, xs, ys):
        with torch.cuda.graph(g):
            gplk.gemv_nvfp4(x, w, sf, y, al)
            gplk.gemv_nvfp4(x, w, sf, y, al, residual=y)
    streams = [torch.cuda.Stream(device=cuda) for _ in range(2)]
    for _ in range(4):
        for x in xs:
            x.copy_(torch.randn(16, 4096, device=cuda, generator=gen))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, y in zip(xs, ys):
            e = torch.empty_like(y)
            gplk.gemv_nvfp4(x, w, sf, e, al)
            gplk.gemv_nvfp4(x, w, sf, e, al, residual=e)
            torch.cuda.synchronize()
            assert torch.equal(y.view(torch.int16), e.view(torch.int16))


def test_python_refusals(gplk, cuda):
    import torch

    w, sf, _ = ref.random_weights(8, 64, _gen(cuda, 1), cuda)
    al = torch.ones(1, device=cuda)
    bf = dict(dtype=torch.bfloat16, device=cuda)
    x, y = torch.zeros(2, 64, **bf), torch.zeros(2, 8, **bf)
    bad = [
        (x.float(), w, sf, y.float(), al, None),
        (x, w, sf, y.half(), al, None),
        (x, w, sf, torch.zeros(3, 8, **bf), al, None),
        (x, w, sf, torch.zeros(2, 9, **bf), al, None),
        (x, w[:, :16], sf, y, al, None),
        (x, w, sf[:100], y, al, None),
        (x, w, sf, y, al.double(), None),
        (x, w, sf, y.cpu(), al, None),
        (x, w, sf, y, al, torch.zeros(1, 8, **bf)),
        (x, w, sf, y, al, y.float()),
        (torch.zeros(64, 2, **bf).T, w, sf, y, al, None),
        (torch.zeros(33, 64, **bf), w, sf, torch.zeros(33, 8, **bf), al, None),
        (x[:, :32], w[:, :16].contiguous(), sf, y, al, None),
    ]
    for a in bad:
        with pytest.raises(gplk.GplkError):
            gplk.gemv_nvfp4(*a[:5], residual=a[5])
    gplk.gemv_nvfp4(x, w, sf, y, al)
    torch.cuda.synchronize()
