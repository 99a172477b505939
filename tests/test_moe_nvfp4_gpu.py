"""gplk_moe_nvfp4 (a mixture-of-experts layer for a few tokens) against the
layer in 64 bits on the same codes, scale bytes and activations: the chosen
experts exactly, weights and outputs within the bounds that
nvfp4_reference.moe derives."""
from __future__ import annotations

import pytest

import nvfp4_reference as ref

pytestmark = pytest.mark.gpu


def _gen(cuda, seed):
    import torch

    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


class Layer:
    """Random experts and router of one layer, in both forms."""

    def __init__(self, e, d, f, dt, gen, cuda, pad_byte=0x7F):
        import torch

        def stack(rows, k):
            parts = [ref.random_weights(rows, k, gen, cuda, pad_byte) for _ in range(e)]
            alpha = (0.5 + torch.rand(e, device=cuda, generator=gen)) / (3 * k ** 0.5)
            op = (torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]), alpha)
            return op, [(p[2], float(a)) for p, a in zip(parts, alpha)]

        self.router = (torch.randn(e, d, device=cuda, generator=gen) / d ** 0.5).to(dt)
        (self.gate, self.gate64), (self.up, self.up64), (self.down, self.down64) = stack(f, d), stack(f, d), stack(d, f)

    def run(self, gplk, x, top, renorm=True, y=None, **kw):
        import torch

        y = torch.empty_like(x) if y is None else y
        ids = torch.full((x.shape[0], top), -7, dtype=torch.int32, device=x.device)
        w = torch.full((x.shape[0], top), float("nan"), device=x.device)
        gplk.moe_nvfp4(x, self.router, self.gate, self.up, self.down, y, ids, w, renormalise=renorm, **kw)
        return y, ids, w

    def check(self, x, top, renorm, y, ids, w):
        import torch

        want, err, wids, ww, dw = ref.moe(x, self.router, self.gate64, self.up64, self.down64, top, renorm)
        assert torch.equal(ids, wids)
        assert bool(((w.double() - ww).abs() <= dw * ww + 2.0 ** -140).all())
        off = ref.off(y, want, err, x.dtype)
        assert off <= 1, off


def _case(gplk, cuda, t, e, top, d, f, dtype="bf16", renorm=True, pad=0, seed=0):
    import torch

    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    gen = _gen(cuda, seed + 1000 * t + 10 * e + d + f)
    layer = Layer(e, d, f, dt, gen, cuda)
    x = torch.randn(t, d + pad, device=cuda, generator=gen).to(dt)[:, :d]
    buf = torch.full((t, d + pad), 7.0, dtype=dt, device=cuda)
    y, ids, w = layer.run(gplk, x, top, renorm, y=buf[:, :d])
    torch.cuda.synchronize()
    layer.check(x, top, renorm, y, ids, w)
    if pad:
        assert bool((buf[:, d:] == 7.0).all()), "columns beyond D were written"


@pytest.mark.parametrize("t", [1, 2, 5, 8, 16, 27, 32])
def test_tokens(t, gplk, cuda):
    _case(gplk, cuda, t, 8, 3, 320, 192)


@pytest.mark.parametrize("e,top", [(1, 1), (2, 2), (3, 1), (16, 16), (33, 5), (100, 8), (512, 16)])
def test_experts(e, top, gplk, cuda):
    _case(gplk, cuda, 3, e, top, 128, 64)


@pytest.mark.parametrize("d,f", [(64, 64), (64, 704), (704, 64), (192, 448), (1088, 320), (2048, 1024)])
@pytest.mark.parametrize("t", [1, 6])
def test_widths(t, d, f, gplk, cuda):
    _case(gplk, cuda, t, 4, 2, d, f)


@pytest.mark.parametrize("t,e,top,d,f", [
    (8, 64, 8, 640, 1024),    # items for resident blocks, an odd number of down's tiles
    (32, 40, 4, 320, 1088),   # the same, tiles cut short, some experts with several tokens
    (32, 2, 2, 192, 128),     # every expert has all 32 tokens: three entries each
    (32, 1, 1, 1024, 20480),  # resident gate / up of one expert in three entries
    (32, 512, 16, 64, 64),    # the most experts, ranks and tokens
    (3, 8, 2, 1024, 8192),    # down accumulates over long K
    (12, 300, 3, 128, 192),   # more experts than four to a lane
])
def test_paths(t, e, top, d, f, gplk, cuda):
    _case(gplk, cuda, t, e, top, d, f)


def test_without_ids_and_weights(gplk, cuda):
    """Through the C ABI with NULL for both: the same y."""
    import ctypes

    import torch

    layer = Layer(6, 128, 192, torch.bfloat16, _gen(cuda, 10), cuda)
    x = torch.randn(5, 128, device=cuda, generator=_gen(cuda, 11)).to(torch.bfloat16)
    y, _, _ = layer.run(gplk, x, 2)
    z = torch.empty_like(y)
    ws = torch.empty(gplk.moe_nvfp4_workspace_bytes(5, 6, 2, 128, 192), dtype=torch.uint8, device=cuda)
    p = lambda a: a.data_ptr()  # noqa: E731
    g, u, d = layer.gate, layer.up, layer.down
    c = gplk.MoeCfg(p(x), p(layer.router), p(g[0]), p(u[0]), p(d[0]), p(g[1]), p(u[1]), p(d[1]), p(g[2]), p(u[2]),
                    p(d[2]), p(z), None, None, p(ws), ws.numel(), 5, 6, 2, 128, 192, 128, 128, 1, 0)
    assert gplk.lib().gplk_moe_nvfp4(ctypes.byref(c), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(y.view(torch.int16), z.view(torch.int16))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_types_weights_strides(dtype, renorm, pad, gplk, cuda):
    _case(gplk, cuda, 4, 6, 2, 256, 192, dtype=dtype, renorm=renorm, pad=pad)


def test_all_tokens_to_one_expert_and_ties(gplk, cuda):
    """Equal router rows tie: the lower index wins. Every token then goes to
    the same experts."""
    import torch

    gen = _gen(cuda, 3)
    layer = Layer(40, 256, 128, torch.bfloat16, gen, cuda)
    layer.router[:] = layer.router[:1]
    x = torch.randn(32, 256, device=cuda, generator=gen).to(torch.bfloat16)
    y, ids, w = layer.run(gplk, x, 4)
    torch.cuda.synchronize()
    assert torch.equal(ids, torch.arange(4, device=cuda, dtype=torch.int32).expand(32, 4))
    assert torch.equal(w, torch.full_like(w, 0.25))
    layer.check(x, 4, True, y, ids, w)


def test_one_expert_far_from_the_others(gplk, cuda):
    """Router weights that give one expert all of the probability: the other
    chosen ones count with weights down to zero."""
    import torch

    gen = _gen(cuda, 4)
    layer = Layer(5, 128, 192, torch.bfloat16, gen, cuda)
    layer.router *= 40
    x = torch.randn(7, 128, device=cuda, generator=gen).to(torch.bfloat16)
    y, ids, w = layer.run(gplk, x, 3, False)
    torch.cuda.synchronize()
    layer.check(x, 3, False, y, ids, w)


def test_zero_tokens_rows(gplk, cuda):
    import torch

    gen = _gen(cuda, 5)
    layer = Layer(4, 128, 128, torch.bfloat16, gen, cuda)
    x = torch.randn(3, 128, device=cuda, generator=gen).to(torch.bfloat16)
    x[1] = 0
    y, ids, w = layer.run(gplk, x, 2)
    torch.cuda.synchronize()
    assert bool((y[1] == 0).all()) and ids[1].tolist() == [0, 1]
    layer.check(x, 2, True, y, ids, w)
    layer.run(gplk, x[:0], 2)


@pytest.mark.parametrize("bad", ["inf", "nan"])
def test_nonfinite_token_stays_in_its_row(bad, gplk, cuda):
    import torch

    gen = _gen(cuda, 6)
    layer = Layer(9, 256, 192, torch.bfloat16, gen, cuda)
    x = torch.randn(4, 256, device=cuda, generator=gen).to(torch.bfloat16)
    clean, cids, _ = layer.run(gplk, x, 3)
    x[2, 5] = float(bad)
    y, ids, _ = layer.run(gplk, x, 3)
    torch.cuda.synchronize()
    keep = [0, 1, 3]
    assert torch.equal(ids[keep], cids[keep])
    assert torch.equal(y[keep].view(torch.int16), clean[keep].view(torch.int16))
    assert not bool(torch.isfinite(y[2]).any())
    assert bool(((ids[2] >= 0) & (ids[2] < 9)).all()) and len(set(ids[2].tolist())) == 3


def test_streams_and_workspaces(gplk, cuda):
    """Calls on several streams at once, each in a block of its own, and calls
    in a caller's workspace full of NaN: the same bits every time."""
    import torch

    gen = _gen(cuda, 7)
    layer = Layer(16, 512, 320, torch.bfloat16, gen, cuda)
    x = torch.randn(6, 512, device=cuda, generator=gen).to(torch.bfloat16)
    first, fids, fw = layer.run(gplk, x, 4)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=cuda) for _ in range(3)]
    outs = [torch.empty_like(x) for _ in range(9)]
    ids = [torch.empty_like(fids) for _ in range(9)]
    ws = [torch.empty_like(fw) for _ in range(9)]
    torch.cuda.synchronize()
    for i in range(9):
        gplk.moe_nvfp4(x, layer.router, layer.gate, layer.up, layer.down, outs[i], ids[i], ws[i], stream=streams[i % 3])
    torch.cuda.synchronize()
    n = gplk.moe_nvfp4_workspace_bytes(6, 16, 4, 512, 320)
    own = torch.full((n,), 0xFF, dtype=torch.uint8, device=cuda)
    for _ in range(2):
        outs.append(layer.run(gplk, x, 4, workspace=own)[0])
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.view(torch.int16), first.view(torch.int16))
    with pytest.raises(gplk.GplkError):
        layer.run(gplk, x, 4, workspace=own[: n - 1])


def test_two_captured_graphs(gplk, cuda):
    """Two graphs captured with automatic workspaces, replayed together on two
    streams over new inputs."""
    import torch

    gen = _gen(cuda, 8)
    layers = [Layer(8, 256, 128, torch.bfloat16, gen, cuda) for _ in range(2)]
    xs = [torch.zeros(3, 256, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    graphs, outs = [], []
    for layer, x in zip(layers, xs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.run(gplk, x, 2))
        graphs.append(g)
    streams = [torch.cuda.Stream(device=cuda) for _ in range(2)]
    for _ in range(3):
        for x in xs:
            x.copy_(torch.randn(3, 256, device=cuda, generator=gen))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for layer, x, (y, ids, w) in zip(layers, xs, outs):
            layer.check(x, 2, True, y, ids, w)


@pytest.mark.parametrize("t,e,top,d,f", [(8, 64, 8, 640, 1024), (3, 32, 4, 512, 320)])
def test_replays_on_other_experts(t, e, top, d, f, gplk, cuda):
    """A captured layer (resident blocks; clusters) replayed back to back on
    inputs that choose other experts each time: the eager call's bits."""
    import torch

    gen = _gen(cuda, 12)
    layer = Layer(e, d, f, torch.bfloat16, gen, cuda)
    x = torch.zeros(t, d, dtype=torch.bfloat16, device=cuda)
    xs = [torch.randn(t, d, device=cuda, generator=gen).to(torch.bfloat16) for _ in range(5)]
    eager = [layer.run(gplk, v, top) for v in xs]
    outs = [torch.empty_like(x) for _ in xs]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, ids, w = layer.run(gplk, x, top)
    for v, o in zip(xs, outs):  # nothing waits between the replays
        x.copy_(v)
        g.replay()
        o.copy_(y)
    torch.cuda.synchronize()
    assert len({tuple(i.flatten().tolist()) for _, i, _ in eager}) == len(xs)
    for (want, _, _), got in zip(eager, outs):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


def test_decoding_block(gplk, cuda):
    """The operators in a row as a decoding block has them: a projection that
    adds the residual stream, the mixture of experts on its output, a
    projection to scores; eager and captured, against 64 bits step by step."""
    import torch

    gen = _gen(cuda, 9)
    d, v, t = 512, 1500, 5
    wo, so, wo64 = ref.random_weights(d, 2 * d, gen, cuda)
    wv, sv, wv64 = ref.random_weights(v, d, gen, cuda)
    ao, av = torch.tensor([4e-3], device=cuda), torch.tensor([7e-3], device=cuda)
    layer = Layer(12, d, 320, torch.bfloat16, gen, cuda)
    bf = dict(dtype=torch.bfloat16, device=cuda)
    a, stream_in = torch.randn(t, 2 * d, device=cuda, generator=gen).to(**bf), torch.randn(t, d, device=cuda, generator=gen).to(**bf)
    h, y, z = torch.empty(t, d, **bf), torch.empty(t, d, **bf), torch.empty(t, v, **bf)
    ids, w = torch.empty(t, 2, dtype=torch.int32, device=cuda), torch.empty(t, 2, device=cuda)

    def block():
        gplk.gemv_nvfp4(a, wo, so, h, ao, residual=stream_in)
        gplk.moe_nvfp4(h, layer.router, layer.gate, layer.up, layer.down, y, ids, w)
        gplk.gemv_nvfp4(y, wv, sv, z, av)

    block()
    torch.cuda.synchronize()
    eager = [q.clone() for q in (h, y, z)]

    def near(got, x, w64, alpha, r=0.0):
        want = alpha * (x.double() @ w64.T) + r
        err = ref.product_error(w64, x, alpha) + 4 * 2.0 ** -24 * want.abs()
        assert bool(((got.double() - want).abs() <= err + ref.rounding(want.abs() + err, torch.bfloat16)).all())

    near(h, a, wo64, float(ao), stream_in.double())
    layer.check(h, 2, True, y, ids, w)
    near(z, y, wv64, float(av))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        block()
    for q in (h, y, z):
        q.fill_(float("nan"))
    g.replay()
    torch.cuda.synchronize()
    for q, e in zip((h, y, z), eager):
        assert torch.equal(q.view(torch.int16), e.view(torch.int16))


def test_python_refusals(gplk, cuda):
    import torch

    layer = Layer(4, 128, 64, torch.bfloat16, _gen(cuda, 1), cuda)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=cuda)
    y, ids, w = torch.empty_like(x), torch.empty(2, 2, dtype=torch.int32, device=cuda), torch.empty(2, 2, device=cuda)
    good = dict(X=x, router=layer.router, gate=layer.gate, up=layer.up, down=layer.down, Y=y, ids=ids, weights=w)
    g0, g1, g2 = layer.gate
    for kw in (dict(X=x.float()), dict(Y=y.half()), dict(Y=y[:1]), dict(router=layer.router.half()),
               dict(router=layer.router[:, :64]), dict(ids=ids.long()), dict(ids=ids[:1]), dict(weights=w.double()),
               dict(weights=w[:, :1]), dict(gate=(g0[:3], g1, g2)), dict(gate=(g0, g1[:, :100], g2)),
               dict(up=(g0, g1, g2.double())), dict(down=layer.gate), dict(gate=(g0[:, :32], g1, g2)),
               dict(ids=torch.empty(2, 5, dtype=torch.int32, device=cuda), weights=torch.empty(2, 5, device=cuda)),
               dict(Y=y.cpu())):
        with pytest.raises(gplk.GplkError):
            gplk.moe_nvfp4(**{**good, **kw})
    gplk.moe_nvfp4(**good)
    torch.cuda.synchronize()
