"""The few-token NVFP4 operators on the paths that tests of other sizes do not
take: FP16, strided rows and tokens that are not finite through the conversion
ahead of the products, the resident blocks and the router of many tokens; and
arguments that only a GPU tensor can carry."""
from __future__ import annotations

import pytest

import nvfp4_reference as ref
from test_gemv_nvfp4_gpu import _check as product
from test_moe_nvfp4_gpu import Layer
from test_moe_nvfp4_gpu import _case as layer_case

pytestmark = pytest.mark.gpu


def _gen(cuda, seed):
    import torch

    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def test_layer_without_a_workspace_is_refused(gplk, cuda):
    import torch

    layer = Layer(4, 128, 64, torch.bfloat16, _gen(cuda, 1), cuda)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(gplk.GplkError):
        layer.run(gplk, x, 2, workspace=None)

@pytest.mark.parametrize("t", [1, 2, 3, 4, 7, 12, 16, 18, 19, 24, 27, 32])
def test_product_f16_tokens(t, gplk, cuda):
    product(gplk, cuda, t, 300, 1088, dtype="f16", pad=1)


@pytest.mark.parametrize("tnk", [(4, 700, 8192), (9, 500, 8192), (17, 1000, 4160), (25, 128, 16384), (32, 130, 16448)])
@pytest.mark.parametrize("pad", [0, 1, 3, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_product_converted_ahead(dtype, pad, tnk, gplk, cuda):
    product(gplk, cuda, *tnk, dtype=dtype, pad=pad, residual="inplace")


@pytest.mark.parametrize("tnk", [(1, 200, 512), (4, 300, 1088), (3, 200, 16384), (9, 500, 8192), (17, 1000, 4160),
                                 (32, 130, 16448)])
@pytest.mark.parametrize("bad", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_product_token_that_is_not_finite(dtype, bad, tnk, gplk, cuda):
    """All of its outputs are NaN, whatever the weights; the others keep their bits."""
    import torch

    t, n, k = tnk
    gen = _gen(cuda, 61 + t + n + k)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    w, sf, _ = ref.random_weights(n, k, gen, cuda)
    w[::2, (k - 1) // 2] &= 0x0F  # zero weights on the bad element in every other row
    al = torch.full((1,), 1e-3, device=cuda)
    x = torch.randn(t, k, device=cuda, generator=gen).to(dt)
    clean, y = (torch.empty(t, n, dtype=dt, device=cuda) for _ in range(2))
    gplk.gemv_nvfp4(x, w, sf, clean, al)
    at = t // 2
    x[at, k - 1] = float(bad)
    gplk.gemv_nvfp4(x, w, sf, y, al)
    torch.cuda.synchronize()
    keep = [i for i in range(t) if i != at]
    assert bool(torch.isnan(y[at]).all())
    assert torch.equal(y[keep].view(torch.int16), clean[keep].view(torch.int16))


# Resident blocks (strided x, several entries an expert, an odd last tile); clusters with the router of many
# tokens; more experts than four to a lane.
LAYERS = [(8, 64, 8, 640, 1024), (32, 40, 4, 320, 1088), (32, 2, 2, 192, 128), (7, 9, 3, 256, 192), (12, 300, 3, 128, 192)]


@pytest.mark.parametrize("size", LAYERS)
@pytest.mark.parametrize("pad", [0, 1, 3])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_layer_types_and_strides(dtype, pad, size, gplk, cuda):
    layer_case(gplk, cuda, *size, dtype=dtype, pad=pad)


@pytest.mark.parametrize("size", LAYERS)
@pytest.mark.parametrize("bad", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_layer_token_that_is_not_finite(dtype, bad, size, gplk, cuda):
    import torch

    t, e, top, d, f = size
    gen = _gen(cuda, 67 + sum(size))
    dt = torch.bfloat16 if dtype == "bf16" else torch.float16
    layer = Layer(e, d, f, dt, gen, cuda)
    x = torch.randn(t, d, device=cuda, generator=gen).to(dt)
    at = t // 2
    x[at, d - 1] = float(bad)
    y, ids, w = layer.run(gplk, x, top)
    torch.cuda.synchronize()
    assert bool(torch.isnan(y[at]).all())
    assert bool(((ids[at] >= 0) & (ids[at] < e)).all()) and len(set(ids[at].tolist())) == top
    keep = [i for i in range(t) if i != at]
    layer.check(x[keep], top, True, y[keep], ids[keep], w[keep])


def test_products_layers_and_gemms_at_once(gplk, cuda):
    """Streams of products, of layers and of GEMMs side by side, whose blocks
    want different parts of an SM: every call ends, with the bits it has alone."""
    import torch

    gen = _gen(cuda, 71)
    bf = dict(dtype=torch.bfloat16, device=cuda)
    sizes = [(1, 2048, 2048), (3, 1000, 4096), (12, 2000, 4096), (32, 4000, 1024)]
    products = []
    for t, n, k in sizes:
        w, sf, _ = ref.random_weights(n, k, gen, cuda)
        products.append((torch.randn(t, k, device=cuda, generator=gen).to(torch.bfloat16), w, sf))
    al = torch.full((1,), 1e-3, device=cuda)
    layers = [(Layer(e, d, f, torch.bfloat16, gen, cuda), torch.randn(t, d, device=cuda, generator=gen).to(**bf), top)
              for t, e, top, d, f in ((2, 8, 2, 512, 256), (8, 64, 8, 640, 1024))]
    p, q = torch.randn(1024, 1024, device=cuda, generator=gen).to(torch.bfloat16), torch.empty(1024, 1024, **bf)

    def product_run(i, stream=None):
        x, w, sf = products[i]
        y = torch.empty(x.shape[0], w.shape[0], **bf)
        gplk.gemv_nvfp4(x, w, sf, y, al, stream=stream)
        return y

    want = [product_run(i) for i in range(len(products))]
    want_layers = [layer.run(gplk, x, top)[0] for layer, x, top in layers]
    gplk.gemm_nn("bf16", p, p, q, 1024, 1024, 1024)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=cuda) for _ in range(4)]
    got, got_layers, got_gemm = [], [], []
    for r in range(12):
        for s, i in zip(streams[:2], (r % 4, (r + 2) % 4)):
            with torch.cuda.stream(s):
                got.append((i, product_run(i)))
        with torch.cuda.stream(streams[2]):
            layer, x, top = layers[r % 2]
            got_layers.append((r % 2, layer.run(gplk, x, top)[0]))
        with torch.cuda.stream(streams[3]):
            g = torch.empty_like(q)
            gplk.gemm_nn("bf16", p, p, g, 1024, 1024, 1024)
            got_gemm.append(g)
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y.view(torch.int16), want[i].view(torch.int16))
    for i, y in got_layers:
        assert torch.equal(y.view(torch.int16), want_layers[i].view(torch.int16))
    for g in got_gemm:
        assert torch.equal(g.view(torch.int16), q.view(torch.int16))


def test_weights_written_by_the_kernel_before(gplk, cuda):
    """Weights and scales that a kernel writes right before each call, in
    streams and in a captured graph: no product or layer starts on older ones."""
    import torch

    gen = _gen(cuda, 73)
    t, n, k = 16, 3000, 4096  # converted ahead: weights are read while that runs
    sets = [ref.random_weights(n, k, gen, cuda)[:2] for _ in range(3)]
    layer, other = (Layer(8, 512, 320, torch.bfloat16, gen, cuda) for _ in range(2))
    al = torch.full((1,), 1e-3, device=cuda)
    x = torch.randn(t, k, device=cuda, generator=gen).to(torch.bfloat16)
    v = torch.randn(3, 512, device=cuda, generator=gen).to(torch.bfloat16)
    stacks = [torch.cat([a.flatten() for op in (q.gate, q.up, q.down) for a in op[:2]]) for q in (layer, other)]

    def product(w, sf):
        y = torch.empty(t, n, dtype=torch.bfloat16, device=cuda)
        gplk.gemv_nvfp4(x, w, sf, y, al)
        return y

    want = [product(*s) for s in sets]
    other.gate, other.up, other.down = ((b[0], b[1], a[2]) for a, b in zip((layer.gate, layer.up, layer.down),
                                                                           (other.gate, other.up, other.down)))
    other.router = layer.router
    want_layers = [q.run(gplk, v, 2)[0] for q in (layer, other)]
    parts = [a for op in (layer.gate, layer.up, layer.down) for a in op[:2]]
    torch.cuda.synchronize()
    w, sf = sets[0][0].clone(), sets[0][1].clone()

    def write(i):
        at = 0
        for a in parts:
            a.view(-1).copy_(stacks[i][at : at + a.numel()])
            at += a.numel()

    def both(i):
        w.copy_(sets[i % 3][0])
        sf.copy_(sets[i % 3][1])
        y = product(w, sf)
        write(i % 2)
        return y, layer.run(gplk, v, 2)[0]

    got = [both(i) for i in range(12)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [both(i) for i in range(6)]
    graph.replay()
    torch.cuda.synchronize()
    for outs in (got, captured):
        for i, (y, z) in enumerate(outs):
            assert torch.equal(y.view(torch.int16), want[i % 3].view(torch.int16))
            assert torch.equal(z.view(torch.int16), want_layers[i % 2].view(torch.int16))


def test_row_distances_beyond_32_bits_are_refused(gplk, cuda):
    """A C int carries them: 2^32 + 64 would arrive as 64, a row distance in bounds
    that is not the tensor's."""
    import torch

    k, n = 64, 128
    w, sf, _ = ref.random_weights(n, k, _gen(cuda, 79), cuda)
    al = torch.ones(1, device=cuda)
    far = torch.empty((1 << 32) + 2 * n, dtype=torch.bfloat16, device=cuda)
    x, y = (far.as_strided((2, width), ((1 << 32) + width, 1)) for width in (k, n))
    x_near, y_near = x.contiguous(), torch.zeros(2, n, dtype=torch.bfloat16, device=cuda)
    for args in ((x, y_near, None), (x_near, y, None), (x_near, y_near, y)):
        with pytest.raises(gplk.GplkError):
            gplk.gemv_nvfp4(args[0], w, sf, args[1], al, residual=args[2])
    layer = Layer(4, 64, 128, torch.bfloat16, _gen(cuda, 80), cuda)
    y_near = torch.zeros_like(x_near)
    for args in ((x, y_near), (x_near, x)):
        with pytest.raises(gplk.GplkError):
            layer.run(gplk, args[0], 2, y=args[1])


def _rows(w, sf, at, k):
    """float64 values of rows `at` of one matrix."""
    import torch

    r, g = at.view(-1, 1), torch.arange(k // 16, device=w.device).view(1, -1)
    return ref.decode(w[at], sf[(r // 128 * -(-k // 64) + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4])


def test_product_offsets_beyond_32_bits(gplk, cuda):
    """8 GiB of codes: rows on both sides of 2^32 bytes, and the last ones."""
    import torch

    n, k = 131072 + 40, 131072
    gen = _gen(cuda, 83)
    w = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=cuda, generator=gen)
    sf = torch.randint(0x28, 0x48, (ref.sf_bytes(n, k),), dtype=torch.uint8, device=cuda, generator=gen)
    x = torch.randn(4, k, device=cuda, generator=gen).to(torch.bfloat16)
    al = torch.full((1,), 1e-3, device=cuda)
    at = torch.cat([torch.arange(65536 - 64, 65536 + 64), torch.arange(n - 100, n)]).to(cuda)
    wd = _rows(w, sf, at, k)
    for workspace in ("auto", None):
        y = torch.empty(4, n, dtype=torch.bfloat16, device=cuda)
        gplk.gemv_nvfp4(x, w, sf, y, al, workspace=workspace)
        want = float(al) * (x.double() @ wd.T)
        err = ref.product_error(wd, x, float(al)) + 2 * 2.0 ** -24 * want.abs()
        assert ref.off(y[:, at], want, err, torch.bfloat16) <= 1


def test_layer_offsets_beyond_32_bits(gplk, cuda):
    """Stacks of 4 GiB and more, of which the last experts are chosen."""
    import torch

    e, d, f, t, top = 512, 4096, 4160, 3, 2
    gen = _gen(cuda, 89)

    def stack(rows, k):
        w = torch.randint(0, 256, (e, rows, k // 2), dtype=torch.uint8, device=cuda, generator=gen)
        sf = torch.randint(0x28, 0x40, (e, ref.sf_bytes(rows, k)), dtype=torch.uint8, device=cuda, generator=gen)
        return w, sf, torch.full((e,), 0.3 / k ** 0.5, device=cuda)

    gate, up, down = stack(f, d), stack(f, d), stack(d, f)
    assert gate[0].numel() > 1 << 32
    x = torch.randn(t, d, device=cuda, generator=gen).to(torch.bfloat16)
    router = torch.randn(e, d, device=cuda, generator=gen) / d ** 0.5
    for i in range(t):  # token i's experts are among the last
        router[e - 1 - i] += x[i].float() / 64
        router[e - 4 - i] += x[i].float() / 128
    router = router.to(torch.bfloat16)
    y, ids, w = torch.empty_like(x), torch.empty(t, top, dtype=torch.int32, device=cuda), torch.empty(t, top, device=cuda)
    gplk.moe_nvfp4(x, router, gate, up, down, y, ids, w)
    assert int(ids.min()) >= e - 8

    class Decoded:
        def __init__(self, op, rows, k):
            self.op, self.rows, self.k = op, rows, k

        def __getitem__(self, i):
            at = torch.arange(self.rows, device=cuda)
            return _rows(self.op[0][i], self.op[1][i], at, self.k), float(self.op[2][i])

    want, err, wids, ww, dw = ref.moe(x, router, Decoded(gate, f, d), Decoded(up, f, d), Decoded(down, d, f), top, True)
    assert torch.equal(ids, wids)
    assert bool(((w.double() - ww).abs() <= dw * ww + 2.0 ** -140).all())
    assert ref.off(y, want, err, x.dtype) <= 1
