"""How exactly 16-bit activations enter the few-token NVFP4 operators: within a
group of 16 whose largest magnitude is at least 2^b, as multiples of 2^b / 2^16
(BF16) or 2^b / 2^19 (FP16). A value down to 2^-9 of 2^b keeps all of its bits
then (BF16 has 8, FP16 11), and any other is off by at most half such a step.
The layer's h, which is FP32, enters down the same way, by the output's type."""
from __future__ import annotations

import pytest

import nvfp4_reference as ref
from test_moe_nvfp4_gpu import Layer

pytestmark = pytest.mark.gpu

HALF_STEP = {"bf16": 2.0 ** -17, "f16": 2.0 ** -20}


def _gen(cuda, seed):
    import torch

    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _dtype(name):
    import torch

    return torch.bfloat16 if name == "bf16" else torch.float16


def _error(w, x, scale, half_step):
    """ref.product_error, with activations off by half_step of their group's
    largest magnitude (and by 2^-14 of that share of the token's, in groups
    that lie further below it); 0: exact activations."""
    t, k = x.shape
    xa = x.double().abs()
    group = xa.view(t, k // 16, 16).amax(2, keepdim=True).expand(t, k // 16, 16).reshape(t, k)
    far = xa.amax(1, keepdim=True) * 2.0 ** -14
    dx = half_step * (group + far) + (2.0 ** -128 if half_step else 0.0)
    wa = w.abs()
    return abs(scale) * (dx @ wa.T + (k / 64 + 16) * 2.0 ** -22 * (xa @ wa.T))


def _beside_outliers(t, k, up, dt, gen, cuda):
    """Tokens with one value near 2^up in every group and the others between
    2^(up - 9) and 2^(up - 6), and the outliers' columns."""
    import torch

    x = torch.rand(t, k, device=cuda, generator=gen) * 7.0 + 1.0  # 1 to 8
    x = x * 2.0 ** (up - 9) * torch.where(torch.rand(t, k, device=cuda, generator=gen) < 0.5, -1.0, 1.0)
    cols = torch.arange(k // 16, device=cuda) * 16 + torch.randint(0, 16, (k // 16,), device=cuda, generator=gen)
    x[:, cols] = 2.0 ** up * (1 + 0.9 * torch.rand(t, k // 16, device=cuda, generator=gen))
    return x.to(dt), cols


def _without(w, wd, cols):
    """Codes (..., rows, k/2) and decoded rows without the columns: zeros, of both signs."""
    import torch

    keep = torch.full((wd.shape[1],), 0xF, dtype=torch.uint8, device=w.device)
    keep[cols] = 0x8
    w &= keep[0::2] | (keep[1::2] << 4)
    wd[:, cols] = 0.0


# one token, activations held in registers; converted by every block; several slices; 26 and more tokens (a second
# 128 rows of B scales); converted ahead of the products
SIZES = [(1, 300, 512), (3, 200, 1088), (5, 130, 4096), (32, 260, 1024), (9, 500, 8192), (16, 260, 8192),
         (32, 130, 16448)]


@pytest.mark.parametrize("tnk", SIZES)
@pytest.mark.parametrize("up", [3, 10])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_values_beside_an_outlier_keep_their_bits(dtype, up, tnk, gplk, cuda):
    """Where the weights of the outliers are zero, only FP32 sums of the exact
    activations and the output's rounding are left."""
    import torch

    t, n, k = tnk
    gen, dt = _gen(cuda, 41 + up + t + n + k), _dtype(dtype)
    x, cols = _beside_outliers(t, k, up, dt, gen, cuda)
    w, sf, wd = ref.random_weights(n, k, gen, cuda, 0x7F)
    _without(w, wd, cols)
    al = torch.tensor([2.0 ** -9 / k ** 0.5], dtype=torch.float32, device=cuda)
    y = torch.empty(t, n, dtype=dt, device=cuda)
    gplk.gemv_nvfp4(x, w, sf, y, al)
    want = float(al) * (x.double() @ wd.T)
    err = _error(wd, x, float(al), 0.0) + 2 * 2.0 ** -24 * want.abs()
    assert ref.off(y, want, err, dt) <= 1


@pytest.mark.parametrize("tnk", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_product_within_half_a_step_of_its_activations(dtype, tnk, gplk, cuda):
    """Normal activations with a few channels far above the rest."""
    import torch

    t, n, k = tnk
    gen, dt = _gen(cuda, 43 + t + n + k), _dtype(dtype)
    x = torch.randn(t, k, device=cuda, generator=gen)
    x[:, ::97] *= 300.0
    x = x.to(dt)
    w, sf, wd = ref.random_weights(n, k, gen, cuda, 0x7F)
    al = torch.tensor([2.0 ** -9 / k ** 0.5], dtype=torch.float32, device=cuda)
    y = torch.empty(t, n, dtype=dt, device=cuda)
    gplk.gemv_nvfp4(x, w, sf, y, al)
    want = float(al) * (x.double() @ wd.T)
    err = _error(wd, x, float(al), HALF_STEP[dtype]) + 2 * 2.0 ** -24 * want.abs()
    assert ref.off(y, want, err, dt) <= 1


# a cluster per item and accumulated down; resident blocks; resident blocks with experts of several tokens
LAYERS = [(3, 8, 2, 128, 64), (8, 64, 8, 640, 1024), (32, 40, 4, 320, 1088)]


@pytest.mark.parametrize("size", LAYERS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_layer_within_half_a_step_of_its_activations(dtype, size, gplk, cuda, monkeypatch):
    import torch

    t, e, top, d, f = size
    gen, dt = _gen(cuda, 47 + sum(size)), _dtype(dtype)
    layer = Layer(e, d, f, dt, gen, cuda)
    x = torch.randn(t, d, device=cuda, generator=gen).to(dt)
    y, ids, w = layer.run(gplk, x, top)
    monkeypatch.setattr(ref, "product_error", lambda wd, v, scale=1.0: _error(wd, v, scale, HALF_STEP[dtype]))
    layer.check(x, top, True, y, ids, w)


@pytest.mark.parametrize("size", LAYERS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_layer_beside_outliers(dtype, size, gplk, cuda, monkeypatch):
    """Outliers that gate and up have no weights for: x is exact, h within
    half a step."""
    import torch

    t, e, top, d, f = size
    gen, dt = _gen(cuda, 53 + sum(size)), _dtype(dtype)
    layer = Layer(e, d, f, dt, gen, cuda)
    x, cols = _beside_outliers(t, d, 8, dt, gen, cuda)
    layer.router[:, cols] = 0
    for op, decoded in ((layer.gate, layer.gate64), (layer.up, layer.up64)):
        for i, (wd, _) in enumerate(decoded):
            _without(op[0][i], wd, cols)
    y, ids, w = layer.run(gplk, x, top)
    monkeypatch.setattr(ref, "product_error", lambda wd, v, scale=1.0: _error(
        wd, v, scale, 0.0 if v.shape[1] == d else HALF_STEP[dtype]))
    layer.check(x, top, True, y, ids, w)
