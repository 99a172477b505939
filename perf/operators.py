"""What is measured of the NVFP4 operators for a few tokens: the cases, their
inputs, each operator in elementary torch operations, and its floor.

Two operators on weights in the framework's NVFP4 layout (E2M1 codes two per
byte, one UE4M3 scale per 16 K-elements in 128-row x 4-scale blocks of 512
bytes, one FP32 scale per matrix), with 16-bit activations:

  gemv   y[t] = alpha * W x[t] (+ r[t]) for 1 to 32 tokens
  moe    a mixture-of-experts layer for 1 to 32 tokens: router product,
         softmax, top-k, gated experts, weighted sum

`own` selects which form run() computes: the elementary one, or the calls a
user makes of the framework.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-power-lab_b200")
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _gplk():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import gplk

    return gplk


# ------------------------------------------------------------ the cases

def listed():
    return [
        # One token through a small square projection, weights resident in L2: what counts is latency.
        {"name": "gemv 1x2048x2048", "op": "gemv", "t": 1, "n": 2048, "k": 2048, "dtype": "bf16", "pad": 0, "residual": False},
        # One token through an output projection that adds the residual stream, FP16 activations.
        {"name": "gemv 1x4096x4096 f16", "op": "gemv", "t": 1, "n": 4096, "k": 4096, "dtype": "f16", "pad": 0, "residual": True},
        # One token through a wide up projection: far larger than a launch, one read of the weights.
        {"name": "gemv 1x16384x8192", "op": "gemv", "t": 1, "n": 16384, "k": 8192, "dtype": "bf16", "pad": 0, "residual": False},
        # A few tokens, a row count off every tile, a short K that ends inside a tile, rows of a wider buffer.
        {"name": "gemv 5x5003x1088", "op": "gemv", "t": 5, "n": 5003, "k": 1088, "dtype": "bf16", "pad": 24, "residual": True},
        # A small batch of sequences decoding together.
        {"name": "gemv 16x8192x8192", "op": "gemv", "t": 16, "n": 8192, "k": 8192, "dtype": "bf16", "pad": 0, "residual": False},
        # The largest: the ladder's largest square at the most tokens.
        {"name": "gemv 32x16384x16384", "op": "gemv", "t": 32, "n": 16384, "k": 16384, "dtype": "bf16", "pad": 0, "residual": False},
        # One token, two of eight small experts: latency.
        {"name": "moe 1 8/2 1024x512", "op": "moe", "t": 1, "e": 8, "top": 2, "d": 1024, "f": 512, "dtype": "bf16", "pad": 0, "renorm": True},
        # One token of a layer of many fine-grained experts: a single stream decoding.
        {"name": "moe 1 64/8 2048x1024", "op": "moe", "t": 1, "e": 64, "top": 8, "d": 2048, "f": 1024, "dtype": "bf16", "pad": 0, "renorm": True},
        # A few tokens, a hidden width that is no multiple of a tile, weights of the softmax over all experts.
        {"name": "moe 4 32/4 2048x704", "op": "moe", "t": 4, "e": 32, "top": 4, "d": 2048, "f": 704, "dtype": "bf16", "pad": 8, "renorm": False},
        # Eight sequences, 128 experts of which some 50 are read.
        {"name": "moe 8 128/8 4096x768", "op": "moe", "t": 8, "e": 128, "top": 8, "d": 4096, "f": 768, "dtype": "bf16", "pad": 0, "renorm": True},
        # Sixteen tokens over few wide experts, several tokens to each, FP16.
        {"name": "moe 16 16/2 4096x4096 f16", "op": "moe", "t": 16, "e": 16, "top": 2, "d": 4096, "f": 4096, "dtype": "f16", "pad": 0, "renorm": True},
        # The largest: 32 tokens that read nearly all of 64 experts.
        {"name": "moe 32 64/6 4096x2048", "op": "moe", "t": 32, "e": 64, "top": 6, "d": 4096, "f": 2048, "dtype": "bf16", "pad": 0, "renorm": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype, pad = rng.choice(["bf16", "bf16", "f16"]), rng.choice([0, 0, 8, 24, 3])
    t = _log(rng, 1, 32)
    if rng.random() < 0.5:
        k = 64 * _log(rng, 4, 256)
        n = _log(rng, 100, min(32768, (1 << 28) // k))
        return {"op": "gemv", "t": t, "n": n, "k": k, "dtype": dtype, "pad": pad, "residual": rng.random() < 0.5}
    e = _log(rng, 4, 128)
    d = 64 * _log(rng, 8, 64)
    f = 64 * _log(rng, 4, max(5, min(64, (1 << 29) // (e * d * 64))))
    return {"op": "moe", "t": t, "e": e, "top": rng.randint(1, min(8, e)), "d": d, "f": f, "dtype": dtype, "pad": pad,
            "renorm": rng.random() < 0.7}


# ------------------------------------------------------------ inputs

def _layout(s8):
    """rows x groups scale bytes in the 128-row x 4-scale block order, zero padded."""
    rows, groups = s8.shape
    r, g = -(-rows // 128) * 128, -(-groups // 4) * 4
    p = torch.zeros(r, g, dtype=torch.uint8, device=s8.device)
    p[:rows, :groups] = s8
    return p.view(r // 128, 4, 32, g // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _quantised(rows, k, gen):
    """A rows x k normal matrix in NVFP4: packed codes, laid-out scales, matrix scale."""
    w = torch.randn(rows, k // 16, 16, device="cuda", generator=gen).mul_(1.0 / math.sqrt(k))
    g = w.abs().max() / (6.0 * 448.0)
    s8 = (w.abs().amax(2) / 6.0 / g).to(torch.float8_e4m3fn)
    w /= (s8.float() * g).clamp_min(1e-30).unsqueeze(2)
    code = torch.bucketize(w.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda"), out_int32=True).to(torch.uint8)
    code |= (w < 0).to(torch.uint8) << 3
    code = code.view(rows, k // 2, 2)
    return code[..., 0] | (code[..., 1] << 4), _layout(s8.view(torch.uint8)), g


def _stack(e, rows, k, gen):
    parts = [_quantised(rows, k, gen) for _ in range(e)]
    return tuple(torch.stack(p) for p in zip(*parts))


def _activations(t, k, pad, dtype, gen):
    """Normal activations with a few channels far above the rest, as a block's
    normed input has them; rows of a buffer `pad` elements wider."""
    x = torch.randn(t, k + pad, device="cuda", generator=gen)
    x[:, :: 97] *= 12.0
    return x.to(dtype)[:, :k]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, t = _TYPES[case["dtype"]], case["t"]
    s = {"case": case}
    if case["op"] == "gemv":
        n, k = case["n"], case["k"]
        s["w"], s["sf"], g = _quantised(n, k, gen)
        s["alpha"] = g.reshape(1)
        s["x"] = _activations(t, k, case["pad"], dtype, gen)
        s["r"] = torch.randn(t, n, device="cuda", generator=gen).to(dtype) if case["residual"] else None
        s["y"] = torch.empty(t, n, dtype=dtype, device="cuda")
        return s
    e, d, f, top = case["e"], case["d"], case["f"], case["top"]
    s["x"] = _activations(t, d, case["pad"], dtype, gen)
    s["router"] = (torch.randn(e, d, device="cuda", generator=gen) / math.sqrt(d)).to(dtype)
    s["gate"], s["up"], s["down"] = _stack(e, f, d, gen), _stack(e, f, d, gen), _stack(e, d, f, gen)
    s["y"] = torch.empty(t, d, dtype=dtype, device="cuda")
    s["ids"] = torch.empty(t, top, dtype=torch.int32, device="cuda")
    s["weights"] = torch.empty(t, top, dtype=torch.float32, device="cuda")
    return s


# ------------------------------------------------------------ one pass

def _values(w, sf):
    """FP32 values (without the matrix scale) of packed codes (..., rows, k/2)
    and their laid-out scales (..., bytes)."""
    m = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=w.device)
    m = torch.cat([m, -m])
    b = torch.arange(256, device=w.device)
    pair = torch.stack([m[b & 15], m[b >> 4]], 1)
    lead, rows, k = w.shape[:-2], w.shape[-2], w.shape[-1] * 2
    v = pair[w.int()].view(*lead, rows, k // 16, 16)
    r, g = -(-rows // 128), -(-k // 64)
    s = sf.view(-1, r, g, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(*lead, r * 128, g * 4)
    s = s[..., :rows, : k // 16].contiguous().view(torch.float8_e4m3fn).float()
    return (v * s.unsqueeze(-1)).view(*lead, rows, k)


def _route(logits, top, renorm):
    """Top-k of the softmax over the experts, ties to the lowest index."""
    p = (logits - logits.amax(1, keepdim=True)).exp()
    p = p / p.sum(1, keepdim=True)
    p, order = torch.sort(p, dim=1, descending=True, stable=True)
    p, ids = p[:, :top], order[:, :top]
    return ids, p / p.sum(1, keepdim=True) if renorm else p


def _plain_gemv(s):
    y = s["x"].float() @ _values(s["w"], s["sf"]).T * s["alpha"]
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(s["x"].dtype)


def _plain_moe(s):
    case, x = s["case"], s["x"]
    t, e, top, d = case["t"], case["e"], case["top"], case["d"]
    # The logits decide which experts answer: in 64 bits.
    ids, w = _route(x.double() @ s["router"].double().T, top, case["renorm"])
    xf, w = x.float(), w.float()
    if t * top <= e:  # fewer pairs than experts: the pairs' own weights
        sel = ids.reshape(-1)
        xs = xf.repeat_interleave(top, 0).unsqueeze(2)
        g, u = ((_values(c[sel], f[sel]) @ xs).squeeze(2) * a[sel].unsqueeze(1) for c, f, a in (s["gate"], s["up"]))
        h = g / (1 + (-g).exp()) * u
        o = (_values(s["down"][0][sel], s["down"][1][sel]) @ h.unsqueeze(2)).squeeze(2) * s["down"][2][sel].unsqueeze(1)
        y = (o.view(t, top, d) * w.unsqueeze(2)).sum(1)
    else:  # every expert on every token, weighted by zero where it is not chosen
        every = torch.zeros(t, e, device=x.device).scatter_(1, ids, w)
        g, u = (torch.matmul(xf, _values(c, f).transpose(1, 2)) * a.view(-1, 1, 1) for c, f, a in (s["gate"], s["up"]))
        h = g / (1 + (-g).exp()) * u * every.T.unsqueeze(2)
        y = (torch.matmul(h, _values(s["down"][0], s["down"][1]).transpose(1, 2)) * s["down"][2].view(-1, 1, 1)).sum(0)
    return {"y": y.to(x.dtype), "ids": ids.int(), "weights": w}


def run(state):
    s = state
    if s["case"]["op"] == "gemv":
        if own:
            _gplk().gemv_nvfp4(s["x"], s["w"], s["sf"], s["y"], s["alpha"], residual=s["r"])
            return s["y"]
        return _plain_gemv(s)
    if own:
        _gplk().moe_nvfp4(s["x"], s["router"], s["gate"], s["up"], s["down"], s["y"], s["ids"], s["weights"],
                          renormalise=s["case"]["renorm"])
        return {"y": s["y"], "ids": s["ids"], "weights": s["weights"]}
    return _plain_moe(s)


def work(case):
    t = case["t"]
    if case["op"] == "gemv":
        n, k = case["n"], case["k"]
        return {"bytes": n * k // 2 + n * k // 16 + 2 * t * k + 2 * t * n * (2 if case["residual"] else 1), "flops": 2 * t * n * k}
    e, top, d, f = case["e"], case["top"], case["d"], case["f"]
    # The experts that t independent choices of `top` out of e are expected to touch.
    read = e * (1 - (1 - top / e) ** t)
    return {"bytes": int(read * 3 * d * f * 9 / 16) + 2 * e * d + 4 * t * d + 8 * t * top, "flops": 2 * t * e * d + 6 * t * top * d * f}


# ------------------------------------------------------------ the definition in 64 bits

def _decoded(w, sf, at):
    """Rows `at` of one matrix in 64 bits: each code and scale byte decoded by
    its fields, each scale fetched from its own place in the layout."""
    k = w.shape[1] * 2
    byte = w[at].long()
    code = torch.stack([byte % 16, byte // 16], 2).reshape(len(at), k)
    sign, ex, man = code // 8, code // 2 % 4, (code % 2).double()
    v = torch.where(ex == 0, man / 2, (1 + man / 2) * 2.0 ** (ex - 1).double()) * (1 - 2 * sign).double()
    r, c = at.view(-1, 1), torch.arange(k // 16, device=w.device).view(1, -1)
    place = (r // 128 * (-(-k // 64)) + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4
    b = sf.long()[place]
    ex, man = b // 8 % 16, (b % 8).double()
    scale = torch.where(ex == 0, man / 8 * 2.0 ** -6, (1 + man / 8) * 2.0 ** (ex - 7).double())
    return (v.view(len(at), -1, 16) * scale.unsqueeze(2)).view(len(at), k)


def _times(w, sf, x):
    """x (t x k) times the matrix's transpose in 64 bits, a band of rows at a time."""
    n, k = w.shape[0], w.shape[1] * 2
    step = max(128, (1 << 26) // k)
    return torch.cat([x.double() @ _decoded(w, sf, torch.arange(i, min(n, i + step), device=w.device)).T for i in range(0, n, step)], 1)


def exact(case, seed):
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "gemv":
        y = _times(s["w"], s["sf"], x) * s["alpha"].double()
        return y if s["r"] is None else y + s["r"].double()
    t, top = case["t"], case["top"]
    logits = torch.einsum("td,ed->te", x, s["router"].double())
    p = torch.softmax(logits, 1)
    # Selection one rank at a time; argmax of a reversed row would break ties upwards, so compare and take the first.
    ids, left = torch.zeros(t, top, dtype=torch.long, device=x.device), p.clone()
    for j in range(top):
        best = (left == left.amax(1, keepdim=True)).int()
        ids[:, j] = torch.where(best > 0, torch.arange(case["e"], device=x.device), case["e"]).amin(1)
        left.scatter_(1, ids[:, j : j + 1], -1.0)
    w = p.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(1, keepdim=True)
    y = torch.zeros(t, case["d"], dtype=torch.float64, device=x.device)
    for e in ids.unique().tolist():
        tok, slot = (ids == e).nonzero(as_tuple=True)
        g, u = (_times(m[0][e], m[1][e], x[tok]) * m[2][e].double() for m in (s["gate"], s["up"]))
        o = _times(s["down"][0][e], s["down"][1][e], g * torch.sigmoid(g) * u) * s["down"][2][e].double()
        y.index_add_(0, tok, o * w[tok, slot].unsqueeze(1))
    return {"y": y, "ids": ids.int(), "weights": w}
