"""The NVFP4 few-token operators in 64 bits, and the tolerances they are held
to. Decodes codes and scale bytes by their fields; shares no code with the
library or the oracle."""
from __future__ import annotations

import torch


def sf_bytes(rows: int, k: int) -> int:
    return -(-rows // 128) * -(-k // 64) * 512


def random_weights(rows: int, k: int, gen, device, pad_byte: int = 0):
    """Random codes (every nibble), random scale bytes over the finite UE4M3
    range with zero and subnormal ones among them, laid out with `pad_byte` in
    the rows that pad the layout, and the decoded float64 matrix (without the
    matrix scale)."""
    w = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, device=device, generator=gen)
    s = torch.randint(0x20, 0x50, (rows, k // 16), dtype=torch.uint8, device=device, generator=gen)
    rare = torch.rand(rows, k // 16, device=device, generator=gen)
    s = torch.where(rare < 0.02, torch.zeros_like(s), s)
    s = torch.where((rare >= 0.02) & (rare < 0.04), s & 7, s)
    s = torch.where(rare > 0.98, torch.full_like(s, 0x7E), s)
    sf = torch.full((sf_bytes(rows, k),), pad_byte, dtype=torch.uint8, device=device)
    r = torch.arange(rows, device=device).view(-1, 1)
    g = torch.arange(k // 16, device=device).view(1, -1)
    sf[(r // 128 * -(-k // 64) + g // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + g % 4] = s
    return w, sf, decode(w, s)


def decode(w, s):
    """float64 values of packed codes (rows, k/2) and scale bytes (rows, k/16)."""
    rows, k = w.shape[0], w.shape[1] * 2
    b = w.long()
    c = torch.stack([b & 15, b >> 4], 2).view(rows, k)
    ex, man = (c >> 1) & 3, (c & 1).double()
    v = torch.where(ex == 0, man * 0.5, (1 + man * 0.5) * torch.pow(2.0, (ex - 1).double()))
    v = torch.where(c >= 8, -v, v)
    sl = s.long()
    se, sm = sl >> 3, (sl & 7).double()
    sv = torch.where(se == 0, sm / 8 * 2.0 ** -6, (1 + sm / 8) * torch.pow(2.0, (se - 7).double()))
    return (v.view(rows, k // 16, 16) * sv.unsqueeze(2)).view(rows, k)


def product_error(w, x, scale=1.0):
    """Bound on what scale * x @ w.T computed by the library is off before its
    output is rounded (w: rows x k float64, x: t x k, any float type).

    Activations: an activation is taken to a multiple of 2^b / 8192, 2^b being
    the power of two at or below the largest magnitude of its 16-group: off by
    at most 2^-14 of that magnitude. A group far below the token's largest
    magnitude (by 2^14 or more) is taken to a multiple of 2^-27 of that one: off
    by at most 2^-28 of it. Groups below 2^-114 are taken to multiples of
    2^-127.
    Sums: products are exact; 64 of them are added in one step that keeps at
    least FP32's 24 bits of the largest term, so a sum of k / 64 steps, and the
    16 additions that join partial sums, are off by (k / 64 + 16) * 2^-22 of the
    sum of magnitudes (two bits for the alignment inside a step)."""
    t, k = x.shape
    xa = x.double().abs()
    group = xa.view(t, k // 16, 16).amax(2, keepdim=True).expand(t, k // 16, 16).reshape(t, k)
    dx = group * 2.0 ** -14 + xa.amax(1, keepdim=True) * 2.0 ** -28 + 2.0 ** -128
    wa = w.abs()
    return abs(scale) * (dx @ wa.T + (k / 64 + 16) * 2.0 ** -22 * (xa @ wa.T))


def rounding(y, dtype):
    """Half a step of `dtype` at y, with the subnormal step as its floor."""
    f = torch.finfo(dtype)
    return y.abs() * (f.eps / 2) + f.tiny * f.eps / 2


def off(got, want, err, dtype) -> float:
    """The largest |got - want| over its bound: `err` before the output is
    rounded and half a step of rounding. An infinity is right where the value
    may lie at or above the largest finite number plus half its step (for FP16
    65504 + 16), which rounds to infinity; it counts as 0 there and as inf
    elsewhere."""
    f = torch.finfo(dtype)
    over = f.max + f.max * f.eps / (4 - 2 * f.eps)  # half of the step eps * 2^e, max = (2 - eps) * 2^e
    inf = torch.isinf(got)
    right = inf & (want.abs() + err >= over) & (torch.sign(got) == torch.sign(want))
    ratio = (got.double() - want).abs() / (err + rounding(want.abs() + err, dtype))
    return float(torch.where(right, torch.zeros_like(want), torch.nan_to_num(ratio, nan=float("inf"))).max())


def moe(x, router, gate, up, down, top, renormalise):
    """y, its error bound before rounding, ids, weights and their relative
    error bound. gate, up, down: lists of (decoded float64 matrix, alpha) per
    expert."""
    t, d = x.shape
    xd, rd = x.double(), router.double()
    p = torch.softmax(xd @ rd.T, 1)
    order = torch.sort(p, dim=1, descending=True, stable=True)
    ids, w = order.indices[:, :top], order.values[:, :top]
    if renormalise:
        w = w / w.sum(1, keepdim=True)
    # FP32 logits, summed in at most d / 64 + 16 steps, are off by that many half
    # steps of the sum of magnitudes; a weight is a quotient of exponentials of
    # their differences (which double the error) and of sums of at most 2^5
    # steps, each exponential and division off by at most 4 half steps.
    dl = ((d / 64 + 16) * 2.0 ** -24 * (xd.abs() @ rd.abs().T)).amax(1, keepdim=True)
    dw = 2 * dl + 64 * 2.0 ** -24
    y = torch.zeros(t, d, dtype=torch.float64, device=x.device)
    err = torch.zeros_like(y)
    for i in range(t):
        row, tail, most = xd[i : i + 1], 0.0, 0.0
        for j in range(top):
            e = int(ids[i, j])
            g, u = gate[e][1] * (row @ gate[e][0].T), up[e][1] * (row @ up[e][0].T)
            dg, du = product_error(gate[e][0], row, gate[e][1]), product_error(up[e][0], row, up[e][1])
            h = g * torch.sigmoid(g) * u
            # |silu'| <= 1.1; the exponential, the quotient and the products round
            # at most 16 half steps in FP32.
            dh = 1.1 * dg * u.abs() + (g * torch.sigmoid(g)).abs() * du + 1.1 * dg * du
            dh = dh + (16 * 2.0 ** -24 + dw[i]) * h.abs()
            wd, ad = down[e]
            c = float(w[i, j]) * ad
            y[i] += c * (h @ wd.T)[0]
            err[i] += abs(c) * (dh @ wd.abs().T + product_error(wd, h))[0]
            # Groups of the weighted h that are far below the token's largest
            # one, whichever expert that is of.
            most = max(most, abs(c) * float(h.abs().max()))
            tail = tail + wd.abs().sum(1)
        err[i] += 2.0 ** -28 * most * tail
    return y, err, ids.int(), w, dw
