"""64-bit restatements of the dense projection, the router and the mixture-of-experts layer, and
the error bounds their tests hold the kernels to.

Bounds (all elementwise, worst case):
  * one rounding to the output type is off by half a step: eps/2 * |y|, and by half the smallest
    subnormal below the normal range;
  * a tensor-core sum over K adds 16 products per instruction to an fp32 accumulator; each
    addition loses at most one fp32 step of the running sum, itself at most S = sum |x w|:
    (K/16 + 16) * 2^-23 * S (the 16: partial sums of a split K range, bias, residual);
  * activations have slope at most 1.13 and are evaluated to 2^-20 of |z| + |act(z)|.
"""
import torch

EPS = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
SLOPE = 1.13

# Coefficients of the rational GELU (erf as t P(t^2) / Q(t^2), argument clipped to +-3.92).
GELU_P = (0.053443748819, 7.5517016694, 101.62808918, 1393.8061484, 5063.7915060, 29639.384698)
GELU_Q = (1.0, 31.212858877, 398.56963806, 3023.1248150, 13243.365831, 26267.224157)


def act64(z, act, gelu="erf"):
    if act == "swiglu":
        g, u = z.chunk(2, dim=-1)
        return g * torch.sigmoid(g) * u
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu" and gelu == "erf":
        return 0.5 * z * (1 + torch.erf(z / 2 ** 0.5))
    if act == "gelu":
        t = (z / 2 ** 0.5).clamp(-3.92, 3.92)
        p, q = torch.zeros_like(t), torch.zeros_like(t)
        for a, b in zip(GELU_P, GELU_Q):
            p, q = p * t * t + a, q * t * t + b
        return 0.5 * z * (1 + t * p / q)
    return z


def sum_error(k, s):
    return (k / 16 + 16) * 2.0 ** -23 * s


def linear64(x, w, bias, residual, act, gelu):
    """(y, bound) of the projection in 64 bits, [rows, N]."""
    x2, k = x.double().reshape(-1, x.shape[-1]), x.shape[-1]
    z = x2 @ w.double().t()
    s = x2.abs() @ w.double().abs().t()
    if bias is not None:
        z, s = z + bias.double(), s + bias.double().abs()
    y = act64(z, act, gelu)
    err = sum_error(k, s) * (1.0 if act == "none" else SLOPE) + 2.0 ** -20 * (z.abs() + y.abs())
    if residual is not None:
        y = y + residual.double().reshape(y.shape)
    return y, err + EPS[x.dtype] / 2 * (y.abs() + err) + TINY[x.dtype]


def route64(x, w, top_k, scoring="softmax", choice_bias=None, renormalize=True, scale=1.0, mask=None):
    """(ids, weights) in 64 bits: stable descending order of the keys, NaN keys last."""
    logits = x.double().reshape(-1, x.shape[-1]) @ w.double().t()
    p = torch.softmax(logits, 1) if scoring == "softmax" else torch.sigmoid(logits)
    key = p if choice_bias is None else p + choice_bias.double()
    key = torch.where(key.isnan(), -torch.inf, key)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top_k]
    wt = p.gather(1, ids)
    wt = (wt / wt.sum(1, keepdim=True) if renormalize else wt) * scale
    if mask is not None:
        live = mask.reshape(-1, 1)
        ids, wt = torch.where(live, ids, -1), torch.where(live, wt, 0.0)
    return ids.to(torch.int32), wt


def moe64(x, ids, weights, w1, w2, act, gelu, residual):
    """(y, bound) of the experts' weighted sum in 64 bits, given choices [rows, k].  The hidden
    value is rounded once: half a step of it reaches the output through |W2|."""
    x2 = x.double().reshape(-1, x.shape[-1])
    m, (e, n, h), k = x2.shape[0], w2.shape, x.shape[-1]
    y = torch.zeros(m, n, dtype=torch.float64, device=x.device)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    half = EPS[x.dtype] / 2
    for i in range(e):
        token, place = torch.nonzero(ids == i, as_tuple=True)
        if not token.numel():
            continue
        a, b = w1[i].double(), w2[i].double()
        z, s = x2[token] @ a.t(), x2[token].abs() @ a.abs().t()
        hid = act64(z, act, gelu)
        dz = sum_error(k, s) + 2.0 ** -20 * z.abs()
        if act == "swiglu":
            (g, u), (dg, du) = z.chunk(2, dim=-1), dz.chunk(2, dim=-1)
            dh = SLOPE * dg * (u.abs() + du) + (g * torch.sigmoid(g)).abs() * du + 2.0 ** -20 * hid.abs()
        else:
            dh = SLOPE * dz + 2.0 ** -20 * hid.abs()
        dh = dh + half * (hid.abs() + dh) + TINY[x.dtype]
        c = weights[token, place].double()[:, None]
        y.index_add_(0, token, (hid @ b.t()) * c)
        size = hid.abs() @ b.abs().t()
        mag.index_add_(0, token, size * c.abs())
        err.index_add_(0, token, (dh @ b.abs().t() + sum_error(h, size)) * c.abs())
    err = err + 2.0 ** -20 * mag
    if residual is not None:
        y = y + residual.double().reshape(y.shape)
    return y, err + half * (y.abs() + err) + TINY[x.dtype]


def assert_within(got, ref, bound, dtype):
    got = got.double().reshape(ref.shape)
    off = (got - ref).abs()
    assert torch.isfinite(got).all()
    worst = (off - bound).max().item()
    assert worst <= 0, f"exceeds the bound by {worst} (largest error {off.max().item()})"
    # Roundings are independent, so in the 2-norm they stay within a step of the type even where
    # the worst-case sums above allow more.
    norm = ref.norm().item()
    assert off.norm().item() <= EPS[dtype] * norm + 1e-30, (off.norm().item() / norm)
