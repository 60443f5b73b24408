"""The dense feed-forward operators written down plainly in 64 bits, forward and backward, and how far a 16-bit result may lie
from them.

Tolerances count roundings. h is half a step of the type (bf16 2^-8, fp16 2^-11: eps / 2 relative to the value). A product of K
terms adds in fp32: on the tensor cores one truncation of at most 2^-23 of the running sum for each 16 terms and a few inside
them, (K / 16 + 8) 2^-23 of the sum of magnitudes; on CUDA cores K roundings of 2^-24. The hardware's exp2 and reciprocal are
good to about 2^-21 each; functions built from them are given 2^-19 of the magnitudes that they are made of.
"""
import math

import torch

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
APPROX = 2.0 ** -19


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the subnormals (results that small are rounded absolutely); bf16 results may also lose a flushed one."""
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def sum_error(K, impl="tcgen05"):
    return K * 2.0 ** -24 if impl == "simt" else (K / 16 + 8) * 2.0 ** -23


def project(x, w, b=None):
    """(z, sum of magnitudes behind each z)"""
    x, w = x.double(), w.double()
    z, m = x @ w.T, x.abs() @ w.abs().T
    return (z, m) if b is None else (z + b.double(), m + b.double().abs())


def gated(z, kind="swiglu", limit=0.0, beta=4.0, linear_beta=25.0):
    """(h, gate, up, dh/dg, dh/du, and the magnitudes that the three are made of) from the pre-activations in 64 bits."""
    n = z.shape[1] // 2
    g, u = z[:, :n], z[:, n:]
    if kind == "situ":
        p, a = torch.sigmoid(g), torch.tanh(g / beta)
        b = torch.tanh(u / linear_beta) if linear_beta > 0 else None
        gate, up, slope_u = beta * a * p, (u if b is None else linear_beta * b), (1.0 if b is None else 1 - b * b)
        return gate * up, up * ((1 - a * a) * p + beta * a * p * (1 - p)), gate * slope_u, \
            (gate * up).abs(), up.abs() * (1 + beta), torch.full_like(g, beta)
    gc, uc = (g.clamp(max=limit), u.clamp(-limit, limit)) if limit > 0 else (g, u)
    p = torch.sigmoid(gc)
    gate = gc * p
    dg, du = uc * (p + gate * (1 - p)), gate
    if limit > 0:
        dg, du = torch.where(g > limit, 0.0, dg), torch.where(u.abs() > limit, 0.0, du)
    return gate * uc, dg, du, (gate * uc).abs(), uc.abs() * (1 + gc.abs()), gc.abs()


def gated_slopes_bound(z, kind, limit, beta=4.0, linear_beta=25.0):
    """How much h moves with the pre-activations: |dh/dg| and |dh/du| are at most these near z."""
    n = z.shape[1] // 2
    g, u = z[:, :n].abs() + 0.1, z[:, n:].abs() + 0.1
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(max=limit)
    if kind == "situ":
        up = u.clamp(max=linear_beta) if linear_beta > 0 else u
        return up * (1.2 + beta / 4), g.clamp(max=beta)
    return 1.1 * u, g


def linear_act(z, act):
    """(value, slope)"""
    if act in (None, "none"):
        return z, torch.ones_like(z)
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)


def gradients(dz, dz_error, x, w, dtype, impl="tcgen05"):
    """dx, dw, db from the gradient of the pre-activations in 64 bits and its error before it is rounded: [(value, bound)] * 3.
    The operand of the products is rounded once more (h), db sums unrounded in fp32."""
    h, x, w = half_step(dtype), x.double(), w.double()
    operand = dz_error + h * (dz.abs() + dz_error) + tiny(dtype)
    out = []
    for value, error, mags, K in ((dz @ w, operand @ w.abs(), dz.abs() @ w.abs(), w.shape[0]),
                                  (dz.T @ x, operand.T @ x.abs(), dz.T.abs() @ x.abs(), x.shape[0]),
                                  (dz.sum(0), dz_error.sum(0), dz.abs().sum(0), x.shape[0])):
        error = error + 1.01 * (sum_error(K, "simt" if value.dim() == 1 else impl) + 2.0 ** -23) * (mags + error)
        out.append((value, error + h * (value.abs() + error) + tiny(dtype)))
    return out


def assert_within(got, value, bound, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN in other places"
    off = (got - value).abs()
    bad = ~((off <= bound) | torch.isnan(value) | (got == value))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off / bound)[bad].max()):.3g} x its bound"
