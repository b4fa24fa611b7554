"""The feed-forward operators and their gradients in 64 bits, and the error bounds that the tests hold the kernels to.

Half a rounding step relative to the value is eps / 2: bf16 2^-8, fp32 2^-24. A sum of fp32 terms whose longest chain of
additions is d is off by at most d * 2^-24 * sum of absolute terms; the tensor core may cut instead of round, so its
additions count 2^-23 each.
"""
import math

import torch

H32, H16 = 2.0 ** -24, 2.0 ** -8


def half_step(dtype):
    return H16 if dtype == torch.bfloat16 else H32


def act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "silu":
        return z * torch.special.expit(z)
    if name == "sigmoid":
        return torch.special.expit(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z * torch.special.expit(math.sqrt(8 / math.pi) * (z + 0.044715 * z ** 3))


def slope(z, name):
    z = z.detach().clone().requires_grad_(True)
    if name == "relu":
        return (z > 0).double().detach()
    act(z, name).sum().backward()
    return z.grad.detach() if z.grad is not None else torch.ones_like(z)


# The slopes of all activations here are at most 1.13 in absolute value (gelu: 1.129 at sqrt(2)). Their second
# derivatives stay below 1.0. exp2 and the reciprocal are good to 2 ulp each and the argument of exp2 is scaled in fp32
# (|z| 2^-24 relative, and z s(1-s) |z| <= 1): value and slope are off by at most 8 * 2^-23 (1 + |value|).
SLOPE = 1.13
ACT_ERR = 8 * 2.0 ** -23


def project(x, w, bias):
    """z and the bound on an fp32 accumulator's error."""
    z = x.double() @ w.double()
    e = (x.shape[1] + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs())
    if bias is not None:
        z = z + bias.double()
        e = e + 2.0 ** -23 * z.abs()
    return z, e


def check(got, want, bound, what):
    """Every element within its bound (no element may be compared with a NaN: those must agree)."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaNs in other places"
    far = ((got - want).abs() > bound) & ~nan & ~(got == want)
    if far.any():
        i = int(torch.nonzero(far.reshape(-1))[0])
        raise AssertionError(f"{what}: {int(far.sum())} of {far.numel()} off, first at {i}: got {got.reshape(-1)[i]}, "
                             f"want {want.reshape(-1)[i]}, bound {bound.expand_as(want).reshape(-1)[i]}")


def check_norm(got, want, bound, what):
    """Frobenius norm of the difference."""
    off = float(torch.linalg.norm(got.double() - want))
    assert off <= bound, f"{what}: off by {off} in norm, bound {bound}"


def spectral(m):
    return float(torch.linalg.matrix_norm(m.double(), 2))


def layernorm(x, gamma, beta, eps):
    """y, mean, rstd and the bounds of their fp32 evaluation (before y's own rounding)."""
    x64, n = x.double(), x.shape[-1]
    mean = x64.mean(-1, keepdim=True)
    var = (x64 - mean).square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    u = (x64 - mean) * rstd
    y = u * gamma.double() + beta.double()
    depth = 64 + n / 256
    e_mean = depth * H32 * x64.abs().mean(-1, keepdim=True) + H32 * mean.abs()
    # sums around a point at most one standard deviation from the mean keep var to (depth + 8) 2^-24 * 4
    e_rstd = rstd * (4 * (depth + 8) * H32 + 4 * H32)
    e_u = rstd * (e_mean + 2 * H32 * (x64.abs() + mean.abs())) + u.abs() * (e_rstd / rstd + 2 * H32)
    e_y = gamma.double().abs() * e_u + 3 * H32 * (y.abs() + beta.double().abs())
    return y, mean[..., 0], rstd[..., 0], e_y, e_mean[..., 0], e_rstd[..., 0]


def layernorm_grads(dy, x, gamma, mean, rstd):
    """(dx, dgamma, dbeta) from the given statistics, and the bounds of their fp32 evaluation."""
    x64, d, g, n = x.double(), dy.double(), gamma.double(), x.shape[-1]
    mu, rs = mean.double()[..., None], rstd.double()[..., None]
    u, w = (x64 - mu) * rs, d * g
    c1, c2 = w.mean(-1, keepdim=True), (w * u).mean(-1, keepdim=True)
    dx = rs * (w - c1 - u * c2)
    e_u = 3 * H32 * (x64.abs() + mu.abs()) * rs
    depth = 64 + n / 256
    e_c1 = (depth + 2) * H32 * w.abs().mean(-1, keepdim=True)
    e_c2 = (depth + 3) * H32 * (w * u).abs().mean(-1, keepdim=True) + (w.abs() * e_u).mean(-1, keepdim=True)
    e_dx = rs * (4 * H32 * (w.abs() + c1.abs() + (u * c2).abs()) + e_c1 + u.abs() * e_c2 + c2.abs() * e_u)
    flat = lambda t: t.reshape(-1, n)  # noqa: E731
    rows = flat(x64).shape[0]
    chain = 64 + rows / 32
    dgamma, dbeta = flat(d * u).sum(0), flat(d).sum(0)
    e_dgamma = (chain + 2) * H32 * flat((d * u).abs()).sum(0) + flat(d.abs() * e_u).sum(0)
    e_dbeta = chain * H32 * flat(d.abs()).sum(0)
    return dx, dgamma, dbeta, e_dx, e_dgamma, e_dbeta
