"""The layer products (GemmEpilogue, GemmActivationGradient, ActivationGradient, GemmGrouped, GemmGroupedGradient) in 64 bits,
and how far a result in the storage type may be from them.

The bounds come from the arithmetic, before any run:
  * a product of depth k summed in fp32 is off by at most (k + 8) 2^-24 times the sum of the absolute products (k roundings of
    partial sums and a few for alpha, bias and the order of additions in the matrix instruction);
  * the activations' Lipschitz constants are below 1.13, so such an error passes through them at most that much larger;
  * act(z) itself: one part in 2^16 for 16-bit results (the fitted Phi is off by 2^-17.6, the hardware's exponential by 2^-22 of
    its argument, at most 90 here: 2^-15.5 of a value below 2^-126), one part in 2^20 for fp32 (a few roundings, and the
    argument of an exponential of up to 90 rounded to 24 bits: 2^-24 * 90 < 2^-17 only where the value is below 1e-30, so an
    absolute 1e-30 is added);
  * act'(z): the same, absolutely (its values lie in -0.13 .. 1.13, sums of terms of either sign);
  * the result's rounding: half a step, relative to the value (2^-8, 2^-11, 2^-24), or half the smallest number.
"""
import math

import torch

ROUNDING = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
FUNCTION = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -16, torch.float32: 2.0 ** -20}
LIPSCHITZ = 1.13


def inner(z):
    return math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)


def phi(z):
    return torch.special.erfc(-z / math.sqrt(2)) / 2


def act(z, kind):
    if kind == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if kind == "gelu":
        return z * phi(z)
    if kind == "gelu_tanh":
        return z * torch.sigmoid(2 * inner(z))
    return z * torch.sigmoid(z) if kind == "silu" else z


def slope(z, kind):
    if kind == "relu":
        return (z > 0).double()
    if kind == "gelu":
        return phi(z) + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        s = torch.sigmoid(2 * inner(z))
        return s + z * s * torch.sigmoid(-2 * inner(z)) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
    if kind == "silu":
        s = torch.sigmoid(z)
        return s + z * s * torch.sigmoid(-z)
    return torch.ones_like(z)


def rounded(value, error, dtype):
    """Bound of a result: the error in front of the rounding, and the rounding of anything that far off"""
    return error + ROUNDING[dtype] * (value.abs() + error) + SMALLEST[dtype]


def epilogue(a, b, dtype, alpha=1.0, bias=None, kind="none", beta=0.0, residual=None):
    """(C, bound, Z, bound) for 64-bit a (m x k) and b (k x n)"""
    k = a.shape[1]
    z = alpha * (a @ b)
    size = abs(alpha) * (a.abs() @ b.abs())
    if bias is not None:
        z = z + bias
        size = size + bias.abs()
    z_error = (k + 8) * 2.0 ** -24 * size
    c = act(z, kind)
    error = LIPSCHITZ * z_error + FUNCTION[dtype] * c.abs() + (1e-30 if kind != "none" else 0.0)
    if beta != 0.0:
        c = c + beta * residual
        error = error + 2.0 ** -23 * (c.abs() + abs(beta) * residual.abs())
    return c, rounded(c, error, dtype), z, rounded(z, z_error, dtype)


def gradient(y, y_error, pre, kind, dtype):
    """(C, bound, column sums, bound) for the 64-bit gradient y in front of the activation, itself off by at most y_error"""
    s = slope(pre, kind)
    c = y * s
    error = y_error * (s.abs() + FUNCTION[dtype]) + y.abs() * (FUNCTION[dtype] if kind not in ("none", "relu") else 0.0) + 2.0 ** -23 * c.abs()
    sums = c.sum(0)
    sums_error = error.sum(0) + (c.shape[0] + 8) * 2.0 ** -24 * (c.abs() + error).sum(0)
    return c, rounded(c, error, dtype), sums, rounded(sums, sums_error, dtype)


def check(got, want, bound, what=""):
    """Every element of `got` within its bound of `want` (both may be empty)"""
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        index = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError("%s: %d of %d elements off, first at %s: %r instead of %r, off by %.3g, allowed %.3g; worst ratio %.3g" % (
            what, int(bad.sum()), bad.numel(), index, float(got[index]), float(want[index]), float(off[index]), float(bound[index]),
            float((off / bound).nan_to_num(float("inf")).max())))
