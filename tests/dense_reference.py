"""The dense operators' definition in float64 on the CPU, and how far a kernel may be from it.

Tolerances are bounds, element by element, from the roundings a kernel makes: a sum of K products in
32 bits is off by at most (K + 4) 2^-23 of the sum of the products' sizes (2^-24 for each addition
rounded to nearest, twice that allows for truncating adders inside the matrix instructions); a value
stored in a type is off by half its epsilon; an activation of 32 bits is off by ACT_ERR of its size;
16-bit backward passes take z and dz rounded to the type.
"""
import math

import numpy as np
import torch

from oracle import rng

RNG_DROPOUT = 8
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
# activations and slopes relative to max(1, |z|): the fit of the normal tail (3.4e-7 in 32 bits, 8.6e-6
# in the form for 16-bit types), and a handful of roundings of v_exp / v_rcp (1 ulp = 1.2e-7 each);
# the exponent's own rounding, e^(z^2 / 2 (1 + 2^-23)), is below 1e-6 where the result is above 1e-7
ACT_ERR = {torch.float32: 3e-6, torch.float16: 1.2e-5, torch.bfloat16: 1.2e-5}
CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "gelu_tanh": 0.85, "silu": 0.5}  # max |a''|
STEEP = 1.13  # max |a'|


def eps2(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps


def keep_mask(m, n, thr, seed, sub):
    """keep [m, n] (bool) of (seed, sub): the halves of Philox words, eight a group."""
    groups = -(-n // 8)
    w = rng.philox_words(m * groups, seed, sub, RNG_DROPOUT, 0)
    h = np.ascontiguousarray(w).view(np.uint16).reshape(m, groups * 8)[:, :n]
    return torch.from_numpy(np.ascontiguousarray(h >= thr))


def scale_of(thr):
    return 65536.0 / (65536 - thr) if thr < 65536 else 0.0


def act(z, name):
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "none":
        return torch.ones_like(z)
    z = z.detach().clone().requires_grad_()
    with torch.enable_grad():
        return torch.autograd.grad(act(z, name).sum(), z)[0]


class Linear:
    """Values and tolerances of one call; every argument is a CPU tensor of the type under test."""

    def __init__(self, x, w, b=None, name="none", r=None, thr=0, seed=0, sub=0, dy=None):
        t, d = x.dtype, lambda v: v.double()  # noqa: E731
        m, k = x.shape
        n = w.shape[1]
        x, w = d(x), d(w)
        z = x @ w
        size = x.abs() @ w.abs()
        if b is not None:
            z, size = z + d(b), size + d(b).abs()
        z_err = (k + 4) * 2.0 ** -23 * size
        s = scale_of(thr)
        keep = keep_mask(m, n, thr, seed, sub).double() if thr else torch.ones_like(z)
        a = act(z, name)
        y = keep * a * s if thr else a
        a_err = 0.0 if name in ("none", "relu") else ACT_ERR[t] * torch.clamp(z.abs(), min=1)
        err = keep * (s if thr else 1.0) * (STEEP * z_err + a_err + 2.0 ** -23 * a.abs())
        if r is not None:
            y = y + d(r)
            err = err + 2.0 ** -23 * y.abs()
        self.y, self.y_tol = y, err * 1.01 + eps2(t) * (y.abs() + err) + tiny(t)
        if dy is None:
            return
        dy = d(dy)
        g = slope(z, name)
        dz = dy * keep * (s if thr else 1.0) * g
        stored = 0.0 if name == "relu" else eps2(t) * z.abs()
        g_err = 0.0 if name in ("none", "relu") else CURVE[name] * (stored + z_err) + ACT_ERR[t] * torch.clamp(z.abs(), min=1)
        dz_err = (dy * keep).abs() * (s if thr else 1.0) * g_err + 2.0 ** -22 * dz.abs()
        in_err = dz_err + eps2(t) * (dz.abs() + dz_err) + tiny(t)  # as the products take it
        self.dx, self.dw, self.db = dz @ w.t(), x.t() @ dz, dz.sum(0)
        self.dx_tol = self._sum(self.dx, in_err @ w.abs().t(), dz.abs() @ w.abs().t(), n, t)
        self.dw_tol = self._sum(self.dw, x.abs().t() @ in_err, x.abs().t() @ dz.abs(), m, t)
        self.db_tol = self._sum(self.db, dz_err.sum(0), dz.abs().sum(0), m, t)

    @staticmethod
    def _sum(v, err, size, count, t):
        err = err + (count + 4) * 2.0 ** -23 * (size + err)
        return err + eps2(t) * (v.abs() + err) + tiny(t)


def check(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - tol).max() if got.numel() else torch.tensor(-1.0)
    if over > 0:
        at = ((got - want).abs() - tol).argmax()
        raise AssertionError(f"{what}: {got.flatten()[at]} for {want.flatten()[at]} +- "
                             f"{tol.flatten()[at]} at {int(at)} of {tuple(got.shape)}")
