"""Dense operators: a matrix product with bias, activation, dropout and residual in its epilogue, and
dropout whose mask comes from the counter-based generator and is never stored.

    z = x W + b        linear:   y = r + s m a(z)        dropout:  y = r + s m x

Both are differentiable (torch.autograd); the backward pass makes the mask again from the same
counters.  They run on torch's current stream of the tensors' device and can be captured by
torch.cuda.graph.  include/dgprf.h (dgprf_linear_t) has the definition of the mask.
"""
import torch

from . import _native as N
from . import engine as E

_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def drop_threshold(p):
    """The share of 65536 that dropout of probability p drops (p is rounded to a multiple of it)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    return int(p * 65536 + 0.5)


def _stream_of(thr, seed, sub):
    """(seed, sub) of this call's mask: as given, or the global generator's key and its next
    subsequence (dgprf.set_seed makes a run's masks repeat)."""
    if thr == 0:
        return 0, 0
    if seed is None:
        seed = E._RNG.seed
    if sub is None:
        sub = E.next_subsequence()
    return E._i64(seed), E._i64(sub)


def _check(name, t):
    if not torch.is_tensor(t):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} is on {t.device}: the dense operators need a HIP device "
                           "(there is no CPU fallback)")


def _rows(t, n):
    """[..., n] as a matrix with unit stride within a row (a view where the strides allow one)."""
    t = t.reshape(-1, n) if t.dim() != 2 else t
    return t if n <= 1 or t.stride(1) == 1 else t.contiguous()


def _row_strides(t):
    """A matrix the kernels can read: rows apart by 0 or by their length and more."""
    s = t.stride(0)
    return t if t.size(0) <= 1 or s == 0 or s >= t.size(1) else t.contiguous()


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, res, act, thr, seed, sub, step):
        save = any(ctx.needs_input_grad[:3])
        y, aux = E.ops().linear(x, w, bias, act, res, thr, seed, sub, step, save)
        ctx.save_for_backward(x, w, aux if act else None, step)
        ctx.args = act, thr, seed, sub
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, aux, step = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            d = _row_strides(_rows(dy, w.shape[1]))
            dx, dw, db = E.ops().linear_backward(d, x, w, aux, *ctx.args, step, *need[:3])
        return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None,
                dy if need[3] else None, None, None, None, None, None)


def linear(x, weight, bias=None, activation="none", residual=None, dropout=0.0, seed=None, sub=None,
           step=None):
    """y = residual + s m a(x W + b).

    x [..., k], weight [k, n] (GPLayer's layout), bias [n], residual of y's shape [..., n]; one type
    of float32, float16 and bfloat16 for all.  activation: none, relu, gelu, gelu_tanh or silu.
    dropout: the probability p of an element's being dropped, rounded to a multiple of 1 / 65536.
    seed / sub: key and number of the mask (default: the global generator, its next subsequence);
    step: an int64 device tensor added to sub when the kernels run, for a captured call — advance it
    after the call's backward pass.  The gradient of the gradient is not available.
    """
    for name, t in (("x", x), ("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None:
            _check(name, t)
    if activation not in N.ACTS:
        raise ValueError(f"activation must be one of {', '.join(N.ACTS)}, got {activation!r}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[0]:
        raise ValueError(f"x [..., k] and weight [k, n] do not fit: {tuple(x.shape)}, "
                         f"{tuple(weight.shape)}")
    k, n = weight.shape
    if k < 1 or n < 1:
        raise ValueError(f"weight must not be empty, got {tuple(weight.shape)}")
    shape = (*x.shape[:-1], n)
    if residual is not None:
        if tuple(residual.shape) != shape:
            raise ValueError(f"residual must have the result's shape {shape}, got "
                             f"{tuple(residual.shape)}")
        residual = _row_strides(_rows(residual, n))
    if bias is not None:
        if tuple(bias.shape) != (n,):
            raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
        bias = bias.contiguous()
    thr = drop_threshold(dropout)
    seed, sub = _stream_of(thr, seed, sub)
    x2, w = _rows(x, k), _rows(weight, n)
    x2 = x2 if x2.stride(0) >= k or x2.size(0) <= 1 else x2.contiguous()
    w = w if w.stride(0) >= n or k <= 1 else w.contiguous()
    act = N.ACTS[activation]
    if thr == 0:
        step = None
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        y = _Linear.apply(x2, w, bias, residual, act, thr, seed, sub, step)
    else:
        y = E.ops().linear(x2, w, bias, act, residual, thr, seed, sub, step, False)[0]
    return y if len(shape) == 2 else y.view(shape)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, thr, seed, sub, step):
        ctx.save_for_backward(step)
        ctx.args = thr, seed, sub
        return E.ops().dropout(x, res, thr, seed, sub, step)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (step,) = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            d = _row_strides(_rows(dy, dy.shape[1]))
            dx = E.ops().dropout(d, None, *ctx.args, step)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(x, p, residual=None, seed=None, sub=None, step=None):
    """y = residual + s m x for x [..., n]: the mask of `linear`'s result of the same rows, (seed, sub)
    and n.  p = 1 drops everything.  Arguments as in `linear`."""
    _check("x", x)
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    thr = drop_threshold(p)
    if residual is not None:
        _check("residual", residual)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got "
                             f"{tuple(residual.shape)}")
    if x.numel() == 0:
        return x.clone() if residual is None else x + residual
    n = x.shape[-1]
    seed, sub = _stream_of(thr, seed, sub)
    x2 = _row_strides(_rows(x, n))
    r2 = None if residual is None else _row_strides(_rows(residual, n))
    if thr == 0:
        step = None
    if torch.is_grad_enabled() and (x.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        y = _Dropout.apply(x2, r2, thr, seed, sub, step)
    else:
        y = E.ops().dropout(x2, r2, thr, seed, sub, step)
    return y if x.dim() == 2 else y.view(x.shape)
