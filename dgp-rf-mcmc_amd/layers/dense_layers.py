"""DenseLayer and DropoutLayer: layers trained by gradient, for the networks beside the random-feature
ones — the deterministic or MC-dropout network that a DGP is compared with, or features trained by it.

They call dgprf.linear / dgprf.dropout (one kernel for product, bias, activation, dropout and residual)
and are differentiable: torch.autograd.grad(loss, layer.trainable_variables) and
experiments.optimizers.Adam.apply_gradients train them (16-bit weights with values and moments in 32
bits).  RBFLayer, ARCLayer and GPLayer take their results as inputs but pass no gradient back: what they
return has no autograd graph, so a DenseLayer in front of them is not trained through them.  The product
is GPLayer's (X W, W [in, out]).
"""
import torch

from dgprf import _native as N
from dgprf import engine as E
from dgprf.dense import dropout, linear
from dgprf.module import Module


def _input(X, W):
    """X [..., in_feature] on the device of W (not the current one) in its type; a tensor that is, is taken
    as it is."""
    if not torch.is_tensor(X):
        X = torch.as_tensor(X)
    if X.dim() < 1 or X.shape[-1] != W.shape[0]:
        raise ValueError(f"X must be [..., {W.shape[0]}], got {tuple(X.shape)}")
    return X.to(device=W.device, dtype=W.dtype)


class DenseLayer(Module):
    """residual + D(a(X W + b)): W ~ N(0, 1 / in_feature), b = 0.

    activation: none, relu, gelu, gelu_tanh or silu; dropout: the probability of an element's being
    dropped, while set_training(True) holds; dtype: float32, float16 or bfloat16."""

    def __init__(self, in_feature, out_feature, activation="none", bias=True, dropout=0.,
                 dtype=torch.float32, name=None):
        super().__init__(name=name)
        if activation not in N.ACTS:
            raise ValueError(f"activation must be one of {', '.join(N.ACTS)}, got {activation!r}")
        if not 0. <= dropout <= 1.:
            raise ValueError(f"dropout probability must be in [0, 1], got {dropout}")
        if dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        self.in_feature, self.out_feature = int(in_feature), int(out_feature)
        self.activation, self.dropout, self.training = activation, float(dropout), False
        w = E.normal((self.in_feature, self.out_feature), N.RNG_W) * self.in_feature ** -0.5
        self.W = w.to(dtype).requires_grad_()
        self.W.trainable, self.W.var_name = True, "dense_layer_W"
        self.b = None
        if bias:
            self.b = torch.zeros(self.out_feature, dtype=dtype, device=w.device, requires_grad=True)
            self.b.trainable, self.b.var_name = True, "dense_layer_b"

    def __call__(self, X, residual=None, seed=None, sub=None, step=None):
        """X [..., in_feature] -> [..., out_feature]; seed, sub, step: the mask's, as in dgprf.linear."""
        X = _input(X, self.W)
        return linear(X, self.W, self.b, self.activation, residual,
                      self.dropout if self.training else 0., seed, sub, step)

    def set_training(self, state):
        self.training = bool(state)


class DropoutLayer(Module):
    """residual + D(X), while set_training(True) holds; X as it is (plus the residual) otherwise."""

    def __init__(self, p, name=None):
        super().__init__(name=name)
        if not 0. <= p <= 1.:
            raise ValueError(f"dropout probability must be in [0, 1], got {p}")
        self.p, self.training = float(p), False

    def __call__(self, X, residual=None, seed=None, sub=None, step=None):
        if self.training:
            return dropout(X, self.p, residual, seed, sub, step)
        return X if residual is None else X + residual

    def set_training(self, state):
        self.training = bool(state)
