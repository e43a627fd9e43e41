"""What the dense operators refuse, and their C structs and scratch sizes: no GPU needed."""
import ctypes
import json
import os
import subprocess

import pytest
import torch

import dgprf
from dgprf import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def linear(**kw):
    a = dict(dtype=N.F32, act=0, m=4, k=8, n=16, ldx=8, ldw=16, ldr=0)
    a.update(kw)
    return N.Linear(**a)


def grad(**kw):
    a = dict(dtype=N.F32, act=0, m=4, k=8, n=16, ldx=8, ldw=16, lddy=16)
    a.update(kw)
    return N.LinearGrad(**a)


def scratch(a):
    need = ctypes.c_int64(-1)
    f = N.lib().dgprf_linear_scratch if isinstance(a, N.Linear) else N.lib().dgprf_linear_grad_scratch
    return f(ctypes.byref(a), ctypes.byref(need)), need.value


def test_struct_layout_matches_c(tmp_path):
    structs = {"dgprf_linear_t": N.Linear, "dgprf_linear_grad_t": N.LinearGrad}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{ROOT}/include/dgprf.h"', 'int main(void){',
             'printf("{\\"x\\": 0");']
    for c, cls in structs.items():
        lines += [f'printf(",\\"{c}.{f}\\": %zu", offsetof({c}, {f}));' for f, _ in cls._fields_]
        lines.append(f'printf(",\\"{c}\\": %zu", sizeof({c}));')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ['printf("}");', 'return 0;}']))
    subprocess.check_call(["gcc", "-std=c99", "-o", str(tmp_path / "layout"), str(src)])
    got = json.loads(subprocess.check_output([str(tmp_path / "layout")]))
    for c, cls in structs.items():
        assert got[c] == ctypes.sizeof(cls)
        assert all(got[f"{c}.{f}"] == getattr(cls, f).offset for f, _ in cls._fields_)


@pytest.mark.parametrize("make", [linear, grad])
@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(act=5), dict(act=-1), dict(drop_thr=-1), dict(drop_thr=65537)])
def test_arguments_refused(make, bad):
    assert scratch(make(**bad))[0] == N.E_ARG


@pytest.mark.parametrize("make", [linear, grad])
@pytest.mark.parametrize("bad", [
    dict(m=-1), dict(k=0), dict(n=0), dict(ldx=7), dict(ldw=15), dict(m=1 << 31), dict(k=(1 << 20) + 1, ldx=(1 << 20) + 1),
    dict(ldw=(1 << 20) + 1), dict(ldx=(1 << 20) + 1)])
def test_shapes_refused(make, bad):
    assert scratch(make(**bad))[0] == N.E_SHAPE


def test_row_numbers_fit():
    """Row numbers up to a tile's end fit 32 bits, and tiles a launch."""
    for make in (linear, grad):
        ones = dict(k=1, n=1, ldx=1, ldw=1)
        assert scratch(make(m=2 ** 31 - 512, **ones))[0] == 0
        assert scratch(make(m=2 ** 31 - 511, **ones))[0] == N.E_SHAPE
        assert scratch(make(m=2 ** 31 - 512, k=1, n=256, ldx=1, ldw=256))[0] == N.E_SHAPE
    some = 1 << 20  # never read
    assert N.lib().dgprf_dropout(0, some, 1, 2 ** 31 - 7, 2 ** 31, None, 0, 1, 0, 0, None, some, None) == N.E_SHAPE


def test_calls_refused_before_anything_is_enqueued():
    lib, e = N.lib(), ctypes.byref
    assert lib.dgprf_linear_forward(None, None, 0, None) == N.E_ARG
    assert lib.dgprf_linear_backward(None, None, 0, None) == N.E_ARG
    assert lib.dgprf_linear_scratch(e(linear()), None) == N.E_ARG
    assert lib.dgprf_linear_forward(e(linear()), None, 0, None) == N.E_ARG      # no tensors
    some = 1 << 20  # never read: refused on the host
    ok = dict(x=some, w=some, y=some, m=1, k=1 << 14, ldx=1 << 14)  # one row of a long K: parts to join
    assert scratch(linear(**ok)) == (0, scratch(linear(**ok))[1]) and scratch(linear(**ok))[1] > 1
    assert lib.dgprf_linear_forward(e(linear(**ok)), None, 0, None) == N.E_ARG   # scratch missing
    assert lib.dgprf_linear_forward(e(linear(**ok)), some, 1, None) == N.E_ARG   # scratch too small
    assert lib.dgprf_linear_forward(e(linear(res=some, ldr=3, **ok)), some, 1 << 30, None) == N.E_SHAPE
    assert lib.dgprf_linear_forward(e(linear(act=2, aux=some + 4, **ok)), some, 1 << 30, None) == N.E_ARG
    g = dict(x=some, w=some, dy=some, dx=some, drop_thr=1)  # dz is a tensor of its own
    assert scratch(grad(**g))[1] > 1
    assert lib.dgprf_linear_backward(e(grad(act=2, **g)), some, 1 << 30, None) == N.E_ARG  # nothing saved
    assert lib.dgprf_linear_backward(e(grad(lddy=3, **g)), some, 1 << 30, None) == N.E_SHAPE
    assert lib.dgprf_linear_backward(e(grad(**g)), None, 0, None) == N.E_ARG
    assert lib.dgprf_linear_backward(e(grad(**{**g, "w": None})), some, 1 << 30, None) == N.E_ARG
    assert lib.dgprf_dropout(9, some, 1, 8, 8, None, 0, 0, 0, 0, None, some, None) == N.E_ARG
    assert lib.dgprf_dropout(0, some, 1, 8, 8, None, 0, 65537, 0, 0, None, some, None) == N.E_ARG
    assert lib.dgprf_dropout(0, some, 2, 8, 4, None, 0, 1, 0, 0, None, some, None) == N.E_SHAPE
    assert lib.dgprf_dropout(0, some, -1, 8, 8, None, 0, 1, 0, 0, None, some, None) == N.E_SHAPE
    assert lib.dgprf_dropout(0, None, 1, 8, 8, None, 0, 1, 0, 0, None, None, None) == N.E_ARG
    # nothing to do
    assert lib.dgprf_linear_forward(e(linear(m=0)), None, 0, None) == 0
    assert lib.dgprf_dropout(0, None, 0, 8, 8, None, 0, 1, 0, 0, None, None, None) == 0


def test_python_refusals():
    x, w = torch.zeros(4, 8), torch.zeros(8, 16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dgprf.linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        dgprf.dropout(x, 0.5)
    with pytest.raises(TypeError):
        dgprf.linear(x.double(), w)
    with pytest.raises((TypeError, RuntimeError)):
        dgprf.linear([[1.0]], w)
    with pytest.raises(ValueError, match="activation"):
        dgprf.linear(x, w, activation="swish")
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            dgprf.dense.drop_threshold(p)
    assert [dgprf.dense.drop_threshold(p) for p in (0, 0.1, 0.5, 1)] == [0, 6554, 32768, 65536]


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_refused(which):
    """A dual tensor need not ask for a gradient; its tangent is not dropped silently."""
    import torch.autograd.forward_ad as fw
    args = [torch.ones(4, 8), torch.ones(8, 16), torch.ones(16), torch.ones(4, 16)]
    with fw.dual_level():
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            dgprf.linear(*args[:3], residual=args[3])
        if which in (0, 3):
            pair = [fw.make_dual(torch.ones(4, 8), torch.ones(4, 8)), torch.ones(4, 8)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                dgprf.dropout(pair[which > 0], 0.5, residual=pair[which == 0])


class _StandIn:
    """dgprf.dropout's operator on the CPU: the mask of (seed, sub) by torch's generator."""

    @staticmethod
    def dropout(x, residual, thr, seed, sub, step):
        g = torch.Generator()
        g.manual_seed((seed * 31 + sub) % 2 ** 62)
        return x * (torch.rand(x.shape, generator=g) >= thr / 65536)


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_masks(monkeypatch, reentrant):
    """A forward pass that activation checkpointing runs again draws no other mask: default numbers are
    refused there, given ones make the same mask."""
    from torch.utils.checkpoint import checkpoint
    monkeypatch.setattr(dgprf.dense.E, "ops", lambda: _StandIn)
    x = torch.linspace(-1, 1, 64).requires_grad_()

    def run(**kw):
        y = checkpoint(lambda v: dgprf.dropout(v, 0.5, **kw).square(), x, use_reentrant=reentrant)
        x.grad = None
        y.sum().backward()
        return y.detach()

    for kw in ({}, dict(seed=3), dict(step=torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="needs sub"):
            run(**kw)
    y = run(seed=3, sub=4)
    assert torch.equal(x.grad != 0, y != 0) and 0 < int((y != 0).sum()) < 64
    run(sub=4)
    # nothing to draw: no mask, and all of it
    monkeypatch.setattr(_StandIn, "dropout", staticmethod(lambda x, r, thr, *a: x * (thr == 0)))
    for p in (0.0, 1.0):
        checkpoint(lambda v: dgprf.dropout(v, p).square(), x, use_reentrant=reentrant).sum().backward()


def test_captured_masks(monkeypatch):
    """A captured call does not draw a number that all its replays would share."""
    seen = []
    monkeypatch.setattr(_StandIn, "dropout", staticmethod(lambda *a: seen.append(a)))
    monkeypatch.setattr(dgprf.dense.E, "ops", lambda: _StandIn)
    monkeypatch.setattr(dgprf.dense, "_captured", lambda x: True, raising=False)
    x, step = torch.ones(8), torch.zeros(1, dtype=torch.int64)
    for kw in ({}, dict(seed=3)):
        with pytest.raises(RuntimeError, match="needs step"):
            dgprf.dropout(x, 0.5, **kw)
    for p, kw in ((0.5, dict(step=step)), (0.5, dict(sub=2)), (0.5, dict(sub=2, step=step)), (0.0, {}), (1.0, {})):
        dgprf.dropout(x, p, **kw)
    assert len(seen) == 5


def test_layer_refusals():
    from layers import DenseLayer, DropoutLayer
    for bad in (lambda: DenseLayer(4, 8, activation="tanh"), lambda: DenseLayer(4, 8, dropout=2.0),
                lambda: DropoutLayer(-0.5)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.complex64, "float32", None])
def test_layer_types_refused(dtype):
    """When the layer is made, not at its first call."""
    from layers import DenseLayer
    with pytest.raises(TypeError, match="dtype"):
        DenseLayer(4, 8, dtype=dtype)


def test_layer_takes_its_own_device(monkeypatch):
    """A layer's input goes to where its weights are, whichever device is current."""
    from layers import DenseLayer, dense_layers
    layer, seen = DenseLayer.__new__(DenseLayer), []
    layer.in_feature, layer.out_feature, layer.activation, layer.dropout, layer.training = 4, 8, "none", 0.0, False
    layer.W, layer.b = torch.zeros(4, 8, dtype=torch.float16), None
    monkeypatch.setattr(dense_layers.E, "device", lambda: torch.device("meta"))
    monkeypatch.setattr(dense_layers, "linear", lambda x, *a: seen.append(x))
    layer(torch.zeros(3, 4))
    layer([[1.0, 2.0, 3.0, 4.0]])
    assert all(x.device == layer.W.device and x.dtype == torch.float16 for x in seen) and len(seen) == 2
    with pytest.raises(ValueError, match="X must be"):
        layer(torch.zeros(3, 5))


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU refusal")
def test_layer_needs_a_device():
    from layers import DenseLayer
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        DenseLayer(4, 8)
