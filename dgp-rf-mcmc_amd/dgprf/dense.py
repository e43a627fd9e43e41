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


def drop_threshold(p):
    """The share of 65536 that dropout of probability p drops (p is rounded to a multiple of it)."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be in [0, 1], got {p}")
    return int(p * 65536 + 0.5)


def _captured(x):
    """Whether calls on x are being captured into a graph."""
    if not (torch.is_tensor(x) and x.is_cuda) or torch._C._cuda_getCurrentRawStream(x.get_device()) == 0:
        return False  # (the null stream cannot be captured, and must not be asked while another is)
    with torch.cuda.device(x.device):
        return torch.cuda.is_current_stream_capturing()


def _stream_of(x, thr, seed, sub, step):
    """(seed, sub) of this call's mask: as given, or the global generator's key and its next
    subsequence (dgprf.set_seed makes a run's masks repeat).  With a step, the call has 2^32 of them to
    itself: step is added to sub, and no other call's masks may come up."""
    if thr == 0:
        return 0, 0
    if sub is None and thr < 65536:  # (p = 1 drops everything whatever the number)
        # A forward pass that a backward pass runs again (activation checkpointing) would draw another
        # mask than the result that it stands for was made with.
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError(
                "dgprf: dropout inside a backward pass (activation checkpointing runs the forward pass again "
                "there) needs sub given: the generator's next number would give another mask than before")
        if step is None and _captured(x):
            raise RuntimeError(
                "dgprf: dropout captured into a graph needs step (a device counter), or sub given for one mask "
                "in every replay: the generator's number would be drawn once, for all replays")
    if seed is None:
        seed = E._RNG.seed
    if sub is None:
        sub = E.next_subsequence() if step is None else (E.next_subsequence() + 1) << 32
    return E._i64(seed), E._i64(sub)


def linear(x, weight, bias=None, activation="none", residual=None, dropout=0.0, seed=None, sub=None,
           step=None):
    """y = residual + s m a(x W + b).

    x [..., k], weight [k, n] (GPLayer's layout), bias [n], residual of y's shape [..., n]; one type
    of float32, float16 and bfloat16 for all.  activation: none, relu, gelu, gelu_tanh or silu.
    dropout: the probability p of an element's being dropped, rounded to a multiple of 1 / 65536.
    seed / sub: key and number of the mask (default: the global generator, its next subsequence; a call
    that activation checkpointing runs again in the backward pass needs sub given, so that it makes the
    same mask, and raises RuntimeError without);
    step: an int64 device tensor added to sub when the kernels run, for a captured call — advance it
    after the call's backward pass, and keep given subs of different calls more than the number of
    steps apart.  A captured call with neither sub nor step raises RuntimeError (its mask would be one for
    all replays); with sub alone it repeats the mask of sub.  The gradient of the gradient is not available.
    """
    act = N.ACTS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(N.ACTS)}, got {activation!r}")
    thr = drop_threshold(dropout) if dropout else 0
    seed, sub = _stream_of(x, thr, seed, sub, step)
    return E.ops().linear(x, weight, bias, act, residual, thr, seed, sub, step)


def dropout(x, p, residual=None, seed=None, sub=None, step=None):
    """y = residual + s m x for x [..., n]: the mask of `linear`'s result of the same rows, (seed, sub)
    and n.  p = 1 drops everything.  Arguments as in `linear`."""
    thr = drop_threshold(p)
    seed, sub = _stream_of(x, thr, seed, sub, step)
    return E.ops().dropout(x, residual, thr, seed, sub, step)
