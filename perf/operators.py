"""What the dense operators are measured on: the matrix product with bias, activation, dropout and
residual in its epilogue (``dgprf.linear``), and dropout from the counter-based generator
(``dgprf.dropout``), forward and backward.

With x [M, K], W [K, N], b [N], r [M, N] and an activation a:

    z = x W + b        y = r + s m a(z)        dropout:  y = r + s m x

m is 0 for a share p = T / 65536 of the elements (T = round(65536 p)) and 1 for the others,
s = 65536 / (65536 - T).  m is never stored: it comes from Philox4x32-10 with the key `seed`.  The
eight elements 8 g .. 8 g + 7 of row i share the call whose counter is (q mod 2^32, sub mod 2^32,
sub div 2^32, 8 2^24 + q div 2^32), q = i ceil(N / 8) + g; element e of them takes the half e mod 2
(0: the low one) of output word e div 2, and is kept when that half is >= T.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def listed():
    """Twelve cases: the single token, small batches, prompts, training passes, dropout alone and
    both operators as a network uses them."""
    return [
        # one token through an up-projection while serving: W is read once, little is computed
        dict(name="token", op="linear", type="bf16", m=1, k=2048, n=8192, act="gelu", bias=True, res=False),
        # a decoding batch's down-projection onto the residual stream
        dict(name="decode batch", op="linear", type="fp16", m=24, k=8192, n=2048, act="none", bias=True, res=True),
        # a whole prompt through one hidden layer
        dict(name="prompt", op="linear", type="bf16", m=4096, k=4096, n=4096, act="gelu_tanh", bias=True, res=False),
        # a prompt whose length, inputs and outputs fit no tile, rows of odd length
        dict(name="prompt odd", op="linear", type="bf16", m=1777, k=1001, n=2049, act="silu", bias=True, res=True),
        # this repository's minibatch (200 rows of 784 pixels, 4096 features), in the type of its engine
        dict(name="pixels", op="linear", type="fp32", m=200, k=784, n=4096, act="relu", bias=False, res=False),
        # a training step's up-projection, with all gradients
        dict(name="train up", op="train", type="bf16", m=8192, k=2048, n=8192, act="gelu", bias=True, res=False, p=0.1),
        # a training step's down-projection onto the residual stream
        dict(name="train down", op="train", type="bf16", m=8192, k=8192, n=2048, act="none", bias=True, res=True, p=0.1),
        # the same in 32 bits, a minibatch of 1024 rows (one of this repository's batch sizes) of 784 pixels
        dict(name="train fp32", op="train", type="fp32", m=1024, k=784, n=2000, act="gelu", bias=True, res=False, p=0.25),
        # a ragged batch with odd widths in the narrow-range type
        dict(name="train odd", op="train", type="fp16", m=777, k=515, n=1283, act="silu", bias=True, res=True, p=0.5),
        # dropout of a minibatch's 1024 features: the smallest call
        dict(name="dropout small", op="dropout", type="fp32", m=200, n=1024, res=False, p=0.5),
        # dropout of a long batch's hidden states onto the residual stream
        dict(name="dropout long", op="dropout", type="bf16", m=16384, n=8192, res=True, p=0.1),
        # the two projections of a block in a training step, one after the other
        dict(name="block", op="block", type="bf16", m=4096, k=2048, n=8192, act="gelu_tanh", bias=True, res=True, p=0.1),
    ]


def _size(rng, low, high):
    """A size between low and high, even over the logarithm, every other one a multiple of 64, 8 or 1."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    to = rng.choice((1, 1, 8, 64))
    return min(high, max(low, v // to * to))


def draw(rng):
    op = rng.choice(("linear", "linear", "train", "train", "dropout", "block"))
    c = dict(op=op, type=rng.choice(("bf16", "fp16", "fp32")))
    if op == "dropout":
        return dict(c, m=_size(rng, 1, 16384), n=_size(rng, 64, 8192), res=rng.random() < 0.5,
                    p=rng.choice((0.05, 0.1, 0.25, 0.5)))
    top = 8192 if op != "block" else 4096
    c.update(m=_size(rng, 1, top), k=_size(rng, 64, 8192 if op != "block" else 2048), n=_size(rng, 64, 8192),
             act=rng.choice(ACTS), bias=rng.random() < 0.75, res=rng.random() < 0.5)
    while c["m"] * c["k"] * c["n"] > 2 ** 36:
        c["k"] = max(64, c["k"] // 2)
    if op != "linear":
        c["p"] = rng.choice((0.0, 0.1, 0.25, 0.5))
        if c["type"] == "fp32" and c["act"] == "relu":
            # its slope jumps at z = 0, where sums in 32 bits fall on one side or the other by their
            # order alone: one of them moves a whole row of dx by more than the type's error
            c["act"] = "silu"
    return c


def prepare(case, seed):
    """Activations of unit size, weights that keep it, a small bias and the gradient that comes
    from above; the key and the call's number of the generator."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    t, m, n = TYPES[case["type"]], case["m"], case["n"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    s = dict(case, seed=(int(seed) * 0x9E3779B97F4A7C15) % 2 ** 64, sub=int(seed) % 1000 + 2 ** 33)
    grad = case["op"] != "linear"
    if case["op"] == "dropout":
        s["x"] = normal(m, n).requires_grad_()
        s["r"] = normal(m, n).requires_grad_() if case["res"] else None
        s["dy"] = normal(m, n)
        return s
    k = case["k"]
    s["x"] = normal(m, k)
    s["w"] = normal(k, n, scale=k ** -0.5)
    s["b"] = normal(n, scale=0.1) if case["bias"] else None
    if case["op"] == "block":
        s["w2"] = normal(n, k, scale=n ** -0.5)
        s["b2"] = normal(k, scale=0.1) if case["bias"] else None
        s["dy"] = normal(m, k)
    else:
        s["r"] = normal(m, n) if case["res"] else None
        s["dy"] = normal(m, n) if grad else None
    if grad:
        for key in ("x", "w", "b", "w2", "b2", "r"):
            if s.get(key) is not None:
                s[key].requires_grad_()
    return s


# ---------------------------------------------------------------- the framework's calls
_dgprf = None


def _framework():
    global _dgprf
    if _dgprf is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dgp-rf-mcmc_amd")
        if at not in sys.path:
            sys.path.insert(0, at)
        import dgprf
        _dgprf = dgprf
    return _dgprf


def _grads(y, dy, named):
    named = {k: v for k, v in named.items() if v is not None}
    got = torch.autograd.grad(y, list(named.values()), dy)
    return {"y": y, **{"d" + k: v for k, v in zip(named, got)}}


def _run_own(s):
    f = _framework()
    rand = dict(seed=s["seed"], sub=s["sub"])
    if s["op"] == "dropout":
        y = f.dropout(s["x"], s["p"], residual=s["r"], **rand)
        return _grads(y, s["dy"], {"x": s["x"], "r": s["r"]})
    if s["op"] == "linear":
        return {"y": f.linear(s["x"], s["w"], s["b"], activation=s["act"], residual=s["r"])}
    if s["op"] == "train":
        y = f.linear(s["x"], s["w"], s["b"], activation=s["act"], residual=s["r"], dropout=s["p"], **rand)
        return _grads(y, s["dy"], {"x": s["x"], "w": s["w"], "b": s["b"], "r": s["r"]})
    h = f.linear(s["x"], s["w"], s["b"], activation=s["act"], dropout=s["p"], **rand)
    y = f.linear(h, s["w2"], s["b2"], residual=s["x"] if s["res"] else None, dropout=s["p"], seed=s["seed"],
                 sub=s["sub"] + 1)
    return _grads(y, s["dy"], {"x": s["x"], "w": s["w"], "b": s["b"], "w2": s["w2"], "b2": s["b2"]})


# ---------------------------------------------------------------- the plain form
LOW = 0xFFFFFFFF


def _keep(m, n, p, seed, sub, device):
    """(keep [m, n], scale).  A product of two 32-bit numbers wraps in int64, but its low half and,
    shifted and masked, its high half come out right."""
    t = int(p * 65536 + 0.5)
    groups = (n + 7) // 8
    q = torch.arange(m * groups, dtype=torch.int64, device=device)
    x, y = q & LOW, torch.full_like(q, sub & LOW)
    z, w = torch.full_like(q, sub >> 32), (q >> 32) | (8 << 24)
    k0, k1 = seed & LOW, seed >> 32
    for _ in range(10):  # the generator's rounds
        a, b = x * 0xD2511F53, z * 0xCD9E8D57
        x, y, z, w = ((b >> 32) & LOW) ^ y ^ k0, b & LOW, ((a >> 32) & LOW) ^ w ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack((x, y, z, w), dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1)
    return (halves >= t).reshape(m, groups * 8)[:, :n], 65536.0 / (65536 - t)


def _drop(v, keep, scale):
    return v if keep is None else torch.where(keep, v * scale, torch.zeros_like(v))


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        u = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + u) + 0.5 * z * (1 - u * u) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        g = 1 / (1 + torch.exp(-z))
        return g * (1 + z * (1 - g))
    return torch.ones_like(z)


def _plain_linear(x, w, b, r, act, p, seed, sub):
    """y in the inputs' type, and what its backward pass takes."""
    z = x.float() @ w.float()
    if b is not None:
        z = z + b.float()
    keep, scale = _keep(*z.shape, p, seed, sub, z.device) if p else (None, 1.0)
    y = _drop(_act(z, act), keep, scale)
    if r is not None:
        y = y + r.float()
    return y.to(x.dtype), (z, keep, scale)


def _plain_backward(dy, x, w, act, kept):
    z, keep, scale = kept
    dz = _drop(dy.float(), keep, scale) * _slope(z, act)
    return (dz @ w.float().t()).to(x.dtype), (x.float().t() @ dz).to(w.dtype), dz.sum(0).to(w.dtype)


@torch.no_grad()
def _run_plain(s):
    dy = s.get("dy")
    if s["op"] == "dropout":
        keep, scale = _keep(s["m"], s["n"], s["p"], s["seed"], s["sub"], dy.device)
        y = _drop(s["x"].float(), keep, scale)
        y = (y if s["r"] is None else y + s["r"].float()).to(dy.dtype)
        return {"y": y, "dx": _drop(dy.float(), keep, scale).to(dy.dtype), **({} if s["r"] is None else {"dr": dy})}
    if s["op"] == "linear":
        return {"y": _plain_linear(s["x"], s["w"], s["b"], s["r"], s["act"], 0.0, 0, 0)[0]}
    if s["op"] == "train":
        y, kept = _plain_linear(s["x"], s["w"], s["b"], s["r"], s["act"], s["p"], s["seed"], s["sub"])
        dx, dw, db = _plain_backward(dy, s["x"], s["w"], s["act"], kept)
        return {"y": y, "dx": dx, "dw": dw, **({} if s["b"] is None else {"db": db}),
                **({} if s["r"] is None else {"dr": dy})}
    res = s["x"] if s["res"] else None
    h, kept = _plain_linear(s["x"], s["w"], s["b"], None, s["act"], s["p"], s["seed"], s["sub"])
    y, kept2 = _plain_linear(h, s["w2"], s["b2"], res, "none", s["p"], s["seed"], s["sub"] + 1)
    dh, dw2, db2 = _plain_backward(dy, h, s["w2"], "none", kept2)
    dx, dw, db = _plain_backward(dh, s["x"], s["w"], s["act"], kept)
    if s["res"]:
        dx = (dx.float() + dy.float()).to(dx.dtype)
    return {"y": y, "dx": dx, "dw": dw, "dw2": dw2, **({} if s["b"] is None else {"db": db, "db2": db2})}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- what it costs, and the exact values
def work(case):
    size = TYPES[case["type"]].itemsize
    m, n, k = case["m"], case["n"], case.get("k", 0)
    res, bias = m * n * bool(case["res"]), bool(case.get("bias"))
    if case["op"] == "dropout":  # x, dy read, y, dx written; eight elements cost ten rounds of ten operations
        return {"bytes": size * (4 * m * n + res), "flops": 2 * m * n * 13}
    if case["op"] == "linear":
        return {"bytes": size * (m * k + k * n + n * bias + res + m * n), "flops": 2 * m * n * k}
    if case["op"] == "train":  # x, W, b, r, dy read; y, dx, dW, db written
        return {"bytes": size * (2 * m * k + 2 * k * n + 2 * n * bias + res + 2 * m * n), "flops": 6 * m * n * k}
    # x, W, W2, b, b2, dy read; y, dx and the gradients of the four weights written
    return {"bytes": size * (4 * m * k + 4 * k * n + 2 * (n + k) * bias), "flops": 12 * m * n * k}


def _exact_keep(m, n, p, seed, sub):
    t, groups = int(p * 65536 + 0.5), -(-n // 8)
    c = [np.arange(m * groups, dtype=np.uint64), np.uint64(sub % 2 ** 32), np.uint64(sub // 2 ** 32), np.uint64(8 << 24)]
    c[3] = c[3] + c[0] // np.uint64(2 ** 32)
    c[0] = c[0] % np.uint64(2 ** 32)
    key, low, half = [seed % 2 ** 32, seed // 2 ** 32], np.uint64(2 ** 32 - 1), np.uint64(32)
    for i in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        k0, k1 = ((key[j] + i * (0x9E3779B9, 0xBB67AE85)[j]) % 2 ** 32 for j in (0, 1))
        c = [(b >> half) ^ c[1] ^ np.uint64(k0), b & low, (a >> half) ^ c[3] ^ np.uint64(k1), a & low]
    halves = np.stack([v.astype(np.uint32) for v in c], axis=1).view(np.uint16)
    keep = (halves >= t).reshape(m, 8 * groups)[:, :n]
    return torch.from_numpy(np.ascontiguousarray(keep)).cuda(), 1.0 / (1.0 - t / 65536.0)


def _exact_linear(x, w, b, r, act, p, seed, sub):
    z = torch.matmul(x, w)
    z = z if b is None else z + b
    if act == "relu":
        y = z * (z > 0)
    elif act == "gelu":
        y = z * torch.special.ndtr(z)
    elif act == "gelu_tanh":
        y = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    else:
        y = z * torch.sigmoid(z) if act == "silu" else z
    if p:
        keep, scale = _exact_keep(*z.shape, p, seed, sub)
        y = y * keep * scale
    return y if r is None else y + r


def exact(case, seed):
    """The definition in 64 bits, its gradients by torch's own differentiation."""
    s = prepare(case, seed)
    v = {k: s[k].detach().double().requires_grad_(case["op"] != "linear") if s.get(k) is not None else None
         for k in ("x", "w", "b", "w2", "b2", "r")}
    p, rand = case.get("p", 0.0), (s["seed"], s["sub"])
    if case["op"] == "dropout":
        keep, scale = _exact_keep(case["m"], case["n"], p, *rand)
        y = v["x"] * keep * scale
        y = y if v["r"] is None else y + v["r"]
    elif case["op"] == "block":
        h = _exact_linear(v["x"], v["w"], v["b"], None, case["act"], p, *rand)
        y = _exact_linear(h, v["w2"], v["b2"], v["x"] if case["res"] else None, "none", p, rand[0], rand[1] + 1)
    else:
        y = _exact_linear(v["x"], v["w"], v["b"], v["r"], case["act"], p, *rand)
    if case["op"] == "linear":
        return {"y": y}
    named = {k: t for k, t in v.items() if t is not None}
    got = torch.autograd.grad(y, list(named.values()), s["dy"].double())
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(named, got)}}
