"""Plain 64-bit implementations of the sequence operators (CPU), step by step from their definitions, and the rounding
bounds that the tests hold the kernels to."""
from __future__ import annotations

import torch

SEGMENT = 512   # steps over which the decay gradient takes the difference of two running sums


def make(seed, B, L, H, Hkv, Dk, Dv, dtype, *, decay="step", state=False, lengths=None, rate=0.3):
    """Operands on the CPU in 64 bits, already rounded to the types that the operator takes."""
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape, to=dtype):
        return torch.randn(*shape, generator=gen, dtype=torch.float64).to(to).double()

    sums = torch.float64 if dtype == torch.float64 else torch.float32
    c = {"q": normal(B, L, H, Dk), "k": normal(B, L, Hkv, Dk), "v": normal(B, L, Hkv, Dv)}
    if decay == "head":
        g = -rate * torch.rand(H, generator=gen, dtype=torch.float64)
    else:
        g = -2 * rate * torch.rand(B, L, H, generator=gen, dtype=torch.float64) ** 3
        if decay == "forget":   # steps that forget everything, some next to each other, the first and last among them
            g[torch.rand(B, L, H, generator=gen) < 0.15] = -float("inf")
            g[:, :1] = -float("inf")
            g[:, -1:] = -float("inf")
        elif decay == "strong":
            g = g * 200
        elif decay == "none":
            g = torch.zeros_like(g)
    c["log_decay"] = g.to(sums).double()
    c["initial_state"] = normal(B, H, Dk, Dv, to=sums) if state else None
    c["lengths"] = lengths
    c["grad_out"] = normal(B, L, H, Dv)
    c["grad_state"] = normal(B, H, Dk, Dv, to=sums) if state else None
    c["scale"] = Dk ** -0.5
    return c


def absolute(c):
    """The same case with absolute values: every sum below then is the sum of the absolute values of its terms."""
    return {n: t.abs() if isinstance(t, torch.Tensor) and n not in ("log_decay", "lengths") else abs(t) if n == "scale" else t
            for n, t in c.items()}


def attention(c, sign=-1.0):
    """Outputs and gradients by the recurrences, one step after another.  ``sign`` is that of the y terms in
    ``pairs`` (x - y per step; +1 for bounds)."""
    q, k, v, scale = c["q"], c["k"], c["v"], c["scale"]
    B, L, H, Dk = q.shape
    Dv, share = v.shape[-1], H // k.shape[2]
    k, v = k.repeat_interleave(share, 2), v.repeat_interleave(share, 2)
    g = c["log_decay"] if c["log_decay"].dim() == 3 else c["log_decay"].expand(B, L, H)
    n = torch.full((B,), L) if c["lengths"] is None else c["lengths"].clamp(0, L).cpu()
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64) if c["initial_state"] is None else c["initial_state"]
    zero = torch.zeros(())
    states, out = [S], torch.zeros(B, L, H, Dv, dtype=torch.float64)
    for t in range(L):
        live = (t < n)[:, None, None]
        kt, vt, qt = (torch.where(live, x[:, t], zero.double()) for x in (k, v, q))
        w = torch.where(live[..., 0], g[:, t], zero.double()).exp()
        S = torch.where(w[..., None, None] == 0, zero.double(), S) * w[..., None, None] + kt[..., :, None] * vt[..., None, :]
        states.append(S)
        out[:, t] = scale * torch.einsum("bhi,bhij->bhj", qt, S)
    got = {"out": out, "state": S}
    A = torch.zeros_like(S) if c["grad_state"] is None else c["grad_state"]
    dq, dk, dv = (torch.zeros(B, L, H, d, dtype=torch.float64) for d in (Dk, Dk, Dv))
    dg, pairs, across = (torch.zeros(B, L, H, dtype=torch.float64) for _ in range(3))
    for t in reversed(range(L)):
        live = (t < n)[:, None, None]
        kt, vt, qt, gt = (torch.where(live, x[:, t], zero.double()) for x in (k, v, q, c["grad_out"]))
        across[:, t] = (A * states[t + 1]).sum((-1, -2))      # pairs that go across the end of step t
        A = A + scale * qt[..., :, None] * gt[..., None, :]
        dq[:, t] = scale * torch.einsum("bhij,bhj->bhi", states[t + 1], gt)
        dk[:, t] = torch.where(live, torch.einsum("bhij,bhj->bhi", A, vt), zero.double())
        dv[:, t] = torch.where(live, torch.einsum("bhij,bhi->bhj", A, kt), zero.double())
        pairs[:, t] = (qt * dq[:, t]).sum(-1) + sign * (kt * dk[:, t]).sum(-1)
        w = torch.where(live[..., 0], g[:, t], zero.double()).exp()
        A = A * w[..., None, None]
        dg[:, t] = torch.where(live[..., 0], (A * states[t]).sum((-1, -2)), zero.double())
    got |= {"grad_q": dq, "grad_k": dk.reshape(B, L, -1, share, Dk).sum(3), "grad_v": dv.reshape(B, L, -1, share, Dv).sum(3),
            "grad_log_decay": dg if c["log_decay"].dim() == 3 else dg.sum((0, 1))}
    if c["initial_state"] is not None:
        got["grad_initial_state"] = A
    got["_pairs"], got["_across"] = pairs, across
    return got


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def lost_below(dtype):
    """A product, exponential or reciprocal below the smallest normal number of the type of sums (2^-126, or 2^-1022)
    may be returned as 0: off by less than that number times what it is multiplied with or summed over, which is below
    2^26 in every test."""
    return 2.0 ** -996 if dtype == torch.float64 else 2.0 ** -100


def attention_bounds(c, dtype, terms=1, chain=None):
    """How far each output may be from its exact value, element by element.

    Every output is a sum of products; with all terms replaced by their absolute values it is some T.  A chain of m
    roundings of at most u each, every one relative to a partial sum, is off by at most m u T (1 + small).  In the
    type of sums the longest chain is two roundings per step of the state (decay and addition), or the sum over a
    piece, plus the sums over a head, the exponentials (2 units each, the argument a sum over a piece) and a few
    products: m = 2 L + Dk + Dv + 64.  Operands of the matrix products in 16 bits are rounded at most twice on the
    way of a term (the state's part or the pair's weight, and the weighted row): 3 half steps of the storage type cover
    both and their products; results in the storage type add a half step of themselves.

    ``terms`` = 2: what enters the products is the value's rounding to bfloat16 and the rounding of what that left, so
    off by a half step of bfloat16 squared (2^-16), three times at most as above: the result is rounded to its type
    once, and nothing before it to so few bits.  ``chain``: m, for operands that are nearly all zero."""
    T = attention(absolute(c), sign=1.0)
    B, L, H, Dk = c["q"].shape
    u = half_step(torch.float64 if dtype == torch.float64 else torch.float32)
    m = chain or 2 * L + Dk + c["v"].shape[-1] + 64
    exact = attention(c)
    bounds = {}
    stored = half_step(dtype)
    for name in exact:
        if name.startswith("_"):
            continue
        t = T[name]
        if name == "grad_log_decay":
            # sums of x and y from the end of the segment, and the pairs across that end, all in absolute values
            pairs, across = T["_pairs"], T["_across"]
            t = torch.zeros_like(pairs)
            for a in range(0, L, SEGMENT):
                b = min(L, a + SEGMENT)
                t[:, a:b] = pairs[:, a:b].flip(1).cumsum(1).flip(1) + across[:, a:b].amax(1, keepdim=True)
            t = t if c["log_decay"].dim() == 3 else t.sum((0, 1))
            bounds[name] = 2 * m * u * t + lost_below(dtype)
        elif name in ("state", "grad_initial_state"):
            bounds[name] = m * u * t + lost_below(dtype)
        else:
            inner = 3 * stored if dtype in (torch.bfloat16, torch.float16) else 0.0
            inner = 3 * half_step(torch.bfloat16) ** 2 if inner and terms == 2 else inner
            bounds[name] = (m * u + inner) * t + stored * exact[name].abs() * 1.01 + lost_below(dtype)
            if dtype == torch.float16:
                bounds[name] = bounds[name] + 2.0 ** -25 * (1 + t.amax())   # below the smallest normal number
    return exact, bounds


def norm(c):
    """The norm around a block in 64 bits (autograd gives its gradients)."""
    x = c["x"]
    h = x / (x.square().mean(-1, keepdim=True) + c["eps"]).sqrt()
    if c["weight"] is not None:
        h = h * c["weight"]
    if c["gate"] is not None:
        h = h * (c["gate"].sigmoid() if c["activation"] == "sigmoid" else c["gate"] * c["gate"].sigmoid())
    if c["residual_scale"] is not None:
        h = h * c["residual_scale"]
    if c["residual"] is not None:
        h = h + c["residual"]
    n = None
    if c["next_weight"] is not None:
        n = h / (h.square().mean(-1, keepdim=True) + c["eps"]).sqrt() * c["next_weight"]
    return h, n


def norm_gradients(c):
    """Outputs and gradients of :func:`norm` by automatic differentiation."""
    names = ("x", "weight", "gate", "residual", "residual_scale", "next_weight")
    leaves = {n: c[n].clone().requires_grad_(True) for n in names if c[n] is not None}
    h, n = norm({**c, **leaves})
    heads = [(h, c["grad_h"])] + ([(n, c["grad_n"])] if n is not None else [])
    grads = torch.autograd.grad([a for a, _ in heads], list(leaves.values()), [b for _, b in heads])
    return {"h": h.detach()} | ({"n": n.detach()} if n is not None else {}) | {"grad_" + k: g for k, g in zip(leaves, grads)}


def norm_bounds(c, dtype):
    """Exact values of the norm and its gradients, and how far each element may be from them.

    As above: every value is a sum of products, and with m roundings of at most u on the way of a term it is off by at
    most m u times the sum of its terms' absolute values.  A gradient through a root mean square is such a difference:
    r (w dz) - x r^3 mean(w dz x) vanishes where w dz is along x (always, nearly, for a row of one element), while its two terms
    do not, so the bound is relative to the terms.  A relative error of r2 = (mean(h^2) + eps)^(-1/2) is that of
    the mean, which for h = residual + u is up to 1 + mean(|h| (|residual| + |u|)) / (mean(h^2) + eps) times that of
    its terms (kappa; r2 enters up to thrice).  The slope of the gate s (1 + g (1 - s)) counts as s (1 + |g|), since 1 - s cancels.
    An element goes through at most 60 roundings besides the sums, which run over 32 lanes or more at once: chains of
    D / 32 + 64 over a row and rows / 32 + 64 over the rows.  Two units are allowed for each."""
    u = half_step(torch.float64 if dtype == torch.float64 else torch.float32)
    stored = half_step(dtype) if dtype in (torch.bfloat16, torch.float16) else 0.0
    rows, D = c["x"].shape
    m = 2 * (60 + 3 * (D / 32 + 64)) * u
    x = c["x"].abs()
    one = torch.ones((), dtype=torch.float64)
    w, cs = (one if c[n] is None else c[n].abs() for n in ("weight", "residual_scale"))
    r = (x.square().mean(-1, keepdim=True) + c["eps"]).rsqrt()
    act, slope = one, one
    if c["gate"] is not None:
        s = c["gate"].sigmoid()
        act, slope = (s, s) if c["activation"] == "sigmoid" else (c["gate"].abs() * s, s * (1 + c["gate"].abs()))
    z = x * r * w
    ha = cs * z * act + (0 if c["residual"] is None else c["residual"].abs())
    exact = norm_gradients(c)
    size = {"h": ha}
    total = c["grad_h"].abs()
    if c["next_weight"] is not None:
        h = exact["h"]
        mean = h.square().mean(-1, keepdim=True) + c["eps"]
        kappa = 1 + (h.abs() * ha).mean(-1, keepdim=True) / mean
        r2, w2, dn = mean.rsqrt(), c["next_weight"].abs(), c["grad_n"].abs()
        size["n"] = kappa * ha * r2 * w2
        total = total + 3 * kappa * (r2 * w2 * dn + ha * r2 ** 3 * (w2 * dn * ha).mean(-1, keepdim=True))
        size["grad_next_weight"] = (kappa * dn * ha * r2).sum(0)
    size["grad_residual"] = total
    size["grad_residual_scale"] = (total * z * act).sum(0)
    size["grad_gate"] = total * cs * z * slope
    dz = total * cs * act
    size["grad_weight"] = (dz * x * r).sum(0)
    size["grad_x"] = r * w * dz + x * r ** 3 * (w * dz * x).mean(-1, keepdim=True)
    bounds = {}
    for name, want in exact.items():
        if name in ("grad_weight", "grad_residual_scale", "grad_next_weight"):
            bounds[name] = (m + 2 * u * (rows / 32 + 64)) * size[name] + lost_below(dtype)
        else:
            bounds[name] = m * size[name] + stored * 1.01 * want.abs() + (2.0 ** -25 if dtype == torch.float16 else lost_below(dtype))
    return exact, bounds
