"""Cases of the sequence operators that stand beside the signature layers: decayed linear attention over the
time axis of a batch of sequences (whole sequences, their gradients, and single time steps on a kept state) and
the norm around a block, fused with the block's gate, the residual sum and the norm before the next block.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes a case's tensors on
the GPU, ``run`` makes one pass: in elementary torch operations, or, where ``own`` is true, through the calls of
``pathsig_b200``.  ``exact`` computes the same outputs from the definitions in 64 bits and ``work`` gives the bytes
and floating-point operations that a pass cannot do without.

Definitions.  Attention, per sequence and head, with state S of shape (Dk, Dv):

    S_t = exp(log_decay_t) * S_{t-1} + k_t v_t^T,      out_t = scale * S_t^T q_t,      scale = Dk ** -0.5

A sequence of length n < L stops at n: later rows of the output are zero and the state is S_n.  Key and value
heads may be shared by consecutive query heads.  Norm, per row:

    rms(x) = x / sqrt(mean(x^2) + eps),   h = residual + residual_scale * (rms(x) * weight * act(gate)),
    n = rms(h) * next_weight                                              (h before it is rounded)
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_EPS = 1e-6
_CHUNK = 64


# ------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # One new observation of one stream: eight heads of 64 on one kept state; latency is all of it.
        _step("step of one stream", "bf16", 1, 8, 8, 64, 64, False),
        # One new observation for each of 256 streams, irregularly spaced in time (a decay for each stream).
        _step("step of 256 streams", "bf16", 256, 16, 4, 128, 128, True),
        # A long history of one stream is read once to build its state: few rows, a long time axis.
        _attention("prefill", "history of one stream", "bf16", 1, 16384, 16, 16, 128, 128, False, False, True),
        # A padded batch of histories of different lengths, continued from kept states, shared key heads.
        _attention("prefill", "ragged histories", "fp16", 13, 1111, 16, 4, 64, 128, True, True, True),
        # 32-bit sequences as the signature layers give them, odd length.
        _attention("prefill", "32-bit sequences", "fp32", 8, 2047, 8, 8, 64, 64, True, False, False),
        # Training on the sequence of 61 window signatures of each of 256 paths, projected to eight heads of 64.
        _attention("train", "train on windows", "bf16", 256, 61, 8, 8, 64, 64, False, False, False),
        # Training on long sequences: the largest case.
        _attention("train", "train on long sequences", "bf16", 8, 4096, 16, 16, 128, 128, True, False, False),
        # Training in 32 bits on one segment after another: the state's gradient comes in and goes out.
        _attention("train", "train in 32 bits", "fp32", 16, 511, 4, 2, 48, 80, True, True, True),
        # One row per stream on its way through the layers of a model that answers step by step.
        _norm("serve", "norm of 32 rows", "bf16", 32, 1024, True, True, True, True),
        # Norms around a block over the tokens of a training batch (256 paths of 61 windows).
        _norm("train", "norm of tokens", "bf16", 15616, 1024, True, True, True, True),
        # Depth-4 signatures of 8-channel paths, normalised and scaled in 32 bits: rows of 4680 features.
        _norm("train", "norm of signatures", "fp32", 15616, 4680, False, False, False, False),
        # The norm of each head's output and its gate, before the heads are mixed: short rows, many of them.
        _norm("train", "norm of heads", "bf16", 262144, 128, True, False, False, False),
    ]


def _attention(kind, name, dtype, B, L, H, Hkv, Dk, Dv, timed, ragged, state):
    return {"name": name, "kind": kind, "dtype": dtype, "B": B, "L": L, "H": H, "Hkv": Hkv, "Dk": Dk, "Dv": Dv,
            "timed": timed, "ragged": ragged, "state": state}


def _step(name, dtype, B, H, Hkv, Dk, Dv, timed):
    return {"name": name, "kind": "step", "dtype": dtype, "B": B, "H": H, "Hkv": Hkv, "Dk": Dk, "Dv": Dv, "timed": timed}


def _norm(mode, name, dtype, rows, D, gate, residual, scale, after):
    return {"name": name, "kind": "norm", "mode": mode, "dtype": dtype, "rows": rows, "D": D, "gate": gate,
            "residual": residual, "scale": scale, "after": after}


def _spread(rng, low, high):
    """A whole number between the two, evenly over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(("step", "prefill", "train", "train", "prefill", "norm", "norm"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "norm":
        rows = _spread(rng, 1, 262144)
        D = _spread(rng, 32, min(8192, max(32, 64_000_000 // rows)))
        D = -(-D // 8) * 8 if rng.random() < 0.6 else D
        gate, residual = rng.random() < 0.6, rng.random() < 0.5
        case = _norm(rng.choice(("serve", "train")), "", dtype, rows, D, gate, residual, residual and rng.random() < 0.6,
                     residual and rng.random() < 0.6)
    else:
        heads = rng.choice((1, 2, 3, 4, 5, 6, 8, 12, 16))
        kv = rng.choice([n for n in range(1, heads + 1) if heads % n == 0] + [heads])
        Dk, Dv = 8 * rng.randint(2, 16), 8 * rng.randint(2, 16)
        timed = rng.random() < 0.5
        if kind == "step":
            case = _step("", dtype, _spread(rng, 1, 256), heads, kv, Dk, Dv, timed)
        else:
            L = _spread(rng, 1, 16384)
            most = 33_554_432 if kind == "train" else 25_165_824
            B = _spread(rng, 1, max(1, min(256, most // (L * heads * max(Dk, Dv)) // (4 if dtype == "fp32" else 1))))
            case = _attention(kind, "", dtype, B, L, heads, kv, Dk, Dv, timed, rng.random() < 0.4, rng.random() < 0.5)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 2 + 1)
    dtype = _TYPES[case["dtype"]]

    def normal(*shape, dtype=dtype, std=1.0):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    if case["kind"] == "norm":
        rows, D = case["rows"], case["D"]
        s = {"x": normal(rows, D, std=2.0), "weight": 1 + normal(D, dtype=torch.float32, std=0.2),
             "gate": normal(rows, D) if case["gate"] else None,
             "residual": normal(rows, D, std=3.0) if case["residual"] else None,
             "residual_scale": normal(D, dtype=torch.float32, std=0.3) if case["scale"] else None,
             "next_weight": 1 + normal(D, dtype=torch.float32, std=0.2) if case["after"] else None}
        if case["mode"] == "train":
            for v in s.values():
                if v is not None:
                    v.requires_grad_(True)
            s["grad_h"] = normal(rows, D)
            s["grad_n"] = normal(rows, D) if case["after"] else None
        return {"kind": "norm", "mode": case["mode"], **s}

    B, H, Hkv, Dk, Dv = (case[n] for n in ("B", "H", "Hkv", "Dk", "Dv"))
    lead = (B,) if case["kind"] == "step" else (B, case["L"])
    q, k, v = normal(*lead, H, Dk), normal(*lead, Hkv, Dk), normal(*lead, Hkv, Dv)
    # rates from about 1/2 down to about 1/1000 per unit of time over the heads; steps of time are 1, or exponential
    rate = torch.exp2(-1.0 - 9.0 * (torch.arange(H, device="cuda", dtype=torch.float32) + torch.rand(H, generator=gen, device="cuda")) / H)
    log_decay = -rate
    if case["timed"]:
        log_decay = rate * torch.log(torch.rand(*lead, 1, generator=gen, device="cuda").clamp_min_(1e-6))
    s = {"kind": case["kind"], "q": q, "k": k, "v": v, "log_decay": log_decay.contiguous()}
    if case["kind"] == "step":
        s["state"] = normal(B, H, Dk, Dv, dtype=torch.float32, std=3.0)
        return s
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(0, case["L"] + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        s["lengths"][0] = case["L"]
    s["initial_state"] = normal(B, H, Dk, Dv, dtype=torch.float32, std=3.0) if case["state"] else None
    s["with_state"] = case["state"]
    if case["kind"] == "train":
        for name in ("q", "k", "v", "log_decay", "initial_state"):
            if s[name] is not None:
                s[name].requires_grad_(True)
        s["grad_out"] = normal(*lead, H, Dv)
        s["grad_state"] = normal(B, H, Dk, Dv, dtype=torch.float32) if case["state"] else None
    return s


# ------------------------------------------------------------------------------------------------- one pass

def run(s):
    if s["kind"] == "step":
        if own:
            import pathsig_b200 as ps
            out = ps.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"])
        else:
            out = _plain_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"])
        return {"out": out, "state": s["state"]}
    if s["kind"] == "norm":
        return _run_norm(s)
    args = (s["q"], s["k"], s["v"], s["log_decay"])
    more = {"initial_state": s["initial_state"], "lengths": s["lengths"]}
    if own:
        import pathsig_b200 as ps
        got = ps.linear_attention(*args, **more, return_state=s["with_state"])
        out, state = got if s["with_state"] else (got, None)
    else:
        out, state = _plain_attention(*args, **more)
        state = state if s["with_state"] else None
    outputs = {"out": out, "state": state}
    if s["kind"] == "train":
        outputs |= _gradients(s, ("q", "k", "v", "log_decay", "initial_state"), [out, state], [s["grad_out"], s["grad_state"]])
    return outputs


def _run_norm(s):
    names = ("x", "weight", "gate", "residual", "residual_scale", "next_weight")
    more = {n: s[n] for n in names[2:]}
    if own:
        import pathsig_b200 as ps
        got = ps.gated_residual_norm(s["x"], s["weight"], **more, eps=_EPS)
        h, n = got if s["next_weight"] is not None else (got, None)
    else:
        h, n = _plain_norm(s["x"], s["weight"], **more)
    outputs = {"h": h, "n": n}
    if s["mode"] == "train":
        outputs |= _gradients(s, names, [h, n], [s["grad_h"], s["grad_n"]])
    return outputs


def _gradients(s, names, outputs, grads):
    names = [n for n in names if s[n] is not None]
    pairs = [(o, g) for o, g in zip(outputs, grads) if o is not None]
    got = torch.autograd.grad([o for o, _ in pairs], [s[n] for n in names], [g for _, g in pairs])
    return {"grad_" + n: g for n, g in zip(names, got)}


def _plain_step(q, k, v, log_decay, state):
    share = q.shape[-2] // k.shape[-2]
    k, v = (t.float().repeat_interleave(share, dim=-2) for t in (k, v))
    decay = log_decay.exp().expand(q.shape[0], -1)[..., None, None]
    state.copy_(state * decay + k[..., :, None] * v[..., None, :])
    out = (q.float() * q.shape[-1] ** -0.5)[..., None, :] @ state
    return out[..., 0, :].to(q.dtype)


def _plain_attention(q, k, v, log_decay, initial_state, lengths):
    """All pieces of 64 time steps at once: pairs inside a piece by their matrix of weights, earlier pieces by the
    states at the pieces' beginnings, which are one product of the pieces' own sums with a matrix of decays."""
    B, L, H, Dk = q.shape
    Dv, dtype, share = v.shape[-1], q.dtype, H // k.shape[2]
    N = -(-L // _CHUNK)

    def pieces(t):  # (B, L, H, X) -> (B, H, N, C, X)
        t = torch.nn.functional.pad(t, (0, 0, 0, 0, 0, N * _CHUNK - L))
        return t.reshape(B, N, _CHUNK, H, -1).permute(0, 3, 1, 2, 4)

    q, k, v = q.float() * Dk ** -0.5, k.float().repeat_interleave(share, dim=2), v.float().repeat_interleave(share, dim=2)
    g = log_decay.double().expand(B, L, H)[..., None]
    if lengths is not None:
        live = (torch.arange(L, device=q.device) < lengths[:, None])[:, :, None, None]
        q, k, v, g = (torch.where(live, t, torch.zeros((), dtype=t.dtype, device=t.device)) for t in (q, k, v, g))
    q, k, v, g = (pieces(t) for t in (q, k, v, g))
    g = g[..., 0].cumsum(-1)                                                     # (B, H, N, C), from each piece's beginning
    steps = torch.arange(_CHUNK, device=q.device)
    inside = (g[..., :, None] - g[..., None, :]).masked_fill(steps[:, None] < steps, -math.inf).exp().float()
    out = ((q @ k.transpose(-1, -2)) * inside) @ v
    own_sums = (k * (g[..., -1:] - g).exp().float()[..., None]).transpose(-1, -2) @ v   # (B, H, N, Dk, Dv)
    total = torch.nn.functional.pad(g[..., -1].cumsum(-1), (1, 0))               # (B, H, N + 1), up to each beginning
    at = torch.arange(N + 1, device=q.device)
    between = (total[..., :, None] - total[..., None, 1:]).masked_fill(at[:, None] <= at[:-1], -math.inf).exp().float()
    states = (between @ own_sums.reshape(B, H, N, Dk * Dv)).reshape(B, H, N + 1, Dk, Dv)
    if initial_state is not None:
        states = states + total.exp().float()[..., None, None] * initial_state[:, :, None]
    out = out + (q * g.exp().float()[..., None]) @ states[:, :, :-1]
    out = out.permute(0, 2, 3, 1, 4).reshape(B, N * _CHUNK, H, Dv)[:, :L]
    return out.to(dtype), states[:, :, -1]


def _plain_norm(x, weight, gate, residual, residual_scale, next_weight):
    dtype = x.dtype
    x = x.float()
    h = x * (x.square().mean(-1, keepdim=True) + _EPS).rsqrt() * weight
    if gate is not None:
        gate = gate.float()
        h = h * gate * gate.sigmoid()
    if residual_scale is not None:
        h = h * residual_scale
    if residual is not None:
        h = residual.float() + h
    n = None
    if next_weight is not None:
        n = (h * (h.square().mean(-1, keepdim=True) + _EPS).rsqrt() * next_weight).to(dtype)
    return h.to(dtype), n


# ------------------------------------------------------------------------------------------------- what it needs

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "norm":
        train, rows, D = case["mode"] == "train", case["rows"], case["D"]
        reads, writes = 1 + case["gate"] + case["residual"], 1 + case["after"]
        vectors = 1 + case["scale"] + case["after"]
        moved = (reads + writes) * (2 if train else 1)
        return {"bytes": moved * rows * D * size + vectors * D * 4 * (2 if train else 1),
                "flops": (8 + 6 * case["gate"] + 2 * case["residual"] + 4 * case["after"]) * (3 if train else 1) * rows * D}
    B, H, Hkv, Dk, Dv = (case[n] for n in ("B", "H", "Hkv", "Dk", "Dv"))
    state = B * H * Dk * Dv * 4
    if case["kind"] == "step":
        return {"bytes": 2 * state + B * size * (H * (Dk + Dv) + Hkv * (Dk + Dv)) + 4 * H * (B if case["timed"] else 1),
                "flops": 5 * B * H * Dk * Dv}
    rows = B * case["L"] * (0.5 if case["ragged"] else 1.0)   # lengths are uniform: half of the rows are live
    ends = B * case["L"] - rows                               # the others are written as zeros
    decay = 4 * H * (rows if case["timed"] else 1)
    inputs, output = rows * size * (H * Dk + Hkv * (Dk + Dv)), size * H * Dv
    need = {"bytes": inputs + (rows + ends) * output + decay, "flops": 4 * rows * H * Dk * Dv}
    if case["state"]:
        need["bytes"] += 2 * state
    if case["kind"] == "train":
        need["bytes"] += inputs + ends * size * (H * Dk + Hkv * (Dk + Dv)) + rows * output + decay + (2 * state if case["state"] else 0)
        need["flops"] += 8 * rows * H * Dk * Dv
    return need


# ------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = {n: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for n, v in prepare(case, seed).items()}
    with torch.no_grad():
        if case["kind"] == "step":
            return _exact_step(s)
        if case["kind"] == "norm":
            return _exact_norm(s)
        return _exact_attention(s)


def _exact_step(s):
    share = s["q"].shape[1] // s["k"].shape[1]
    heads = torch.arange(s["q"].shape[1], device="cuda") // share
    k, v = s["k"][:, heads], s["v"][:, heads]
    decay = torch.exp(s["log_decay"])
    decay = decay[None, :] if decay.dim() == 1 else decay
    state = torch.einsum("bhij,bh->bhij", s["state"], decay.expand(k.shape[0], -1)) + torch.einsum("bhi,bhj->bhij", k, v)
    return {"out": torch.einsum("bhi,bhij->bhj", s["q"], state) / math.sqrt(k.shape[-1]), "state": state}


def _exact_attention(s):
    """The double sum over pairs of time steps, a few heads at a time, and its derivatives."""
    q, k, v, S0, lengths = s["q"], s["k"], s["v"], s["initial_state"], s["lengths"]
    B, L, H, Dk = q.shape
    share, scale, train = H // k.shape[2], 1 / math.sqrt(Dk), s["kind"] == "train"
    got = {"out": torch.zeros(B, L, H, v.shape[-1], dtype=torch.float64, device="cuda"),
           "state": torch.zeros(B, H, Dk, v.shape[-1], dtype=torch.float64, device="cuda") if s["with_state"] else None}
    per_step = s["log_decay"].dim() == 3
    if train:
        got |= {"grad_" + n: torch.zeros_like(s[n]) for n in ("q", "k", "v", "log_decay", "initial_state") if s[n] is not None}
    for b in range(B):
        n = L if lengths is None else int(lengths[b])
        if n == 0:
            if s["with_state"]:
                got["state"][b] = S0[b]
                if train:
                    got["grad_initial_state"][b] = s["grad_state"][b]
            continue
        at_once = max(1, min(H, 120_000_000 // (n * n)))
        at = torch.arange(n, device="cuda")
        for first in range(0, H, at_once):
            hs = torch.arange(first, min(H, first + at_once), device="cuda")
            Q, K, V = q[b, :n, hs].transpose(0, 1), k[b, :n, hs // share].transpose(0, 1), v[b, :n, hs // share].transpose(0, 1)
            g = s["log_decay"][b, :n, hs].t() if per_step else s["log_decay"][hs][:, None].expand(-1, n)
            G = g.cumsum(1)
            W = (G[:, :, None] - G[:, None, :]).masked_fill_(at[:, None] < at, -math.inf).exp_()
            P = torch.einsum("hti,hsi->hts", Q, K).mul_(W).mul_(scale)
            O = torch.einsum("hts,hsj->htj", P, V)
            head, tail = G.exp(), (G[:, -1:] - G).exp()
            if S0 is not None:
                O += scale * head[..., None] * torch.einsum("hti,hij->htj", Q, S0[b, hs])
            got["out"][b, :n, hs] = O.transpose(0, 1)
            if s["with_state"]:
                last = torch.einsum("hs,hsi,hsj->hij", tail, K, V) + (head[:, -1, None, None] * S0[b, hs] if S0 is not None else 0)
                got["state"][b, hs] = last
            if not train:
                continue
            dO = s["grad_out"][b, :n, hs].transpose(0, 1)
            dV = torch.einsum("hts,htj->hsj", P, dO)
            R = torch.einsum("htj,hsj->hts", dO, V)
            pair = P.mul_(R)                                   # what each pair adds to <grad_out, out>
            dG = pair.sum(2) - pair.sum(1)
            R.mul_(W).mul_(scale)
            dQ, dK = torch.einsum("hts,hsi->hti", R, K), torch.einsum("hts,hti->hsi", R, Q)
            if S0 is not None:
                x = scale * head[..., None] * torch.einsum("htj,hij->hti", dO, S0[b, hs])
                dQ += x
                dG += (Q * x).sum(2)
                dS0 = scale * torch.einsum("ht,hti,htj->hij", head, Q, dO)
            if s["with_state"]:
                A = s["grad_state"][b, hs]
                kA = tail[..., None] * torch.einsum("hsj,hij->hsi", V, A)
                dK += kA
                dV += tail[..., None] * torch.einsum("hsi,hij->hsj", K, A)
                dG -= (K * kA).sum(2)
                dG[:, -1] += (A * last).sum((1, 2))
                dS0 += head[:, -1, None, None] * A
            dg = dG.flip(1).cumsum(1).flip(1)
            got["grad_q"][b, :n, hs] = dQ.transpose(0, 1)
            for name, d in (("grad_k", dK), ("grad_v", dV)):
                got[name][b, :n].index_add_(1, hs // share, d.transpose(0, 1))
            if per_step:
                got["grad_log_decay"][b, :n, hs] = dg.t()
            else:
                got["grad_log_decay"][hs] += dg.sum(1)
            if S0 is not None:
                got["grad_initial_state"][b, hs] = dS0
    return got


def _exact_norm(s):
    D = s["x"].shape[1]
    names = ("x", "weight", "gate", "residual", "residual_scale", "next_weight")
    got = {"h": torch.empty_like(s["x"]), "n": None if s["next_weight"] is None else torch.empty_like(s["x"])}
    train = s["mode"] == "train"
    if train:
        got |= {"grad_" + n: torch.zeros_like(s[n]) for n in names if s[n] is not None}
    one = torch.ones((), dtype=torch.float64, device="cuda")
    w, c = s["weight"], one if s["residual_scale"] is None else s["residual_scale"]
    for a in range(0, s["x"].shape[0], max(1, 16_000_000 // D)):
        rows = slice(a, a + max(1, 16_000_000 // D))
        x = s["x"][rows]
        r = 1 / torch.sqrt((x * x).sum(1, keepdim=True) / D + _EPS)
        gate = None if s["gate"] is None else s["gate"][rows]
        sig = None if gate is None else 1 / (1 + torch.exp(-gate))
        act = one if gate is None else gate * sig
        z = x * r * w
        h = c * z * act + (0 if s["residual"] is None else s["residual"][rows])
        got["h"][rows] = h
        if s["next_weight"] is not None:
            r2 = 1 / torch.sqrt((h * h).sum(1, keepdim=True) / D + _EPS)
            got["n"][rows] = h * r2 * s["next_weight"]
        if not train:
            continue
        dh = s["grad_h"][rows]
        if s["next_weight"] is not None:
            dn = s["grad_n"][rows]
            got["grad_next_weight"] += (dn * h * r2).sum(0)
            u = dn * s["next_weight"]
            dh = dh + r2 * u - h * r2 ** 3 * (u * h).sum(1, keepdim=True) / D
        if s["residual"] is not None:
            got["grad_residual"][rows] = dh
        if s["residual_scale"] is not None:
            got["grad_residual_scale"] += (dh * z * act).sum(0)
        if gate is not None:
            got["grad_gate"][rows] = dh * c * z * sig * (1 + gate * (1 - sig))
        dz = dh * c * act
        got["grad_weight"] += (dz * x * r).sum(0)
        u = dz * w
        got["grad_x"][rows] = r * u - x * r ** 3 * (u * x).sum(1, keepdim=True) / D
    return got
