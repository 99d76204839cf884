"""The norm around a block (gate, residual, next norm) on the GPU against 64-bit formulas and their autograd gradients."""
from __future__ import annotations

import subprocess
import sys

import pytest
import torch

from . import sequence_oracle as so
from . import util
from .conftest import ROOT

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]
NAMES = ("x", "weight", "gate", "residual", "residual_scale", "next_weight")
FORMS = [  # weight, gate, activation, residual, residual_scale, next_weight
    (False, None, False, False, False),
    (True, None, False, False, False),
    (True, "silu", False, False, False),
    (True, "sigmoid", True, False, True),
    (True, "silu", True, True, True),
    (False, None, True, True, True),
    (True, None, False, True, True),
]


@pytest.fixture(scope="module")
def ps():
    import pathsig_b200
    return pathsig_b200


def _make(seed, rows, D, dtype, form, eps=1e-6):
    gen = torch.Generator().manual_seed(seed)
    sums = torch.float64 if dtype == torch.float64 else torch.float32

    def normal(*shape, to=dtype, std=1.0, mean=0.0):
        return (mean + std * torch.randn(*shape, generator=gen, dtype=torch.float64)).to(to).double()

    weight, act, residual, scale, after = form
    return {"x": normal(rows, D, std=2.0), "weight": normal(D, to=sums, std=0.2, mean=1.0) if weight else None,
            "gate": normal(rows, D) if act else None, "residual": normal(rows, D, std=3.0) if residual else None,
            "residual_scale": normal(D, to=sums, std=0.5) if scale else None,
            "next_weight": normal(D, to=sums, std=0.2, mean=1.0) if after else None,
            "grad_h": normal(rows, D), "grad_n": normal(rows, D) if after else None, "activation": act or "silu", "eps": eps}


def _gpu(c, dtype):
    sums = torch.float64 if dtype == torch.float64 else torch.float32
    wide = ("weight", "residual_scale", "next_weight")
    return {n: t.to(sums if n in wide else dtype).to(DEV) if isinstance(t, torch.Tensor) else t for n, t in c.items()}


def _run(f, c):
    leaves = {n: c[n].detach().requires_grad_(True) if c[n] is not None else None for n in NAMES}
    h, n = f(leaves)
    heads, grads = [h], [c["grad_h"]]
    if n is not None:
        heads.append(n)
        grads.append(c["grad_n"])
    wanted = {k: t for k, t in leaves.items() if t is not None}
    got = {"grad_" + k: g for k, g in zip(wanted, torch.autograd.grad(heads, list(wanted.values()), grads))}
    return got | {"h": h.detach()} | ({"n": n.detach()} if n is not None else {})


def _ours(ps, eps):
    def f(leaves):
        activation = leaves.get("activation", "silu")
        got = ps.gated_residual_norm(leaves["x"], leaves["weight"], gate=leaves["gate"], residual=leaves["residual"],
                                     residual_scale=leaves["residual_scale"], next_weight=leaves["next_weight"],
                                     activation=activation, eps=eps)
        return got if leaves["next_weight"] is not None else (got, None)
    return f


def _check(ps, c, dtype):
    ours = _run(lambda t: _ours(ps, c["eps"])(dict(t, activation=c["activation"])), _gpu(c, dtype))
    exact, bounds = so.norm_bounds(c, dtype)
    assert set(ours) == set(exact)
    for name, want in exact.items():
        assert ours[name].shape == want.shape, name
        off = (ours[name].double().cpu() - want).abs()
        bad = ~(off <= bounds[name])
        assert not bad.any(), (name, int(bad.sum()), float(off[bad].max()), float((off / bounds[name].clamp_min(1e-300)).max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (5, 7), (33, 32), (64, 64), (7, 100), (130, 128), (9, 340), (40, 1024),
                                    (3, 1001), (2, 4680), (2, 4096)])
def test_outputs_and_gradients(ps, rows, D, form, dtype):
    c = _make(rows + D, rows, D, dtype, form)
    _check(ps, c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,D", [(2, 8192), (2, 9001), (3, 16384), (1, 30000), (2, 69904)])
def test_wide_rows(ps, rows, D, dtype):
    """The widest: depth-4 signatures of 16 channels."""
    c = _make(D, rows, D, dtype, FORMS[4])
    _check(ps, c, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D", [(20000, 16), (3001, 128), (2500, 1000), (1500, 2048)])
def test_many_rows(ps, rows, D, dtype):
    c = _make(D, rows, D, dtype, FORMS[4])
    _check(ps, c, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_zero_rows_and_large_values(ps, dtype):
    """A row of zeros (eps alone under the root), rows of large and of tiny values, gates far out on both sides."""
    c = _make(1, 4, 64, dtype, FORMS[2], eps=1e-5)
    c["x"][0] = 0
    c["x"][1] = (c["x"][1] * 1000).to(dtype).double()      # the operands of both sides are of the type
    c["x"][2] = (c["x"][2] * 2.0 ** -7).to(dtype).double()
    c["gate"][3, :8] = torch.tensor([-300.0, 300.0, -90.0, 90.0, 0.0, -20.0, 20.0, -5.0], dtype=torch.float64).to(dtype).double()
    _check(ps, c, dtype)


def test_gradients_against_differences(ps):
    c = _gpu(_make(4, 3, 5, torch.float64, FORMS[4]), torch.float64)
    leaves = [c[n].requires_grad_(True) for n in NAMES]
    for activation in ("silu", "sigmoid"):
        assert torch.autograd.gradcheck(
            lambda x, w, g, r, s, n: ps.gated_residual_norm(x, w, gate=g, residual=r, residual_scale=s, next_weight=n,
                                                            activation=activation), leaves, eps=1e-6, atol=1e-8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shapes_strides_and_16_bit_parameters(ps, dtype):
    x = torch.randn(2, 3, 5, 64, device=DEV).to(dtype)
    w = torch.rand(64, device=DEV).to(dtype).requires_grad_(True)
    want = ps.gated_residual_norm(x, w.detach().float())
    assert want.shape == x.shape and want.dtype == dtype
    got = ps.gated_residual_norm(x.transpose(0, 1).contiguous().transpose(0, 1), w)
    assert torch.equal(got, want)
    odd = torch.nn.functional.pad(x.reshape(-1), (1, 0))[1:].view_as(x)      # rows that start off a 16-byte boundary
    # the row's sum may run in another order: a chain of 8 squares and 3 levels or of 2 squares and 6 (11 roundings at
    # most, half of them under the root), the root (2 units), two products and the result: under 14 units of 2^-24 on
    # each side.  In 16 bits such a difference can turn a rounding: both results are within a half step of their values.
    apart = 28 * so.half_step(torch.float32) + (0 if dtype == torch.float32 else 2 * so.half_step(dtype))
    assert util.rel_error(ps.gated_residual_norm(odd, w), want) < apart
    got.float().sum().backward()
    assert w.grad.dtype == dtype and w.grad.shape == (64,)
    assert ps.gated_residual_norm(x[0, 0, 0]).shape == (64,)
    assert ps.gated_residual_norm(x[:0]).shape == (0, 3, 5, 64)


def test_only_the_next_norm_is_used(ps):
    c = _gpu(_make(8, 6, 96, torch.float32, FORMS[4]), torch.float32)
    r = c["residual"].requires_grad_(True)
    _, n = ps.gated_residual_norm(c["x"], c["weight"], gate=c["gate"], residual=r, residual_scale=c["residual_scale"],
                                  next_weight=c["next_weight"])
    got, = torch.autograd.grad(n, r, c["grad_n"])
    wide = {k: t.detach().double().cpu() if isinstance(t, torch.Tensor) else t for k, t in c.items()}
    wide["residual"].requires_grad_(True)
    want, = torch.autograd.grad(so.norm(wide)[1], wide["residual"], wide["grad_n"])
    assert util.rel_error(got, want) < 200 * so.half_step(torch.float32)


def test_empty_rows_have_zero_parameter_gradients(ps):
    x = torch.zeros(0, 16, device=DEV)
    w = torch.ones(16, device=DEV, requires_grad=True)
    ps.gated_residual_norm(x, w).sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_bits_every_run_on_streams_and_in_graphs(ps, dtype):
    c = _gpu(_make(5, 700, 1024, dtype, FORMS[4]), dtype)
    first = _run(_ours(ps, 1e-6), c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _run(_ours(ps, 1e-6), c)
    torch.cuda.current_stream().wait_stream(side)
    args = [c[n] for n in NAMES]
    with torch.cuda.stream(side):
        torch.ops.pathsig_b200.gated_residual_norm_backward(*args, c["grad_h"], c["grad_n"], 0, 1e-6)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, n = torch.ops.pathsig_b200.gated_residual_norm(*args, 0, 1e-6)
        grads = torch.ops.pathsig_b200.gated_residual_norm_backward(*args, c["grad_h"], c["grad_n"], 0, 1e-6)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    third = {"h": h, "n": n, **{"grad_" + name: g for name, g in zip(NAMES, grads)}}
    for name in first:
        assert torch.equal(first[name], second[name]) and torch.equal(first[name], third[name]), name


def test_a_mixing_block_on_window_signatures(ps):
    """The operators as they are used together: window signatures, norm before the block, projections, decayed
    attention, norm of each head with its gate, projection, norm after the block with the scaled residual and the norm
    before the next block; outputs and the gradients of all parameters and of the paths, in 64 bits."""
    B, d, depth, E, H = 3, 3, 3, 24, 2
    x = util.brownian_path(B, 65, d, seed=2, dtype=torch.float64)
    win = torch.tensor([[8 * i, 8 * i + 16] for i in range(7)], dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(5)
    width = d + d ** 2 + d ** 3

    def weight(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float64) / shape[0] ** 0.5

    p = {"win": weight(width, E), "wqkvg": weight(E, 4 * E), "wo": weight(E, E), "n1": 1 + 0.1 * weight(width),
         "nh": 1 + 0.1 * weight(E // H), "n2": 1 + 0.1 * weight(E), "n3": 1 + 0.1 * weight(E), "s": 0.3 * weight(E),
         "decay": -torch.rand(H, generator=gen, dtype=torch.float64)}
    sig_gpu = ps.Signature(depth=depth, windows=win)

    def block(sig, p, norm, attention):
        t = norm(sig, p["n1"]) @ p["win"]
        q, k, v, g = (norm(t, None) @ p["wqkvg"]).unflatten(-1, (4, H, E // H)).unbind(-3)
        o = norm(attention(q, k, v, p["decay"]), p["nh"], gate=g).flatten(-2) @ p["wo"]
        h, n = norm(o, p["n2"], residual=t, residual_scale=p["s"], next_weight=p["n3"])
        return h, n

    def plain_norm(x, w, gate=None, residual=None, residual_scale=None, next_weight=None):
        h, n = so.norm({"x": x, "weight": w, "gate": gate, "residual": residual, "residual_scale": residual_scale,
                        "next_weight": next_weight, "activation": "silu", "eps": 1e-6})
        return h if next_weight is None else (h, n)

    def plain_attention(q, k, v, decay):
        S, outs = torch.zeros(B, H, E // H, E // H, dtype=torch.float64), []
        for t in range(q.shape[1]):
            S = S * decay.exp()[:, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
            outs.append((q[:, t, :, None, :] @ S)[..., 0, :] * (E // H) ** -0.5)
        return torch.stack(outs, 1)

    xg = x.to(DEV).requires_grad_(True)
    pg = {n: t.to(DEV).requires_grad_(True) for n, t in p.items()}
    sig = sig_gpu(xg)
    h, n = block(sig, pg, ps.gated_residual_norm, ps.linear_attention)
    (h.square().sum() + n.sin().sum()).backward()
    sig_cpu = sig.detach().cpu().requires_grad_(True)
    pc = {n: t.clone().requires_grad_(True) for n, t in p.items()}
    h2, n2 = block(sig_cpu, pc, plain_norm, plain_attention)
    (h2.square().sum() + n2.sin().sum()).backward()
    assert util.rel_error(h, h2) < 1e-12 and util.rel_error(n, n2) < 1e-12
    for name in p:
        assert util.rel_error(pg[name].grad, pc[name].grad) < 1e-11, name
    want, = torch.autograd.grad(sig_gpu(xg), xg, sig_cpu.grad.to(DEV))
    assert util.rel_error(xg.grad, want) < 1e-11


def test_refusals_on_the_gpu(ps):
    x = torch.zeros(4, 8, device=DEV)
    for more, error in [(dict(weight=torch.ones(7, device=DEV)), "weight"), (dict(gate=torch.zeros(4, 7, device=DEV)), "gate"),
                        (dict(gate=torch.zeros(4, 8, device=DEV, dtype=torch.bfloat16)), "gate"), (dict(residual=torch.zeros(8, device=DEV)), "residual"),
                        (dict(next_weight=torch.ones(8, device=DEV, dtype=torch.float64)), "next_weight"), (dict(weight=torch.ones(8)), "weight")]:
        with pytest.raises(RuntimeError, match=error):
            ps.gated_residual_norm(x, **more)
    with pytest.raises(RuntimeError, match="float32"):
        ps.gated_residual_norm(x.int())
    with pytest.raises(RuntimeError, match="D >= 1"):
        ps.gated_residual_norm(torch.zeros(3, 0, device=DEV))


def test_second_derivatives_are_refused(ps):
    """A gradient with a graph of its own is the plain gradient; its gradient is refused, not left out."""
    x = torch.randn(5, 24, device=DEV, requires_grad=True)
    w = torch.randn(24, device=DEV, requires_grad=True)
    plain = torch.autograd.grad(ps.gated_residual_norm(x, w).square().sum(), (x, w))
    graph = torch.autograd.grad(ps.gated_residual_norm(x, w).square().sum(), (x, w), create_graph=True)
    for a, b in zip(plain, graph):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="differentiable once"):
        graph[0].sum().backward()


@pytest.mark.parametrize("rows,D,dtype,form", [
    (2400, 612, "float32", 4), (2400, 764, "float32", 5), (2400, 1020, "float32", 2), (2400, 1528, "float32", 1),
    (2400, 3056, "bfloat16", 1), (2400, 6104, "bfloat16", 0)])
def test_rings_that_just_fit_the_default_shared_memory(rows, D, dtype, form):
    """Rings of rows that, with the kernel's own 256 bytes, are just above the 48 KB that need no consent.  Each in a
    process of its own, where no wider ring has been launched before."""
    code = (f"import torch, pathsig_b200 as ps; from tests import test_gpu_residual_norm as t; "
            f"t._check(ps, t._make(1, {rows}, {D}, torch.{dtype}, t.FORMS[{form}]), torch.{dtype})")
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", FORMS[3:])
@pytest.mark.parametrize("rows,D", [(1, 8), (1, 128), (17, 64), (33, 100), (3, 1001)])
def test_no_eps(ps, rows, D, form, dtype):
    """eps = 0, with row counts that leave some of a block's teams without a row (or none, where a block holds one)."""
    c = _make(rows * D, rows, D, dtype, form, eps=0.0)
    _check(ps, c, dtype)


@pytest.mark.parametrize("rows,D,dtype,form", [(2400, 1528, "float32", 1), (2400, 1024, "bfloat16", 4), (3000, 200, "bfloat16", 6)])
def test_a_wait_for_a_row_that_runs_out_ends_its_block(ps, rows, D, dtype, form):
    """With no poll allowed the blocks that stream rows leave at the first, count that, and wait for the copies in flight;
    later calls are as ever."""
    from pathsig_b200 import _load
    lib = _load.ensure_loaded()
    dtype = getattr(torch, dtype)
    c = _gpu(_make(2, rows, D, dtype, FORMS[form]), dtype)
    args = [c[n] for n in NAMES]

    def backward():
        got = torch.ops.pathsig_b200.gated_residual_norm_backward(*args, c["grad_h"], c["grad_n"], 0, 1e-6)
        torch.cuda.synchronize()
        return got

    want = backward()
    assert lib.psig_sequence_wait_timeouts() == 0
    try:
        assert lib.psig_set_norm_wait_polls(0) == 0
        backward()
        assert lib.psig_sequence_wait_timeouts() > 0
        assert lib.psig_sequence_wait_timeouts() == 0      # read and cleared
    finally:
        assert lib.psig_set_norm_wait_polls(-1) == 0
    with pytest.raises(RuntimeError, match="ran out"):
        backward()
    for a, b in zip(backward(), want):
        assert torch.equal(a, b)
    assert lib.psig_sequence_wait_timeouts() == 0


def test_a_wait_that_ran_out_is_an_error_of_the_next_call(ps):
    """The call itself has been enqueued and has returned by then; the one after it raises, once, whichever operator it is."""
    from pathsig_b200 import _load
    lib = _load.ensure_loaded()
    c = _gpu(_make(3, 2400, 1024, torch.bfloat16, FORMS[4]), torch.bfloat16)
    args = [c[n] for n in NAMES]
    backward = torch.ops.pathsig_b200.gated_residual_norm_backward
    want = backward(*args, c["grad_h"], c["grad_n"], 0, 1e-6)
    q, d = torch.randn(1, 3, 2, 8, device=DEV), torch.zeros(2, device=DEV)
    for following in (lambda: backward(*args, c["grad_h"], c["grad_n"], 0, 1e-6), lambda: ps.gated_residual_norm(c["x"]),
                      lambda: ps.linear_attention(q, q, q, d),
                      lambda: ps.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], d, torch.zeros(1, 2, 8, 8, device=DEV))):
        try:
            assert lib.psig_set_norm_wait_polls(0) == 0
            backward(*args, c["grad_h"], c["grad_n"], 0, 1e-6)
            torch.cuda.synchronize()
        finally:
            assert lib.psig_set_norm_wait_polls(-1) == 0
        with pytest.raises(RuntimeError, match="ran out"):
            following()
        following()
        assert lib.psig_sequence_wait_timeouts() > 0
    for a, b in zip(backward(*args, c["grad_h"], c["grad_n"], 0, 1e-6), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32])
@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
@pytest.mark.parametrize("D", [8, 16384])
def test_gates_far_out_are_good_to_the_types_last_bits(ps, D, activation, dtype):
    """Gates of -85 to 85, each value relative to itself.  Units of half a step: the root 9 (eight squares and their sum, halved by
    the root: 4; mean and eps 1; the root 4; for the long row its sums run over 32 lanes and 16 warps or more, 1024 / 32 + 20 more
    at most), the exponential 4, the sum, quotient and product 3, three more products: below 24, and 80 for the long row.  The slope
    of the gate, s (1 + g (1 - s)), is looked at below -3, where neither difference cancels by more than half.  The gate's value
    and slope are normal numbers (above exp(-85)), but their product with a small x or gradient, the last on its way, may lie below
    2^-126: it is then a multiple of 2^-149, off by half of that."""
    c = _make(D, 3, D, dtype, (False, activation, False, False, False))
    c["gate"] = torch.linspace(-85, 85, 3 * D, dtype=torch.float64).to(dtype).double().reshape(3, D)
    c["activation"] = activation
    got = _run(lambda t: _ours(ps, c["eps"])(dict(t, activation=activation)), _gpu(c, dtype))
    exact, _ = so.norm_bounds(c, dtype)
    units = (24 if D == 8 else 80) * so.half_step(dtype)
    for name, where in (("h", c["gate"] == c["gate"]), ("grad_gate", c["gate"] < -3)):
        off = (got[name].double().cpu() - exact[name]).abs()[where]
        assert not (off > units * exact[name].abs()[where] + 2.0 ** -150).any(), (name, float((off / exact[name].abs()[where]).max() / so.half_step(dtype)))


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing is set up at a first call that a capture forbids: attributes of kernels, the word that tells of failures, tensor maps."""
    code = """
import torch, pathsig_b200 as ps
x = torch.randn(2400, 1528, device="cuda")
w = torch.ones(1528, device="cuda")
q = torch.randn(2, 300, 4, 64, device="cuda")
d = torch.full((4,), -0.1, device="cuda")
s = torch.zeros(2, 4, 64, 64, device="cuda")
torch.cuda.synchronize()
op = torch.ops.pathsig_b200
def calls(s):
    return (ps.gated_residual_norm(x, w), *op.gated_residual_norm_backward(x, w, None, None, None, None, x, None, 0, 1e-6)[:2],
            ps.linear_attention(q, q, q, d), ps.linear_attention(q.half(), q.half(), q.half(), d), ps.linear_attention(*(3 * [q.bfloat16()]), d),
            *op.linear_attention_backward(q, q, q, d, None, None, q, None, 0.1, True)[:4], ps.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], d, s), s)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls(s)
graph.replay()
torch.cuda.synchronize()
for a, b in zip(got, calls(torch.zeros_like(s))):
    assert torch.equal(a, b)
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
