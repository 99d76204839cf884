"""Decayed linear attention on the GPU against a 64-bit recurrence (sequence_oracle.py), element by element within
rounding bounds derived there: sizes, types, shared heads, lengths, decays that forget everything, strides, states
handed from one call to the next, single steps, streams, graphs, refusals."""
from __future__ import annotations

import pytest
import torch

from . import sequence_oracle as so
from . import util

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float64, torch.float32, torch.bfloat16, torch.float16]
NAMES = ("q", "k", "v", "log_decay", "initial_state")


@pytest.fixture(scope="module")
def ps():
    import pathsig_b200
    return pathsig_b200


def _on_gpu(c, dtype):
    sums = torch.float64 if dtype == torch.float64 else torch.float32
    kinds = {"q": dtype, "k": dtype, "v": dtype, "grad_out": dtype, "log_decay": sums, "initial_state": sums,
             "grad_state": sums}
    got = {n: c[n].to(t).to(DEV) if c[n] is not None else None for n, t in kinds.items()}
    got["lengths"] = c["lengths"].to(DEV) if c["lengths"] is not None else None
    return got


def _run(ps, g, scale=None):
    leaves = [g[n].detach().requires_grad_(True) if g[n] is not None else None for n in NAMES]
    got = ps.linear_attention(*leaves[:4], initial_state=leaves[4], lengths=g["lengths"], return_state=True, scale=scale)
    outputs = {"out": got[0].detach(), "state": got[1].detach()}
    heads, grads = [got[0]], [g["grad_out"]]
    if g["grad_state"] is not None:
        heads.append(got[1])
        grads.append(g["grad_state"])
    wanted = [(n, t) for n, t in zip(NAMES, leaves) if t is not None]
    for (n, _), d in zip(wanted, torch.autograd.grad(heads, [t for _, t in wanted], grads)):
        outputs["grad_" + n] = d
    return outputs


def _check(got, exact, bounds):
    for name, want in exact.items():
        if name.startswith("_") or name not in got:
            continue
        off = (got[name].double().cpu() - want).abs()
        assert got[name].shape == want.shape, name
        bad = ~(off <= bounds[name])
        assert not bad.any(), (name, int(bad.sum()), float(off[bad].max()), float((off / bounds[name].clamp_min(1e-300)).nan_to_num(0).max()))


SHAPES = [  # B, L, H, Hkv, Dk, Dv
    (1, 1, 1, 1, 1, 1),
    (2, 2, 2, 1, 3, 5),
    (3, 17, 4, 2, 16, 32),
    (2, 61, 8, 8, 64, 64),
    (1, 63, 2, 1, 64, 128),
    (2, 64, 3, 3, 40, 24),
    (1, 65, 2, 2, 128, 64),
    (2, 127, 2, 1, 48, 80),
    (1, 128, 2, 2, 128, 128),
    (2, 129, 4, 1, 72, 120),
    (1, 257, 2, 2, 33, 65),
    (1, 513, 2, 1, 64, 64),
    (1, 640, 1, 1, 128, 128),
    (1, 70, 2, 1, 256, 200),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_outputs_and_gradients(ps, shape, dtype):
    state = shape[1] % 2 == 1
    decay = ("step", "head")[sum(shape) % 2]
    c = so.make(sum(shape), *shape, dtype, decay=decay, state=state)
    _check(_run(ps, _on_gpu(c, dtype)), *so.attention_bounds(c, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("decay", ["none", "strong", "forget"])
@pytest.mark.parametrize("shape", [(2, 150, 2, 1, 64, 64), (1, 520, 2, 2, 32, 128)])
def test_extreme_decays(ps, shape, decay, dtype):
    c = so.make(7, *shape, dtype, decay=decay, state=True)
    got = _run(ps, _on_gpu(c, dtype))
    _check(got, *so.attention_bounds(c, dtype))
    if decay == "forget":
        assert not got["grad_log_decay"][torch.isinf(c["log_decay"]).to(DEV)].any()
        assert not got["grad_initial_state"].any()    # the first step forgets it


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_lengths_leave_later_rows_alone(ps, dtype, kind):
    """Lengths of zero, one, past a piece's end, the whole, and out of range; rows behind them hold NaN and infinities."""
    lengths = torch.tensor([0, 1, 64, 65, 128, 129, 200, 999, -3], dtype=kind)
    c = so.make(3, 9, 200, 4, 2, 64, 32, dtype, state=True, lengths=lengths)
    exact, bounds = so.attention_bounds(c, dtype)
    g = _on_gpu(c, dtype)
    behind = torch.arange(200, device=DEV) >= lengths.to(DEV).clamp(0, 200)[:, None]
    for name in ("q", "k", "v", "grad_out", "log_decay"):
        g[name][behind] = float("nan")
    g["q"][8] = float("inf")
    got = _run(ps, g)
    _check(got, exact, bounds)
    for name in ("out", "grad_q", "grad_k", "grad_v", "grad_log_decay"):
        assert not got[name][behind].any(), name
    assert torch.equal(got["state"][0], g["initial_state"][0]) and torch.equal(got["grad_initial_state"][0], g["grad_state"][0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(ps, dtype):
    """Slices of one fused projection, a transposed batch, an odd offset and a last dimension that is not dense."""
    B, L, H, D = 2, 140, 4, 64
    c = so.make(11, B, L, H, H, D, D, dtype)
    g = _on_gpu(c, dtype)
    want = _run(ps, g)
    _check(want, *so.attention_bounds(c, dtype))
    fused = torch.cat([g["q"], g["k"], g["v"]], dim=2).reshape(B, L, 3, H, D)
    forms = {
        "fused": [fused[:, :, i] for i in range(3)],
        "heads first": [g[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v")],
        "time first": [g[n].transpose(0, 1).contiguous().transpose(0, 1) for n in ("q", "k", "v")],
        "odd offset": [torch.nn.functional.pad(g[n].reshape(-1), (1, 0))[1:].view(B, L, H, D) for n in ("q", "k", "v")],
        "odd rows": [torch.nn.functional.pad(g[n], (0, 3))[..., :D] for n in ("q", "k", "v")],
        "last not dense": [torch.stack([g[n], g[n]], dim=-1)[..., 0] for n in ("q", "k", "v")],
    }
    for form, (q, k, v) in forms.items():
        got = _run(ps, dict(g, q=q, k=k, v=v, grad_out=g["grad_out"].transpose(1, 2).contiguous().transpose(1, 2)))
        _check(got, *so.attention_bounds(c, dtype))


def test_broadcast_operands_get_summed_gradients(ps):
    c = so.make(5, 3, 40, 2, 2, 16, 16, torch.float64)
    g = _on_gpu(c, torch.float64)
    k0 = g["k"][:1, :, :1].clone().requires_grad_(True)
    d0 = g["log_decay"][:1].clone().requires_grad_(True)
    out = ps.linear_attention(g["q"], k0.expand(3, -1, 2, -1), g["v"], d0.expand(3, -1, -1))
    out.backward(torch.ones((), dtype=out.dtype, device=DEV).expand_as(out))
    c |= {"k": k0.detach().cpu().expand(3, -1, 2, -1), "log_decay": d0.detach().cpu().expand(3, -1, -1).clone(),
          "grad_out": torch.ones_like(c["grad_out"])}
    want = so.attention(c)
    assert util.rel_error(k0.grad, want["grad_k"].sum((0, 2), keepdim=True)) < 1e-12
    assert util.rel_error(d0.grad, want["grad_log_decay"].sum(0, keepdim=True)) < 1e-12


@pytest.mark.parametrize("decay", ["step", "head"])
def test_gradients_against_differences(ps, decay):
    c = so.make(9, 2, 9, 2, 1, 3, 4, torch.float64, decay=decay, state=True, lengths=torch.tensor([9, 6]))
    g = _on_gpu(c, torch.float64)
    leaves = [g[n].requires_grad_(True) for n in NAMES]
    assert torch.autograd.gradcheck(
        lambda q, k, v, d, s: ps.linear_attention(q, k, v, d, initial_state=s, lengths=g["lengths"], return_state=True),
        leaves, eps=1e-6, atol=1e-8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pieces_and_steps_give_the_whole(ps, dtype):
    """A sequence in one call, in three calls that hand the state on, and one step at a time; shared heads."""
    c = so.make(13, 2, 150, 4, 2, 64, 40, dtype, state=True)
    exact, bounds = so.attention_bounds(c, dtype)
    g = _on_gpu(c, dtype)
    args = [g[n] for n in ("q", "k", "v", "log_decay")]
    state, outs = g["initial_state"], []
    for a, b in ((0, 1), (1, 100), (100, 150)):
        o, state = ps.linear_attention(*[t[:, a:b] for t in args], initial_state=state, return_state=True)
        outs.append(o)
    _check({"out": torch.cat(outs, 1), "state": state}, exact, bounds)
    state, outs = g["initial_state"].clone(), []
    for t in range(150):
        outs.append(ps.linear_attention_step(*[x[:, t] for x in args], state))
    _check({"out": torch.stack(outs, 1), "state": state}, exact, bounds)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,H,Hkv,Dk,Dv", [(1, 1, 1, 1, 1), (3, 4, 2, 5, 33), (2, 8, 8, 64, 64), (5, 6, 2, 48, 80),
                                           (300, 16, 4, 128, 128), (2, 2, 1, 256, 256), (2, 3, 3, 31, 100)])
@pytest.mark.parametrize("decay", ["step", "head"])
def test_single_steps(ps, B, H, Hkv, Dk, Dv, dtype, decay):
    c = so.make(B + Dk, B, 1, H, Hkv, Dk, Dv, dtype, decay=decay, state=True)
    exact, bounds = so.attention_bounds(c, dtype)
    g = _on_gpu(c, dtype)
    state = g["initial_state"]
    d = g["log_decay"] if decay == "head" else g["log_decay"][:, 0]
    out = ps.linear_attention_step(g["q"][:, 0], g["k"][:, 0], g["v"][:, 0], d, state)
    _check({"out": out[:, None], "state": state}, exact, bounds)


def test_step_forgets_and_keeps_dtype(ps):
    c = so.make(1, 2, 1, 2, 2, 8, 8, torch.float16, decay="forget", state=True)
    g = _on_gpu(c, torch.float16)
    state = g["initial_state"]
    out = ps.linear_attention_step(g["q"][:, 0], g["k"][:, 0], g["v"][:, 0], g["log_decay"][:, 0], state)
    assert out.dtype == torch.float16 and state.dtype == torch.float32
    assert torch.equal(state, g["k"][:, 0, :, :, None].float() * g["v"][:, 0, :, None, :].float())


def test_second_degree_of_the_signature(ps):
    """Without decay, with keys x_{t-1} - x_0 + dx_t / 2 and values dx_t, the state is the degree-2 part of Signature."""
    d, L = 5, 90
    x = util.brownian_path(4, L, d, seed=3, dtype=torch.float64).to(DEV).requires_grad_(True)
    dx = x.diff(dim=1)
    keys = x[:, :-1] - x[:, :1] + dx / 2
    _, state = ps.linear_attention(keys[:, :, None], keys[:, :, None], dx[:, :, None], torch.zeros(1, dtype=torch.float64, device=DEV),
                                   return_state=True)
    sig = ps.Signature(depth=2)(x)[:, d:]
    assert util.rel_error(state.flatten(1), sig) < 1e-12
    g = torch.randn(4, d * d, dtype=torch.float64, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    ours, = torch.autograd.grad(state.flatten(1), x, g)
    theirs, = torch.autograd.grad(sig, x, g)
    assert util.rel_error(ours, theirs) < 1e-12


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_only_some_gradients(ps, dtype):
    c = so.make(2, 2, 70, 2, 1, 64, 64, dtype, state=True)
    exact, bounds = so.attention_bounds(dict(c, grad_out=torch.zeros_like(c["grad_out"])), dtype)
    g = _on_gpu(c, dtype)
    v = g["v"].requires_grad_(True)
    s = g["initial_state"].requires_grad_(True)
    out, state = ps.linear_attention(g["q"], g["k"], v, g["log_decay"], initial_state=s, return_state=True)
    dv, ds = torch.autograd.grad(state, (v, s), g["grad_state"])     # nothing comes in through the output
    _check({"grad_v": dv, "grad_initial_state": ds}, exact, bounds)
    out = ps.linear_attention(g["q"], g["k"], v.detach(), g["log_decay"])
    assert not out.requires_grad


def test_empty_sizes(ps):
    z = torch.zeros
    out, s = ps.linear_attention(z(0, 5, 2, 8, device=DEV), z(0, 5, 2, 8, device=DEV), z(0, 5, 2, 4, device=DEV), z(2, device=DEV), return_state=True)
    assert out.shape == (0, 5, 2, 4) and s.shape == (0, 2, 8, 4)
    init = torch.randn(3, 2, 8, 4, device=DEV).requires_grad_(True)
    q = z(3, 0, 2, 8, device=DEV, requires_grad=True)
    out, s = ps.linear_attention(q, q.detach(), z(3, 0, 2, 4, device=DEV), z(2, device=DEV), initial_state=init, return_state=True)
    assert out.shape == (3, 0, 2, 4) and torch.equal(s, init)
    assert torch.equal(torch.autograd.grad(s.sum() + out.sum(), init)[0], torch.ones_like(init))
    assert ps.linear_attention_step(z(0, 2, 8, device=DEV), z(0, 2, 8, device=DEV), z(0, 2, 4, device=DEV), z(2, device=DEV),
                                    z(0, 2, 8, 4, device=DEV)).shape == (0, 2, 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_bits_every_run_and_on_another_stream(ps, dtype):
    c = so.make(21, 3, 700, 4, 2, 64, 64, dtype, state=True, lengths=torch.tensor([700, 333, 0]))
    g = _on_gpu(c, dtype)
    first = _run(ps, g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _run(ps, g)
    torch.cuda.current_stream().wait_stream(side)
    for name in first:
        assert torch.equal(first[name], second[name]), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_replayed(ps, dtype):
    """Two captured graphs (forward with backward, and a step) replayed on new contents of the same buffers, in turn."""
    one, two = (so.make(s, 2, 130, 4, 2, 64, 64, dtype, state=True) for s in (1, 2))
    static, other = _on_gpu(one, dtype), _on_gpu(two, dtype)
    step_state = static["initial_state"].clone()

    def grads():
        go, gs = static["grad_out"], static["grad_state"]
        return torch.ops.pathsig_b200.linear_attention_backward(
            static["q"], static["k"], static["v"], static["log_decay"], static["initial_state"], None, go, gs, 0.125, True)

    def step():
        return ps.linear_attention_step(static["q"][:, 0], static["k"][:, 0], static["v"][:, 0], static["log_decay"][:, 0], step_state)

    def whole():
        return ps.linear_attention(static["q"], static["k"], static["v"], static["log_decay"],
                                   initial_state=static["initial_state"], return_state=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        whole(), grads(), step()
    torch.cuda.current_stream().wait_stream(side)
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a):
        out, state = whole()
        got = grads()
    with torch.cuda.graph(b):
        stepped = step()
    for name in NAMES + ("grad_out", "grad_state"):
        static[name].copy_(other[name])
    step_state.copy_(other["initial_state"])
    a.replay(), b.replay(), a.replay()
    torch.cuda.synchronize()
    exact, bounds = so.attention_bounds(two, dtype)
    _check({"out": out, "state": state, **{"grad_" + n: t for n, t in zip(NAMES, got)}}, exact, bounds)
    first = {n: (t[:, :1] if isinstance(t, torch.Tensor) and n in ("q", "k", "v", "log_decay", "grad_out") else t) for n, t in two.items()}
    exact, bounds = so.attention_bounds(first, dtype)
    _check({"out": stepped[:, None], "state": step_state}, exact, bounds)


def test_traced_by_torch_compile(ps):
    c = so.make(4, 2, 40, 2, 2, 16, 16, torch.float32)
    g = _on_gpu(c, torch.float32)
    f = torch.compile(lambda q, k, v, d: ps.linear_attention(q, k, v, d).square().sum(), backend="aot_eager", fullgraph=True)
    leaves = [g[n].clone().requires_grad_(True) for n in NAMES[:4]]
    f(*leaves).backward()
    plain = [g[n].clone().requires_grad_(True) for n in NAMES[:4]]
    ps.linear_attention(*plain).square().sum().backward()
    for a, b in zip(leaves, plain):
        assert torch.equal(a.grad, b.grad)


def test_many_sequences_and_heads(ps):
    """More (sequence, head) pairs than one grid dimension of 65535 holds."""
    c = so.make(6, 9000, 2, 8, 8, 4, 4, torch.float32)
    _check(_run(ps, _on_gpu(c, torch.float32)), *so.attention_bounds(c, torch.float32))


LONG = [  # few long sequences are swept in parts, many short ones several to a block
    ((1, 1200, 2, 1, 64, 64), None),
    ((2, 1100, 2, 2, 128, 96), [1100, 700]),
    ((1, 1700, 1, 1, 40, 128), None),
    ((3, 1030, 1, 1, 64, 64), [0, 1030, 130]),
    ((1, 1153, 1, 1, 128, 128), [1]),
    ((50, 150, 4, 2, 64, 32), "random"),
    ((70, 61, 4, 4, 32, 64), None),
    ((40, 300, 4, 1, 96, 128), "random"),
]


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("shape,lengths", LONG)
@pytest.mark.parametrize("state", [False, True])
def test_sequences_in_parts_and_several_to_a_block(ps, shape, lengths, state, dtype):
    if lengths is not None:
        gen = torch.Generator().manual_seed(shape[1])
        lengths = torch.randint(0, shape[1] + 1, (shape[0],), generator=gen) if lengths == "random" else torch.tensor(lengths)
    c = so.make(sum(shape), *shape, dtype, state=state, lengths=lengths, rate=0.02)
    _check(_run(ps, _on_gpu(c, dtype)), *so.attention_bounds(c, dtype))
    _no_timeouts()


def _no_timeouts():
    from pathsig_b200 import _load
    assert _load.ensure_loaded().psig_sequence_wait_timeouts() == 0


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("shape", [(2, 61, 8, 8, 64, 64), (1, 300, 4, 2, 128, 72)])
def test_kernels_of_every_size_at_the_sizes_of_the_others(ps, shape, dtype):
    c = so.make(17, *shape, dtype, state=True)
    ps.ops.set_algorithm("generic")
    try:
        got = _run(ps, _on_gpu(c, dtype))
    finally:
        ps.ops.set_algorithm("auto")
    _check(got, *so.attention_bounds(c, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, 1.0, -2.5])
def test_scales(ps, dtype, scale):
    c = so.make(23, 2, 140, 2, 1, 64, 64, dtype, state=True) | {"scale": scale}
    got = _run(ps, _on_gpu(c, dtype), scale=scale)
    _check(got, *so.attention_bounds(c, dtype))
    if scale == 0.0:
        assert not got["out"].any() and not got["grad_q"].any()


def test_float16_scores_and_states_beyond_its_range(ps):
    """Scores of 128 * 300 * 300 and sums of 200 such products do not fit float16; the results do."""
    c = so.make(29, 1, 200, 1, 1, 128, 64, torch.float16, decay="none")
    for n, size in (("q", 300.0), ("k", 300.0), ("v", 2.0 ** -14), ("grad_out", 2.0 ** -14)):
        c[n] = (c[n].sign() * size * (1 + c[n].abs() / 64)).to(torch.float16).double()
    c["q"], c["k"] = c["q"].abs(), c["k"].abs()
    exact, bounds = so.attention_bounds(c, torch.float16)
    got = _run(ps, _on_gpu(c, torch.float16))
    assert float(exact["out"].abs().max()) < 65504
    _check({n: got[n] for n in ("out", "state")}, exact, bounds)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_offsets_beyond_32_bits(ps, dtype):
    """Operands of more than 2^31 elements: the last heads of the last steps against a call on those heads alone."""
    L, H, D = 65664, 256, 128
    gen = torch.Generator(DEV).manual_seed(3)
    big = torch.randn(1, L, H, D, device=DEV, generator=gen, dtype=dtype)
    assert big.numel() > 2 ** 31
    decay = -torch.rand(H, device=DEV, generator=gen)
    out, state = ps.linear_attention(big, big, big, decay, return_state=True)
    few = big[:, :, -2:].contiguous()
    want, want_state = ps.linear_attention(few, few, few, decay[-2:], return_state=True)
    # the few heads are swept in parts, so sums run in another order: one rounding of the storage type, and of sums
    apart = 2 * so.half_step(dtype) if dtype == torch.bfloat16 else 3e-6
    assert util.rel_error(out[:, -3000:, -2:], want[:, -3000:]) < apart
    assert util.rel_error(state[:, -2:], want_state) < 3e-6
    del out, big
    torch.cuda.empty_cache()


def test_concurrent_host_threads_and_streams(ps):
    import threading
    c = so.make(31, 3, 300, 4, 2, 64, 64, torch.bfloat16, state=True)
    g = _on_gpu(c, torch.bfloat16)
    want = _run(ps, g)
    torch.cuda.synchronize()
    results, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    results[i] = _run(ps, g)
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for got in results.values():
        for name in want:
            assert torch.equal(got[name], want[name]), name
    _no_timeouts()


def test_refusals_on_the_gpu(ps):
    f = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device=DEV)
    q, k, v, d = f(2, 5, 4, 8), f(2, 5, 2, 8), f(2, 5, 2, 6), f(4)
    ps.linear_attention(q, k, v, d)
    bad = [
        (dict(q=f(2, 5, 3, 8), d=f(3)), "multiple"), (dict(k=f(2, 5, 2, 9)), "head size"), (dict(v=f(2, 4, 2, 6)), "agree"),
        (dict(v=f(2, 5, 4, 6)), "same number of heads"), (dict(d=f(5)), "log_decay"), (dict(d=f(2, 5, 2)), "log_decay"),
        (dict(d=f(4, t=torch.float64)), "log_decay"), (dict(k=f(2, 5, 2, 8, t=torch.bfloat16)), "k must be"),
        (dict(q=f(5, 4, 8)), "shape"), (dict(q=f(2, 5, 4, 300), k=f(2, 5, 2, 300)), "256"),
        (dict(q=torch.zeros(2, 5, 4, 8, dtype=torch.int32, device=DEV)), "float32"),
    ]
    for change, message in bad:
        a = {"q": q, "k": k, "v": v, "d": d} | change
        with pytest.raises(RuntimeError, match=message):
            ps.linear_attention(a["q"], a["k"], a["v"], a["d"])
    for more, message in [(dict(initial_state=f(2, 4, 8, 5)), "initial_state"), (dict(initial_state=f(2, 4, 8, 6, t=torch.bfloat16)), "initial_state"),
                          (dict(lengths=torch.zeros(3, dtype=torch.int32, device=DEV)), "lengths"), (dict(lengths=f(2)), "lengths"),
                          (dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths")]:
        with pytest.raises(RuntimeError, match=message):
            ps.linear_attention(q, k, v, d, **more)
    with pytest.raises(ValueError, match="scale"):
        ps.linear_attention(q, k, v, d, scale=float("nan"))
    state = f(2, 4, 8, 6)
    step = (q[:, 0], k[:, 0], v[:, 0], d)
    with pytest.raises(RuntimeError, match="contiguous"):
        ps.linear_attention_step(*step, f(2, 4, 6, 8).transpose(2, 3))
    with pytest.raises(RuntimeError, match="share memory"):
        ps.linear_attention_step(state.view(-1)[: 2 * 4 * 8].view(2, 4, 8), *step[1:], state)
    with pytest.raises(RuntimeError, match="not differentiable"):
        ps.linear_attention_step(q[:, 0].clone().requires_grad_(True), *step[1:], state)
    with pytest.raises(RuntimeError, match="state"):
        ps.linear_attention_step(*step, f(1, 4, 8, 6))
    many = torch.zeros(1, 1, 1, 1, device=DEV)
    for heads in (65536, 2 ** 32 + 1):   # would be 1 in 32 bits
        with pytest.raises(RuntimeError, match="65535 heads"):
            ps.linear_attention(many.expand(1, 1, heads, 1), many, many, f(1))


def test_second_derivatives_are_refused(ps):
    """A gradient with a graph of its own is the plain gradient; its gradient is refused, not left out."""
    q, k, v = (torch.randn(1, 6, 2, 8, device=DEV, requires_grad=True) for _ in range(3))
    d = torch.full((2,), -0.1, device=DEV, requires_grad=True)
    leaves = (q, k, v, d)
    plain = torch.autograd.grad(ps.linear_attention(*leaves).square().sum(), leaves)
    graph = torch.autograd.grad(ps.linear_attention(*leaves).square().sum(), leaves, create_graph=True)
    for a, b in zip(plain, graph):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="differentiable once"):
        graph[0].sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("steps", [1, 2, 3, 16, 17])
def test_short_sequences_on_both_sides_of_the_kernels_limits(ps, steps, state, dtype):
    c = so.make(steps + 40, 2, steps, 4, 2, 40, 72, dtype, state=state)
    g = _on_gpu(c, dtype)
    exact, bounds = so.attention_bounds(c, dtype)
    _check(_run(ps, g), exact, bounds)
    out = ps.linear_attention(*(g[n] for n in NAMES[:4]), initial_state=g["initial_state"])   # no state asked for
    _check({"out": out}, exact, bounds)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("shape", [(2, 61, 8, 8, 64, 64), (2, 127, 2, 1, 48, 80), (1, 300, 2, 1, 128, 128), (1, 640, 1, 1, 128, 72),
                                   (1, 1200, 2, 1, 64, 64)])
def test_16_bit_results_are_rounded_once(ps, shape, state, dtype):
    """Weights of pairs and states enter the products as two 16-bit terms: outputs and gradients are as near as 32-bit
    arithmetic and one rounding bring them."""
    c = so.make(sum(shape) + 1, *shape, dtype, state=state, rate=0.05)
    g = _on_gpu(c, dtype)
    exact, bounds = so.attention_bounds(c, dtype, terms=2)
    _check(_run(ps, g), exact, bounds)
    out = ps.linear_attention(*(g[n] for n in NAMES[:4]), initial_state=g["initial_state"])   # no state asked for
    _check({"out": out}, exact, bounds)
    leaves = [g[n].detach().requires_grad_(True) for n in NAMES[:3]]                          # no decay gradient
    out, last = ps.linear_attention(*leaves, g["log_decay"], initial_state=g["initial_state"], return_state=True)
    heads, grads = ([out, last], [g["grad_out"], g["grad_state"]]) if state else ([out], [g["grad_out"]])
    got = torch.autograd.grad(heads, leaves, grads)
    _check({"grad_" + n: t for n, t in zip(NAMES, got)}, exact, bounds)
    _no_timeouts()


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 72)])
def test_weights_next_to_steps_that_forget(ps, Dk, Dv, dtype):
    """Pairs of steps on one side of steps that forget everything (or nearly: exp(-60)), with small decays between the two.
    One entry of one row in 32 is not zero, so a sum has at most ten terms here and its error is that of their weights: four
    exponentials on the way of a term (4 units each: 2^-22), their arguments (below 4, or the weight does not count), the sum
    of ten and two dozen products and splits: 64 units of 2^-24 cover them."""
    B, L, H = 2, 300, 4
    c = so.make(41, B, L, H, H, Dk, Dv, dtype, state=True, rate=0.01)
    gen = torch.Generator().manual_seed(9)
    for h, resets in enumerate((0, 1, 5, 15)):
        for b in range(B):
            for t0 in range(0, L, 32):
                at = t0 + torch.randperm(32, generator=gen)[:resets]
                c["log_decay"][b, at[at < L], h] = -float("inf") if b == 0 else -60.0
    for name, at in (("q", 23), ("k", 3), ("v", 3), ("grad_out", 23)):
        few = torch.zeros_like(c[name])
        for t in range(L):
            if t % 32 == at or name in ("q", "k") and t % 32 in (3, 4, 23, 24):
                few[:, t, :, 5] = c[name][:, t, :, 5]
        c[name] = few
    _check(_run(ps, _on_gpu(c, dtype)), *so.attention_bounds(c, dtype, terms=2, chain=64))
    _no_timeouts()


def test_a_state_stepped_while_a_graph_holds_it(ps):
    c = so.make(47, 2, 6, 4, 2, 16, 24, torch.float32, state=True)
    g = _on_gpu(c, torch.float32)
    args = [g[n][:, 0] for n in NAMES[:4]]
    q = g["q"].clone().requires_grad_(True)
    out = ps.linear_attention(q, *(g[n] for n in NAMES[1:4]), initial_state=g["initial_state"])
    with torch.no_grad():
        ps.linear_attention_step(*args, g["initial_state"])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    out = ps.linear_attention(q, *(g[n] for n in NAMES[1:4]), initial_state=g["initial_state"].clone())
    with torch.no_grad():
        ps.linear_attention_step(*args, g["initial_state"])
    out.sum().backward()
    assert torch.isfinite(q.grad).all()
    with torch.inference_mode():                # a state without a version
        state = c["initial_state"].to(torch.float32).to(DEV)
        out = ps.linear_attention_step(*args, state)
    other = c["initial_state"].to(torch.float32).to(DEV)
    assert torch.equal(out, ps.linear_attention_step(*args, other)) and torch.equal(state, other)


def test_operators_by_torchs_own_checks(ps):
    """Schemas (what is written in place, what aliases what), fake implementations, registration of the formulas."""
    ops = torch.ops.pathsig_b200
    c = so.make(53, 2, 20, 4, 2, 16, 24, torch.float32, state=True)
    g = _on_gpu(c, torch.float32)
    leaves = [g[n].clone().requires_grad_(True) for n in NAMES]
    lengths = torch.tensor([20, 7], device=DEV)
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(ops.linear_attention.default, (*leaves, lengths, 0.25, True), test_utils=tests)
    torch.library.opcheck(ops.linear_attention_backward.default, (*(g[n] for n in NAMES), lengths, g["grad_out"], g["grad_state"], 0.25, True),
                          test_utils=tests[:2])
    torch.library.opcheck(ops.linear_attention_step.default, (*(g[n][:, 0] for n in NAMES[:4]), g["initial_state"], 0.25), test_utils=tests[:2])
    x = torch.randn(6, 40, device=DEV)
    w = [torch.randn(40, device=DEV) for _ in range(3)]
    leaves = [t.clone().requires_grad_(True) for t in (x, w[0], x, x, w[1], w[2])]
    torch.library.opcheck(ops.gated_residual_norm.default, (*leaves, 0, 1e-6), test_utils=tests)
    torch.library.opcheck(ops.gated_residual_norm_backward.default, (x, w[0], x, x, w[1], w[2], x, x, 0, 1e-6), test_utils=tests[:2])


def test_step_and_norm_traced_by_torch_compile(ps):
    c = so.make(59, 2, 3, 2, 2, 16, 16, torch.float32, state=True)
    g = _on_gpu(c, torch.float32)
    w = torch.rand(16, device=DEV)

    def f(q, k, v, d, state, w):
        out = ps.linear_attention_step(q, k, v, d, state)
        h, n = ps.gated_residual_norm(out, w, gate=q, residual=v, next_weight=w)
        return h.square().sum() + n.sum() + state.sum()

    step = [g[n][:, 0] for n in NAMES[:4]]
    one, two = g["initial_state"].clone(), g["initial_state"].clone()
    with torch.no_grad():
        want = f(*step, one, w)
        got = torch.compile(f, backend="aot_eager", fullgraph=True)(*step, two, w)
    assert torch.equal(got, want) and torch.equal(one, two)

    def norm(x, w, r):
        h, n = ps.gated_residual_norm(x, w, gate=x, residual=r, residual_scale=w, next_weight=w)
        return h.square().sum() + n.square().sum()

    leaves = [torch.randn(5, 40, device=DEV), torch.randn(40, device=DEV), torch.randn(5, 40, device=DEV)]
    a, b = ([t.clone().requires_grad_(True) for t in leaves] for _ in range(2))
    norm(*a).backward()
    torch.compile(norm, backend="aot_eager", fullgraph=True)(*b).backward()
    for x, y in zip(a, b):
        assert torch.equal(x.grad, y.grad)


@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("steps,D", [(3, 128), (4, 128), (6, 64), (7, 64), (12, 32), (13, 32), (16, 24), (17, 24)])
def test_short_bfloat16_sequences_by_head_size(ps, steps, D, state):
    """Either side of the limit of steps by head size; both kernels give results that are rounded once."""
    c = so.make(steps + D, 3, steps, 4, 2, D, D, torch.bfloat16, state=state)
    g = _on_gpu(c, torch.bfloat16)
    exact, bounds = so.attention_bounds(c, torch.bfloat16, terms=2)
    _check(_run(ps, g), exact, bounds)
    out = ps.linear_attention(*(g[n] for n in NAMES[:4]), initial_state=g["initial_state"])
    _check({"out": out}, exact, bounds)
    _no_timeouts()
