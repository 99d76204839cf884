"""CPU tests of the sequence operators' host side: entry points' checks without a GPU, shapes of fake tensors,
refusals, and the oracle against automatic differentiation."""
from __future__ import annotations

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode

import pathsig_b200 as ps
from pathsig_b200 import _load

from . import sequence_oracle as so


def _attn(**change):
    d = _load.AttnDesc()
    d.dtype, d.dk, d.dv, d.H, d.Hkv, d.B, d.L, d.scale = 0, 8, 8, 4, 2, 2, 5, 1.0
    for n, v in change.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("change,status", [(dict(dtype=4), -2), (dict(dtype=-1), -2), (dict(Hkv=3), -4), (dict(H=0), -4), (dict(B=-1), -4),
                                           (dict(dk=257), -8), (dict(dv=0), -4), (dict(B=2 ** 30), -8)])
def test_attention_descriptions_are_checked(change, status):
    lib = _load.ensure_loaded()
    d = ctypes.byref(_attn(**change))
    assert lib.psig_attn_forward_workspace(d) == status
    assert lib.psig_attn_backward_workspace(d) == status
    assert lib.psig_attn_forward(d, *[None] * 8, 0, None) == status
    assert lib.psig_attn_backward(d, *[None] * 13, 0, None) == status
    assert lib.psig_attn_step(d, *[None] * 7) == status


def test_missing_pointers_and_workspaces_are_refused():
    lib = _load.ensure_loaded()
    d = ctypes.byref(_attn())
    one = ctypes.c_void_p(256)     # never dereferenced: every call below is refused on the host
    assert lib.psig_attn_forward(d, *[None] * 8, 0, None) == -1
    assert lib.psig_attn_step(d, *[None] * 7) == -1
    assert lib.psig_attn_backward(d, *[None] * 13, 0, None) == -1
    need = lib.psig_attn_backward_workspace(d)
    assert need > 0
    assert lib.psig_attn_backward(d, *[one] * 12, None, need, None) == -6
    assert lib.psig_attn_backward(d, *[one] * 12, one, need - 1, None) == -6
    assert lib.psig_attn_forward(None, *[None] * 8, 0, None) == -1
    n = _load.NormDesc()
    n.dtype, n.rows, n.D, n.eps = 0, 3, 8, 1e-6
    assert lib.psig_norm_forward(ctypes.byref(n), *[None] * 9) == -1
    need = lib.psig_norm_backward_workspace(ctypes.byref(n))
    assert need > 0
    assert lib.psig_norm_backward(ctypes.byref(n), one, None, None, None, None, None, one, None, *[None] * 6, one, need - 1, None) == -6
    n.activation = 2
    assert lib.psig_norm_forward(ctypes.byref(n), *[None] * 9) == -4
    n.activation, n.dtype = 0, 9
    assert lib.psig_norm_backward_workspace(ctypes.byref(n)) == -2


def test_parts_of_long_sequences_need_a_workspace():
    lib = _load.ensure_loaded()
    one = ctypes.c_void_p(256)
    short, long = _attn(B=1, H=2, L=500), _attn(B=1, H=2, L=16384)
    assert lib.psig_attn_forward_workspace(ctypes.byref(short)) == 0
    need = lib.psig_attn_forward_workspace(ctypes.byref(long))
    assert need >= 2 * 2 * 4 * 64 * 64          # two heads, two parts or more, a tile of states each
    assert lib.psig_attn_forward(ctypes.byref(long), one, one, one, one, None, one, None, None, 0, None) == -6
    assert lib.psig_attn_forward(ctypes.byref(long), one, one, one, one, None, one, None, one, need - 1, None) == -6
    assert lib.psig_attn_backward_workspace(ctypes.byref(long)) > need
    many = _attn(B=64, H=16, L=16384)           # enough blocks without
    assert lib.psig_attn_forward_workspace(ctypes.byref(many)) == 0


def test_nothing_to_do_is_no_error():
    lib = _load.ensure_loaded()
    d = ctypes.byref(_attn(B=0))
    assert lib.psig_attn_forward(d, *[None] * 8, 0, None) == 0
    assert lib.psig_attn_step(d, *[None] * 7) == 0
    assert lib.psig_attn_backward(d, *[None] * 13, 0, None) == 0


def test_fake_tensors_give_the_shapes():
    with FakeTensorMode():
        op = torch.ops.pathsig_b200
        q, k, v = (torch.empty(2, 9, h, d, device="cuda", dtype=torch.bfloat16) for h, d in ((4, 16), (2, 16), (2, 24)))
        decay = torch.empty(2, 9, 4, device="cuda")
        out, state = ps.linear_attention(q, k, v, decay, return_state=True)
        assert out.shape == (2, 9, 4, 24) and out.dtype == torch.bfloat16
        assert state.shape == (2, 4, 16, 24) and state.dtype == torch.float32
        grads = op.linear_attention_backward(q, k, v, decay, state, None, out, None, 1.0, True)
        assert [g.shape for g in grads] == [t.shape for t in (q, k, v, decay, state)]
        assert ps.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay[:, 0], state).shape == (2, 4, 24)
        x = torch.empty(3, 5, 32, device="cuda")
        w = torch.empty(32, device="cuda")
        h, n = ps.gated_residual_norm(x, w, gate=x, next_weight=w)
        assert h.shape == n.shape == x.shape
        assert ps.gated_residual_norm(x).shape == x.shape
        grads = op.gated_residual_norm_backward(x, w, None, x, None, w, h, n, 0, 1e-6)
        assert [g.shape for g in grads] == [x.shape, w.shape, (0,), x.shape, (0,), w.shape]


def test_refusals_without_a_gpu():
    z = torch.zeros
    with pytest.raises(NotImplementedError):
        ps.linear_attention(z(1, 2, 1, 4), z(1, 2, 1, 4), z(1, 2, 1, 4), z(1))
    with pytest.raises(NotImplementedError):
        ps.gated_residual_norm(z(2, 4))
    with pytest.raises(RuntimeError, match="not differentiable"):
        ps.linear_attention_step(z(1, 1, 4, requires_grad=True), z(1, 1, 4), z(1, 1, 4), z(1), z(1, 1, 4, 4))
    with pytest.raises(ValueError, match="activation"):
        ps.gated_residual_norm(z(2, 4), activation="relu")
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            ps.gated_residual_norm(z(2, 4), eps=eps)
    for scale in (float("inf"), float("nan"), z(1)):
        with pytest.raises(ValueError, match="scale"):
            ps.linear_attention(z(1, 2, 1, 4), z(1, 2, 1, 4), z(1, 2, 1, 4), z(1), scale=scale)


@pytest.mark.parametrize("decay", ["step", "head"])
def test_oracle_gradients_against_automatic_differentiation(decay):
    c = so.make(3, 2, 12, 4, 2, 3, 5, torch.float64, decay=decay, state=True, lengths=torch.tensor([12, 7]))
    names = ("q", "k", "v", "log_decay", "initial_state")
    leaves = {n: c[n].clone().requires_grad_(True) for n in names}
    got = so.attention({**c, **leaves})
    want = torch.autograd.grad((got["out"] * c["grad_out"]).sum() + (got["state"] * c["grad_state"]).sum(), list(leaves.values()))
    plain = so.attention(c)
    for n, w in zip(names, want):
        assert torch.allclose(plain["grad_" + n], w, rtol=1e-11, atol=1e-12), n


def test_the_step_raises_the_version_of_its_state():
    """By which a graph that has saved the state refuses its backward pass, as with torch's own operators in place."""
    with FakeTensorMode():
        q, k, v = (torch.empty(2, 4, 8, device="cuda") for _ in range(3))
        decay, state = torch.empty(4, device="cuda"), torch.empty(2, 4, 8, 8, device="cuda")
        view = state[0]
        for n in range(1, 4):
            ps.linear_attention_step(q, k, v, decay, state)
            assert state._version == n and view._version == n
        assert q._version == k._version == v._version == decay._version == 0
        with torch.no_grad():
            ps.linear_attention_step(q, k, v, decay, state)
        assert state._version == 4
        with torch.inference_mode():
            ps.linear_attention_step(q, k, v, decay, state)
            ps.linear_attention_step(q, k, v, decay, torch.empty(2, 4, 8, 8, device="cuda"))   # has no version


@pytest.mark.parametrize("namespace", ["pathsig_b200", "pathsig"])
def test_forward_mode_is_refused(namespace):
    """An operand with a tangent, whether or not another requires a gradient; by the compiled operators, so under both names."""
    ps.ops.register_namespace("pathsig")
    op = getattr(torch.ops, namespace)
    with FakeTensorMode(), forward_ad.dual_level():
        z = lambda *s: torch.empty(*s, device="cuda")
        attention = (z(2, 5, 4, 8), z(2, 5, 2, 8), z(2, 5, 2, 6), z(4), z(2, 4, 8, 6))
        norm = (z(3, 8), z(8), z(3, 8), z(3, 8), z(8), z(8))
        step = (z(2, 4, 8), z(2, 2, 8), z(2, 2, 6), z(4), z(2, 4, 8, 6))
        out, state = z(2, 5, 4, 6), z(2, 4, 8, 6)
        calls = {
            "linear_attention": (attention, lambda a: op.linear_attention(*a, None, 1.0, True)),
            "linear_attention_backward": (attention + (out, state),
                                          lambda a: op.linear_attention_backward(*a[:5], None, *a[5:], 1.0, True)),
            "linear_attention_step": (step, lambda a: op.linear_attention_step(*a, 1.0)),
            "gated_residual_norm": (norm, lambda a: op.gated_residual_norm(*a, 0, 1e-6)),
            "gated_residual_norm_backward": (norm + (norm[0], norm[0]), lambda a: op.gated_residual_norm_backward(*a, 0, 1e-6)),
        }
        for name, (operands, call) in calls.items():
            call(operands)
            for i, t in enumerate(operands):
                dual = list(operands)
                dual[i] = forward_ad.make_dual(t, torch.empty_like(t))
                with pytest.raises(RuntimeError, match=name + " has no forward-mode"):
                    call(dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(dual)


def test_the_other_namespace_runs_the_same_operators():
    ps.ops.register_namespace("pathsig")
    with FakeTensorMode():
        q, k, v = (torch.empty(2, 9, h, d, device="cuda") for h, d in ((4, 16), (2, 16), (2, 24)))
        decay = torch.empty(4, device="cuda", requires_grad=True)
        out, state = torch.ops.pathsig.linear_attention(q, k, v, decay, None, None, 1.0, True)
        assert out.shape == (2, 9, 4, 24) and state.shape == (2, 4, 16, 24) and out.requires_grad and state.requires_grad
        state = state.detach()
        torch.ops.pathsig.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay.detach(), state, 1.0)
        assert state._version == 1
    with pytest.raises(NotImplementedError):
        torch.ops.pathsig.gated_residual_norm(torch.zeros(2, 4), None, None, None, None, None, 0, 1e-6)
