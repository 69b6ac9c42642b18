"""Calls of the token-attention operators that are not the ordinary one: tracing and forward mode, captured backwards of leaves that the
call converts, positions made in another mode, sizes at the launch limits; and how exact the fp32 products are, normwise."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx

import mono_vifi_amd  # noqa: F401
from mono_vifi_amd import ops

gpu = pytest.mark.gpu


def heads(device="cpu", B=1, Lq=3, Lk=5, H=2, D=8):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(B, n, H, D, generator=g).to(device) for n in (Lq, Lk, Lk)]


def calls(device="cpu"):
    """(name, function, tensors) of both operators."""
    q, k, v = heads(device)
    w = torch.linspace(0.5, 1.5, q.shape[-1], device=device)
    return [("cross_attention", lambda q, k, v: ops.cross_attention(q, k, v), [q, k, v]),
            ("qk_norm_rope", lambda q, k, wq, wk: ops.qk_norm_rope(q, k, wq, wk)[0], [q, k, w, w.clone()])]


# ------------------------------------------------------------------------------------------------ routes past the operators
def refuses_forward_mode(device):
    for name, f, xs in calls(device):
        for i in range(len(xs)):
            for grad in (False, True):
                with fwAD.dual_level():
                    args = [x.clone().requires_grad_(grad) for x in xs]
                    args[i] = fwAD.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                        f(*args)


def refuses_tracing(device):
    for name, f, xs in calls(device):
        for grad in (False, True):
            args = tuple(x.clone().requires_grad_(grad) for x in xs)
            with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
                torch.jit.trace(f, args)
            with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
                make_fx(f)(*args)


def test_forward_mode_is_refused():
    """A tangent that would be dropped: refused before the device is looked at, whichever input carries it."""
    refuses_forward_mode("cpu")


def test_tracing_is_refused():
    """A trace would hold the allocation of the output and not the kernels that fill it."""
    refuses_tracing("cpu")
    from mono_vifi_amd import layers
    m = layers.CrossAttention(16, 2)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(m, (torch.zeros(1, 3, 16), torch.zeros(1, 4, 16)), check_trace=False)


@gpu
def test_other_routes_are_refused_on_the_device():
    refuses_forward_mode("cuda")
    refuses_tracing("cuda")
    for _, f, xs in calls("cuda"):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, tuple(xs), tuple(torch.ones_like(x) for x in xs))
        with pytest.raises(RuntimeError):
            torch.vmap(f)(*(torch.stack([x, x]) for x in xs))


@gpu
def test_a_backward_under_another_route_is_refused():
    """The gradient that arrives carries a tangent, or the backward runs while a trace is recorded."""
    for name, f, xs in calls("cuda"):
        leaves = [x.requires_grad_(True) for x in xs]
        out = f(*leaves)
        go = torch.ones_like(out)
        want = torch.autograd.grad(out, leaves, go, retain_graph=True)
        with fwAD.dual_level():
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(out, leaves, fwAD.make_dual(go, go), retain_graph=True)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda g: torch.autograd.grad(out, leaves, g, retain_graph=True))(go)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, go), want))
