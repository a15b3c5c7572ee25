"""Refusals and the CPU path of ops.nn.linear_act (no GPU)."""

import math

import pytest
import torch

from cerebro_ds_kpgi_amd.ops import nn as P
from cerebro_ds_kpgi_amd.runtime.arena import Arena, ModelLayout, ParamRef, ParamSpec

F = torch.nn.functional
ACT64 = {"none": lambda z: z, "relu": F.relu, "relu6": F.relu6, "gelu": F.gelu,
         "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}


def make(G=2, N=3, K=5, dtype=torch.float32, bias=True, trainable=True, device="cpu"):
    specs = [ParamSpec("d/kernel", (N, K), "weight")]
    if bias:
        specs.append(ParamSpec("d/bias", (N,), "bias"))
    arena = Arena(ModelLayout(specs), G, device, dtype, trainable=trainable)
    refs = [ParamRef(arena, s) for s in specs]
    gen = torch.Generator().manual_seed(N * 1000 + K)
    refs[0].master().copy_((torch.randn(G, N, K, generator=gen) / math.sqrt(K)).to(dtype))
    if bias:
        refs[1].master().copy_(torch.randn(G, N, generator=gen).to(dtype))
    arena.sync_work()
    return arena, refs[0], refs[1] if bias else None


@pytest.mark.parametrize("act", sorted(ACT64))
@pytest.mark.parametrize("residual", [False, True])
def test_cpu_path_matches_64_bits(act, residual):
    G, M, N, K = 2, 4, 3, 5
    arena, w, b = make(G, N, K)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, M // 2, G * K, generator=gen, requires_grad=True)
    r = torch.randn(2, M // 2, G * N, generator=gen, requires_grad=True) if residual else None
    dy = torch.randn(2, M // 2, G * N, generator=gen)
    y = P.linear_act(x, w, b, act, r)
    y.backward(dy)
    x64 = x.detach().double().requires_grad_(True)
    w64 = w.work().double().requires_grad_(True)
    b64 = b.work().double().requires_grad_(True)
    z = torch.stack([F.linear(x64.view(M, G, K)[:, g], w64[g], b64[g]) for g in range(G)], 1)
    y64 = ACT64[act](z).reshape(x.shape[:-1] + (G * N,))
    if residual:
        y64 = y64 + r.detach().double()
    y64.backward(dy.double())
    # sums of K = 5 and N = 3 terms of size ~1 in fp32
    kw = dict(rtol=16 * 2 ** -24, atol=64 * 2 ** -24)
    torch.testing.assert_close(y.detach().double(), y64.detach(), **kw)
    torch.testing.assert_close(x.grad.double(), x64.grad, **kw)
    torch.testing.assert_close(w.grad().double(), w64.grad, **kw)
    torch.testing.assert_close(b.grad().double(), b64.grad, **kw)
    if residual:
        assert torch.equal(r.grad, dy)


def test_cpu_bf16_and_empty():
    arena, w, b = make(dtype=torch.bfloat16)
    x = torch.randn(4, 10).bfloat16().requires_grad_(True)
    y = P.linear_act(x, w, b, "silu")
    assert y.dtype == torch.bfloat16 and y.shape == (4, 6)
    y.sum().backward()
    assert x.grad.dtype == torch.bfloat16 and w.grad().abs().sum() > 0
    e = torch.zeros(0, 10, dtype=torch.bfloat16, requires_grad=True)
    P.linear_act(e, w, b, "silu").sum().backward()
    assert not w.grad().any() and not b.grad().any() and e.grad.shape == (0, 10)


def test_refusals():
    arena, w, b = make()
    x = torch.zeros(4, 10)
    with pytest.raises(ValueError, match="not one of"):
        P.linear_act(x, w, b, "tanh")
    with pytest.raises(ValueError, match="G\\*K"):
        P.linear_act(torch.zeros(4, 9), w, b)
    with pytest.raises(TypeError, match="computes in"):
        P.linear_act(x.bfloat16(), w, b)
    with pytest.raises(TypeError, match="computes in"):
        P.linear_act(x.half(), w, b)
    with pytest.raises(ValueError, match="residual"):
        P.linear_act(x, w, b, "none", torch.zeros(3, 6))
    with pytest.raises(ValueError, match="residual"):
        P.linear_act(x, w, b, "none", torch.zeros(1, 6))
    with pytest.raises(TypeError, match="residual"):
        P.linear_act(x, w, b, "none", torch.zeros(4, 6).double())
    with pytest.raises(ValueError, match="bias"):
        P.linear_act(x, w, make()[2])
    with pytest.raises(ValueError, match="bias"):
        P.linear_act(x, w, w)
    with pytest.raises(ValueError, match="\\[N, K\\]"):
        P.linear_act(x, b)
    hl = x.clone()
    hl._cer_hl = True
    with pytest.raises(ValueError, match="HL"):
        P.linear_act(hl, w, b)
    _, w2, b2 = make(trainable=False)
    with pytest.raises(ValueError, match="no gradients"):
        P.linear_act(x.clone().requires_grad_(True), w2, b2)
    with torch.no_grad():
        assert P.linear_act(x, w2, b2).shape == (4, 6)
    _, w3, b3 = make(dtype=torch.bfloat16, trainable=False)
    with pytest.raises(ValueError, match="parks"):
        P.linear_act(x.bfloat16(), w3, b3)


def test_kernels_refuse_tracers_and_dual_numbers():
    """At the door of the compiled calls, before anything is looked at."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from cerebro_ds_kpgi_amd.ops import _hip
    arena, w, b = make()
    n = _hip.nodes()
    i32 = torch.int32

    def linear(x, r=None):
        return n.linear_act(x, None, r, arena.work, arena.grad, w.spec.offset, b.spec.offset, 3, 5,
                            0, False)

    def distill(z, val=torch.zeros(2, 4, 1), tau=torch.ones(2)):
        return n.distill_ce(z, torch.zeros(2, 4, dtype=i32), torch.zeros(2, 4), 2, val,
                            torch.zeros(2, 4, 1, dtype=i32), None, 0.5, tau, 0.0, False, False)

    def top(z):
        return n.top_logits(z, 2, 1)
    x, r = torch.randn(4, 10), torch.randn(4, 6)
    for f, t in ((lambda t: linear(t), x), (lambda t: distill(t), r), (lambda t: top(t), r)):
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            torch.jit.trace(f, (t,))
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            make_fx(f)(t)
    with torch.autograd.forward_ad.dual_level():
        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        for f in (lambda: linear(dual(x)), lambda: linear(x, dual(r)), lambda: distill(dual(r)),
                  lambda: distill(r, dual(torch.zeros(2, 4, 1))),
                  lambda: distill(r, tau=dual(torch.ones(2)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()


def test_rows_beyond_the_kernels_integers_are_refused():
    """Row numbers are ints, with room for the last tile and the last range of
    rows; a launch has fewer than 2^32 threads."""
    import ctypes
    from cerebro_ds_kpgi_amd.ops import _hip
    ws = _hip.lib().cer_dense_ws
    ws.restype = ctypes.c_int64
    for bf16 in (0, 1):
        for act in (0, 1, 7):
            for kind in (0, 1):
                assert ws(kind, 2 ** 29 + 3, 1, 1, 1, bf16, act) >= 0
                assert ws(kind, 2 ** 31 - 2 ** 21, 4, 1, 1, bf16, act) >= 0
                for M in (2 ** 31 - 2 ** 20, 2 ** 31 - 1):
                    assert ws(kind, M, 1, 1, 1, bf16, act) == -1
            # 2^31 x 2^21 outputs: no tile covers them in one launch
            assert ws(0, 2 ** 31 - 2 ** 21, 2 ** 21, 1, 1, bf16, act) == -1
    arena, w, b = make(1, 1, 1)
    for M in (2 ** 31 - 1, 2 ** 31 + 5):
        with pytest.raises(ValueError, match="32-bit|2\\^31"):
            _hip.nodes().linear_act(torch.zeros(1, 1).expand(M, 1), None, None, arena.work,
                                    arena.grad, w.spec.offset, b.spec.offset, 1, 1, 0, False)


def test_no_second_derivative_on_the_cpu():
    """The weights are no leaves, so a second derivative would lack their part."""
    arena, w, b = make()
    x = torch.randn(4, 10, requires_grad=True)
    y = P.linear_act(x, w, b, "silu")
    with pytest.raises(RuntimeError, match="second derivative"):
        d, = torch.autograd.grad((y * y).sum(), [x], create_graph=True)
        torch.autograd.grad(d.sum(), [x])


def test_statistics_and_parameters_of_other_layouts_are_refused():
    """A running mean lies behind the parameters, where the gradients have
    nothing: its gradient would be written past their end."""
    from cerebro_ds_kpgi_amd.ops import _hip
    spec = [ParamSpec("d/kernel", (3, 5), "weight"), ParamSpec("bn/mean", (3,), "running_mean")]
    arena = Arena(ModelLayout(spec), 2, "cpu", torch.float32)
    big = ModelLayout([ParamSpec("a", (300, 5), "weight"), ParamSpec("b", (3,), "bias")]).specs[1]
    w = ParamRef(arena, spec[0])
    x = torch.randn(4, 10)
    for other in (spec[1], big):
        with pytest.raises(ValueError, match="no trainable parameter"):
            _hip.nodes().linear_act(x, None, None, arena.work, arena.grad, spec[0].offset,
                                    other.offset, 3, 5, 0, True)
        with pytest.raises((ValueError, RuntimeError)):
            P.linear_act(x, w, ParamRef(arena, other))
