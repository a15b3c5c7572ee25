"""ops.loss.distill_ce and top_logits on the GPU against 64-bit arithmetic
(tolerances: test_distill.check), and the dense layer, both of them and the
optimizer run together."""

import math

import pytest
import torch

from cerebro_ds_kpgi_amd.ops import backend
from cerebro_ds_kpgi_amd.ops import loss as L
from cerebro_ds_kpgi_amd.ops import nn as P
from test_distill import check, hits, inputs, reference, top_reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])


@pytest.fixture(autouse=True)
def _hip_backend():
    backend.set_backend("hip")
    backend.force_torch_ops([])
    yield


# rows of one element to rows of several slices, either side of every change of
# block size (256, 512, 1024, 2048, 4096, ... elements)
SIZES = [(1, 1, 1, 1), (2, 6, 2, 2), (3, 5, 7, 3), (16, 8, 257, 10), (2, 33, 1000, 20),
         (1, 4, 1025, 64), (1, 4, 2049, 100), (2, 3, 4099, 7), (1, 3, 8191, 200), (1, 3, 16390, 5),
         (1, 2, 40001, 1024), (2, 2, 65537, 64), (1, 3, 150001, 33)]


@pytest.mark.parametrize("unit", [True, False])
@DTYPES
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_sizes(size, dtype, unit):
    check(*size, dtype, unit, device=DEV)


@DTYPES
def test_many_rows(dtype):
    check(2, 3000, 10, 3, dtype, device=DEV)
    check(1, 70001, 4, 2, dtype, unit=False, device=DEV)


@pytest.mark.parametrize("unit", [True, False])
@pytest.mark.parametrize("N", [9, 1000, 5000, 70001, 140001])
@DTYPES
def test_masked_classes_and_extremes(dtype, N, unit):
    """Classes at the type's lowest value and at -inf, logits of +-1e4."""
    z, lab, val, idx, alpha, tau = inputs(2, 6, N, 3, dtype, ragged=False, device=DEV)
    zz = z.view(6, 2, N)
    zz[:, :, N // 2:N // 2 + N // 4] = torch.finfo(dtype).min
    zz[:, :, -(N // 4):] = -math.inf
    zz[2] *= 1000
    zz[3] = torch.finfo(dtype).min                # nothing but the lowest value
    lab.clamp_(max=N // 2 - 1)
    idx = idx % (N // 2)
    val[0, 0, 0] = -math.inf                      # an entry that is none
    val[1, 3] = -math.inf                         # a row of them
    check(2, 6, N, 3, dtype, unit, device=DEV, args=(z, lab, val, idx, alpha, tau))


@pytest.mark.parametrize("N", [50, 70001, 140001])
@DTYPES
def test_rows_without_terms_may_hold_anything(dtype, N):
    z, lab, val, idx, alpha, tau = inputs(1, 5, N, 4, dtype, ragged=False, device=DEV)
    z[1] = float("nan")
    z[3] = -math.inf
    lab[0, 1] = lab[0, 3] = -1
    idx[0, 1] = idx[0, 3] = -1
    for unit in (True, False):
        x = z.clone().requires_grad_(True)
        loss = L.distill_ce(x, lab, torch.zeros(1, 4, device=DEV), 1, val, idx, alpha, tau,
                            unit=unit)
        d, = torch.autograd.grad(loss, [x], torch.ones(1, device=DEV))
        assert torch.isfinite(loss).all() and torch.isfinite(d).all()
        assert not d[1].any() and not d[3].any()


@pytest.mark.parametrize("N", [50, 70001, 140001])
@DTYPES
def test_nan_and_bad_classes_reach_their_row_only(dtype, N):
    for what in ("nan", "label", "entry", "empty"):
        z, lab, val, idx, alpha, tau = inputs(1, 4, N, 4, dtype, ragged=False, device=DEV)
        if what == "nan":
            z[2, N - 1] = float("nan")
        elif what == "label":
            lab[0, 2] = N
        elif what == "entry":
            idx[0, 2, 3] = 2 ** 31 - 1
        else:
            z[2] = -math.inf
        for unit in (True, False):
            x = z.clone().requires_grad_(True)
            loss = L.distill_ce(x, lab, torch.zeros(1, 4, device=DEV), 1, val, idx, alpha, tau,
                                unit=unit)
            d, = torch.autograd.grad(loss, [x], torch.ones(1, device=DEV))
            assert torch.isnan(loss).all() and torch.isnan(d[2]).all(), what
            assert torch.isfinite(d[[0, 1, 3]]).all(), what


@DTYPES
def test_every_entry_the_same_class(dtype):
    """A class named K times gets the whole mass, the label among them."""
    z, lab, val, idx, alpha, tau = inputs(2, 4, 30, 9, dtype, ragged=False, device=DEV)
    idx[:] = 11
    lab[0] = 11
    check(2, 4, 30, 9, dtype, device=DEV, args=(z, lab, val, idx, alpha, tau))


@pytest.mark.parametrize("N", [30, 5000, 70001])
@DTYPES
def test_negative_and_zero_loss_gradients_and_tau_of_one(dtype, N):
    z, lab, val, idx, alpha, tau = inputs(3, 6, N, 5, dtype, device=DEV)
    tau = torch.tensor([1.0, 2.0, 1.0], device=DEV)
    dloss = torch.tensor([-2.0, 0.0, 0.7], device=DEV)
    x = z.clone().requires_grad_(True)
    loss = L.distill_ce(x, lab, torch.zeros(3, 4, device=DEV), 3, val, idx, alpha, tau)
    d, = torch.autograd.grad(loss, [x], dloss)
    _, _, want, mag = reference(z, lab, val, idx, alpha, tau, dloss)
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    tol = 2.0 ** -20 * 40 * mag
    tol = tol + half * (want.abs() + tol) + 1e-30
    assert ((d.double() - want).abs() <= tol).all()
    check(3, 6, N, 5, dtype, True, device=DEV, args=(z, lab, val, idx, alpha, tau))


@pytest.mark.parametrize("N", [70, 1000, 5003, 49999, 70001])
@DTYPES
def test_places_near_the_fifth(dtype, N):
    """Labels with 0 to 8 larger logits, gathered or spread, and up to 6 equal
    ones before and after the label: one row per configuration."""
    gen = torch.Generator().manual_seed(N)
    rows, labs = [], []
    for larger in (0, 1, 3, 4, 5, 8):
        for same in (0, 1, 2, 6):
            for near in (True, False):
                z = -1.0 - torch.rand(N, generator=gen)
                where = (torch.randperm(60, generator=gen) + torch.randint(0, N - 60, (1,), generator=gen)
                         if near else torch.randperm(N, generator=gen))
                z[where[:larger]] = 2.0 + torch.arange(larger)
                z[where[larger:larger + same + 1]] = 1.0
                rows.append(z)
                labs.append(where[larger])
    G = len(rows)
    z = torch.cat(rows)[None].to(dtype).to(DEV)
    lab = torch.stack(labs).int().view(G, 1).to(DEV)
    acc = torch.zeros(G, 4, device=DEV)
    idx = torch.zeros(G, 1, 1, dtype=torch.int32, device=DEV)
    val = torch.zeros(G, 1, 1, device=DEV)
    L.distill_ce(z.requires_grad_(True), lab, acc, G, val, idx, 0.5, 2.0, unit=True)
    first, fifth = hits(z.detach(), lab)
    assert torch.equal(acc[:, 1].long(), first) and torch.equal(acc[:, 2].long(), fifth)
    assert 0 < first.sum() < fifth.sum() < G


def test_alpha_of_zero_and_one():
    z, lab, val, idx, _, _ = inputs(3, 6, 40, 5, ragged=False, device=DEV)
    alpha = torch.tensor([0.0, 1.0, 0.5], device=DEV)
    tau = torch.tensor([2.0, 1.5, 1.0], device=DEV)
    idx0 = idx.clone()
    idx0[0] = 999                                  # alpha 0: not looked at
    z0 = z.clone()
    z0[:, 40 + 3] = -math.inf                      # config 1, alpha 1: its label is hopeless
    idx0[1] = torch.where(idx0[1] == 3, 4, idx0[1])
    lab[1] = 3
    check(3, 6, 40, 5, device=DEV, args=(z0, lab, val, idx0.clamp(max=39), alpha, tau))
    loss = L.distill_ce(z0, lab, torch.zeros(3, 4, device=DEV), 3, val, idx0, alpha, tau)
    assert torch.isfinite(loss).all()


@pytest.mark.parametrize("unit", [True, False])
@pytest.mark.parametrize("N", [50, 70001])
def test_weights_as_numbers(N, unit):
    z, lab, val, idx, _, _ = inputs(2, 3, N, 4, device=DEV)
    outs = []
    for a, t in ((0.25, 2.0), (torch.full((2,), 0.25, device=DEV), 2.0),
                 (0.25, torch.full((2,), 2.0, device=DEV))):
        x = z.clone().requires_grad_(True)
        loss = L.distill_ce(x, lab, torch.zeros(2, 4, device=DEV), 2, val, idx, a, t, unit=unit)
        outs.append((loss.detach(), torch.autograd.grad(loss, [x], torch.ones(2, device=DEV))[0]))
    assert all(torch.equal(p, q) for o in outs[1:] for p, q in zip(o, outs[0]))


def test_layouts_and_mixed_types():
    """Pitched logits, a shared teacher, fp32 values beside bf16 logits and the
    other way round, strided entries."""
    z, lab, val, idx, alpha, tau = inputs(2, 5, 37, 6, ragged=False, device=DEV)
    big = torch.zeros(5, 2 * 37 + 3, device=DEV)
    big[:, 1:75] = z

    def one(z, val, idx):
        x = z.detach().requires_grad_(True)
        acc = torch.zeros(2, 4, device=DEV)
        loss = L.distill_ce(x, lab, acc, 2, val, idx, alpha, tau, unit=True)
        d, = torch.autograd.grad(loss, [x], torch.ones(2, device=DEV))
        return loss.detach(), d, acc
    want = one(z, val, idx)
    # rows that start elsewhere in a 16-byte vector are summed in another order:
    # the same tolerance as any result, not the same bits
    check(2, 5, 37, 6, device=DEV, args=(big[:, 1:75], lab, val, idx, alpha, tau))
    for got in (one(z.t().contiguous().t(), val, idx),
                one(z, val.transpose(0, 1).contiguous().transpose(0, 1),
                    idx.permute(2, 0, 1).contiguous().permute(1, 2, 0))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    shared = one(z, val[0], idx[0])
    full = one(z, val[:1].repeat(2, 1, 1), idx[:1].repeat(2, 1, 1))
    assert all(torch.equal(a, b) for a, b in zip(shared, full))
    vb = val.bfloat16()
    assert all(torch.equal(a, b) for a, b in zip(one(z, vb, idx), one(z, vb.float(), idx)))
    zb = z.bfloat16()
    assert all(torch.equal(a, b) for a, b in zip(one(zb, vb, idx), one(zb, vb.float(), idx)))
    with torch.no_grad():
        assert not L.distill_ce(z.requires_grad_(True), lab, want[2], 2, val, idx).requires_grad


@DTYPES
def test_no_teacher_entries_at_all(dtype):
    """K = 0: the hard term alone, its metrics as softmax_ce counts them."""
    for N in (11, 70001):
        check(2, 4, N, 0, dtype, device=DEV)
    z, lab, val, idx, _, _ = inputs(2, 6, 40, 0, torch.float32, ragged=False, device=DEV)
    a1, a2 = torch.zeros(2, 4, device=DEV), torch.zeros(2, 4, device=DEV)
    one = L.distill_ce(z, lab, a1, 2, val, idx, alpha=0.0)
    two = L.softmax_ce(z, lab, a2, 2)
    # both sum six rows' lse - z_y of size below 20 in fp32
    assert (one - two).abs().max() <= 20 * 2.0 ** -20
    assert torch.equal(a1[:, 1:], a2[:, 1:])


@pytest.mark.parametrize("unit", [True, False])
def test_backward_twice_and_second_derivatives(unit):
    z, lab, val, idx, alpha, tau = inputs(1, 3, 20, 4, device=DEV)
    z.requires_grad_(True)

    def loss():
        return L.distill_ce(z, lab, torch.zeros(1, 4, device=DEV), 1, val, idx, alpha, tau,
                            unit=unit)
    y = loss()
    y.sum().backward(retain_graph=True)
    first = z.grad.clone()
    y.sum().backward()
    assert torch.equal(z.grad, first + first)
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(loss().sum(), [z], create_graph=True)


def test_gradient_against_differences():
    z, lab, val, idx, alpha, tau = inputs(2, 3, 12, 4, device=DEV, scale=1.0)

    def f(x):
        return L.distill_ce(x, lab, torch.zeros(2, 4, device=DEV), 2, val, idx, alpha, tau)
    x = z.clone().requires_grad_(True)
    d, = torch.autograd.grad(f(x).sum(), [x])
    v = torch.randn_like(z)
    h = 2.0 ** -5
    num = (f(z + h * v).double().sum() - f(z - h * v).double().sum()) / (2 * h)
    # third directional derivative of a log-sum-exp: below 2 (max |v|)^3 a term,
    # weights below 1 + tau^2; rounding 2^-20 of losses below 40
    bound = h * h / 6 * 2 * float(v.abs().max()) ** 3 * 10 * 2 + 2 * 40 * 2.0 ** -20 / h
    assert abs(float(num) - float((d.double() * v.double()).sum())) <= bound


@pytest.mark.parametrize("N", [1000, 70001])
def test_repeats_and_replays(N):
    """Bitwise equal passes; two captured graphs replayed in turn with other
    inputs between eager passes and synchronisations."""
    z, lab, val, idx, alpha, tau = inputs(2, 5, N, 9, device=DEV)
    x = z.clone().requires_grad_(True)

    def step(unit):
        acc = torch.zeros(2, 4, device=DEV)
        loss = L.distill_ce(x, lab, acc, 2, val, idx, alpha, tau, unit=unit)
        d, = torch.autograd.grad(loss, [x], ones)
        return loss.detach(), d, acc
    ones = torch.ones(2, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a, b = step(True), step(False)
        a2 = step(True)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(a, a2))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs = []
    for unit in (True, False):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(unit)
        graphs.append((g, out))
    for it in range(4):
        with torch.no_grad():
            x.copy_(torch.randn_like(x) * 3)
        g, out = graphs[it % 2]
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, step(it % 2 == 0))), it


# ---------------------------------------------------------------------------
def top_check(z, G, k):
    v, i = L.top_logits(z, G, k)
    vr, ir = top_reference(z, G, k)
    assert v.dtype == z.dtype and i.dtype == torch.int32
    assert torch.equal(i.cpu(), ir)
    as_int = torch.int32 if z.dtype == torch.float32 else torch.int16
    assert torch.equal(v.cpu().contiguous().view(as_int), vr.contiguous().view(as_int))


TOP_SIZES = [(1, 1, 1, 1), (2, 3, 2, 2), (3, 5, 7, 3), (2, 4, 255, 255), (8, 32, 1000, 10),
             (1, 3, 1000, 1000), (1, 4, 2049, 64), (1, 2, 4097, 1024), (1, 3, 8193, 5),
             (2, 2, 16385, 200), (1, 130, 20000, 3), (1, 2, 40001, 1024), (1, 130, 33000, 300),
             (1, 3, 131071, 200), (1, 2, 300007, 1024), (1, 1, 1000003, 1024), (1, 129, 70001, 100)]


@DTYPES
@pytest.mark.parametrize("size", TOP_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_top_sizes(size, dtype):
    G, B, N, k = size
    gen = torch.Generator(device=DEV).manual_seed(N)
    top_check((torch.randn(B, G * N, generator=gen, device=DEV) * 3).to(dtype), G, k)


@DTYPES
@pytest.mark.parametrize("N", [64, 1000, 3000, 5000, 40000, 140000])
@pytest.mark.parametrize("k", [1, 10, 64])
def test_top_of_awkward_rows(N, k, dtype):
    """Rows that defeat a filter: constants, two values, sorted, all of -inf,
    signed zeros, NaN, the type's lowest value."""
    rows = []
    rows.append(torch.full((N,), 1.5))
    rows.append((torch.arange(N) % 2).float())
    rows.append(torch.arange(N).float() / N)
    rows.append(-torch.arange(N).float() / N)
    rows.append(torch.full((N,), -math.inf))
    rows.append(torch.zeros(N) * torch.where(torch.arange(N) % 3 == 0, -1.0, 1.0))
    r = torch.randn(N, generator=torch.Generator().manual_seed(N))
    r[[0, N // 2, N - 1]] = float("nan")
    r[N // 3] = -float("nan")
    rows.append(r)
    rows.append(torch.full((N,), float("nan")))
    r = torch.full((N,), torch.finfo(dtype).min)
    r[N // 2] = math.inf
    rows.append(r)
    r = torch.randn(N, generator=torch.Generator().manual_seed(1))
    r[N // 2:N // 2 + 32] += 1000                 # the largest side by side
    rows.append(r)
    r = torch.full((N,), -math.inf)
    r[N - 3:] = -1.0
    rows.append(r)
    top_check(torch.stack(rows).to(dtype).to(DEV), 1, k)


def test_top_of_pitched_rows_and_large_k_ties():
    big = torch.randn(6, 2 * 501 + 9, device=DEV)
    top_check(big[:, 4:4 + 1002], 2, 30)
    v, i = L.top_logits(big[:, 4:4 + 1002], 2, 30)
    v2, i2 = L.top_logits(big[:, 4:4 + 1002].t().contiguous().t(), 2, 30)
    assert torch.equal(v, v2) and torch.equal(i, i2)
    # a few distinct values and k in the hundreds: ties cross the last place
    z = (torch.randn(3, 50000, device=DEV) * 2).round()
    for k in (700, 1024):
        top_check(z, 1, k)


def test_top_replays():
    z = torch.randn(3, 40000, device=DEV)
    L.top_logits(z, 1, 50)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        v, i = L.top_logits(z, 1, 50)
    for _ in range(3):
        z.copy_(torch.randn(3, 40000, device=DEV))
        g.replay()
        torch.cuda.synchronize()
        got = v.clone(), i.clone()
        want = L.top_logits(z, 1, 50)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
def _mlp(G, dims, dtype, seed):
    from cerebro_ds_kpgi_amd.runtime.arena import Arena, ModelLayout, ParamRef, ParamSpec
    specs = []
    for n, (k, o) in enumerate(zip(dims[:-1], dims[1:])):
        specs += [ParamSpec("l%d/kernel" % n, (o, k), "weight"), ParamSpec("l%d/bias" % n, (o,),
                                                                           "bias")]
    arena = Arena(ModelLayout(specs), G, DEV, dtype)
    for g in range(G):
        arena.init_model(g, seed + g)
        arena.set_hparams(g, 1e-2, 0.0)
    return arena, [ParamRef(arena, s) for s in specs]


@DTYPES
def test_teacher_to_student_step(dtype):
    """A step as it is used: a teacher's top logits, a student of residual
    blocks, the loss, its backward and the optimizer -- captured and replayed
    against eager steps from the same state, and the first step's weight
    gradients against 64-bit differentiation of the whole student."""
    from cerebro_ds_kpgi_amd.ops.optim import adam_step
    G, B, D, N, K = 2, 24, 40, 50, 6
    tar, tref = _mlp(1, (D, 64, N), dtype, 7)
    sar, sref = _mlp(G, (D, D, D, N), dtype, 3)
    x = torch.randn(B, D, device=DEV).to(dtype)
    lab = torch.randint(0, N, (G, B), device=DEV, dtype=torch.int32)
    alpha, tau = torch.tensor([0.3, 0.8], device=DEV), torch.tensor([1.0, 2.0], device=DEV)
    anchor = torch.zeros((), device=DEV, requires_grad=True)
    acc = torch.zeros(G, 4, device=DEV)

    def forward():
        with torch.no_grad():
            t = P.linear_act(P.linear_act(x, *tref[:2], "gelu"), *tref[2:])
            val, idx = L.top_logits(t, 1, K)
        h = x.repeat(1, G)
        h = P.linear_act(h, *sref[:2], "silu", h, anchor=anchor)
        h = P.linear_act(h, *sref[2:4], "gelu", h)
        z = P.linear_act(h, *sref[4:])
        return L.distill_ce(z, lab, acc, G, val[0], idx[0], alpha, tau, unit=True), val, idx

    def step():
        loss, val, idx = forward()
        torch.autograd.backward(loss, torch.ones(G, device=DEV))
        out = loss.detach().clone()
        adam_step(sar)
        return out

    # gradients of the whole student
    loss, val, idx = forward()
    torch.autograd.backward(loss, torch.ones(G, device=DEV))
    del loss
    F = torch.nn.functional
    for g in range(G):
        w = [r.work()[g].double().requires_grad_(True) for r in sref]
        h = x.double()
        h = h + F.silu(F.linear(h, w[0], w[1]))
        h = h + F.gelu(F.linear(h, w[2], w[3]))
        z = F.linear(h, w[4], w[5])
        a, t = float(alpha[g]), float(tau[g])
        p = torch.softmax(val[0].double() / t, 1)
        kl = (p * (torch.log(p) - torch.log_softmax(z / t, 1).gather(1, idx[0].long()))).sum(1)
        ce = F.cross_entropy(z, lab[g].long(), reduction="none")
        ref = ((1 - a) * ce + a * t * t * kl).mean()
        grads = torch.autograd.grad(ref, w)
        for r, want in zip(sref, grads):
            # norms: two-plane products (fp32) or three roundings of the
            # activations and four of the gradients on the way (bf16)
            rel = float((r.grad()[g].double() - want).norm() / want.norm())
            assert rel < (2.0 ** -14 if dtype == torch.float32 else 8 * 2.0 ** -8), (r.spec.name,
                                                                                     rel)
    # captured against eager, from the same state
    state = sar.state.clone()

    def restore():
        sar.state.copy_(state)
        sar.sync_work()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    restore()
    eager = [step() for _ in range(4)]
    after = sar.state.clone()
    restore()
    for want in eager:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(sar.state, after)


def test_more_than_two_to_the_31_elements():
    """17 000 rows of 131 072 classes (2.2e9 logits): loss, gradient and top
    logits of the last rows."""
    B, N, K = 17_000, 131_072, 8
    gen = torch.Generator(device=DEV).manual_seed(0)
    z = torch.empty(B, N, dtype=torch.bfloat16, device=DEV)
    for i in range(0, B, 1000):
        z[i:i + 1000] = (torch.randn(1000, N, generator=gen, device=DEV) * 3).bfloat16()
    val, idx = L.top_logits(z, 1, K)
    tail = slice(B - 40, B)
    vr, ir = top_reference(z[tail], 1, K)
    assert torch.equal(idx[:, tail].cpu(), ir) and torch.equal(val[:, tail].cpu(), vr)
    lab = torch.randint(0, N, (1, B), generator=gen, device=DEV, dtype=torch.int32)
    alpha, tau = torch.tensor([0.4], device=DEV), torch.tensor([2.0], device=DEV)
    z.requires_grad_(True)
    grads = []
    for unit in (True, False):
        loss = L.distill_ce(z, lab, torch.zeros(1, 4, device=DEV), 1, val, idx, alpha, tau, unit=unit)
        grads.append(torch.autograd.grad(loss, [z], torch.ones(1, device=DEV))[0])
        del loss
    assert torch.equal(grads[0], grads[1])
    one = torch.ones(1, device=DEV)
    _, _, d, dm = reference(z.detach()[tail], lab[:, tail], val[:, tail], idx[:, tail], alpha, tau, one)
    d, dm = d * 40 / B, dm * 40 / B
    tol = 2.0 ** -20 * 40 * dm
    assert ((grads[0][tail].double() - d).abs() <= tol + 2.0 ** -8 * (d.abs() + tol) + 1e-30).all()


def test_inputs_written_before_the_backward_are_refused():
    """The general gradient reads labels, entries and weights again; the unit
    gradient is finished in the forward."""
    for name in ("logits", "labels", "top_val", "top_idx", "alpha", "tau", None):
        for unit in (False, True):
            z, lab, val, idx, alpha, tau = inputs(2, 6, 30, 4, device=DEV)
            x = z.clone().requires_grad_(True)
            h = x * 1.0
            t = {"logits": h, "labels": lab, "top_val": val, "top_idx": idx, "alpha": alpha,
                 "tau": tau}
            loss = L.distill_ce(h, lab, torch.zeros(2, 4, device=DEV), 2, val, idx, alpha, tau,
                                unit=unit)
            if name is not None:
                t[name].mul_(1)                         # a write, whatever it writes
            if name is None or unit:
                d, = torch.autograd.grad(loss, [x], torch.ones(2, device=DEV))
                assert torch.isfinite(d).all()
            else:
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    torch.autograd.grad(loss, [x], torch.ones(2, device=DEV))


def test_teacher_made_in_inference_mode():
    """Such tensors count no writes: the gradient is of the values at the call."""
    z, lab, val, idx, alpha, tau = inputs(2, 6, 30, 4, device=DEV)
    with torch.inference_mode():
        ival, iidx, ialpha = val.clone(), idx.clone(), alpha.clone()
    grads = []
    for v, i, a in ((val, idx, alpha), (ival, iidx, ialpha)):
        x = z.clone().requires_grad_(True)
        loss = L.distill_ce(x, lab, torch.zeros(2, 4, device=DEV), 2, v, i, a, tau)
        if v is ival:
            with torch.inference_mode():
                ival.zero_()
                iidx.zero_()
                ialpha.zero_()
        grads.append(torch.autograd.grad(loss, [x], torch.ones(2, device=DEV))[0])
    assert torch.equal(*grads)


@pytest.mark.parametrize("unit", [True, False])
def test_gradients_of_a_kept_graph_are_the_callers(unit):
    z, lab, val, idx, alpha, tau = inputs(2, 6, 30, 4, device=DEV)
    x = z.clone().requires_grad_(True)
    ones = torch.ones(2, device=DEV)
    loss = L.distill_ce(x, lab, torch.zeros(2, 4, device=DEV), 2, val, idx, alpha, tau, unit=unit)
    first, = torch.autograd.grad(loss, [x], ones, retain_graph=True)
    want = first.clone()
    first.mul_(100.0)                            # a caller that scales or clips in place
    second, = torch.autograd.grad(loss, [x], ones, retain_graph=True)
    assert torch.equal(second, want)
    loss.backward(ones, retain_graph=True)
    x.grad.zero_()
    third, = torch.autograd.grad(loss, [x], ones)
    assert torch.equal(third, want)


def test_tracers_and_dual_numbers_are_refused():
    """Neither can see into the kernels: a trace would hold empty outputs, a dual
    number would come back without its tangent."""
    from test_linear_act import make
    from torch.autograd import forward_ad
    arena, w, b = make(device=DEV)
    z, lab, val, idx, alpha, tau = inputs(2, 4, 6, 3, device=DEV)
    x = torch.randn(4, 10, device=DEV)

    def loss(z):
        return L.distill_ce(z, lab, torch.zeros(2, 4, device=DEV), 2, val, idx, alpha, tau)
    for f, t in ((lambda x: P.linear_act(x, w, b, "silu"), x), (loss, z),
                 (lambda z: L.top_logits(z, 2, 2), z)):
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            torch.jit.trace(f, (t,))
    with forward_ad.dual_level():
        for f, t in ((lambda x: P.linear_act(x, w, b, "silu"), x), (loss, z),
                     (lambda r: P.linear_act(x, w, b, "silu", r), torch.randn(4, 6, device=DEV))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(forward_ad.make_dual(t, torch.ones_like(t)))
        # a teacher's logits have no derivative to lose
        L.top_logits(forward_ad.make_dual(z, torch.ones_like(z)), 2, 2)


def test_a_single_row_of_any_pitch():
    from test_distill import one_row_layouts
    z, lab, val, idx, alpha, tau = inputs(2, 1, 60, 4, device=DEV)

    def run(x):
        x = x.detach().requires_grad_(True)
        acc = torch.zeros(2, 4, device=DEV)
        loss = L.distill_ce(x, lab, acc, 2, val, idx, alpha, tau)
        return [loss.detach(), acc, torch.autograd.grad(loss.sum(), [x])[0], *L.top_logits(x, 2, 7)]
    want = run(z)
    for x in one_row_layouts(z):
        assert all(torch.equal(a, b) for a, b in zip(run(x), want))


@pytest.mark.parametrize("unit", [True, False])
@pytest.mark.parametrize("B", [1, 6])
def test_hooks_and_checkpoints_see_what_is_saved(B, unit):
    from torch.autograd.graph import saved_tensors_hooks
    from torch.utils.checkpoint import checkpoint
    z, lab, val, idx, alpha, tau = inputs(2, B, 30, 4, device=DEV)
    x = z.clone().requires_grad_(True)
    ones = torch.ones(2, device=DEV)

    def loss(x):
        return L.distill_ce(x, lab, torch.zeros(2, 4, device=DEV), 2, val, idx[:1].expand(2, -1, -1),
                            alpha, tau, unit=unit)
    want, = torch.autograd.grad(loss(x), [x], ones)
    packed = []

    def pack(t):
        packed.append(tuple(t.shape))
        return t.cpu()

    def unpack(t):
        return t.to(DEV) if t.dim() < 2 else t.transpose(-1, -2).contiguous().to(DEV).transpose(-1, -2)
    with saved_tensors_hooks(pack, unpack):
        y = loss(x)
    assert (B, 60) in packed
    assert unit or (2, B, 4) in packed and (2, B) in packed and (2,) in packed
    assert torch.equal(torch.autograd.grad(y, [x], ones)[0], want)
    y = checkpoint(loss, x, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(y, [x], ones)[0], want)


@pytest.mark.parametrize("N", [1000, 70001, 140001])
@DTYPES
def test_lowest_values_beside_a_huge_one(dtype, N):
    """The type's lowest value below a maximum of 1e37: their difference is beyond
    fp32, the probability zero all the same -- also of a slice of nothing else."""
    z = torch.full((2, N), torch.finfo(dtype).min, dtype=dtype, device=DEV)
    z[:, 5] = 1e37
    lab = torch.full((1, 2), 5, dtype=torch.int32, device=DEV)
    idx = torch.full((1, 2, 1), 5, dtype=torch.int32, device=DEV)
    val = torch.zeros(1, 2, 1, device=DEV)
    for unit in (True, False):
        for tau in (1.0, 2.0):
            x = z.clone().requires_grad_(True)
            loss = L.distill_ce(x, lab, torch.zeros(1, 4, device=DEV), 1, val, idx, 0.5, tau, unit=unit)
            d, = torch.autograd.grad(loss, [x], torch.ones(1, device=DEV))
            assert float(loss) == 0 and not d.any()


@pytest.mark.parametrize("unit", [True, False])
@pytest.mark.parametrize("B,N", [(8192, 1000), (512, 40000), (64, 70001)])
def test_fp32_gradient_is_as_near_as_its_exponentials(B, N, unit):
    """Logits in [-1, 0]: a term's exponent is off by two roundings (2^-24 |x|
    each, |x| <= 1), its exponential and its sum by 2^-23 each, quotient, product
    and sum by 2^-24 each.  Independent and uniform, their squares add up to
    (2/3 + 4 + 4 + 3) / 3 2^-48: a norm of 1.97 2^-24, below 2^-23."""
    gen = torch.Generator(device=DEV).manual_seed(N)
    z = -torch.rand(B, N, generator=gen, device=DEV)
    z[:, 7] = 0.0
    lab = torch.randint(0, N, (1, B), generator=gen, device=DEV, dtype=torch.int32)
    idx = torch.randint(0, N, (1, B, 4), generator=gen, device=DEV, dtype=torch.int32)
    val = torch.randn(1, B, 4, generator=gen, device=DEV)
    alpha, tau = torch.tensor([0.4], device=DEV), torch.tensor([2.0], device=DEV)
    x = z.clone().requires_grad_(True)
    one = torch.ones(1, device=DEV)
    loss = L.distill_ce(x, lab, torch.zeros(1, 4, device=DEV), 1, val, idx, alpha, tau, unit=unit)
    d, = torch.autograd.grad(loss, [x], one)
    _, _, want, _ = reference(z, lab, val, idx, alpha, tau, one)
    # the named classes, near -c whatever the softmax, are left out
    rest = torch.ones_like(z, dtype=torch.bool)
    rest.scatter_(1, lab[0].long()[:, None], False).scatter_(1, idx[0].long(), False)
    err = (d.double() - want)[rest]
    assert float(err.norm() / want[rest].norm()) <= 2.0 ** -23


def test_hooks_that_give_back_something_else_are_refused():
    from torch.autograd.graph import saved_tensors_hooks
    z, lab, val, idx, alpha, tau = inputs(2, 6, 30, 4, device=DEV)
    x = z.clone().requires_grad_(True)
    for unit, shapes in ((True, [(6, 60)]), (False, [(6, 60), (2, 6), (2, 6, 4), (2,), (48,)])):
        for wrong in (lambda t: t.double(), lambda t: t.cpu(), lambda t: t[:1], lambda t: t[None]):
            for shape in shapes:
                with saved_tensors_hooks(lambda t: t, lambda t: wrong(t) if t.shape == shape else t):
                    loss = L.distill_ce(x, lab, torch.zeros(2, 4, device=DEV), 2, val, idx, alpha, tau,
                                        unit=unit)
                with pytest.raises(RuntimeError, match="a hook on saved tensors"):
                    torch.autograd.grad(loss, [x], torch.ones(2, device=DEV))
