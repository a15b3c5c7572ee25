"""ops.loss.distill_ce and top_logits: the CPU path against 64-bit arithmetic,
and the refusals (no GPU)."""

import math

import pytest
import torch

from cerebro_ds_kpgi_amd.ops import loss as L


def inputs(G, B, N, K, dtype=torch.float32, ragged=True, device="cpu", seed=0, scale=3.0):
    gen = torch.Generator(device=device).manual_seed(seed + N)
    z = (torch.randn(B, G * N, generator=gen, device=device) * scale).to(dtype)
    idx = torch.stack([torch.randperm(N, generator=gen, device=device)[:K]
                       for _ in range(min(G * B, 64))])
    idx = idx.repeat(-(-G * B // len(idx)), 1)[:G * B].view(G, B, K).to(torch.int32)
    val = (torch.randn(G, B, K, generator=gen, device=device) * scale).to(dtype)
    lab = torch.randint(0, N, (G, B), generator=gen, device=device, dtype=torch.int32)
    if ragged:
        drop = torch.rand(G, B, K, generator=gen, device=device) < 0.3
        idx = torch.where(drop, torch.full_like(idx, -1), idx)
        row = torch.arange(G * B, device=device).view(G, B)
        idx[row % 5 == 4] = -1                      # no entry
        lab[row % 3 == 2] = -1                      # no label
        if B > 2 and K > 1:
            idx[0, 0, 1] = idx[0, 0, 0]             # the same class twice
            lab[0, 1] = max(int(idx[0, 1, 0]), 0)   # the label is the teacher's choice
    alpha = torch.linspace(0.2, 0.9, G, device=device)
    tau = torch.linspace(1.0, 3.0, G, device=device)
    return z, lab, val, idx, alpha, tau


def reference(z, lab, val, idx, alpha, tau, dloss):
    """Row losses, their magnitude, and the gradient with the magnitude of its
    terms, from the definition in 64 bits, config by config."""
    G, B = lab.shape
    N = z.shape[1] // G
    rows, mags, grads, gmags = [], [], [], []
    for g in range(G):
        zg = z[:, g * N:(g + 1) * N].double()
        a, t = float(alpha[g].double()), float(tau[g].double())
        row = torch.zeros(B, dtype=torch.float64, device=z.device)
        mag, d, dm = row.clone(), torch.zeros_like(zg), torch.zeros_like(zg)
        y = lab[g].long()
        has = (y >= 0).nonzero().squeeze(1)
        if a != 1:
            p1 = torch.softmax(zg, 1)
            lse = torch.logsumexp(zg, 1)
            zy = zg[has, y[has]]
            row[has] += (1 - a) * (lse[has] - zy)
            mag[has] += (1 - a) * (lse[has].abs() + zy.abs())
            d[has] += (1 - a) * p1[has]
            dm[has] += (1 - a) * p1[has]
            d[has, y[has]] -= 1 - a
            dm[has, y[has]] += 1 - a
        if a != 0 and idx.shape[2]:
            i = idx[g].long()
            th = (i >= 0) & (val[g] != -math.inf)
            hv = th.any(1).nonzero().squeeze(1)
            if len(hv):
                v = (val[g].double() / t).masked_fill(~th, -math.inf)[hv]
                p = torch.softmax(v, 1)
                logp = torch.log_softmax(v, 1)
                zq = zg[hv] / t
                lq = torch.log_softmax(zq, 1)
                logq = lq.gather(1, i[hv].clamp(min=0))
                term = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p))
                row[hv] += a * t * t * term.sum(1)
                big = zq.abs().gather(1, i[hv].clamp(min=0)) + torch.logsumexp(zq, 1).abs()[:, None]
                vb = v.abs().masked_fill(~th[hv], 0) + torch.logsumexp(v, 1).abs()[:, None]
                mag[hv] += a * t * t * (p * (big + vb)).sum(1)
                m = torch.zeros_like(zg[hv]).scatter_add_(1, i[hv].clamp(min=0), p)
                d[hv] += a * t * (lq.exp() - m)
                dm[hv] += a * t * (lq.exp() + m)
        rows.append(row)
        mags.append(mag)
        grads.append(d * float(dloss[g]) / B)
        gmags.append(dm * abs(float(dloss[g])) / B)
    return torch.stack(rows), torch.stack(mags), torch.cat(grads, 1), torch.cat(gmags, 1)


def hits(z, lab):
    G, B = lab.shape
    N = z.shape[1] // G
    zg = z.reshape(B, G, N).double().transpose(0, 1)
    y = lab.long().clamp(min=0).unsqueeze(2)
    zy = zg.gather(2, y)
    cols = torch.arange(N, device=z.device)
    rank = ((zg > zy) | ((zg == zy) & (cols < y))).sum(2)
    ok = lab >= 0
    top5 = ((rank < 5) & ok).sum(1) if N > 2 else torch.full((G,), B, device=z.device)
    return ((rank < 1) & ok).sum(1), top5


def check(G, B, N, K, dtype=torch.float32, unit=True, ragged=True, device="cpu", seed=0, args=None,
          **kw):
    """Tolerances: a softmax term exp(x), x = (z - max) / tau, carries the
    rounding of x (|x| 2^-23) and of exp, the sums a few steps: 2^-20 (2 + max|x|)
    of every term; a row loss 2^-20 of the magnitudes that it adds and the
    softmax's relative error.  Then half a step of the output's type."""
    z, lab, val, idx, alpha, tau = args or inputs(G, B, N, K, dtype, ragged, device, seed, **kw)
    acc = torch.full((G, 4), 2.0, device=device)
    dloss = torch.ones(G, device=device) if unit else torch.linspace(0.5, 2, G, device=device)
    z = z.detach().requires_grad_(True)
    loss = L.distill_ce(z, lab, acc, G, val, idx, alpha, tau, unit=unit)
    dz, = torch.autograd.grad(loss, [z], dloss)
    assert loss.dtype == torch.float32 and dz.dtype == dtype and dz.shape == z.shape
    rows, mags, d, dm = reference(z.detach(), lab, val, idx, alpha, tau, dloss)
    zf = z.detach().double().reshape(B, G, -1)
    fin = torch.where(torch.isfinite(zf) & (zf.abs() < 1e30), zf, zf.new_zeros(()))
    span = 2 + (fin.max(2).values - fin.min(2).values)                          # [B, G]
    e = 2.0 ** -20 * span
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    tol = e.repeat_interleave(z.shape[1] // G, 1) * dm
    tol = tol + half * (d.abs() + tol) + 1e-30
    err = (dz.double() - d).abs()
    assert (err <= tol).all(), ("dz", float((err / tol).max()))
    rt = (2.0 ** -20 * mags + 2 * e.t() * (mags > 0)).mean(1) + 2.0 ** -24 * rows.abs().mean(1)
    lerr = (loss.detach().double() - rows.mean(1)).abs()
    assert (lerr <= rt).all(), ("loss", lerr, rt)
    t1, t5 = hits(z.detach(), lab)
    assert torch.equal(acc[:, 1] - 2, t1.float()) and torch.equal(acc[:, 2] - 2, t5.float())
    assert (acc[:, 3] == 2 + B).all()
    serr = (acc[:, 0].double() - 2 - rows.sum(1)).abs()
    assert (serr <= B * rt + 2.0 ** -23 * (2 + rows.sum(1).abs())).all()
    return loss.detach(), dz


@pytest.mark.parametrize("unit", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (2, 6, 2, 2), (3, 7, 11, 4), (2, 5, 300, 0)],
                         ids=lambda s: "x".join(map(str, s)))
def test_cpu_path(size, dtype, unit):
    check(*size, dtype, unit)


def test_weights_of_zero_are_not_computed():
    z, lab, val, idx, _, _ = inputs(2, 4, 6, 3, ragged=False)
    acc = torch.zeros(2, 4)
    z2 = z.clone()
    z2[:, 0] = -math.inf                                   # hopeless for class 0 of config 0
    lab[0] = 0
    ones = torch.ones(2)
    loss = L.distill_ce(z2, lab, acc, 2, val, torch.where(idx == 0, 1, idx).int(), ones, ones)
    assert torch.isfinite(loss).all()                      # alpha = 1: labels do not matter
    idx2 = torch.full_like(idx, 99)
    loss = L.distill_ce(z, lab, acc, 2, val, idx2, 0.0, 1.0)
    assert torch.isfinite(loss).all()                      # alpha = 0: entries do not matter
    want = torch.nn.functional.cross_entropy(z[:, :6].double(), lab[0].long())
    assert abs(float(loss[0]) - float(want)) < 1e-5


def test_out_of_range_classes_poison_their_row():
    z, lab, val, idx, alpha, tau = inputs(1, 4, 6, 3, ragged=False)
    for what in ("label", "entry"):
        lab2, idx2 = lab.clone(), idx.clone()
        if what == "label":
            lab2[0, 2] = 6
        else:
            idx2[0, 2, 1] = 6
        x = z.clone().requires_grad_(True)
        loss = L.distill_ce(x, lab2, torch.zeros(1, 4), 1, val, idx2, alpha, tau)
        d, = torch.autograd.grad(loss.sum(), [x])
        assert torch.isnan(loss).all() and torch.isnan(d[2]).all()
        assert torch.isfinite(d[[0, 1, 3]]).all()


def test_shared_teacher():
    z, lab, val, idx, alpha, tau = inputs(3, 4, 9, 3, ragged=False)
    a1, a2 = torch.zeros(3, 4), torch.zeros(3, 4)
    one = L.distill_ce(z, lab, a1, 3, val[0], idx[0], alpha, tau)
    two = L.distill_ce(z, lab, a2, 3, val[:1].repeat(3, 1, 1), idx[:1].repeat(3, 1, 1), alpha, tau)
    assert torch.equal(one, two) and torch.equal(a1, a2)


def test_refusals():
    z, lab, val, idx, alpha, tau = inputs(2, 4, 6, 3)
    acc = torch.zeros(2, 4)
    good = dict(logits=z, labels=lab, acc=acc, G=2, top_val=val, top_idx=idx, alpha=alpha, tau=tau)
    L.distill_ce(**good)

    def bad(exc, match, **kw):
        with pytest.raises(exc, match=match):
            L.distill_ce(**dict(good, **kw))
    bad(ValueError, "G\\*N", G=5)
    bad(ValueError, "no rows", logits=z[:0])
    bad(TypeError, "fp32 or bf16", logits=z.half())
    bad(ValueError, "labels", labels=lab.long())
    bad(ValueError, "labels", labels=lab[:, :3])
    bad(ValueError, "acc", acc=torch.zeros(2, 3))
    bad(ValueError, "acc", acc=torch.zeros(4, 2).t())
    bad(ValueError, "top_val", top_val=val.double())
    bad(ValueError, "top_idx", top_idx=idx[:, :, :2])
    bad(ValueError, "top_idx", top_idx=idx.long())
    bad(ValueError, "alpha", alpha=1.5)
    bad(ValueError, "alpha", alpha=torch.zeros(3))
    bad(ValueError, "tau", tau=0.0)
    bad(ValueError, "tau", tau=float("nan"))
    bad(ValueError, "at most", top_val=torch.zeros(2, 4, 1025),
        top_idx=torch.zeros(2, 4, 1025, dtype=torch.int32))
    for k in (0, 7, -1):
        with pytest.raises(ValueError, match="top_logits: k"):
            L.top_logits(z, 2, k)
    with pytest.raises(ValueError, match="top_logits: k"):
        L.top_logits(torch.zeros(1, 2000), 1, 1025)
    with pytest.raises(TypeError, match="top_logits"):
        L.top_logits(z.double(), 2, 1)
    with pytest.raises(ValueError, match="top_logits"):
        L.top_logits(z[0], 2, 1)


def top_reference(z, G, k):
    """By a stable sort in 64 bits on the host: NaN first, +0 equal to -0."""
    zc = z.detach().double().cpu()
    B = zc.shape[0]
    x = zc.view(B, G, -1).transpose(0, 1)
    nan = torch.isnan(x)
    order = torch.argsort(torch.where(nan, torch.full_like(x, math.inf), x), dim=2,
                          descending=True, stable=True)
    late = torch.argsort(nan.gather(2, order).int(), dim=2, descending=True, stable=True)
    i = order.gather(2, late)[:, :, :k]
    v = z.detach().cpu().view(B, G, -1).transpose(0, 1).gather(2, i)
    return v, i.to(torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_top_logits_cpu(dtype):
    z = (torch.randn(5, 3 * 40, generator=torch.Generator().manual_seed(0)) * 2).round().to(dtype)
    z[1, 5] = float("nan")
    z[2, :40] = 0.0
    z[2, 7] = -0.0
    for k in (1, 3, 40):
        v, i = L.top_logits(z, 3, k)
        vr, ir = top_reference(z, 3, k)
        assert torch.equal(i, ir) and v.dtype == dtype
        assert torch.equal(v.nan_to_num(9e9), vr.nan_to_num(9e9))
    zz = z.clone().requires_grad_(True)
    assert not L.top_logits(zz, 3, 2)[0].requires_grad


@pytest.mark.parametrize("unit", [True, False])
def test_gradients_of_a_kept_graph_are_the_callers(unit):
    z, lab, val, idx, alpha, tau = inputs(2, 6, 30, 4)
    x = z.clone().requires_grad_(True)
    loss = L.distill_ce(x, lab, torch.zeros(2, 4), 2, val, idx, alpha, tau, unit=unit)
    first, = torch.autograd.grad(loss, [x], torch.ones(2), retain_graph=True)
    want = first.clone()
    first.mul_(100.0)
    assert torch.equal(torch.autograd.grad(loss, [x], torch.ones(2))[0], want)


def one_row_layouts(z):
    """[1, W] views of a row whose pitch is below W."""
    col = z.reshape(-1).clone()[:, None]                        # [W, 1]
    yield col.t()
    yield z.contiguous().as_strided(z.shape, (0, 1))
    yield torch.cat([col, col], 1)[:, :1].t()


def test_a_single_row_has_a_pitch():
    z = torch.randn(1, 10)
    for x in one_row_layouts(z):
        assert x.stride(0) < 10
        rows, N = L._logit_rows("test", x, 2)
        assert rows.stride() == (10, 1) and N == 5 and torch.equal(rows, z)
    # one class and one config: any stride between elements that are not there
    assert L._logit_rows("test", torch.randn(6, 3)[:, 1:2], 1)[0].stride(0) >= 1


def test_sizes_beyond_the_kernels_are_refused():
    """Classes are ints (2^32 + 5 of them were taken for 5), a launch has fewer
    than 2^32 threads and 65536 configurations."""
    import ctypes
    from cerebro_ds_kpgi_amd.ops import _hip
    lib, n = _hip.lib(), _hip.nodes()
    ws, top = lib.cer_distill_ws, lib.cer_top_ws
    ws.restype = top.restype = ctypes.c_int64
    for bf16 in (0, 1):
        assert ws(2 ** 26 - 1, 1, 2, bf16) > 0 and ws(2 ** 26, 1, 2, bf16) == -1
        assert ws(2 ** 24 - 1, 1, 600, bf16) > 0 and ws(2 ** 24, 1, 600, bf16) == -1
        assert ws(2 ** 20, 1, 2 ** 24, bf16) == -1 and ws(1, 1, 2 ** 31 - 1, bf16) == -1
        assert ws(1, 65535, 5, bf16) > 0 and ws(1, 65536, 5, bf16) == -1
        assert top(2 ** 26 - 1, 1, 2, 1, bf16) == 0 and top(2 ** 26, 1, 2, 1, bf16) == -1
        assert top(1, 2 ** 24, 600, 1, bf16) == -1 and top(2 ** 22, 1, 70000, 1, bf16) == -1
    i32 = torch.int32
    for N in (2 ** 31 - 1, 2 ** 31 + 8, 2 ** 32 + 5):
        z = torch.zeros(1, 1).expand(1, N)
        with pytest.raises(ValueError, match="grids|2\\^31"):
            n.top_logits(z, 1, 3)
        with pytest.raises(ValueError, match="grids|2\\^31"):
            n.distill_ce(z, torch.zeros(1, 1, dtype=i32), torch.zeros(1, 4), 1, torch.zeros(1, 1, 1),
                         torch.zeros(1, 1, 1, dtype=i32), None, 0.5, None, 1.0, False, False)


def test_no_second_derivative_on_the_cpu():
    """Not even in part: through the loss gradient of a squared loss."""
    z, lab, val, idx, alpha, tau = inputs(2, 4, 6, 3)
    for unit in (True, False):
        x = z.clone().requires_grad_(True)
        loss = L.distill_ce(x, lab, torch.zeros(2, 4), 2, val, idx, alpha, tau, unit=unit)
        with pytest.raises(RuntimeError, match="second derivative"):
            d, = torch.autograd.grad((loss * loss).sum(), [x], create_graph=True)
            torch.autograd.grad(d.sum(), [x])
