"""Fused softmax cross-entropy + top-1/top-5 metrics for G packed configs.

logits ``[B, G*N]`` (config g owns columns ``g*N:(g+1)*N``), labels
``[G, B]`` int32.  Per config: mean CE over the batch (= Keras
``categorical_crossentropy`` / torch ``CrossEntropyLoss``), and the metric
accumulator ``acc[g] += (loss_sum, top1_correct, top5_correct, count)``
on device — no host sync per step (reference metrics: SURVEY.md §5.5,
``cerebro_gpdb/run_pytorchddp.py:181-201``).  For N == 2 (Criteo) top-5 is
reported as 1 (reference binary-accuracy path).
"""

import torch

from .backend import use_hip


class SoftmaxCE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, acc, G, head=None, unit=False):
        B = logits.shape[0]
        N = logits.shape[1] // G
        ctx.unit = unit
        if unit and logits.dtype == torch.float32 and use_hip("loss", logits):
            # training step: the caller seeds a unit gradient and reads the
            # metrics from ``acc`` -- no loss values, and the head's bias
            # gradient comes out of this kernel (``head`` = (bias ref, box))
            from . import _hip
            dlogits = _hip.softmax_ce_train(logits, labels, acc, G,
                                            head[0] if head is not None else None)
            if head is not None:
                head[1][0] = True
            ctx.save_for_backward(dlogits)
            ctx.dtype = logits.dtype
            return logits.new_empty(G)
        if use_hip("loss", logits):
            from . import _hip
            loss, dlogits = _hip.softmax_ce_fwd(logits, labels, acc, G)
        else:
            z = logits.view(B, G, N).float()
            lse = torch.logsumexp(z, dim=2)                             # [B, G]
            lab = labels.t().long()                                     # [B, G]
            picked = z.gather(2, lab.unsqueeze(2)).squeeze(2)
            nll = lse - picked                                          # [B, G]
            loss = nll.mean(0)                                          # [G]
            p = torch.softmax(z, dim=2)
            onehot = torch.zeros_like(p).scatter_(2, lab.unsqueeze(2), 1.0)
            dlogits = ((p - onehot) / B).reshape(B, G * N)
            with torch.no_grad():
                k = min(5, N)
                top = z.topk(k, dim=2).indices                          # [B, G, k]
                hit = top == lab.unsqueeze(2)
                top1 = hit[:, :, 0].float().sum(0)
                top5 = hit.any(2).float().sum(0) if N > 2 else torch.full_like(top1, float(B))
                acc += torch.stack([nll.sum(0), top1, top5, torch.full_like(top1, float(B))], 1)
        ctx.save_for_backward(dlogits)
        ctx.dtype = logits.dtype
        return loss

    @staticmethod
    def backward(ctx, dloss):
        dlogits, = ctx.saved_tensors
        if ctx.unit:                    # dloss is ones by the caller's contract
            return dlogits.to(ctx.dtype), None, None, None, None, None
        B, GN = dlogits.shape
        G = dloss.shape[0]
        d = dlogits.view(B, G, GN // G) * dloss.view(1, G, 1)
        return d.reshape(B, GN).to(ctx.dtype), None, None, None, None, None


def softmax_ce(logits, labels, acc, G, head=None, unit=False):
    """Per-config mean CE ``[G]``.  ``unit=True``: the caller back-propagates
    a gradient of ones (``torch.autograd.backward(loss, ones)``), so the
    backward returns dlogits as they are; on the fp32 HIP path the returned
    loss values are then not computed (metrics live in ``acc``).  ``head``:
    ``logits._cer_head`` of an act-free Dense (ops.nn.PackedLinear) whose
    bias gradient the loss kernel then accumulates."""
    return SoftmaxCE.apply(logits, labels, acc, G, head, unit)


def eval_metrics(logits, labels, acc, G):
    """Validation: same accumulators, no gradient."""
    with torch.no_grad():
        if use_hip("loss", logits):
            from . import _hip
            _hip.softmax_ce_fwd(logits, labels, acc, G, need_grad=False)
            return
        SoftmaxCE.forward(_Ctx(), logits, labels, acc, G)


class _Ctx(object):
    def save_for_backward(self, *a):
        pass


# ---------------------------------------------------------------------------
# distillation from a teacher's top logits
# ---------------------------------------------------------------------------
MAX_TOP = 1024          # teacher entries of a row (csrc/hip/distill.hip KMAX)


def _logit_rows(what, logits, G):
    """[B, G*N] logits with adjacent columns; (rows, N)."""
    if logits.dim() != 2 or G < 1 or logits.shape[1] % G or logits.shape[1] == 0:
        raise ValueError("{}: logits {} are not [B, G*N] for G = {}".format(
            what, tuple(logits.shape), G))
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("{}: logits are {}, not fp32 or bf16".format(what, logits.dtype))
    if logits.shape[0] == 0:
        raise ValueError("{}: no rows".format(what))
    if logits.stride(1) != 1 or logits.stride(0) < logits.shape[1]:
        # the reshape gives a single row its own length as pitch, whatever it had
        logits = logits.reshape(-1, logits.shape[1]).contiguous()
    return logits, logits.shape[1] // G


def top_logits(logits, G, k):
    """The ``k`` largest logits of every row and their classes.

    logits ``[B, G*N]`` (fp32 or bf16) -> values ``[G, B, k]`` in the logits'
    dtype and classes ``[G, B, k]`` int32, in descending order, equal values by
    class number (+0 equals -0, NaN counts as largest); 1 <= k <= min(N, 1024).
    No gradient: this is what a teacher hands to ``distill_ce``.
    """
    if logits.requires_grad:
        logits = logits.detach()
    z, N = _logit_rows("top_logits", logits, G)
    if not 1 <= k <= min(N, MAX_TOP):
        raise ValueError("top_logits: k = {} is not in 1 .. min(N = {}, {})".format(k, N, MAX_TOP))
    if use_hip("top_logits", z):
        from . import _hip
        return _hip.nodes().top_logits(z, G, k)
    v, i = torch.sort(z.reshape(-1, G, N).transpose(0, 1), dim=2, descending=True, stable=True)
    return v[:, :, :k].contiguous(), i[:, :, :k].to(torch.int32)


class DistillCE(torch.autograd.Function):
    """The oracle."""

    @staticmethod
    def forward(ctx, logits, labels, acc, G, val, idx, alpha, tau, unit):
        ctx.unit, ctx.G, ctx.dtype = unit, G, logits.dtype
        loss, d = _distill_torch(logits, labels, acc, G, val, idx, alpha, tau)
        ctx.save_for_backward(d)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        if torch.is_grad_enabled():
            raise RuntimeError("distill_ce has no second derivative (its backward ran with "
                               "create_graph=True)")
        d, = ctx.saved_tensors
        if not ctx.unit:                # else dloss is ones by the caller's contract
            d = (d.view(d.shape[0], ctx.G, -1) * dloss.view(1, ctx.G, 1)).view(d.shape)
        # a copy: the caller may write its gradient and run a kept graph again
        return (d.to(ctx.dtype, copy=True),) + (None,) * 8


def _distill_torch(logits, labels, acc, G, val, idx, alpha, tau):
    """Loss [G] and its gradient [B, G*N] (fp32, for dloss = 1); the oracle."""
    B = logits.shape[0]
    N = logits.shape[1] // G
    inf = float("inf")
    z = logits.detach().reshape(B, G, N).float()
    lab = labels.t().long()                                             # [B, G]
    v, i = val.transpose(0, 1).float(), idx.transpose(0, 1).long()      # [B, G, K]
    a, ta = (x.view(1, G) if isinstance(x, torch.Tensor) else
             torch.full((1, G), x, dtype=torch.float32, device=z.device) for x in (alpha, tau))
    hard_on = (lab >= 0) & (a != 1)
    there = (i >= 0) & (v != -inf) & (a != 0).unsqueeze(2)
    bad = (lab >= N) | ((i >= N) & (a != 0).unsqueeze(2)).any(2)
    there = there & (i < N)
    soft_on = there.any(2)
    yi = lab.clamp(0, N - 1).unsqueeze(2)
    ii = i.clamp(0, N - 1)

    zy = z.gather(2, yi)
    lse = torch.logsumexp(z, dim=2)
    hard = torch.where(hard_on, lse - zy.squeeze(2), torch.zeros_like(lse))
    vt = torch.where(there, v, torch.full_like(v, -inf)) / ta.unsqueeze(2)
    vt = torch.where(soft_on.unsqueeze(2), vt, torch.zeros_like(vt))
    p = torch.where(there, torch.softmax(vt, dim=2), torch.zeros_like(vt))
    logp = torch.log_softmax(vt, dim=2)
    logq = torch.log_softmax(z / ta.unsqueeze(2), dim=2)
    kl = torch.where(p > 0, p * (logp - logq.gather(2, ii)), p)
    soft = torch.where(soft_on, kl.sum(2), torch.zeros_like(lse))
    row = torch.where(hard_on, (1 - a) * hard, torch.zeros_like(hard))
    row = row + torch.where(soft_on, a * ta * ta * soft, torch.zeros_like(soft))
    row = torch.where(bad, torch.full_like(row, float("nan")), row)

    onehot = torch.zeros_like(z).scatter_(2, yi, 1.0)
    d = torch.where(hard_on.unsqueeze(2), (1 - a).unsqueeze(2) * (torch.softmax(z, 2) - onehot),
                    torch.zeros_like(z))
    mass = torch.zeros_like(z).scatter_add_(2, ii, p)
    d = d + torch.where(soft_on.unsqueeze(2), (a * ta).unsqueeze(2) * (logq.exp() - mass),
                        torch.zeros_like(z))
    d = torch.where(bad.unsqueeze(2), torch.full_like(d, float("nan")), d) / B

    known = (lab >= 0) & (lab < N)
    cols = torch.arange(N, device=z.device).view(1, 1, N)
    rank = ((z > zy) | ((z == zy) & (cols < yi))).sum(2)
    top1 = ((rank < 1) & known).float().sum(0)
    top5 = (((rank < 5) & known).float().sum(0) if N > 2 else torch.full_like(top1, float(B)))
    acc += torch.stack([row.sum(0), top1, top5, torch.full_like(top1, float(B))], 1)
    return row.mean(0), d.reshape(B, G * N)


def _per_config(what, x, G, device, lo, hi):
    """A hyper-parameter: a range-checked number or an fp32 [G] tensor."""
    if isinstance(x, torch.Tensor):
        if tuple(x.shape) != (G,) or x.dtype != torch.float32 or x.device != device:
            raise ValueError("distill_ce: {} must be a number or an fp32 [{}] tensor on {}".format(
                what, G, device))
        x = x.detach() if x.requires_grad else x
        return x if x.is_contiguous() else x.contiguous()
    x = float(x)
    if not lo <= x <= hi:
        raise ValueError("distill_ce: {} = {} is not in [{}, {}]".format(what, x, lo, hi))
    return x


def _refuse_teacher(G, B, dev, **tensors):
    K = tensors["top_val"].shape[-1]
    f32, i32 = torch.float32, torch.int32
    for name, dt, shape in (("labels", (i32,), (G, B)), ("acc", (f32,), (G, 4)),
                            ("top_val", (f32, torch.bfloat16), (G, B, K)),
                            ("top_idx", (i32,), (G, B, K))):
        t = tensors[name]
        if tuple(t.shape) != shape or t.dtype not in dt or t.device != dev:
            raise ValueError("distill_ce: {} is {} {} on {}, not {} {} on {}".format(
                name, tuple(t.shape), t.dtype, t.device, shape,
                " or ".join(str(d) for d in dt), dev))
    if K > MAX_TOP:
        raise ValueError("distill_ce: {} teacher entries, at most {}".format(K, MAX_TOP))
    raise ValueError("distill_ce: acc must be contiguous")


def distill_ce(logits, labels, acc, G, top_val, top_idx, alpha=0.5, tau=1.0, unit=False):
    """Per-config mean ``[G]`` of cross-entropy mixed with distillation from a
    teacher known by its top logits (``top_logits``), with metrics.

    Row (g, b), student logits z, label y, teacher entries (i_k, v_k)::

        p = softmax_k(v_k / tau)      q = softmax(z / tau)
        (1 - alpha) (lse(z) - z_y) + alpha tau^2 sum_k p_k (log p_k - log q_{i_k})

    ``logits [B, G*N]`` fp32 or bf16; ``labels [G, B]`` int32, negative = no
    label; ``top_val`` (fp32 or bf16) and ``top_idx`` (int32) ``[G, B, K]``, or
    ``[B, K]`` for one teacher of all configurations, 0 <= K <= 1024: a negative
    class or a value of -inf is no entry, a class named twice counts twice.
    ``alpha`` in [0, 1] and ``tau`` > 0 are numbers or fp32 ``[G]`` device
    tensors (not range-checked there).  A row without a label has no first term,
    one without entries no second, and a term of weight zero is not computed;
    a label or class >= N makes the row's loss and gradient NaN.  The mean is
    over all B rows.

    ``acc [G, 4]`` fp32 += (sum of the rows' losses, top-1, top-5, B), as in
    ``softmax_ce``; unlabelled rows are no hits (with N == 2 every row is a top-5
    hit).  Gradient in ``logits`` only.  ``unit=True``: the caller
    back-propagates a gradient of ones, and the forward writes the gradient in
    the same pass over the logits.  Otherwise the backward reads logits, labels,
    entries, alpha and tau again: one that was written in between is refused.  No
    second or forward-mode derivatives, no tracing.  (Capturing a backward: see
    ``nn.linear_act``.)
    """
    z, N = _logit_rows("distill_ce", logits, G)
    B, dev = z.shape[0], z.device
    if top_val.dim() == 2:
        top_val = top_val.unsqueeze(0).expand(G, -1, -1)
    if top_idx.dim() == 2:
        top_idx = top_idx.unsqueeze(0).expand(G, -1, -1)
    K = top_val.shape[-1]
    if (labels.shape != (G, B) or labels.dtype is not torch.int32 or labels.device != dev
            or acc.shape != (G, 4) or acc.dtype is not torch.float32 or acc.device != dev
            or not acc.is_contiguous() or top_val.shape != (G, B, K)
            or top_val.dtype not in (torch.float32, torch.bfloat16) or top_val.device != dev
            or top_idx.shape != (G, B, K) or top_idx.dtype is not torch.int32
            or top_idx.device != dev or K > MAX_TOP):
        _refuse_teacher(G, B, dev, labels=labels, acc=acc, top_val=top_val, top_idx=top_idx)
    alpha = _per_config("alpha", alpha, G, dev, 0.0, 1.0)
    tau = _per_config("tau", tau, G, dev, 1e-6, 1e6)
    if K and top_val.stride(2) != 1:
        top_val = top_val.contiguous()
    if K and top_idx.stride(2) != 1:
        top_idx = top_idx.contiguous()
    if top_val.requires_grad:
        top_val = top_val.detach()
    labels = labels.contiguous()
    if use_hip("distill", z):
        from . import _hip
        a, a0 = (alpha, 0.0) if isinstance(alpha, torch.Tensor) else (None, alpha)
        t, t0 = (tau, 0.0) if isinstance(tau, torch.Tensor) else (None, tau)
        return _hip.nodes().distill_ce(z, labels, acc, G, top_val, top_idx, a, a0, t, t0, unit,
                                       torch.is_grad_enabled() and z.requires_grad)
    return DistillCE.apply(z, labels, acc, G, top_val, top_idx, alpha, tau, unit)
