"""Operators of the packed training and serving paths, as timed and compared cases.

Three kinds of case, each over G packed configurations:

* ``linear``  -- ``ops.nn.linear_act``: y = residual + act(x W^T + b) for config
  g's column block, and in training its input, weight and bias gradients;
* ``distill`` -- ``ops.loss.distill_ce``: cross-entropy on labels mixed with the
  KL divergence from a teacher known by its top logits, with the gradient;
* ``top``     -- ``ops.loss.top_logits``: the k largest logits of a teacher and
  their classes, in descending order, ties by class number.

``own`` False computes a case with elementary torch operations in 32 bits,
True through the framework's entry points.
"""

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_SMOOTH = ("none", "gelu", "gelu_tanh", "silu")
# relu and relu6 are drawn for the forward pass only: among millions of random
# pre-activations some lie closer to the kink than 32 bits of any order of
# summation resolve, and each of those moves the weight gradient by a whole term
_ACTS = _SMOOTH + ("relu", "relu6")


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the ResNet-50 head of one configuration at the grid's batch of 32:
        # a training step's smallest dense layer, where launches count
        {"name": "linear_head", "kind": "linear", "dtype": "fp32", "G": 1, "M": 32, "K": 2048,
         "N": 1000, "act": "none", "bias": True, "residual": False, "train": True},
        # Criteo confA's second layer, 16 configurations of the grid at batch 256
        {"name": "linear_criteo", "kind": "linear", "dtype": "fp32", "G": 16, "M": 256, "K": 1000,
         "N": 500, "act": "silu", "bias": True, "residual": False, "train": True},
        # VGG-16's fc1 on 112 x 112 images, 8 configurations at batch 32:
        # weights and their gradients are the traffic
        {"name": "linear_fc1", "kind": "linear", "dtype": "fp32", "G": 8, "M": 32, "K": 4608,
         "N": 4096, "act": "gelu_tanh", "bias": True, "residual": False, "train": True},
        # a residual block's dense layer over many rows (tokens, patches) in
        # the bf16 compute mode; the largest case
        {"name": "linear_block_bf16", "kind": "linear", "dtype": "bf16", "G": 1, "M": 8192,
         "K": 4096, "N": 4096, "act": "gelu", "bias": True, "residual": True, "train": True},
        # the same kind of layer in fp32, two configurations, ragged rows
        {"name": "linear_block_fp32", "kind": "linear", "dtype": "fp32", "G": 2, "M": 2047,
         "K": 1536, "N": 2048, "act": "silu", "bias": True, "residual": True, "train": True},
        # one row at a time: serving a trained residual block
        {"name": "linear_serve", "kind": "linear", "dtype": "bf16", "G": 1, "M": 1, "K": 4096,
         "N": 4096, "act": "relu", "bias": True, "residual": True, "train": False},
        # a ResNet-50 student of one configuration, 1000 classes, batch 32
        {"name": "distill_head", "kind": "distill", "dtype": "fp32", "G": 1, "B": 32, "N": 1000,
         "k": 10, "unit": True, "ragged": False},
        # 8 packed students at the grid's larger batch, some rows unlabelled
        # or without a teacher, a general gradient from above
        {"name": "distill_pack", "kind": "distill", "dtype": "fp32", "G": 8, "B": 256, "N": 1000,
         "k": 20, "unit": False, "ragged": True},
        # token-level distillation over a large, odd vocabulary
        {"name": "distill_wide", "kind": "distill", "dtype": "bf16", "G": 1, "B": 4096, "N": 49999,
         "k": 64, "unit": True, "ragged": True},
        # top logits of 8 packed teachers over 1000 classes
        {"name": "top_head", "kind": "top", "dtype": "fp32", "G": 8, "B": 32, "N": 1000, "k": 10},
        # top logits of a token-level teacher: many rows, long axis
        {"name": "top_wide", "kind": "top", "dtype": "bf16", "G": 1, "B": 2048, "N": 65536,
         "k": 64},
        # few rows over a long axis: the axis is what there is to split
        {"name": "top_few", "kind": "top", "dtype": "fp32", "G": 1, "B": 3, "N": 131071, "k": 200},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "distill", "top"])
    dtype = rng.choice(["fp32", "bf16"])
    if kind == "linear":
        train = rng.random() < 0.75
        while True:
            G = _log_int(rng, 1, 16)
            M = _log_int(rng, 1, 8192)
            K = _log_int(rng, 4, 8192)
            N = _log_int(rng, 2, 8192)
            if rng.random() < 0.5:          # widths of real layers are mostly even
                K, N = (K + 7) // 8 * 8, (N + 7) // 8 * 8
            if G * N * K <= 1 << 26 and G * M * N * K <= 1 << (37 if dtype == "bf16" else 35):
                break
        return {"kind": "linear", "dtype": dtype, "G": G, "M": M, "K": K, "N": N,
                "act": rng.choice(_SMOOTH if train else _ACTS), "bias": rng.random() < 0.8,
                "residual": rng.random() < 0.5, "train": train}
    while True:
        G = _log_int(rng, 1, 16)
        B = _log_int(rng, 1, 8192)
        N = _log_int(rng, 2, 131072)
        if G * B * N <= 1 << 27:
            break
    k = _log_int(rng, 1, min(256, N))
    if kind == "distill":
        return {"kind": "distill", "dtype": dtype, "G": G, "B": B, "N": N, "k": k,
                "unit": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    return {"kind": "top", "dtype": dtype, "G": G, "B": B, "N": N, "k": k}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _inputs(case, seed):
    """The tensors of a case, made from the seed alone."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    G = case["G"]
    if case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        t = {"x": normal(M, G * K).to(dt),
             "w": (normal(G, N, K) * math.sqrt(2.0 / K)).to(dt),
             "b": (normal(G, N) * 0.1).to(dt) if case["bias"] else None,
             "r": normal(M, G * N).to(dt) if case["residual"] else None}
        if case["train"]:
            t["dy"] = (normal(M, G * N) / M).to(dt)
        return t
    B, N = case["B"], case["N"]
    logits = normal(B, G * N).mul_(3.0)
    if case["kind"] == "top":
        return {"logits": logits.to(dt)}
    k = case["k"]
    # a teacher that mostly agrees with the student; its top logits
    teacher = logits.view(B, G, N) * 0.8 + normal(B, G, N).mul_(1.5)
    val, idx = torch.topk(teacher, k, dim=2)
    del teacher
    val = val.transpose(0, 1).to(dt).contiguous()                       # [G, B, k]
    idx = idx.transpose(0, 1).to(torch.int32).contiguous()
    labels = torch.randint(0, N, (G, B), generator=gen, device=dev, dtype=torch.int32)
    # half of the labels are the teacher's first choice
    first = torch.rand(G, B, generator=gen, device=dev) < 0.5
    labels = torch.where(first, idx[:, :, 0], labels)
    if case["ragged"]:
        # padded classes at the type's lowest value (never the teacher's
        # choice), rows with fewer or no teacher entries, unlabelled rows
        pad = N // 100
        if pad:
            cols = torch.arange(N, device=dev) >= N - pad
            idx = torch.where(cols[idx.long()], torch.full_like(idx, -1), idx)
            labels = torch.where(cols[labels.long()], torch.full_like(labels, -1), labels)
            logits.view(B, G, N).masked_fill_(cols, torch.finfo(dt).min)
        keep = torch.randint(0, k + 1, (G, B, 1), generator=gen, device=dev)
        short = torch.rand(G, B, 1, generator=gen, device=dev) < 0.3
        gone = short & (torch.arange(k, device=dev) >= keep)
        idx = torch.where(gone, torch.full_like(idx, -1), idx)
        unlab = torch.rand(G, B, generator=gen, device=dev) < 0.2
        labels = torch.where(unlab, torch.full_like(labels, -1), labels)
    return {"logits": logits.to(dt), "labels": labels, "val": val, "idx": idx,
            "alpha": torch.rand(G, generator=gen, device=dev) * 0.8 + 0.1,
            "tau": torch.rand(G, generator=gen, device=dev) * 3.0 + 1.0,
            "dloss": (torch.ones(G, device=dev) if case["unit"] else
                      torch.rand(G, generator=gen, device=dev) + 0.5)}


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    if own and case["kind"] == "linear":
        # the parameters live in the configurations' arena
        from cerebro_ds_kpgi_amd.runtime.arena import Arena, ModelLayout, ParamRef, ParamSpec
        specs = [ParamSpec("dense/kernel", (case["N"], case["K"]), "weight")]
        if case["bias"]:
            specs.append(ParamSpec("dense/bias", (case["N"],), "bias"))
        arena = Arena(ModelLayout(specs), case["G"], "cuda", _DTYPES[case["dtype"]])
        refs = [ParamRef(arena, s) for s in specs]
        refs[0].master().copy_(t["w"])
        if case["bias"]:
            refs[1].master().copy_(t["b"])
        arena.sync_work()
        state["wref"], state["bref"] = refs[0], refs[1] if case["bias"] else None
    if own and case.get("train"):
        t["x"].requires_grad_(True)
        if t["r"] is not None:
            t["r"].requires_grad_(True)
    if own and case["kind"] == "distill":
        t["logits"].requires_grad_(True)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    case, t = state["case"], state["t"]
    return {"linear": _linear, "distill": _distill, "top": _top}[case["kind"]](case, t, state)


def _act(z, act):
    """act(z) and act'(z)."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.clamp(z, min=0.0), (z > 0).to(z.dtype)
    if act == "relu6":
        return torch.clamp(z, 0.0, 6.0), ((z > 0) & (z < 6)).to(z.dtype)
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z * z * z))
        return (0.5 * z * (1.0 + th),
                0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * c * (1.0 + 0.134145 * z * z))
    s = 1.0 / (1.0 + torch.exp(-z))
    return z * s, s * (1.0 + z * (1.0 - s))


def _linear(case, t, state):
    G, M, K, N = case["G"], case["M"], case["K"], case["N"]
    if own:
        from cerebro_ds_kpgi_amd.ops import nn as P
        if not case["train"]:
            with torch.no_grad():
                return {"y": P.linear_act(t["x"], state["wref"], state["bref"], case["act"],
                                          t["r"])}
        y = P.linear_act(t["x"], state["wref"], state["bref"], case["act"], t["r"])
        leaves = [t["x"]] + ([t["r"]] if case["residual"] else [])
        grads = torch.autograd.grad(y, leaves, t["dy"])
        out = {"y": y.detach(), "dx": grads[0], "dw": state["wref"].grad()}
        if case["bias"]:
            out["db"] = state["bref"].grad()
        if case["residual"]:
            out["dr"] = grads[1]
        return out
    dt = t["x"].dtype
    xg = t["x"].view(M, G, K).float().transpose(0, 1).contiguous()          # [G, M, K]
    w = t["w"].float()
    z = torch.bmm(xg, w.transpose(1, 2).contiguous())                        # [G, M, N]
    if case["bias"]:
        z = z + t["b"].float().unsqueeze(1)
    a, d = _act(z, case["act"])
    y = a.transpose(0, 1).reshape(M, G * N)
    if case["residual"]:
        y = y + t["r"].float()
    if not case["train"]:
        return {"y": y.to(dt)}
    dz = t["dy"].view(M, G, N).float().transpose(0, 1) * d                   # [G, M, N]
    dx = torch.bmm(dz, w).transpose(0, 1).reshape(M, G * K)
    out = {"y": y.to(dt), "dx": dx.to(dt),
           "dw": torch.bmm(dz.transpose(1, 2).contiguous(), xg)}
    if case["bias"]:
        out["db"] = dz.sum(1)
    if case["residual"]:
        out["dr"] = t["dy"]
    return out


def _distill(case, t, state):
    G, B, N = case["G"], case["B"], case["N"]
    if own:
        from cerebro_ds_kpgi_amd.ops import loss as L
        acc = torch.zeros(G, 4, device="cuda")
        loss = L.distill_ce(t["logits"], t["labels"], acc, G, t["val"], t["idx"], t["alpha"],
                            t["tau"], unit=case["unit"])
        dlogits, = torch.autograd.grad(loss, [t["logits"]], t["dloss"])
        return {"loss": loss.detach(), "acc": acc, "dlogits": dlogits}
    z = t["logits"].view(B, G, N).float()
    lab = t["labels"].t().long()                                             # [B, G]
    idx = t["idx"].transpose(0, 1).long()                                    # [B, G, k]
    val = t["val"].transpose(0, 1).float()
    alpha, tau = t["alpha"].view(1, G), t["tau"].view(1, G)
    has_y = (lab >= 0).float()
    yi = lab.clamp(min=0).unsqueeze(2)
    have = idx >= 0
    ii = idx.clamp(min=0)
    has_t = have.any(2).float()

    mx = z.max(2, keepdim=True).values
    e1 = torch.exp(z - mx)
    s1 = e1.sum(2, keepdim=True)
    e2 = torch.exp((z - mx) / tau.unsqueeze(2))
    s2 = e2.sum(2, keepdim=True)
    # teacher's distribution over its entries
    v = val / tau.unsqueeze(2)
    v = torch.where(have, v, torch.full_like(v, -math.inf))
    vm = torch.where(has_t.unsqueeze(2) > 0, v.max(2, keepdim=True).values,
                     torch.zeros_like(v[:, :, :1]))
    p = torch.exp(v - vm)
    ps = p.sum(2, keepdim=True).clamp(min=1e-30)
    p = p / ps
    logp = torch.where(have, v - vm - torch.log(ps), torch.zeros_like(v))
    logq = (z.gather(2, ii) - mx) / tau.unsqueeze(2) - torch.log(s2)
    zy = z.gather(2, yi)
    hard = has_y * (torch.log(s1) + mx - zy).squeeze(2)                       # [B, G]
    soft = torch.where(have, p * (logp - logq), torch.zeros_like(p)).sum(2)
    row = (1 - alpha) * hard + alpha * tau * tau * soft
    # gradient
    c1 = ((1 - alpha) * has_y).unsqueeze(2)
    c2 = (alpha * tau * has_t).unsqueeze(2)
    d = e1.mul_(c1 / s1).add_(e2.mul_(c2 / s2))
    d.scatter_add_(2, yi, -c1)
    d.scatter_add_(2, ii, torch.where(have, -c2 * p, torch.zeros_like(p)))
    d = d * (t["dloss"].view(1, G, 1) / B)
    # metrics: the label's rank, ties by class number
    cols = torch.arange(N, device=z.device).view(1, 1, N)
    rank = ((z > zy) | ((z == zy) & (cols < yi))).sum(2)
    top1 = ((rank < 1) * has_y).sum(0)
    top5 = ((rank < 5) * has_y).sum(0) if N > 2 else torch.full_like(top1, float(B))
    acc = torch.stack([row.sum(0), top1, top5, torch.full_like(top1, float(B))], 1)
    return {"loss": row.mean(0), "acc": acc, "dlogits": d.reshape(B, G * N).to(t["logits"].dtype)}


def _top(case, t, state):
    G, B, N, k = case["G"], case["B"], case["N"], case["k"]
    if own:
        from cerebro_ds_kpgi_amd.ops import loss as L
        val, idx = L.top_logits(t["logits"], G, k)
        return {"val": val, "idx": idx}
    z = t["logits"].view(B, G, N).transpose(0, 1).float()
    val, idx = torch.sort(z, dim=2, descending=True, stable=True)
    return {"val": val[:, :, :k].to(t["logits"].dtype), "idx": idx[:, :, :k].to(torch.int32)}


# ---------------------------------------------------------------------------
# cost and 64-bit values
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    G = case["G"]
    if case["kind"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        x, w, y = M * G * K, G * N * K, M * G * N
        b = G * N if case["bias"] else 0
        r = y if case["residual"] else 0
        nbytes = e * (x + w + b + r + y)
        flops = 2 * G * M * N * K
        if case["train"]:
            nbytes += e * (y + x) + 4 * (w + b)      # dy in; dx, dw, db out (dr is dy)
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    B, N, k = case["B"], case["N"], case["k"]
    n = B * G * N
    if case["kind"] == "distill":
        # logits in, gradient out, the teacher's entries and the labels in
        return {"bytes": 2 * e * n + G * B * (k * (e + 4) + 4), "flops": 8 * n}
    return {"bytes": e * n + G * B * k * (e + 4), "flops": n}


def exact(case, seed):
    t = _inputs(case, seed)
    G = case["G"]
    if case["kind"] == "linear":
        return _exact_linear(case, t)
    B, N, k = case["B"], case["N"], case["k"]
    if case["kind"] == "top":
        val, idx = [], []
        for g in range(G):
            z = t["logits"][:, g * N:(g + 1) * N].double()
            order = torch.argsort(z, dim=1, descending=True, stable=True)[:, :k]
            val.append(z.gather(1, order))
            idx.append(order.to(torch.int32))
        return {"val": torch.stack(val), "idx": torch.stack(idx)}
    loss, acc, dlogits = [], [], torch.empty(B, G * N, dtype=torch.float64, device="cuda")
    for g in range(G):
        z = t["logits"][:, g * N:(g + 1) * N].double().requires_grad_(True)
        al, ta = float(t["alpha"][g].double()), float(t["tau"][g].double())
        rows = torch.zeros(B, dtype=torch.float64, device="cuda")
        lab = t["labels"][g].long()
        y = (lab >= 0).nonzero().squeeze(1)
        logq1 = torch.log_softmax(z, 1)
        rows = rows.index_add(0, y, -(1 - al) * logq1[y, lab[y]])
        idx = t["idx"][g].long()
        for_t = (idx >= 0).any(1).nonzero().squeeze(1)
        if len(for_t):
            logq = torch.log_softmax(z / ta, 1)[for_t]
            have = idx[for_t] >= 0
            v = (t["val"][g][for_t].double() / ta).masked_fill(~have, -math.inf)
            logp = torch.log_softmax(v, 1).masked_fill(~have, 0.0)
            p = torch.softmax(v, 1)
            kl = (p * (logp - logq.gather(1, idx[for_t].clamp(min=0)))).sum(1)
            rows = rows.index_add(0, for_t, al * ta * ta * kl)
        mean = rows.mean()
        d, = torch.autograd.grad(mean * float(t["dloss"][g].double()), [z])
        dlogits[:, g * N:(g + 1) * N] = d
        with torch.no_grad():
            zl = z.detach()
            own_z = zl.gather(1, lab.clamp(min=0).unsqueeze(1))
            lower = torch.arange(N, device="cuda").unsqueeze(0) < lab.unsqueeze(1)
            ahead = (zl > own_z).sum(1) + ((zl == own_z) & lower).sum(1)
            hit1 = float(((ahead < 1) & (lab >= 0)).sum())
            hit5 = float(((ahead < 5) & (lab >= 0)).sum()) if N > 2 else float(B)
        loss.append(mean.detach())
        acc.append(torch.tensor([float(rows.detach().sum()), hit1, hit5, float(B)],
                                dtype=torch.float64, device="cuda"))
    return {"loss": torch.stack(loss), "acc": torch.stack(acc), "dlogits": dlogits}


def _exact_linear(case, t):
    """The layer config by config in 64 bits; gradients by differentiation."""
    F = torch.nn.functional
    fn = {"none": lambda z: z, "relu": F.relu, "relu6": F.relu6, "gelu": F.gelu,
          "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}[case["act"]]
    G, M, K, N = case["G"], case["M"], case["K"], case["N"]
    y = torch.empty(M, G * N, dtype=torch.float64, device="cuda")
    out = {"y": y}
    if case["train"]:
        out["dx"] = torch.empty(M, G * K, dtype=torch.float64, device="cuda")
        out["dw"] = torch.empty(G, N, K, dtype=torch.float64, device="cuda")
        if case["bias"]:
            out["db"] = torch.empty(G, N, dtype=torch.float64, device="cuda")
        if case["residual"]:
            out["dr"] = t["dy"].double()
    for g in range(G):
        rows, cols = slice(g * K, (g + 1) * K), slice(g * N, (g + 1) * N)
        x = t["x"][:, rows].double().requires_grad_(case["train"])
        w = t["w"][g].double().requires_grad_(case["train"])
        b = t["b"][g].double().requires_grad_(case["train"]) if case["bias"] else None
        v = fn(F.linear(x, w, b))
        if case["train"]:
            wrt = [x, w] + ([b] if case["bias"] else [])
            d = torch.autograd.grad(v, wrt, t["dy"][:, cols].double())
            out["dx"][:, rows], out["dw"][g] = d[0], d[1]
            if case["bias"]:
                out["db"][g] = d[2]
        y[:, cols] = v.detach() + (t["r"][:, cols].double() if case["residual"] else 0.0)
    return out
