"""Workloads of the linear head's losses: softmax cross entropy over a large
vocabulary and distillation from a teacher's top logits, with their gradients
and without keeping the logits.

With hidden states h [T, D], head weights w [V, D] and logits
s = logit_scale * h w^T:

  cross entropy   loss_t = lse_t - s[t, y_t]
  distillation    loss_t = tau^2 (sum_k p_tk (log p_tk - s[t, i_tk]) + lse_t),  logit_scale = 1 / tau,
                  p_t = softmax of the teacher's entries / tau

A row whose target is IGNORE, or whose teacher has no entry, has loss 0, lse 0
and no gradient.  A case's "mode" says what one pass is:

  score     loss and lse
  train     loss, lse, dh and dw in one call
  backprop  dh and dw from the lse that an earlier forward pass returned

"mean" cases reduce the loss to its mean over the rows that count; the others
return a loss per row and take an upstream gradient per row.
"""

from __future__ import annotations

import math

import torch

own = False

IGNORE = -100


def listed():
    return [
        # one token scored by a served model: bound by reading the head once
        dict(name="xent score 1 token", op="xent", mode="score", dtype="bf16", T=1, V=32000, D=4096, K=1,
             keep=1.0, tau=1.0, mean=False, columns=False),
        # a toy model's step: launches and latency, odd extents everywhere
        dict(name="xent train tiny", op="xent", mode="train", dtype="f32", T=33, V=1021, D=257, K=1, keep=0.9,
             tau=1.0, mean=True, columns=False),
        # log-probabilities of a prompt, its first part not counted
        dict(name="xent score prompt", op="xent", mode="score", dtype="bf16", T=2000, V=50001, D=2048, K=1,
             keep=0.7, tau=1.0, mean=False, columns=False),
        # an ordinary training step of a head over 32000 words
        dict(name="xent train 32k words", op="xent", mode="train", dtype="bf16", T=4096, V=32000, D=4096, K=1,
             keep=1.0, tau=1.0, mean=True, columns=False),
        # fine-tuning on answers: a third of the rows counts; the backward node of an autograd graph
        dict(name="xent backprop answers", op="xent", mode="backprop", dtype="bf16", T=8192, V=50001, D=1024, K=1,
             keep=0.33, tau=1.0, mean=False, columns=False),
        # the Float32 output of this framework's MLP (1024 features, column-major) under a head
        dict(name="xent train mlp f32", op="xent", mode="train", dtype="f32", T=2048, V=32000, D=1024, K=1,
             keep=1.0, tau=1.0, mean=True, columns=True),
        # the largest step: 8192 tokens over 131072 words
        dict(name="xent train 128k words", op="xent", mode="train", dtype="bf16", T=8192, V=131072, D=4096, K=1,
             keep=1.0, tau=1.0, mean=True, columns=False),
        # a toy student: launches and latency
        dict(name="distill train tiny", op="distill", mode="train", dtype="bf16", T=17, V=4099, D=192, K=5,
             keep=0.9, tau=2.0, mean=True, columns=False),
        # a short sequence under a wide head: reading and writing the head bounds it
        dict(name="distill train 64 tokens", op="distill", mode="train", dtype="bf16", T=64, V=131072, D=2048, K=32,
             keep=1.0, tau=1.5, mean=False, columns=False),
        # an ordinary student's step from 64 stored teacher logits a token
        dict(name="distill train 32k words", op="distill", mode="train", dtype="bf16", T=4096, V=32000, D=2048,
             K=64, keep=0.95, tau=2.0, mean=True, columns=False),
        # evaluation in Float32
        dict(name="distill score f32", op="distill", mode="score", dtype="f32", T=1000, V=32000, D=2048, K=16,
             keep=0.9, tau=1.0, mean=False, columns=False),
        # the largest student, 128 teacher logits a token; the backward node of an autograd graph
        dict(name="distill backprop 128k words", op="distill", mode="backprop", dtype="bf16", T=4096, V=131072,
             D=4096, K=128, keep=0.95, tau=2.0, mean=False, columns=False),
    ]


def draw(rng):
    def log_uniform(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    while True:
        op = rng.choice(["xent", "distill"])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        T, V, D = log_uniform(1, 8192), log_uniform(500, 131072), log_uniform(64, 4096)
        if rng.random() < 0.5:  # heads are mostly whole multiples of 64 wide
            D = max(64, D // 64 * 64)
        if D == 3072 or V == 3072 or T == 3072:
            continue
        if dtype == "f32" and T * V * D > 2.5e11:  # Float32 heads are the smaller ones
            continue
        if T * V * D < 2e6:
            continue
        return dict(op=op, mode=rng.choice(["score", "train", "backprop"]), dtype=dtype, T=T, V=V, D=D,
                    K=1 if op == "xent" else log_uniform(1, 128), keep=rng.choice([1.0, 0.9, 0.4]),
                    tau=1.0 if op == "xent" else rng.choice([1.0, 1.5, 2.0, 4.0]), mean=rng.random() < 0.5,
                    columns=rng.random() < 0.25)


def _inputs(case, seed):
    """The inputs of a case: states and weights of a partly trained head (the
    true word's logit stands out by 0 to 12), and its targets or teacher."""
    T, V, D, K = case["T"], case["V"], case["D"], case["K"]
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    std = 1.0 / math.sqrt(D)
    w = torch.randn(V, D, generator=gen, device=dev).mul_(std).to(dtype)
    y = torch.randint(0, V, (T,), generator=gen, device=dev)
    h = torch.randn(T, D, generator=gen, device=dev)
    h += (12.0 * uniform(T, 1)) * w[y].float()
    h = h.to(dtype)
    if case["columns"]:
        h = h.t().contiguous().t()
    dropped = uniform(T) >= case["keep"]
    if T > 1:
        dropped[T // 2] = False
    else:
        dropped[:] = False
    s = dict(case=dict(case), h=h, w=w)
    if case["op"] == "xent":
        s["targets"] = torch.where(dropped, torch.full_like(y, IGNORE), y).to(torch.int32)
    else:
        # the teacher's best word is the student's true one; the others lie at
        # a random step, so that a row's entries are distinct; some rows keep
        # fewer than K entries
        step = (uniform(T, 1) * max(1, V // K - 1)).long().clamp_(min=1) if V >= K else 1
        index = (y[:, None] + step * torch.arange(K, device=dev)[None, :]) % V
        gaps = -torch.log(uniform(T, K).clamp_(min=1e-6)) * (8.0 / K ** 0.5)
        logits = 20.0 - torch.cumsum(gaps, dim=1)
        kept = 1 + (uniform(T, 1) * (2 * K)).long().clamp_(max=K - 1)
        absent = (torch.arange(K, device=dev)[None, :] >= kept) | dropped[:, None]
        s["teacher_index"] = index.masked_fill(absent, -1).to(torch.int32).contiguous()
        s["teacher_logits"] = logits.masked_fill(absent, -math.inf).contiguous()
    if case["mean"]:
        s["upstream"] = 0.5 + uniform(1)
    else:
        s["upstream"] = (0.5 + uniform(T)) / T
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["mode"] == "backprop":
        logits = torch.matmul(s["h"].float(), s["w"].float().t()).mul_(1.0 / case["tau"])
        s["lse"] = torch.where(_counted(s), torch.logsumexp(logits, dim=1), torch.zeros((), device="cuda"))
        del logits
    return s


def _counted(s):
    if s["case"]["op"] == "xent":
        return s["targets"] != IGNORE
    return (s["teacher_index"] >= 0).any(dim=1)


def _plain(s):
    case = s["case"]
    h, w = s["h"].float(), s["w"].float()
    scale, mode = 1.0 / case["tau"], case["mode"]
    logits = torch.matmul(h, w.t())
    logits *= scale
    counted = _counted(s)
    if case["op"] == "xent":
        index = s["targets"].long().clamp(min=0)[:, None]
        p = counted[:, None].float()
        entropy = torch.zeros_like(p)
        factor = 1.0
    else:
        index = s["teacher_index"].long().clamp(min=0)
        there = s["teacher_index"] >= 0
        t = torch.where(there, s["teacher_logits"] * scale, -torch.inf)
        t = t - torch.where(counted, t.amax(dim=1), 0.0)[:, None]
        e = torch.exp(t)
        total = torch.where(counted, e.sum(dim=1), 1.0)[:, None]
        p = e / total
        entropy = torch.where(there, p * (t - torch.log(total)), 0.0)
        factor = case["tau"] ** 2
    out = {}
    if mode == "backprop":
        lse = s["lse"]
    else:
        top = logits.amax(dim=1)
        lse = top + torch.log(torch.exp(logits - top[:, None]).sum(dim=1))
        picked = torch.gather(logits, 1, index)
        loss = factor * (lse + (entropy - torch.where(p > 0, p * picked, 0.0)).sum(dim=1))
        loss = torch.where(counted, loss, 0.0)
        out["loss"] = loss.sum() / counted.sum() if case["mean"] else loss
        out["lse"] = torch.where(counted, lse, 0.0)
    if mode != "score":
        upstream = s["upstream"] / counted.sum() if case["mean"] else s["upstream"]
        g = torch.where(counted, upstream * (factor * scale), 0.0)[:, None]
        grad = torch.exp(logits - lse[:, None])
        grad.scatter_add_(1, index, -p)
        grad *= g
        out["dh"] = torch.matmul(grad, w).to(s["h"].dtype)
        out["dw"] = torch.matmul(grad.t(), h).to(s["w"].dtype)
    return out


def _kernels(s):
    from strideweave_b200 import kernels

    case, h, w = s["case"], s["h"], s["w"]
    mode = case["mode"]
    out, grads = {}, {}
    if mode == "backprop":
        lse, loss = s["lse"], None
    else:
        lse = out["lse"] = torch.empty(case["T"], dtype=torch.float32, device=h.device)
        loss = out["loss"] = torch.empty(() if case["mean"] else case["T"], dtype=torch.float32, device=h.device)
    if mode != "score":
        dh, dw = torch.empty(h.shape, dtype=h.dtype, device=h.device), torch.empty_like(w)
        out["dh"], out["dw"] = dh, dw
        grads = dict(upstream_ptr=s["upstream"].data_ptr(), dh_ptr=dh.data_ptr(), dh_strides=dh.stride(),
                     dw_ptr=dw.data_ptr(), dw_strides=dw.stride())
    common = dict(loss_ptr=loss.data_ptr() if loss is not None else 0, lse_ptr=lse.data_ptr(),
                  reduction="mean" if case["mean"] else "none", stream=torch.cuda.current_stream().cuda_stream, **grads)
    head = ("BFloat16" if case["dtype"] == "bf16" else "Float32", h.data_ptr(), h.stride(), w.data_ptr(), w.stride(),
            case["T"], case["V"], case["D"])
    if case["op"] == "xent":
        kernels.linear_cross_entropy(*head, s["targets"].data_ptr(), ignore_index=IGNORE, **common)
    else:
        kernels.linear_distillation(*head, s["teacher_index"].data_ptr(), s["teacher_logits"].data_ptr(), case["K"],
                                    temperature=case["tau"], **common)
    return out


def run(state):
    return _kernels(state) if own else _plain(state)


def work(case):
    T, V, D, K = case["T"], case["V"], case["D"], case["K"]
    size = 2 if case["dtype"] == "bf16" else 4
    rows = T if case["keep"] == 1.0 else max(1, round(T * case["keep"]))  # rows that count
    grads = case["mode"] != "score"
    nbytes = size * (rows * D + V * D) + 8 * T + (4 if case["op"] == "xent" else 8 * K) * T
    if grads:
        nbytes += size * (T * D + V * D)
    return {"bytes": nbytes, "flops": (6 if grads else 2) * rows * V * D}


def exact(case, seed):
    """The definition in binary64, a block of rows at a time."""
    s = prepare(case, seed)
    tau, T, D = case["tau"], case["T"], case["D"]
    w = s["w"].double()
    f64 = dict(dtype=torch.float64, device=w.device)
    loss, lse_all = torch.zeros(T, **f64), torch.zeros(T, **f64)
    dh, dw = torch.zeros(T, D, **f64), torch.zeros(w.shape, **f64)
    if case["op"] == "xent":
        entries = s["targets"].long()[:, None]
        valid = entries != IGNORE
        weight = valid.double()
        own_entropy = torch.zeros(T, **f64)
    else:
        entries = s["teacher_index"].long()
        valid = entries >= 0
        raw = s["teacher_logits"].double() / tau
        raw[~valid] = -math.inf
        weight = torch.nan_to_num(torch.softmax(raw, dim=1), nan=0.0)
        own_entropy = torch.xlogy(weight, weight).sum(dim=1)
    rows = valid.any(dim=1).nonzero()[:, 0]
    up = s["upstream"].double()
    up = (up / len(rows)).expand(T) if case["mean"] else up
    for block in rows.split(1024):
        z = s["h"][block].double() @ w.t() / tau
        lse = s["lse"][block].double() if case["mode"] == "backprop" else torch.logsumexp(z, dim=1)
        q = torch.zeros_like(z)
        q.scatter_add_(1, entries[block].clamp(min=0), weight[block])
        lse_all[block] = lse
        loss[block] = tau ** 2 * (own_entropy[block] + lse - torch.where(q > 0, q * z, 0.0).sum(dim=1))
        if case["mode"] != "score":
            q.neg_().add_(torch.exp(z.sub_(lse[:, None])))
            q.mul_((up[block] * tau)[:, None])
            dh[block] = q @ w
            dw += q.t() @ s["h"][block].double()
    out = {}
    if case["mode"] != "backprop":
        out["loss"] = loss.sum() / len(rows) if case["mean"] else loss
        out["lse"] = lse_all
    if case["mode"] != "score":
        out["dh"], out["dw"] = dh, dw
    return out
