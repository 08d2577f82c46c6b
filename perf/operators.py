"""Vocabulary losses measured: cross entropy and per-token log-probabilities taken
straight from hidden states and the output projection, and distillation from a
teacher's top logits.

Three operators, with N tokens, D hidden units, V vocabulary entries:

    z = hidden @ weight.T                       (N, V), held nowhere
    linear_cross_entropy:          mean_i / sum_i / each  lse(z_i) - z_i[t_i] + z_loss * lse(z_i)^2
    linear_selective_log_softmax:  z_i[t_i] - lse(z_i)
    topk_distillation_loss:        T^2 * KL(p_i || softmax(logits_i / T)), p_i the softmax of the
                                   teacher's kept logits / T; entries of index -1 are padding

`run` makes one pass: the loss, and in training its gradients too.
"""
import math

import torch

own = False

IGNORE = -100

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def _ce(name, n, d, v, dtype, ignored, reduction, z_loss, upstream):
    case = {"op": "ce", "n": n, "d": d, "v": v, "dtype": dtype, "ignored": ignored,
            "reduction": reduction, "z_loss": z_loss, "upstream": upstream}
    return dict(case, name=name) if name else case


def _logp(name, b, t, d, v, dtype, train):
    case = {"op": "logp", "b": b, "t": t, "d": d, "v": v, "dtype": dtype, "train": train}
    return dict(case, name=name) if name else case


def _distill(name, n, v, k, dtype, temperature, padded, reduction, train):
    case = {"op": "distill", "n": n, "v": v, "k": k, "dtype": dtype, "temperature": temperature,
            "padded": padded, "reduction": reduction, "train": train}
    return dict(case, name=name) if name else case


def listed():
    return [
        # a fine-tuning step of 8192 tokens, a quarter of them prompt tokens without a target
        _ce("ce_train_8192x4096x128256_bf16", 8192, 4096, 128256, "bf16", 0.25, "mean", 0.0, 1.0),
        # mixed-precision training under loss scaling with the log-normaliser held near zero
        _ce("ce_train_2048x2048x50257_fp16", 2048, 2048, 50257, "fp16", 0.0, "mean", 1e-4, 4096.0),
        # a ragged batch whose tokens carry weights of their own, odd vocabulary, half padding
        _ce("ce_train_1023x1000x32003_bf16", 1023, 1000, 32003, "bf16", 0.5, "none", 0.0, 1.0),
        # one small microbatch: latency
        _ce("ce_train_48x256x4099_bf16", 48, 256, 4099, "bf16", 0.0, "mean", 0.0, 1.0),
        # scoring one generated token while serving
        _logp("logp_1x1x4096x128256_bf16", 1, 1, 4096, 128256, "bf16", False),
        # scoring finished rollouts: every token but the last of each sequence predicts the next
        _logp("logp_4x1023x2048x128256_bf16", 4, 1023, 2048, 128256, "bf16", False),
        # scoring a batch of generated tokens
        _logp("logp_17x1x1024x50257_fp16", 17, 1, 1024, 50257, "fp16", False),
        # a policy-gradient step: one upstream weight for each token
        _logp("logp_train_2x511x2048x32000_bf16", 2, 511, 2048, 32000, "bf16", True),
        # distillation steps
        _distill("distill_train_2048x128256_bf16_k64", 2048, 128256, 64, "bf16", 1.0, 0.1, "mean", True),
        _distill("distill_train_512x128256_fp32_k32", 512, 128256, 32, "fp32", 2.0, 0.0, "mean", True),
        _distill("distill_train_333x50257_fp16_k100", 333, 50257, 100, "fp16", 1.5, 0.25, "none", True),
        # validation on a few tokens
        _distill("distill_eval_4x128256_fp32_k20", 4, 128256, 20, "fp32", 1.0, 0.0, "sum", False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(n, d, v):
    return n * d * v


def draw(rng):
    limit = 8192 * 4096 * 128256 * 0.75
    op = rng.choice(["ce", "ce", "logp", "logp", "distill", "distill"])
    if op == "ce":
        while True:
            n, v = _log_int(rng, 1, 8192), _log_int(rng, 1000, 128256)
            d = _log_int(rng, 64, 8192)
            d = d if rng.random() < 0.15 else max(64, d // 8 * 8)
            ignored = rng.choice([0.0, 0.0, 0.1, 0.25, 0.5, 0.9])
            # the fp32 logits of the plain form hold n * v elements
            if _cost(n, d, v) * (1 - ignored) <= limit and v * d <= 128256 * 4096:
                break
        reduction = rng.choice(["mean", "mean", "sum", "none"])
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        # 16-bit floats with few exponent bits are trained under loss scaling
        upstream = 4096.0 if dtype == "fp16" else rng.choice([1.0, 0.125, 1024.0])
        return _ce(None, n, d, v, dtype, ignored, reduction, rng.choice([0.0, 0.0, 1e-4, 1e-2]), upstream)
    if op == "logp":
        train = rng.random() < 0.4
        while True:
            b, t = rng.choice([1, 2, 3, 4, 8]), _log_int(rng, 1, 1023)
            v = _log_int(rng, 1000, 128256)
            d = max(64, _log_int(rng, 64, 8192) // 8 * 8)
            if _cost(b * t, d, v) <= limit / 8 and v * d <= 128256 * 4096:
                break
        return _logp(None, b, t, d, v, rng.choice(["bf16", "bf16", "fp16"]), train)
    while True:
        n, v = _log_int(rng, 1, 4096), _log_int(rng, 1000, 128256)
        if n * v <= 2048 * 128256:
            break
    return _distill(None, n, v, _log_int(rng, 1, 256), rng.choice(["bf16", "fp16", "fp32"]),
                    rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]), rng.choice([0.0, 0.1, 0.25]),
                    rng.choice(["mean", "sum", "none"]), rng.random() < 0.75)


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------
def _zipf(n, v, g):
    """Token ids whose frequency falls with their rank, over the whole vocabulary."""
    u = torch.rand(n, device="cuda", generator=g)
    return (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1)


def _projection(n, d, v, dtype, g):
    """Normalised hidden states, an output projection that gives logits a spread of
    about two, targets, and a pull of some tokens toward their target, from tokens
    that the model has no idea of to tokens that it is sure of."""
    weight = (torch.randn(v, d, device="cuda", generator=g) * (2.0 / math.sqrt(d))).to(dtype)
    target = _zipf(n, v, g)
    hidden = torch.randn(n, d, device="cuda", generator=g)
    pull = 3.0 * torch.rand(n, 1, device="cuda", generator=g)
    hidden = (hidden + pull * weight[target].float()).to(dtype)
    return hidden, weight, target


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "ce":
        n = case["n"]
        hidden, weight, target = _projection(n, case["d"], case["v"], dtype, g)
        dropped = torch.rand(n, device="cuda", generator=g) < case["ignored"]
        dropped[0] = False
        target = torch.where(dropped, torch.full_like(target, IGNORE), target)
        if case["reduction"] == "none":
            upstream = torch.rand(n, device="cuda", generator=g) * case["upstream"] / n
        else:
            # a summed loss is brought to a mean by its caller
            share = 1.0 if case["reduction"] == "mean" else 1.0 / n
            upstream = torch.full((), case["upstream"] * share, device="cuda")
        return {"case": case, "hidden": hidden.requires_grad_(), "weight": weight.requires_grad_(),
                "target": target, "upstream": upstream}
    if case["op"] == "logp":
        b, t, d, v = case["b"], case["t"], case["d"], case["v"]
        hidden, weight, index = _projection(b * t, d, v, dtype, g)
        # the rows of a (b, t + 1, d) tensor without each sequence's last token
        full = torch.zeros(b, t + 1, d, device="cuda", dtype=dtype)
        full[:, :t] = hidden.view(b, t, d)
        hidden = full[:, :t]
        scale = 4096.0 if case["dtype"] == "fp16" else 1.0
        upstream = torch.randn(b, t, device="cuda", generator=g) * (scale / (b * t))
        if case["train"]:
            hidden.requires_grad_()
            weight.requires_grad_()
        return {"case": case, "hidden": hidden, "weight": weight, "index": index.view(b, t),
                "upstream": upstream}
    n, v, k = case["n"], case["v"], case["k"]
    student = 2.0 * torch.randn(n, v, device="cuda", generator=g)
    teacher = torch.randn(n, v, device="cuda", generator=g).mul_(1.5).add_(student, alpha=0.7)
    top, index = torch.topk(teacher, min(k, v), dim=-1)
    del teacher
    top = 1.5 * top
    # some rows keep fewer than k entries, and padding tokens keep none
    keep = torch.full((n, 1), k, device="cuda")
    short = torch.rand(n, 1, device="cuda", generator=g) < case["padded"]
    keep = torch.where(short, (torch.rand(n, 1, device="cuda", generator=g) * k).long(), keep)
    keep[0] = k
    index = torch.where(torch.arange(k, device="cuda") < keep, index, torch.full_like(index, -1))
    logits = student.to(dtype)
    del student
    # fp16 gradients are taken under loss scaling: about 256 for each row
    each = 256.0 if case["dtype"] == "fp16" else 1.0 / n
    if case["reduction"] == "none":
        upstream = torch.rand(n, device="cuda", generator=g) * each
    else:
        upstream = torch.full((), each * n if case["reduction"] == "mean" else each, device="cuda")
    if case["train"]:
        logits.requires_grad_()
    return {"case": case, "logits": logits, "teacher_logits": top.to(dtype), "teacher_index": index,
            "upstream": upstream}


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"ce": _own_ce, "logp": _own_logp, "distill": _own_distill}[op](state)
    with torch.no_grad():
        return {"ce": _plain_ce, "logp": _plain_logp, "distill": _plain_distill}[op](state)


def _own_ce(state):
    import fuselse_b200
    case = state["case"]
    hidden, weight = state["hidden"], state["weight"]
    loss = fuselse_b200.linear_cross_entropy(hidden, weight, state["target"], ignore_index=IGNORE,
                                             reduction=case["reduction"], z_loss=case["z_loss"])
    grad_hidden, grad_weight = torch.autograd.grad(loss, (hidden, weight), state["upstream"])
    return loss.detach(), grad_hidden, grad_weight


def _own_logp(state):
    import fuselse_b200
    hidden, weight = state["hidden"], state["weight"]
    logp = fuselse_b200.linear_selective_log_softmax(hidden, weight, state["index"])
    if not state["case"]["train"]:
        return logp
    grad_hidden, grad_weight = torch.autograd.grad(logp, (hidden, weight), state["upstream"])
    return logp.detach(), grad_hidden, grad_weight


def _own_distill(state):
    import fuselse_b200
    case = state["case"]
    loss = fuselse_b200.topk_distillation_loss(state["logits"], state["teacher_logits"],
                                               state["teacher_index"],
                                               temperature=case["temperature"],
                                               reduction=case["reduction"])
    if not case["train"]:
        return loss
    (grad_logits,) = torch.autograd.grad(loss, (state["logits"],), state["upstream"])
    return loss.detach(), grad_logits


def _row_lse(z):
    """Log-sum-exp of each row of z, as a column."""
    top = z.amax(dim=-1, keepdim=True)
    return top + torch.log(torch.exp(z - top).sum(dim=-1, keepdim=True))


def _plain_ce(state):
    case = state["case"]
    hidden, weight = state["hidden"].float(), state["weight"].float()
    target = state["target"]
    rows = torch.nonzero(target != IGNORE).squeeze(-1)
    kept, picked = hidden[rows], target[rows].unsqueeze(-1)
    z = kept @ weight.t()
    lse = _row_lse(z)
    each = (lse - z.gather(-1, picked) + case["z_loss"] * lse * lse).squeeze(-1)
    if case["reduction"] == "none":
        loss = torch.zeros(target.numel(), device=target.device)
        loss[rows] = each
        g = state["upstream"][rows].unsqueeze(-1)
    else:
        share = 1.0 / rows.numel() if case["reduction"] == "mean" else 1.0
        loss = (each.double().sum() * share).float()
        g = (state["upstream"] * share).expand(rows.numel(), 1)
    # d loss / d z = g * (softmax * (1 + 2 * z_loss * lse) - onehot)
    grad_z = torch.exp(z.sub_(lse)).mul_(g * (1.0 + 2.0 * case["z_loss"] * lse))
    del z
    grad_z.scatter_add_(-1, picked, -g.contiguous())
    grad_hidden = torch.zeros_like(hidden)
    grad_hidden[rows] = grad_z @ weight
    grad_weight = grad_z.t() @ kept
    dtype = state["hidden"].dtype
    return loss, grad_hidden.to(dtype), grad_weight.to(dtype)


def _plain_logp(state):
    d = state["case"]["d"]
    hidden, weight = state["hidden"].reshape(-1, d).float(), state["weight"].float()
    index = state["index"].reshape(-1, 1)
    z = hidden @ weight.t()
    lse = _row_lse(z)
    logp = (z.gather(-1, index) - lse).view(state["index"].shape)
    if not state["case"]["train"]:
        return logp
    g = state["upstream"].reshape(-1, 1)
    grad_z = torch.exp(z.sub_(lse)).mul_(-g)
    del z
    grad_z.scatter_add_(-1, index, g)
    dtype = state["hidden"].dtype
    grad_hidden = (grad_z @ weight).view(state["hidden"].shape)
    return logp, grad_hidden.to(dtype), (grad_z.t() @ hidden).to(dtype)


def _plain_distill(state):
    case = state["case"]
    temp = case["temperature"]
    z = state["logits"].float() / temp
    index = state["teacher_index"]
    kept = index >= 0
    live = kept.any(dim=-1, keepdim=True)
    t = (state["teacher_logits"].float() / temp).masked_fill(~kept, -math.inf)
    # a row without entries gets a finite stand-in and is zeroed at the end
    t = torch.where(live, t, torch.zeros_like(t))
    log_p = t - _row_lse(t)
    p = torch.where(kept, torch.exp(log_p), torch.zeros_like(t))
    lse = _row_lse(z)
    slot = index.clamp(min=0)
    gap = torch.where(kept, log_p - (z.gather(-1, slot) - lse), torch.zeros_like(p))
    each = (temp * temp * (p * gap).sum(dim=-1)) * live.squeeze(-1)
    if case["reduction"] == "none":
        loss, g = each, state["upstream"].unsqueeze(-1)
    else:
        total = each.double().sum()
        share = 1.0 / live.sum().double() if case["reduction"] == "mean" else 1.0
        loss = (total * share).float()
        g = (state["upstream"].double() * share).float().expand(z.shape[0], 1)
    if not case["train"]:
        return loss
    # d loss / d logits = g * T * (softmax(logits / T) - p)
    scale = g * temp * live
    grad = torch.exp(z.sub_(lse)).mul_(scale)
    grad.scatter_add_(-1, slot, -(p * scale))
    return loss, grad.to(state["logits"].dtype)


# --------------------------------------------------------------------------
# The definition in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.enable_grad():
        if case["op"] == "distill":
            return _exact_distill(case, state)
        return _exact_projection(case, state)


def _exact_projection(case, state):
    """Blocks of tokens, each one's gradients by automatic differentiation."""
    d = case["d"]
    hidden = state["hidden"].detach().double().reshape(-1, d)
    weight = state["weight"].detach().double()
    ce = case["op"] == "ce"
    train = ce or case["train"]
    target = (state["target"] if ce else state["index"]).reshape(-1)
    live = (target != IGNORE) if ce else torch.ones_like(target, dtype=torch.bool)
    n = target.numel()
    if not ce or case["reduction"] == "none":
        upstream = state["upstream"].double().reshape(-1)
    else:
        count = float(live.sum()) if case["reduction"] == "mean" else 1.0
        upstream = (state["upstream"].double() / count).expand(n)
    values = torch.zeros(n, dtype=torch.float64, device="cuda")
    grad_hidden = torch.zeros_like(hidden) if train else None
    grad_weight = torch.zeros_like(weight) if train else None
    block = max(1, (1 << 28) // case["v"])
    for lo in range(0, n, block):
        rows = torch.arange(lo, min(n, lo + block), device="cuda")
        rows = rows[live[rows]]
        if rows.numel() == 0:
            continue
        h = hidden[rows].requires_grad_(train)
        z = (h @ weight.t()).detach().requires_grad_(train)
        logp = torch.log_softmax(z, dim=-1)
        value = logp[torch.arange(rows.numel(), device="cuda"), target[rows]]
        if ce:
            lse = torch.logsumexp(z, dim=-1)
            value = case["z_loss"] * lse ** 2 - value
        values[rows] = value.detach()
        if train:
            (grad_z,) = torch.autograd.grad((value * upstream[rows]).sum(), (z,))
            grad_hidden[rows] = grad_z @ weight
            grad_weight += grad_z.t() @ hidden[rows]
    if not ce:
        out = values.view(state["index"].shape)
    elif case["reduction"] == "none":
        out = values
    else:
        out = values.sum() / (live.sum() if case["reduction"] == "mean" else 1.0)
    if not train:
        return out
    return out, grad_hidden.view(state["hidden"].shape), grad_weight


def _exact_distill(case, state):
    temp, n, v = case["temperature"], case["n"], case["v"]
    index = state["teacher_index"]
    z = state["logits"].detach().double().requires_grad_(case["train"])
    log_q = torch.log_softmax(z / temp, dim=-1)
    # the teacher's distribution over its kept entries, row by row in a dense table
    t = torch.full((n, v + 1), -math.inf, dtype=torch.float64, device="cuda")
    slot = torch.where(index >= 0, index, torch.full_like(index, v))
    t.scatter_(-1, slot, state["teacher_logits"].double() / temp)
    t = t[:, :v]
    live = (index >= 0).any(dim=-1)
    p = torch.softmax(t, dim=-1)
    p[~live] = 0.0
    each = temp ** 2 * (torch.special.xlogy(p, p) - p * log_q).sum(dim=-1)
    if case["reduction"] == "none":
        loss = each
    elif case["reduction"] == "sum":
        loss = each.sum()
    else:
        loss = each.sum() / live.sum()
    if not case["train"]:
        return loss.detach()
    (grad,) = torch.autograd.grad(loss, (z,), state["upstream"].double())
    return loss.detach(), grad


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    if case["op"] == "distill":
        n, v, k = case["n"], case["v"], case["k"]
        size = 4 if case["dtype"] == "fp32" else 2
        out = 4 * n if case["reduction"] == "none" else 4
        moved = n * v * size + n * k * (size + 8) + out
        if case["train"]:
            moved += n * v * size
        return {"bytes": moved, "flops": n * v * (8 if case["train"] else 4)}
    d, v = case["d"], case["v"]
    if case["op"] == "ce":
        n = case["n"]
        live = max(1, round(n * (1 - case["ignored"])))
        out = 4 * n if case["reduction"] == "none" else 4
        train = True
    else:
        n = live = case["b"] * case["t"]
        out, train = 4 * n, case["train"]
    moved = 2 * (live * d + v * d) + 8 * n + out
    flops = 2 * live * d * v
    if train:
        moved += 2 * (n * d + v * d)
        flops *= 3
    return {"bytes": moved, "flops": flops}
