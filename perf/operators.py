"""Cases, plain forms and 64-bit values of the operators on a model's output distribution.

Four operators, each forward and (where a case says so) backward:

``token_logprobs``       log-probability of given tokens, entropy and the k most likely alternatives, from logits
``distill_loss``         distillation from a teacher's top logits, from the student's logits
``head_token_logprobs``  log-probability and entropy from hidden states and the head's weight, no logits kept
``head_distill_loss``    cross-entropy, L2Wrap and distillation in one pass over the head, no logits kept

With ``own`` false :func:`run` computes them in elementary torch operations in 32 bits, with ``own`` true it makes the
calls that a user of ``rwkv7m_b200.ops`` makes.
"""

import math

import torch

own = False

L2WRAP = 1e-4
_CHUNK = 2048        # rows of [rows, vocabulary] temporaries that the plain form holds at a time
_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one sequence decoding with the log-probability of its token and five alternatives: latency of one row
        {"name": "logprobs_decode_one", "op": "token_logprobs", "rows": 1, "vocab": 65536, "dtype": "bf16",
         "top_k": 5, "temperature": 1.0, "backward": False},
        # a serving batch at a sampling temperature, twenty alternatives for each sequence
        {"name": "logprobs_serving_batch", "op": "token_logprobs", "rows": 64, "vocab": 65536, "dtype": "bf16",
         "top_k": 20, "temperature": 0.8, "backward": False},
        # a prompt's scores with alternatives from 32-bit logits over a vocabulary of odd size
        {"name": "logprobs_prompt_odd", "op": "token_logprobs", "rows": 1021, "vocab": 50021, "dtype": "fp32",
         "top_k": 10, "temperature": 1.0, "backward": False},
        # a policy-gradient step with an entropy bonus on logits that the caller holds
        {"name": "logprobs_policy_step", "op": "token_logprobs", "rows": 4096, "vocab": 65536, "dtype": "bf16",
         "top_k": 0, "temperature": 1.0, "backward": True},
        # a small student on the host model's logits: a few short sequences, small vocabulary, odd row count
        {"name": "distill_small", "op": "distill_loss", "rows": 127, "vocab": 2048, "dtype": "fp32",
         "top_k": 8, "temperature": 1.0, "backward": True},
        # a distillation step of a student whose logits exist: one sequence of 4096 tokens, 64 alternatives
        {"name": "distill_step", "op": "distill_loss", "rows": 4096, "vocab": 65536, "dtype": "bf16",
         "top_k": 64, "temperature": 2.0, "backward": True},
        # the last tokens of a few candidate answers, scored in one call: streams the head's weight once
        {"name": "head_logprobs_rerank", "op": "head_token_logprobs", "rows": 24, "vocab": 65536, "width": 1024,
         "dtype": "bf16", "temperature": 1.0, "backward": False},
        # a long document scored token by token
        {"name": "head_logprobs_document", "op": "head_token_logprobs", "rows": 8192, "vocab": 65536, "width": 2048,
         "dtype": "bf16", "temperature": 1.0, "backward": False},
        # a policy-gradient step through the head: ragged answers, packed, so an odd number of rows
        {"name": "head_logprobs_policy", "op": "head_token_logprobs", "rows": 4093, "vocab": 65536, "width": 2560,
         "dtype": "bf16", "temperature": 1.0, "backward": True},
        # the smallest configuration distilled on one sequence shorter than its context
        {"name": "head_distill_small", "op": "head_distill_loss", "rows": 509, "vocab": 65536, "width": 768,
         "dtype": "bf16", "top_k": 16, "temperature": 1.0, "backward": True},
        # four sequences of 4096 tokens of the 2048-wide model, the step that distillation runs
        {"name": "head_distill_step", "op": "head_distill_loss", "rows": 16384, "vocab": 65536, "width": 2048,
         "dtype": "bf16", "top_k": 32, "temperature": 2.0, "backward": True},
        # the widest configuration on one sequence, an odd vocabulary and many alternatives
        {"name": "head_distill_wide", "op": "head_distill_loss", "rows": 4096, "vocab": 65529, "width": 4096,
         "dtype": "bf16", "top_k": 128, "temperature": 2.0, "backward": True},
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["token_logprobs", "distill_loss", "head_token_logprobs", "head_distill_loss"])
    temperature = rng.choice([1.0, 1.0, round(rng.uniform(0.5, 3.0), 2)])
    if op == "token_logprobs":
        backward = rng.random() < 0.4
        vocab = _log_uniform(rng, 1000, 65536)
        rows = _log_uniform(rng, 1, 4096)
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "fp32"]),
                "top_k": rng.choice([0, rng.randint(1, 32)]), "temperature": temperature, "backward": backward}
    if op == "distill_loss":
        return {"op": op, "rows": _log_uniform(rng, 16, 4096), "vocab": _log_uniform(rng, 2000, 65536),
                "dtype": rng.choice(["bf16", "fp32"]), "top_k": _log_uniform(rng, 4, 128), "temperature": temperature,
                "backward": True}
    width = 64 * _log_uniform(rng, 8, 64)
    vocab = _log_uniform(rng, 8000, 65536)
    if op == "head_token_logprobs":
        backward = rng.random() < 0.5
        rows = _log_uniform(rng, 1, 8192)
        return {"op": op, "rows": rows, "vocab": vocab, "width": width, "dtype": "bf16", "temperature": temperature,
                "backward": backward}
    return {"op": op, "rows": _log_uniform(rng, 100, 8192), "vocab": vocab, "width": width, "dtype": "bf16",
            "top_k": _log_uniform(rng, 4, 128), "temperature": temperature, "backward": True}


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _tokens(gen, rows, vocab):
    """Token ids with the skew of a text corpus: low ids are frequent, every id occurs."""
    u = torch.rand(rows, generator=gen, device="cuda")
    return (u * u * u * vocab).long().clamp_(max=vocab - 1)


def _logits(gen, rows, vocab, dtype, target):
    """Logits of a language model: a slope over the vocabulary, noise, and the seen token ahead in most rows."""
    out = torch.empty(rows, vocab, dtype=dtype, device="cuda")
    slope = -0.6 * torch.log1p(torch.arange(vocab, device="cuda", dtype=torch.float32))
    for s in range(0, rows, _CHUNK):
        e = min(rows, s + _CHUNK)
        z = torch.randn(e - s, vocab, generator=gen, device="cuda").mul_(2.0).add_(slope)
        boost = torch.rand(e - s, 1, generator=gen, device="cuda").mul_(9.0)
        z.scatter_add_(1, target[s:e, None], boost)
        out[s:e] = z.to(dtype)
    return out


def _teacher(gen, rows, vocab, k, dtype):
    """A teacher's alternatives: ids skewed like tokens, logits in falling order, one row in 16 cut short (id -1) and one
    in 64 without any."""
    j = torch.arange(k, device="cuda", dtype=torch.float32)
    u = (j + torch.rand(rows, k, generator=gen, device="cuda")) / k
    ids = (u * u * vocab).long().clamp_(max=vocab - 1)
    order = torch.rand(rows, k, generator=gen, device="cuda").argsort(dim=1)
    ids = ids.gather(1, order)
    steps = torch.rand(rows, k, generator=gen, device="cuda").clamp_(min=1e-4).log().neg_().mul_(6.0 / (1.0 + j))
    logits = 14.0 - steps.cumsum(dim=1)
    kept = torch.full((rows, 1), k, device="cuda", dtype=torch.long)
    short = torch.rand(rows, 1, generator=gen, device="cuda")
    some = torch.randint(0, k, (rows, 1), generator=gen, device="cuda")
    kept = torch.where(short < 1 / 16, some, kept)
    kept = torch.where(short < 1 / 64, torch.zeros_like(kept), kept)
    ids = torch.where(torch.arange(k, device="cuda")[None, :] < kept, ids, torch.full_like(ids, -1))
    return ids.to(torch.int32), logits.to(dtype)


def _mask(gen, rows):
    """Rows that count: padding and prompt rows, a twelfth of all, do not."""
    return (torch.rand(rows, generator=gen, device="cuda") > 1 / 12).float()


def prepare(case, seed):
    gen = _generator(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], _DTYPES[case["dtype"]]
    target = _tokens(gen, rows, vocab)
    st = {"case": case, "ids": target.to(torch.int32)}
    if case["op"] in ("token_logprobs", "distill_loss"):
        st["logits"] = _logits(gen, rows, vocab, dtype, target)
    else:
        C = case["width"]
        w = torch.empty(vocab, C, dtype=dtype, device="cuda")
        for s in range(0, vocab, 8192):
            e = min(vocab, s + 8192)
            w[s:e] = (torch.randn(e - s, C, generator=gen, device="cuda") * (2.0 / math.sqrt(C))).to(dtype)
        # a layer norm's output that leans towards the seen token's row of the head in most rows
        lean = torch.rand(rows, 1, generator=gen, device="cuda") * 2.5
        h = torch.randn(rows, C, generator=gen, device="cuda") + lean * w[target].float()
        st["hidden"] = (h * torch.rsqrt(h.square().mean(dim=1, keepdim=True))).to(dtype)
        st["weight"] = w
    if case["op"] in ("distill_loss", "head_distill_loss"):
        st["mask"] = _mask(gen, rows)
        # stored teachers come in 16 bits beside a 16-bit student
        st["teacher_ids"], st["teacher_logits"] = _teacher(gen, rows, vocab, case["top_k"], dtype)
    elif case["backward"]:
        # advantages and the entropy bonus's weight, averaged over the rows
        st["g_logprob"] = -torch.randn(rows, generator=gen, device="cuda") / rows
        st["g_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda")
    return st


# ---- one pass ------------------------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    from rwkv7m_b200 import ops

    case = st["case"]
    tau = case["temperature"]
    grad = case["backward"]
    if case["op"] == "token_logprobs":
        z = st["logits"].detach().requires_grad_(grad)
        out = ops.token_logprobs(z, st["ids"], top_k=case["top_k"], temperature=tau)
        res = {"logprob": out.logprob.detach(), "entropy": out.entropy.detach()}
        if case["top_k"]:
            res["top_ids"], res["top_logprobs"] = out.top_ids, out.top_logprobs.detach()
        if grad:
            res["dlogits"], = torch.autograd.grad((out.logprob, out.entropy), (z,), (st["g_logprob"], st["g_entropy"]))
        return res
    if case["op"] == "distill_loss":
        z = st["logits"].detach().requires_grad_(grad)
        kd, count = ops.distill_loss(z, st["teacher_ids"], st["teacher_logits"], st["mask"], temperature=tau)
        dz, = torch.autograd.grad(kd / count.clamp(min=1.0), (z,))
        return {"kd_total": kd.detach(), "kd_count": count, "dlogits": dz}
    h = st["hidden"].detach().requires_grad_(grad)
    w = st["weight"].detach().requires_grad_(grad)
    if case["op"] == "head_token_logprobs":
        logprob, entropy = ops.head_token_logprobs(h, w, st["ids"], temperature=tau)
        res = {"logprob": logprob.detach(), "entropy": entropy.detach()}
        if grad:
            res["dhidden"], res["dweight"] = torch.autograd.grad((logprob, entropy), (h, w),
                                                                 (st["g_logprob"], st["g_entropy"]))
        return res
    ce, ce_n, l2, l2_n, kd, kd_n = ops.head_distill_loss(h, w, st["ids"], st["mask"], st["teacher_ids"],
                                                         st["teacher_logits"], temperature=tau)
    loss = 0.5 * ce / ce_n.clamp(min=1.0) + 0.5 * kd / kd_n.clamp(min=1.0) + l2 / l2_n
    dh, dw = torch.autograd.grad(loss, (h, w))
    return {"ce_total": ce.detach(), "ce_count": ce_n, "l2_total": l2.detach(), "l2_count": l2_n,
            "kd_total": kd.detach(), "kd_count": kd_n, "dhidden": dh, "dweight": dw}


def _top_plain(z, k):
    """Ids of the k largest entries of each row, ties to the lowest index: the value's bits in an order that integers
    share, the index below them."""
    bits = (z + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = (bits.long() << 32) | (0xFFFFFFFF - torch.arange(z.shape[1], device=z.device))
    top = torch.topk(key, k, dim=1).values
    return 0xFFFFFFFF - (top & 0xFFFFFFFF)


def _softmax_parts(z):
    """Row maximum taken out, exponentials, their sum, and the logarithm of the sum of exponentials, in 32 bits."""
    m = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - m)
    s = e.sum(dim=1, keepdim=True)
    return e / s, m + torch.log(s)


def _logprob_rows(z, ids, tau, g_lp, g_h):
    """Log-probability, entropy and (with upstream gradients) the gradient with respect to these rows of logits."""
    zt = z / tau
    p, lse = _softmax_parts(zt)
    logp = zt - lse
    lp = logp.gather(1, ids[:, None])
    h = -(p * logp).sum(dim=1, keepdim=True)
    dz = None
    if g_lp is not None:
        g_lp, g_h = g_lp[:, None], g_h[:, None]
        dz = p * (-g_lp - g_h * (logp + h))
        dz.scatter_add_(1, ids[:, None], g_lp)
        dz = dz / tau
    return lp[:, 0], h[:, 0], dz


def _teacher_weights(ids, logits, vocab, tau):
    """The teacher's distribution over its alternatives, absent ones at zero; rows without any are all zero."""
    there = (ids >= 0) & (ids < vocab)
    x = torch.where(there, logits.float() / tau, torch.full_like(logits, -math.inf, dtype=torch.float32))
    m = x.max(dim=1, keepdim=True).values
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(x - m)
    return e / e.sum(dim=1, keepdim=True).clamp(min=1e-30), torch.where(there, ids, torch.zeros_like(ids)).long()


def _distill_rows(z, t_ids, t_logits, mask, tau):
    """Masked distillation loss of these rows and its gradient for a unit upstream gradient."""
    p_t, idx = _teacher_weights(t_ids, t_logits, z.shape[1], tau)
    zt = z / tau
    q, lse = _softmax_parts(zt)
    logq = zt.gather(1, idx) - lse
    logp = torch.log(p_t.clamp(min=1e-38))
    row = (p_t * (logp - logq)).sum(dim=1) * (tau * tau)
    dz = q * p_t.sum(dim=1, keepdim=True)
    dz.scatter_add_(1, idx, -p_t)
    return (row * mask).sum(), dz * (tau * mask[:, None])


def _run_plain(st):
    case = st["case"]
    tau, rows = case["temperature"], case["rows"]
    head = case["op"].startswith("head")
    dtype = _DTYPES[case["dtype"]]
    ids = st["ids"].long()
    parts = {}

    def keep(name, value):
        parts.setdefault(name, []).append(value)

    w32 = st["weight"].float() if head else None
    dw = torch.zeros_like(w32) if head and case["backward"] else None
    count = st["mask"].sum() if "mask" in st else None
    for s in range(0, rows, _CHUNK):
        e = min(rows, s + _CHUNK)
        if head:
            h32 = st["hidden"][s:e].float()
            z = h32 @ w32.t()
        else:
            z = st["logits"][s:e].float()
        if "logprobs" in case["op"]:
            g_lp = st["g_logprob"][s:e] if case["backward"] else None
            g_h = st["g_entropy"][s:e] if case["backward"] else None
            lp, ent, dz = _logprob_rows(z, ids[s:e], tau, g_lp, g_h)
            keep("logprob", lp)
            keep("entropy", ent)
            if case.get("top_k"):
                top = _top_plain(z, case["top_k"])
                keep("top_ids", top.to(torch.int32))
                keep("top_logprobs", z.gather(1, top) / tau - _softmax_parts(z / tau)[1])
        else:
            kd, dz = _distill_rows(z, st["teacher_ids"][s:e], st["teacher_logits"][s:e], st["mask"][s:e], tau)
            keep("kd_total", kd)
            if head:
                dz = dz * (0.5 / count.clamp(min=1.0))
                p, lse = _softmax_parts(z)
                mx, am = z.max(dim=1, keepdim=True)
                keep("ce_total", ((lse - z.gather(1, ids[s:e, None]))[:, 0] * st["mask"][s:e]).sum())
                keep("l2_total", 0.5 * L2WRAP * mx.square().sum())
                g = st["mask"][s:e, None] * (0.5 / count.clamp(min=1.0))
                dz += p * g
                dz.scatter_add_(1, ids[s:e, None], -g)
                dz.scatter_add_(1, am, (L2WRAP / rows) * mx)
            else:
                dz = dz / count.clamp(min=1.0)
        if dz is not None:
            if head:
                keep("dhidden", (dz @ w32).to(dtype))
                dw += dz.t() @ h32
            else:
                keep("dlogits", dz.to(dtype))
    res = {k: (torch.stack(v).sum() if k.endswith("_total") else torch.cat(v)) for k, v in parts.items()}
    if dw is not None:
        res["dweight"] = dw.to(dtype)
    if count is not None:
        res["kd_count"] = count
        if head:
            res["ce_count"] = count.clone()
            res["l2_count"] = torch.full_like(count, float(rows))
    if case["op"] == "head_distill_loss":
        order = ("ce_total", "ce_count", "l2_total", "l2_count", "kd_total", "kd_count", "dhidden", "dweight")
        return {k: res[k] for k in order}
    if case["op"] == "distill_loss":
        return {k: res[k] for k in ("kd_total", "kd_count", "dlogits")}
    return res


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    k = case.get("top_k", 0)
    distill = case["op"] in ("distill_loss", "head_distill_loss")
    # ids or alternatives in, per-row results out (or the mask and a few scalars)
    small = rows * (k * (4 + size) + 8) if distill else rows * (4 + 8 + 8 * k + (8 if case["backward"] else 0))
    passes = 2 if case["backward"] else 1
    if case["op"].startswith("head"):
        C = case["width"]
        # three products: logits, gradient of the hidden states, gradient of the weight
        return {"bytes": passes * size * (rows * C + vocab * C) + small,
                "flops": (6 if case["backward"] else 2) * rows * vocab * C}
    # per element: shift, scale, exponential, two sums; and as many for the gradient
    return {"bytes": passes * size * rows * vocab + small, "flops": 5 * passes * rows * vocab}


# ---- 64-bit values ---------------------------------------------------------------------------------------------------------


def exact(case, seed):
    """From the definitions, by automatic differentiation in 64 bits, a few rows at a time."""
    st = prepare(case, seed)
    rows, tau, vocab = case["rows"], float(case["temperature"]), case["vocab"]
    step = max(1, min(rows, (1 << 26) // vocab))
    head, grad = case["op"].startswith("head"), case["backward"]
    w = st["weight"].double().requires_grad_(grad) if head else None
    dw = torch.zeros_like(w) if head and grad else None
    out = {}
    weight_sum = st["mask"].double().sum() if "mask" in st else None
    for s in range(0, rows, step):
        rng = slice(s, min(rows, s + step))
        leaf = (st["hidden"] if head else st["logits"])[rng].double().requires_grad_(grad)
        z = leaf @ w.T if head else leaf
        ids = st["ids"][rng].long()[:, None]
        logq = torch.log_softmax(z / tau, dim=-1)
        if case["op"].endswith("token_logprobs"):
            got = {"logprob": logq.gather(1, ids)[:, 0], "entropy": -(logq.exp() * logq).sum(-1)}
            if case.get("top_k"):
                order = torch.sort(z.detach(), dim=-1, descending=True, stable=True).indices[:, : case["top_k"]]
                got["top_ids"], got["top_logprobs"] = order.to(torch.int32), logq.gather(1, order)
            if grad:
                loss = (got["logprob"] * st["g_logprob"][rng].double()).sum() + \
                       (got["entropy"] * st["g_entropy"][rng].double()).sum()
        else:
            t_ids = st["teacher_ids"][rng].long()
            t = st["teacher_logits"][rng].double() / tau
            absent = t_ids < 0
            logp = torch.log_softmax(t.masked_fill(absent, -1e300), dim=-1)
            p = logp.exp().masked_fill(absent, 0.0)
            diff = logp.masked_fill(absent, 0.0) - logq.gather(1, t_ids.clamp(min=0))
            m = st["mask"][rng].double()
            got = {"kd_total": (tau * tau * (p * diff).sum(-1) * m).sum()}
            loss = got["kd_total"] / weight_sum.clamp(min=1.0)
            if head:
                got["ce_total"] = -(torch.log_softmax(z, dim=-1).gather(1, ids)[:, 0] * m).sum()
                got["l2_total"] = 0.5 * L2WRAP * z.amax(dim=-1).square().sum()
                loss = 0.5 * loss + 0.5 * got["ce_total"] / weight_sum.clamp(min=1.0) + got["l2_total"] / rows
        if grad:
            if head:
                dleaf, dwp = torch.autograd.grad(loss, (leaf, w))
                dw += dwp
                got["dhidden"] = dleaf
            else:
                got["dlogits"], = torch.autograd.grad(loss, (leaf,))
        for name, value in got.items():
            out.setdefault(name, []).append(value.detach())
    res = {k: (torch.stack(v).sum() if k.endswith("_total") else torch.cat(v)) for k, v in out.items()}
    if case["op"] == "head_distill_loss":
        return {"ce_total": res["ce_total"], "ce_count": weight_sum, "l2_total": res["l2_total"],
                "l2_count": torch.tensor(float(rows), dtype=torch.float64, device=weight_sum.device),
                "kd_total": res["kd_total"], "kd_count": weight_sum, "dhidden": res["dhidden"], "dweight": dw}
    if case["op"] == "distill_loss":
        return {"kd_total": res["kd_total"], "kd_count": weight_sum, "dlogits": res["dlogits"]}
    if dw is not None:
        res["dweight"] = dw
    return res
