"""Performance cases of the vocabulary-sized losses: cross entropy and top-k distillation straight from the hidden states (the logits are
never kept) and top-k distillation on given logits.

``run`` computes a case in its plain form (elementary torch operations in 32 bits), or, where ``own`` is true, through the framework's
operators (``deeplearning4j_amd.ops.vocab_loss``). ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# most work of a listed case: N * D * V of the largest training step, N * V of the largest given logits
MOST_NDV = 8192 * 2048 * 65536
MOST_NV = 8192 * 65536


def _linear(name, op, n, d, v, dtype, train, bias=False, layout="vd", ignored=0.0, smoothing=0.0, k=0, temperature=1.0):
    return {"name": name, "op": op, "n": n, "d": d, "v": v, "dtype": dtype, "train": train, "bias": bias, "layout": layout,
            "ignored": ignored, "smoothing": smoothing, "k": k, "temperature": temperature}


def listed():
    return [
        # the score of one generated token: one row against the whole word table (vocabulary and width of the BERT configuration)
        _linear("ce_score_one_token", "ce", 1, 768, 30522, "bf16", False, bias=True),
        # perplexity of a short text
        _linear("ce_score_text", "ce", 512, 1024, 50001, "bf16", False),
        # masked-LM step on 32 x 128 tokens: 85 % of the positions carry no label; width and vocabulary of the BERT configuration
        _linear("ce_train_masked", "ce", 4096, 768, 30522, "bf16", True, bias=True, ignored=0.85),
        # character model: a small fp32 output layer [nIn, nOut] as the recurrent networks keep it, odd vocabulary
        _linear("ce_train_char_fp32", "ce", 1600, 512, 98, "fp32", True, bias=True, layout="dv"),
        # word-level model in the framework's default type
        _linear("ce_train_fp32", "ce", 2048, 768, 30522, "fp32", True),
        # ragged batch in half precision with smoothed labels, odd sizes everywhere
        _linear("ce_train_ragged_fp16", "ce", 3001, 1000, 50001, "fp16", True, bias=True, ignored=0.3, smoothing=0.1),
        # a large step: 8192 tokens, 65536 words
        _linear("ce_train_large", "ce", 8192, 2048, 65536, "bf16", True),
        # student step against a teacher's 64 best words
        _linear("distil_train", "distil", 4096, 1024, 32000, "bf16", True, k=64, temperature=2.0),
        # small distillation batch in the default type, some rows without teacher entries
        _linear("distil_train_small_fp32", "distil", 96, 768, 30522, "fp32", True, bias=True, ignored=0.2, k=8, temperature=1.5),
        # the same loss where the network has its logits already
        {"name": "distil_logits_small", "op": "distil_logits", "n": 64, "v": 1000, "dtype": "fp32", "train": True, "ignored": 0.0, "k": 16,
         "temperature": 1.0},
        {"name": "distil_logits_train", "op": "distil_logits", "n": 4096, "v": 30522, "dtype": "bf16", "train": True, "ignored": 0.2, "k": 64,
         "temperature": 2.0},
        {"name": "distil_logits_large", "op": "distil_logits", "n": 8192, "v": 65536, "dtype": "bf16", "train": True, "ignored": 0.0, "k": 128,
         "temperature": 4.0},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "distil", "distil_logits"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    v = _log_uniform(rng, 98, 65536)
    ignored = rng.choice([0.0, 0.0, 0.3, 0.85])
    k = min(_log_uniform(rng, 4, 128), v // 2)
    temperature = rng.choice([1.0, 1.5, 2.0, 4.0])
    if op == "distil_logits":
        n = min(_log_uniform(rng, 1, 8192), MOST_NV // v)
        return {"op": op, "n": n, "v": v, "dtype": dtype, "train": rng.random() < 0.7, "ignored": ignored, "k": k, "temperature": temperature}
    d = _log_uniform(rng, 64, 4096)
    if rng.random() < 0.75:
        d = (d + 7) // 8 * 8                                    # most models; the others keep an odd width
    n = _log_uniform(rng, 1, 8192)
    # fp32 products cost the plain form and the kernels several times as much as 16-bit ones
    n = max(1, min(n, (MOST_NDV // (8 if dtype == "fp32" else 1)) // (d * v)))
    case = _linear("", op, n, d, v, dtype, rng.random() < 0.7, bias=rng.random() < 0.5, layout=rng.choice(["vd", "vd", "dv"]),
                   ignored=ignored, smoothing=rng.choice([0.0, 0.0, 0.1]) if op == "ce" else 0.0,
                   k=k if op == "distil" else 0, temperature=temperature if op == "distil" else 1.0)
    del case["name"]
    return case


def _teacher(case, gen, dev):
    """Indices of a teacher's k best words (distinct, in no order of the vocabulary's) and their logits, best first; rows without
    entries are filled with -1."""
    n, v, k = case["n"], case["v"], case["k"]
    step = torch.randint(1, max(2, v // k), (n, k), generator=gen, device=dev)
    idx = (torch.randint(0, v, (n, 1), generator=gen, device=dev) + step.cumsum(1)) % v
    t = 9.0 - torch.rand(n, k, generator=gen, device=dev).mul_(0.5).cumsum(1)
    if case["ignored"]:
        idx[torch.rand(n, generator=gen, device=dev) < case["ignored"]] = -1
    return idx, t


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt, n, v = DTYPES[case["dtype"]], case["n"], case["v"]
    s = {"case": case}
    if case["op"] == "distil_logits":
        s["logits"] = torch.randn(n, v, generator=gen, device=dev).mul_(2.5).to(dt).requires_grad_(case["train"])
    else:
        d = case["d"]
        # hidden states as behind a layer norm; a trained table gives logits a spread of a few units
        s["hidden"] = torch.randn(n, d, generator=gen, device=dev).to(dt).requires_grad_(case["train"])
        w = torch.randn(v, d, generator=gen, device=dev).mul_(2.5 / math.sqrt(d)).to(dt)
        s["weights"] = (w if case["layout"] == "vd" else w.t().contiguous()).requires_grad_(case["train"])
        s["bias"] = torch.randn(v, generator=gen, device=dev).mul_(0.5).to(dt).requires_grad_(case["train"]) if case["bias"] else None
    if case["op"] == "ce":
        labels = torch.randint(0, v, (n,), generator=gen, device=dev)
        if case["ignored"]:
            labels[torch.rand(n, generator=gen, device=dev) < case["ignored"]] = IGNORE
        s["labels"] = labels
    else:
        s["indices"], s["teacher"] = _teacher(case, gen, dev)
    # gradient of the rows' losses: a mean over the rows with per-row weights around 1
    s["dloss"] = (torch.rand(n, generator=gen, device=dev) + 0.5) / max(1.0, n * (1.0 - case["ignored"]))
    return s


def _leaves(s):
    return {k: s[k] for k in ("hidden", "weights", "bias", "logits") if s.get(k) is not None}


def _own(s):
    from deeplearning4j_amd.ops import vocab_loss
    case = s["case"]
    if case["op"] == "distil_logits":
        loss = vocab_loss.topk_distillation(s["logits"], s["indices"], s["teacher"], temperature=case["temperature"])
    else:
        w = s["weights"] if case["layout"] == "vd" else s["weights"].t()
        if case["op"] == "ce":
            loss = vocab_loss.linear_cross_entropy(s["hidden"], w, s["labels"], bias=s["bias"], ignore_index=IGNORE,
                                                   label_smoothing=case["smoothing"])
        else:
            loss = vocab_loss.linear_topk_distillation(s["hidden"], w, s["indices"], s["teacher"], bias=s["bias"],
                                                       temperature=case["temperature"])
    if not case["train"]:
        return {"loss": loss}
    leaves = _leaves(s)
    grads = torch.autograd.grad(loss, list(leaves.values()), grad_outputs=s["dloss"])
    return {"loss": loss.detach(), **{"d_" + k: g for k, g in zip(leaves, grads)}}


def _plain(s):
    case = s["case"]
    if case["op"] == "distil_logits":
        z = s["logits"].float()
    else:
        h = s["hidden"].float()
        w = s["weights"].float() if case["layout"] == "vd" else s["weights"].float().t()
        z = h @ w.t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
    if case["op"] == "ce":
        keep = s["labels"] != IGNORE
        at = s["labels"].clamp(min=0).unsqueeze(1)
        e, v = case["smoothing"], case["v"]
        m = z.max(1, keepdim=True).values
        lse = m + (z - m).exp().sum(1, keepdim=True).log()
        loss = lse - (1 - e) * z.gather(1, at) - (e * z.mean(1, keepdim=True) if e else 0.0)
        loss = torch.where(keep, loss.squeeze(1), 0.0)
        if not case["train"]:
            return {"loss": loss}
        c = torch.where(keep, s["dloss"], 0.0).unsqueeze(1)
        g = ((z - lse).exp() - (e / v if e else 0.0)) * c
        g.scatter_add_(1, at, -(1 - e) * c)
    else:
        T = case["temperature"]
        there = s["indices"] >= 0
        at = s["indices"].clamp(min=0)
        t = torch.where(there, s["teacher"].float() / T, -math.inf)
        top = t.max(1, keepdim=True).values.clamp(min=-3e38)
        p = (t - top).exp()
        p = p / p.sum(1, keepdim=True).clamp(min=1e-30)
        z = z / T
        m = z.max(1, keepdim=True).values
        lse = m + (z - m).exp().sum(1, keepdim=True).log()
        logp = torch.where(p > 0, p.clamp(min=1e-38).log(), 0.0)
        loss = T * T * (p * (logp - (z.gather(1, at) - lse))).sum(1)
        if not case["train"]:
            return {"loss": loss}
        c = (T * s["dloss"]).unsqueeze(1)
        g = (z - lse).exp() * (c * p.sum(1, keepdim=True))
        g.scatter_add_(1, at, -c * p)
        if case["op"] == "distil_logits":
            return {"loss": loss, "d_logits": g.to(s["logits"].dtype)}
    out = {"loss": loss, "d_hidden": (g @ w).to(s["hidden"].dtype)}
    dw = g.t() @ h if case["layout"] == "vd" else h.t() @ g
    out["d_weights"] = dw.to(s["weights"].dtype)
    if s["bias"] is not None:
        out["d_bias"] = g.sum(0).to(s["bias"].dtype)
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def _valid(case):
    return max(1.0, case["n"] * (1.0 - case["ignored"]))


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    n, v, rows = case["n"], case["v"], _valid(case)
    side = rows * case["k"] * 12 if case["k"] else n * 8
    if case["op"] == "distil_logits":
        return {"bytes": rows * v * size + (n * v * size if case["train"] else 0) + side + n * 4, "flops": rows * v * (8 if case["train"] else 4)}
    d = case["d"]
    tables = (rows * d + v * d + (v if case["bias"] else 0)) * size
    grads = (n * d + v * d + (v if case["bias"] else 0)) * size if case["train"] else 0
    return {"bytes": tables + grads + side + n * 4, "flops": rows * d * v * (6 if case["train"] else 2)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact(case, s)


def _exact(case, s):
    """In 64 bits, a few rows at a time."""
    f64, n, v = torch.float64, case["n"], case["v"]
    linear = case["op"] != "distil_logits"
    loss = torch.zeros(n, dtype=f64, device="cuda")
    if linear:
        W = s["weights"].to(f64)
        if case["layout"] == "dv":
            W = W.t().contiguous()
        b = None if s["bias"] is None else s["bias"].to(f64)
        dh, dW, db = torch.zeros(n, case["d"], dtype=f64, device="cuda"), torch.zeros_like(W), torch.zeros(v, dtype=f64, device="cuda")
    else:
        dz = torch.zeros(n, v, dtype=f64, device="cuda") if case["train"] else None
    rows = max(1, 2 ** 26 // v)
    for a in range(0, n, rows):
        sl = slice(a, min(n, a + rows))
        if linear:
            h = s["hidden"][sl].to(f64)
            z = torch.mm(h, W.t())
            if b is not None:
                z += b
        else:
            z = s["logits"][sl].to(f64)
        T = case["temperature"] if case["op"] != "ce" else 1.0
        logq = torch.log_softmax(z / T, dim=1)
        if case["op"] == "ce":
            y = s["labels"][sl]
            weight = (y != IGNORE).to(f64)
            target = torch.full_like(z, case["smoothing"] / v)
            target[torch.arange(y.numel(), device="cuda"), y.clamp(min=0)] += 1.0 - case["smoothing"]
            loss[sl] = -(target * logq).sum(1) * weight
            mass = weight
            target *= weight[:, None]
        else:
            idx = s["indices"][sl]
            t = torch.where(idx >= 0, s["teacher"][sl].to(f64) / T, torch.tensor(-math.inf, dtype=f64, device="cuda"))
            p = torch.nan_to_num(torch.softmax(t, dim=1), nan=0.0)
            target = torch.zeros_like(z).scatter_add_(1, idx.clamp(min=0), p)
            loss[sl] = T * T * (torch.xlogy(p, p).sum(1) - (target * logq).sum(1))
            mass = p.sum(1)
        if not case["train"]:
            continue
        g = (logq.exp() * mass[:, None] - target) * (T * s["dloss"][sl].to(f64))[:, None]
        if linear:
            dh[sl] = torch.mm(g, W)
            dW += torch.mm(g.t(), h)
            db += g.sum(0)
        else:
            dz[sl] = g
    if not case["train"]:
        return {"loss": loss}
    if not linear:
        return {"loss": loss, "d_logits": dz}
    out = {"loss": loss, "d_hidden": dh, "d_weights": dW if case["layout"] == "vd" else dW.t().contiguous()}
    if s["bias"] is not None:
        out["d_bias"] = db
    return out
