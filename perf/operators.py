"""Cases that measure the token-model operators: layer norm, embedding and token log-probabilities, each with its gradient.

`run` computes an operator in elementary torch operations where `own` is false and through `tlcuda` where it is true.
"""
import math
import os
import sys

import numpy as np
import torch

own = False
EPS = 1e-5
DEV = "cuda"


def _binding():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torchlite-cpp_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import tlcuda
    return tlcuda


# ---- the cases -------------------------------------------------------------------------------------------------------


def listed():
    return [
        # the norm in front of a layer while one token is generated: pure latency
        {"name": "norm 1 x 768", "op": "norm", "rows": 1, "dim": 768, "gap": 0},
        # a training batch of an encoder: 16 sequences of 512, width 768
        {"name": "norm 8192 x 768", "op": "norm", "rows": 8192, "dim": 768, "gap": 0},
        # an odd width, rows read out of a wider buffer
        {"name": "norm 4099 x 5001", "op": "norm", "rows": 4099, "dim": 5001, "gap": 7},
        # the gradient for the encoder's batch
        {"name": "norm grad 8192 x 768", "op": "norm grad", "rows": 8192, "dim": 768, "gap": 0},
        # the gradient in a wide model
        {"name": "norm grad 8192 x 8192", "op": "norm grad", "rows": 8192, "dim": 8192, "gap": 0},
        # the last tokens of 48 requests that are being answered
        {"name": "embed 48 x 768", "op": "embed", "batch": 48, "seq": 1, "vocab": 32000, "dim": 768, "bits": 64, "pad": False},
        # a long training batch of a wide model, sequences of unequal length
        {"name": "embed 32768 x 4096", "op": "embed", "batch": 16, "seq": 2048, "vocab": 131072, "dim": 4096, "bits": 64, "pad": True},
        # the encoder's batch: the table's gradient is larger than what flows into it
        {"name": "embed grad 8192 x 768", "op": "embed grad", "batch": 16, "seq": 512, "vocab": 32000, "dim": 768, "bits": 64, "pad": True},
        # a large batch into a table of an odd number of rows
        {"name": "embed grad 65536 x 2048", "op": "embed grad", "batch": 16, "seq": 4096, "vocab": 100003, "dim": 2048, "bits": 32, "pad": False},
        # the answer to one request: its token's log-probability and 20 alternatives, part of the vocabulary masked
        {"name": "logp 1 x 131072 top 20", "op": "logp", "batch": 1, "seq": 1, "vocab": 131072, "top": 20, "bits": 64, "scale": 1.0, "shift": False, "masked": True},
        # scoring prompts: each position scores the next token, with 5 alternatives, odd vocabulary
        {"name": "logp 4095 x 50001 top 5", "op": "logp", "batch": 5, "seq": 820, "vocab": 50001, "top": 5, "bits": 64, "scale": 1.0, "shift": True, "masked": False},
        # the gradient of a policy's log-probabilities and entropy at a temperature
        {"name": "logp grad 4096 x 50001", "op": "logp grad", "batch": 8, "seq": 512, "vocab": 50001, "top": 0, "bits": 32, "scale": 0.8, "shift": False, "masked": False},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm grad", "embed", "embed grad", "logp", "logp grad"])
    bits = rng.choice([32, 64])
    if op.startswith("norm"):
        dim = _log(rng, 16, 16384)
        return {"op": op, "rows": _log(rng, 1, min(65536, (1 << 26) // dim)), "dim": dim, "gap": rng.choice([0, 0, 8, 37])}
    batch = rng.randint(1, 16)
    if op.startswith("embed"):
        dim = _log(rng, 32, 8192)
        vocab = _log(rng, 256, min(131072, 200_000_000 // dim))
        seq = _log(rng, 1, max(1, min(131072, 120_000_000 // dim) // batch))
        return {"op": op, "batch": batch, "seq": seq, "vocab": vocab, "dim": dim, "bits": bits, "pad": rng.random() < 0.5}
    vocab = _log(rng, 100, 262144)
    shift = op == "logp" and rng.random() < 0.5
    seq = _log(rng, 2 if shift else 1, max(2, min(8192, 200_000_000 // vocab) // batch))
    return {"op": op, "batch": batch, "seq": seq, "vocab": vocab, "top": rng.choice([0, 1, 5, 20]) if op == "logp" else 0,
            "bits": bits, "scale": rng.choice([1.0, 1.0, 0.7, 1.25]), "shift": shift, "masked": rng.random() < 0.4}


# ---- their inputs ----------------------------------------------------------------------------------------------------


def _tokens(case, gen):
    """Token numbers that fall off as 1 / rank, as words do; -1 behind each sequence's end where there is padding."""
    shape = (case["batch"], case["seq"])
    u = torch.rand(shape, generator=gen, device=DEV, dtype=torch.float64)
    t = torch.exp(u * math.log(case["vocab"] + 1)).sub(1).floor().long().clamp(0, case["vocab"] - 1)
    if case.get("pad"):
        length = torch.randint(case["seq"] // 2, case["seq"] + 1, (case["batch"], 1), generator=gen, device=DEV)
        t = torch.where(torch.arange(case["seq"], device=DEV) < length, t, -1)
    return t.to(torch.int32 if case["bits"] == 32 else torch.int64)


def _logp_stats(logits, scale):
    """What the forward pass left for the backward: (the row's maximum, the log of its sum of exponentials) and its entropy."""
    rows = logits.reshape(-1, logits.shape[-1])
    stats, entropy = torch.empty(rows.shape[0], 2, device=DEV), torch.empty(rows.shape[0], device=DEV)
    for at in range(0, rows.shape[0], 1024):
        x = rows[at:at + 1024].double()
        m = x.amax(-1, keepdim=True)
        z = scale * (x - m)
        e = torch.exp(z)
        total = e.sum(-1)
        stats[at:at + 1024, 0], stats[at:at + 1024, 1] = m[:, 0], total.log()
        entropy[at:at + 1024] = total.log() - torch.where(e > 0, e * z, 0).sum(-1) / total
    return stats.view(*logits.shape[:-1], 2), entropy.view(logits.shape[:-1])


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEV)

    op = case["op"]
    s = {"case": case}
    if op.startswith("norm"):
        rows, dim = case["rows"], case["dim"]
        # a residual stream: columns of unequal size, some of them far larger, about a mean that is not zero
        size = 0.5 + torch.rand(dim, generator=gen, device=DEV)
        size[torch.randint(0, dim, (1 + dim // 256,), generator=gen, device=DEV)] *= 12
        wide = torch.zeros(rows, dim + case["gap"], device=DEV)
        wide[:, :dim] = normal(rows, dim) * size + 0.3 * normal(dim)
        s["x"] = wide[:, :dim]
        s["weight"], s["bias"] = 1 + 0.2 * normal(dim), 0.1 * normal(dim)
        if op == "norm grad":
            s["grad"] = normal(rows, dim)
            s["stats"] = torch.empty(rows, 2, device=DEV)
            for at in range(0, rows, 1024):
                x = s["x"][at:at + 1024].double()
                mean = x.mean(-1, keepdim=True)
                s["stats"][at:at + 1024, 0] = mean[:, 0]
                s["stats"][at:at + 1024, 1] = ((x - mean) ** 2).mean(-1).add(EPS).rsqrt()
        return s
    tokens = _tokens(case, gen)
    if op.startswith("embed"):
        s["tokens"], s["scale"] = tokens, math.sqrt(case["dim"])
        if op == "embed":
            s["weight"] = 0.02 * normal(case["vocab"], case["dim"])
        else:
            s["grad"] = normal(case["batch"], case["seq"], case["dim"])
        return s
    logits = 2.5 * normal(case["batch"], case["seq"], case["vocab"])
    if case["shift"]:  # position i scores token i + 1
        logits, tokens = logits[:, :-1], tokens[:, 1:]
    if case["masked"]:  # a grammar or a tool's schema leaves part of the vocabulary
        logits[..., torch.rand(case["vocab"], generator=gen, device=DEV) < 0.3] = -math.inf
    at = tokens.long().unsqueeze(-1)
    logits.scatter_(-1, at, 5 + 2 * normal(*at.shape))  # a trained model is often right
    s["logits"], s["tokens"] = logits, tokens
    if op == "logp grad":
        s["stats"], s["entropy"] = _logp_stats(logits, case["scale"])
        s["grad_logprobs"], s["grad_entropy"] = normal(*tokens.shape), 0.01 * normal(*tokens.shape)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------


def _own(s, case):
    tl, op = _binding(), case["op"]
    if op == "norm":
        return tl.layer_norm(s["x"], s["weight"], s["bias"], EPS)
    if op == "norm grad":
        return tl.layer_norm_backward(s["grad"], s["x"], s["stats"], s["weight"])
    if op == "embed":
        return tl.embedding(s["weight"], s["tokens"], scale=s["scale"])
    if op == "embed grad":
        return tl.embedding_backward(s["grad"], s["tokens"], case["vocab"], scale=s["scale"])
    if op == "logp":
        return tl.token_logprobs(s["logits"], s["tokens"], scale=case["scale"], top=case["top"])
    return tl.token_logprobs_backward(s["logits"], s["tokens"], s["stats"], s["grad_logprobs"], s["grad_entropy"],
                                      s["entropy"], scale=case["scale"])


def _norm(s):
    x = s["x"]
    mean = x.mean(-1, keepdim=True)
    off = x - mean
    rstd = ((off * off).mean(-1, keepdim=True) + EPS).rsqrt()
    return off * rstd * s["weight"] + s["bias"], torch.cat([mean, rstd], -1)


def _norm_grad(s):
    mean, rstd = s["stats"][:, :1], s["stats"][:, 1:]
    hat = (s["x"] - mean) * rstd
    gw = s["grad"] * s["weight"]
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))
    return dx, (s["grad"] * hat).sum(0), s["grad"].sum(0)


def _embed(s):
    t = s["tokens"].long()
    return torch.where((t >= 0).unsqueeze(-1), s["weight"][t.clamp(min=0)] * s["scale"], 0.0)


def _embed_grad(s, vocab):
    t, dim = s["tokens"].long().reshape(-1), s["grad"].shape[-1]
    d = torch.zeros(vocab, dim, device=t.device)
    d.index_add_(0, t.clamp(min=0), torch.where((t >= 0).unsqueeze(-1), s["grad"].reshape(-1, dim), 0.0))
    return d * s["scale"]


def _logp(s, scale, top):
    x, t = s["logits"], s["tokens"].long()
    m = x.amax(-1, keepdim=True)
    z = (x - m) * scale
    e = torch.exp(z)
    total = e.sum(-1)
    log_total = total.log()
    logp = torch.where(t >= 0, z.gather(-1, t.clamp(min=0).unsqueeze(-1))[..., 0] - log_total, 0.0)
    entropy = log_total - torch.where(e > 0, e * z, 0.0).sum(-1) / total
    out = [logp, entropy, torch.stack([m[..., 0], log_total], -1)]
    if top:
        value, index = torch.sort(x, dim=-1, descending=True, stable=True)
        out += [(value[..., :top] - m) * scale - log_total.unsqueeze(-1), index[..., :top].to(s["tokens"].dtype)]
    return out


def _logp_grad(s, scale):
    x, t = s["logits"], s["tokens"].long()
    logp = (x - s["stats"][..., :1]) * scale - s["stats"][..., 1:]
    p = torch.exp(logp)
    g = s["grad_logprobs"].unsqueeze(-1) * (t >= 0).unsqueeze(-1)
    d = -g * p - s["grad_entropy"].unsqueeze(-1) * torch.where(p > 0, p * (logp + s["entropy"].unsqueeze(-1)), 0.0)
    d.scatter_add_(-1, t.clamp(min=0).unsqueeze(-1), g)
    return d * scale


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    op = case["op"]
    if op == "norm":
        return _norm(s)
    if op == "norm grad":
        return _norm_grad(s)
    if op == "embed":
        return _embed(s)
    if op == "embed grad":
        return _embed_grad(s, case["vocab"])
    if op == "logp":
        return _logp(s, case["scale"], case["top"])
    return _logp_grad(s, case["scale"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def _distinct(case):
    """How many different tokens a batch is expected to hold."""
    edge = np.log(np.arange(1, case["vocab"] + 2)) / math.log(case["vocab"] + 1)
    n = case["batch"] * case["seq"] * (0.75 if case["pad"] else 1.0)
    return float(np.sum(1 - np.exp(n * np.log1p(-np.minimum(np.diff(edge), 1 - 1e-12)))))


def work(case):
    op = case["op"]
    if op.startswith("norm"):
        n, rows, dim = case["rows"] * case["dim"], case["rows"], case["dim"]
        if op == "norm":
            return {"bytes": 8 * n + 8 * dim + 8 * rows, "flops": 8 * n}
        return {"bytes": 12 * n + 12 * dim + 8 * rows, "flops": 14 * n}
    count = case["batch"] * (case["seq"] - (1 if case.get("shift") else 0))
    index = count * case["bits"] // 8
    if op == "embed":
        return {"bytes": index + int(4 * case["dim"] * (count + _distinct(case))), "flops": count * case["dim"]}
    if op == "embed grad":
        n = int(count * (0.75 if case["pad"] else 1.0)) * case["dim"]
        return {"bytes": index + 4 * n + 4 * case["vocab"] * case["dim"], "flops": 2 * n}
    n = count * case["vocab"]
    if op == "logp":
        return {"bytes": 4 * n + index + count * (16 + case["top"] * (4 + case["bits"] // 8)), "flops": 6 * n}
    return {"bytes": 8 * n + index + 20 * count, "flops": 9 * n}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------


def _exact_logp(s, case):
    x = s["logits"].reshape(-1, case["vocab"])
    tokens = s["tokens"].reshape(-1)
    logp, entropy, stats, best, which = [], [], [], [], []
    for at in range(0, x.shape[0], 512):
        part, t = x[at:at + 512].double(), tokens[at:at + 512].long()
        whole = torch.logsumexp(part * case["scale"], -1, keepdim=True)
        every = part * case["scale"] - whole
        p = every.exp()
        logp.append(every[torch.arange(len(t), device=t.device), t])
        entropy.append(-(p * every.clamp(min=-1e30)).sum(-1))
        top1 = part.max(-1, keepdim=True).values
        stats.append(torch.cat([top1, whole - case["scale"] * top1], -1))
        if case["top"]:
            order = torch.argsort(-part, dim=-1, stable=True)[:, :case["top"]]
            which.append(order.to(tokens.dtype))
            best.append(every.gather(-1, order))
    shape = s["tokens"].shape
    out = [torch.cat(logp).view(shape), torch.cat(entropy).view(shape), torch.cat(stats).view(*shape, 2)]
    return out + [torch.cat(v).view(*shape, case["top"]) for v in (best, which) if case["top"]]


def _exact_logp_grad(s, case):
    x, tokens = s["logits"].reshape(-1, case["vocab"]), s["tokens"].reshape(-1)
    gl, gh = s["grad_logprobs"].reshape(-1), s["grad_entropy"].reshape(-1)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for at in range(0, x.shape[0], 512):
        part, t = x[at:at + 512].double() * case["scale"], tokens[at:at + 512].long()
        logp = torch.log_softmax(part, -1).clamp(min=-1e30)
        p = logp.exp()
        entropy = -(p * logp).sum(-1, keepdim=True)
        one = torch.zeros_like(p)
        one[torch.arange(len(t), device=t.device), t] = 1.0
        a, b = gl[at:at + 512].double().unsqueeze(-1), gh[at:at + 512].double().unsqueeze(-1)
        out[at:at + 512] = case["scale"] * (a * (one - p) - b * p * (logp + entropy))
    return out.view(*s["tokens"].shape, case["vocab"])


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        scale = 1 / torch.sqrt(var + EPS)
        return (x - mean) * scale * s["weight"].double() + s["bias"].double(), torch.cat([mean, scale], -1)
    if op == "norm grad":
        x, g = s["x"].double(), s["grad"].double()
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS)
        hat = (x - mean) / sd
        # the Jacobian of x -> hat is (1 - 1/D - hat hat^T / D) / sd
        back = g * s["weight"].double()
        dot = torch.einsum("rd,rd->r", back, hat).unsqueeze(-1)
        dx = (back - (back.sum(-1, keepdim=True) + hat * dot) / case["dim"]) / sd
        return dx, torch.einsum("rd,rd->d", g, hat), torch.einsum("rd->d", g)
    if op == "embed":
        table = torch.cat([s["weight"].double() * s["scale"], torch.zeros(1, case["dim"], dtype=torch.float64, device=DEV)])
        return table[s["tokens"].long()]  # -1 is the last row
    if op == "embed grad":
        d = torch.zeros(case["vocab"] + 1, case["dim"], dtype=torch.float64, device=DEV)
        t = s["tokens"].long().reshape(-1) % (case["vocab"] + 1)
        d.index_put_((t,), s["grad"].reshape(-1, case["dim"]).double(), accumulate=True)
        return d[:-1] * s["scale"]
    return _exact_logp(s, case) if op == "logp" else _exact_logp_grad(s, case)
