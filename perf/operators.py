"""Measured cases of the generator's tuning operators: layer norm, the clipped policy loss, the preference loss, and
the global gradient norm with clipping. With `own` false every pass is computed from elementary torch operations; with
`own` true it goes through ldrs_amd.hip.ops. The sizes are those of the framework's own workloads (vocabularies of 10k,
20k and 50k words, sentences of 15 to 41 tokens, hidden sizes 256 to 1024, the 825-wide highway input) and odd ones
around them."""
import math

import torch

own = False

F32, BF16 = "float32", "bfloat16"
KINDS = ("layer_norm", "policy", "preference", "clip")


def _dt(case):
    return torch.float32 if case["dtype"] == F32 else torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the hidden rows of one sentence's beams between two decoding steps: nothing but latency
        {"name": "layer norm, 10 beams", "kind": "layer_norm", "rows": 10, "cols": 800, "dtype": F32, "train": False},
        # the encoder's highway input of a 64 x 20 batch: an odd width, rows that start on no 16-byte boundary
        {"name": "layer norm, highway input", "kind": "layer_norm", "rows": 1280, "cols": 825, "dtype": F32,
         "train": True},
        # the generator's hidden states of eight 256 x 41 batches
        {"name": "layer norm, eight batches", "kind": "layer_norm", "rows": 83968, "cols": 1024, "dtype": BF16,
         "train": True},
        # one sentence of 15 words and its end token over the small vocabulary
        {"name": "policy, one sentence", "kind": "policy", "seqs": 1, "len": 16, "vocab": 10000, "dtype": F32,
         "kl": 0.0, "inv_tau": 1.0, "banned": False},
        # the default training batch: 64 sentences of up to 21 tokens, 20k words
        {"name": "policy, 64 sentences", "kind": "policy", "seqs": 64, "len": 21, "vocab": 20000, "dtype": F32,
         "kl": 0.05, "inv_tau": 1.25, "banned": True},
        # the large-vocabulary batch: 256 sentences of up to 41 tokens, 50k words, bf16 logits
        {"name": "policy, large vocabulary", "kind": "policy", "seqs": 256, "len": 41, "vocab": 50000, "dtype": BF16,
         "kl": 0.05, "inv_tau": 1.0, "banned": False},
        # a single pair of sentences
        {"name": "preference, one pair", "kind": "preference", "pairs": 1, "len": 16, "vocab": 10000, "dtype": F32,
         "smooth": 0.0, "inv_tau": 1.0, "banned": False},
        # 32 pairs, a vocabulary of odd size: rows start on no 16-byte boundary
        {"name": "preference, 32 pairs", "kind": "preference", "pairs": 32, "len": 21, "vocab": 20001, "dtype": F32,
         "smooth": 0.1, "inv_tau": 1.0, "banned": True},
        # 64 pairs of the large-vocabulary model
        {"name": "preference, large vocabulary", "kind": "preference", "pairs": 64, "len": 41, "vocab": 50000,
         "dtype": BF16, "smooth": 0.0, "inv_tau": 1.0, "banned": False},
        # the gradients of one text classifier: three convolutions and a linear layer, weights and biases
        {"name": "clip, discriminator", "kind": "clip", "tensors": 8, "total": 361502, "dtype": F32, "adam": False},
        # sixty matrices and vectors, half of them bf16
        {"name": "clip, sixty tensors", "kind": "clip", "tensors": 60, "total": 30000000, "dtype": BF16, "adam": False},
        # the large-vocabulary generator's parameters (its output layer is 50000 x 1024), clipped inside the Adam update
        {"name": "clip in Adam, generator arena", "kind": "clip", "tensors": 1, "total": 64000000, "dtype": F32,
         "adam": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(KINDS)
    dtype = rng.choice((F32, BF16))
    size = 4 if dtype == F32 else 2
    if kind == "layer_norm":
        cols = _log_int(rng, 16, 4096)
        rows = _log_int(rng, 1, max(1, 160_000_000 // (cols * size)))
        return {"kind": kind, "rows": rows, "cols": cols, "dtype": dtype, "train": rng.random() < 0.75}
    if kind in ("policy", "preference"):
        vocab, length = _log_int(rng, 500, 60000), rng.randint(1, 48)
        most = (1_000_000_000 if kind == "policy" else 500_000_000) // (vocab * size * length)
        c = {"kind": kind, "len": length, "vocab": vocab, "dtype": dtype, "inv_tau": rng.choice((1.0, 1.25, 0.7)),
             "banned": rng.random() < 0.3}
        if kind == "policy":
            return {**c, "seqs": _log_int(rng, 1, max(1, min(256, most))), "kl": rng.choice((0.0, 0.02, 0.1))}
        return {**c, "pairs": _log_int(rng, 1, max(1, min(64, most // 2))), "smooth": rng.choice((0.0, 0.1))}
    adam = rng.random() < 0.4
    total = _log_int(rng, 1000, 50_000_000)
    return {"kind": kind, "tensors": 1 if adam else rng.randint(1, 60), "total": total, "dtype": F32 if adam else dtype,
            "adam": adam}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    return {"case": case, **{"layer_norm": _prepare_norm, "policy": _prepare_policy, "preference": _prepare_pairs,
                             "clip": _prepare_clip}[case["kind"]](case, _gen(seed))}


def _prepare_norm(case, g):
    R, C = case["rows"], case["cols"]
    x = torch.randn(R, C, device="cuda", generator=g)
    x = x * (0.5 + torch.rand(R, 1, device="cuda", generator=g)) + torch.randn(R, 1, device="cuda", generator=g)
    s = {"x": x.to(_dt(case)), "weight": 1.0 + 0.1 * torch.randn(C, device="cuda", generator=g),
         "bias": 0.1 * torch.randn(C, device="cuda", generator=g)}
    if case["train"]:
        s["dy"] = (0.1 * torch.randn(R, C, device="cuda", generator=g)).to(_dt(case))
    return s


def _logits(case, rows, g):
    """Logits of a trained generator: a normal spread and a few likely words a row; a banned word is never produced."""
    V = case["vocab"]
    x = torch.empty(rows, V, device="cuda", dtype=_dt(case))
    x.normal_(0.0, 1.5, generator=g)
    likely = torch.randint(0, V, (rows, 8), device="cuda", generator=g)
    x.scatter_(1, likely, (5.0 + 3.0 * torch.rand(rows, 8, device="cuda", generator=g)).to(x.dtype))
    if case["banned"]:
        x[:, 0] = -math.inf
    pick = torch.randint(0, 8, (rows, 1), device="cuda", generator=g)
    odd = torch.randint(1, V, (rows, 1), device="cuda", generator=g)
    take = torch.rand(rows, 1, device="cuda", generator=g) < 0.8
    target = torch.where(take, likely.gather(1, pick).clamp(min=1), odd).view(-1)
    return x, target


def _lengths(case, seqs, g):
    """1 where the sentence still runs, 0 behind its end: lengths are spread evenly over 1..len."""
    n = torch.randint(1, case["len"] + 1, (seqs, 1), device="cuda", generator=g)
    return (torch.arange(case["len"], device="cuda")[None] < n).float()


def _logp64(x, target, inv_tau, rows=2048):
    parts = [torch.log_softmax(x[i:i + rows].double() * inv_tau, 1).gather(1, target[i:i + rows, None])[:, 0]
             for i in range(0, x.shape[0], rows)]
    return torch.cat(parts)


def _prepare_policy(case, g):
    S, T = case["seqs"], case["len"]
    x, target = _logits(case, S * T, g)
    mask = _lengths(case, S, g)
    lp = _logp64(x, target, case["inv_tau"])
    # the log-ratio to the sampling policy, kept off the two borders where the loss has a kink
    d = 0.15 * torch.randn(S * T, device="cuda", generator=g).double()
    for edge in (math.log(0.8), math.log(1.2)):
        d = torch.where((d - edge).abs() < 2e-3, d + 5e-3, d)
    return {"logits": x, "target": target, "weight": (mask / mask.sum()).view(-1),
            "advantage": torch.randn(S, 1, device="cuda", generator=g).expand(S, T).reshape(-1).contiguous(),
            "old": (lp - d).float(), "ref": (lp + 0.2 * torch.randn(S * T, device="cuda", generator=g)).float(),
            "dlogits": torch.empty_like(x)}


def _prepare_pairs(case, g):
    P, T = case["pairs"], case["len"]
    x, target = _logits(case, 2 * P * T, g)
    mask = _lengths(case, 2 * P, g)
    S = (_logp64(x, target, case["inv_tau"]) * mask.view(-1)).view(2 * P, T).sum(1)
    side = torch.randint(0, 2, (P,), device="cuda", generator=g).double() * 2 - 1
    gain = side * (1.0 + 2.0 * torch.rand(P, device="cuda", generator=g).double())
    return {"logits": x, "target": target, "weight": mask, "ref": (S - torch.cat((gain, -gain))).float(),
            "dlogits": torch.empty_like(x)}


def _sizes(case):
    """`tensors` sizes that add up to `total`: every fourth one a vector, the rest matrices of uneven widths."""
    n, total = case["tensors"], case["total"]
    share = [(1 + (i * 7) % 5) * (0.01 if i % 4 == 3 else 1.0) for i in range(n)]
    sizes = [max(1, int(total * s / sum(share))) for s in share]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


def _prepare_clip(case, g):
    if case["adam"]:
        n = case["total"]
        grad = 0.01 * torch.randn(n, device="cuda", generator=g)
        return {"g": grad, "p": 0.1 * torch.randn(n, device="cuda", generator=g),
                "m": 0.01 * torch.randn(n, device="cuda", generator=g),
                "v": 1e-4 * (0.1 + torch.rand(n, device="cuda", generator=g)), "max_norm": 0.0063 * math.sqrt(n)}
    grads = [0.01 * torch.randn(n, device="cuda", generator=g) for n in _sizes(case)]
    grads = [t.to(torch.bfloat16) if case["dtype"] == BF16 and i % 2 == 0 else t for i, t in enumerate(grads)]
    return {"grads": grads, "out": [torch.empty_like(t) for t in grads], "max_norm": 0.0063 * math.sqrt(case["total"])}


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
EPS, CLIP, BETA, LR, STEP = 1e-5, 0.2, 0.1, 1e-3, 10


def run(s):
    return {"layer_norm": _run_norm, "policy": _run_policy, "preference": _run_pairs,
            "clip": _run_clip}[s["case"]["kind"]](s)


def _run_norm(s):
    if own:
        from ldrs_amd.hip import ops
        y, mean, rstd = ops.layer_norm_fwd(s["x"], s["weight"], s["bias"], EPS)
        if not s["case"]["train"]:
            return {"y": y}
        dx, dw, db = ops.layer_norm_bwd(s["dy"], s["x"], s["weight"], mean, rstd)
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    xh = d * rstd
    y = (xh * s["weight"] + s["bias"]).to(s["x"].dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * xh).sum(0, dtype=torch.float64).float(),
            "dbias": dy.sum(0, dtype=torch.float64).float()}


def _plain_rows(s):
    """(log-probabilities of the targets, probabilities) of every row, in 32 bits."""
    x = s["logits"].float() * s["case"]["inv_tau"]
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    return x.gather(1, s["target"][:, None])[:, 0] - torch.log(total[:, 0]), e / total


def _plain_dlogits(s, p, coef):
    """coef * (1 at the target - p), zero in the rows of weight zero."""
    live = s["weight"].reshape(-1, 1) != 0
    c = (coef * s["case"]["inv_tau"])[:, None]
    d = (p * -c).scatter_add(1, s["target"][:, None], c)
    return torch.where(live, d, 0.0).to(s["logits"].dtype)


def _run_policy(s):
    c = s["case"]
    if own:
        from ldrs_amd.hip import ops
        loss, logp = ops.policy_loss(s["logits"], s["target"], s["advantage"], s["weight"], old_logp=s["old"],
                                     ref_logp=s["ref"] if c["kl"] else None, clip=(CLIP, CLIP), kl_coef=c["kl"],
                                     inv_tau=c["inv_tau"], dlogits=s["dlogits"])
        return {"loss": loss, "logp": logp, "dlogits": s["dlogits"]}
    lp, p = _plain_rows(s)
    w, A = s["weight"], s["advantage"]
    ratio = torch.exp(lp - s["old"])
    kept = torch.minimum(ratio * A, ratio.clamp(1 - CLIP, 1 + CLIP) * A)
    cut = ((A > 0) & (ratio > 1 + CLIP)) | ((A < 0) & (ratio < 1 - CLIP))
    k = s["ref"] - lp
    loss = torch.where(w != 0, w * (c["kl"] * (torch.exp(k) - k - 1) - kept), 0.0)
    coef = w * (c["kl"] * (1 - torch.exp(k)) - torch.where(cut, 0.0, ratio * A))
    return {"loss": loss.sum(dtype=torch.float64).float().view(1), "logp": torch.where(w != 0, lp, 0.0),
            "dlogits": _plain_dlogits(s, p, coef)}


def _run_pairs(s):
    c = s["case"]
    if own:
        from ldrs_amd.hip import ops
        loss, margin, seq_logp = ops.preference_loss(s["logits"], s["target"], s["weight"], s["ref"], beta=BETA,
                                                     label_smoothing=c["smooth"], inv_tau=c["inv_tau"],
                                                     dlogits=s["dlogits"])
        return {"loss": loss, "margin": margin, "seq_logp": seq_logp, "dlogits": s["dlogits"]}
    P, e = c["pairs"], c["smooth"]
    lp, p = _plain_rows(s)
    S = torch.where(s["weight"] != 0, s["weight"] * lp.view(2 * P, -1), 0.0).sum(1, dtype=torch.float64)
    gain = S - s["ref"]
    m = BETA * (gain[:P] - gain[P:])
    loss = ((1 - e) * torch.log1p(torch.exp(-m)) + e * torch.log1p(torch.exp(m))).mean()
    up = -(BETA / P) * ((1 - e) * torch.sigmoid(-m) - e * torch.sigmoid(m))
    coef = (torch.cat((up, -up))[:, None] * s["weight"]).float().view(-1)
    return {"loss": loss.float().view(1), "margin": m.float(), "seq_logp": S.float(),
            "dlogits": _plain_dlogits(s, p, coef)}


def _run_clip(s):
    if s["case"]["adam"]:
        if own:
            from ldrs_amd.hip import ops
            norm = ops.adam(s["p"], s["g"], s["m"], s["v"], LR, STEP, max_norm=s["max_norm"])
            return {"norm": norm, "p": s["p"], "m": s["m"], "v": s["v"]}
        p, m, v = s["p"], s["m"], s["v"]
        norm = s["g"].double().square().sum().sqrt()
        g = s["g"] * (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
        m.add_((g - m) * (1 - 0.9))
        v.mul_(0.999).add_(g * g * (1 - 0.999))
        p.sub_(LR / (1 - 0.9 ** STEP) * (m / (v.sqrt() / math.sqrt(1 - 0.999 ** STEP) + 1e-8)))
        return {"norm": norm.float().view(1), "p": p, "m": m, "v": v}
    if own:
        from ldrs_amd.hip import ops
        norm = ops.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])
        return {"norm": norm, "out": s["out"]}
    norm = torch.stack([t.double().square().sum() for t in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    return {"norm": norm.float().view(1), "out": [o.copy_(t.float() * coef) for o, t in zip(s["out"], s["grads"])]}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == F32 else 2
    if case["kind"] == "layer_norm":
        n, C = case["rows"] * case["cols"], case["cols"]
        if not case["train"]:
            return {"bytes": 2 * n * size + 8 * C, "flops": 8 * n}
        return {"bytes": 4 * n * size + 16 * C, "flops": 22 * n}
    if case["kind"] in ("policy", "preference"):
        seqs = case["seqs"] if case["kind"] == "policy" else 2 * case["pairs"]
        rows = seqs * case["len"]
        live = seqs * (case["len"] + 1) / 2  # rows of weight zero are not read, only written
        return {"bytes": (live + rows) * case["vocab"] * size + 28 * rows, "flops": 8 * live * case["vocab"]}
    if case["adam"]:
        return {"bytes": 28 * case["total"], "flops": 18 * case["total"]}
    n = _sizes(case)
    size = [2 if case["dtype"] == BF16 and i % 2 == 0 else 4 for i in range(len(n))]
    return {"bytes": 2 * sum(a * b for a, b in zip(n, size)), "flops": 3 * sum(n)}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"layer_norm": _exact_norm, "policy": _exact_policy, "preference": _exact_pairs,
            "clip": _exact_clip}[case["kind"]](s)


def _exact_norm(s):
    w, b = s["weight"].double(), s["bias"].double()
    ys, dxs, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(w)
    for i in range(0, s["x"].shape[0], 8192):
        x = s["x"][i:i + 8192].double()
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        xh = (x - mean) / torch.sqrt(var + EPS)
        ys.append(xh * w + b)
        if s["case"]["train"]:
            dy = s["dy"][i:i + 8192].double()
            dw += (dy * xh).sum(0)
            db += dy.sum(0)
            g = dy * w
            g = g - g.mean(1, keepdim=True)
            dxs.append((g - xh * (g * xh).mean(1, keepdim=True)) / torch.sqrt(var + EPS))
    if not s["case"]["train"]:
        return {"y": torch.cat(ys)}
    return {"y": torch.cat(ys), "dx": torch.cat(dxs), "dweight": dw, "dbias": db}


def _exact_dlogits(s, coef, rows=1024):
    """The gradient of sum(coef * log-probability) over the rows that count, by the rows of the softmax."""
    out = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    for i in torch.nonzero(coef).view(-1).split(rows):
        q = torch.softmax(s["logits"][i].double() * s["case"]["inv_tau"], 1).neg_()
        q[torch.arange(len(i), device="cuda"), s["target"][i]] += 1.0
        out[i] = q * (coef[i] * s["case"]["inv_tau"])[:, None]
    return out


def _exact_policy(s):
    c = s["case"]
    lp = _logp64(s["logits"], s["target"], c["inv_tau"]).requires_grad_()
    w, A, old, ref = (s[k].double() for k in ("weight", "advantage", "old", "ref"))
    ratio = (lp - old).exp()
    kl = (ref - lp).exp() - (ref - lp) - 1
    loss = (w * (c["kl"] * kl - torch.minimum(ratio * A, ratio.clamp(1 - CLIP, 1 + CLIP) * A))).sum()
    loss.backward()
    return {"loss": loss.detach().view(1), "logp": lp.detach() * (w != 0), "dlogits": _exact_dlogits(s, lp.grad)}


def _exact_pairs(s):
    c, P = s["case"], s["case"]["pairs"]
    lp = _logp64(s["logits"], s["target"], c["inv_tau"]).requires_grad_()
    S = (lp.view(2 * P, -1) * s["weight"].double()).sum(1)
    gain = S - s["ref"].double()
    m = BETA * (gain[:P] - gain[P:])
    loss = -((1 - c["smooth"]) * torch.sigmoid(m).log() + c["smooth"] * torch.sigmoid(-m).log()).mean()
    loss.backward()
    return {"loss": loss.detach().view(1), "margin": m.detach(), "seq_logp": S.detach(),
            "dlogits": _exact_dlogits(s, lp.grad)}


def _exact_clip(s):
    grads = [s["g"]] if s["case"]["adam"] else s["grads"]
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads))
    coef = min(1.0, s["max_norm"] / (norm + 1e-6))
    total = torch.tensor([norm], dtype=torch.float64, device="cuda")
    if not s["case"]["adam"]:
        return {"norm": total, "out": [t.double() * coef for t in grads]}
    g = s["g"].double() * coef
    m = 0.9 * s["m"].double() + 0.1 * g
    v = 0.999 * s["v"].double() + 0.001 * g * g
    step = (m / (1 - 0.9 ** STEP)) / ((v / (1 - 0.999 ** STEP)).sqrt() + 1e-8)
    return {"norm": total, "p": s["p"].double() - LR * step, "m": m, "v": v}
