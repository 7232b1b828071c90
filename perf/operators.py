"""Measured cases of the preference / policy tuning operators.

Five operators, each forward and backward in one pass, as a training step runs
them around the QLoRA model:

* ``logps``      per-token log-probabilities and entropies of the lm_head, with
                 the gradient of the hidden states (and of a trained head);
* ``preference`` paired log-ratio loss over chosen / rejected sequences;
* ``policy``     clipped importance-ratio loss with a KL term;
* ``window``     causal grouped-query attention with a sliding window and a few
                 first tokens that stay visible (sinks);
* ``swiglu8``    SwiGLU whose backward reads gate and up from 8-bit codes.

``run`` computes the plain form (elementary torch operations in 32 or 64 bits,
rounded once at the end) unless ``own`` is set; then it makes the calls that a
user makes of the framework.
"""

import math

import numpy as np
import torch

own = False

IGNORE = -100
HEAD_DIM = 128
Q_BLOCK = 64  # elements that share one scale in the 8-bit format

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one short answer pair scored against the Qwen2.5-1.5B head: few rows, the head is read once
        {"name": "logps_short", "op": "logps", "batch": 2, "seq": 64, "vocab": 151936, "dim": 1536,
         "prompt": 0.3, "train_head": False},
        # a preference batch of the benchmark's shape (4 x 1024 tokens), prompts unlabelled, head frozen
        {"name": "logps_pairs", "op": "logps", "batch": 4, "seq": 1024, "vocab": 151936, "dim": 1536,
         "prompt": 0.3, "train_head": False},
        # a trained head of a smaller model with an odd vocabulary and odd rows: its gradient too
        {"name": "logps_head", "op": "logps", "batch": 3, "seq": 333, "vocab": 32003, "dim": 896,
         "prompt": 0.15, "train_head": True},
        # two pairs per step at the task's 512-token limit: the smallest call, latency counts
        {"name": "preference_small", "op": "preference", "pairs": 2, "seq": 512, "loss": "sigmoid",
         "smoothing": 0.0, "prompt": 0.3},
        # accumulated evaluation batch of long pairs, odd length
        {"name": "preference_large", "op": "preference", "pairs": 96, "seq": 4095, "loss": "sigmoid",
         "smoothing": 0.1, "prompt": 0.3},
        # one prompt's group of 8 sampled answers
        {"name": "policy_small", "op": "policy", "batch": 8, "seq": 512, "reduction": "token",
         "kl": 0.04, "per_token": False, "prompt": 0.3},
        # 256 prompts x 8 answers of one optimisation round
        {"name": "policy_large", "op": "policy", "batch": 2048, "seq": 2048, "reduction": "sequence",
         "kl": 0.04, "per_token": False, "prompt": 0.3},
        # a short batch of the QLoRA step's heads with a narrow window
        {"name": "window_short", "op": "window", "batch": 4, "heads": 12, "kv_heads": 2, "seq": 512,
         "window": 128, "sinks": 4},
        # the step's 4 x 2048 tokens with a window a quarter of the sequence
        {"name": "window_step", "op": "window", "batch": 4, "heads": 12, "kv_heads": 2, "seq": 2048,
         "window": 512, "sinks": 4},
        # one long document, odd length, window that ends inside a tile
        {"name": "window_long", "op": "window", "batch": 1, "heads": 12, "kv_heads": 2, "seq": 16001,
         "window": 1000, "sinks": 16},
        # MLP of a short batch, gate / up as column halves of one projection
        {"name": "swiglu8_short", "op": "swiglu8", "rows": 130, "cols": 8960, "dtype": "bf16"},
        # MLP of the 4 x 2048-token step
        {"name": "swiglu8_step", "op": "swiglu8", "rows": 8192, "cols": 8960, "dtype": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logps", "preference", "policy", "window", "swiglu8"])
    if op == "logps":
        return {"op": op, "batch": rng.randint(1, 4), "seq": _log_uniform(rng, 9, 900),
                "vocab": _log_uniform(rng, 1000, 151936), "dim": 8 * _log_uniform(rng, 8, 192),
                "prompt": rng.uniform(0.0, 0.5), "train_head": rng.random() < 0.4}
    if op == "preference":
        return {"op": op, "pairs": _log_uniform(rng, 1, 90), "seq": _log_uniform(rng, 17, 4000),
                "loss": rng.choice(["sigmoid", "hinge", "ipo"]), "smoothing": 0.0,
                "prompt": rng.uniform(0.0, 0.5)}
    if op == "policy":
        return {"op": op, "batch": _log_uniform(rng, 1, 1500), "seq": _log_uniform(rng, 17, 2047),
                "reduction": rng.choice(["token", "sequence"]), "kl": rng.choice([0.0, 0.04]),
                "per_token": rng.random() < 0.5, "prompt": rng.uniform(0.0, 0.5)}
    if op == "window":
        kv = rng.choice([1, 2, 4])
        seq = _log_uniform(rng, 33, 6000)
        return {"op": op, "batch": rng.randint(1, 2), "heads": kv * rng.choice([1, 3, 6]) if kv < 4 else 8,
                "kv_heads": kv, "seq": seq, "window": _log_uniform(rng, 8, max(9, seq)),
                "sinks": rng.choice([0, 1, 4, 130])}
    return {"op": op, "rows": _log_uniform(rng, 3, 8000), "cols": _log_uniform(rng, 500, 8960),
            "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}


# ------------------------------------------------------------------ inputs ----
def _label_mask(batch, seq, prompt, seed):
    """[batch, seq] bool: the answer tokens between a prompt and the padding."""
    rs = np.random.RandomState(seed % (2 ** 31))
    start = np.floor(seq * prompt * rs.uniform(0.5, 1.5, size=(batch, 1)))
    stop = seq - np.floor(seq * 0.1 * rs.uniform(0.0, 2.0, size=(batch, 1)))
    pos = np.arange(seq)[None, :]
    return torch.from_numpy((pos >= start) & (pos < stop))


def _labelled(case, rows):
    """Expected labelled tokens of ``rows`` sequences of the case."""
    return rows * case["seq"] * max(0.0, 0.9 - case["prompt"])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    op = case["op"]
    st = {"case": case}
    if op == "logps":
        b, s, v, d = case["batch"], case["seq"], case["vocab"], case["dim"]
        weight = randn(v, d, dtype=torch.bfloat16).mul_(0.02)
        ids = torch.randint(0, v, (b, s), generator=g, device=dev)
        # hidden states that favour their target by 0 to 15 in the logit
        lift = 15.0 * torch.rand(b, s, 1, generator=g, device=dev) / (d * 0.02 ** 2)
        hidden = (randn(b, s, d) + lift * weight[ids].float()).to(torch.bfloat16)
        mask = _label_mask(b, s, case["prompt"], seed).to(dev)
        st["labels"] = torch.where(mask, ids, torch.full_like(ids, IGNORE))
        st["hidden"] = hidden.requires_grad_(own)
        st["weight"] = weight.requires_grad_(own and case["train_head"])
        st["dlogps"] = randn(b, s) / (b * s)
    elif op == "preference":
        n, s = 2 * case["pairs"], case["seq"]
        logps = -torch.rand(n, s, generator=g, device=dev).mul_(0.999).add_(0.001).log_().abs_() * 1.5
        mask = _label_mask(n, s, case["prompt"], seed).to(dev)
        ids = torch.randint(0, 151936, (n, s), generator=g, device=dev)
        st["labels"] = torch.where(mask, ids, torch.full_like(ids, IGNORE))
        st["ref_logps"] = torch.where(mask, logps + 0.1 * randn(n, s), torch.zeros_like(logps))
        st["logps"] = torch.where(mask, logps, torch.zeros_like(logps)).requires_grad_(own)
    elif op == "policy":
        b, s = case["batch"], case["seq"]
        logps = -torch.rand(b, s, generator=g, device=dev).mul_(0.999).add_(0.001).log_().abs_() * 1.5
        mask = _label_mask(b, s, case["prompt"], seed).to(dev)
        ids = torch.randint(0, 151936, (b, s), generator=g, device=dev)
        zero = torch.zeros_like(logps)
        st["labels"] = torch.where(mask, ids, torch.full_like(ids, IGNORE))
        st["old_logps"] = torch.where(mask, logps + 0.12 * randn(b, s), zero)
        st["ref_logps"] = torch.where(mask, logps + 0.2 * randn(b, s), zero) if case["kl"] else None
        st["advantages"] = randn(b, s) if case["per_token"] else randn(b)
        st["logps"] = torch.where(mask, logps, zero).requires_grad_(own)
    elif op == "window":
        b, h, hk, s = case["batch"], case["heads"], case["kv_heads"], case["seq"]
        d = HEAD_DIM
        u = randn(d)
        # a common direction of the queries that the first keys answer to, as sinks do
        q = (randn(b, s, h, d) + 0.4 * u).to(torch.bfloat16)
        k = randn(b, s, hk, d)
        k[:, :max(1, case["sinks"])] += 0.8 * u
        k = k.to(torch.bfloat16)
        v = randn(b, s, hk, d, dtype=torch.bfloat16)
        # projections [B, S, heads, D] handed over as [B, heads, S, D] views
        for name, t in (("q", q), ("k", k), ("v", v)):
            st[name] = t.transpose(1, 2).requires_grad_(own)
        st["dout"] = randn(b, s, h, d, dtype=torch.bfloat16)
        st["scale"] = d ** -0.5
    else:
        r, c, dt = case["rows"], case["cols"], _DTYPES[case["dtype"]]
        both = randn(r, 2 * c).mul_(1.5).to(dt)
        st["gate"] = both[:, :c].requires_grad_(own)
        st["up"] = both[:, c:].requires_grad_(own)
        st["dy"] = randn(r, c, dtype=dt)
    return st


# --------------------------------------------------------------- own calls ----
def _run_own(st):
    from auspex_soup_demo_b200 import kernels

    case = st["case"]
    op = case["op"]
    if op == "logps":
        logps, ent = kernels.head_token_logps(st["hidden"], st["weight"], st["labels"])
        leaves = [st["hidden"]] + ([st["weight"]] if case["train_head"] else [])
        grads = torch.autograd.grad(logps, leaves, st["dlogps"])
        out = {"logps": logps.detach(), "entropies": ent, "dhidden": grads[0]}
        if case["train_head"]:
            out["dweight"] = grads[1]
        return out
    if op == "preference":
        loss, chosen, rejected = kernels.preference_loss(
            st["logps"], st["ref_logps"], st["labels"], beta=0.1, label_smoothing=case["smoothing"],
            loss_type=case["loss"])
        (grad,) = torch.autograd.grad(loss, [st["logps"]])
        return {"loss": loss.detach(), "chosen": chosen, "rejected": rejected, "dlogps": grad}
    if op == "policy":
        loss, kl, clipped = kernels.policy_loss(
            st["logps"], st["advantages"], st["labels"], old_logps=st["old_logps"],
            ref_logps=st["ref_logps"], clip_low=0.2, clip_high=0.28, kl_coef=case["kl"],
            reduction=case["reduction"])
        (grad,) = torch.autograd.grad(loss, [st["logps"]])
        return {"loss": loss.detach(), "kl": kl, "clipped": clipped, "dlogps": grad}
    if op == "window":
        out = kernels.window_attention(st["q"], st["k"], st["v"], st["scale"], case["window"],
                                       case["sinks"])
        grads = torch.autograd.grad(out, [st["q"], st["k"], st["v"]], st["dout"])
        return {"out": out.detach(), "dq": grads[0], "dk": grads[1], "dv": grads[2]}
    h = kernels.swiglu_8bit(st["gate"], st["up"])
    dg, du = torch.autograd.grad(h, [st["gate"], st["up"]], st["dy"])
    return {"h": h.detach(), "dg": dg, "du": du}


# -------------------------------------------------------------- plain form ----
def _plain_logps(st):
    case = st["case"]
    v, d = case["vocab"], case["dim"]
    labels = st["labels"].reshape(-1)
    h = st["hidden"].detach().reshape(-1, d).float()
    w = st["weight"].detach().float()
    g = st["dlogps"].reshape(-1)
    n = h.shape[0]
    logps = torch.zeros(n, device=h.device)
    ents = torch.zeros(n, device=h.device)
    dh = torch.empty(n, d, device=h.device)
    dw = torch.zeros(v, d, device=h.device) if case["train_head"] else None
    step = max(1, (1 << 30) // v)
    for a in range(0, n, step):
        lab = labels[a:a + step]
        keep = lab != IGNORE
        z = h[a:a + step] @ w.t()
        m = z.max(1, keepdim=True).values
        e = torch.exp(z - m)
        total = e.sum(1, keepdim=True)
        p = e / total
        lse = (m + torch.log(total)).squeeze(1)
        idx = torch.where(keep, lab, torch.zeros_like(lab))
        zt = z.gather(1, idx[:, None]).squeeze(1)
        zero = torch.zeros_like(lse)
        logps[a:a + step] = torch.where(keep, zt - lse, zero)
        ents[a:a + step] = torch.where(keep, lse - (p * z).sum(1), zero)
        gk = torch.where(keep, g[a:a + step], zero)
        dz = -p * gk[:, None]
        dz[torch.arange(len(lab), device=dz.device), idx] += gk
        dh[a:a + step] = dz @ w
        if dw is not None:
            dw += dz.t() @ h[a:a + step]
    shape = st["labels"].shape
    out = {"logps": logps.view(shape), "entropies": ents.view(shape),
           "dhidden": dh.to(st["hidden"].dtype).view(st["hidden"].shape)}
    if dw is not None:
        out["dweight"] = dw.to(st["weight"].dtype)
    return out


def _plain_preference(st, beta=0.1):
    case = st["case"]
    x, ref = st["logps"].detach(), st["ref_logps"]
    mask = st["labels"] != IGNORE
    n, p = x.shape[0], x.shape[0] // 2
    # sums over thousands of tokens, and the few values per pair, in 64 bits
    diff = torch.where(mask, x - ref, torch.zeros_like(x)).sum(1, dtype=torch.float64)
    count = mask.sum(1).double()
    per = 1.0 / torch.clamp(count, min=1.0)
    rew = beta * diff
    score = diff * per if case["loss"] == "ipo" else diff
    hh = score[:p] - score[p:]
    if case["loss"] == "sigmoid":
        eps = case["smoothing"]
        soft_neg = torch.clamp(-beta * hh, min=0.0) + torch.log1p(torch.exp(-(beta * hh).abs()))
        soft_pos = torch.clamp(beta * hh, min=0.0) + torch.log1p(torch.exp(-(beta * hh).abs()))
        losses = (1.0 - eps) * soft_neg + eps * soft_pos
        sig = 1.0 / (1.0 + torch.exp(beta * hh))
        dh = -beta * ((1.0 - eps) * sig - eps * (1.0 - sig))
    elif case["loss"] == "hinge":
        losses = torch.clamp(1.0 - beta * hh, min=0.0)
        dh = torch.where(1.0 - beta * hh > 0, torch.full_like(hh, -beta), torch.zeros_like(hh))
    else:
        t = hh - 1.0 / (2.0 * beta)
        losses = t * t
        dh = 2.0 * t
    coef = torch.cat([dh, -dh]) / p
    if case["loss"] == "ipo":
        coef = coef * per
    grad = torch.where(mask, coef.float()[:, None].expand(n, x.shape[1]), torch.zeros_like(x))
    return {"loss": losses.mean().float(), "chosen": rew[:p].float(), "rejected": rew[p:].float(),
            "dlogps": grad}


def _plain_policy(st, lo=0.2, hi=0.28):
    case = st["case"]
    x, old, adv = st["logps"].detach(), st["old_logps"], st["advantages"]
    adv = adv if adv.dim() == 2 else adv[:, None].expand_as(x)
    mask = st["labels"] != IGNORE
    zero = torch.zeros_like(x)
    # which side of the clip border a ratio lies on is told in 64 bits
    side = torch.exp(x.double() - old.double())
    clipped = ((adv > 0) & (side > 1.0 + hi)) | ((adv < 0) & (side < 1.0 - lo))
    r = torch.exp(x - old)
    obj = torch.where(clipped, torch.where(adv > 0, zero + (1.0 + hi), zero + (1.0 - lo)) * adv, r * adv)
    tok = -obj
    grad = torch.where(clipped, zero, -adv * r)
    kl = zero
    if case["kl"]:
        delta = st["ref_logps"] - x
        kl = torch.exp(delta) - delta - 1.0
        tok = tok + case["kl"] * kl
        grad = grad + case["kl"] * (1.0 - torch.exp(delta))
    count = mask.sum(1, keepdim=True)
    total = torch.clamp(count.sum(), min=1)
    if case["reduction"] == "token":
        wgt = (1.0 / total.double()).expand_as(count)
    else:
        wgt = 1.0 / (torch.clamp(count, min=1).double() * x.shape[0])
    sums = torch.where(mask, tok, zero).sum(1, keepdim=True, dtype=torch.float64)
    return {"loss": (sums * wgt).sum().float(),
            "kl": (torch.where(mask, kl, zero).sum(dtype=torch.float64) / total).float(),
            "clipped": ((clipped & mask).sum() / total.double()).float(),
            "dlogps": torch.where(mask, grad * wgt.float(), zero)}


def _plain_window(st):
    case = st["case"]
    b, h, hk, s = case["batch"], case["heads"], case["kv_heads"], case["seq"]
    q, k, v = (st[n].detach().float() for n in ("q", "k", "v"))
    do = st["dout"].float()
    i = torch.arange(s, device=q.device)[:, None]
    j = torch.arange(s, device=q.device)[None, :]
    seen = (j <= i) & ((i - j < case["window"]) | (j < case["sinks"]))
    out = torch.empty(b, s, h, HEAD_DIM, device=q.device)
    dq = torch.empty(b, h, s, HEAD_DIM, device=q.device)
    dk = torch.zeros(b, hk, s, HEAD_DIM, device=q.device)
    dv = torch.zeros(b, hk, s, HEAD_DIM, device=q.device)
    for bi in range(b):
        for hi in range(h):
            g = hi // (h // hk)
            p = (q[bi, hi] @ k[bi, g].t()) * st["scale"]
            p = torch.where(seen, p, torch.full_like(p, -math.inf))
            p = torch.exp(p - p.max(1, keepdim=True).values)
            p = p / p.sum(1, keepdim=True)
            o = p @ v[bi, g]
            out[bi, :, hi] = o
            dv[bi, g] += p.t() @ do[bi, :, hi]
            dp = do[bi, :, hi] @ v[bi, g].t()
            ds = p * (dp - (do[bi, :, hi] * o).sum(1, keepdim=True)) * st["scale"]
            dq[bi, hi] = ds @ k[bi, g]
            dk[bi, g] += ds.t() @ q[bi, hi]
    return {"out": out.to(torch.bfloat16), "dq": dq.to(torch.bfloat16), "dk": dk.to(torch.bfloat16),
            "dv": dv.to(torch.bfloat16)}


def _plain_q8(x):
    """What a row's 8-bit codes stand for: blocks of Q_BLOCK columns share absmax / 127."""
    r, c = x.shape
    pad = (-c) % Q_BLOCK
    xp = torch.cat([x, torch.zeros(r, pad, device=x.device)], 1).view(r, -1, Q_BLOCK)
    top = xp.abs().max(2, keepdim=True).values
    tiny = top < 2.0 ** -100
    full = torch.full_like(top, 127.0)  # a tensor: dividing by a number multiplies by its reciprocal
    inv = torch.where(tiny, torch.zeros_like(top), full / top)
    return (torch.round(xp * inv) * (top / full)).view(r, c + pad)[:, :c]


def _plain_swiglu8(st):
    dt = st["gate"].dtype
    g, u, dy = st["gate"].detach().float(), st["up"].detach().float(), st["dy"].float()
    h = g / (1.0 + torch.exp(-g)) * u
    gq, uq = _plain_q8(g), _plain_q8(u)
    sig = 1.0 / (1.0 + torch.exp(-gq))
    du = dy * gq * sig
    dg = dy * uq * sig * (1.0 + gq * (1.0 - sig))
    return {"h": h.to(dt), "dg": dg.to(dt), "du": du.to(dt)}


_PLAIN = {"logps": _plain_logps, "preference": _plain_preference, "policy": _plain_policy,
          "window": _plain_window, "swiglu8": _plain_swiglu8}


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------- work ----
def work(case):
    op = case["op"]
    if op == "logps":
        n, v, d = case["batch"] * case["seq"], case["vocab"], case["dim"]
        lab = _labelled(case, case["batch"])  # unlabelled rows need no product
        wts = 2 * v * d
        flops = 2.0 * lab * v * d * (3 if case["train_head"] else 2)
        nbytes = wts + lab * d * 2 + n * 8 + n * 4 * 3 + n * d * 2 + (wts if case["train_head"] else 0)
        return {"bytes": float(nbytes), "flops": flops}
    if op == "preference":
        t = 2 * case["pairs"] * case["seq"]
        lab = _labelled(case, 2 * case["pairs"])
        return {"bytes": t * 8.0 + lab * 8.0 + t * 4.0 + 8.0 * case["pairs"], "flops": 2.0 * lab}
    if op == "policy":
        t = case["batch"] * case["seq"]
        lab = _labelled(case, case["batch"])
        arrays = 2 + (1 if case["kl"] else 0) + (1 if case["per_token"] else 0)
        return {"bytes": t * 8.0 + lab * 4.0 * arrays + t * 4.0 + 4.0 * case["batch"], "flops": 12.0 * lab}
    if op == "window":
        b, h, hk, s = case["batch"], case["heads"], case["kv_heads"], case["seq"]
        win, sinks = min(case["window"], s), min(case["sinks"], s)
        pairs = s * win - win * (win - 1) / 2.0  # keys within the window
        for j in range(sinks):  # the sinks that the window has left behind
            pairs += max(0, s - j - win)
        q = b * s * h * HEAD_DIM * 2
        kv = b * s * hk * HEAD_DIM * 2
        return {"bytes": float(4 * q + 4 * kv), "flops": 7 * 2.0 * b * h * pairs * HEAD_DIM}
    size = _DTYPES[case["dtype"]].itemsize
    t = case["rows"] * case["cols"]
    # forward: gate, up, h and the codes; backward: codes, dy, dg, du
    return {"bytes": t * (6.0 * size) + 2 * 2 * t * (1.0 + 4.0 / Q_BLOCK), "flops": 30.0 * t}


# ------------------------------------------------------------------ exact ----
def _exact_logps(st):
    case = st["case"]
    v, d = case["vocab"], case["dim"]
    lab = st["labels"].reshape(-1)
    rows = torch.nonzero(lab >= 0).squeeze(1)  # only these have values
    hid = st["hidden"].detach().reshape(-1, d)
    w = st["weight"].detach().to(torch.float64)
    up = st["dlogps"].reshape(-1).to(torch.float64)
    lp = torch.zeros(lab.numel(), dtype=torch.float64, device=hid.device)
    en = torch.zeros_like(lp)
    dh = torch.zeros(lab.numel(), d, dtype=torch.float64, device=hid.device)
    dw = torch.zeros(v, d, dtype=torch.float64, device=hid.device) if case["train_head"] else None
    step = max(1, (1 << 28) // v)
    for part in rows.split(step):
        x = hid[part].to(torch.float64)
        logp = torch.log_softmax(torch.mm(x, w.T), dim=-1)
        prob = logp.exp()
        tgt = lab[part].unsqueeze(1)
        lp[part] = logp.gather(1, tgt).squeeze(1)
        en[part] = -(prob * logp).sum(-1)
        prob.neg_().scatter_add_(1, tgt, torch.ones_like(tgt, dtype=torch.float64))
        prob *= up[part].unsqueeze(1)
        dh[part] = torch.mm(prob, w)
        if dw is not None:
            dw.addmm_(prob.T, x)
    shape = st["labels"].shape
    out = {"logps": lp.reshape(shape), "entropies": en.reshape(shape),
           "dhidden": dh.reshape(st["hidden"].shape)}
    if dw is not None:
        out["dweight"] = dw
    return out


def _exact_preference(st):
    case, beta = st["case"], 0.1
    x = st["logps"].detach().to(torch.float64).requires_grad_(True)
    keep = (st["labels"] >= 0).to(torch.float64)
    ratios = ((x - st["ref_logps"].to(torch.float64)) * keep).sum(-1)
    scores = ratios / keep.sum(-1).clamp_min(1.0) if case["loss"] == "ipo" else ratios
    chosen, rejected = scores.chunk(2)
    margin = chosen - rejected
    if case["loss"] == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        loss = -(1 - case["smoothing"]) * ls(beta * margin) - case["smoothing"] * ls(-beta * margin)
    elif case["loss"] == "hinge":
        loss = torch.relu(1.0 - beta * margin)
    else:
        loss = (margin - 0.5 / beta).square()
    loss = loss.mean()
    (grad,) = torch.autograd.grad(loss, [x])
    rc, rr = (beta * ratios.detach()).chunk(2)
    return {"loss": loss.detach(), "chosen": rc, "rejected": rr, "dlogps": grad}


def _exact_policy(st):
    case = st["case"]
    rows, cols = torch.nonzero(st["labels"] >= 0, as_tuple=True)
    x = st["logps"].detach()[rows, cols].to(torch.float64)
    a = st["advantages"].to(torch.float64)
    a = a[rows, cols] if a.dim() == 2 else a[rows]
    ratio = (x - st["old_logps"][rows, cols].to(torch.float64)).exp()
    bounded = ratio.clamp(1 - 0.2, 1 + 0.28)
    gain = torch.minimum(ratio * a, bounded * a)
    cut = bounded * a < ratio * a
    loss = -gain
    grad = torch.where(cut, torch.zeros_like(a), -a * ratio)
    kl = torch.zeros_like(x)
    if case["kl"]:
        gap = st["ref_logps"][rows, cols].to(torch.float64) - x
        kl = torch.expm1(gap) - gap
        loss = loss + case["kl"] * kl
        grad = grad - case["kl"] * torch.expm1(gap)
    n = max(1, rows.numel())
    per_row = torch.bincount(rows, minlength=case["batch"]).to(torch.float64).clamp_min(1.0)
    share = 1.0 / (per_row[rows] * case["batch"]) if case["reduction"] == "sequence" else 1.0 / n
    full = torch.zeros(st["labels"].shape, dtype=torch.float64, device=x.device)
    full[rows, cols] = grad * share
    return {"loss": (loss * share).sum(), "kl": kl.sum() / n,
            "clipped": cut.to(torch.float64).sum() / n, "dlogps": full}


def _exact_window(st):
    """Query blocks against the sinks and the keys that the block's windows reach."""
    case = st["case"]
    b, h, hk, s = case["batch"], case["heads"], case["kv_heads"], case["seq"]
    win, sinks, rep, f64 = case["window"], case["sinks"], h // hk, torch.float64
    q, k, v = (st[n].detach().to(f64) for n in ("q", "k", "v"))
    do = st["dout"].to(f64).transpose(1, 2)
    dev = q.device
    o, dq = torch.empty_like(q), torch.empty_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for lo in range(0, s, 1024):
        hi = min(s, lo + 1024)
        first = max(0, lo - win + 1)
        cols = torch.cat([torch.arange(0, min(sinks, first), device=dev),
                          torch.arange(first, hi, device=dev)])
        dist = torch.arange(lo, hi, device=dev)[:, None] - cols[None, :]
        hidden = (dist < 0) | ((dist >= win) & (cols[None, :] >= sinks))
        kk, vv = k[:, :, cols], v[:, :, cols]
        qb = q[:, :, lo:hi].reshape(b, hk, rep, hi - lo, -1)
        gb = do[:, :, lo:hi].reshape(b, hk, rep, hi - lo, -1)
        logits = torch.einsum("bgrid,bgjd->bgrij", qb, kk) * st["scale"]
        prob = torch.softmax(logits.masked_fill_(hidden, -math.inf), dim=-1)
        ob = torch.einsum("bgrij,bgjd->bgrid", prob, vv)
        o[:, :, lo:hi] = ob.reshape(b, h, hi - lo, -1)
        dv.index_add_(2, cols, torch.einsum("bgrij,bgrid->bgjd", prob, gb))
        dlog = torch.einsum("bgrid,bgjd->bgrij", gb, vv)
        dlog = prob * (dlog - (prob * dlog).sum(-1, keepdim=True)) * st["scale"]
        dq[:, :, lo:hi] = torch.einsum("bgrij,bgjd->bgrid", dlog, kk).reshape(b, h, hi - lo, -1)
        dk.index_add_(2, cols, torch.einsum("bgrij,bgrid->bgjd", dlog, qb))
    return {"out": o.transpose(1, 2), "dq": dq, "dk": dk, "dv": dv}


def _exact_swiglu8(st):
    def held(t):
        # the format's own definition: 32-bit absmax / 127 and 127 / absmax, nearest even code
        t = t.detach().float()
        out = torch.empty(t.shape, dtype=torch.float64, device=t.device)
        for blk, dst in zip(t.split(Q_BLOCK, dim=1), out.split(Q_BLOCK, dim=1)):
            top = blk.abs().amax(1, keepdim=True)
            most = torch.full_like(top, 127.0)
            inv = torch.where(top < 2.0 ** -100, torch.zeros_like(top), torch.div(most, top))
            dst.copy_(torch.round(blk * inv).to(torch.float64) * torch.div(top, most).to(torch.float64))
        return out

    g, u, dy = (st[n].detach().to(torch.float64) for n in ("gate", "up", "dy"))
    h = g * torch.sigmoid(g) * u
    gq, uq = held(st["gate"]), held(st["up"])
    s = torch.sigmoid(gq)
    return {"h": h, "dg": dy * uq * (s + gq * s * (1 - s)), "du": dy * gq * s}


_EXACT = {"logps": _exact_logps, "preference": _exact_preference, "policy": _exact_policy,
          "window": _exact_window, "swiglu8": _exact_swiglu8}


def exact(case, seed):
    with torch.enable_grad():
        return _EXACT[case["op"]](prepare(case, seed))
