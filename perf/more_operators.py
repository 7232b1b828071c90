"""Measured cases of the operators around a step of many adapters on one base model.

* ``adapters``  a shared frozen projection with the low-rank adapters of many
                requests beside it: single tokens (no gradient) and training
                batches (forward and backward);
* ``qknorm``    norms of queries and keys for each head with the rotation in the
                same pass, from cos / sin tables, forward and backward;
* ``axes``      rotary positions with several axes (time, height, width), angles
                formed from the positions, with or without the norms;
* ``adamw``     one AdamW step over many tensors, states in 8 or 32 bits, with the
                gradients' global norm clipped.

``run`` computes the plain form (elementary torch operations in 32 or 64 bits,
rounded once at the end) unless ``own`` is set; then it makes the calls that a
user makes of the framework.
"""

import math

import numpy as np
import torch

own = False

STATE_BLOCK = 256  # elements that share one scale of an 8-bit optimiser state
LR, BETAS, EPS, DECAY = 2e-4, (0.9, 0.999), 1e-8, 0.01

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # a few requests' next tokens through the q/k/v projection: the smallest call, latency counts
        {"name": "adapters_few", "op": "adapters", "tokens": 4, "requests": 4, "adapters": 8, "rank": 16,
         "in": 1536, "out": 2048, "bias": True, "train": False},
        # 48 requests' next tokens, each with its own adapter of 64, through gate/up
        {"name": "adapters_tokens", "op": "adapters", "tokens": 48, "requests": 48, "adapters": 64, "rank": 16,
         "in": 1536, "out": 17920, "bias": False, "train": False},
        # requests of ragged lengths, some without an adapter, down projection, trained
        {"name": "adapters_ragged", "op": "adapters", "tokens": 2999, "requests": 21, "adapters": 24, "rank": 8,
         "in": 8960, "out": 1536, "bias": False, "train": True},
        # four adapters trained at once on the step's 4 x 2048 tokens, gate/up
        {"name": "adapters_step", "op": "adapters", "tokens": 8192, "requests": 8, "adapters": 4, "rank": 16,
         "in": 1536, "out": 17920, "bias": False, "train": True},
        # the next tokens of 32 requests: latency counts
        {"name": "qknorm_tokens", "op": "qknorm", "batch": 32, "seq": 1, "heads": 12, "kv_heads": 2, "dim": 128,
         "dtype": "bf16", "train": False},
        # the step's 4 x 2048 tokens
        {"name": "qknorm_step", "op": "qknorm", "batch": 4, "seq": 2048, "heads": 12, "kv_heads": 2, "dim": 128,
         "dtype": "bf16", "train": True},
        # long documents of odd length, many heads
        {"name": "qknorm_long", "op": "qknorm", "batch": 2, "seq": 16001, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "train": True},
        # short prompts with an image each, small heads, rotation alone
        {"name": "axes_image", "op": "axes", "batch": 4, "seq": 1111, "heads": 14, "kv_heads": 2, "dim": 64,
         "dtype": "f16", "norm": False, "interleaved": True, "start": 0, "train": True},
        # a long video after a long text: far positions, norms too
        {"name": "axes_video", "op": "axes", "batch": 1, "seq": 24000, "heads": 12, "kv_heads": 2, "dim": 128,
         "dtype": "bf16", "norm": True, "interleaved": False, "start": 90000, "train": True},
        # the trained norm weights of 28 layers: many tiny tensors, latency counts
        {"name": "adamw_norms", "op": "adamw", "kind": "rows", "tensors": 57, "size": 1536, "dtype": "f32",
         "bits": 32, "clip": True},
        # the rank-16 factors of every projection of the 28 layers
        {"name": "adamw_lora", "op": "adamw", "kind": "lora", "tensors": 392, "size": 16, "dtype": "f32",
         "bits": 8, "clip": True},
        # a trained head beside its norm
        {"name": "adamw_head", "op": "adamw", "kind": "head", "tensors": 2, "size": 1536, "dtype": "bf16",
         "bits": 8, "clip": False},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adapters", "qknorm", "axes", "adamw"])
    if op == "adapters":
        train = rng.random() < 0.6
        tokens = _log_uniform(rng, 33, 4000) if train else _log_uniform(rng, 1, 200)
        return {"op": op, "tokens": tokens, "requests": min(tokens, _log_uniform(rng, 1, 40 if train else 200)),
                "adapters": _log_uniform(rng, 1, 64), "rank": rng.choice([8, 16, 24, 32]),
                "in": 8 * _log_uniform(rng, 8, 640), "out": 8 * _log_uniform(rng, 8, 1120),
                "bias": rng.random() < 0.5, "train": train}
    if op in ("qknorm", "axes"):
        kv = rng.choice([1, 2, 4, 8])
        train = rng.random() < 0.7
        c = {"op": op, "batch": rng.randint(1, 4) if train else _log_uniform(rng, 1, 200),
             "seq": _log_uniform(rng, 3, 6000) if train else 1, "heads": kv * rng.choice([1, 3, 4, 7]),
             "kv_heads": kv, "dim": rng.choice([64, 96, 128, 256]),
             "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "train": train}
        if op == "axes":
            c.update(norm=rng.random() < 0.5, interleaved=rng.random() < 0.5,
                     start=rng.choice([0, 1000, 100000]))
        return c
    kind = rng.choice(["rows", "lora", "head"])
    size = {"rows": _log_uniform(rng, 65, 9000), "lora": rng.choice([8, 16, 32]),
            "head": _log_uniform(rng, 100, 1536)}[kind]
    return {"op": op, "kind": kind, "tensors": {"rows": _log_uniform(rng, 2, 400), "lora": 14 * rng.randint(1, 28),
                                                "head": 2}[kind],
            "size": size, "dtype": rng.choice(["f32", "bf16"]) if kind != "lora" else "f32",
            "bits": rng.choice([8, 32]), "clip": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs ----
def _request_lengths(tokens, requests, seed):
    """Ragged lengths of at least one token."""
    rs = np.random.RandomState(seed % (2 ** 31))
    cuts = np.sort(rs.choice(tokens - 1, requests - 1, replace=False)) + 1 if requests > 1 else np.zeros(0, int)
    return np.diff(np.concatenate([[0], cuts, [tokens]]))


def _axis_of(half, interleaved):
    """(sections, axis of each frequency) of time, height and width."""
    h = 3 * half // 8
    sections = (half - 2 * h, h, h)
    if not interleaved:
        return sections, np.repeat(np.arange(3), sections)
    i = np.arange(half)
    axis = np.where((i % 3 != 0) & (i < 3 * h), i % 3, 0)
    return sections, axis


def _positions(case, seed):
    """[3, batch, seq]: a text, then the patches of an image or a video, row by row."""
    b, s, start = case["batch"], case["seq"], case["start"]
    rs = np.random.RandomState(seed % (2 ** 31))
    out = np.empty((3, b, s), np.int64)
    for i in range(b):
        text = int(rs.randint(0, s // 4 + 1))
        n = np.arange(s)
        first = start + text
        w = int(rs.randint(4, 40))
        h = int(rs.randint(4, 40))
        p = n - text
        out[0, i] = np.where(p < 0, start + n, first + p // (w * h))
        out[1, i] = np.where(p < 0, start + n, first + p // w % h)
        out[2, i] = np.where(p < 0, start + n, first + p % w)
    return torch.from_numpy(out)


def _tensor_shapes(case):
    k, n = case["kind"], case["tensors"]
    if k == "rows":
        return [(case["size"],)] * n
    if k == "lora":
        r = case["size"]
        layer = [(1536, 1536), (1536, 256), (1536, 256), (1536, 1536), (1536, 8960), (1536, 8960), (8960, 1536)]
        both = [s for i, o in layer for s in ((r, i), (o, r))]
        return [both[j % len(both)] for j in range(n)]
    return [(151936, case["size"]), (case["size"],)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    op = case["op"]
    st = {"case": case}
    bf16 = torch.bfloat16
    if op == "adapters":
        t, k, n, na, r = case["tokens"], case["in"], case["out"], case["adapters"], case["rank"]
        rs = np.random.RandomState(seed % (2 ** 31))
        lengths = _request_lengths(t, case["requests"], seed)
        # as many different adapters as there are, then any; one request in eight uses none
        ids = rs.permutation(np.arange(len(lengths)) % na)
        ids = np.where(rs.rand(len(lengths)) < 0.125, -1, ids)
        st["ids"] = torch.from_numpy(np.repeat(ids, lengths)).to(dev)
        grad = own and case["train"]
        st["x"] = randn(t, k, dtype=bf16).requires_grad_(grad)
        st["weight"] = randn(n, k, dtype=bf16).mul_(0.02)
        st["a"] = randn(na, r, k, dtype=bf16).mul_(k ** -0.5).requires_grad_(grad)
        st["b"] = randn(n, na, r, dtype=bf16).mul_(0.05).requires_grad_(grad)
        st["scaling"] = 0.5 + 2.0 * torch.rand(na, generator=g, device=dev)
        st["bias"] = randn(n, dtype=bf16) if case["bias"] else None
        if case["train"]:
            st["dy"] = randn(t, n, dtype=bf16)
    elif op in ("qknorm", "axes"):
        b, s, h, hk, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
        dt = _DTYPES[case["dtype"]]
        grad = own and case["train"]
        # column ranges of one projection [B, S, (h + 2 hk) D], as a grouped q/k/v product hands them over
        both = randn(b, s, (h + 2 * hk) * d, dtype=dt)
        st["q"] = both[..., :h * d].view(b, s, h, d).transpose(1, 2).requires_grad_(grad)
        st["k"] = both[..., h * d:(h + hk) * d].view(b, s, hk, d).transpose(1, 2).requires_grad_(grad)
        if op == "qknorm" or case["norm"]:
            st["qw"] = (1 + 0.2 * randn(d)).to(dt).requires_grad_(grad)
            st["kw"] = (1 + 0.2 * randn(d)).to(dt).requires_grad_(grad)
        inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device=dev).float() / d))
        if op == "qknorm":
            first = torch.randint(0, 30000, (b, 1), generator=g, device=dev) if s == 1 else \
                torch.zeros(b, 1, dtype=torch.int64, device=dev)
            ang = (first + torch.arange(s, device=dev)).double()[..., None] * inv.double()
            st["cos"] = torch.cat([ang.cos()] * 2, -1).to(dt)
            st["sin"] = torch.cat([ang.sin()] * 2, -1).to(dt)
        else:
            st["positions"] = _positions(case, seed).to(dev)
            st["inv_freq"] = inv
            st["sections"], axis = _axis_of(d // 2, case["interleaved"])
            st["axis"] = torch.from_numpy(axis).to(dev)
        if case["train"]:
            # gradients as attention hands them back: [B, heads, S, D]
            st["dq"], st["dk"] = randn(b, h, s, d, dtype=dt), randn(b, hk, s, d, dtype=dt)
    else:
        _prepare_adamw(st, case, randn)
    return st


def _prepare_adamw(st, case, randn):
    dt = _DTYPES[case["dtype"]]
    shapes = _tensor_shapes(case)
    sizes = np.array([int(np.prod(s)) for s in shapes], np.int64)
    blocks = -(-sizes // STATE_BLOCK)
    offs = np.concatenate([[0], np.cumsum(blocks)]) * STATE_BLOCK
    total = int(offs[-1])
    # parameters and gradients are views of two buffers, as the trainer lays them out;
    # each tensor starts at a whole block, and what lies between the tensors is 0
    p, gr = randn(total, dtype=dt).mul_(0.02), randn(total, dtype=dt).mul_(1e-3)
    m, v = randn(total).mul_(3e-4), randn(total).mul_(1e-3).square_()
    if case["kind"] == "head":  # embedding rows that rarely occur: tiny second moments beside large ones
        rare = 10.0 ** (-2.0 * randn(total // 64 + 1).abs().clamp_(max=3.0)).repeat_interleave(64)[:total]
        v.mul_(rare)
        m.mul_(rare.sqrt_())
    used = torch.zeros(total, dtype=torch.bool, device=p.device)
    view = []
    for s, o, k in zip(shapes, offs, sizes):
        used[int(o):int(o + k)] = True
        view.append((int(o), int(k), s))
    for t in (p, gr, m, v):
        t.masked_fill_(~used, 0)
    st.update(flat_param=p, flat_grad=gr, step=torch.full((), 7.0, device=p.device))
    if case["bits"] == 8:
        st["m"], st["m_scale"] = _to_8bit(m)
        st["v"], st["v_scale"] = _root_to_8bit(v)
    else:
        st["m"], st["v"] = m, v
    if own:
        from auspex_soup_demo_b200.optim import MultiTensorAdamW

        params = []
        for o, k, s in view:
            q = torch.nn.Parameter(p[o:o + k].view(s))
            q.grad = gr[o:o + k].view(s)
            params.append(q)
        opt = MultiTensorAdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
                               state_bits=case["bits"], max_grad_norm=1.0 if case["clip"] else None)
        held = opt.flat_state()
        for name in ("m", "v", "m_scale", "v_scale"):
            if name in st:
                held[name].copy_(st[name].view(held[name].shape))
        held["step"].copy_(st["step"])
        st["opt"], st["held"] = opt, held


# --------------------------------------------------------------- own calls ----
def _run_own(st):
    from auspex_soup_demo_b200 import kernels

    case = st["case"]
    op = case["op"]
    if op == "adapters":
        args = (st["x"], st["weight"], st["a"], st["b"], st["ids"], st["scaling"], st["bias"])
        if not case["train"]:
            return {"y": kernels.multi_lora_linear(*args)}
        y = kernels.multi_lora_linear(*args)
        dx, da, db = torch.autograd.grad(y, [st["x"], st["a"], st["b"]], st["dy"])
        return {"y": y.detach(), "dx": dx, "da": da, "db": db}
    if op == "adamw":
        st["opt"].step()
        return _adamw_out(st, st["held"])
    if op == "qknorm":
        q, k = kernels.apply_qk_norm_rope(st["q"], st["k"], st["qw"], st["kw"], st["cos"], st["sin"])
    else:
        q, k = kernels.apply_multi_axis_rope(
            st["q"], st["k"], st["positions"], st["inv_freq"],
            kernels.rope_axes(st["sections"], st["case"]["interleaved"]), st.get("qw"), st.get("kw"))
    if not case["train"]:
        return {"q": q, "k": k}
    names = [n for n in ("q", "k", "qw", "kw") if n in st]
    grads = torch.autograd.grad([q, k], [st[n] for n in names], [st["dq"], st["dk"]])
    return {"q": q.detach(), "k": k.detach(), **{"d" + n: x for n, x in zip(names, grads)}}


def _adamw_out(st, held):
    out = {"param": st["flat_param"], "m": held["m"].reshape(-1), "v": held["v"].reshape(-1)}
    if st["case"]["bits"] == 8:
        out.update(m_scale=held["m_scale"].reshape(-1), v_scale=held["v_scale"].reshape(-1))
    return out


# -------------------------------------------------------------- plain form ----
def _plain_adapters(st):
    case = st["case"]
    x, w = st["x"].detach().float(), st["weight"].float()
    na, r = case["adapters"], case["rank"]
    a = st["a"].detach().float().reshape(na * r, -1)
    b = st["b"].detach().float().reshape(-1, na * r)
    ids = st["ids"]
    owner = torch.arange(na * r, device=x.device) // r
    sel = torch.where(owner[None, :] == ids[:, None], st["scaling"][owner][None, :], 0.0)
    xa = (x @ a.t()) * sel
    y = x @ w.t() + xa @ b.t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    out = {"y": y.to(torch.bfloat16)}
    if case["train"]:
        dy = st["dy"].float()
        dxa = (dy @ b) * sel
        out["dx"] = (dy @ w + dxa @ a).to(torch.bfloat16)
        out["da"] = (dxa.t() @ x).to(torch.bfloat16).view(st["a"].shape)
        out["db"] = (dy.t() @ xa).to(torch.bfloat16).view(st["b"].shape)
    return out


def _plain_rotate(st, cos, sin, eps=1e-6):
    """Norm (where there are weights) and rotation of q and k, and their gradients."""
    out = {}
    for n in ("q", "k"):
        x = st[n].detach().float()
        half = x.shape[-1] // 2
        w = st[n + "w"].detach().float() if n + "w" in st else None
        if w is not None:
            rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
            hat = x * rstd
            y = hat * w
        else:
            y = x
        y1, y2 = y[..., :half], y[..., half:]
        out[n] = torch.cat([y1 * cos - y2 * sin, y1 * sin + y2 * cos], -1).to(st[n].dtype)
        if not st["case"]["train"]:
            continue
        g = st["d" + n].float()
        g1, g2 = g[..., :half], g[..., half:]
        g = torch.cat([g1 * cos + g2 * sin, g2 * cos - g1 * sin], -1)
        if w is not None:
            out["d" + n + "w"] = (g * hat).sum((0, 1, 2), dtype=torch.float64).to(st[n + "w"].dtype)
            g = g * w
            g = rstd * (g - hat * (g * hat).mean(-1, keepdim=True))
        out["d" + n] = g.to(st[n].dtype)
    return out


def _plain_qknorm(st):
    half = st["case"]["dim"] // 2
    return _plain_rotate(st, st["cos"][:, None, :, :half].float(), st["sin"][:, None, :, :half].float())


def _plain_axes(st):
    # angles of far positions in 64 bits
    pos = st["positions"].permute(1, 2, 0)[..., st["axis"]].double()
    ang = (pos * st["inv_freq"].double())[:, None]
    return _plain_rotate(st, torch.cos(ang).float(), torch.sin(ang).float())


def _to_8bit(x):
    """(e4m3 values, scales) of blocks of STATE_BLOCK that share absmax / 448."""
    x = x.view(-1, STATE_BLOCK)
    scale = x.abs().max(1, keepdim=True).values / torch.full((1, 1), 448.0, device=x.device)
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    return y.to(torch.float8_e4m3fn), scale


def _root_to_8bit(v):
    """The same of second moments, held as their square roots. One that is not 0 does
    not become 0: beside a first moment that is not 0 it would make a huge step."""
    x = torch.sqrt(v).view(-1, STATE_BLOCK)
    code, scale = _to_8bit(x)
    least = torch.full((1, 1), 2.0 ** -9, device=x.device).to(code.dtype)
    return torch.where((x > 0) & (code.float() == 0), least, code), scale


def _from_8bit(code, scale):
    return (code.view(-1, STATE_BLOCK).float() * scale.view(-1, 1)).view(-1)


def _plain_adamw(st):
    case = st["case"]
    p, g = st["flat_param"], st["flat_grad"].float()
    (b1, b2), eight = BETAS, case["bits"] == 8
    if case["clip"]:
        norm = torch.sqrt((g.double() * g.double()).sum())
        g = g * torch.clamp(1.0 / (norm + 1e-6), max=1.0).float()
    m = _from_8bit(st["m"], st["m_scale"]) if eight else st["m"]
    v = _from_8bit(st["v"], st["v_scale"]) if eight else st["v"]
    if eight:
        v = v * v
    st["step"] += 1
    t = st["step"].double()
    m = m + (1 - b1) * (g - m)
    v = b2 * v + (1 - b2) * (g * g)
    step_size = (LR / (1 - b1 ** t)).float()
    root = torch.sqrt(v) * (1.0 / torch.sqrt(1 - b2 ** t)).float()
    new = p.float() * (1 - LR * DECAY) - step_size * m / (root + EPS)
    p.copy_(new)
    if eight:
        for n, held in (("m", _to_8bit(m)), ("v", _root_to_8bit(v))):
            st[n].copy_(held[0])
            st[n + "_scale"].copy_(held[1])
    else:
        st["m"].copy_(m)
        st["v"].copy_(v)
    return _adamw_out(st, st)


_PLAIN = {"adapters": _plain_adapters, "qknorm": _plain_qknorm, "axes": _plain_axes, "adamw": _plain_adamw}


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------- work ----
def work(case):
    op = case["op"]
    if op == "adapters":
        t, k, n, r = case["tokens"], case["in"], case["out"], case["rank"]
        used = min(case["adapters"], case["requests"])
        factors = 2.0 * used * r * (k + n)
        nbytes = 2.0 * n * k + 2.0 * t * (k + n) + factors + 8.0 * t
        flops = 2.0 * t * n * k + 2.0 * t * r * (k + n)
        if case["train"]:
            # backward: dy, W and the factors read, dx and the factors' gradients (of every adapter) written
            nbytes += 2.0 * n * k + 2.0 * t * (2 * k + n) + factors + 2.0 * case["adapters"] * r * (k + n)
            flops += 2.0 * t * n * k + 6.0 * t * r * (k + n) - 2.0 * t * r * k
        return {"bytes": nbytes, "flops": flops}
    if op in ("qknorm", "axes"):
        tok = float(case["batch"] * case["seq"])
        es = _DTYPES[case["dtype"]].itemsize
        rows = tok * (case["heads"] + case["kv_heads"]) * case["dim"] * es
        table = tok * (case["dim"] * es if op == "qknorm" else 24.0)  # half of cos and of sin, or three positions
        norm = op == "qknorm" or case["norm"]
        passes = 2 + ((3 if norm else 2) if case["train"] else 0)
        return {"bytes": passes * rows + table * (2 if case["train"] else 1),
                "flops": (10.0 + (25.0 if case["train"] else 0.0)) * rows / es}
    n = float(sum(int(np.prod(s)) for s in _tensor_shapes(case)))
    es = _DTYPES[case["dtype"]].itemsize
    state = 4.0 * (1 + 4.0 / STATE_BLOCK) if case["bits"] == 8 else 16.0
    return {"bytes": n * (3 * es + state), "flops": 20.0 * n}


# ------------------------------------------------------------------ exact ----
def _exact_adapters(st):
    case, f64 = st["case"], torch.float64
    x, w = st["x"].detach().to(f64), st["weight"].to(f64)
    a, b = st["a"].detach().to(f64), st["b"].detach().to(f64)
    y = torch.mm(x, w.T)
    if st["bias"] is not None:
        y += st["bias"].to(f64)
    dy = st["dy"].to(f64) if case["train"] else None
    dx = torch.mm(dy, w) if case["train"] else None
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for i in range(case["adapters"]):
        rows = torch.nonzero(st["ids"] == i).squeeze(1)
        if not rows.numel():
            continue
        s = st["scaling"][i].to(f64)
        low = torch.mm(x[rows], a[i].T)
        y[rows] += s * torch.mm(low, b[:, i].T)
        if case["train"]:
            up = s * torch.mm(dy[rows], b[:, i])
            dx[rows] += torch.mm(up, a[i])
            da[i] = torch.mm(up.T, x[rows])
            db[:, i] = s * torch.mm(dy[rows].T, low)
    return {"y": y, "dx": dx, "da": da, "db": db} if case["train"] else {"y": y}


def _exact_heads(st):
    """Rotation as a complex product, gradients by automatic differentiation, in 64 bits."""
    case = st["case"]
    half = case["dim"] // 2
    if case["op"] == "qknorm":
        unit = torch.complex(st["cos"][..., :half].double(), st["sin"][..., :half].double())
    else:
        pos = torch.stack([st["positions"][int(j)] for j in st["axis"].tolist()], -1).double()
        unit = torch.polar(torch.ones_like(pos), pos * st["inv_freq"].double())
    unit = unit.unsqueeze(1)
    out = {}
    for n in ("q", "k"):
        x = st[n].detach().double().requires_grad_(case["train"])
        w = st[n + "w"].detach().double().requires_grad_(case["train"]) if n + "w" in st else None
        y = x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        z = torch.complex(y[..., :half], y[..., half:]) * unit
        y = torch.cat([z.real, z.imag], -1)
        out[n] = y.detach()
        if case["train"]:
            leaves = [x] if w is None else [x, w]
            for name, gr in zip((n, n + "w"), torch.autograd.grad(y, leaves, st["d" + n].double())):
                out["d" + name] = gr
    return out


def _exact_adamw(st):
    case, f64 = st["case"], torch.float64
    g = st["flat_grad"].to(f64)
    if case["clip"]:
        g = g * min(1.0, 1.0 / (float(torch.linalg.vector_norm(g)) + 1e-6))
    if case["bits"] == 8:
        m, r = ((st[n].to(f64).view(-1, STATE_BLOCK) * st[n + "_scale"].to(f64).view(-1, 1)).flatten()
                for n in ("m", "v"))
        v = r.square()
    else:
        m, v = st["m"].to(f64), st["v"].to(f64)
    t = int(st["step"]) + 1
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * g.square()
    m_hat, v_hat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
    p = st["flat_param"].to(f64) * (1 - LR * DECAY) - LR * m_hat / (v_hat.sqrt() + EPS)
    if case["bits"] == 32:
        return {"param": p, "m": m, "v": v}
    # the new states are rounded to 8 bits: only their scales have values of their own
    return {"param": p, "m": None, "v": None,
            "m_scale": m.view(-1, STATE_BLOCK).abs().amax(1) / 448,
            "v_scale": v.view(-1, STATE_BLOCK).amax(1).sqrt() / 448}


_EXACT = {"adapters": _exact_adapters, "qknorm": _exact_heads, "axes": _exact_heads, "adamw": _exact_adamw}


def exact(case, seed):
    with torch.enable_grad():
        return _EXACT[case["op"]](prepare(case, seed))
