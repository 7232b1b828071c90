"""Plain 64-bit forms of the preference / policy tuning operators, for the tests."""

import math

import torch

IGNORE = -100


def logps64(hidden, weight, labels, g=None):
    """(logps, entropies, softmax, dhidden, dweight) in 64 bits; g: dL/dlogps."""
    h = hidden.detach().reshape(-1, hidden.shape[-1]).double()
    w = weight.detach().double()
    t = labels.reshape(-1)
    keep = t != IGNORE
    z = h @ w.t()
    lsm = z - torch.logsumexp(z, 1, keepdim=True)
    p = lsm.exp()
    idx = torch.where(keep, t, torch.zeros_like(t))
    zero = torch.zeros(len(t), dtype=torch.float64, device=h.device)
    lp = torch.where(keep, lsm.gather(1, idx[:, None])[:, 0], zero)
    ent = torch.where(keep, -(p * lsm).sum(1), zero)
    if g is None:
        return lp, ent, p, None, None
    gk = torch.where(keep, g.reshape(-1).double(), zero)
    dz = -p * gk[:, None]
    dz[torch.arange(len(t), device=h.device), idx] += gk
    return lp, ent, p, dz @ w, dz.t() @ h


def preference64(x, ref, labels, beta, smoothing, kind):
    """(loss, chosen rewards, rejected rewards, dloss/dx) in 64 bits."""
    x = x.detach().double().requires_grad_(True)
    keep = labels != IGNORE
    zero = torch.zeros_like(x)
    r = torch.where(keep, x, zero).sum(1)
    if ref is not None:
        r = r - (torch.where(keep, ref.double(), zero).sum(1) if ref.dim() == 2 else ref.double())
    n = r.shape[0] // 2
    s = r / keep.sum(1).clamp(min=1) if kind == "ipo" else r
    h = s[:n] - s[n:]
    if kind == "sigmoid":
        loss = (-(1 - smoothing) * torch.nn.functional.logsigmoid(beta * h)
                - smoothing * torch.nn.functional.logsigmoid(-beta * h))
    elif kind == "hinge":
        loss = torch.relu(1 - beta * h)
    else:
        loss = (h - 1 / (2 * beta)) ** 2
    loss = loss.mean()
    (grad,) = torch.autograd.grad(loss, [x])
    r = (beta * r).detach()
    return loss.detach(), r[:n], r[n:], grad


def policy64(x, adv, labels, old, ref, lo, hi, c, reduction):
    """(loss, kl, clipped, dloss/dx, size of dloss/dx's terms) in 64 bits."""
    keep = labels != IGNORE
    zero = torch.zeros(x.shape, dtype=torch.float64, device=x.device)

    def pick(t):
        return torch.where(keep, t.detach().double(), zero)

    x64 = pick(x)
    a = pick(adv if adv.dim() == 2 else adv[:, None].expand(x.shape))
    delta = x64 - pick(old) if old is not None else zero
    r = delta.exp()
    cut = keep & (((a > 0) & (r > 1 + hi)) | ((a < 0) & (r < 1 - lo)))
    tok = -torch.minimum(r * a, r.clamp(1 - lo, 1 + hi) * a)
    grad = torch.where(cut, zero, -a * r)
    size = (a * r).abs()
    kl = zero
    if ref is not None:
        d = pick(ref) - x64
        kl = torch.expm1(d) - d
        tok = tok + c * kl
        grad = grad - c * torch.expm1(d)
        size = size + c * torch.expm1(d).abs()
    cnt = keep.sum(1, keepdim=True).double()
    total = cnt.sum().clamp(min=1)
    w = 1 / total if reduction == "token" else 1 / (cnt.clamp(min=1) * x.shape[0])
    w = torch.where(keep, w.expand(x.shape) if w.dim() else w, zero)
    return ((tok * w).sum(), torch.where(keep, kl, zero).sum() / total, cut.double().sum() / total,
            grad * w, size * w)


def window64(q, k, v, do, scale, window, sinks):
    """out, dq, dk, dv and, per output, a bound of the bf16 kernel's error in 64 bits.

    The kernel rounds P, dS and the outputs to bf16 (half a step: 2^-8 of the value)
    and takes D = rowsum(dO O) from the rounded O; its other arithmetic is fp32 with a
    base-2 exponential good to 2^-22 of an exponent of at most about 2^7, i.e. 2^-15
    of P, well below 2^-8."""
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    B, H, S, D = q.shape
    rep = H // k.shape[1]
    kk, vv = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    i = torch.arange(S, device=q.device)
    dist = i[:, None] - i[None, :]
    seen = (dist >= 0) & ((dist < window) | (i[None, :] < sinks))
    p = torch.softmax((q @ kk.transpose(2, 3) * scale).masked_fill(~seen, -math.inf), -1)
    o = p @ vv
    g = do.transpose(1, 2)
    dp = g @ vv.transpose(2, 3)
    dsum = (g * o).sum(-1, keepdim=True)
    ds = p * (dp - dsum)
    u = 2.0 ** -8 * 1.03
    e_o = u * (p @ vv.abs() + o.abs())
    e_ds = u * (ds.abs() + p * ((g.abs() * o.abs()).sum(-1, keepdim=True)
                                + dp.abs() * 2.0 ** -6 + dsum.abs() * 2.0 ** -6))
    e_p = u * p

    def grouped(t):
        return t.view(B, H // rep, rep, S, D).sum(2)

    dq, e_dq = ds @ kk * scale, e_ds @ kk.abs() * scale
    dk, e_dk = grouped(ds.transpose(2, 3) @ q * scale), grouped(e_ds.transpose(2, 3) @ q.abs() * scale)
    dv, e_dv = grouped(p.transpose(2, 3) @ g), grouped(e_p.transpose(2, 3) @ g.abs())
    val = (o.transpose(1, 2), dq, dk, dv)
    bound = (e_o.transpose(1, 2), e_dq + u * dq.abs(), e_dk + u * dk.abs(), e_dv + u * dv.abs())
    return val, bound


def kept8(x):
    """What the 8-bit codes of x [rows, n] stand for (fp32 arithmetic of the format)."""
    out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    for c in range(0, x.shape[1], 64):
        b = x[:, c:c + 64].detach().float()
        top = b.abs().amax(1, keepdim=True)
        most = torch.full_like(top, 127.0)  # torch divides by a plain number through its reciprocal
        inv = torch.where(top < 2.0 ** -100, torch.zeros_like(top), most / top)
        out[:, c:c + 64] = torch.round(b * inv) * (top / most)
    return out


def swiglu64(g, u, dy):
    g, u, dy = (t.double() for t in (g, u, dy))
    s = torch.sigmoid(g)
    return g * s * u, dy * u * s * (1 + g * (1 - s)), dy * g * s, (dy * u * s).abs() * (1 + g.abs())
