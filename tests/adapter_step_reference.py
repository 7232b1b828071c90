"""Plain 64-bit forms of the operators of a step with several adapters, written from
their formulas, and error bounds that count roundings."""

import torch

BLOCK = 256


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def multi_lora(x, w, a, b, ids, scale, bias, dy=None):
    """(values, bounds) of y and, with dy, dx, da, db for x [T, K], ids [T]: every bound
    counts the outputs' rounding, the rounding of the rank products to bf16 and 2^-24 of
    the absolute sums for each term added."""
    f = torch.float64
    x, w, a, b, scale = (t.detach().to(f) for t in (x, w, a, b, scale))
    na, r, k = a.shape
    n = w.shape[0]
    h, e = half_step(torch.bfloat16), 2.0 ** -24
    af, bf = a.reshape(na * r, k), b.reshape(n, na * r)
    owner = torch.arange(na * r, device=x.device) // r
    sel = torch.where(owner[None] == ids[:, None], scale[owner][None], torch.zeros((), dtype=f, device=x.device))
    u, ua = (x @ af.t()) * sel, (x.abs() @ af.abs().t()) * sel.abs()
    y = x @ w.t() + u @ bf.t()
    ya = x.abs() @ w.abs().t()
    if bias is not None:
        y = y + bias.to(f)
        ya = ya + bias.to(f).abs()
    u_err = h * u.abs() + (k + 2) * e * (1 + h) * ua  # rounded, summed in 32 bits, scaled
    err = u_err @ bf.abs().t() + (k + 66 * 64) * e * (ya + u.abs() @ bf.abs().t())
    out = {"y": (y, (1 + h) * err + h * y.abs())}
    if dy is None:
        return out
    g = dy.detach().to(f)
    t = x.shape[0]
    v, va = (g @ bf) * sel, (g.abs() @ bf.abs()) * sel.abs()
    v_err = h * v.abs() + (n + 2) * e * (1 + h) * va
    dx = g @ w + v @ af
    err = v_err @ af.abs() + (n + 66 * 64) * e * (g.abs() @ w.abs() + v.abs() @ af.abs())
    out["dx"] = (dx, (1 + h) * err + h * dx.abs())
    da = v.t() @ x
    err = v_err.t() @ x.abs() + t * e * (v.abs().t() @ x.abs())
    out["da"] = (da.view(na, r, k), ((1 + h) * err + h * da.abs()).view(na, r, k))
    db = g.t() @ u
    err = g.abs().t() @ u_err + t * e * (g.abs().t() @ u.abs())
    out["db"] = (db.view(n, na, r), ((1 + h) * err + h * db.abs()).view(n, na, r))
    return out


def rotate(x, w, cos, sin, eps, g=None, angle_error=0.0):
    """(values, bounds) of the normalised (w not None) and rotated rows of x [B, H, S, D];
    cos, sin [B | 1, 1, S, D / 2] in 64 bits; with g also of dx and dw. 2^-24 for each
    addition of a row's sums and for each of the few products after them."""
    f = torch.float64
    dt, d = x.dtype, x.shape[-1]
    h, e = half_step(dt), (d + 16) * 2.0 ** -24
    if w is None:
        e = 4 * 2.0 ** -24
    x = x.detach().to(f)
    half = d // 2
    rstd = torch.ones_like(x[..., :1])
    hat = x
    if w is not None:
        rstd = 1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
        hat = x * rstd
    ww = torch.ones(d, dtype=f, device=x.device) if w is None else w.detach().to(f)
    n = hat * ww
    n1, n2 = n[..., :half], n[..., half:]
    y = torch.cat([n1 * cos - n2 * sin, n1 * sin + n2 * cos], -1)
    a = n1.abs() + n2.abs()
    top = torch.cat([a, a], -1)
    out = {"y": (y, h * y.abs() + (1 + h) * (e + angle_error) * top)}
    if g is None:
        return out
    g = g.detach().to(f)
    g1, g2 = g[..., :half], g[..., half:]
    dn = torch.cat([g1 * cos + g2 * sin, g2 * cos - g1 * sin], -1)
    ga = g1.abs() + g2.abs()
    dna = torch.cat([ga, ga], -1)  # bounds |dn|
    if w is None:
        out["dx"] = (dn, h * dn.abs() + (1 + h) * (e + angle_error) * dna)
        return out
    dx = rstd * (dn * ww - hat * (dn * ww * hat).mean(-1, keepdim=True))
    mag = rstd * (dna * ww.abs() + hat.abs() * (dna * ww.abs() * hat.abs()).mean(-1, keepdim=True))
    out["dx"] = (dx, h * dx.abs() + (1 + h) * (4 * e + 2 * angle_error) * mag)
    dw = (dn * hat).sum((0, 1, 2))
    count = x.numel() // d
    hw = half_step(w.dtype)
    err = (count * 2.0 ** -24 + 2 * e + angle_error) * (dna * hat.abs()).sum((0, 1, 2))
    out["dw"] = (dw, hw * dw.abs() + (1 + hw) * err)
    return out


def adamw(p, g, m, v, t, lr, betas, eps, wd, clip=1.0):
    """New (p, m, v) in 64 bits after step t."""
    f = torch.float64
    p, g, m, v = (x.detach().to(f) for x in (p, g, m, v))
    g = g * clip
    m = m + (1 - betas[0]) * (g - m)
    v = betas[1] * v + (1 - betas[1]) * g * g
    upd = lr / (1 - betas[0] ** t) * m / (torch.sqrt(v / (1 - betas[1] ** t)) + eps)
    return p * (1 - lr * wd) - upd, m, v, upd


def check(name, got, ref):
    """got within the bounds of ref = (value, bound), everywhere."""
    value, bound = ref
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got.detach().to(torch.float64) - value).abs()
    # 1 % for the bounds' own second-order terms, and the smallest numbers of a type
    over = off - 1.01 * bound - 1e-30
    assert torch.isfinite(got).all(), name
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 0.0, (name, worst, float(off.max()), float((off / (bound + 1e-300)).max()))
