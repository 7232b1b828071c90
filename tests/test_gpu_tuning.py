"""The preference / policy tuning operators on the GPU against plain 64-bit forms.

Tolerances follow from the arithmetic: a rounding to type t is off by at most
half a step, eps(t) / 2 of the value (bf16 2^-8, fp16 2^-11, fp32 2^-24); each
test states which roundings its bound counts.
"""

import math

import pytest
import torch

import tuning_reference as ref64
from auspex_soup_demo_b200 import _lib, kernels
from auspex_soup_demo_b200.kernels import chunked_ce

pytestmark = pytest.mark.gpu

IGNORE = -100
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _labels(n, s, v, g, keep=0.6):
    ids = torch.randint(0, v, (n, s), generator=g, device=DEV)
    return torch.where(torch.rand(n, s, generator=g, device=DEV) < keep, ids, torch.full_like(ids, IGNORE))


def _within(a, b, tol, name):
    bad = ((a.double() - b).abs() - tol)
    assert not torch.isnan(bad).any(), name
    assert float(bad.max()) <= 0, (name, float(bad.max()), float((a.double() - b).abs().max()))


# ------------------------------------------------------------- log-probabilities --
def _logps_inputs(n, d, v, dtype=torch.bfloat16, seed=0, keep=0.6):
    g = _gen(seed)
    w = (torch.randn(v, d, generator=g, device=DEV) * 0.05).to(dtype)
    lab = _labels(1, n, v, g, keep)[0]
    lift = 8 * torch.rand(n, 1, generator=g, device=DEV) / (d * 0.0025)
    h = (torch.randn(n, d, generator=g, device=DEV) + lift * w[lab.clamp(min=0)].float()).to(dtype)
    return h, w, lab, torch.randn(n, generator=g, device=DEV)


def _logps_check(h, w, lab, up, out, grads):
    lp, ent, p, dh, dw = ref64.logps64(h, w, lab, up)
    h2, w2 = h.detach().double().reshape(-1, h.shape[-1]), w.detach().double()
    d = h2.shape[1]
    # fp32 accumulation of d products (random signs of the roundings), then lse in fp32
    mag = float((h2.abs() @ w2.abs().t()).max())
    tol = 4 * math.sqrt(d) * 2.0 ** -24 * mag + 2.0 ** -20 * (1 + lp.abs())
    _within(out[0].reshape(-1), lp, tol, "logps")
    _within(out[1].reshape(-1), ent, 16 * tol, "entropies")  # weighted by |z - lse|, below 16 here
    t = lab.reshape(-1)
    gk = torch.where(t != IGNORE, up.reshape(-1).double(), torch.zeros_like(lp)).abs()
    pt = p.clone()
    rows = torch.arange(len(t), device=DEV)
    idx = t.clamp(min=0)
    pt[rows, idx] = 1 - pt[rows, idx]
    dz = pt * gk[:, None]  # |dz|
    u = 2.0 ** -8 * 1.02
    # dz's factor is rounded to bf16 (and, for fp16 operands, the weight), the result to its dtype
    wr = 2 if h.dtype != torch.bfloat16 else 1
    end = torch.finfo(h.dtype).eps / 2
    _within(grads[0].reshape(-1, d), dh, wr * u * (dz @ w2.abs()) + end * dh.abs() + 1e-7, "dhidden")
    if len(grads) > 1:  # the scaled hidden rows are rounded to bf16 too
        _within(grads[1], dw, 2 * u * (dz.t() @ h2.abs()) + torch.finfo(w.dtype).eps / 2 * dw.abs() + 1e-7,
                "dweight")


@pytest.mark.parametrize("n,d,v,dtype", [
    (1, 64, 300, torch.bfloat16),       # one token, an odd vocabulary
    (77, 72, 1000, torch.bfloat16),     # ragged rows and width
    (300, 128, 4099, torch.bfloat16),   # over one row tile, odd vocabulary
    (513, 256, 2048, torch.bfloat16),
    (130, 64, 777, torch.float16),
    (70, 64, 500, torch.float32),
])
@pytest.mark.parametrize("train_head", [False, True])
def test_head_token_logps(n, d, v, dtype, train_head):
    h, w, lab, up = _logps_inputs(n, d, v, dtype, seed=n + v)
    if dtype == torch.float32:  # operands are rounded to fp16: start from values that are
        h, w = h.half().float(), w.half().float()
    h.requires_grad_(True)
    w.requires_grad_(train_head)
    out = kernels.head_token_logps(h, w, lab)
    grads = torch.autograd.grad(out[0], [h] + [w] * train_head, up)
    assert _lib.device_error(h.device) == 0
    if dtype == torch.float32:  # compared to bf16 rounding, the formula's own error
        grads = tuple(t.clone() for t in grads)
    assert out[0].dtype == out[1].dtype == torch.float32 and grads[0].dtype == dtype
    assert not out[1].requires_grad
    _logps_check(h, w, lab, up, out, grads)


def test_head_token_logps_shapes_modules_and_labels():
    h, w, lab, up = _logps_inputs(60, 64, 500, seed=3)
    head = torch.nn.Linear(64, 500, bias=False, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        head.weight.copy_(w)
    ref = kernels.head_token_logps(h, w, lab)
    h3 = torch.empty(4, 30, 128, device=DEV, dtype=torch.bfloat16)[:, ::2, :64]  # strided rows
    h3.copy_(h.view(4, 15, 64))
    lab3 = torch.empty(4, 30, device=DEV, dtype=torch.int32)[:, ::2]
    lab3.copy_(lab.view(4, 15))
    with torch.no_grad():
        lp, ent = kernels.head_token_logps(h3, head, lab3)
    assert lp.shape == (4, 15) and not lp.requires_grad
    assert torch.equal(lp.view(-1), ref[0]) and torch.equal(ent.view(-1), ref[1])


def test_head_token_logps_all_ignored_and_outside():
    h, w, lab, up = _logps_inputs(40, 64, 500, seed=4)
    h.requires_grad_(True)
    lp, ent = kernels.head_token_logps(h, w, torch.full_like(lab, IGNORE))
    (dh,) = torch.autograd.grad(lp, [h], torch.full_like(up, float("nan")))
    assert not lp.any() and not ent.any() and not dh.any()
    lab[3], lab[7] = 500, -1
    lp, _ = kernels.head_token_logps(h, w, lab)
    bad = torch.zeros_like(lab, dtype=torch.bool)
    bad[3] = bad[7] = True
    assert torch.equal(torch.isnan(lp), bad)


def test_head_token_logps_masked_rows_do_not_leak():
    """NaN and infinities in unlabelled hidden rows and their weights stay there."""
    h, w, lab, up = _logps_inputs(300, 64, 900, seed=5)
    off = lab == IGNORE
    h[off] = float("nan")
    up[off] = float("inf")
    h.requires_grad_(True)
    w.requires_grad_(True)
    out = kernels.head_token_logps(h, w, lab)
    dh, dw = torch.autograd.grad(out[0], [h, w], up)
    assert not dh[off].any()
    clean = torch.where(off[:, None], torch.zeros_like(h), h).detach()
    _logps_check(clean, w, lab, torch.where(off, torch.zeros_like(up), up), out, (dh, dw))


def test_head_token_logps_blocks_and_repeated_backward(monkeypatch):
    h, w, lab, up = _logps_inputs(700, 64, 1500, seed=6)
    h.requires_grad_(True)
    w.requires_grad_(True)
    lp, ent = kernels.head_token_logps(h, w, lab)
    a = torch.autograd.grad(lp, [h, w], up, retain_graph=True)
    b = torch.autograd.grad(lp, [h, w], up)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    monkeypatch.setattr(chunked_ce, "CE_WORKSPACE_BYTES", 1 << 20)
    lp2, ent2 = kernels.head_token_logps(h, w, lab)
    assert torch.equal(lp, lp2) and torch.equal(ent, ent2)
    _logps_check(h, w, lab, up, (lp2, ent2), torch.autograd.grad(lp2, [h, w], up))


def test_head_token_logps_wide_logits():
    """Rows whose maximum lies far above the target's logit (the overflow fallback)."""
    h, w, lab, up = _logps_inputs(64, 64, 600, seed=7, keep=1.0)
    w = w.clone()
    w[0] = 0.5
    w[1] = -0.5
    h = (h.float() + 3.0).to(torch.bfloat16)  # z_0 near +96, z_1 near -96
    lab[:32] = 1
    h.requires_grad_(True)
    lp, ent = kernels.head_token_logps(h, w, lab)
    (dh,) = torch.autograd.grad(lp, [h], up)
    assert float(lp[:32].max()) < -100
    _logps_check(h, w, lab, up, (lp, ent), (dh,))


def test_head_token_logps_directional_difference():
    h, w, lab, up = _logps_inputs(50, 64, 400, torch.float16, seed=8)
    h.requires_grad_(True)
    lp, _ = kernels.head_token_logps(h, w, lab)
    (dh,) = torch.autograd.grad(lp, [h], up)
    step = torch.randn(h.shape, generator=_gen(9), device=DEV) * 0.02
    hi, lo = (h.detach() + step).half(), (h.detach() - step).half()
    diff = ((kernels.head_token_logps(hi, w, lab)[0] - kernels.head_token_logps(lo, w, lab)[0]).double()
            * up.double()).sum()
    along = (dh.double() * (hi.double() - lo.double())).sum()
    scale = (dh.double() * (hi.double() - lo.double())).norm()
    # bf16 factors (2^-8 per term, random) and the third-order term of 0.02 steps
    assert abs(float(diff - along)) <= 0.02 * float(scale) + 0.005 * abs(float(along))


# ----------------------------------------------------------------- preference -----
@pytest.mark.parametrize("pairs,s", [(1, 1), (1, 7), (2, 512), (3, 4096), (5, 4097), (300, 33), (2, 20001), (1, 8192), (1, 2049)])
@pytest.mark.parametrize("kind,eps", [("sigmoid", 0.0), ("sigmoid", 0.1), ("hinge", 0.0), ("ipo", 0.0)])
def test_preference_loss(pairs, s, kind, eps):
    g = _gen(pairs * 31 + s)
    x = -torch.rand(2 * pairs, s, generator=g, device=DEV) * 3
    r = x + torch.randn(2 * pairs, s, generator=g, device=DEV) * (2 / math.sqrt(s))
    lab = _labels(2 * pairs, s, 1000, g)
    x.requires_grad_(True)
    for ref in (r, torch.where(lab != IGNORE, r, torch.zeros_like(r)).sum(1), None):
        if ref is None and s > 4096:
            continue
        loss, c, j = kernels.preference_loss(x, ref, lab, beta=0.3, label_smoothing=eps, loss_type=kind)
        (dx,) = torch.autograd.grad(loss * 2.5, [x])
        want = ref64.preference64(x, ref, lab, 0.3, eps, kind)
        # beta reaches the kernel in fp32 (2^-24 of h); exp / log1p are good to 2^-22
        bh = float(torch.cat([want[1], want[2]]).abs().max()) * 2 + 1
        t = 2.0 ** -21
        _within(c, want[1], t * want[1].abs() + 1e-30, "chosen")
        _within(j, want[2], t * want[2].abs() + 1e-30, "rejected")
        per = 1.0 if kind != "ipo" else 1 / 0.3 ** 2
        _within(loss.detach(), want[0], t * (want[0].abs() + bh * per), "loss")
        _within(dx, 2.5 * want[3], t * (bh + 4) * (2.5 * want[3].abs() + 1e-12) +
                (t * 2.5 * bh * per / pairs if kind == "ipo" else 0), "dlogps")
        assert not c.requires_grad and not j.requires_grad


def test_preference_loss_masked_values_and_empty_sequences():
    g = _gen(5)
    x = -torch.rand(4, 50, generator=g, device=DEV)
    r = -torch.rand(4, 50, generator=g, device=DEV)
    lab = _labels(4, 50, 100, g)
    lab[1] = IGNORE
    off = lab == IGNORE
    dirty = torch.where(off, torch.full_like(x, float("nan")), x).requires_grad_(True)
    rdirty = torch.where(off, torch.full_like(x, float("-inf")), r)
    for kind in ("sigmoid", "hinge", "ipo"):
        loss, c, j = kernels.preference_loss(dirty, rdirty, lab, loss_type=kind)
        (dx,) = torch.autograd.grad(loss, [dirty])
        want = ref64.preference64(x, r, lab, 0.1, 0.0, kind)
        assert abs(float(loss) - float(want[0])) <= 1e-5 and not dx[off].any() and not dx[1].any()
        _within(dx, want[3], 1e-5 * want[3].abs() + 1e-12, "dlogps")
        assert float(c[1]) == 0.0


def test_preference_loss_extreme_margins():
    """Margins where exp overflows or underflows keep a finite loss and gradient."""
    x = torch.tensor([[-1.0], [-4000.0], [-3000.0], [-2.0]], device=DEV, requires_grad=True)
    lab = torch.zeros(4, 1, dtype=torch.int64, device=DEV)
    loss, _, _ = kernels.preference_loss(x, None, lab, beta=1.0)
    (dx,) = torch.autograd.grad(loss, [x])
    want = ref64.preference64(x, None, lab, 1.0, 0.0, "sigmoid")
    assert abs(float(loss) - float(want[0])) <= 2.0 ** -20 * float(want[0])
    _within(dx, want[3], 2.0 ** -20 * want[3].abs(), "dlogps")


# --------------------------------------------------------------------- policy -----
@pytest.mark.parametrize("b,s", [(1, 1), (3, 7), (8, 512), (2, 4097), (1500, 33), (2, 8192), (4, 2049)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("case", ["full", "no_old", "no_ref", "plain"])
def test_policy_loss(b, s, reduction, case):
    g = _gen(b + s)
    x = -torch.rand(b, s, generator=g, device=DEV) * 3
    old = x + 0.2 * torch.randn(b, s, generator=g, device=DEV) if case in ("full", "no_ref") else None
    ref = x + 0.3 * torch.randn(b, s, generator=g, device=DEV) if case in ("full", "no_old") else None
    c = 0.1 if ref is not None else 0.0
    lab = _labels(b, s, 1000, g)
    x.requires_grad_(True)
    for adv in (torch.randn(b, generator=g, device=DEV), torch.randn(b, s, generator=g, device=DEV)):
        loss, kl, cut = kernels.policy_loss(x, adv, lab, old, ref, 0.2, 0.3, c, reduction)
        (dx,) = torch.autograd.grad(loss * -3.0, [x])
        want = ref64.policy64(x, adv, lab, old, ref, 0.2, 0.3, c, reduction)
        # expf / expm1f to 2^-22, a handful of fp32 roundings at 2^-24 of the terms
        t = 2.0 ** -20
        _within(dx, -3.0 * want[3], t * 3.0 * want[4] + 1e-30, "dlogps")
        size = float(want[4].sum()) + 2.0 * float(want[4].gt(0).any())
        _within(loss.detach(), want[0], torch.tensor(t * size + 1e-30, device=DEV), "loss")
        _within(kl, want[1], t * (want[1].abs() + 0.3), "kl")
        _within(cut, want[2], 2.0 ** -24 * want[2], "clipped")


def test_policy_loss_masked_values_empty_rows_and_borders():
    g = _gen(6)
    x = -torch.rand(5, 64, generator=g, device=DEV)
    lab = _labels(5, 64, 100, g)
    lab[2] = IGNORE
    off = lab == IGNORE
    nan = torch.full_like(x, float("nan"))
    dirty = torch.where(off, nan, x).requires_grad_(True)
    old = torch.where(off, nan, x - 0.1)
    ref = torch.where(off, -nan, x + 0.1)
    adv = torch.where(off, nan, torch.ones_like(x))
    for red in ("token", "sequence"):
        loss, kl, cut = kernels.policy_loss(dirty, adv, lab, old, ref, kl_coef=0.1, reduction=red)
        (dx,) = torch.autograd.grad(loss, [dirty])
        want = ref64.policy64(x, torch.ones_like(x), lab, x - 0.1, x + 0.1, 0.2, 0.2, 0.1, red)
        assert abs(float(loss) - float(want[0])) <= 1e-6 and not dx[off].any()
        _within(dx, want[3], 1e-6 * want[4] + 1e-30, "dlogps")
    # nothing labelled at all
    loss, kl, cut = kernels.policy_loss(dirty, adv, torch.full_like(lab, IGNORE))
    (dx,) = torch.autograd.grad(loss, [dirty])
    assert float(loss) == float(kl) == float(cut) == 0.0 and not dx.any()
    # an advantage of 0 clips nothing; ratios on either side of the border
    x1 = torch.zeros(1, 3, device=DEV, requires_grad=True)
    o1 = -torch.log(torch.tensor([[1.2 - 1e-6, 1.2 + 1e-6, 9.0]], device=DEV, dtype=torch.float64)).float()
    a1 = torch.tensor([[1.0, 1.0, 0.0]], device=DEV)
    loss, _, cut = kernels.policy_loss(x1, a1, torch.zeros(1, 3, dtype=torch.int64, device=DEV), o1)
    (dx,) = torch.autograd.grad(loss, [x1])
    assert abs(float(cut) - 1 / 3) < 1e-6
    assert float(dx[0, 0]) < -0.39 and float(dx[0, 1]) == 0.0 and float(dx[0, 2]) == 0.0


def test_loss_directional_differences():
    g = _gen(7)
    x = -torch.rand(6, 200, generator=g, device=DEV)
    lab = _labels(6, 200, 100, g)
    old, ref, adv = x + 0.05, x - 0.2, torch.randn(6, generator=g, device=DEV)
    d = torch.randn(6, 200, generator=g, device=DEV)
    calls = [lambda y: kernels.policy_loss(y, adv, lab, old, ref, kl_coef=0.5)[0],
             lambda y: kernels.preference_loss(y, ref, lab, beta=0.2)[0],
             lambda y: kernels.preference_loss(y, ref, lab, beta=0.2, loss_type="ipo")[0]]
    for f in calls:
        y = x.clone().requires_grad_(True)
        (gy,) = torch.autograd.grad(f(y), [y])
        h = 2.0 ** -7
        num = (float(f(x + h * d)) - float(f(x - h * d))) / (2 * h)
        ana = float((gy.double() * d.double()).sum())
        # loss good to 2^-22 of a few units over 2 h, and the step's third-order term
        assert abs(num - ana) <= 5e-4 * (1 + abs(ana)), (num, ana)


# --------------------------------------------------------------------- window -----
def _qkv(B, H, Hk, S, seed, layout="hf"):
    g = _gen(seed)
    D = 128
    if layout == "hf":
        q, k, v = (torch.randn(B, S, n, D, generator=g, device=DEV).bfloat16().transpose(1, 2)
                   for n in (H, Hk, Hk))
    else:
        q, k, v = (torch.randn(B, n, S, D, generator=g, device=DEV).bfloat16() for n in (H, Hk, Hk))
    do = torch.randn(B, S, H, D, generator=g, device=DEV).bfloat16()
    return q, k, v, do


def _window_check(q, k, v, do, window, sinks, scale=128 ** -0.5):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = kernels.window_attention(q, k, v, scale, window, sinks)
    got = (out,) + torch.autograd.grad(out, [q, k, v], do)
    torch.cuda.synchronize()
    assert _lib.device_error(q.device) == 0
    val, tol = ref64.window64(q, k, v, do, scale, window, sinks)
    for name, a, b, t in zip(("out", "dq", "dk", "dv"), got, val, tol):
        assert a.shape == b.shape and a.dtype == torch.bfloat16
        _within(a, b, t + 2.0 ** -14 * float(b.abs().max()), name)


@pytest.mark.parametrize("B,H,Hk,S,window,sinks", [
    (1, 1, 1, 1, 1, 0),          # one token
    (2, 2, 1, 5, 2, 1),
    (1, 2, 2, 128, 1, 0),        # each query sees itself alone
    (1, 2, 1, 129, 64, 4),       # one row in the last tile
    (2, 12, 2, 384, 100, 4),     # the QLoRA step's heads
    (1, 6, 3, 400, 128, 0),      # window = tile
    (1, 4, 1, 513, 129, 130),    # sinks over a tile's end
    (1, 2, 2, 700, 300, 257),
    (1, 3, 1, 1000, 7, 1),       # a window far below a tile
    (1, 2, 1, 640, 640, 3),      # window = sequence: plain causal
    (1, 2, 1, 333, 5000, 9000),  # both beyond the sequence
    (1, 8, 1, 300, 40, 2),       # eight heads of one KV head, few key tiles: heads split over CTAs
    (1, 7, 1, 200, 70, 1),       # a head count that no split divides
    (6, 10, 5, 900, 64, 140),    # many key tiles: one CTA for all heads; sinks in segments
    (2, 2, 2, 2500, 130, 129),   # sink segments, two sink tiles
])
def test_window_attention(B, H, Hk, S, window, sinks):
    _window_check(*_qkv(B, H, Hk, S, S + window), window, sinks)


def test_window_attention_layouts():
    q, k, v, do = _qkv(2, 4, 2, 200, 1, layout="bhsd")
    _window_check(q, k, v, do, 50, 4)
    # slices of one fused projection, and layouts the kernels cannot read in place
    big = torch.randn(2, 200, 8 * 128, generator=_gen(2), device=DEV).bfloat16()
    q = big[..., :512].view(2, 200, 4, 128).transpose(1, 2)
    k = big[..., 512:768].view(2, 200, 2, 128).transpose(1, 2)
    v = big[..., 768:].view(2, 200, 2, 128).transpose(1, 2)
    _window_check(q, k, v, do, 50, 4)
    odd = torch.randn(2, 4, 200, 129, generator=_gen(3), device=DEV).bfloat16()[..., 1:]
    _window_check(odd, k, v, do, 50, 4)
    _window_check(q, k[:, :1].expand(2, 2, 200, 128), v, do, 50, 4)
    _window_check(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, do, 50, 4)


def test_window_attention_large_logits():
    """Sinks far above and far below the window's logits."""
    q, k, v, do = _qkv(1, 2, 1, 600, 4)
    u = torch.randn(128, generator=_gen(5), device=DEV)
    q = (q.float() + 2 * u).bfloat16()
    for f in (3.0, -3.0):
        k2 = k.float().clone()
        k2[:, :, :4] += f * u
        _window_check(q, k2.bfloat16(), v, do, 90, 4)


def test_window_attention_equals_causal_when_the_window_covers_all():
    from auspex_soup_demo_b200.kernels.attention import flash_attention

    q, k, v, do = _qkv(2, 4, 2, 500, 6)
    a, b = [], []
    for f, res in ((lambda *t: kernels.window_attention(*t, 0.1, 500), a),
                   (lambda *t: flash_attention(*t, 0.1, True), b)):
        ts = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = f(*ts)
        res += [out, *torch.autograd.grad(out, ts, do)]
    # two kernels that both round P, dS (2^-8 of each) and their outputs to bf16
    for x, y in zip(a, b):
        assert float((x.double() - y.double()).norm() / y.double().norm()) <= 2 * 2.0 ** -8


def test_window_attention_directional_difference():
    q, k, v, do = _qkv(1, 2, 1, 300, 8)
    ts = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = kernels.window_attention(*ts, 0.09, 70, 2)
    grads = torch.autograd.grad(out, ts, do)
    for i in range(3):
        step = torch.randn(ts[i].shape, generator=_gen(i), device=DEV) * 0.05
        hi, lo = list(map(torch.detach, ts)), list(map(torch.detach, ts))
        hi[i], lo[i] = (hi[i] + step).bfloat16(), (lo[i] - step).bfloat16()
        num = ((kernels.window_attention(*hi, 0.09, 70, 2).double()
                - kernels.window_attention(*lo, 0.09, 70, 2).double()) * do.double()).sum()
        term = grads[i].double() * (hi[i].double() - lo[i].double())
        # outputs rounded to bf16 (2^-8 of values below 4, random over the elements), gradients too
        noise = 2.0 ** -8 * 2 * math.sqrt(out.numel()) * float((out.double() * do.double()).std())
        assert abs(float(num - term.sum())) <= noise + 0.02 * abs(float(term.sum()))


# ----------------------------------------------------------------- 8-bit SwiGLU ----
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 8), (2, 63), (5, 64), (7, 65), (130, 200), (33, 1000), (4, 8960)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("strided", [False, True])
def test_swiglu_8bit(rows, n, dtype, strided):
    g = _gen(rows * n)
    if strided:
        both = (torch.randn(rows, 2 * n, generator=g, device=DEV) * 2).to(dtype)
        gate, up = both[:, :n], both[:, n:]
    else:
        gate, up = ((torch.randn(rows, n, generator=g, device=DEV) * 2).to(dtype) for _ in range(2))
    dy = torch.randn(rows, n, generator=g, device=DEV).to(dtype)
    gate, up = gate.detach().requires_grad_(True), up.detach().requires_grad_(True)
    h = kernels.swiglu_8bit(gate, up)
    dg, du = torch.autograd.grad(h, [gate, up], dy)
    gq, uq = ref64.kept8(gate), ref64.kept8(up)
    for x, want in ((gate, gq), (up, uq)):
        codes, scales = kernels.quantize_8bit(x)
        assert torch.equal(codes.float() * scales.repeat_interleave(64, 1)[:, :n], want)
    wh = ref64.swiglu64(gate, up, dy)[0]
    _, wg, wu, size = ref64.swiglu64(gq, uq, dy)
    e = torch.finfo(dtype).eps / 2
    # the rounding to the dtype, and a few fp32 operations (2^-24) with an exponential good to 2^-21
    s = 2.0 ** -19
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # half a subnormal step
    _within(h.detach(), wh, (e + s) * wh.abs() + tiny, "h")
    _within(dg, wg, e * wg.abs() + s * size + tiny, "dg")
    _within(du, wu, (e + s) * wu.abs() + tiny, "du")


def test_swiglu_8bit_special_values():
    n = 192
    gate = torch.randn(3, n, device=DEV, generator=_gen(1))
    up = torch.randn(3, n, device=DEV, generator=_gen(2))
    gate[0, :64] = 0
    gate[0, 64:128] = 1e-38  # a block too small for its scale
    gate[1, 70] = float("inf")
    up[2, 5] = float("nan")
    gate.requires_grad_(True)
    up.requires_grad_(True)
    for f in (lambda t: t, lambda t: t[:, :n - 1]):  # vector and scalar paths
        h = kernels.swiglu_8bit(f(gate), f(up))
        dg, du = torch.autograd.grad(h, [gate, up], torch.ones_like(h))
        assert not du[0, :128].any() and torch.isfinite(dg[0]).all()
        assert torch.isnan(du[1, 64:128]).all() and torch.isfinite(du[1, :64]).all()
        assert torch.isnan(dg[2, :64]).all() and torch.isfinite(dg[2, 64:]).all()
    e = torch.empty(0, 16, device=DEV, requires_grad=True)
    assert kernels.swiglu_8bit(e, e).shape == (0, 16)


def test_swiglu_8bit_gradient_close_to_exact():
    """Against the exact gradient: the kept values are within absmax / 254."""
    g = _gen(3)
    gate, up, dy = (torch.randn(64, 512, generator=g, device=DEV) for _ in range(3))
    gate.requires_grad_(True)
    up.requires_grad_(True)
    h = kernels.swiglu_8bit(gate, up)
    dg, du = torch.autograd.grad(h, [gate, up], dy)
    _, wg, wu, _ = ref64.swiglu64(gate.detach(), up.detach(), dy)
    # half a code of the block with the largest maximum (above 4.5 for some draws of
    # 32768 normal values), and the fp32 roundings of code and value (2^-22)
    step = float(torch.maximum(gate.detach().abs().max(), up.detach().abs().max())) / 254 * (1 + 2.0 ** -20)
    # |d silu| <= 1.1, |d^2 silu| <= 0.5
    _within(du, wu, dy.abs().double() * 1.1 * step + 1e-5, "du")
    _within(dg, wg, dy.abs().double() * step * (1.1 + 0.5 * up.detach().abs().double() + 0.5 * step) + 1e-5,
            "dg")


# ------------------------------------------------------ streams, graphs, together ----
def _chain(st):
    """Log-probabilities, policy loss and their gradients, as a training step runs them."""
    lp, _ = kernels.head_token_logps(st["h"], st["w"], st["lab"])
    loss, kl, cut = kernels.policy_loss(lp, st["adv"], st["lab"], st["old"], st["ref"], kl_coef=0.1)
    pref, _, _ = kernels.preference_loss(lp, st["ref"], st["lab"])
    return (loss, kl, cut, pref) + torch.autograd.grad(loss + pref, [st["h"], st["w"]])


def _chain_inputs(seed):
    h, w, lab, _ = _logps_inputs(4 * 90, 64, 700, seed=seed)
    g = _gen(seed + 1)
    lp = kernels.head_token_logps(h, w, lab)[0].view(4, 90)
    return {"h": h.view(4, 90, 64), "w": w, "lab": lab.view(4, 90),
            "adv": torch.randn(4, generator=g, device=DEV),
            "old": lp + 0.1 * torch.randn(4, 90, generator=g, device=DEV),
            "ref": lp + 0.1 * torch.randn(4, 90, generator=g, device=DEV)}


def test_chain_against_64_bit():
    st = _chain_inputs(11)
    st["h"].requires_grad_(True)
    st["w"].requires_grad_(True)
    loss, kl, cut, pref, dh, dw = _chain(st)
    lp64 = ref64.logps64(st["h"], st["w"], st["lab"])[0].view(4, 90)
    a = ref64.policy64(lp64, st["adv"], st["lab"], st["old"], st["ref"], 0.2, 0.2, 0.1, "token")
    b = ref64.preference64(lp64, st["ref"], st["lab"], 0.1, 0.0, "sigmoid")
    assert abs(float(loss) - float(a[0])) <= 1e-4 and abs(float(pref) - float(b[0])) <= 1e-4
    lp = kernels.head_token_logps(st["h"], st["w"], st["lab"])
    _logps_check(st["h"], st["w"], st["lab"], a[3] + b[3], lp, (dh, dw))


def test_chain_on_side_streams_and_in_graphs():
    ins = [_chain_inputs(s) for s in (21, 22)]
    for st in ins:
        st["h"].requires_grad_(True)
        st["w"].requires_grad_(True)
    want = [[t.detach().clone() for t in _chain(st)] for st in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    outs = []
    for st, s in zip(ins, streams):  # both at once
        with torch.cuda.stream(s):
            for _ in range(3):
                o = _chain(st)
            outs.append(o)
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    # two captured graphs on one static input, replayed with other inputs, in turn and together
    statics, graphs, res = [], [], []
    for k in range(2):
        st = {n: t.detach().clone() for n, t in ins[0].items()}
        st["h"].requires_grad_(True)
        st["w"].requires_grad_(True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = _chain(st)
        statics.append(st)
        graphs.append(graph)
        res.append(r)
    for k, order in ((0, (0, 1)), (1, (1, 0))):
        with torch.no_grad():
            for j in range(2):
                for n in statics[j]:
                    statics[j][n].copy_(ins[order[j]][n])
        torch.cuda.synchronize()
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                graphs[j].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert all(torch.equal(x, y) for x, y in zip(res[j], want[order[j]]))
    assert _lib.device_error(torch.device(DEV)) == 0


def test_window_and_swiglu8_in_graphs():
    q, k, v, do = _qkv(1, 4, 2, 300, 31)
    ts = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    gu = [torch.randn(60, 200, device=DEV, generator=_gen(i)).bfloat16().requires_grad_(True) for i in (1, 2)]

    def run():
        o = kernels.window_attention(*ts, 0.1, 80, 4)
        h = kernels.swiglu_8bit(*gu)
        return (o, h) + torch.autograd.grad([o, h], ts + gu, [do, torch.ones_like(h)])

    # detached: an eager graph of the same leaves must not outlive into the capture
    want = [t.detach().clone() for t in run()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = run()
    for _ in range(2):
        for t in res:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_window_on_two_streams_at_once():
    """More CTAs than SMs on each stream, with the head's products between them."""
    st = _chain_inputs(41)
    st["h"].requires_grad_(True)
    st["w"].requires_grad_(True)
    ins = [[t.detach().requires_grad_(True) for t in qkv] + [do]
           for *qkv, do in (_qkv(2, 12, 2, 1300, 32), _qkv(3, 8, 4, 1111, 33))]

    def run(i):
        *qkv, do = ins[i]
        o = kernels.window_attention(*qkv, 0.09, 300 - 100 * i, 70)
        return [o.detach()] + list(torch.autograd.grad(o, qkv, do)) + [t.detach() for t in _chain(st)]

    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    outs = [None, None]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i] = run(i)
    torch.cuda.synchronize()
    for a, b in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert _lib.device_error(torch.device(DEV)) == 0


# ------------------------------------------------------------------- the model ----
def _model(layers=2, attention="sdpa", **over):
    from auspex_soup_demo_b200 import apply, qlora

    apply()
    cfg = qlora.qwen2_1p5b_config(layers, attention, hidden_size=256, intermediate_size=512,
                                  num_attention_heads=2, num_key_value_heads=1, vocab_size=1000, **over)
    model = qlora.build_qwen2_qlora(cfg, seed=1)
    g = _gen(2)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "lora_B" in n:
                p.copy_(torch.randn(p.shape, generator=g, device=DEV) * 0.05)
    return model


def test_trainer_preference_and_policy_steps():
    from auspex_soup_demo_b200 import qlora

    model = _model()
    tr = qlora.QLoRATrainer(model, lr=0.0)
    ids = torch.randint(0, 1000, (4, 64), generator=_gen(3), device=DEV)
    lab = qlora.causal_labels(ids)
    lab[:, :20] = IGNORE
    ref = tr.token_logps(ids, lab)
    assert ref.shape == (4, 64) and not ref.requires_grad
    loss, c, r = tr.preference_step(ids, lab, ref)
    # the policy is the reference: no margin
    assert abs(float(loss) - math.log(2)) <= 1e-5 and float(c.abs().max()) <= 1e-5
    assert torch.isfinite(tr.flat_grad).all() and float(tr.flat_grad.abs().max()) > 0
    adv = torch.randn(4, generator=_gen(4), device=DEV)
    loss, kl, cut = tr.policy_step(ids, lab, adv, old_logps=ref, ref_logps=ref, kl_coef=0.1)
    n = (lab != IGNORE).sum(1)
    assert abs(float(loss) + float((adv * n).sum() / n.sum())) <= 1e-5
    assert float(cut) == 0.0 and abs(float(kl)) <= 1e-9
    # its gradient is that of -A times the mean log-probability, through plain autograd
    got = tr.flat_grad.clone()
    tr.flat_grad.zero_()
    hid = tr._hidden(ids)
    lsm = torch.log_softmax(hid.float() @ model.lm_head.weight.float().t(), -1)
    lp = lsm.gather(-1, lab.clamp(min=0)[..., None])[..., 0]
    (-(lp * adv[:, None])[lab != IGNORE].sum() / n.sum()).backward()
    want = tr.flat_grad
    cos = float((got.double() @ want.double()) / (got.double().norm() * want.double().norm()))
    assert cos >= 0.999 and abs(float(got.norm() / want.norm()) - 1) <= 0.02


def test_mlp_kept_in_8_bits():
    from auspex_soup_demo_b200 import qlora
    from auspex_soup_demo_b200.kernels import swiglu

    ids = torch.randint(0, 1000, (2, 128), generator=_gen(5), device=DEV)
    lab = qlora.causal_labels(ids)
    grads, losses, peaks = [], [], []
    old = (swiglu.CHECKPOINT_8BIT, swiglu.RECOMPUTE)
    try:
        for keep8, recompute in ((False, False), (True, False), (True, True)):
            swiglu.CHECKPOINT_8BIT, swiglu.RECOMPUTE = keep8, recompute
            tr = qlora.QLoRATrainer(_model(), lr=0.0)
            loss, _ = tr.step(ids, lab, 254.0)
            losses.append(float(loss))
            grads.append(tr.flat_grad.double().clone())
    finally:
        swiglu.CHECKPOINT_8BIT, swiglu.RECOMPUTE = old
    assert losses[0] == losses[1] == losses[2]  # the forward does not change
    assert torch.equal(grads[1], grads[2])
    a, b = grads[0], grads[1]
    # kept values are off by at most 1/254 of their block's maximum (about 2.5 of its
    # standard deviations): below 1 % of the gradient, random over the terms
    assert float(a @ b / (a.norm() * b.norm())) >= 0.9995
    assert abs(float(a.norm() / b.norm()) - 1) <= 0.005


def test_mlp_kept_in_8_bits_ungrouped():
    """The patched MLP of a model whose projections are plain linears."""
    from transformers.models.qwen2 import modeling_qwen2
    from auspex_soup_demo_b200 import apply, qlora
    from auspex_soup_demo_b200.kernels import swiglu

    apply()
    cfg = qlora.qwen2_1p5b_config(1, hidden_size=128, intermediate_size=320, num_attention_heads=1,
                                  num_key_value_heads=1, vocab_size=100)
    torch.manual_seed(0)
    mlp = modeling_qwen2.Qwen2MLP(cfg).to(DEV, torch.bfloat16).train()
    x = torch.randn(2, 40, 128, device=DEV, generator=_gen(6)).bfloat16()
    res = []
    old = (swiglu.CHECKPOINT_8BIT, swiglu.RECOMPUTE)
    try:
        for keep8 in (False, True):
            swiglu.CHECKPOINT_8BIT, swiglu.RECOMPUTE = keep8, False
            y = x.clone().requires_grad_(True)
            out = mlp(y)
            res.append((out.detach(), torch.autograd.grad(out.float().square().sum(), [y])[0]))
    finally:
        swiglu.CHECKPOINT_8BIT, swiglu.RECOMPUTE = old
    assert torch.equal(res[0][0], res[1][0])
    a, b = res[0][1].double().flatten(), res[1][1].double().flatten()
    assert float(a @ b / (a.norm() * b.norm())) >= 0.9995


def test_model_with_sliding_window_layers():
    kw = dict(use_sliding_window=True, sliding_window=20, max_window_layers=1)
    ids = torch.randint(0, 1000, (2, 150), generator=_gen(7), device=DEV)
    a = _model(2, "soup", **kw)
    b = _model(2, "sdpa", **kw)
    assert a.config.layer_types == ["full_attention", "sliding_attention"]
    with torch.no_grad():
        x, y = a(ids).logits.double(), b(ids).logits.double()
    # two bf16 attention kernels through two layers
    assert float((x - y).norm() / y.norm()) <= 0.02
    wide = _model(2, "soup")
    with torch.no_grad():
        z = wide(ids).logits.double()
    assert float((x - z).norm() / z.norm()) > 0.05  # the window does change the result
    a.config.attention_sink_tokens = 150  # every key is a sink: the window hides nothing
    with torch.no_grad():
        x = a(ids).logits.double()
    assert float((x - z).norm() / z.norm()) <= 0.02


def test_model_with_sliding_window_layers_and_a_cache():
    kw = dict(use_sliding_window=True, sliding_window=20, max_window_layers=1)
    ids = torch.randint(0, 1000, (2, 70), generator=_gen(8), device=DEV)
    a = _model(2, "soup", **kw)
    with torch.no_grad():
        whole = a(ids).logits.double()
        first = a(ids[:, :60], use_cache=True)
        rest = [first.logits]
        cache = first.past_key_values
        for i in range(60, 70):
            step = a(ids[:, i:i + 1], past_key_values=cache, use_cache=True)
            cache = step.past_key_values
            rest.append(step.logits)
    rest = torch.cat(rest, 1).double()
    # the same model by two bf16 attention kernels through two layers
    assert float((whole - rest).norm() / whole.norm()) <= 0.02


def test_second_derivatives_are_refused():
    lab = torch.tensor([[1, -100, 2], [3, 4, -100]], device=DEV)
    x = torch.randn(2, 3, device=DEV, generator=_gen(51)).requires_grad_(True)
    h = torch.randn(2, 3, 64, device=DEV, generator=_gen(52)).bfloat16().requires_grad_(True)
    w = torch.randn(40, 64, device=DEV, generator=_gen(53)).bfloat16()
    q = torch.randn(1, 2, 9, 128, device=DEV, generator=_gen(54)).bfloat16().requires_grad_(True)
    calls = [(lambda: kernels.preference_loss(x, None, lab)[0], x),
             (lambda: kernels.policy_loss(x, torch.ones(2, device=DEV), lab)[0], x),
             (lambda: kernels.head_token_logps(h, w, lab)[0].sum(), h),
             (lambda: kernels.window_attention(q, q, q, 0.1, 4).float().sum(), q),
             (lambda: kernels.swiglu_8bit(h, h).float().sum(), h)]
    for f, leaf in calls:
        plain = torch.autograd.grad(f(), [leaf])[0]
        (g,) = torch.autograd.grad(f(), [leaf], create_graph=True)
        assert torch.equal(g.detach(), plain)
        # torch: a backward whose incoming gradient is a constant gives a constant
        with pytest.raises(RuntimeError, match="does not require grad"):
            torch.autograd.grad(g.float().square().sum(), [leaf])
        factor = torch.ones((), device=DEV, requires_grad=True)
        (g,) = torch.autograd.grad(f() * factor, [leaf], create_graph=True)
        assert torch.equal(g.detach(), plain)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.float().square().sum().backward()
