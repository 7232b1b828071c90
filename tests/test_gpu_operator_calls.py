"""The preference / policy tuning operators in calls that a training program makes around
them: offloaded activations, far references, caches, short batches.

Where two calls have to agree bit for bit, the kernels sum in a fixed order and the
inputs are the same; other tolerances are derived at their test.
"""

import pytest
import torch

from auspex_soup_demo_b200 import _lib, kernels

pytestmark = pytest.mark.gpu

IGNORE = -100
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ----------------------------------------------------------- saved-tensor hooks ----
def _offload(pin):
    return torch.autograd.graph.save_on_cpu(pin_memory=pin)


def _same_under_offload(call, leaves):
    """Outputs and gradients of ``call`` under save_on_cpu equal those without."""
    def run():
        out = call()
        out = out if isinstance(out, tuple) else (out,)
        dout = torch.randn(out[0].shape, generator=_gen(99), device=DEV).to(out[0].dtype)
        return [t.detach().clone() for t in out], dout, out[0]

    want, dout, first = run()
    want += torch.autograd.grad(first, leaves, dout)
    for pin in (True, False):
        with _offload(pin):
            got, dout, first = run()
            got += torch.autograd.grad(first, leaves, dout)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), pin
    assert _lib.device_error(torch.device(DEV)) == 0


@pytest.mark.parametrize("source", ["transposed", "fused projection"])
def test_window_attention_under_offload(source):
    B, H, Hk, S, D = 2, 4, 2, 200, 128
    if source == "transposed":
        q, k, v = (torch.randn(B, S, h, D, generator=_gen(h), device=DEV).bfloat16().transpose(1, 2)
                   for h in (H, Hk, Hk))
    else:
        big = torch.randn(B, S, (H + 2 * Hk) * D, generator=_gen(1), device=DEV).bfloat16()
        q, k, v = (big[..., a * D:(a + h) * D].view(B, S, h, D).transpose(1, 2)
                   for a, h in ((0, H), (H, Hk), (H + Hk, Hk)))
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    _same_under_offload(lambda: kernels.window_attention(q, k, v, 0.1, 50, 4), [q, k, v])


@pytest.mark.parametrize("S", [200, 256])
def test_causal_attention_under_offload(S):
    from auspex_soup_demo_b200.kernels.attention import flash_attention

    q, k, v = (torch.randn(2, S, h, 128, generator=_gen(h), device=DEV).bfloat16().transpose(1, 2)
               .requires_grad_(True) for h in (4, 2, 2))
    _same_under_offload(lambda: flash_attention(q, k, v, 0.1), [q, k, v])


def _logp_batch(n, s, seed):
    """logps [n, s], and labels as a slice of a wider tensor."""
    g = _gen(seed)
    ids = torch.randint(0, 1000, (n, s + 1), generator=g, device=DEV)
    ids = torch.where(torch.rand(n, s + 1, generator=g, device=DEV) < 0.6, ids, torch.full_like(ids, IGNORE))
    x = -torch.rand(n, s, generator=g, device=DEV) * 3
    return x.requires_grad_(True), ids[:, 1:], g


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
def test_preference_loss_under_offload(kind):
    x, lab, g = _logp_batch(6, 33, 2)
    ref = x.detach() + 0.1
    _same_under_offload(lambda: kernels.preference_loss(x, ref, lab, loss_type=kind), [x])


def test_policy_loss_under_offload():
    x, lab, g = _logp_batch(5, 33, 3)
    adv = torch.randn(5, 66, generator=g, device=DEV)[:, ::2]
    old = x.detach() + 0.1
    _same_under_offload(lambda: kernels.policy_loss(x, adv, lab, old, old, kl_coef=0.1), [x])


@pytest.mark.parametrize("budget", [None, 1 << 20], ids=["one block", "blocks"])
def test_head_token_logps_under_offload(monkeypatch, budget):
    from auspex_soup_demo_b200.kernels import chunked_ce

    if budget:
        monkeypatch.setattr(chunked_ce, "CE_WORKSPACE_BYTES", budget)
    g = _gen(4)
    h = torch.randn(10, 70, 128, generator=g, device=DEV).bfloat16()[..., :64].requires_grad_(True)
    w = (torch.randn(900, 64, generator=g, device=DEV) * 0.1).bfloat16().requires_grad_(True)
    lab = torch.randint(0, 900, (10, 71), generator=g, device=DEV)[:, 1:]
    _same_under_offload(lambda: kernels.head_token_logps(h, w, lab), [h, w])


def test_swiglu_8bit_under_offload():
    both = torch.randn(40, 400, generator=_gen(5), device=DEV).bfloat16()
    gate, up = (both[:, i * 200:(i + 1) * 200].requires_grad_(True) for i in (0, 1))
    _same_under_offload(lambda: kernels.swiglu_8bit(gate, up), [gate, up])


def test_mlp_kept_in_8_bits_under_offload():
    """The QLoRA step's MLP: the codes and scales of [gate | up] come back from the host."""
    from auspex_soup_demo_b200 import apply, qlora
    from auspex_soup_demo_b200.kernels import swiglu

    apply()
    cfg = qlora.qwen2_1p5b_config(1, hidden_size=256, intermediate_size=512, num_attention_heads=2,
                                  num_key_value_heads=1, vocab_size=500)
    tr = qlora.QLoRATrainer(qlora.build_qwen2_qlora(cfg, seed=1), lr=0.0)
    with torch.no_grad():
        for n, p in tr.model.named_parameters():
            if "lora_B" in n:
                p.copy_(torch.randn(p.shape, generator=_gen(6), device=DEV) * 0.05)
    ids = torch.randint(0, 500, (2, 128), generator=_gen(7), device=DEV)
    lab = qlora.causal_labels(ids)
    old = swiglu.CHECKPOINT_8BIT
    try:
        swiglu.CHECKPOINT_8BIT = True
        tr.step(ids, lab, 254.0)
        want = tr.flat_grad.clone()
        with _offload(True):
            tr.step(ids, lab, 254.0)
    finally:
        swiglu.CHECKPOINT_8BIT = old
    assert float(want.abs().max()) > 0 and torch.equal(tr.flat_grad, want)


# ------------------------------------------------------------------ policy loss ----
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_loss_reference_for_the_metric_alone(reduction):
    """kl_coef = 0: the reference enters mean_kl and nothing else, however far it is."""
    x, lab, g = _logp_batch(6, 300, 8)
    adv = torch.randn(6, generator=g, device=DEV)
    old = x.detach() + 0.1

    def run(ref):
        loss, kl, cut = kernels.policy_loss(x, adv, lab, old, ref, kl_coef=0.0, reduction=reduction)
        return loss.detach(), kl, cut, torch.autograd.grad(loss, [x])[0]

    loss, _, cut, dx = run(None)
    for shift, finite in ((100.0, False), (-100.0, True), (0.5, True), (float("nan"), False)):
        got = run(x.detach() + shift)
        assert torch.equal(got[0], loss) and torch.equal(got[2], cut) and torch.equal(got[3], dx), shift
        assert bool(torch.isfinite(got[1])) == finite


@pytest.mark.parametrize("ref", [False, True])
@pytest.mark.parametrize("bad,old", [
    ("nan", False), ("nan", True), ("inf", False), ("-inf", False),  # with old_logps a ratio of inf or 0
])
def test_policy_loss_keeps_a_broken_log_probability_visible(bad, old, ref):
    x, lab, g = _logp_batch(4, 70, 9)
    o = x.detach() - 0.05 if old else None
    r = x.detach() + 0.05 if ref else None
    lab = lab.clone()
    lab[2, 5], lab[1, 3] = 7, IGNORE
    with torch.no_grad():
        x[2, 5] = float(bad)
        x[1, 3] = float("nan")  # unlabelled: not used
    for adv in (torch.ones(4, device=DEV), -torch.ones(4, device=DEV)):
        loss, _, _ = kernels.policy_loss(x, adv, lab, o, r, kl_coef=0.1 if ref else 0.0)
        (dx,) = torch.autograd.grad(loss, [x])
        assert torch.isnan(loss)
        nan = torch.isnan(dx)
        assert bool(nan[2, 5]) and int(nan.sum()) == 1


def test_policy_loss_of_a_label_outside_the_vocabulary():
    g = _gen(10)
    h = torch.randn(2, 30, 64, generator=g, device=DEV).bfloat16().requires_grad_(True)
    w = (torch.randn(200, 64, generator=g, device=DEV) * 0.1).bfloat16()
    lab = torch.randint(0, 200, (2, 30), generator=g, device=DEV)
    lab[1, 4] = 200
    logps, _ = kernels.head_token_logps(h, w, lab)
    loss, _, _ = kernels.policy_loss(logps, torch.ones(2, device=DEV), lab)
    (dh,) = torch.autograd.grad(loss, [h])
    assert torch.isnan(loss) and torch.isnan(dh[1, 4]).all() and int(torch.isnan(dh).any(-1).sum()) == 1


@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e-3, 1e-2, 0.1, 0.45, 0.55, 1.0, 3.0])
@pytest.mark.parametrize("n", [(1, 1), (7, 100)])
def test_policy_loss_kl_near_the_reference(size, n):
    """The KL estimate keeps its digits for a policy that has hardly left its reference.

    d = ref - logps is rounded to fp32 (2^-24, twice that in d^2), the estimate takes a
    few more roundings; from |d| = 0.5 on expm1(d) - d loses a factor of up to 5 of
    expm1's 2^-23, below that nothing cancels. Every term is positive, so the bound of a
    term, 2^-20 of it, is that of the mean."""
    g = _gen(11)
    x = -1 - torch.rand(*n, generator=g, device=DEV)
    d = size * (0.9 + 0.2 * torch.rand(*n, generator=g, device=DEV))
    ref = x + torch.where(torch.rand(*n, generator=g, device=DEV) < 0.5, d, -d)
    lab = torch.zeros(*n, dtype=torch.int64, device=DEV)
    _, kl, _ = kernels.policy_loss(x, torch.ones(n[0], device=DEV), lab, None, ref, kl_coef=0.1)
    d = ref.double() - x.double()
    # in 64 bits the first terms of the series, whose cancellation expm1 would leave at small d
    small = d * d * (0.5 + d * (1 / 6 + d * (1 / 24 + d * (1 / 120 + d / 720))))
    want = torch.where(d.abs() < 0.02, small, torch.expm1(d) - d).mean()
    assert abs(float(kl) - float(want)) <= 2.0 ** -20 * float(want)


# ---------------------------------------------------------------- sliding layers ----
def _model(attention, **over):
    from auspex_soup_demo_b200 import apply, qlora

    apply()
    cfg = qlora.qwen2_1p5b_config(2, attention, hidden_size=256, intermediate_size=512, num_attention_heads=2,
                                  num_key_value_heads=1, vocab_size=1000, use_sliding_window=True,
                                  sliding_window=20, max_window_layers=1, **over)
    return qlora.build_qwen2_qlora(cfg, seed=1).eval()


def test_token_against_a_long_cache_takes_little_memory():
    from auspex_soup_demo_b200.kernels.attention import soup_attention

    class Layer(torch.nn.Module):
        is_causal, num_key_value_groups = True, 6

    q, k, v = (torch.randn(1, h, n, 128, generator=_gen(n + h), device=DEV).bfloat16()
               for h, n in ((12, 1), (2, 32768), (2, 32768)))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    out, _ = soup_attention(Layer(), q, k, v, None, sliding_window=4096)
    # keys and values once for every query head (6 groups each), not 32768^2 distances
    assert torch.cuda.max_memory_allocated() - base <= 16 * (k.nbytes + v.nbytes)
    see = slice(32768 - 4096, None)
    kk, vv = (t[:, :, see].double().repeat_interleave(6, 1) for t in (k, v))
    want = torch.softmax(q.double() @ kk.transpose(2, 3) * 128 ** -0.5, -1) @ vv
    # P and the output rounded to bf16 (2^-8 each, P's averaging out over 4096 keys)
    err = (out.transpose(1, 2).double() - want).abs()
    assert bool((err <= 2.0 ** -8 * 1.03 * want.abs() + 2.0 ** -8 * float(want.abs().max())).all())


def test_padded_batches_of_a_model_with_sliding_layers(monkeypatch):
    a, b = _model("soup"), _model("sdpa")
    ids = torch.randint(0, 1000, (3, 150), generator=_gen(20), device=DEV)
    calls = []
    call = _lib.call
    monkeypatch.setattr(_lib, "call", lambda fn, *args: (calls.append(fn), call(fn, *args))[1])
    for kind in ("none", "right", "left"):
        mask = torch.ones(3, 150, dtype=torch.long, device=DEV)
        if kind == "right":
            mask[0, 90:] = 0
        if kind == "left":
            mask[1, :40] = 0
        calls.clear()
        with torch.no_grad():
            x = a(ids, attention_mask=mask).logits[mask.bool()].double()
            on_kernels = {"soup_attention_window_fwd", "soup_attention_fwd"} <= set(calls)
            y = b(ids, attention_mask=mask).logits[mask.bool()].double()
        # two bf16 attention kernels through two layers
        assert float((x - y).norm() / y.norm()) <= 0.02, kind
        assert on_kernels == (kind != "left")


def test_chunks_against_a_cache_of_a_model_with_sliding_layers():
    a = _model("soup")
    ids = torch.randint(0, 1000, (2, 70), generator=_gen(21), device=DEV)
    with torch.no_grad():
        whole = a(ids).logits.double()
        cache, parts = None, []
        for lo, hi in ((0, 15), (15, 30), (30, 31), (31, 70)):
            r = a(ids[:, lo:hi], past_key_values=cache, use_cache=True)
            cache = r.past_key_values
            parts.append(r.logits)
    rest = torch.cat(parts, 1).double()
    assert float((whole - rest).norm() / whole.norm()) <= 0.02  # as above


# ------------------------------------------------------- window attention's key ranges ----
@pytest.mark.parametrize("S,window,sinks", [(500, 7, 493), (500, 7, 500), (300, 1, 299), (640, 320, 320),
                                            (129, 128, 1), (1, 1, 0)])
def test_window_and_sinks_that_hide_nothing(S, window, sinks):
    """Bit for bit the causal case, in which no key is hidden either."""
    q, k, v = (torch.randn(2, S, h, 128, generator=_gen(S + h), device=DEV).bfloat16().transpose(1, 2)
               .requires_grad_(True) for h in (4, 2, 2))
    do = torch.randn(2, S, 4, 128, generator=_gen(S), device=DEV).bfloat16()

    def run(*span):
        out = kernels.window_attention(q, k, v, 0.09, *span)
        return [out.detach()] + list(torch.autograd.grad(out, [q, k, v], do))

    assert all(torch.equal(a, b) for a, b in zip(run(window, sinks), run(S, 0)))
    assert _lib.device_error(torch.device(DEV)) == 0


# ------------------------------------------------------------------ 8-bit codes ----
def test_quantize_8bit_shapes():
    codes, scales = kernels.quantize_8bit(torch.empty(0, 70, device=DEV))
    assert codes.shape == (0, 70) and scales.shape == (0, 2)
    x = torch.randn(3, 4, 70, generator=_gen(30), device=DEV)
    want = kernels.quantize_8bit(x.view(12, 70))
    for t in (x, x.transpose(0, 1).contiguous().transpose(0, 1)):
        assert all(torch.equal(a, b) for a, b in zip(kernels.quantize_8bit(t), want))


# ---------------------------------------------------------------------- no tokens ----
@pytest.mark.parametrize("shape", [(0,), (2, 0)])
@pytest.mark.parametrize("trained", ["states", "head", "both"])
def test_head_token_logps_of_no_tokens(shape, trained):
    h = torch.empty(*shape, 64, device=DEV, dtype=torch.bfloat16).requires_grad_(trained != "head")
    w = torch.randn(100, 64, device=DEV).bfloat16().requires_grad_(trained != "states")
    lp, ent = kernels.head_token_logps(h, w, torch.empty(*shape, dtype=torch.int64, device=DEV))
    assert lp.shape == ent.shape == shape and lp.dtype == torch.float32 and not ent.requires_grad
    leaves = [t for t in (h, w) if t.requires_grad]
    for t, g in zip(leaves, torch.autograd.grad(lp.sum(), leaves)):
        assert g.shape == t.shape and not g.any()


# ------------------------------------------------------------------- large vocabulary ----
def test_head_token_logps_at_offsets_past_32_bits():
    """15000 tokens x 151936: the kept exponentials pass 2^31 elements. Rows at both ends
    against 64 bits; tolerances as in the tests of small sizes: fp32 accumulation of 64
    products, lse in fp32, dz's factor and the result rounded to bf16 (2^-8 each)."""
    n, d, v = 15000, 64, 151936
    g = _gen(40)
    w = (torch.randn(v, d, generator=g, device=DEV) * 0.05).bfloat16()
    lab = torch.randint(0, v, (n,), generator=g, device=DEV)
    lab[5::97] = IGNORE
    h = torch.randn(n, d, generator=g, device=DEV).bfloat16().requires_grad_(True)
    up = torch.randn(n, generator=g, device=DEV)
    lp, ent = kernels.head_token_logps(h, w, lab)
    (dh,) = torch.autograd.grad(lp, [h], up)
    assert _lib.device_error(torch.device(DEV)) == 0
    rows = torch.cat([torch.arange(20, device=DEV), torch.arange(n - 300, n, device=DEV)])
    z = h.detach()[rows].double() @ w.double().t()
    lsm = torch.log_softmax(z, 1)
    keep = lab[rows] != IGNORE
    idx = lab[rows].clamp(min=0)[:, None]
    want = torch.where(keep, lsm.gather(1, idx)[:, 0], torch.zeros_like(lsm[:, 0]))
    mag = float((h.detach()[rows].double().abs() @ w.double().abs().t()).max())
    tol = 4 * 8 * 2.0 ** -24 * mag + 2.0 ** -20 * (1 + want.abs())
    assert bool(((lp[rows].double() - want).abs() <= tol).all())
    p = lsm.exp()
    we = torch.where(keep, -(p * lsm).sum(1), torch.zeros_like(want))
    assert bool(((ent[rows].double() - we).abs() <= 16 * tol).all())
    gk = torch.where(keep, up[rows].double(), torch.zeros_like(want))
    p.scatter_add_(1, idx, -torch.ones_like(idx, dtype=torch.float64))  # -dz / gk
    wd = -(p @ w.double()) * gk[:, None]
    u = 2.0 ** -8 * 1.02
    bound = u * (p.abs() @ w.double().abs()) * gk.abs()[:, None] + 2.0 ** -8 * wd.abs() + 1e-7
    assert bool(((dh[rows].double() - wd).abs() <= bound).all())


def test_padded_batch_in_a_graph():
    """Under capture no value of the padding mask is looked at: it is applied by SDPA."""
    a = _model("soup")
    ids = torch.randint(0, 1000, (2, 150), generator=_gen(41), device=DEV)
    mask = torch.ones(2, 150, dtype=torch.long, device=DEV)
    mask[0, :30] = 0
    with torch.no_grad():
        want = a(ids, attention_mask=mask).logits[mask.bool()].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = a(ids, attention_mask=mask).logits
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(out[mask.bool()], want)


# ------------------------------------------------------------------------ small sizes ----
@pytest.mark.parametrize("n,d,v", [(1, 8, 1), (3, 8, 2), (2, 16, 9), (257, 8, 3), (1, 8, 70000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("trained", ["states", "head", "both"])
def test_head_token_logps_smallest_sizes(n, d, v, dtype, trained):
    """fp32 accumulation of 8 or 16 products and an lse in fp32; gradients through factors
    rounded to bf16 (2^-8; twice for the head and for fp16's bf16 copy of it)."""
    g = _gen(n + v)
    h = torch.randn(n, d, generator=g, device=DEV).to(dtype).requires_grad_(trained != "head")
    w = torch.randn(v, d, generator=g, device=DEV).to(dtype).requires_grad_(trained != "states")
    lab = torch.randint(0, v, (n,), generator=g, device=DEV)
    up = torch.randn(n, generator=g, device=DEV)
    lp, ent = kernels.head_token_logps(h, w, lab)
    leaves = [t for t in (h, w) if t.requires_grad]
    grads = dict(zip(map(id, leaves), torch.autograd.grad(lp, leaves, up)))
    h6, w6 = h.detach().double(), w.detach().double()
    z = h6 @ w6.t()
    lsm = torch.log_softmax(z, 1)
    p = lsm.exp()
    want = lsm.gather(1, lab[:, None])[:, 0]
    mag = float((h6.abs() @ w6.abs().t()).max())
    tol = 16 * 2.0 ** -24 * mag + 2.0 ** -20 * (1 + want.abs())
    assert bool(((lp.double() - want).abs() <= tol).all())
    assert bool(((ent.double() + (p * lsm).sum(1)).abs() <= 40 * tol.max()).all())  # |z - lse| below 40
    dz = -p
    dz.scatter_add_(1, lab[:, None], torch.ones_like(want)[:, None])
    dz = dz * up.double()[:, None]
    u = 2 * 2.0 ** -8 * 1.02
    # dz itself is off by the logits' error: p (1 - p) of it
    slack = (p * up.double().abs()[:, None] + dz.abs()) * 4 * tol.max()
    for t, a, size in ((h, dz @ w6, (dz.abs() * u + slack) @ w6.abs()),
                       (w, dz.t() @ h6, (dz.abs() * u + slack).t() @ h6.abs())):
        if id(t) in grads:
            got = grads[id(t)].double()
            assert bool(((got - a).abs() <= size + 2.0 ** -8 * a.abs() + 1e-7).all())
