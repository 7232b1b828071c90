"""GPU: calls of the operators of a step with several adapters whose outcome their
documentation promises: gradients that are not finite, second moments near the smallest
numbers, parameters that were given other memory, tangents, rows that
overlap, base weights that are not kept,
positions of several axes in a call of the model, the trainer's choice of moments."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwad
import torch.nn.functional as F

import adapter_step_reference as ref
import test_gpu_adapter_model as model_tests
from auspex_soup_demo_b200 import _lib, kernels, qlora
from auspex_soup_demo_b200.multi_adapter import AdapterIds, MultiLoRANF4Linear
from auspex_soup_demo_b200.optim import MultiTensorAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error(torch.device("cuda:0")) == 0


def _flat(opt):
    """Parameters aside, what an optimiser holds of its one parameter: bytes of m and v, scales."""
    st = opt.flat_state()
    out = {k: st[k].view(torch.uint8).view(-1) if opt.state_bits == 8 else st[k].view(-1) for k in ("m", "v")}
    return out, {k: st[k] for k in ("m_scale", "v_scale") if k in st}


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("clip", [None, 1.0])
def test_gradients_that_are_not_finite_leave_their_neighbours(bits, dtype, what, clip):
    """One step with such gradients, then two sound ones, beside a copy that sees 0 in their
    places (everywhere, where a norm that is infinite scales all others to 0): every other
    element's parameter and moments are the copy's, bit for bit, and it moves in each sound
    step; in 8 bits the blocks' scales are the copy's too."""
    if clip is not None and math.isnan(what):
        pytest.skip("a norm that is not a number reaches every element")
    n, bad = 600, [3, 300, 301, 599]
    keep = torch.ones(n, dtype=torch.bool, device=DEV)
    keep[bad] = False
    g = torch.Generator(device=DEV).manual_seed(3)
    start = (0.05 * torch.randn(n, generator=g, device=DEV)).to(dtype)
    ps = [torch.nn.Parameter(start.clone()) for _ in range(2)]
    opts = [MultiTensorAdamW([p], lr=1e-2, state_bits=bits, max_grad_norm=clip) for p in ps]
    for step in range(3):
        grad = (1.0 + 0.1 * torch.randn(n, generator=g, device=DEV)).to(dtype)
        grad[bad] = 0.0
        before = ps[0].detach().clone()
        for p, o, first in zip(ps, opts, (True, False)):
            p.grad = grad.clone()
            if step == 0 and first:
                p.grad[bad] = what
            elif step == 0 and clip is not None:
                p.grad.zero_()
            o.step()
        assert torch.equal(ps[0].detach()[keep], ps[1].detach()[keep])
        assert not torch.isfinite(ps[0].detach()[~keep]).any()
        (states, scales), (states2, scales2) = map(_flat, opts)
        for k, s in states.items():
            assert torch.equal(s[:n][keep], states2[k][:n][keep]), (step, k)
            assert not s[n:].any()
        for k, s in scales.items():
            assert torch.equal(s, scales2[k]), (step, k)
        if step > 0:
            # gradients within a few tenths of 1 move an element by about lr
            assert float((ps[0].detach() - before).abs()[keep].min()) >= 2e-3, step


@pytest.mark.parametrize("change", [lambda p: p[:4].clone(), lambda p: p.cpu(), lambda p: p.bfloat16(),
                                    lambda p: p.view(4, 2).t()])
def test_parameters_given_other_memory_are_refused(change):
    """Another size, place, type or layout under a gradient that stays; before anything is written."""
    ps = [torch.nn.Parameter(torch.ones(8, device=DEV)) for _ in range(3)]
    opt = MultiTensorAdamW(ps, lr=1e-2, max_grad_norm=1.0)
    for p in ps:
        p.grad = torch.ones(8, device=DEV)
    opt.step()
    before = [p.detach().clone() for p in ps]
    old = ps[1].data
    ps[1].data = change(ps[1].data)
    with pytest.raises(ValueError, match="parameters must stay"):
        opt.step()
    assert torch.equal(ps[0], before[0]) and torch.equal(ps[2], before[2]) and torch.equal(old, before[1])
    assert float(opt.flat_state()["step"]) == 1.0
    ps[1].data = torch.zeros(8, device=DEV)  # other memory of the same form is the parameter's
    opt.step()
    assert ps[1].detach().all() and float(opt.flat_state()["step"]) == 2.0


def test_steps_are_seen_by_autograd():
    """A backward pass that needs the values before a step raises, as after torch's optimisers."""
    w = torch.nn.Parameter(torch.ones(300, device=DEV))
    unused = torch.nn.Parameter(torch.ones(8, device=DEV))
    loss = (w * w).sum()
    opt = MultiTensorAdamW([w, unused], lr=1e-2)
    w.grad = torch.ones_like(w)
    versions = w._version, unused._version
    opt.step()
    assert w._version > versions[0] and unused._version == versions[1]  # no gradient: not written
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("eps", [1e-8, 4e-12, 3e-12, 1e-26])
def test_second_moments_near_the_smallest_numbers(bits, eps):
    """Gradients of 1e-21 to 1e-16, whose second moments are subnormal or close to it, and an
    eps that is larger or smaller than their roots, against 64 bits: each of v's four
    operations rounds by 2^-24 of its result or by 2^-150, half of the smallest number; the
    rest are a dozen roundings of the update. Beside an eps of 3.5e-12 or more (for this
    beta2) roots may be low by 2.1e-20, less than eps' own rounding."""
    n, lr, betas = 256, 1e-3, (0.9, 0.99)
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = MultiTensorAdamW([p], lr=lr, betas=betas, eps=eps, state_bits=bits)
    e, tiny = 2.0 ** -24, 2.0 ** -150
    g = 10.0 ** torch.linspace(-21, -16, n, device=DEV)
    p.grad = g.clone()
    opt.step()
    want, m, v, _ = ref.adamw(torch.zeros_like(g), g, torch.zeros_like(g), torch.zeros_like(g), 1, lr, betas, eps, 0.0)
    slack = 8 * e * v + 4 * tiny
    least, most = torch.sqrt((v - slack).clamp_(min=0.0)), torch.sqrt(v + slack)
    step = lr / (1 - betas[0]) * m
    small, large = (step / (r / math.sqrt(1 - betas[1]) + eps) for r in (most, least))
    got = -p.detach().double()
    assert (got >= (1 - 12 * e) * small).all() and (got <= (1 + 12 * e) * large).all()
    st = opt.flat_state()
    if bits == 32:
        assert ((st["v"].double().view(-1) - v).abs() <= slack).all()
    else:
        low = 2.1e-20 if eps > 3.5e-12 else 0.0
        root, scale = st["v"].float().double().view(-1) * st["v_scale"].double(), float(st["v_scale"])
        assert abs(scale - float(torch.sqrt(v).max()) / 448) <= 8 * e * scale + low / 448
        code = (2.0 ** -4 + 4 * e) * most + 2.0 ** -9 * scale  # half a step of 2^-4, or the smallest code
        assert (root >= least - code - low).all() and (root <= most + code).all()


def test_forward_mode_derivatives_are_refused():
    """As the other operators': a tangent is refused, not dropped."""
    x, w = torch.randn(10, 64, device=DEV).bfloat16(), torch.randn(32, 64, device=DEV).bfloat16()
    a, b = torch.randn(2, 8, 64, device=DEV).bfloat16(), torch.randn(32, 2, 8, device=DEV).bfloat16()
    ids = torch.zeros(10, dtype=torch.int64, device=DEV)
    q, k = torch.randn(1, 2, 5, 8, device=DEV), torch.randn(1, 1, 5, 8, device=DEV)
    nw, cos, sin = torch.ones(8, device=DEV), torch.rand(5, 8, device=DEV), torch.rand(5, 8, device=DEV)
    pos, inv = torch.zeros(1, 5, dtype=torch.int64, device=DEV), torch.rand(4, device=DEV)
    calls = [(lambda t: kernels.multi_lora_linear(t, w, a, b, ids), x),
             (lambda t: kernels.multi_lora_linear(x, w, t, b, ids), a),
             (lambda t: kernels.multi_lora_linear(x, w, a, t, ids), b),
             (lambda t: kernels.apply_qk_norm_rope(t, k, nw, nw, cos, sin), q),
             (lambda t: kernels.apply_qk_norm_rope(q, k, nw, t, cos, sin), nw),
             (lambda t: kernels.apply_multi_axis_rope(q, t, pos, inv, (0,) * 4), k)]
    for grad in (True, False):
        for fn, t in calls:
            with torch.set_grad_enabled(grad), fwad.dual_level():
                with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                    fn(fwad.make_dual(t, torch.ones_like(t)))
                fn(t)  # no tangent: nothing to refuse


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_overlap(dtype):
    """Rows one element apart, and shared by all heads: any strides with a contiguous head dim
    are allowed. Results and gradients (those of each row by itself) against 64 bits."""
    b, h, s, d = 2, 3, 5, 8
    buf = torch.randn(4000, device=DEV).to(dtype)
    k = torch.randn(b, 1, s, d, device=DEV).to(dtype).requires_grad_(True)
    w = (1 + torch.rand(d, device=DEV)).requires_grad_(True)
    cos, sin = torch.rand(s, d, device=DEV), torch.rand(s, d, device=DEV)
    pos, inv = torch.arange(s, device=DEV)[None], torch.rand(d // 2, device=DEV)
    ang = (pos[0].double()[:, None] * inv.double())[None, None]
    g = torch.randn(b, h, s, d, device=DEV).to(dtype)
    tables = [t[None, None, :, :d // 2].double() for t in (cos, sin)]
    for strides in ((500, 100, 1, 1), (500, 0, 1, 1), (0, 1, 0, 1), (1, 0, 0, 1)):
        q = buf.as_strided((b, h, s, d), strides).requires_grad_(True)
        for norm in (True, False):
            if norm:
                qo, ko = kernels.apply_qk_norm_rope(q, k, w, w, cos, sin)
                want = ref.rotate(q, w, *tables, 1e-6, g)
            else:
                qo, ko = kernels.apply_multi_axis_rope(q, k, pos, inv, (0,) * (d // 2))
                want = ref.rotate(q, None, ang.cos(), ang.sin(), 0.0, g, angle_error=2.0 ** -21)
            (dq,) = torch.autograd.grad([qo, ko], [q], [g, torch.zeros_like(k)])
            assert qo.stride(-1) == ko.stride(-1) == 1
            ref.check("y", qo, want["y"])
            ref.check("dx", dq, want["dx"])


@pytest.mark.parametrize("tokens", [9, 300])
def test_base_weights_that_are_not_kept(tokens, monkeypatch):
    """With KEEP_BASE_WEIGHTS off nothing of the dense weight's size stays between the passes of
    an NF4 linear, and results and gradients are the same bits."""
    ids = AdapterIds(3)
    torch.manual_seed(0)
    lin = MultiLoRANF4Linear(torch.nn.Linear(256, 192, device=DEV, dtype=torch.bfloat16), ids, r=8)
    with torch.no_grad():
        lin.lora_B.normal_(std=0.1)
    x = torch.randn(1, tokens, 256, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn(1, tokens, 192, device=DEV, dtype=torch.bfloat16)
    ids.set((torch.arange(tokens, device=DEV) % 4 - 1)[None])
    runs = []
    for keep in (True, False):
        monkeypatch.setattr(qlora, "KEEP_BASE_WEIGHTS", keep)
        for grad in (True, False):  # with and without x's gradient, which needs the weight
            held = []
            leaves = [lin.lora_A, lin.lora_B] + ([x.requires_grad_(True)] if grad else [])
            x.requires_grad_(grad)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: held.append(tuple(t.shape)) or t, lambda t: t):
                y = lin(x)
            assert ((192, 256) in held) == (keep and grad)
            runs.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    for one, two in ((runs[0], runs[2]), (runs[1], runs[3]), (runs[0], runs[1])):
        for a, b in zip(one, two):
            assert torch.equal(a, b)


@pytest.mark.parametrize("attention", ["sdpa", "soup"])
def test_positions_of_several_axes_in_a_call_of_the_model(attention):
    """The model called with [axes, B, S] positions, beside its body with a prepared mask (no mask:
    causal) as the trainer calls it: at most an attention kernel apart, 16 roundings of bf16."""
    m = model_tests._model(attention=attention)
    ids, _, pos = model_tests._batch()
    m.adapter_ids.set(torch.tensor([0, 2, -1], device=DEV))
    with torch.no_grad():
        got = m(ids, position_ids=pos).logits
        want = m.lm_head(m.model(input_ids=ids, attention_mask={"full_attention": None}, position_ids=pos)[0])
        text = m(ids).logits
    assert float((got - want).abs().max()) <= 16 * 2.0 ** -8 * float(want.abs().max())
    assert not torch.equal(got, text)


def _one_adapter():
    cfg = qlora.qwen2_1p5b_config(1, hidden_size=256, intermediate_size=512, num_attention_heads=2,
                                  num_key_value_heads=1, vocab_size=1000, head_dim=128)
    return qlora.build_qwen2_qlora(cfg, device=DEV, r=8, alpha=16)


def test_clipping_alone_does_not_choose_8_bit_moments():
    """The trainer's own choice keeps fp32 moments; with a norm that clips nothing its steps are
    those of the flat optimiser: 16 roundings of 2^-24 of a parameter and its update a step,
    and an update is lr at most but for a few percent."""
    ids, labels, _ = model_tests._batch()
    den = float((labels != -100).sum())
    trainers = [qlora.QLoRATrainer(_one_adapter(), max_grad_norm=1e9), qlora.QLoRATrainer(_one_adapter(), optimizer="soup"),
                qlora.QLoRATrainer(_one_adapter(), optimizer="soup32", max_grad_norm=1e-3),
                qlora.QLoRATrainer(_one_adapter(), optimizer="soup8", max_grad_norm=1e-3)]
    assert [t.opt and t.opt.state_bits for t in trainers] == [32, None, 32, 8]
    for t in trainers:
        loss, _ = t.step(ids, labels, den)
        assert torch.isfinite(loss)
    one, two = (t.flat_param for t in trainers[:2])
    assert float((one - two).abs().max()) <= 16 * 2.0 ** -24 * (float(two.abs().max()) + 2e-4)
    assert float(trainers[0].opt.grad_norm) > 1e-3
    for bad in ("soup", "torch"):
        with pytest.raises(ValueError, match="soup32"):
            qlora.QLoRATrainer(_one_adapter(), optimizer=bad, max_grad_norm=1.0)


@pytest.mark.parametrize("again", [lambda w: w[:-8], lambda w: w[:, :-8], lambda w: w.float(), lambda w: w.cpu()])
def test_a_weight_formed_again_is_checked(again):
    x, w = torch.randn(20, 64, device=DEV).bfloat16().requires_grad_(True), torch.randn(32, 64, device=DEV).bfloat16()
    a, b = torch.randn(2, 8, 64, device=DEV).bfloat16(), torch.randn(32, 2, 8, device=DEV).bfloat16()
    ids = torch.zeros(20, dtype=torch.int64, device=DEV)
    y = kernels.multi_lora_linear(x, w, a, b, ids, weight_fn=lambda: again(w))
    with pytest.raises(ValueError, match="weight_fn"):
        y.float().sum().backward()
    y = kernels.multi_lora_linear(x, w, a, b, ids, weight_fn=lambda: w.t().contiguous().t())  # any strides
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    (want,) = torch.autograd.grad(kernels.multi_lora_linear(x, w, a, b, ids), x, torch.ones_like(y))
    assert torch.equal(dx, want)


@pytest.mark.parametrize("sections", [None, model_tests.SECTIONS])
@pytest.mark.parametrize("quantize", [False, True])
def test_heads_beside_grouped_projections(quantize, sections):
    """One adapter, norms and axes of heads, q/k/v and gate/up as one product each or by
    themselves: the same gradients but for the roundings between them (some 40 of 2^-9 rms in
    either, a cosine of 0.9998; asked for are 0.995)."""
    cfg = qlora.qwen2_1p5b_config(2, hidden_size=256, intermediate_size=512, num_attention_heads=2,
                                  num_key_value_heads=1, vocab_size=1000, head_dim=128)
    ids, labels, pos = model_tests._batch()
    runs = []
    for group in (True, False):
        m = qlora.build_qwen2_qlora(cfg, device=DEV, r=8, alpha=16, quantize=quantize, qk_norm=True, train_norms=True,
                                    rope_sections=sections, group=group)
        g = torch.Generator(device=DEV).manual_seed(1)
        with torch.no_grad():
            for n, p in m.named_parameters():
                if "lora_B" in n:
                    p.copy_(0.05 * torch.randn(p.shape, generator=g, device=DEV))
        runs.append(model_tests._loss_and_grads(m, ids, labels, None, pos if sections else None))
    (loss, grads), (loss2, grads2) = runs
    assert abs(loss - loss2) <= 2e-2 * abs(loss2) and any("q_norm" in n for n in grads)
    for n, x in grads.items():
        assert float(F.cosine_similarity(x.double().flatten(), grads2[n].double().flatten(), dim=0)) >= 0.995, n
