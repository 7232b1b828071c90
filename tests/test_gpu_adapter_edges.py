"""GPU: calls of the adapters', norms' and optimiser's entry points that are allowed and rare:
masked rows that are not finite, tensors saved on the host, addresses off the vector grid,
groups added to a captured optimiser, offsets that pass 32 bits."""

import math

import pytest
import torch

import adapter_step_reference as ref
from auspex_soup_demo_b200 import _lib, kernels
from auspex_soup_demo_b200.optim import MultiTensorAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error(torch.device("cuda:0")) == 0


def _lora(t, k, n, na, r, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device=DEV).bfloat16()

    scale = 0.5 + torch.rand(na, generator=g, device=DEV)
    return randn(t, k), randn(n, k) * 0.05, randn(na, r, k) * k ** -0.5, randn(n, na, r) * 0.2, scale, randn(t, n)


@pytest.mark.parametrize("what", [math.nan, math.inf])
@pytest.mark.parametrize("t,per", [(60, 1), (200, 7), (700, 50)])
def test_masked_rows_that_are_not_finite_reach_no_gradient(t, per, what):
    """Rows without an adapter, and of an adapter of another rank block, in x and in dy."""
    k, n, na, r = 192, 136, 6, 16  # columns 0-63: adapters 0-3, the others: 4 and 5
    x, w, a, b, scale, dy = _lora(t, k, n, na, r, t)
    ids = torch.tensor([0, -1, 3, 6, 5, 1], device=DEV).repeat_interleave(per).repeat(-(-t // (6 * per)))[:t]
    masked = (ids < 0) | (ids > 5)
    gone = masked | (ids == 5)
    keep = [0, 1, 2, 3]
    want = ref.multi_lora(torch.where(gone[:, None], 0, x), w, a, b, ids, scale, None, torch.where(gone[:, None], 0, dy))
    x[gone] = what
    dy[gone] = what
    leaves = [v.requires_grad_(True) for v in (x, a, b)]
    y = kernels.multi_lora_linear(x, w, a, b, ids, scale)
    dx, da, db = torch.autograd.grad(y, leaves, dy)
    rows = ~gone
    for name, got in (("y", y), ("dx", dx)):
        whole = want[name]
        ref.check(name, got[rows], tuple(v[rows] for v in whole) if isinstance(whole, tuple) else whole[rows])
    for name, got, pick in (("da", da, lambda v: v[keep]), ("db", db, lambda v: v[:, keep])):
        whole = want[name]
        ref.check(name, pick(got), tuple(pick(v) for v in whole) if isinstance(whole, tuple) else pick(whole))


@pytest.mark.parametrize("t,k,n,na,r", [(1, 8, 8, 1, 8), (17, 8, 24, 2, 4), (130, 16, 8, 8, 1), (300, 8, 8, 3, 8),
                                        (257, 24, 40, 1, 64), (600, 8, 264, 40, 1)])
def test_smallest_widths_and_ranks(t, k, n, na, r):
    x, w, a, b, scale, dy = _lora(t, k, n, na, r, t + k)
    ids = torch.arange(t, device=DEV) % (na + 1) - 1
    leaves = [v.requires_grad_(True) for v in (x, a, b)]
    y = kernels.multi_lora_linear(x, w, a, b, ids, scale)
    grads = torch.autograd.grad(y, leaves, dy)
    want = ref.multi_lora(x, w, a, b, ids, scale, None, dy)
    for name, got in zip(("y", "dx", "da", "db"), (y, *grads)):
        ref.check(name, got, want[name])


@pytest.mark.parametrize("t", [8, 200, 1200])
def test_bias_and_rows_at_any_address(t):
    k, n = 136, 9344 if t == 200 else 200
    x, w, a, b, scale, _ = _lora(t, k, n, 3, 8, 2)
    ids = torch.arange(t, device=DEV) % 4 - 1
    bias = torch.randn(n, device=DEV).bfloat16()
    wide = torch.zeros(t, k + 24, device=DEV, dtype=torch.bfloat16)
    wide[:, 3:3 + k] = x  # rows off the 16-byte grid
    far = torch.zeros(n + 1, device=DEV, dtype=torch.bfloat16)
    far[1:] = bias
    cols = w.t().contiguous().t()  # a weight of column order
    with torch.no_grad():
        want = kernels.multi_lora_linear(x, w, a, b, ids, scale, bias)
        assert torch.equal(kernels.multi_lora_linear(wide[:, 3:3 + k], cols, a, b, ids, scale, far[1:]), want)


def _leaves(seed=0):
    x, w, a, b, scale, dy = _lora(100, 128, 64, 4, 8, seed)
    return x, w, a, b, scale, torch.arange(100, device=DEV) // 30, dy


def test_saved_on_the_host():
    x, w, a, b, scale, ids, dy = _leaves()
    q = torch.randn(2, 3, 20, 64, device=DEV, dtype=torch.bfloat16).transpose(1, 2).contiguous().transpose(1, 2)
    k = torch.randn(2, 1, 20, 64, device=DEV, dtype=torch.bfloat16)
    nw = torch.rand(2, 64, device=DEV).bfloat16()
    cos, sin = torch.rand(2, 20, 64, device=DEV)
    pos = torch.arange(40, device=DEV).view(2, 20).t().expand(20, 2).t()[None]
    inv = torch.rand(32, device=DEV)

    def run():
        leaves = [v.detach().clone().requires_grad_(True) for v in (x, a, b, q, k, nw[0], nw[1])]
        y = kernels.multi_lora_linear(leaves[0], w, leaves[1], leaves[2], ids, scale)
        q1, k1 = kernels.apply_qk_norm_rope(*leaves[3:], cos, sin)
        q2, k2 = kernels.apply_multi_axis_rope(q1, k1, pos, inv, (0,) * 32)
        return torch.autograd.grad([y, q2, k2], leaves, [dy, torch.ones_like(q2), torch.ones_like(k2)])

    want = run()
    with torch.autograd.graph.save_on_cpu():
        got = run()
    for p, g in zip(want, got):
        assert torch.equal(p, g)


def test_second_derivatives_are_refused():
    x, w, a, b, scale, ids, dy = _leaves()
    a.requires_grad_(True)
    (da,) = torch.autograd.grad(kernels.multi_lora_linear(x, w, a, b, ids, scale), a, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        da.float().square().sum().backward()


def test_training_calls_in_a_graph():
    """Forward and backward captured, on new contents of the same buffers."""
    x, w, a, b, scale, ids, dy = _leaves(3)
    q = torch.randn(1, 4, 100, 64, device=DEV, dtype=torch.bfloat16)
    k = torch.randn(1, 2, 100, 64, device=DEV, dtype=torch.bfloat16)
    nw = torch.rand(64, device=DEV).bfloat16()
    pos, inv = torch.arange(100, device=DEV)[None], torch.rand(32, device=DEV)
    leaves = [v.requires_grad_(True) for v in (x, a, b, q, k, nw)]

    def run():
        y = kernels.multi_lora_linear(leaves[0], w, leaves[1], leaves[2], ids, scale)
        qo, ko = kernels.apply_multi_axis_rope(leaves[3], leaves[4], pos, inv, (0,) * 32, leaves[5], leaves[5])
        return torch.autograd.grad([y, qo, ko], leaves, [dy, qo.detach(), ko.detach()])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    with torch.no_grad():
        x.mul_(-0.5)
        ids.copy_(ids.flip(0))
        q.add_(1.0)
        pos.add_(9)
    graph.replay()
    for got, want in zip(held, run()):
        assert torch.equal(got, want)


def test_adamw_groups_added_later_and_empty_ones():
    """A captured step keeps its workspace when a later group needs a larger one."""
    ps = [torch.nn.Parameter(torch.ones(40, device=DEV)) for _ in range(2)]
    opt = MultiTensorAdamW([{"params": []}, {"params": ps[:1]}], lr=1e-2, max_grad_norm=1.0)
    for p in ps:
        p.grad = torch.full_like(p, 2.0)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.add_param_group({"params": [ps[1]], "lr": 0.0})
    junk = [torch.zeros(1 << 14, device=DEV) for _ in range(8)]  # where a freed workspace would be
    graph.replay()
    torch.cuda.synchronize()
    assert abs(float(opt.grad_norm) - 2.0 * 40 ** 0.5) <= 1e-5
    assert not any(j.any() for j in junk)
    opt.step()
    assert abs(float(opt.grad_norm) - 2.0 * 80 ** 0.5) <= 1e-5
    assert torch.equal(ps[1], torch.ones_like(ps[1]))


def test_adamw_parameters_that_moved_are_refused():
    ps = [torch.nn.Parameter(torch.ones(8, device=DEV)) for _ in range(2)]
    opt = MultiTensorAdamW(ps, lr=1e-2)
    ps[1].data = ps[1].data.cpu()
    ps[1].grad = torch.ones(8)
    ps[0].grad = torch.ones(8, device=DEV)
    with pytest.raises(ValueError, match="gradients must be"):
        opt.step()


def test_two_optimisers_on_two_streams():
    def steps(opt, p, n=20):
        for i in range(n):
            p.grad = torch.sin(p.detach() * (i + 1))
            opt.step()
        return p.detach()

    def pair():
        ps = [torch.nn.Parameter(torch.linspace(-1, 1, 5000 + 7 * i, device=DEV)) for i in range(2)]
        return ps, [MultiTensorAdamW([p], lr=1e-2, max_grad_norm=0.5) for p in ps]

    want = [steps(o, p) for p, o in zip(*pair())]
    ps, opts = pair()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s, p, o in zip(streams, ps, opts):
        with torch.cuda.stream(s):
            steps(o, p)
    torch.cuda.synchronize()
    for p, w in zip(ps, want):
        assert torch.equal(p.detach(), w)


# ------------------------------------------------------- offsets that pass 32 bits ----
def test_rotation_of_more_than_2_to_31_elements():
    h, hk, s, d, tail = 66, 1, 257000, 128, 70
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.zeros(1, h, s, d, device=DEV, dtype=torch.bfloat16)
    k = torch.zeros(1, hk, s, d, device=DEV, dtype=torch.bfloat16)
    assert q.numel() > 1 << 31
    q[:, :, -tail:] = torch.randn(1, h, tail, d, generator=g, device=DEV)
    k[:, :, -tail:] = torch.randn(1, hk, tail, d, generator=g, device=DEV)
    w = [(1 + torch.rand(d, device=DEV)).bfloat16().requires_grad_(True) for _ in range(2)]
    pos, inv = torch.arange(s, device=DEV)[None], torch.rand(d // 2, device=DEV)

    def run(q, k, pos):
        q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        out = kernels.apply_multi_axis_rope(q, k, pos, inv, (0,) * (d // 2), *w)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, [q, k, *w], [q.detach(), k.detach()]))

    whole = run(q, k, pos)
    part = run(q[:, :, -tail:].contiguous(), k[:, :, -tail:].contiguous(), pos[:, -tail:])
    for i in range(4):
        assert torch.equal(whole[i][:, :, -tail:], part[i])
    for i in (4, 5):  # rows of zeros add zeros, in another order of sums
        torch.testing.assert_close(whole[i], part[i], rtol=2 ** -7, atol=2 ** -7 * float(part[i].abs().max()))


def test_adapters_with_more_than_2_to_31_outputs():
    t, n, k, tail = 131072, 16512, 64, 256
    assert t * n > 1 << 31
    x, w, a, b, scale, _ = _lora(t, k, n, 4, 16, 5)
    ids = torch.arange(t, device=DEV) // 1000 % 5 - 1
    with torch.no_grad():
        y = kernels.multi_lora_linear(x, w, a, b, ids, scale)
        want = ref.multi_lora(x[-tail:], w, a, b, ids[-tail:], scale, None)["y"]
    ref.check("y", y[-tail:], want)
    x.requires_grad_(True)
    dy = torch.zeros_like(y)
    dy[-tail:] = torch.randn(tail, n, device=DEV)
    leaves = [x, a.requires_grad_(True), b.requires_grad_(True)]
    dx, da, db = torch.autograd.grad(kernels.multi_lora_linear(x, w, a, b, ids, scale), leaves, dy)
    want = ref.multi_lora(x[-tail:], w, a, b, ids[-tail:], scale, None, dy[-tail:])
    ref.check("dx", dx[-tail:], want["dx"])
    assert not dx[:-tail].any()
    ref.check("da", da, want["da"])
    ref.check("db", db, want["db"])


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_of_more_than_2_to_31_elements(bits):
    n = (1 << 31) + 1000
    g = torch.randn(1000, device=DEV).bfloat16()
    big = torch.nn.Parameter(torch.ones(n, device=DEV, dtype=torch.bfloat16))
    big.grad = torch.zeros_like(big)
    big.grad[-1000:] = g
    small = torch.nn.Parameter(torch.ones(1000, device=DEV, dtype=torch.bfloat16))
    small.grad = g.clone()
    norms = []
    for p in (big, small):  # 2^31 is a multiple of 256: the same blocks at the end
        opt = MultiTensorAdamW([p], lr=0.1, state_bits=bits, max_grad_norm=5.0)
        for _ in range(2):
            opt.step()
        norms.append(opt.grad_norm.clone())
        del opt
    assert torch.equal(big.detach()[-1000:], small.detach())
    assert bool((big.detach()[:-1000] == 1).all())
    torch.testing.assert_close(norms[0], norms[1], rtol=1e-6, atol=0)
