"""GPU: projections with several adapters, norms of queries and keys with their
rotation, positions of several axes and AdamW over many tensors, against 64 bits."""

import math

import pytest
import torch

import adapter_step_reference as ref
from auspex_soup_demo_b200 import _lib, kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert _lib.device_error(torch.device("cuda:0")) == 0


# ------------------------------------------------------------ several adapters ----
def _lora_inputs(t, k, n, na, r, seed, runs=None, bias=False):
    g = _gen(seed)
    bf = torch.bfloat16
    x = _randn(g, t, k, dtype=bf)
    w = _randn(g, n, k, dtype=bf) * 0.05
    a = _randn(g, na, r, k, dtype=bf) * k ** -0.5
    b = _randn(g, n, na, r, dtype=bf) * 0.2
    scale = 0.5 + torch.rand(na, generator=g, device=DEV)
    if runs is None:  # every token its own
        ids = torch.randint(-1, na, (t,), generator=g, device=DEV)
    else:  # runs of equal ids
        ids = torch.randint(-1, na, (-(-t // runs),), generator=g, device=DEV).repeat_interleave(runs)[:t]
    return x, w, a, b, ids, scale, _randn(g, n, dtype=bf) if bias else None


LORA = [
    # tokens, K, N, adapters, rank, run length, bias
    (1, 64, 64, 1, 8, 1, False),
    (1, 1536, 2048, 7, 16, 1, True),
    (5, 200, 136, 3, 8, None, True),
    (16, 512, 384, 40, 16, None, False),
    (17, 1536, 640, 64, 16, None, True),
    (33, 264, 1000, 5, 24, None, False),
    (64, 1536, 2048, 128, 32, None, False),
    (65, 1536, 2048, 64, 64, None, True),
    (128, 392, 712, 12, 16, 3, False),
    (200, 1536, 640, 31, 16, None, True),
    (256, 264, 9600, 3, 8, 9, True),
    (256, 264, 9344, 3, 8, 9, True),
    (127, 72, 88, 2, 4, 50, False),
    (129, 640, 512, 9, 16, 13, True),
    (300, 512, 264, 300, 8, 1, False),
    (257, 128, 320, 256, 16, None, False),
    (1000, 896, 1160, 24, 8, 91, True),
    (2050, 1536, 2048, 4, 16, 700, False),
]


@pytest.mark.parametrize("t,k,n,na,r,runs,bias", LORA)
def test_multi_lora_against_64_bits(t, k, n, na, r, runs, bias):
    x, w, a, b, ids, scale, bi = _lora_inputs(t, k, n, na, r, t + k, runs, bias)
    dy = _randn(_gen(9), t, n, dtype=torch.bfloat16)
    want = ref.multi_lora(x, w, a, b, ids, scale, bi, dy)
    with torch.no_grad():
        y0 = kernels.multi_lora_linear(x, w, a, b, ids, scale, bi)
    ref.check("y", y0, want["y"])
    for t_ in (x, a, b):
        t_.requires_grad_(True)
    y = kernels.multi_lora_linear(x, w, a, b, ids.to(torch.int32), scale, bi)
    assert torch.equal(y, y0)
    grads = torch.autograd.grad(y, [x, a, b], dy)
    for name, got in zip(("dx", "da", "db"), grads):
        assert got.dtype == torch.bfloat16
        ref.check(name, got, want[name])


@pytest.mark.parametrize("which", [(True, False, False), (False, True, False), (False, False, True)])
def test_multi_lora_single_gradients(which):
    x, w, a, b, ids, scale, _ = _lora_inputs(200, 256, 192, 6, 16, 3, 40)
    dy = _randn(_gen(4), 200, 192, dtype=torch.bfloat16)
    leaves = [t.requires_grad_(f) for t, f in zip((x, a, b), which)]
    y = kernels.multi_lora_linear(x, w, a, b, ids, scale)
    leaf = [t for t in leaves if t.requires_grad]
    (got,) = torch.autograd.grad(y, leaf, dy)
    name = ("dx", "da", "db")[which.index(True)]
    ref.check(name, got, ref.multi_lora(x, w, a, b, ids, scale, None, dy)[name])


def test_multi_lora_ids_of_sequences_strides_and_fp32_factors():
    """[B, S, K] with an id a sequence, rows of a wider buffer, fp32 factors."""
    g = _gen(5)
    bsz, s, k, n, na, r = 3, 77, 320, 256, 4, 8
    wide = _randn(g, bsz * s, k + 64, dtype=torch.bfloat16)
    x = wide[:, 32:32 + k].view(bsz, s, k)
    _, w, a, b, _, scale, _ = _lora_inputs(1, k, n, na, r, 6)
    a32 = (a.float() + 1e-4).requires_grad_(True)
    b32 = (b.float() - 1e-4).requires_grad_(True)
    ids = torch.tensor([2, -1, 0], device=DEV)
    y = kernels.multi_lora_linear(x, w, a32, b32, ids, scale)
    dy = _randn(g, n, bsz, s, dtype=torch.bfloat16).permute(1, 2, 0)  # strided gradient
    da, db = torch.autograd.grad(y, [a32, b32], dy)
    assert da.dtype == db.dtype == torch.float32
    want = ref.multi_lora(x.reshape(-1, k), w, a32.bfloat16(), b32.bfloat16(), ids.repeat_interleave(s), scale, None,
                          dy.reshape(-1, n))
    ref.check("y", y.reshape(-1, n), want["y"])
    ref.check("da", da, want["da"])
    ref.check("db", db, want["db"])
    assert not da[1].any() and not da[3].any() and not db[:, 1].any()


def test_multi_lora_no_adapter_at_all_and_ids_out_of_range():
    x, w, a, b, ids, scale, bias = _lora_inputs(150, 128, 192, 3, 16, 8, 10, True)
    for bad in (-1, 3, -(1 << 40), 1 << 40):
        xs = x.clone().requires_grad_(True)
        aa, bb = a.clone().requires_grad_(True), b.clone().requires_grad_(True)
        y = kernels.multi_lora_linear(xs, w, aa, bb, torch.full_like(ids, bad), scale, bias)
        none = torch.full_like(ids, -1)
        dy = torch.ones_like(y)
        want = ref.multi_lora(x, w, a, b, none, scale, bias, dy)
        ref.check("y", y, want["y"])
        dx, da, db = torch.autograd.grad(y, [xs, aa, bb], dy)
        ref.check("dx", dx, want["dx"])
        assert not da.any() and not db.any()


def test_multi_lora_unused_adapters_may_hold_anything():
    """NaN in the factors of an adapter whose rank block no token reads changes nothing; in
    a block that is read, only that adapter's own gradients would be touched by zeros."""
    x, w, a, b, ids, scale, _ = _lora_inputs(128, 128, 128, 8, 64, 11, 16)
    ids = torch.where(ids == 5, torch.full_like(ids, 2), ids)
    y0 = kernels.multi_lora_linear(x, w, a, b, ids, scale)
    a[5] = math.nan
    b[:, 5] = math.inf
    assert torch.equal(kernels.multi_lora_linear(x, w, a, b, ids, scale), y0)


def test_multi_lora_no_tokens():
    _, w, a, b, _, scale, _ = _lora_inputs(1, 64, 72, 2, 8, 1)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    a.requires_grad_(True)
    y = kernels.multi_lora_linear(x, w, a, b, torch.empty(0, dtype=torch.int64, device=DEV), scale)
    assert y.shape == (0, 72)
    dx, da = torch.autograd.grad(y, [x, a], torch.empty_like(y))
    assert dx.shape == x.shape and not da.any()


def test_multi_lora_repeats_bitwise_and_on_two_streams():
    x, w, a, b, ids, scale, _ = _lora_inputs(900, 1024, 640, 16, 16, 21, 33)
    dy = _randn(_gen(2), 900, 640, dtype=torch.bfloat16)

    def once():
        xs, aa, bb = (t.detach().clone().requires_grad_(True) for t in (x, a, b))
        y = kernels.multi_lora_linear(xs, w, aa, bb, ids, scale)
        return [y.detach(), *torch.autograd.grad(y, [xs, aa, bb], dy)]

    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(once())
    torch.cuda.synchronize()
    for res in results:
        for p, q in zip(first, res):
            assert torch.equal(p, q)


@pytest.mark.parametrize("t", [8, 320])
def test_multi_lora_in_a_graph_with_new_ids(t):
    x, w, a, b, ids, scale, _ = _lora_inputs(t, 256, 512, 10, 16, 31, 5)
    static = ids.clone()
    with torch.no_grad():
        kernels.multi_lora_linear(x, w, a, b, static, scale)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = kernels.multi_lora_linear(x, w, a, b, static, scale)
        for shift in range(3):
            new = (ids + 1 + shift) % 11 - 1
            static.copy_(new)
            g.replay()
            ref.check("y", y, ref.multi_lora(x, w, a, b, new, scale, None)["y"])


# --------------------------------------------------- norms and rotation of q and k ----
def _tables(s, d, dtype, batch=None, seed=0):
    inv = 1.0 / (1e4 ** (torch.arange(0, d, 2, device=DEV).double() / d))
    pos = torch.arange(s, device=DEV).double()
    if batch is not None:
        pos = pos[None] + 17.0 * torch.arange(batch, device=DEV)[:, None]
    ang = pos[..., None] * inv
    emb = torch.cat([ang, ang], -1)
    return emb.cos().to(dtype), emb.sin().to(dtype)


def _qk(b, h, hk, s, d, dtype, seed, packed):
    g = _gen(seed)
    if packed:
        both = _randn(g, b, s, (h + hk + 1) * d, dtype=dtype)
        q = both[..., :h * d].view(b, s, h, d).transpose(1, 2)
        k = both[..., h * d:(h + hk) * d].view(b, s, hk, d).transpose(1, 2)
    else:
        q, k = _randn(g, b, h, s, d, dtype=dtype), _randn(g, b, hk, s, d, dtype=dtype)
    return q, k


QK = [
    # B, H, Hk, S, D, dtype, packed
    (1, 1, 1, 1, 2, torch.float32, False),
    (1, 12, 2, 1, 128, torch.bfloat16, True),
    (3, 12, 2, 70, 128, torch.bfloat16, True),
    (2, 7, 1, 33, 64, torch.float16, False),
    (2, 4, 4, 19, 96, torch.bfloat16, True),
    (1, 3, 1, 50, 80, torch.float32, False),
    (2, 5, 5, 9, 34, torch.bfloat16, False),
    (1, 16, 8, 21, 256, torch.bfloat16, True),
    (1, 2, 1, 40, 512, torch.float32, False),
    (1, 2, 1, 11, 512, torch.float16, False),
    (2, 64, 8, 130, 128, torch.bfloat16, False),
    (5, 6, 3, 1200, 64, torch.bfloat16, True),
]


@pytest.mark.parametrize("b,h,hk,s,d,dtype,packed", QK)
def test_qk_norm_rope_against_64_bits(b, h, hk, s, d, dtype, packed):
    q, k = _qk(b, h, hk, s, d, dtype, s + d, packed)
    g = _gen(1)
    qw, kw = (1 + 0.3 * _randn(g, d)).to(dtype), (1 + 0.3 * _randn(g, d)).to(dtype)
    cos, sin = _tables(s, d, dtype, batch=b)
    gq, gk = _randn(g, b, h, s, d, dtype=dtype), _randn(g, b, s, hk, d, dtype=dtype).transpose(1, 2)
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    qo, ko = kernels.apply_qk_norm_rope(q, k, qw, kw, cos, sin, 1e-5)
    grads = torch.autograd.grad([qo, ko], leaves, [gq, gk])
    c, sn = cos.double()[:, None, :, :d // 2], sin.double()[:, None, :, :d // 2]
    for x, w, o, gr, dx, dw in ((q, qw, qo, gq, grads[0], grads[2]), (k, kw, ko, gk, grads[1], grads[3])):
        want = ref.rotate(x, w, c, sn, 1e-5, gr)
        assert o.dtype == dtype and dw.dtype == w.dtype
        ref.check("y", o, want["y"])
        ref.check("dx", dx, want["dx"])
        ref.check("dw", dw, want["dw"])


def test_qk_norm_rope_forms_of_tables_and_weights():
    b, h, hk, s, d = 2, 4, 2, 37, 64
    q, k = _qk(b, h, hk, s, d, torch.bfloat16, 3, True)
    g = _gen(2)
    qw, kw = 1 + 0.1 * _randn(g, d), 1 + 0.1 * _randn(g, d)  # fp32 weights beside bf16 rows
    cos, sin = _tables(s, d, torch.float32)
    base = kernels.apply_qk_norm_rope(q, k, qw, kw, cos, sin)
    for c, sn in ((cos[None], sin[None]), (cos[None, None].expand(b, 1, s, d), sin[None, None].expand(b, 1, s, d)),
                  (cos.t().contiguous().t(), sin), (cos[None].expand(b, s, d).contiguous(), sin[None].expand(b, s, d))):
        got = kernels.apply_qk_norm_rope(q, k, qw, kw, c, sn)
        assert torch.equal(got[0], base[0]) and torch.equal(got[1], base[1])
    ref.check("y", base[0], ref.rotate(q, qw, cos.double()[None, None, :, :32], sin.double()[None, None, :, :32],
                                       1e-6)["y"])
    # one gradient alone, and rows that are not contiguous
    q2 = q.transpose(2, 3).contiguous().transpose(2, 3).requires_grad_(True)
    qo, ko = kernels.apply_qk_norm_rope(q2, k, qw, kw, cos, sin)
    assert torch.equal(qo, base[0])
    (dq,) = torch.autograd.grad(qo.float().square().sum(), [q2])
    gr = 2 * base[0]
    ref.check("dx", dq, ref.rotate(q, qw, cos.double()[None, None, :, :32], sin.double()[None, None, :, :32], 1e-6,
                                   gr)["dx"])


def test_qk_norm_rope_rows_of_zeros_and_infinities():
    """A row of zeros has rstd 1 / sqrt(eps); a row with NaN or infinity stays its own affair."""
    b, h, hk, s, d = 1, 2, 1, 6, 128
    q, k = _qk(b, h, hk, s, d, torch.bfloat16, 4, False)
    q[0, 0, 1] = 0
    q[0, 1, 3, 5] = math.inf
    q[0, 0, 4, 7] = math.nan
    w = torch.ones(d, device=DEV, dtype=torch.bfloat16)
    cos, sin = _tables(s, d, torch.float32)
    qs = q.clone().requires_grad_(True)
    qo, ko = kernels.apply_qk_norm_rope(qs, k, w, w, cos, sin)
    bad = torch.zeros(b, h, s, dtype=torch.bool, device=DEV)
    bad[0, 1, 3] = bad[0, 0, 4] = True
    assert torch.isfinite(qo[~bad]).all() and not torch.isfinite(qo[bad]).all()
    assert not qo[0, 0, 1].any()
    (dq,) = torch.autograd.grad(qo, [qs], torch.ones_like(qo))
    assert torch.isfinite(dq[~bad]).all()
    want = ref.rotate(torch.zeros_like(q[:, :1, 1:2]), w, cos.double()[None, None, 1:2, :64],
                      sin.double()[None, None, 1:2, :64], 1e-6, torch.ones_like(q[:, :1, 1:2]))
    ref.check("dx", dq[:, :1, 1:2], want["dx"])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("far", [0, 1 << 20])
def test_multi_axis_rope_against_64_bits(dtype, norm, interleaved, far):
    b, h, hk, s, d = 2, 6, 2, 45, 128
    q, k = _qk(b, h, hk, s, d, dtype, 6, True)
    g = _gen(3)
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device=DEV).float() / d))
    pos = torch.randint(-5, 400, (3, b, s), generator=g, device=DEV) + far
    sections = (16, 24, 24)
    axes = kernels.rope_axes(sections, interleaved)
    ang = pos[list(axes)].permute(1, 2, 0).double() * inv.double()
    c, sn = ang.cos()[:, None], ang.sin()[:, None]
    w = (1 + 0.2 * _randn(g, d)).to(dtype), (1 + 0.2 * _randn(g, d)).to(dtype)
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    leaves = [q.requires_grad_(True), k.requires_grad_(True)]
    if norm:
        leaves += [t.requires_grad_(True) for t in w]
    args = w if norm else (None, None)
    for p in (pos, pos.to(torch.int32)):
        qo, ko = kernels.apply_multi_axis_rope(q, k, p, inv, axes, *args)
        grads = torch.autograd.grad([qo, ko], leaves, [gq, gk])
        for i, (x, o, gr) in enumerate(((q, qo, gq), (k, ko, gk))):
            # the reduced angle in 32 bits (pi 2^-24) and sincospi's two last places
            want = ref.rotate(x, args[i], c, sn, 1e-6, gr, angle_error=2.0 ** -21)
            ref.check("y", o, want["y"])
            ref.check("dx", grads[i], want["dx"])
            if norm:
                ref.check("dw", grads[2 + i], want["dw"])


def test_multi_axis_rope_of_equal_axes_is_the_rotation_by_tables():
    b, h, hk, s, d = 2, 3, 1, 20, 64
    q, k = _qk(b, h, hk, s, d, torch.float32, 7, False)
    inv = 1.0 / (1e4 ** (torch.arange(0, d, 2, device=DEV).float() / d))
    axes = kernels.rope_axes((8, 12, 12))
    pos = torch.arange(s, device=DEV)
    ang = pos.double()[:, None] * inv.double()
    cos, sin = (torch.cat([f(ang)] * 2, -1).float() for f in (torch.cos, torch.sin))
    want = kernels.apply_fast_rope_qk(q, k, cos, sin)
    for p in (pos.expand(3, s), pos.expand(3, b, s), pos.expand(3, 1, s).contiguous()):
        got = kernels.apply_multi_axis_rope(q, k, p, inv, axes)
        for x, y, z in zip(got, want, (q, k)):
            # two tables that differ by 2^-21 on each of two terms
            assert float((x - y).abs().max()) <= 2.0 ** -20 * float(z.abs().max())


def test_qk_norm_rope_gradients_against_differences():
    """Central differences of a fp32 loss, steps of 2^-6: their own error is the third
    derivative's h^2 / 6 (a few 1e-4 here) and 2^-24 of the loss over h."""
    b, h, hk, s, d = 1, 2, 1, 3, 16
    q, k = _qk(b, h, hk, s, d, torch.float32, 9, False)
    g = _gen(4)
    w = 1 + 0.2 * _randn(g, d), 1 + 0.2 * _randn(g, d)
    cos, sin = _tables(s, d, torch.float32)
    cq, ck = _randn(g, b, h, s, d), _randn(g, b, hk, s, d)

    def loss(q, k, a, c):
        qo, ko = kernels.apply_qk_norm_rope(q, k, a, c, cos, sin)
        return ((qo.double() * cq).sum() + (ko.double() * ck).sum())

    leaves = [t.clone().requires_grad_(True) for t in (q, k, *w)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    step = 2.0 ** -6
    for i, t in enumerate(leaves):
        for at in (0, 5, t.numel() - 1):
            vals = []
            for sign in (1, -1):
                moved = [x.detach().clone() for x in leaves]
                moved[i].view(-1)[at] += sign * step
                vals.append(float(loss(*moved)))
            diff = (vals[0] - vals[1]) / (2 * step)
            assert abs(diff - float(grads[i].reshape(-1)[at])) <= 2e-3 * (1 + abs(diff)), (i, at)


def test_rotations_in_a_graph_and_empty():
    b, h, hk, s, d = 2, 4, 2, 8, 128
    q, k = _qk(b, h, hk, s, d, torch.bfloat16, 12, False)
    inv = 1.0 / (1e4 ** (torch.arange(0, d, 2, device=DEV).float() / d))
    axes = kernels.rope_axes((16, 24, 24))
    pos = torch.zeros(3, b, s, dtype=torch.int64, device=DEV)
    with torch.no_grad():
        kernels.apply_multi_axis_rope(q, k, pos, inv, axes)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qo, _ = kernels.apply_multi_axis_rope(q, k, pos, inv, axes)
        pos.copy_(torch.randint(0, 1000, pos.shape, device=DEV))
        g.replay()
        assert torch.equal(qo, kernels.apply_multi_axis_rope(q, k, pos, inv, axes)[0])
        e = kernels.apply_multi_axis_rope(q[:, :, :0], k[:, :, :0], pos[..., :0], inv, axes)
        assert e[0].shape == (b, h, 0, d) and e[1].shape == (b, hk, 0, d)


# ------------------------------------------------------- AdamW over many tensors ----
def _optim():
    from auspex_soup_demo_b200 import optim

    return optim


SIZES = {
    "one": [(1,)],
    "odd": [(7,), (256,), (257,), (3, 5, 11), (2048,), (2049,), (1, 1), (4097,)],
    "rows": [(513,)] * 70,
    "large": [(1000, 1003), (64, 64)],
    "many": [(33,)] * 1500,
}


def _params(shapes, dtype, seed, offset=0):
    """Separate tensors; with offset, views that start that many elements into a buffer."""
    g = _gen(seed)
    out = []
    for s in shapes:
        n = math.prod(s)
        t = (0.05 * _randn(g, n + offset))[offset:].view(s) if not offset else \
            (0.05 * _randn(g, n + offset)).to(dtype)[offset:].view(s)
        out.append(torch.nn.Parameter(t.to(dtype) if not offset else t))
    return out


def _blocks(opt, i, n, name, scale=None):
    st = opt.state[opt.param_groups[0]["params"][i]]
    v = st[name].float()
    if scale:
        v = v * st[scale][:, None]
    return v.reshape(-1)[:n], st[name].float().reshape(-1)[n:], st.get(scale)


@pytest.mark.parametrize("kind", list(SIZES))
@pytest.mark.parametrize("dtype,bits", [(torch.float32, 8), (torch.float32, 32), (torch.bfloat16, 8),
                                        (torch.float16, 32)])
@pytest.mark.parametrize("clip", [None, 0.37])
def test_adamw_multi_against_64_bits(kind, dtype, bits, clip):
    """Three steps, each against 64 bits from the states that were held before it."""
    lr, betas, eps, wd = 3e-3, (0.9, 0.99), 1e-8, 0.1
    params = _params(SIZES[kind], dtype, 5, offset=1 if kind == "odd" else 0)
    opt = _optim().MultiTensorAdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=bits,
                                    max_grad_norm=clip)
    h = ref.half_step(dtype)
    e = 2.0 ** -24
    for step in (1, 2, 3):
        g = _gen(40 + step)
        for p in params:
            p.grad = (_randn(g, *p.shape) * 10.0 ** (2 * torch.rand(1, generator=g, device=DEV) - 2)).to(dtype)
        norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
        coef = 1.0 if clip is None else min(1.0, clip / (norm + 1e-6))
        old = []
        picks = range(len(params)) if len(params) < 80 else list(range(0, len(params), 97)) + [len(params) - 1]
        for i in picks:
            n = params[i].numel()
            m, _, _ = _blocks(opt, i, n, "exp_avg", "exp_avg_scale" if bits == 8 else None)
            v, _, _ = _blocks(opt, i, n, "exp_avg_sq", "exp_avg_sq_scale" if bits == 8 else None)
            v = v.double().square() if bits == 8 else v
            old.append((params[i].detach().clone().view(-1), m.clone(), v.clone()))
        opt.step()
        if clip is not None:
            assert abs(float(opt.grad_norm) - norm) <= 1e-6 * norm
        for i, (p0, m0, v0) in zip(picks, old):
            p, n = params[i], params[i].numel()
            want, m, v, upd = ref.adamw(p0, p.grad.view(-1), m0, v0, step, lr, betas, eps, wd, coef)
            # a dozen roundings of 2^-24 on the update, two on the rest, then p's own
            # (m's terms may cancel, so they count in full)
            top_m = m0.double().abs() + p.grad.view(-1).double().abs()
            rel = lr / (1 - betas[0] ** step) / (torch.sqrt(v / (1 - betas[1] ** step)) + eps)
            err = 12 * e * upd.abs() + 6 * e * rel * top_m + 4 * e * p0.double().abs()
            # fp16's subnormals: half of its smallest number
            tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
            ref.check("param", p.detach().view(-1), (want, h * want.abs() + (1 + h) * err + tiny))
            gm, pad_m, sm = _blocks(opt, i, n, "exp_avg", "exp_avg_scale" if bits == 8 else None)
            gv, pad_v, sv = _blocks(opt, i, n, "exp_avg_sq", "exp_avg_sq_scale" if bits == 8 else None)
            assert not pad_m.any() and not pad_v.any()
            if bits == 32:
                ref.check("m", gm, (m, 4 * e * top_m))
                ref.check("v", gv, (v, 8 * e * v))
            else:
                # half a step of 2^-4, or half of (a root: all of) the smallest code
                nb = sm.numel()
                for got, val, s, least, slack in ((gm, m, sm, 2.0 ** -10, 4 * e * top_m),
                                                  (gv, torch.sqrt(v), sv, 2.0 ** -9, 8 * e * torch.sqrt(v))):
                    sc = s.double().repeat_interleave(256)[:n]
                    ref.check("state", got, (val, (2.0 ** -4 + 4 * e) * val.abs() + least * sc + slack))
                    pad = torch.zeros(nb * 256, dtype=torch.float64, device=DEV)
                    pad[:n] = val.abs()
                    top = pad.view(nb, 256).amax(1)
                    ref.check("scale", s, (top / 448, 16 * e * top + float(top.max() > 0) * 1e-30
                                           + 6 * e * float(top_m.max()) / 448))
                assert ((gv > 0) | (v == 0)).all()
    assert float(opt.flat_state()["step"]) == 3.0


def test_adamw_multi_is_torch_adamw_with_32_bit_states():
    """Against torch's own, 20 steps: every step adds at most a few 2^-24 of p and of its update."""
    a, b = _params(SIZES["odd"], torch.float32, 6), _params(SIZES["odd"], torch.float32, 6)
    kw = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.05)
    x, y = _optim().MultiTensorAdamW(a, state_bits=32, **kw), torch.optim.AdamW(b, **kw)
    g = _gen(7)
    for _ in range(20):
        for p, q in zip(a, b):
            p.grad = _randn(g, *p.shape)
            q.grad = p.grad.clone()
        x.step()
        y.step()
    for p, q in zip(a, b):
        p, q = p.detach(), q.detach()
        assert float((p - q).abs().max()) <= 20 * 16 * 2.0 ** -24 * (float(q.abs().max()) + 1e-2)


def test_adamw_multi_groups_missing_gradients_and_layouts():
    ps = _params([(40, 30), (500,), (64, 2), (300,)], torch.float32, 8)
    half = _params([(100,)], torch.bfloat16, 9)
    opt = _optim().MultiTensorAdamW([{"params": ps[:2], "lr": 1e-3}, {"params": ps[2:] + half, "lr": 0.0}],
                                    weight_decay=0.0, state_bits=8, max_grad_norm=1e9)
    before = [p.detach().clone() for p in ps + half]
    ps[0].grad = torch.ones(30, 40, device=DEV).t()  # not contiguous
    ps[2].grad = torch.ones_like(ps[2])
    half[0].grad = torch.ones_like(half[0])
    opt.step()
    assert torch.equal(ps[1], before[1]) and torch.equal(ps[3], before[3])  # no gradient
    assert torch.equal(ps[2], before[2]) and torch.equal(half[0], before[4])  # lr 0
    # the first step of equal gradients is lr everywhere (up to eps 1e-8 and a rounding of 0.2 and of lr)
    assert float((before[0] - ps[0] - 1e-3).abs().max()) <= 1e-3 * (1e-7 + 16 * 2.0 ** -24) + 2.0 ** -25
    assert abs(float(opt.grad_norm) - math.sqrt(1200 + 128 + 100)) <= 1e-5
    assert not opt.state[ps[1]]["exp_avg"].float().any()
    opt.zero_grad()
    opt.step()  # nothing to do
    assert float(opt.flat_state()["step"]) == 1.0


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_multi_not_finite_gradient_reaches_its_own_element(bits):
    (p,) = _params([(600,)], torch.float32, 10)
    opt = _optim().MultiTensorAdamW([p], lr=1e-3, state_bits=bits)
    p.grad = torch.ones_like(p)
    p.grad[300] = math.inf
    p.grad[301] = math.nan
    opt.step()
    p.grad = torch.ones_like(p)
    opt.step()
    bad = torch.zeros(600, dtype=torch.bool, device=DEV)
    bad[300:302] = True
    assert torch.isfinite(p[~bad]).all() and not torch.isfinite(p[bad]).any()
    for name in ("m", "v"):
        assert torch.isfinite(opt.flat_state()[name].float().view(-1)[:600][~bad]).all()


def test_adamw_multi_zero_gradients_and_zero_states():
    (p,) = _params([(300,)], torch.float32, 11)
    before = p.detach().clone()
    opt = _optim().MultiTensorAdamW([p], lr=1e-3, state_bits=8, weight_decay=0.0, max_grad_norm=1.0)
    p.grad = torch.zeros_like(p)
    opt.step()
    assert torch.equal(p, before) and float(opt.grad_norm) == 0.0


def test_adamw_multi_tiny_second_moments_beside_large_ones():
    """Gradients over 12 decades in one block: no element moves by more than a few lr."""
    (p,) = _params([(256,)], torch.float32, 12)
    opt = _optim().MultiTensorAdamW([p], lr=1e-3, state_bits=8)
    g = 10.0 ** torch.linspace(-12, 0, 256, device=DEV)
    last = p.detach().clone()
    for _ in range(5):
        p.grad = g.clone()
        opt.step()
        # m <= 1.07 g (1 - b1^t) and sqrt(v) >= 0.93 g sqrt(1 - b2^t), or v's floor, which is above
        assert float((p.detach() - last).abs().max()) <= 1.3e-3
        last = p.detach().clone()


def test_adamw_multi_in_a_graph():
    ps = _params(SIZES["odd"], torch.float32, 13)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    kw = dict(lr=1e-3, state_bits=8, max_grad_norm=0.5, weight_decay=0.01)
    a, b = _optim().MultiTensorAdamW(ps, **kw), _optim().MultiTensorAdamW(qs, **kw)
    grads = [torch.randn_like(p) for p in ps]
    for p, q, g in zip(ps, qs, grads):
        p.grad, q.grad = g, g.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        b.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    assert float(a.flat_state()["step"]) == 4.0


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_multi_state_dict(bits):
    def make(seed):
        ps = _params(SIZES["odd"], torch.float32, seed)
        return ps, _optim().MultiTensorAdamW(ps, lr=1e-3, state_bits=bits)

    def step(ps, opt, seed):
        g = _gen(seed)
        for p in ps:
            p.grad = _randn(g, *p.shape)
        opt.step()

    ps, a = make(14)
    step(ps, a, 1)
    qs, b = make(15)
    b.load_state_dict(a.state_dict())
    with torch.no_grad():
        for p, q in zip(ps, qs):
            q.copy_(p)
    step(ps, a, 2)
    step(qs, b, 2)
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    with pytest.raises(ValueError, match="bits"):
        _optim().MultiTensorAdamW(_params(SIZES["odd"], torch.float32, 1), state_bits=40 - bits
                                  ).load_state_dict(a.state_dict())
    with pytest.raises(ValueError, match="sizes"):
        _optim().MultiTensorAdamW(_params(SIZES["one"], torch.float32, 1), state_bits=bits
                                  ).load_state_dict(a.state_dict())
