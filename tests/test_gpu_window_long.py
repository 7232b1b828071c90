"""Window attention over a long sequence: many key blocks a query tile and many steps a key
tile, against a plain 64-bit form, and the same bits on every repeat."""

import math

import pytest
import torch

from auspex_soup_demo_b200 import _lib, kernels

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _blocked64(q, k, v, do, scale, window, sinks):
    """Values and error bounds of (out, dq, dk, dv), query blocks of 1024 against the keys
    that they see. The kernel rounds P, dS and its results to bf16, half a step (2^-8) of
    each, and takes D = rowsum(dO O) from the rounded O; its other arithmetic is fp32
    with exponentials good to 2^-13 (the cubic's 7.5e-5), well below."""
    q, k, v, g = (t.detach().double() for t in (q, k, v, do.transpose(1, 2)))
    B, H, S, D = q.shape
    rep = H // k.shape[1]
    u = 2.0 ** -8 * 1.03
    val = [torch.zeros_like(t) for t in (q, q, k, k)]
    tol = [torch.zeros_like(t) for t in (q, q, k, k)]

    def grouped(t):
        return t.view(B, H // rep, rep, *t.shape[2:]).sum(2)

    for lo in range(0, S, 1024):
        hi = min(S, lo + 1024)
        first = max(0, lo - window + 1)
        cols = torch.cat([torch.arange(min(sinks, first), device=DEV), torch.arange(first, hi, device=DEV)])
        dist = torch.arange(lo, hi, device=DEV)[:, None] - cols
        seen = (dist >= 0) & ((dist < window) | (cols < sinks))
        kk, vv = (t[:, :, cols].repeat_interleave(rep, 1) for t in (k, v))
        qb, gb = q[:, :, lo:hi], g[:, :, lo:hi]
        p = torch.softmax((qb @ kk.transpose(2, 3) * scale).masked_fill(~seen, -math.inf), -1)
        o = p @ vv
        dp = gb @ vv.transpose(2, 3)
        dsum = (gb * o).sum(-1, keepdim=True)
        ds = p * (dp - dsum)
        e_ds = u * (ds.abs() + p * ((gb.abs() * o.abs()).sum(-1, keepdim=True)
                                    + dp.abs() * 2.0 ** -6 + dsum.abs() * 2.0 ** -6))
        val[0][:, :, lo:hi], tol[0][:, :, lo:hi] = o, u * (p @ vv.abs() + o.abs())
        val[1][:, :, lo:hi], tol[1][:, :, lo:hi] = ds @ kk * scale, e_ds @ kk.abs() * scale
        val[2].index_add_(2, cols, grouped(ds.transpose(2, 3) @ qb * scale))
        tol[2].index_add_(2, cols, grouped(e_ds.transpose(2, 3) @ qb.abs() * scale))
        val[3].index_add_(2, cols, grouped(p.transpose(2, 3) @ gb))
        tol[3].index_add_(2, cols, grouped(u * p.transpose(2, 3) @ gb.abs()))
    for i in (1, 2, 3):
        tol[i] += u * val[i].abs()
    val[0], tol[0] = val[0].transpose(1, 2), tol[0].transpose(1, 2)
    return val, tol


@pytest.mark.parametrize("B,H,Hk,S,window,sinks", [
    (1, 6, 2, 16001, 1000, 16),  # a long document, its window ending inside a tile
    (1, 2, 1, 9000, 129, 300),   # sinks over three tiles, each seen by all later queries
    (2, 2, 2, 4097, 4000, 1),    # nearly causal: 64 blocks a query tile, 32 steps a key tile
])
def test_long_window(B, H, Hk, S, window, sinks):
    g = torch.Generator(device=DEV).manual_seed(S)
    q, k, v = (torch.randn(B, S, h, 128, generator=g, device=DEV).bfloat16().transpose(1, 2)
               .requires_grad_(True) for h in (H, Hk, Hk))
    do = torch.randn(B, S, H, 128, generator=g, device=DEV).bfloat16()

    def run():
        out = kernels.window_attention(q, k, v, 128 ** -0.5, window, sinks)
        return [out.detach()] + list(torch.autograd.grad(out, [q, k, v], do))

    got = run()
    torch.cuda.synchronize()
    assert _lib.device_error(torch.device(DEV)) == 0
    val, tol = _blocked64(q, k, v, do, 128 ** -0.5, window, sinks)
    for name, a, b, t in zip(("out", "dq", "dk", "dv"), got, val, tol):
        # 2^-14 of the largest: fp32 accumulation over thousands of terms
        assert bool(((a.double() - b).abs() <= t + 2.0 ** -14 * float(b.abs().max())).all()), name
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(run(), got))
    torch.cuda.synchronize()
    assert _lib.device_error(torch.device(DEV)) == 0


@pytest.mark.parametrize("B,H,Hk,S,window,sinks", [
    (1, 4, 2, 6000, 128, 3000),  # sink tiles in long segments
    (1, 2, 1, 5000, 1, 4990),    # nearly all keys are sinks
    (3, 6, 3, 2100, 70, 1000),
    (1, 8, 1, 3000, 200, 900),   # heads split over CTAs beside the segments
])
def test_many_sinks(B, H, Hk, S, window, sinks):
    test_long_window(B, H, Hk, S, window, sinks)
