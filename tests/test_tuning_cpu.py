"""CPU checks of the preference / policy tuning operators: what they refuse, before
any kernel runs, and the key tile lists of the window attention kernels."""

import math

import pytest
import torch

from auspex_soup_demo_b200 import _lib, kernels


def _cpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


LAB = torch.zeros(4, 6, dtype=torch.int64)


@pytest.mark.parametrize("call,error", [
    # CPU tensors
    (lambda: kernels.preference_loss(_cpu(4, 6), None, LAB), ValueError),
    (lambda: kernels.policy_loss(_cpu(4, 6), _cpu(4), LAB), ValueError),
    (lambda: kernels.head_token_logps(_cpu(4, 8), _cpu(9, 8), LAB[0, :4]), ValueError),
    (lambda: kernels.swiglu_8bit(_cpu(4, 8), _cpu(4, 8)), ValueError),
    (lambda: kernels.window_attention(*[_cpu(1, 1, 4, 128, dtype=torch.bfloat16)] * 3, 1.0, 2), ValueError),
    # shapes
    (lambda: kernels.preference_loss(_cpu(4), None, LAB[0, :4]), ValueError),
    (lambda: kernels.preference_loss(_cpu(4, 0), None, LAB[:, :0]), ValueError),
    (lambda: kernels.preference_loss(_cpu(4, 5), None, LAB), ValueError),
    (lambda: kernels.policy_loss(_cpu(0, 6), _cpu(0), LAB[:0]), ValueError),
    (lambda: kernels.head_token_logps(_cpu(4, 8), _cpu(9, 16), LAB[0, :4]), ValueError),
    (lambda: kernels.head_token_logps(_cpu(4, 8), _cpu(9, 8), LAB[0, :3]), ValueError),
    (lambda: kernels.head_token_logps(_cpu(4, 8), object(), LAB[0, :4]), ValueError),
    (lambda: kernels.swiglu_8bit(_cpu(4, 8), _cpu(4, 7)), ValueError),
    (lambda: kernels.swiglu_8bit(_cpu(4, 0), _cpu(4, 0)), ValueError),
    (lambda: kernels.window_attention(_cpu(4, 128), _cpu(4, 128), _cpu(4, 128), 1.0, 2), ValueError),
    # types
    (lambda: kernels.preference_loss(_cpu(4, 6, dtype=torch.float64), None, LAB), TypeError),
    (lambda: kernels.preference_loss(_cpu(4, 6), None, _cpu(4, 6)), TypeError),
    (lambda: kernels.policy_loss(_cpu(4, 6, dtype=torch.bfloat16), _cpu(4), LAB), TypeError),
    (lambda: kernels.policy_loss(_cpu(4, 6), _cpu(4), LAB.bool()), TypeError),
    (lambda: kernels.head_token_logps(_cpu(4, 8), _cpu(9, 8), _cpu(4)), TypeError),
    (lambda: kernels.head_token_logps(_cpu(4, 8, dtype=torch.float64), _cpu(9, 8), LAB[0, :4]), TypeError),
    (lambda: kernels.swiglu_8bit(_cpu(4, 8), _cpu(4, 8, dtype=torch.float16)), TypeError),
    (lambda: kernels.swiglu_8bit(*[_cpu(4, 8, dtype=torch.int32)] * 2), TypeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


class _Cuda:
    """Stands for a CUDA tensor where only the argument checks look at it."""

    def __init__(self, t):
        self.t = t
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.mark.parametrize("kw", [
    dict(beta=0.0), dict(beta=-1.0), dict(beta=math.nan), dict(beta=math.inf), dict(label_smoothing=0.5),
    dict(label_smoothing=-0.1), dict(loss_type="hinge", label_smoothing=0.1), dict(loss_type="other"),
    dict(ref=_cpu(4, 5)), dict(ref=_cpu(3)), dict(ref=_cpu(4, 6).requires_grad_(True)),
])
def test_preference_options(kw):
    kw = dict(kw)
    ref = kw.pop("ref", None)
    with pytest.raises(ValueError):
        kernels.preference_loss(_Cuda(_cpu(4, 6)), ref, LAB, **kw)


def test_preference_odd_rows():
    with pytest.raises(ValueError, match="as many chosen as rejected"):
        kernels.preference_loss(_Cuda(_cpu(3, 6)), None, LAB[:3])


@pytest.mark.parametrize("kw", [
    dict(clip_low=1.0), dict(clip_low=-0.1), dict(clip_high=-0.1), dict(clip_high=math.inf),
    dict(clip_high=math.nan), dict(kl_coef=0.1), dict(kl_coef=-1.0, ref_logps=_cpu(4, 6)),
    dict(reduction="mean"), dict(old_logps=_cpu(4, 5)), dict(ref_logps=_cpu(4)), dict(adv=_cpu(6)),
    dict(old_logps=_cpu(4, 6).requires_grad_(True)),
])
def test_policy_options(kw):
    kw = dict(kw)
    adv = kw.pop("adv", _cpu(4))
    with pytest.raises(ValueError):
        kernels.policy_loss(_Cuda(_cpu(4, 6)), adv, LAB, **kw)


@pytest.mark.parametrize("scale,window,sinks", [(0.0, 4, 0), (math.nan, 4, 0), (math.inf, 4, 0),
                                                (1.0, 0, 0), (1.0, -3, 0), (1.0, 4, -1)])
def test_window_options(scale, window, sinks):
    t = _Cuda(_cpu(1, 2, 4, 128, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        kernels.window_attention(t, t, t, scale, window, sinks)


def test_window_head_dim_and_groups():
    t = _Cuda(_cpu(1, 2, 4, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="head dim"):
        kernels.window_attention(t, t, t, 1.0, 4)
    q, k = (_Cuda(_cpu(1, h, 4, 128, dtype=torch.bfloat16)) for h in (3, 2))
    with pytest.raises(ValueError, match="multiple"):
        kernels.window_attention(q, k, k, 1.0, 4)


def test_entry_points_refuse_bad_arguments():
    lib = _lib.lib()
    p, st = 256, _lib.i64_array([128, 128, 128])  # a pointer that no check follows
    bad = _lib.SOUP_ERR_INVALID
    assert lib.soup_attention_window_fwd(p, st, p, st, p, st, 1, 1, 1, 4, 128, 1.0, 0, 0, p, p, 0) == bad
    assert lib.soup_attention_window_bwd(p, st, p, st, p, st, p, p, p, 1, 1, 1, 4, 128, 1.0, 3, -1, p, p, p,
                                         p, 1 << 20, 0) == bad
    assert lib.soup_attention_window_fwd(p, st, p, st, p, st, 1, 1, 1, 4, 64, 1.0, 3, 0, p, p,
                                         0) == _lib.SOUP_ERR_UNSUPPORTED
    assert b"soup_attention_window_fwd" in lib.soup_last_error()
    f = lib.soup_preference_loss_fwd
    ok = [p, 6, p, 6, 1, p, 6, 2, 6, -100, 0.1, 0.0, 0, p, p, p, p, 1 << 20, 0]
    for i, v in ((0, 0), (1, 5), (2, 0), (3, 5), (4, 3), (6, 5), (7, 0), (8, 0), (10, 0.0), (11, 0.5),
                 (12, 3), (13, 0), (16, 0)):
        a = list(ok)
        a[i] = v
        assert f(*a) == bad, i
    a = list(ok)
    a[17] = 16
    assert f(*a) == _lib.SOUP_ERR_WORKSPACE
    f = lib.soup_policy_loss_fwd
    ok = [p, 6, p, 6, p, 6, p, 0, p, 6, 2, 6, -100, 0.2, 0.2, 0.1, 0, p, p, p, p, p, p, 1 << 20, 0]
    for i, v in ((0, 0), (1, 5), (3, 5), (5, 5), (6, 0), (7, 3), (9, 5), (10, 0), (11, 0), (13, 1.0),
                 (14, -1.0), (15, -1.0), (16, 2), (17, 0), (20, 0), (22, 0)):
        a = list(ok)
        a[i] = v
        assert f(*a) == bad, i
    assert lib.soup_preference_loss_bwd(0, p, p, 6, 2, 6, -100, p, 0) == bad
    assert lib.soup_policy_loss_bwd(p, p, 0, 2, 6, p, 0) == bad
    assert lib.soup_head_logps_fwd(0, 8, p, 8, 2, p, 4, 9, 8, -100, p, p, 0, 0, p, 1 << 20, 0) == bad
    assert lib.soup_head_logps_fwd(p, 8, p, 8, 0, p, 4, 9, 8, -100, p, p, 0, 0, p, 1 << 20, 0) == bad
    assert lib.soup_head_logps_bwd(p, 1 << 20, p, 8, 2, 0, 8, p, 4, 9, 8, p, 2, 0, 2, 0, p, 1 << 20,
                                   0) == bad
    assert lib.soup_swiglu_q8_fwd(p, 8, p, 8, p, 8, p, p, 7, p, p, 1, 4, 8, 2, 0) == bad
    assert lib.soup_swiglu_q8_fwd(p, 65, p, 65, p, 65, p, p, 65, p, p, 1, 4, 65, 2, 0) == bad
    assert lib.soup_swiglu_q8_bwd(p, 8, p, p, 8, p, p, 1, p, 8, p, 8, p, 7, 4, 8, 2, 0) == bad
    assert lib.soup_q8_quantize(p, 8, p, 8, p, 1, 4, 8, 9, 0) == bad


def test_workspace_sizes():
    lib = _lib.lib()
    assert lib.soup_preference_loss_workspace_bytes(0, 5) == 0
    assert lib.soup_policy_loss_workspace_bytes(3, 4097) > lib.soup_policy_loss_workspace_bytes(3, 4096)
    assert lib.soup_head_logps_state_bytes(10, 0, 8) == 0


# ---- the key blocks of a window (the kernels' index arithmetic, 64-key blocks) -------
def _blocks(qt, S, window, sinks):
    first = qt * 128 - window + 1
    lo = first // 64 if first > 0 else 0
    n_sink = min(-(-sinks // 64), lo)
    return n_sink, lo, n_sink + min(2 * qt + 2, -(-S // 64)) - lo


@pytest.mark.parametrize("S", [1, 127, 128, 129, 300, 640, 1000])
@pytest.mark.parametrize("window", [1, 2, 64, 127, 128, 129, 130, 300, 5000])
@pytest.mark.parametrize("sinks", [0, 1, 127, 128, 129, 400, 5000])
def test_window_block_lists_cover_every_visible_key(S, window, sinks):
    window, sinks = min(window, S), min(sinks, S)
    nq, nq64 = -(-S // 128), -(-S // 64)

    def needed(qt):
        blocks = set()
        for q in range(qt * 128, min(S, qt * 128 + 128)):
            blocks |= set(range(max(0, q - window + 1) // 64, q // 64 + 1))
            blocks |= set(range(0, -(-min(sinks, q + 1) // 64)))
        return blocks

    for qt in range(nq):  # one query tile (forward and dQ)
        n_sink, lo, n = _blocks(qt, S, window, sinks)
        blocks = [i if i < n_sink else lo + i - n_sink for i in range(n)]
        assert len(set(blocks)) == n >= 1 and all(0 <= i < nq64 for i in blocks)
        assert needed(qt) <= set(blocks)
    for kt in range(nq):  # the 128-query steps of a key tile (dK / dV)
        first, n = kt, nq - kt
        if kt * 128 >= sinks:
            n = min((kt * 128 + 127 + window - 1) // 128, nq - 1) - first + 1
        assert n >= 1 and first + n <= nq
        for key in range(kt * 128, min(S, kt * 128 + 128)):
            last = S - 1 if key < sinks else min(S - 1, key + window - 1)
            assert first <= key // 128 and last // 128 < first + n


class _Layer(torch.nn.Module):
    """What soup_attention reads of a transformers attention layer."""

    def __init__(self, groups, sinks=0):
        super().__init__()
        self.is_causal, self.num_key_value_groups = True, groups
        self.config = type("Config", (), {"attention_sink_tokens": sinks})()


@pytest.mark.parametrize("n_q,n_k,window,sinks", [
    (13, 13, 4, 0), (13, 13, 4, 2), (13, 13, 1, 0), (13, 13, 40, 3), (3, 13, 4, 0), (1, 13, 4, 0),
    (1, 4, 4, 0), (5, 8, 4, 0), (1, 1, 1, 0),
])
def test_sliding_layer_off_the_kernels(n_q, n_k, window, sinks):
    """Prefill, chunks and single tokens against a cache; fp64, so only the sums' order differs."""
    from auspex_soup_demo_b200.kernels.attention import soup_attention

    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(2, h, n, 16, generator=g, dtype=torch.float64)
               for h, n in ((4, n_q), (2, n_k), (2, n_k)))
    out, _ = soup_attention(_Layer(2, sinks), q, k, v, None, scaling=0.3, sliding_window=window)
    ref = torch.empty(2, n_q, 4, 16, dtype=torch.float64)
    for h in range(4):
        for i in range(n_q):
            pos = n_k - n_q + i
            see = [j for j in range(pos + 1) if pos - j < window or j < sinks]
            p = torch.softmax(0.3 * (k[:, h // 2, see] @ q[:, h, i, :, None])[..., 0], -1)
            ref[:, i, h] = (p[:, None] @ v[:, h // 2, see])[:, 0]
    assert (out - ref).abs().max() <= 1e-13 * v.abs().max()


@pytest.mark.parametrize("n_q,n_k", [(1, 4), (1, 13), (5, 8)])
def test_sliding_layer_refuses_sinks_beyond_a_cache(n_q, n_k):
    from auspex_soup_demo_b200.kernels.attention import soup_attention

    q, k = torch.zeros(1, 2, n_q, 16), torch.zeros(1, 2, n_k, 16)
    with pytest.raises(ValueError, match="attention_sink_tokens"):
        soup_attention(_Layer(1, 2), q, k, k, None, sliding_window=4)
