"""Calls at the edge of what the operators take, as far as they can be checked without a
GPU: what is refused, and which pointers, strides and masks reach the kernels."""

import pytest
import torch

from auspex_soup_demo_b200 import _lib, kernels


# ------------------------------------------------------------- host tensors ----
@pytest.mark.parametrize("call", [
    lambda t: _lib.stream_of(t),
    lambda t: kernels.fast_swiglu(t, t),
    lambda t: kernels.fast_rms_norm(t, t[0], 1e-6),
], ids=["stream_of", "fast_swiglu", "fast_rms_norm"])
def test_host_tensors_are_refused_before_a_launch(call):
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        call(torch.zeros(4, 8))


@pytest.mark.parametrize("x,error", [
    (torch.zeros(4, 8), ValueError), (torch.zeros(()), ValueError), (torch.zeros(4, 0), ValueError),
    (torch.zeros(4, 8, dtype=torch.int32), TypeError), (torch.zeros(4, 8, dtype=torch.float64), TypeError),
])
def test_quantize_8bit_refusals(x, error):
    with pytest.raises(error, match="quantize_8bit|unsupported dtype"):
        kernels.quantize_8bit(x)


# ------------------------------------------------- saved tensors in other layouts ----
def _relaid(t, layout):
    """The values of t as a saved-tensor hook may hand them back."""
    if layout == "contiguous":  # torch.autograd.graph.save_on_cpu
        return t.detach().clone(memory_format=torch.contiguous_format)
    if layout == "gaps" and t.dim() == 1:
        wide = t.new_empty(2 * t.numel())[::2]
        return wide.copy_(t.detach())
    if layout == "gaps":
        wide = t.new_empty(*t.shape[:-1], t.shape[-1] + 64)
        wide[..., :t.shape[-1]] = t.detach()
        return wide[..., :t.shape[-1]]
    flat = t.new_empty(t.numel() + 1)  # one element off
    flat[1:] = t.detach().reshape(-1)
    return flat[1:].view(t.shape)


class _Calls:
    """Records the library calls of host tensors instead of making them, and hands saved
    tensors back in another layout."""

    def __init__(self, monkeypatch, layout):
        self.calls, self.back, self.layout = {}, [], layout
        monkeypatch.setattr(_lib, "call", lambda fn, dev, *args: self.calls.__setitem__(fn, args))
        monkeypatch.setattr(_lib, "stream_of", lambda t: 0)

    def hooks(self):
        def unpack(t):
            self.back.append(_relaid(t, self.layout))
            return self.back[-1]

        return torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack)


LAYOUTS = ["contiguous", "gaps", "odd"]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("source", ["transposed", "fused projection"])
def test_window_backward_reads_what_came_back(monkeypatch, layout, source):
    from auspex_soup_demo_b200.kernels import attention

    rec = _Calls(monkeypatch, layout)
    monkeypatch.setattr(attention, "_window_workspace_bytes", lambda *sizes: 256)
    B, H, Hk, S, D = 2, 4, 2, 200, 128
    if source == "transposed":
        q, k, v = (torch.randn(B, S, h, D).bfloat16().transpose(1, 2) for h in (H, Hk, Hk))
    else:
        big = torch.randn(B, S, (H + 2 * Hk) * D).bfloat16()
        q, k, v = (big[..., a * D:(a + h) * D].view(B, S, h, D).transpose(1, 2)
                   for a, h in ((0, H), (H, Hk), (H + Hk, Hk)))
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    with rec.hooks():
        out = attention.WindowAttentionFunction.apply(q, k, v, 0.1, 50, 4)
    out.backward(torch.zeros_like(out))
    fwd, bwd = rec.calls["soup_attention_window_fwd"], rec.calls["soup_attention_window_bwd"]
    for i, t in enumerate((q, k, v)):
        assert fwd[2 * i] == t.data_ptr() and list(fwd[2 * i + 1]) == list(t.stride()[:3])
        got = rec.back[i]
        strides = list(bwd[2 * i + 1])
        if layout == "odd":  # not readable in place
            assert bwd[2 * i] != got.data_ptr() and bwd[2 * i] % 16 == 0
            assert strides == [t.shape[1] * S * D, S * D, D]
        else:
            assert bwd[2 * i] == got.data_ptr() and strides == list(got.stride()[:3])
    for i, got in ((6, rec.back[3]), (8, rec.back[4])):  # out, log-sum-exp: contiguous
        assert bwd[i] % 16 == 0 and (bwd[i] == got.data_ptr()) == (layout == "contiguous")


@pytest.mark.parametrize("S", [128, 200])
def test_causal_backward_under_hooks(monkeypatch, S):
    """The log-sum-exp's padded buffer comes back, whatever the length."""
    from auspex_soup_demo_b200.kernels import attention

    rec = _Calls(monkeypatch, "contiguous")
    monkeypatch.setattr(_lib, "scratch", lambda dev, n: torch.empty(max(n, 16), dtype=torch.uint8))
    monkeypatch.setattr(attention, "_check", lambda q, k, v: (*q.shape[:2], k.shape[1], *q.shape[2:]))
    q, k, v = (torch.randn(2, S, h, 128).bfloat16().transpose(1, 2).requires_grad_(True) for h in (4, 2, 2))
    with rec.hooks():
        out = attention.flash_attention(q, k, v, 0.1)
    out.backward(torch.zeros_like(out))
    bwd = rec.calls["soup_attention_bwd"]
    assert rec.back[4].shape == (2, 4, -(-S // 128) * 128) and bwd[8] == rec.back[4].data_ptr()
    for i in range(3):
        assert bwd[2 * i] == rec.back[i].data_ptr()
        assert list(bwd[2 * i + 1]) == list(rec.back[i].stride()[:3])


@pytest.mark.parametrize("layout", LAYOUTS)
def test_preference_backward_reads_what_came_back(monkeypatch, layout):
    rec = _Calls(monkeypatch, layout)
    x = torch.randn(4, 8).requires_grad_(True)
    labels = torch.arange(36).view(4, 9)[:, 1:]
    with rec.hooks():
        loss, _, _ = kernels.tuning_loss.PreferenceLossFunction.apply(x, None, labels, 0.1, 0.0, 0, -100)
    loss.backward(torch.ones(()))
    fwd, bwd = rec.calls["soup_preference_loss_fwd"], rec.calls["soup_preference_loss_bwd"]
    assert (fwd[5], fwd[6]) == (labels.data_ptr(), 9)
    ws, lab = rec.back
    # rows are read where they are (an int64 pointer is aligned to its element)
    assert (bwd[2], bwd[3]) == (lab.data_ptr(), {"contiguous": 8, "gaps": 8 + 64, "odd": 8}[layout])
    off = fwd[15] - fwd[16]  # the coefficients, behind the workspace
    assert (bwd[1] - off) % 16 == 0 and (bwd[1] == ws.data_ptr() + off) == (layout == "contiguous")


@pytest.mark.parametrize("layout", LAYOUTS)
def test_policy_backward_reads_what_came_back(monkeypatch, layout):
    rec = _Calls(monkeypatch, layout)
    x = torch.randn(4, 8).requires_grad_(True)
    with rec.hooks():
        loss, _, _ = kernels.tuning_loss.PolicyLossFunction.apply(
            x, torch.randn(4), torch.arange(36).view(4, 9)[:, 1:], None, None, 0.2, 0.2, 0.0, 0, -100, True)
    loss.backward(torch.ones(()))
    fwd, bwd = rec.calls["soup_policy_loss_fwd"], rec.calls["soup_policy_loss_bwd"]
    (ws,), off = rec.back, fwd[20] - fwd[22]
    assert bwd[2] - bwd[1] == fwd[21] - fwd[20] == 16
    assert (bwd[1] - off) % 16 == 0 and (bwd[1] == ws.data_ptr() + off) == (layout == "contiguous")


@pytest.mark.parametrize("layout", LAYOUTS)
def test_swiglu_8bit_backward_reads_what_came_back(monkeypatch, layout):
    from auspex_soup_demo_b200.kernels import swiglu

    rec = _Calls(monkeypatch, layout)
    g, u = (torch.randn(3, 70).requires_grad_(True) for _ in range(2))
    with rec.hooks():
        h = swiglu.SwiGLU8BitFunction.apply(g, u)
    h.backward(torch.zeros_like(h))
    fwd, bwd = rec.calls["soup_swiglu_q8_fwd"], rec.calls["soup_swiglu_q8_bwd"]
    codes, scales = (bwd[2], bwd[3]), (bwd[5], bwd[6])
    base = scales[0]
    assert base % 16 == 0 and (base == rec.back[0].data_ptr()) == (layout == "contiguous")
    assert [p - base for p in codes + scales] == [p - fwd[9] for p in fwd[6:8] + fwd[9:11]]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("blocks", [False, True])
def test_token_logps_backward_reads_what_came_back(monkeypatch, layout, blocks):
    from auspex_soup_demo_b200.kernels import chunked_ce, token_logps

    rec = _Calls(monkeypatch, layout)
    monkeypatch.setattr(token_logps, "_state_bytes", lambda n, v, d: 512 * n)
    monkeypatch.setattr(token_logps, "_workspace_bytes", lambda n, v, d, b: 512 * n)
    if blocks:
        monkeypatch.setattr(chunked_ce, "CE_WORKSPACE_BYTES", 1)
    hidden = torch.randn(300, 64).bfloat16().requires_grad_(True)
    weight = torch.randn(70, 64).bfloat16().requires_grad_(True)
    labels = torch.randint(0, 70, (300,))
    with rec.hooks():
        logps, _ = token_logps.HeadTokenLogpsFunction.apply(hidden, weight, labels, -100, True)
    rec.calls.clear()
    logps.backward(torch.zeros_like(logps))
    bwd = rec.calls["soup_head_logps_bwd"]
    back_w, back_t, *back = rec.back
    state, h = (None, back[0]) if blocks else back
    same = layout == "contiguous"
    inplace = layout != "odd"  # rows with gaps are read where they are
    last = 256 * 64 * 2 if blocks else 0  # the last block starts at row 256
    gap = 128 if layout == "gaps" else 64
    assert (bwd[2] - (last * gap // 64) == h.data_ptr()) == inplace and bwd[2] % 16 == 0
    assert bwd[3] == gap and bwd[6] == gap and (bwd[5] == back_w.data_ptr()) == inplace
    if blocks:
        again = rec.calls["soup_head_logps_fwd"]
        assert again[1] == again[3] == gap and (again[5] - 256 * 8 == back_t.data_ptr()) == same
    else:
        assert bwd[0] % 16 == 0 and (bwd[0] == state.data_ptr()) == same


# ------------------------------------------------------- attention against a cache ----
class _Layer(torch.nn.Module):
    """What soup_attention reads of a transformers attention layer."""

    def __init__(self, groups, sinks=0):
        super().__init__()
        self.is_causal, self.num_key_value_groups = True, groups
        self.config = type("Config", (), {"attention_sink_tokens": sinks})()


@pytest.mark.parametrize("n_q,n_k,window,sinks", [
    (4, 12, 12, 0), (4, 12, 64, 0), (4, 12, None, 0), (2, 3, None, 0), (11, 12, 12, 0), (4, 12, 13, 3),
    (4, 12, 11, 0), (1, 12, None, 0), (12, 12, None, 2), (12, 12, 12, 2),
])
@pytest.mark.parametrize("explicit", [False, True])
def test_chunk_against_a_cache(n_q, n_k, window, sinks, explicit):
    """The queries are the last tokens of the keys; fp64, so only the sums' order differs."""
    from auspex_soup_demo_b200.kernels.attention import soup_attention

    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(2, h, n, 16, generator=g, dtype=torch.float64)
               for h, n in ((4, n_q), (2, n_k), (2, n_k)))
    kw = {"is_causal": True} if explicit and n_q > 1 else {}
    out, _ = soup_attention(_Layer(2, sinks), q, k, v, None, scaling=0.3, sliding_window=window, **kw)
    for h in range(4):
        for i in range(n_q):
            pos = n_k - n_q + i
            see = [j for j in range(pos + 1) if window is None or pos - j < window or j < sinks]
            p = torch.softmax(0.3 * (k[:, h // 2, see] @ q[:, h, i, :, None])[..., 0], -1)
            want = (p[:, None] @ v[:, h // 2, see])[:, 0]
            assert (out[:, i, h] - want).abs().max() <= 1e-13 * v.abs().max()


def _tiny_model(impl, **over):
    from transformers import Qwen2Config, Qwen2ForCausalLM

    from auspex_soup_demo_b200.kernels import attention

    attention.register()
    torch.manual_seed(0)
    cfg = Qwen2Config(vocab_size=50, hidden_size=32, intermediate_size=64, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, attn_implementation=impl, **over)
    return Qwen2ForCausalLM(cfg).eval()


SLIDING = dict(use_sliding_window=True, sliding_window=4, max_window_layers=1)


@pytest.mark.parametrize("over", [{}, SLIDING, dict(SLIDING, sliding_window=30)],
                         ids=["full", "sliding", "wide window"])
def test_model_continues_a_cache_with_a_chunk(over):
    a = _tiny_model("soup_b200", **over)
    ids = torch.randint(0, 50, (2, 14), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        whole = a(ids).logits
        cache, parts = None, []
        for lo, hi in ((0, 5), (5, 11), (11, 12), (12, 14)):
            r = a(ids[:, lo:hi], past_key_values=cache, use_cache=True)
            cache = r.past_key_values
            parts.append(r.logits)
    # the same fp32 sums in another order; logits are below 1
    assert (torch.cat(parts, 1) - whole).abs().max() <= 1e-5


@pytest.mark.parametrize("n_q,n_k,window", [(1, 8192, 100), (3, 8192, None)])
def test_cached_attention_takes_memory_of_the_queries_alone(n_q, n_k, window):
    from torch.utils._python_dispatch import TorchDispatchMode

    from auspex_soup_demo_b200.kernels.attention import soup_attention

    class Largest(TorchDispatchMode):
        numel = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            for t in out if isinstance(out, (tuple, list)) else (out,):
                if isinstance(t, torch.Tensor):
                    self.numel = max(self.numel, t.untyped_storage().nbytes())
            return out

    q, k, v = (torch.randn(1, 2, n, 16) for n in (n_q, n_k, n_k))
    with Largest() as seen:
        out, _ = soup_attention(_Layer(1), q, k, v, None, sliding_window=window)
    assert out.shape == (1, n_q, 2, 16)
    assert 0 < seen.numel <= 4 * k.numel() * k.element_size()  # [n_k, n_k] would be 64 times that and more


# ------------------------------------------------------------- masks of a model ----
def _padded(kind):
    m = torch.ones(2, 12, dtype=torch.long)
    if kind == "left":
        m[0, :3] = 0
    elif kind == "right":
        m[0, 9:] = 0
    elif kind == "hole":
        m[1, 5:7] = 0
    return m


@pytest.mark.parametrize("kind", ["none", "left", "right", "hole"])
@pytest.mark.parametrize("over", [{}, SLIDING], ids=["full", "sliding"])
def test_padded_batch_as_with_sdpa(kind, over):
    ids = torch.randint(0, 50, (2, 12), generator=torch.Generator().manual_seed(2))
    mask = _padded(kind)
    a, b = (_tiny_model(impl, **over) for impl in ("soup_b200", "sdpa"))
    with torch.no_grad():
        x, y = (m(ids, attention_mask=mask).logits[mask.bool()] for m in (a, b))
    assert (x - y).abs().max() <= 1e-6  # the same fp32 sums, perhaps in another order


@pytest.mark.parametrize("over", [{}, SLIDING], ids=["full", "sliding"])
@pytest.mark.parametrize("static", [False, True])
def test_generation_from_a_padded_batch_as_with_sdpa(over, static):
    ids = torch.randint(0, 50, (2, 12), generator=torch.Generator().manual_seed(3))
    kw = dict(cache_implementation="static") if static else {}
    a, b = (_tiny_model(impl, **over).generate(ids, attention_mask=_padded("left"), max_new_tokens=5,
                                               do_sample=False, pad_token_id=0, output_scores=True,
                                               return_dict_in_generate=True, **kw)
            for impl in ("soup_b200", "sdpa"))
    assert torch.equal(a.sequences, b.sequences)
    assert max((x - y).abs().max() for x, y in zip(a.scores, b.scores)) <= 1e-5


def _mask(kind=None, q=12, k=12, offset=0, local=None, sinks=0, **kw):
    from auspex_soup_demo_b200.kernels.attention import soup_mask
    from transformers.masking_utils import causal_mask_function

    config = type("Config", (), {"sliding_window": 4, "attention_sink_tokens": sinks})()
    return soup_mask(batch_size=2, q_length=q, kv_length=k, q_offset=offset, kv_offset=0,
                     mask_function=causal_mask_function, attention_mask=kind and _padded(kind).bool(),
                     local_size=local, config=config, **kw)


@pytest.mark.parametrize("local", [None, 4])
def test_masks_that_the_kernels_need_not(local):
    """Whole sequences, also with padding behind them, stay on the kernels."""
    for kind in (None, "none", "right"):
        assert _mask(kind, local=local, sinks=3) is None
    for kind in ("left", "hole"):
        assert _mask(kind, local=local).shape == (2, 1, 12, 12)
    assert _mask(None, local=local, allow_is_causal_skip=False).shape[-2:] == (12, 12)
    assert _mask(None, 3, 12, 9, local=local).shape[-2:] == (3, 12)
    assert _mask(None, local=5).shape[-2:] == (12, 12)  # not this layer type's window: chunks


@pytest.mark.parametrize("call", [
    lambda: _mask("left", local=4, sinks=2),
    lambda: _mask(None, 1, 4, 11, local=4, sinks=2),
    lambda: _mask(None, 3, 12, torch.tensor(9), local=4, sinks=2, allow_is_causal_skip=False),
])
def test_sinks_refuse_masks_they_are_not_in(call):
    with pytest.raises(ValueError, match="attention_sink_tokens"):
        call()


# -------------------------------------------------- workspace of the window backward ----
@pytest.mark.parametrize("S,window,sinks", [(16384, 128, 16384), (16384, 128, 16256), (5000, 1, 5000),
                                            (5000, 2500, 2500), (700, 699, 1)])
def test_window_and_sinks_that_hide_nothing_take_no_more_than_the_causal_case(S, window, sinks):
    size = _lib.lib().soup_attention_window_bwd_workspace_bytes
    assert size(1, 32, 8, S, window, sinks) == size(1, 32, 8, S, S, 0) > 0


def _dkv_plan(B, H, Hk, S, window, sinks, sms=148):
    """The host's cut of the dK / dV work, restated."""
    nt, rep = -(-S // 128), H // Hk
    window, sinks = min(window, S), min(sinks, S)
    if window + sinks >= S:
        window, sinks = S, 0
    ns = -(-sinks // 128)
    tile_steps = min((128 + window - 2) // 128 + 1, nt)
    g = max(1, min(rep, -(-(sms * 4 // 5) // (B * Hk * nt))))
    heads_per = -(-rep // g)
    groups = -(-rep // heads_per)
    work = B * Hk * groups * (ns * nt - ns * (ns - 1) // 2 + (nt - ns) * tile_steps)
    seg_steps = max(4, min(nt, max(tile_steps, -(-work // (4 * sms)))))
    return nt, ns, groups, heads_per, seg_steps


# batch, heads, KV heads, length, window, sinks
CUTS = [(1, 32, 8, 16384, 128, 8192), (1, 12, 2, 16001, 1000, 16), (4, 12, 2, 2048, 512, 4),
        (2, 6, 3, 5000, 1, 4998), (1, 8, 1, 131072, 128, 65536), (1, 7, 1, 1000, 70, 129), (1, 1, 1, 1, 1, 0),
        (3, 4, 4, 4097, 700, 0), (2, 8, 2, 1300, 1300, 5)]


@pytest.mark.parametrize("sizes", CUTS)
def test_partial_slots_of_the_window_backward(sizes):
    """Every partial has a slot of its own inside the workspace; the sink tiles' segments cover
    their steps."""
    B, H, Hk, S, _, _ = sizes
    nt, ns, groups, heads_per, seg_steps = _dkv_plan(*sizes)
    before, used = 0, set()
    starts = []
    for kt in range(ns):
        n = nt - kt
        q, r = divmod(nt - kt, seg_steps)
        q0, r0 = divmod(nt, seg_steps)
        closed = (seg_steps * q0 * (q0 + 1) // 2 + r0 * (q0 + 1)) - (seg_steps * q * (q + 1) // 2 + r * (q + 1))
        assert closed == before  # the kernels' closed form of the segments of earlier tiles
        starts.append((before, -(-n // seg_steps)))
        before += -(-n // seg_steps)
    for bhk in range(B * Hk):
        for first, count in starts:
            for g in range(groups):
                for seg in range(count):
                    slot = (bhk * before + first) * groups + g * count + seg
                    assert slot not in used
                    used.add(slot)
    rest = B * Hk * (nt - ns) * groups if groups > 1 else 0
    assert used == set(range(B * Hk * before * groups))
    assert (groups - 1) * heads_per < H // Hk <= groups * heads_per
    vectors = 2 * (-(-B * H * nt * 128 * 4 // 256) * 256)
    got = _lib.lib().soup_attention_window_bwd_workspace_bytes(*sizes)
    assert got == vectors + (len(used) + rest) * 2 * 128 * 128 * 4


@pytest.mark.parametrize("sizes", CUTS)
def test_partials_stay_linear_in_the_sink_tiles(sizes):
    B, H, Hk, S, _, _ = sizes
    nt, ns, groups, _, _ = _dkv_plan(*sizes)
    partials = (_lib.lib().soup_attention_window_bwd_workspace_bytes(*sizes)
                - 2 * (-(-B * H * nt * 128 * 4 // 256) * 256)) // (2 * 128 * 128 * 4)
    # one slot a sink tile (and a tile, when few tiles split their heads), and four an SM
    assert partials <= B * Hk * groups * (nt if groups > 1 else ns) + 4 * 148


# -------------------------------------------------------------- 8-bit checkpoints ----
@pytest.mark.parametrize("keep8", [False, True])
def test_mlp_that_cannot_keep_8_bits_says_so(keep8):
    """A grouped MLP off the one-Function form (here: fp16 states) recomputes."""
    import warnings

    from auspex_soup_demo_b200 import qlora

    class Group:
        interleaved, outs = True, [8]

        def swiglu(self, x, recompute):
            return x * (2.0 if recompute else 3.0)

    x = torch.ones(2, 8, dtype=torch.float16)
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        y = qlora.LoRAProjectionGroup.mlp(Group(), x, lambda h: h, False, keep8)
    assert y[0, 0] == (2.0 if keep8 else 3.0)
    assert [w for w in seen if "CHECKPOINT_8BIT" in str(w.message)] != [] if keep8 else not seen


# ------------------------------------------------------- the exponential on the FMA pipe ----
def test_cubic_exponential_over_its_range():
    """The window backward's 2^x on the FMA pipe, restated in numpy with the source's
    constants: 7.5e-5 of the value for -126 <= x <= 127, never below 2^-126."""
    import os
    import re

    import numpy as np

    src = open(os.path.join(os.path.dirname(_lib.__file__), "csrc", "attention_window.cu")).read()
    body = src[src.index("void exp2_fma("):]
    body = body[:body.index("\n}")]
    c3, c2, c1, c0 = (float(x) for x in dict.fromkeys(re.findall(r"f2_pack\((0\.\d+)f", body)))
    f32 = np.float32
    x = np.concatenate([np.linspace(-126, 127, 400001), np.arange(-126, 128), np.arange(-126, 127) + 0.5,
                        [-1e30, -200.0, -126.5]]).astype(f32)
    lo = np.maximum(x, f32(-126))
    magic = f32(12582912 + 127)
    t = (lo + magic).astype(f32)
    f = (lo.astype(np.float64) - (t - magic).astype(f32)).astype(f32)  # exact: n is near x

    def fma(a, b, c):  # one rounding: the product of two fp32 values is exact in 64 bits
        return (a.astype(np.float64) * b.astype(np.float64) + np.float64(f32(c))).astype(f32)

    y = fma(f, np.full_like(f, c3), c2)
    y = fma(f, y, c1)
    y = fma(f, y, c0)
    scale = (t.view(np.uint32) << np.uint32(23)).view(f32)
    with np.errstate(over="ignore"):
        got = (y * scale).astype(np.float64)
    want = np.exp2(lo.astype(np.float64))
    assert np.abs(f).max() <= 0.5
    assert (np.abs(got / want - 1) <= 7.6e-5).all()
    assert (got >= 2.0 ** -126 * (1 - 7.6e-5)).all()


def test_window_mask_takes_a_byte_a_pair():
    """A whole sequence off the kernels: no [n, n] tensor of distances beside the mask."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from auspex_soup_demo_b200.kernels.attention import soup_attention

    wide = []

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            for t in out if isinstance(out, (tuple, list)) else (out,):
                if isinstance(t, torch.Tensor) and not t.is_floating_point() and t.numel() >= 500 * 500:
                    wide.append(t.element_size())
            return out

    q = torch.randn(1, 1, 500, 16)
    with Seen():
        soup_attention(_Layer(1), q, q, q, None, sliding_window=30)
    assert wide and max(wide) == 1
