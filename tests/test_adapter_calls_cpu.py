"""CPU: what the operators of a step with several adapters check of tensors that changed
between two calls, and calls of the model built of them (in plain torch)."""

import array
import copy
import ctypes
import io
import json
import threading

import pytest
import torch
from transformers import DynamicCache

import test_gpu_adapter_model as plain
from auspex_soup_demo_b200 import _lib, adapter, kernels, optim, qlora


# --------------------------------------------------- tensors of an optimiser's step ----
def _sizes(*n):
    return array.array("q", n)


def test_addresses_of_many_tensors():
    """The compiled table of addresses against each tensor's own answers."""
    cpu = torch.device("cpu")
    base = torch.zeros(5000)
    good = [base, base[3:50], torch.zeros(4, 5, 6), torch.zeros(7, 1, 3).expand(7, 1, 3), torch.zeros(()),
            torch.nn.Parameter(torch.zeros(2, 2)), torch.zeros(4, 8, 2).transpose(0, 0), torch.zeros(6, 1).t()]
    out = _lib.tensor_addresses(good, _sizes(*[t.numel() for t in good]), _lib.F32, cpu)
    assert out.tolist() == [t.data_ptr() for t in good]
    for dtype, code in ((torch.float16, _lib.F16), (torch.bfloat16, _lib.BF16)):
        t = torch.zeros(9, dtype=dtype)
        assert _lib.tensor_addresses([t], _sizes(9), code, cpu).tolist() == [t.data_ptr()]
    for other in (torch.zeros(9), torch.zeros(11), torch.zeros(20)[::2], torch.zeros(5, 2).t(), torch.zeros(1).expand(10),
                  torch.zeros(10, dtype=torch.bfloat16), torch.zeros(10, dtype=torch.float64),
                  torch.zeros(10, dtype=torch.int32), torch.zeros(0)):
        assert _lib.tensor_addresses([good[0], other], _sizes(5000, 10), _lib.F32, cpu) == 1, other
    assert _lib.tensor_addresses([torch.zeros(9, dtype=torch.float16)], _sizes(9), _lib.BF16, cpu) == 0
    assert _lib.tensor_addresses([base, None], _sizes(5000, 1), _lib.F32, cpu) == 1
    with pytest.raises(ValueError, match="sizes"):
        _lib.tensor_addresses([base], _sizes(5000, 1), _lib.F32, cpu)
    # expected on a GPU, found on the host
    assert _lib.tensor_addresses([base], _sizes(5000), _lib.F32, torch.device("cuda", 0)) == 0
    with pytest.raises(Exception):
        _lib.tensor_addresses([torch.zeros(3, 3).to_sparse()], _sizes(9), _lib.F32, cpu)


def test_addresses_c_arguments():
    lib, p = _lib.lib(), ctypes.c_void_p(16)  # never followed: validation fails first
    r, half, empty = ((ctypes.c_void_p * 3)(*v) for v in ((16, 16, 16), (16, 0, 16), (0, 16, 16)))
    for args in ((None, p, p, 1, 0, 1, 0, p), (half, p, p, 1, 0, 1, 0, p), (empty, p, p, 1, 0, 1, 0, p),
                 (r, None, p, 1, 0, 1, 0, p), (r, p, None, 1, 0, 1, 0, p), (r, p, p, 0, 0, 1, 0, p),
                 (r, p, p, 1, 7, 1, 0, p), (r, p, p, 1, 0, 1, 0, None)):
        assert lib.soup_tensor_addresses(*args) == _lib.SOUP_ERR_INVALID


def _held(params):
    h = optim._Held()
    h.params, h.sizes = params, [p.numel() for p in params]
    h.by_dtype = [(_lib.F32, torch.float32, params, _sizes(*h.sizes), array.array("i", range(len(params))))]
    return h


@pytest.mark.parametrize("change", [lambda p: torch.zeros(4), lambda p: torch.zeros(40), lambda p: torch.zeros(4, 2).t(),
                                    lambda p: torch.zeros(2, 4, dtype=torch.bfloat16), lambda p: p[:, ::2],
                                    lambda p: torch.zeros(2, 4).to_sparse()])
def test_parameters_given_other_memory_are_refused(change):
    """p.data = ... under a gradient that stays: nothing is launched over the old sizes."""
    opt = object.__new__(optim.MultiTensorAdamW)
    ps = [torch.nn.Parameter(torch.zeros(2, 4)) for _ in range(3)]
    for p in ps:
        p.grad = torch.ones(2, 4)
    held, cpu = _held(ps), torch.device("cpu")
    (_, addresses, grads, sizes, *_), = opt._tables(held, cpu)
    assert addresses.tolist() == [p.data_ptr() for p in ps] and grads.tolist() == [p.grad.data_ptr() for p in ps]
    new = change(torch.zeros(2, 8))
    try:
        ps[1].data = new
    except (RuntimeError, NotImplementedError, TypeError):
        pytest.skip("torch refuses that itself")
    with pytest.raises(ValueError, match="parameters must stay"):
        opt._tables(held, cpu)
    ps[1].grad = None  # then it has no part in the step
    (_, addresses, _, sizes, *_), = opt._tables(held, cpu)
    assert addresses.tolist() == [ps[0].data_ptr(), ps[2].data_ptr()] and sizes.tolist() == [8, 8]


def test_gradients_of_another_size_are_refused():
    opt = object.__new__(optim.MultiTensorAdamW)
    p = torch.nn.Parameter(torch.zeros(2, 4))
    held = _held([p])
    p.data = torch.zeros(4)
    p.grad = torch.ones(4)
    p.data = torch.zeros(2, 4)
    with pytest.raises(ValueError, match="gradients must be"):
        opt._tables(held, torch.device("cpu"))
    p.grad = None
    p.grad = torch.ones(4, 2).t()  # another order: copied
    (_, _, grads, _, _, kept, *_), = opt._tables(held, torch.device("cpu"))
    assert kept[0].is_contiguous() and grads[0] == kept[0].data_ptr()


# -------------------------------------------------------------- the model itself ----
def _model(monkeypatch, attention="sdpa", seed=0):
    """A small model on the host, its operators in plain torch."""
    monkeypatch.setattr(kernels, "multi_lora_linear", plain._plain_lora)
    monkeypatch.setattr(kernels, "apply_multi_axis_rope", plain._plain_axes)
    cfg = qlora.qwen2_1p5b_config(2, hidden_size=64, intermediate_size=96, num_attention_heads=2,
                                  num_key_value_heads=1, vocab_size=100, head_dim=32)
    cfg._attn_implementation = attention
    m = qlora.build_qwen2_qlora(cfg, device="cpu", seed=seed, r=8, alpha=16, quantize=False, adapters=3, qk_norm=True,
                                train_norms=True, rope_sections=(4, 6, 6), dtype=torch.float32)
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        for n, p in m.named_parameters():
            if "lora_B" in n:
                p.copy_(0.1 * torch.randn(p.shape, generator=g))
            if "_norm.weight" in n and "self_attn" in n:
                p.copy_(1 + 0.2 * torch.randn(p.shape, generator=g))
    return m


def _batch(b, s=12, seed=3):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 100, (b, s), generator=g)
    pos = torch.arange(s).expand(3, b, s).clone()
    pos[1:, :, s // 2:] = torch.randint(0, 9, (2, b, s - s // 2), generator=g)
    return ids, pos


@pytest.mark.parametrize("attention", ["sdpa", "eager"])
@pytest.mark.parametrize("b", [1, 2, 3])
def test_positions_of_several_axes_in_a_call_of_the_model(b, attention, monkeypatch):
    """model(ids, position_ids=[axes, B, S]) is the body with a prepared causal mask; a padded
    batch's rows are those of the sequences alone."""
    m = _model(monkeypatch, attention)
    ids, pos = _batch(b)
    m.adapter_ids.set(torch.arange(b))
    with torch.no_grad():
        got = m(ids, position_ids=pos).logits
        assert not torch.allclose(got, m(ids).logits)  # the axes count
        # the same positions on every axis, given as [B, S] and as [axes, B, S]
        text = torch.arange(12).expand(b, 12)
        one, two = m(ids, position_ids=text).logits, m(ids, position_ids=text.expand(3, b, 12)).logits
        assert torch.equal(one, two) and torch.equal(one, m(ids).logits)
        for i in range(b):
            m.adapter_ids.set(torch.tensor([i]))
            alone = m(ids[i:i + 1, :9], position_ids=pos[:, i:i + 1, :9]).logits
            # the same sums in products of other row counts, 200 roundings of 2^-24 of numbers of a few units
            assert float((got[i, :9] - alone[0]).abs().max()) <= 200 * 2.0 ** -24 * 8
        mask = torch.ones(b, 12, dtype=torch.int64)
        mask[:, 9:] = 0
        m.adapter_ids.set(torch.arange(b))
        padded = m(ids, attention_mask=mask, position_ids=pos).logits
        assert float((padded[:, :9] - got[:, :9]).abs().max()) <= 200 * 2.0 ** -24 * 8
        (last,) = m.model(ids, None, pos, return_dict=False)[:1]  # by place
        assert torch.equal(m.lm_head(last), got)
        with pytest.raises(ValueError, match="position_ids"):
            m(ids, position_ids=pos[:2])
        assert torch.equal(m(ids).logits, one)  # nothing of a refused call is left


def _grads(m, hidden):
    m.zero_grad()
    hidden.square().sum().backward()
    return [p.grad for p in m.parameters() if p.requires_grad]


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_layers_run_again_with_the_ids_of_their_forward(reentrant, monkeypatch):
    """Two forward passes of different ids, and a call without a gradient, before the first
    one's backward pass: gradients of each are those without checkpointing."""
    m = _model(monkeypatch)
    m.train()
    (one, pos), (two, _) = _batch(2, seed=1), _batch(2, seed=2)
    a, b, c = (torch.tensor(v) for v in ([0, 1], [2, -1], [1, 1]))

    def run():
        m.adapter_ids.set(a)
        h1 = m.model(one, position_ids=pos)[0]
        m.adapter_ids.set(b)
        h2 = m.model(two)[0]
        with torch.no_grad():
            h3 = m.model(one, adapter_ids=c)[0]
        assert m.adapter_ids.ids is b  # an argument holds for its call alone
        return h3, _grads(m, h1), _grads(m, h2)

    want = run()
    m.enable_input_require_grads()
    m.gradient_checkpointing_enable({"use_reentrant": reentrant})
    got = run()
    assert torch.equal(want[0], got[0])
    for w, g in zip(want[1:], got[1:]):
        for x, y in zip(w, g):
            torch.testing.assert_close(x, y, rtol=1e-5, atol=1e-6 * float(x.abs().max() + 1e-3))
    assert not m.adapter_ids._running


def test_adapter_ids_of_a_call(monkeypatch):
    m = _model(monkeypatch)
    ids, pos = _batch(2)
    with torch.no_grad():
        with pytest.raises(ValueError, match="not set"):
            m(ids)
        with pytest.raises(ValueError, match="adapter ids"):
            m(ids, adapter_ids=torch.zeros(2))
        m.adapter_ids.set(torch.tensor([2, 2]))
        one = m(ids).logits
        assert torch.equal(one, m(ids, adapter_ids=torch.tensor([2, 2])).logits)
        assert not torch.equal(one, m(ids, adapter_ids=torch.tensor([0, 2])).logits)
        assert torch.equal(one, m(ids).logits)
        assert not m.adapter_ids._running  # also after the refusals


def test_norms_that_were_trained_are_in_the_adapters_file(tmp_path, monkeypatch):
    """A step, saved and loaded into a fresh model: the same logits, also where the fresh model
    does not train its norms; a file without them is refused where the model does."""
    m = _model(monkeypatch)
    ids, pos = _batch(2)
    a = torch.tensor([1, 2])
    m(ids, position_ids=pos, adapter_ids=a).logits.square().mean().backward()
    norms = {n: p for n, p in m.named_parameters() if "q_norm" in n or "k_norm" in n}
    assert len(norms) == 4
    with torch.no_grad():
        for p in m.parameters():
            if p.grad is not None:
                assert p.grad.any()
                p.sub_(0.1 * p.grad / p.grad.norm())
        want = m(ids, position_ids=pos, adapter_ids=a).logits
    for i in (1, 2):
        adapter.save_adapter(m, str(tmp_path / str(i)), index=i)
    cfg = json.load(open(tmp_path / "1" / "adapter_config.json"))
    assert cfg["modules_to_save"] == ["k_norm", "q_norm"]
    listing = adapter.header_listing(str(tmp_path / "1" / "adapter_model.safetensors"))
    assert listing["base_model.model.model.layers.1.self_attn.q_norm.weight"] == ["F32", [32]]
    for trained in (True, False):
        fresh = _model(monkeypatch)
        for n, p in fresh.named_parameters():
            if "q_norm" in n or "k_norm" in n:
                p.requires_grad_(trained)
        for i in (1, 2):
            adapter.load_adapter(fresh, str(tmp_path / str(i)), index=i)
        with torch.no_grad():
            assert torch.equal(fresh(ids, position_ids=pos, adapter_ids=a).logits, want)
        assert all(p.requires_grad == trained for n, p in fresh.named_parameters() if "q_norm" in n)
        assert torch.equal(fresh.lm_head.weight, m.lm_head.weight)  # frozen, and in no file
    for n, p in fresh.named_parameters():
        if "_norm" in n:
            p.requires_grad_(False)
    adapter.save_adapter(fresh, str(tmp_path / "bare"), index=0)
    assert json.load(open(tmp_path / "bare" / "adapter_config.json"))["modules_to_save"] is None
    with pytest.raises(KeyError, match="parameters that the model trains"):
        adapter.load_adapter(m, str(tmp_path / "bare"), index=0)
    adapter.load_adapter(m, str(tmp_path / "bare"), strict=False, index=0)
    # a model without such norms has no place for them
    other = qlora.build_qwen2_qlora(m.config, device="cpu", r=8, alpha=16, quantize=False, adapters=3,
                                    dtype=torch.float32)
    with pytest.raises(KeyError, match="unexpected"):
        adapter.load_adapter(other, str(tmp_path / "1"), index=1)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3.4e38])  # the last one as bfloat16
def test_factors_that_are_not_finite_stay_out_of_a_model_with_several_adapters(bad, tmp_path, monkeypatch):
    m = _model(monkeypatch)
    before = m.model.layers[0].mlp.up_proj.lora_B.detach().clone()
    other = _model(monkeypatch, seed=1)
    with torch.no_grad():
        other.model.layers[0].mlp.up_proj.lora_B[3, 1, 2] = bad
    adapter.save_adapter(other, str(tmp_path), index=1)
    with pytest.raises(ValueError, match="not finite"):
        adapter.load_adapter(m, str(tmp_path), index=1)
    assert torch.equal(m.model.layers[0].mlp.up_proj.lora_B, before)
    adapter.save_adapter(other, str(tmp_path), index=2)
    adapter.load_adapter(m, str(tmp_path), index=2)


def test_two_calls_of_a_model_at_once(monkeypatch):
    """Two threads, each with its own ids and positions: a call's are its own, whatever the
    other one does between its layers."""
    m = _model(monkeypatch)
    (one, pos), (two, pos2) = _batch(2, seed=1), _batch(2, seed=2)
    jobs = [(one, pos.flip(1), torch.tensor([0, 1])), (two, pos2, torch.tensor([2, -1]))]

    def call(job):
        with torch.no_grad():
            return m(job[0], position_ids=job[1], adapter_ids=job[2]).logits

    want = [call(j) for j in jobs]
    # the layers and the rotary embedding of both calls in turn
    turn = threading.Barrier(2, timeout=60)

    def wait(*args):
        turn.wait()

    for mod in [m.model.rotary_emb, *m.model.layers, *(layer.self_attn.q_proj for layer in m.model.layers)]:
        mod.register_forward_pre_hook(wait)
    got = [None, None]

    def run(i):
        try:
            got[i] = call(jobs[i])
        except BaseException:
            turn.abort()
            raise

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for w, g in zip(want, got):
        assert torch.equal(w, g)
    assert not m.adapter_ids._running and not m.model.rotary_emb.positions


def test_copies_of_a_model(monkeypatch):
    """Deep copies and pickled models are models of their own, heads and adapters with them."""
    m = _model(monkeypatch)
    ids, pos = _batch(2)
    m.adapter_ids.set(torch.tensor([0, 2]))
    buf = io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    with torch.no_grad():
        want = m(ids, position_ids=pos).logits
        for other in (copy.deepcopy(m), torch.load(buf, weights_only=False)):
            assert torch.equal(other(ids, position_ids=pos).logits, want)
            other.adapter_ids.set(torch.tensor([1, 1]))
            for p in other.model.layers[0].self_attn.q_norm.parameters():
                p.mul_(2.0)
            assert not torch.equal(other(ids, position_ids=pos).logits, want)
            assert torch.equal(m(ids, position_ids=pos).logits, want)


@pytest.mark.parametrize("attention", ["sdpa", "eager"])
def test_single_tokens_against_a_cache(attention, monkeypatch):
    """A prompt, a token and a chunk of tokens against a cache, with positions of several axes:
    the logits of the whole sequence (200 roundings of 2^-24 of numbers of a few units)."""
    m = _model(monkeypatch, attention)
    ids, pos = _batch(2)
    m.adapter_ids.set(torch.tensor([0, 2]))
    cache = DynamicCache(config=m.config)
    with torch.no_grad():
        want = m(ids, position_ids=pos).logits
        got = [m(ids[:, a:b], position_ids=pos[..., a:b], past_key_values=cache, use_cache=True).logits
               for a, b in ((0, 7), (7, 8), (8, 12))]
    assert float((torch.cat(got, 1) - want).abs().max()) <= 200 * 2.0 ** -24 * 8
