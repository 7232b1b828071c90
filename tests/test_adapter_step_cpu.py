"""CPU: refusals of the operators of a step with several adapters, and the index
arithmetic of their kernels."""

import ctypes

import pytest
import torch

from auspex_soup_demo_b200 import _lib, adapter, kernels
from auspex_soup_demo_b200.kernels import qk_norm_rope
from auspex_soup_demo_b200.multi_adapter import AdapterIds, MultiLoRADenseLinear
from auspex_soup_demo_b200.optim import MultiTensorAdamW

BF = torch.bfloat16


# ----------------------------------------------------------- several adapters ----
def _lora(t=4, k=64, n=32, na=2, r=8, dtype=BF):
    return dict(x=torch.zeros(t, k, dtype=dtype), weight=torch.zeros(n, k, dtype=dtype),
                lora_a=torch.zeros(na, r, k, dtype=dtype), lora_b=torch.zeros(n, na, r, dtype=dtype),
                adapter_ids=torch.zeros(t, dtype=torch.int64))


@pytest.mark.parametrize("change,error,text", [
    (dict(x=torch.zeros(4, 56, dtype=BF)), ValueError, "fit together"),
    (dict(weight=torch.zeros(32, 64, 1, dtype=BF)), ValueError, "weight"),
    (dict(lora_a=torch.zeros(2, 8, 60, dtype=BF)), ValueError, "fit together"),
    (dict(lora_b=torch.zeros(2, 32, 8, dtype=BF)), ValueError, "fit together"),
    (dict(lora_a=torch.zeros(16, 64, dtype=BF)), ValueError, "lora_a"),
    (dict(x=torch.zeros(4, 64)), TypeError, "bfloat16"),
    (dict(), ValueError, "CUDA"),
])
def test_multi_lora_refuses(change, error, text):
    with pytest.raises(error, match=text):
        kernels.multi_lora_linear(**{**_lora(), **change})


def test_multi_lora_refuses_sizes():
    for bad in (dict(k=60), dict(n=36), dict(na=3, r=3), dict(na=257, r=16)):
        with pytest.raises(ValueError, match="multiples of 8"):
            kernels.multi_lora_linear(**_lora(**bad))


def test_multi_lora_c_arguments():
    lib = _lib.lib()
    p = ctypes.c_void_p(16)  # never dereferenced: validation fails first

    def fwd(t=4, n=64, k=64, na=2, r=8, ldx=64, state=1 << 20, x=p):
        return lib.soup_multi_lora_fwd(x, ldx, p, 64, None, p, p, p, p, 0, 1, t, n, k, na, r, p, n, p, state, None)

    assert fwd(t=0) == _lib.SOUP_ERR_INVALID
    assert fwd(t=(1 << 21) + 1) == _lib.SOUP_ERR_INVALID
    assert fwd(na=4097, r=1) == _lib.SOUP_ERR_INVALID
    assert fwd(x=None) == _lib.SOUP_ERR_INVALID
    assert fwd(n=60) == _lib.SOUP_ERR_UNSUPPORTED
    assert fwd(ldx=63) == _lib.SOUP_ERR_INVALID
    assert fwd(ldx=68) == _lib.SOUP_ERR_UNSUPPORTED  # rows that are not 16-byte aligned
    assert fwd(state=16) == _lib.SOUP_ERR_WORKSPACE
    assert fwd(x=ctypes.c_void_p(24)) == _lib.SOUP_ERR_UNSUPPORTED
    rc = lib.soup_multi_lora_bwd(p, 64, None, 64, p, 64, p, p, p, p, 0, 1, 4, 64, 64, 2, 8, p, 1 << 20, None, 64, p,
                                 _lib.BF16, None, 0, p, 1 << 20, None)
    assert rc == _lib.SOUP_ERR_INVALID  # lora_a's gradient without x
    rc = lib.soup_multi_lora_bwd(p, 64, p, 64, p, 64, p, p, p, p, 0, 1, 4, 64, 64, 2, 8, p, 1 << 20, p, 64, p,
                                 _lib.F16, None, 0, p, 1 << 20, None)
    assert rc == _lib.SOUP_ERR_INVALID  # a gradient in fp16
    rc = lib.soup_multi_lora_bwd(p, 64, p, 64, p, 64, p, p, p, p, 0, 1, 4, 64, 64, 2, 8, p, 1 << 20, p, 64, None, 0,
                                 None, 0, None, 0, None)
    assert rc == _lib.SOUP_ERR_WORKSPACE


@pytest.mark.parametrize("tokens,adapters,rank", [(1, 1, 8), (64, 3, 8), (65, 1, 64), (1000, 24, 8), (8192, 256, 16)])
def test_multi_lora_state_layout(tokens, adapters, rank):
    """Two words of 64- and one of 256-token blocks, then U at a 128-byte boundary, none overlapping."""
    m64 = (tokens + 63) // 64 * 8 * 2
    m256 = (m64 + 15) // 16 * 16
    u = m256 + ((tokens + 255) // 256 * 8 + 127) // 128 * 128
    u = (u + 127) // 128 * 128
    assert m256 >= m64 and u >= m256 + (tokens + 255) // 256 * 8
    assert _lib.lib().soup_multi_lora_state_bytes(tokens, adapters, rank) == u + tokens * adapters * rank * 2


def _bits(adapter, rank):
    lo, hi = adapter * rank // 64, (adapter * rank + rank - 1) // 64
    upto = (1 << 64) - 1 if hi == 63 else (1 << (hi + 1)) - 1
    return upto & ~((1 << lo) - 1)


@pytest.mark.parametrize("rank", [1, 3, 8, 16, 24, 48, 64, 100, 4096])
def test_rank_block_bits_cover_an_adapters_columns(rank):
    for a in range(4096 // rank):
        want = 0
        for c in range(a * rank, (a + 1) * rank):
            want |= 1 << (c // 64)
        assert _bits(a, rank) == want < 1 << 64


def _walk(bits, rank, ks):
    """The k blocks of CTA ``rank`` of a cluster of ks, as the kernel lists them."""
    words = [sum(b << i for i, b in enumerate(bits[w:w + 32])) for w in range(0, len(bits), 32)]
    count = sum(bin(w).count("1") for w in words)
    skip = count * rank // ks
    left = count * (rank + 1) // ks - skip
    out, w, cur = [], -1, 0
    while left:
        if cur == 0:
            w += 1
            cur = words[w]
            n = bin(cur).count("1")
            if skip >= n:
                skip -= n
                cur = 0
            continue
        b = (cur & -cur).bit_length() - 1
        cur &= cur - 1
        if skip:
            skip -= 1
            continue
        out.append(w * 32 + b)
        left -= 1
    return out


@pytest.mark.parametrize("ks", [1, 2, 3, 7, 16])
def test_token_blocks_are_shared_out_once_each(ks):
    g = torch.Generator().manual_seed(ks)
    for n in (1, 5, 32, 33, 64, 200):
        for p in (0.0, 0.1, 0.5, 1.0):
            bits = (torch.rand(n, generator=g) < p).int().tolist()
            got = [k for r in range(ks) for k in _walk(bits, r, ks)]
            assert got == [i for i, b in enumerate(bits) if b]


def test_division_by_a_sequence_length_as_a_product():
    for d in [1, 2, 3, 5, 7, 127, 128, 1000, 16001, 65535, 65537, (1 << 30) + 1, (1 << 31) - 1]:
        l = 0
        while (1 << l) < d:
            l += 1
        m = ((1 << (31 + l)) + d - 1) // d
        assert m < 1 << 32
        for n in {0, 1, d - 1, d, d + 1, 2 * d - 1, 7 * d + 3, (1 << 31) - 1, (1 << 31) - 2, (1 << 31) // d * d - 1}:
            if 0 <= n < 1 << 31:
                assert (n * m) >> (31 + l) == n // d, (n, d)


# ------------------------------------------------------- norms and rotation ----
def test_rope_axes():
    assert kernels.rope_axes((2, 1, 1)) == (0, 0, 1, 2)
    assert kernels.rope_axes([3, 0, 2]) == (0, 0, 0, 2, 2)
    assert kernels.rope_axes((4, 2, 2), interleaved=True) == (0, 1, 2, 0, 1, 2, 0, 0)
    a = kernels.rope_axes((16, 24, 24), interleaved=False)
    assert [a.count(i) for i in range(3)] == [16, 24, 24]
    a = kernels.rope_axes((24, 20, 20), interleaved=True)
    assert [a.count(i) for i in range(3)] == [24, 20, 20] and a[:6] == (0, 1, 2, 0, 1, 2)
    for bad in ((), (0, 0), (-1, 3), (1.5, 2)):
        with pytest.raises(ValueError, match="sections"):
            kernels.rope_axes(bad)


def _heads(b=1, h=2, hk=1, s=3, d=8, dtype=BF):
    return dict(q=torch.zeros(b, h, s, d, dtype=dtype), k=torch.zeros(b, hk, s, d, dtype=dtype),
                q_weight=torch.ones(d, dtype=dtype), k_weight=torch.ones(d, dtype=dtype),
                cos=torch.ones(s, d), sin=torch.zeros(s, d))


@pytest.mark.parametrize("change,error,text", [
    (dict(q=torch.zeros(2, 3, 8, dtype=BF)), ValueError, "B, H, S, D"),
    (dict(k=torch.zeros(1, 1, 4, 8, dtype=BF)), ValueError, "share"),
    (dict(k=torch.zeros(1, 1, 3, 8)), ValueError, "share"),
    (dict(), ValueError, "CUDA"),
])
def test_qk_norm_rope_refuses(change, error, text):
    with pytest.raises(error, match=text):
        kernels.apply_qk_norm_rope(**{**_heads(), **change})


@pytest.mark.parametrize("d", [7, 514, 1024])
def test_qk_norm_rope_refuses_head_dims(d):
    with pytest.raises(ValueError, match="head_dim"):
        kernels.apply_qk_norm_rope(**_heads(d=d))


def _desc(**kw):
    f = dict(batch=1, seq=2, d=8, hq=2, hk=1, dtype=2, wdtype=2, tdtype=2, source=0, inverse=0, table=(0, 0, 8),
             strides=(16, 8, 8, 1) * 6, eps=1e-6)
    f.update(kw)
    return qk_norm_rope._DESC.pack(f["batch"], f["seq"], f["d"], f["hq"], f["hk"], f["dtype"], f["wdtype"],
                                   f["tdtype"], f["source"], f["inverse"], *f["table"], *f["strides"], f["eps"])


def test_qk_norm_rope_descriptor_is_the_headers():
    text = open(_lib.__file__.replace("auspex_soup_demo_b200/_lib.py", "include/soupb200.h")).read()
    body = text[text.index("int64_t batch, seq, head_dim, hq, hk;"):text.index("} soup_qk_rope;")]
    assert qk_norm_rope._DESC.size == 8 * (5 + 5 + 3 + 16 + 8 + 1)
    order = [body.index(w) for w in ("batch", "dtype", "w_dtype", "table_dtype", "source", "inverse", "table[3]",
                                     "q[4]", "q_out[4]", "k[4]", "k_out[4]", "q_grad[4]", "k_grad[4]", "eps")]
    assert order == sorted(order)


@pytest.mark.parametrize("change", [dict(batch=0), dict(seq=0), dict(d=9), dict(d=514), dict(hq=0), dict(hk=0),
                                    dict(batch=1 << 30, seq=2), dict(strides=(16, 8, 8, 2) * 6), dict(eps=-1.0),
                                    dict(eps=float("nan")), dict(wdtype=1), dict(dtype=7, wdtype=7), dict(source=3),
                                    dict(tdtype=9), dict(inverse=1)])
def test_qk_norm_rope_c_arguments(change):
    p = ctypes.c_void_p(16)
    lib = _lib.lib()
    assert lib.soup_qk_norm_rope(p, p, p, p, p, p, p, p, None, _desc(**change), None) == _lib.SOUP_ERR_INVALID
    assert lib.soup_qk_norm_rope(p, p, p, p, None, p, p, p, None, _desc(), None) == _lib.SOUP_ERR_INVALID
    assert lib.soup_qk_norm_rope(p, p, p, p, p, p, p, p, None, None, None) == _lib.SOUP_ERR_INVALID
    assert lib.soup_qk_norm_rope(p, p, p, p, p, p, p, p, None, _desc(source=2), None) == _lib.SOUP_ERR_INVALID
    assert lib.soup_qk_norm_rope_bwd(p, p, p, p, p, p, p, p, p, None, p, p, None, _desc(), None, 0,
                                     None) == _lib.SOUP_ERR_WORKSPACE


def test_multi_axis_rope_refuses():
    q, k = torch.zeros(1, 2, 3, 8, dtype=BF), torch.zeros(1, 1, 3, 8, dtype=BF)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.apply_multi_axis_rope(q, k, torch.zeros(3, 1, 3, dtype=torch.int64), torch.ones(4), (0, 0, 1, 2))
    with pytest.raises(ValueError, match="both"):
        meta = torch.zeros(1, 2, 3, 8, dtype=BF, device="meta")
        qk_norm_rope._check("f", _FakeCuda(meta), _FakeCuda(k.to("meta")), torch.ones(8), None, 1e-6)


class _FakeCuda:
    """A tensor that says it is on a CUDA device, for checks that come after that one."""

    def __init__(self, t):
        self._t = t
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self._t, name)


# --------------------------------------------------------------------- AdamW ----
@pytest.mark.parametrize("kw,text", [(dict(state_bits=16), "state_bits"), (dict(max_grad_norm=0.0), "max_grad_norm"),
                                     (dict(max_grad_norm=float("inf")), "max_grad_norm"), (dict(lr=-1.0), "lr"),
                                     (dict(betas=(1.0, 0.9)), "betas"), (dict(eps=0.0), "eps"),
                                     (dict(eps=1e-40), "eps"), (dict(weight_decay=-0.1), "weight_decay"),
                                     (dict(), "CUDA")])
def test_adamw_multi_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        MultiTensorAdamW([torch.nn.Parameter(torch.zeros(4))], **kw)


def test_adamw_multi_c_arguments():
    lib = _lib.lib()
    p = ctypes.c_void_p(16)
    ptrs = (ctypes.c_void_p * 2)(16, 16)
    sizes = _lib.i64_array([4, 4])
    blocks = (ctypes.c_int32 * 2)(0, 1)

    def step(params=ptrs, n=sizes, count=2, dtype=0, bits=8, b1=0.9, eps=1e-8, coefs=p, scale=p, partials=0):
        return lib.soup_adamw_multi(params, ptrs, n, blocks, count, dtype, bits, p, p, scale, scale, 1e-3, b1, 0.99,
                                    eps, 0.0, 0.0, None, partials, None, p, 1, coefs, None)

    for bad in (dict(params=None), dict(count=0), dict(n=_lib.i64_array([4, 0])), dict(bits=16), dict(b1=1.0),
                dict(eps=0.0), dict(eps=1e-38 / 1e2), dict(coefs=None), dict(coefs=ctypes.c_void_p(8)),
                dict(scale=None), dict(partials=1), dict(dtype=5)):
        assert step(**bad) == _lib.SOUP_ERR_INVALID, bad
    used = ctypes.c_int(0)
    assert lib.soup_grad_square(ptrs, sizes, 2, 0, p, 8, ctypes.byref(used), None) == _lib.SOUP_ERR_WORKSPACE
    assert lib.soup_grad_square(None, sizes, 2, 0, p, 1 << 20, ctypes.byref(used), None) == _lib.SOUP_ERR_INVALID


# ------------------------------------------------------- linears and adapter files ----
def test_multi_adapter_linear_and_its_files(tmp_path):
    torch.manual_seed(0)

    class Body(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.ids = AdapterIds(3)
            self.q_proj = MultiLoRADenseLinear(torch.nn.Linear(16, 8, bias=False), self.ids, 4, [8, 16, 10])

    m = Body()
    assert m.q_proj.lora_A.shape == (3, 4, 16) and m.q_proj.lora_B.shape == (8, 3, 4)
    assert m.q_proj.scaling.tolist() == [2.0, 4.0, 2.5]
    m.to(torch.bfloat16)
    assert m.q_proj.scaling.dtype == torch.float32 and m.q_proj.weight.dtype == torch.bfloat16
    m.to(torch.float32)
    with torch.no_grad():
        m.q_proj.lora_B.normal_()
    with pytest.raises(ValueError, match="which"):
        adapter.save_adapter(m, str(tmp_path))
    with pytest.raises(IndexError):
        adapter.save_adapter(m, str(tmp_path), index=3)
    adapter.save_adapter(m, str(tmp_path), index=2)
    other = Body()
    with pytest.raises(ValueError, match="scale"):
        adapter.load_adapter(other, str(tmp_path), index=0)
    assert adapter.load_adapter(other, str(tmp_path), index=2)["lora_alpha"] == 10
    assert torch.equal(other.q_proj.lora_A[2], m.q_proj.lora_A[2])
    assert torch.equal(other.q_proj.lora_B[:, 2], m.q_proj.lora_B[:, 2])
    with pytest.raises(ValueError, match="not set"):
        m.q_proj(torch.zeros(1, 16))
    with pytest.raises(ValueError, match="adapter ids"):
        m.ids.set(torch.zeros(2))


def test_rotations_refuse_what_has_no_form():
    """More axes than a byte counts, and heads of q or k alone."""
    meta = _FakeCuda(torch.zeros(1, 2, 3, 8, dtype=BF, device="meta"))
    pos = torch.zeros(300, 3, dtype=torch.int64, device="meta")
    with pytest.raises(ValueError, match=r"axes must be in \[0, 256\)"):
        kernels.apply_multi_axis_rope(meta, meta, pos, torch.ones(4, device="meta"), (0, 1, 2, 256))
    none = _FakeCuda(torch.zeros(1, 0, 3, 8, dtype=BF, device="meta"))
    with pytest.raises(ValueError, match="both have heads"):
        qk_norm_rope._check("f", meta, none, None, None, 1e-6)


def test_adamw_multi_refuses_a_parameter_twice():
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.warns(UserWarning), pytest.raises(ValueError, match="twice"):
        MultiTensorAdamW([p, p])
