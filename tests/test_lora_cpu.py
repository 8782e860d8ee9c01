"""CPU tests of the low-rank adapters: the eager form against the float64 oracle and autograd, the
module and the decoder with adapters, and the refusals."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from experiment_swa_kda_amd import LoraLinear, _lib, lora_linear, ops
from experiment_swa_kda_amd.kda import Linear
from experiment_swa_kda_amd.model import GPT, GPTConfig
from oracle import post_training as P


def case(B, T, K, N, R, n, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    shapes = dict(x=(B, T, K), w=(N, K), a=(n, R, K), b=(n, N, R), dy=(B, T, N))
    d = {k: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype) for k, s in shapes.items()}
    d["scale"] = torch.rand(n, generator=g) + 0.5
    return d


def n64(t):
    return t.detach().double().numpy()


@pytest.mark.parametrize("ids", [[0, 2, -1], [1, 1, 1], [5, -7, 0], [[0, 1, 2, -1], [2, 2, 0, 0], [9, 1, 1, 1]]])
def test_eager_matches_oracle_and_its_gradients_differences(ids):
    d = case(3, 4, 6, 5, 2, 3)
    ids = torch.tensor(ids, dtype=torch.int32)
    rows = (ids if ids.ndim == 2 else ids[:, None].expand(3, 4)).flatten().tolist()
    leaves = [d[k].clone().requires_grad_() for k in ("x", "w", "a", "b")]
    y = lora_linear(*leaves, ids, d["scale"])
    grads = torch.autograd.grad(y, leaves, d["dy"])
    want = P.lora(n64(d["x"]).reshape(12, 6), *(n64(d[k]) for k in ("w", "a", "b")), rows, n64(d["scale"]),
                  n64(d["dy"]).reshape(12, 5))
    for got, ref in zip((y, *grads), want):
        np.testing.assert_allclose(n64(got).reshape(ref.shape), ref, rtol=1e-10, atol=1e-12)
    assert torch.autograd.gradcheck(lambda *v: lora_linear(*v, ids, d["scale"]), leaves)


def test_a_row_without_an_adapter_and_another_adapters_nan():
    d = case(2, 3, 6, 5, 2, 3)
    ids = torch.tensor([-1, 1], dtype=torch.int32)
    d["a"][0] = float("nan")
    d["b"][2] = float("inf")
    y = lora_linear(d["x"], d["w"], d["a"], d["b"], ids, d["scale"])
    assert torch.equal(y[0], torch.nn.functional.linear(d["x"], d["w"])[0]) and torch.isfinite(y).all()


def test_module_and_decoder_with_adapters():
    torch.manual_seed(0)
    m = LoraLinear(6, 5, 3, 2, alpha=4.0)
    x, ids = torch.randn(2, 4, 6), torch.tensor([1, -1], dtype=torch.int32)
    base = Linear.forward(m, x)
    assert torch.equal(m(x), base)
    m.adapter_ids = ids
    assert torch.equal(m(x), base)  # a fresh adapter changes nothing
    with torch.no_grad():
        m.lora_b.normal_()
    y = m(x)
    assert torch.equal(y[1], base[1]) and not torch.allclose(y[0], base[0])
    want = base[0] + 2.0 * (x[0] @ m.lora_a[1].t()) @ m.lora_b[1].t()
    assert torch.allclose(y[0], want, atol=1e-5)

    gpt = GPT(GPTConfig(sequence_len=16, vocab_size=50, n_layer=2, n_head=1, n_embd=64, mode="reference"))
    gpt.init_weights()
    torch.nn.init.normal_(gpt.lm_head.weight, 0.0, 0.3)
    idx = torch.randint(0, 50, (3, 5))
    before = gpt(idx)
    names = {k for k, _ in gpt.named_parameters()}
    new = gpt.add_adapters(4, 8)
    assert len(new) == 2 * (3 * 2 + 1) and names < {k for k, _ in gpt.named_parameters()}
    assert torch.equal(gpt(idx), before)
    with torch.no_grad():
        for p in new:
            p.normal_(0.0, 0.05)
    gpt.use_adapters(torch.tensor([2, -1, 0], dtype=torch.int32))
    mixed = gpt(idx)
    assert torch.allclose(mixed[1], before[1], atol=1e-6)
    for row, a in ((0, 2), (2, 0)):  # a batch of requests gives each what it gets alone
        gpt.use_adapters(torch.tensor([a], dtype=torch.int32))
        assert torch.allclose(gpt(idx[row:row + 1])[0], mixed[row], atol=1e-5)
        assert not torch.allclose(mixed[row], before[row], atol=1e-3)
    gpt.use_adapters(torch.tensor([2, -1, 0], dtype=torch.int32))
    loss = gpt(idx, idx)
    grads = torch.autograd.grad(loss, new)
    assert all(torch.isfinite(g).all() for g in grads)
    assert all(not g[[1, 3]].any() and g[[0, 2]].any() for g in grads)  # the adapters in use alone
    with pytest.raises(ValueError, match="once"):
        gpt.add_adapters(4, 8)


def test_adapters_are_added_to_all_projections_or_none():
    gpt = GPT(GPTConfig(sequence_len=16, vocab_size=50, n_layer=2, n_head=1, n_embd=64, mode="reference"))
    with pytest.raises(ValueError, match="no adapters"):
        gpt.use_adapters(torch.tensor([0], dtype=torch.int32))
    gpt.use_adapters(None)
    with pytest.raises(ValueError, match="rank"):
        gpt.add_adapters(2, 0)
    gpt.transformer.h[1].mlp.c_proj = LoraLinear(256, 64, 1, 8)
    with pytest.raises(ValueError, match="plain Linear"):
        gpt.add_adapters(2, 8)
    assert type(gpt.transformer.h[0].attn.o_proj) is Linear and type(gpt.lm_head) is Linear


def test_kept_copies_follow_an_adapter_put_in_a_slot():
    m = LoraLinear(16, 8, 3, 8)
    kept = m.keep_adapters_bf16()
    assert m._adapters16() is kept
    with torch.no_grad():
        m.lora_b[1] = 0.5
    now = m._adapters16()
    assert now is not kept and torch.equal(now[1], m.lora_b.detach().bfloat16())
    kept = m.keep_adapters_bf16()
    assert m._adapters16() is kept
    m.lora_a = torch.nn.Parameter(torch.ones(3, 8, 16))
    assert torch.equal(m._adapters16()[0], torch.ones(3, 8, 16).bfloat16())
    m.drop_adapters_bf16()
    assert m._lora16 is None


def test_refusals():
    d = case(3, 4, 8, 16, 8, 3, dtype=torch.float32)
    ids = torch.zeros(3, dtype=torch.int32)
    args = [d["x"], d["w"], d["a"], d["b"], ids, d["scale"]]

    def refused(words, **change):
        new = list(args)
        for k, v in change.items():
            new["x w a b ids scale".split().index(k)] = v
        with pytest.raises(ValueError, match=words):
            lora_linear(*new)

    refused("weight", w=d["w"][:, :4])
    refused("lora_a", a=d["a"][:2])
    refused("lora_a", b=d["b"].transpose(1, 2))
    refused("scaling", scale=d["scale"][:2])
    refused("adapter_ids", ids=ids[:2])
    refused("adapter_ids", ids=ids.float())
    refused("expected", x=d["x"][0, 0])
    refused("constant", scale=d["scale"].clone().requires_grad_())
    with pytest.raises(RuntimeError, match="ROCm device"):
        ops.lora_forward(*(d[k].bfloat16() for k in ("x", "w", "a", "b")), ids, d["scale"])


@pytest.mark.skipif(not _lib.is_built(), reason="library not built")
def test_c_abi_refuses_bad_calls_without_gpu():
    lib = _lib.load()
    p, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)

    def refused(rc, words):
        assert rc != 0 and words in lib.kda_last_error().decode()

    shrink, expand, grad = lib.kda_lora_shrink, lib.kda_lora_expand, lib.kda_lora_grad
    refused(shrink(4, 12, 8, 2, p, 1, p, 16, p, 0, p, p, None), "multiples of 8")
    refused(shrink(4, 16, 12, 2, p, 1, p, 16, p, 0, p, p, None), "rank")
    refused(shrink(4, 16, 136, 2, p, 1, p, 16, p, 0, p, p, None), "rank")
    refused(shrink(4, 16, 8, 0, p, 1, p, 16, p, 0, p, p, None), "number of adapters")
    refused(shrink(4, 16, 8, 2, None, 1, p, 16, p, 0, p, p, None), "ids")
    refused(shrink(4, 16, 8, 2, p, 0, p, 16, p, 0, p, p, None), "rows per id")
    refused(shrink(4, 16, 8, 2, p, 1, odd, 16, p, 0, p, p, None), "unaligned")
    refused(shrink(4, 16, 8, 2, p, 1, p, 20, p, 0, p, p, None), "rows of x")
    refused(expand(4, 16, 8, 2, p, 1, p, None, 0, p, 16, None), "null")
    refused(expand(4, 16, 8, 2, p, 1, p, p, 0, p, 8, None), "rows of y")
    refused(grad(4, 16, 8, 2, p, 1, p, 16, None, 0, p, p, None), "null")
    refused(grad(4, 16, 8, 2, p, 1, p, 16, p, 0, None, p, None), "null")
    rows, linear, forward, backward = (getattr(lib, f"kda_lora_{k}") for k in ("linear_rows", "linear", "forward", "backward"))
    refused(rows(513, 16, 32, 8, 2, p, 1, p, 32, p, p, p, p, p, p, None), "at most 512 rows")
    refused(rows(4, 12, 24, 8, 2, p, 1, p, 24, p, p, p, p, p, p, None), "out_dim must be a multiple of 8")
    refused(linear(4, 12, 16, 8, 2, p, 1, p, 16, p, 0, p, p, p, None), "multiples of 8")
    refused(linear(4, 16, 16, 8, 2, p, 1, p, 16, p, 0, None, p, p, None), "null")
    refused(forward(4, 16, 32, 8, 2, p, 1, p, 32, p, p, p, p, 3, p, p, None), "unknown way")
    refused(forward(513, 16, 32, 8, 2, p, 1, p, 32, p, p, p, p, 0, p, p, None), "at most 512 rows")
    refused(backward(4, 16, 32, 8, 2, p, 1, p, 32, p, 16, p, p, p, p, p, 0, p, p, p, p, None), "unknown way")
    refused(backward(4, 16, 32, 8, 2, p, 1, p, 32, p, 16, p, p, p, p, p, 1, p, p, p, None, None), "null")
    assert lib.kda_lora_grad_scratch_bytes(32, 128, 16, 4) == 0  # one range is the result itself
    assert lib.kda_lora_grad_scratch_bytes(8192, 128, 16, 4) > 0
