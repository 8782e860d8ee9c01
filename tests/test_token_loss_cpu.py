"""CPU tests of the post-training losses: the float64 oracle against autograd and differences, the
eager forms against the oracle, and the refusals."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from experiment_swa_kda_amd import _lib, ops
from experiment_swa_kda_amd.model import GPT, GPTConfig, policy_loss, preference_loss, softcap_log_probs
from oracle import post_training as P

VOCAB, COLS, CAP = 37, 40, 15.0


def case(rows, seed, ignore_every=4):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, COLS, generator=g, dtype=torch.float64) * 4
    t = torch.randint(0, VOCAB, (rows,), generator=g)
    t[::ignore_every] = -1
    row = [torch.randn(rows, generator=g, dtype=torch.float64) for _ in range(4)]
    return x, t, row


def n(t):
    return None if t is None else t.detach().double().numpy()


def difference(f, x, eps=1e-6):
    """Central differences of a scalar function of a float64 array."""
    out = np.zeros(x.size)
    for i in range(x.size):
        hi, lo = x.copy(), x.copy()
        hi.flat[i] += eps
        lo.flat[i] -= eps
        out[i] = (f(hi) - f(lo)) / (2 * eps)
    return out.reshape(x.shape)


def test_oracle_log_probs_match_torch_and_differences():
    x, t, (g, h, *_) = case(9, 1)
    logp, ent, z, p = P.rows(n(x), t.tolist(), VOCAB, CAP)
    q = torch.log_softmax(CAP * torch.tanh(x[:, :VOCAB] / CAP), -1)
    keep = t >= 0
    np.testing.assert_allclose(logp[keep], q[keep].gather(1, t[keep, None])[:, 0].numpy(), rtol=1e-12)
    np.testing.assert_allclose(ent[keep], torch.distributions.Categorical(logits=q[keep]).entropy().numpy(), rtol=1e-12)
    assert not logp[~keep.numpy()].any() and not ent[~keep.numpy()].any()

    def scalar(a):
        lp, en, _, _ = P.rows(a, t.tolist(), VOCAB, CAP)
        return lp @ n(g) + en @ n(h)

    grad = P.logit_grad(n(x), t.tolist(), VOCAB, CAP, n(g), n(h))
    np.testing.assert_allclose(grad, difference(scalar, n(x)), atol=1e-8)


def test_oracle_slopes_match_differences():
    _, t, (logp, old, adv, ref) = case(16, 2)
    w = torch.rand(16, dtype=torch.float64)
    for weights, r in ((None, n(ref)), (n(w), n(ref)), (n(w), None)):
        args = (t.tolist(), n(old), n(adv), r, weights, 0.8, 1.3, 0.1)
        slope = P.policy(n(logp), *args)[3]
        np.testing.assert_allclose(slope, difference(lambda a: P.policy(a, *args)[0], n(logp)), atol=1e-8)
    for average in (False, True):
        args = (t.tolist(), [0, 3, 3, 9, 15], n(ref)[:4], 0.7, 0.1, average)
        masked = np.where(t.numpy() >= 0, n(logp), 0.0)
        slope = P.preference(masked, *args)[3]
        np.testing.assert_allclose(slope, difference(lambda a: P.preference(a, *args)[0], masked), atol=1e-8)


def test_eager_log_probs_match_oracle():
    x, t, (g, h, *_) = case(12, 3)
    t[5] = VOCAB  # out of range
    x[4, 7] = float("nan")  # a masked row
    leaf = x.clone().requires_grad_()
    logp, ent = softcap_log_probs(leaf, t, VOCAB, CAP, entropy=True)
    e_logp, e_ent, _, _ = P.rows(np.nan_to_num(n(x)), t.tolist(), VOCAB, CAP)
    np.testing.assert_allclose(n(logp), e_logp, rtol=1e-12, atol=1e-12)
    np.testing.assert_allclose(n(ent), e_ent, rtol=1e-12, atol=1e-12)
    ok = torch.arange(12) != 5
    (grad,) = torch.autograd.grad([logp[ok], ent[ok]], leaf, [g[ok], h[ok]])
    t[5] = -1
    np.testing.assert_allclose(n(grad), P.logit_grad(np.nan_to_num(n(x)), t.tolist(), VOCAB, CAP, n(g), n(h)), atol=1e-12)


@pytest.mark.parametrize("weighted,with_ref", [(False, True), (True, True), (True, False)])
def test_eager_policy_loss_matches_oracle(weighted, with_ref):
    x, t, (noise, adv, ref, w) = case(24, 4)
    logp = P.rows(n(x), t.tolist(), VOCAB, CAP)[0]
    old, ref = torch.from_numpy(logp) + 0.3 * noise, torch.from_numpy(logp) + 0.2 * ref
    w = w.abs() if weighted else None
    if weighted:
        w[3] = 0.0
        x[3, 0] = float("nan")  # a row of no weight
    leaf = x.clone().requires_grad_()
    r = policy_loss(leaf, t, old, adv, VOCAB, CAP, ref_log_probs=ref if with_ref else None, clip=0.1, clip_high=0.2,
                    kl_coef=0.3, weights=w)
    f32 = [n(v.float()) if v is not None else None for v in (old, adv, ref if with_ref else None, w)]
    loss, kl, share, slope = P.policy(logp, t.tolist(), *f32, 0.9, 1.2, 0.3)
    assert abs(r.loss.item() - loss) < 1e-9 and abs(r.kl.item() - kl) < 1e-9 and abs(r.clip_fraction.item() - share) < 1e-9
    (grad,) = torch.autograd.grad(r.loss, leaf)
    keep = np.flatnonzero(slope)
    np.testing.assert_allclose(n(grad)[keep], P.logit_grad(np.nan_to_num(n(x)), t.tolist(), VOCAB, CAP, slope)[keep],
                               atol=1e-9)


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_eager_preference_loss_matches_oracle(average, packed):
    x, t, (ref, *_) = case(24, 5)
    starts = [0, 1, 7, 7, 22] if packed else [0, 6, 12, 18, 24]
    lx, lt = (x, t) if packed else (x.view(4, 6, COLS), t.view(4, 6))
    leaf = lx.clone().requires_grad_()
    r = preference_loss(leaf, lt, VOCAB, CAP, beta=0.4, ref_log_probs=ref[:4], label_smoothing=0.2, average=average,
                        cu_seqlens=torch.tensor(starts, dtype=torch.int32) if packed else None)
    logp = P.rows(n(x), t.tolist(), VOCAB, CAP)[0]
    loss, seq, m, slope = P.preference(logp, t.tolist(), starts, n(ref[:4].float()), 0.4, 0.2, average)
    np.testing.assert_allclose(n(r.log_probs), seq, rtol=1e-12)
    np.testing.assert_allclose(n(r.margins), m, rtol=1e-10)
    assert abs(r.loss.item() - loss) < 1e-12
    (grad,) = torch.autograd.grad(r.loss, leaf)
    np.testing.assert_allclose(n(grad).reshape(24, COLS), P.logit_grad(n(x), t.tolist(), VOCAB, CAP, slope), atol=1e-12)


def test_model_methods_run_on_cpu():
    torch.manual_seed(0)
    cfg = GPTConfig(sequence_len=16, vocab_size=50, n_layer=1, n_head=1, n_embd=64, mode="reference")
    m = GPT(cfg)
    m.init_weights()
    torch.nn.init.normal_(m.lm_head.weight, 0.0, 0.5)
    idx = torch.randint(0, 50, (4, 6))
    t = torch.randint(0, 50, (4, 6))
    t[:, :2] = -1
    logp, ent = m.token_log_probs(idx, t, entropy=True)
    q = torch.log_softmax(m(idx), -1)
    want = q.gather(2, t.clamp(min=0)[..., None])[..., 0] * (t >= 0)
    assert torch.allclose(logp, want, atol=1e-5) and logp.shape == ent.shape == (4, 6)
    r = m.policy_loss(idx, t, logp.detach(), torch.randn(4, 6), ref_log_probs=logp.detach(), kl_coef=0.1)
    assert abs(r.kl.item()) < 1e-6 and r.clip_fraction.item() == 0
    s = m.preference_loss(idx, t, beta=0.5)
    assert torch.allclose(s.log_probs, logp.sum(1), atol=1e-4)
    for loss in (r.loss, s.loss):
        grads = torch.autograd.grad(loss, [m.lm_head.weight, m.transformer.wte.weight], retain_graph=True)
        assert all(torch.isfinite(g).all() and g.abs().sum() > 0 for g in grads)


def test_refusals():
    x, t, (row, *_) = case(8, 6)
    with pytest.raises(ValueError, match="one target"):
        softcap_log_probs(x, t[:4], VOCAB)
    with pytest.raises(ValueError, match="vocab"):
        softcap_log_probs(x, t, COLS + 1)
    with pytest.raises(ValueError, match="row value"):
        policy_loss(x, t, row[:3], row, VOCAB)
    with pytest.raises(ValueError, match="clip"):
        policy_loss(x, t, row, row, VOCAB, clip=1.5)
    with pytest.raises(ValueError, match="2 P, T"):
        preference_loss(x, t, VOCAB)
    with pytest.raises(ValueError, match="even number"):
        preference_loss(x.view(1, 8, COLS), t.view(1, 8), VOCAB)
    with pytest.raises(ValueError, match="ref_log_probs"):
        preference_loss(x.view(4, 2, COLS), t.view(4, 2), VOCAB, ref_log_probs=row[:3])
    with pytest.raises(ValueError, match="label_smoothing"):
        preference_loss(x.view(4, 2, COLS), t.view(4, 2), VOCAB, label_smoothing=2.0)
    with pytest.raises(ValueError, match="int32"):
        preference_loss(x, t, VOCAB, cu_seqlens=torch.tensor([0, 4, 8]))
    with pytest.raises(ValueError, match="within the rows"):
        preference_loss(x, t, VOCAB, cu_seqlens=torch.tensor([0, 4, 9], dtype=torch.int32))
    for call in (lambda: ops.softcap_log_probs_forward(x.bfloat16(), t, VOCAB, CAP),
                 lambda: ops.policy_rows(t, row.float(), row.float(), row.float(), None, None, 0.8, 1.2, 0.0)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            call()


@pytest.mark.skipif(not _lib.is_built(), reason="library not built")
def test_c_abi_refuses_bad_calls_without_gpu():
    lib = _lib.load()
    ptr = ctypes.c_void_p(1 << 20)

    def refused(rc, words):
        assert rc != 0 and words in lib.kda_last_error().decode()

    fwd, bwd = lib.kda_softcap_log_probs_forward, lib.kda_softcap_log_probs_backward
    refused(fwd(4, 37, 36, 15.0, ptr, ptr, -1, ptr, None, ptr, None, None), "stride")
    refused(fwd(4, 37, 44, 15.0, ptr, ptr, -1, ptr, None, ptr, None, None), "stride")
    refused(fwd(4, 37, 40, 0.0, ptr, ptr, -1, ptr, None, ptr, None, None), "softcap")
    refused(fwd(4, 37, 40, 15.0, ptr, ptr, -1, None, None, ptr, None, None), "null output")
    refused(fwd(4, 37, 40, 15.0, ctypes.c_void_p(8), ptr, -1, ptr, None, ptr, None, None), "aligned")
    refused(bwd(4, 37, 40, 15.0, ptr, ptr, -1, ptr, None, None, None, None, ptr, None), "null")
    refused(bwd(4, 37, 40, 15.0, ptr, ptr, -1, ptr, None, ptr, ptr, None, ptr, None), "entropies")
    rows = lib.kda_policy_rows
    refused(rows(4, ptr, -1, ptr, ptr, ptr, None, None, 1.1, 1.2, 0.0, ptr, ptr, None, None), "hold 1")
    refused(rows(4, ptr, -1, ptr, None, ptr, None, None, 0.8, 1.2, 0.0, ptr, ptr, None, None), "null")
    pairs = lib.kda_preference_pairs
    refused(pairs(9, 2, 2, None, ptr, -1, ptr, None, 0.1, 0.0, 0, ptr, ptr, ptr, None, ptr, None), "seq_len")
    refused(pairs(8, 2, 0, None, ptr, -1, ptr, None, 0.1, 0.0, 0, ptr, ptr, ptr, None, ptr, None), "pairs")
    refused(pairs(8, 2, 2, None, ptr, -1, ptr, None, 0.1, 1.5, 0, ptr, ptr, ptr, None, ptr, None), "label_smoothing")
    refused(pairs(8, 2, 2, None, ptr, -1, ptr, None, 0.1, 0.0, 0, ptr, ptr, ptr, None, None, None), "null")
