"""GPU parity of the post-training losses (log-probabilities, policy and preference loss) with the
float64 oracle.

Tolerances.  A table entry e^z has z = cap tanh(l / cap) from f32 functions of about 2 ulp: |dz| <=
cap 2^-22, and e^z itself 2^-22 more.  A row of V columns is summed by 64 lanes, V / 512 adds in a
row and 16 more in a vector and across lanes: (V / 512 + 16) 2^-24 relative.  So a log-probability is
off by EPS = cap 2^-22 + 2^-22 + (V / 512 + 16) 2^-24 and its own f32 rounding 2^-24 |logp|; an
entropy (sums of p z with |z| <= cap) by 2 cap EPS.  A gradient is rounded to bf16, 2^-8 of the
value, after an error of EPS in p, 2^-21 in 1 - tanh^2 and 2 cap EPS in z - lse + H.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import post_training as P

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from experiment_swa_kda_amd.model import GPT, GPTConfig, policy_loss, preference_loss, softcap_log_probs

CAP = 15.0


def eps_of(vocab, cap=CAP):
    return (cap + 1) * 2.0 ** -22 + (vocab / 512 + 16) * 2.0 ** -24


def n(t):
    return None if t is None else t.detach().double().cpu().numpy()


def case(rows, vocab, cols, seed, scale=3.0, ignore_every=5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * scale).bfloat16()
    t = torch.randint(0, vocab, (rows,), generator=g)
    if ignore_every:
        t[::ignore_every] = -1
    row = [torch.randn(rows, generator=g) for _ in range(4)]
    return x, t, row


def check_rows(logp, ent, x, t, vocab, cap=CAP):
    e_logp, e_ent, _, _ = P.rows(n(x), t.tolist(), vocab, cap)
    eps = eps_of(vocab, cap)
    assert np.all(np.abs(n(logp) - e_logp) <= (t.numpy() >= 0) * (eps + 2.0 ** -23 * np.abs(e_logp)))
    if ent is not None:
        assert np.all(np.abs(n(ent) - e_ent) <= 2 * cap * eps + 2.0 ** -23 * np.abs(e_ent))


def check_grad(grad, x, t, vocab, g, h=None, cap=CAP, slack=0.0):
    """``slack``: relative error of the row gradients g that the caller allows."""
    want = P.logit_grad(n(x), t.tolist(), vocab, cap, g, h)
    _, ent, z, p = P.rows(n(x), t.tolist(), vocab, cap)
    eps = eps_of(vocab, cap) + slack
    one = np.zeros_like(p)
    for r, v in enumerate(t.tolist()):
        if v >= 0:
            one[r, v] = 1
    size = np.abs(g)[:, None] * (p + one)
    if h is not None:
        size = size + np.abs(h)[:, None] * p * (2 * cap + np.abs(np.log(p) + ent[:, None]))
    size = np.pad(size, ((0, 0), (0, want.shape[1] - vocab)))
    off = np.abs(n(grad) - want)
    assert np.all(off <= 2.0 ** -8 * 1.01 * np.abs(want) + 2 * (eps + 2.0 ** -21) * size + 1e-38)
    assert not n(grad)[:, vocab:].any() and not n(grad)[t.numpy() < 0].any()


SHAPES = [
    (1, 8, 8), (1, 1, 8), (3, 7, 8),          # one vector, padding in it
    (300, 1000, 1024),                        # less than a chunk
    (65, 4097, 4104), (33, 8003, 8064),       # a chunk and a ragged rest
    (5, 32768, 32768), (7, 32000, 32000),
    (3, 70001, 70016),                        # more than the registers of a workgroup hold
    (2100, 264, 264),                         # more rows than waves of some grids
]


@pytest.mark.parametrize("rows,vocab,cols", SHAPES)
@pytest.mark.parametrize("entropy", [False, True])
def test_log_probs_match_oracle(rows, vocab, cols, entropy):
    x, t, (g, h, *_) = case(rows, vocab, cols, rows + vocab)
    leaf = x.cuda().requires_grad_()
    out = softcap_log_probs(leaf, t.cuda(), vocab, CAP, entropy=entropy)
    logp, ent = out if entropy else (out, None)
    check_rows(logp, ent, x, t, vocab)
    if entropy:
        (grad,) = torch.autograd.grad([logp, ent], leaf, [g.cuda(), h.cuda()])
        check_grad(grad, x, t, vocab, n(g), n(h))
    else:
        (grad,) = torch.autograd.grad(logp, leaf, g.cuda())
        check_grad(grad, x, t, vocab, n(g))
    with torch.no_grad():
        again = softcap_log_probs(x.cuda(), t.cuda(), vocab, CAP, entropy=entropy)
    assert torch.equal(again[0] if entropy else again, logp)


def test_log_probs_leading_shape_strides_and_partial_gradients():
    x, t, (g, h, *_) = case(24, 500, 512, 3)
    wide = torch.zeros(4, 6, 1024, dtype=torch.bfloat16, device="cuda")
    wide[..., 8:520] = x.view(4, 6, 512).cuda()
    view = wide[..., 8:520].requires_grad_()  # rows of another stride, not at the storage's start
    logp, ent = softcap_log_probs(view, t.view(4, 6).cuda(), 500, CAP, entropy=True)
    assert logp.shape == ent.shape == (4, 6)
    check_rows(logp.flatten(), ent.flatten(), x, t, 500)
    (only_ent,) = torch.autograd.grad(ent, view, h.view(4, 6).cuda(), retain_graph=True)
    check_grad(only_ent.reshape(24, 512), x, t, 500, np.zeros(24), n(h))
    (one,) = torch.autograd.grad(logp[1, 3], view)  # every other row's gradient is zero
    check_grad(one.reshape(24, 512), x, t, 500, np.eye(24)[9])


@pytest.mark.parametrize("cap", [15.0, 60.0])
def test_log_probs_extreme_logits(cap):
    """Zeros, denormals, huge and infinite logits, the target's too: tanh's limits."""
    x, t, (g, *_) = case(24, 8190, 8192, 11, ignore_every=0)
    special = torch.tensor([0.0, -0.0, 1e-40, 3e-8, 600.0, -600.0, 3e38, float("inf"), float("-inf"), -511.0])
    for r in range(24):
        x[r, r:8000:97] = special[torch.arange(len(x[r, r:8000:97])) % 10].bfloat16()
        x[r, t[r]] = special[r % 10].bfloat16()
    leaf = x.cuda().requires_grad_()
    logp = softcap_log_probs(leaf, t.cuda(), 8190, cap)
    check_rows(logp, None, x, t, 8190, cap)
    (grad,) = torch.autograd.grad(logp, leaf, g.cuda())
    check_grad(grad, x, t, 8190, n(g), cap=cap)


@pytest.mark.parametrize("vocab,cols", [(8192, 8192), (8003, 8064), (40000, 40000)])
def test_nan_stays_in_its_row_and_masked_places_are_not_read(vocab, cols):
    x, t, row = case(16, vocab, cols, 5)
    clean = x.clone()
    x[t < 0] = float("nan")               # rows without a target
    x[:, vocab:] = float("nan")           # padding columns
    x[7, vocab - 1] = float("nan")        # a row that counts
    t[8] = vocab                          # a target that is none
    leaf = x.cuda().requires_grad_()
    logp, ent = softcap_log_probs(leaf, t.cuda(), vocab, CAP, entropy=True)
    (grad,) = torch.autograd.grad([logp, ent], leaf, [row[0].cuda(), row[1].cuda()])
    bad = torch.zeros(16, dtype=torch.bool)
    bad[[7, 8]] = True
    assert torch.isnan(logp.cpu()[bad]).all() and torch.isnan(grad.cpu()[bad][:, :vocab]).all()
    t2 = torch.where(bad, -1, t)
    check_rows(logp.cpu()[~bad], ent.cpu()[~bad], clean[~bad], t2[~bad], vocab)
    check_grad(grad.cpu()[~bad], clean[~bad], t2[~bad], vocab, n(row[0])[~bad.numpy()], n(row[1])[~bad.numpy()])
    # through the losses: a NaN row that does not count leaves nothing behind
    t2 = t2.cuda()
    leaf = x.cuda().requires_grad_()
    r = policy_loss(leaf, t2, logp.detach().nan_to_num(), row[0].cuda(), vocab, CAP)
    (grad,) = torch.autograd.grad(r.loss, leaf)
    assert torch.isfinite(r.loss) and torch.isfinite(grad).all()


def policy_case(rows, vocab, cols, seed, **kw):
    """Ratios on both sides of the clipping borders, none within 1e-3 of one (a rounding error
    of the log-probability would pick the side)."""
    x, t, (noise, adv, ref, w) = case(rows, vocab, cols, seed, **kw)
    logp = P.rows(n(x), t.tolist(), vocab, CAP)[0]
    noise = (0.2 * noise).double()
    for border in np.log([0.85, 1.25]):
        noise = torch.where((noise - border).abs() < 1e-3, border + 2e-3, noise)
    old = (torch.from_numpy(logp) - noise).float()
    return x, t, logp, old, adv, (torch.from_numpy(logp) + 0.3 * ref.double()).float(), w.abs()


@pytest.mark.parametrize("rows,vocab,cols", SHAPES)
@pytest.mark.parametrize("weighted,with_ref", [(False, True), (True, False)])
def test_policy_loss_matches_oracle(rows, vocab, cols, weighted, with_ref):
    x, t, logp, old, adv, ref, w = policy_case(rows, vocab, cols, rows + vocab, ignore_every=5 if rows > 1 else 0)
    w = w / rows if weighted else None
    ref = ref if with_ref else None
    leaf = x.cuda().requires_grad_()
    cuda = [None if v is None else v.cuda() for v in (old, adv, ref, w)]
    opts = dict(ref_log_probs=cuda[2], clip=0.15, clip_high=0.25, kl_coef=0.1, weights=cuda[3])
    r = policy_loss(leaf, t.cuda(), cuda[0], cuda[1], vocab, CAP, **opts)
    loss, kl, share, slope = P.policy(logp, t.tolist(), n(old), n(adv), n(ref), n(w), 0.85, 1.25, 0.1)
    check_rows(r.log_probs, None, x, t, vocab)
    # a row's terms move by |slope| (<= rho |A| + c |e^d - 1|) times the log-probability's error, then f32 rounding
    _, _, _, unit = P.policy(logp, t.tolist(), n(old), n(adv), n(ref), np.ones(rows), 0.0, 99.0, 0.1)
    off = eps_of(vocab) + 2.0 ** -23 * np.abs(logp).max() + 2.0 ** -21
    total = np.ones(rows) / max(1, int((t >= 0).sum())) if w is None else n(w)
    room = off * np.sum(total * (np.abs(unit) + np.abs(n(adv)) * 2 + 1)) + 1e-7
    assert abs(r.loss.item() - loss) <= room and abs(r.kl.item() - kl) <= room
    assert abs(r.clip_fraction.item() - share) <= 1e-6 * max(1.0, total.sum())
    # the gradient is formed for an upstream gradient of 1, rounded to bf16, v (1 + a) with |a| <= 2^-8, and
    # then times 2.5 rounded again, 2.5 v (1 + a) (1 + b): off by up to 2 2^-8 + 2^-16, two half-steps; formed
    # for 2.5 at once, or in the backward, by one
    (grad,) = torch.autograd.grad(2.5 * r.loss, leaf)
    grads = [(grad, 2)]
    for expected in (2.5, None):
        again = policy_loss(leaf, t.cuda(), cuda[0], cuda[1], vocab, CAP, expected_grad=expected, **opts)
        assert abs(again.loss.item() - r.loss.item()) <= 1e-6 * max(1.0, abs(loss))
        grads.append((torch.autograd.grad(2.5 * again.loss, leaf)[0], 1))
    # the slope's own error: that of the ratio and of e^d - 1, relative to |rho A| + c e^d
    ratio = np.exp(logp - n(old))
    size = total * (np.abs(ratio * n(adv)) + (0 if ref is None else 0.1 * np.exp(n(ref) - logp)))
    want = P.logit_grad(n(x), t.tolist(), vocab, CAP, 2.5 * slope)
    _, _, z, p = P.rows(n(x), t.tolist(), vocab, CAP)
    one = np.zeros_like(p)
    one[np.flatnonzero(t >= 0), t[t >= 0].numpy()] = 1
    for grad, roundings in grads:
        room = roundings * 2.0 ** -8 * 1.01 * np.abs(want[:, :vocab]) + \
            2.5 * 2 * (size[:, None] * off + np.abs(slope)[:, None] * off) * (p + one)
        assert np.all(np.abs(n(grad)[:, :vocab] - want[:, :vocab]) <= room + 1e-38)
        assert not n(grad)[:, vocab:].any() and not n(grad)[t.numpy() < 0].any()
    with torch.no_grad():
        plain = policy_loss(x.cuda(), t.cuda(), cuda[0], cuda[1], vocab, CAP, **opts)
    assert abs(plain.loss.item() - loss) <= 1e-4 * max(1, abs(loss))


def test_policy_loss_of_no_rows_and_of_no_weight():
    x, t, (old, adv, *_) = case(6, 100, 104, 2)
    none = torch.full_like(t, -1).cuda()
    leaf = x.cuda().requires_grad_()
    r = policy_loss(leaf, none, old.cuda(), adv.cuda(), 100)
    assert torch.isnan(r.loss)  # the mean of nothing, as the cross entropy's
    (grad,) = torch.autograd.grad(r.loss, leaf)
    assert not grad.any()
    r = policy_loss(leaf, t.cuda(), old.cuda(), adv.cuda(), 100, weights=torch.zeros(6, device="cuda"))
    (grad,) = torch.autograd.grad(r.loss, leaf)
    assert r.loss.item() == 0 and not grad.any()
    # no advantage and a ratio beyond f32: counts nothing
    r = policy_loss(leaf, t.cuda(), torch.full((6,), -1e4, device="cuda"), torch.zeros(6, device="cuda"), 100)
    assert r.loss.item() == 0
    empty = torch.empty(0, 104, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    nothing = torch.empty(0, device="cuda")
    assert torch.isnan(policy_loss(empty, nothing.long(), nothing, nothing, 100).loss)
    assert softcap_log_probs(empty, nothing.long(), 100).shape == (0,)


@pytest.mark.parametrize("lens,vocab,cols,packed", [
    ([4, 4], 50, 56, False), ([64] * 8, 8192, 8192, False), ([1, 300, 0, 77], 1000, 1024, True),
    ([61, 117, 1, 250, 77, 33, 128, 95], 8003, 8064, True), ([2] * 200, 264, 264, True), ([3, 2], 70001, 70016, True),
])
@pytest.mark.parametrize("average", [False, True])
def test_preference_loss_matches_oracle(lens, vocab, cols, packed, average):
    starts = np.concatenate([[0], np.cumsum(lens)])
    rows, S = int(starts[-1]) + (3 if packed else 0), len(lens)  # packed: rows behind the last sequence
    x, t, _ = case(rows, vocab, cols, rows + vocab)
    logp = P.rows(n(x), t.tolist(), vocab, CAP)[0]
    seq = P.preference(logp, t.tolist(), starts, None, 0.5, 0.1, average)[1]
    ref = torch.from_numpy(seq + np.linspace(-2, 2, S)).float()
    leaf = x.cuda().requires_grad_()
    view, tv = (leaf, t) if packed else (leaf.view(S, lens[0], cols), t.view(S, -1))
    r = preference_loss(view, tv.cuda(), vocab, CAP, beta=0.5, ref_log_probs=ref.cuda(), label_smoothing=0.1,
                        average=average, cu_seqlens=torch.tensor(starts, dtype=torch.int32).cuda() if packed else None)
    loss, seq, m, slope = P.preference(logp, t.tolist(), starts, n(ref), 0.5, 0.1, average)
    # sums of f64 rows: EPS a row, then one f32 rounding of the sum
    count = np.maximum(1, [(t[a:b] >= 0).sum() for a, b in zip(starts, starts[1:])])
    off = eps_of(vocab) * (1 if average else count)
    assert np.all(np.abs(n(r.log_probs) - seq) <= off + 2.0 ** -24 * np.abs(seq))
    off_m = 0.5 * (off * np.ones(S)).reshape(2, -1).sum(0)
    assert np.all(np.abs(n(r.margins) - m) <= off_m + 2.0 ** -24 * np.abs(m))
    assert abs(r.loss.item() - loss) <= off_m.mean() + 2.0 ** -24 * loss
    (grad,) = torch.autograd.grad(0.5 * r.loss, leaf)
    # |d slope / d margin| <= 1/4, against a slope of at least beta / P sigmoid(-|m|) less smoothing: relative to beta / P
    slack = np.max(off_m) / 4
    size = 0.5 * 0.5 / (S // 2) / (1 if not average else np.repeat(count, lens).astype(float))
    want = P.logit_grad(n(x), t.tolist(), vocab, CAP, 0.5 * slope)
    _, _, z, p = P.rows(n(x), t.tolist(), vocab, CAP)
    one = np.zeros_like(p)
    one[np.flatnonzero(t >= 0), t[t >= 0].numpy()] = 1
    size = np.concatenate([size * np.ones(int(starts[-1])), np.zeros(rows - int(starts[-1]))])
    room = 2.0 ** -8 * 1.01 * np.abs(want[:, :vocab]) + \
        (2 * eps_of(vocab) + slack + 2.0 ** -21) * 2 * size[:, None] * (p + one)
    assert np.all(np.abs(n(grad)[:, :vocab] - want[:, :vocab]) <= room + 1e-38)
    assert not n(grad)[:, vocab:].any() and not n(grad)[t.numpy() < 0].any() and not n(grad)[int(starts[-1]):].any()


def test_preference_loss_bad_bounds_are_nan_and_extreme_margins_finite():
    x, t, _ = case(12, 100, 104, 4)
    for cu in ([0, 4, 2, 6, 8], [0, 4, 8, 12, 16], [-1, 2, 4, 6, 8], [8, 6, 4, 2, 0]):
        leaf = x.cuda().requires_grad_()
        r = preference_loss(leaf, t.cuda(), 100, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        assert torch.isnan(r.loss) and torch.isnan(r.margins).all() and torch.isnan(r.log_probs).all()
    ref = torch.tensor([4e4, -4e4, -4e4, 4e4], device="cuda")
    leaf = x.cuda().requires_grad_()
    r = preference_loss(leaf.view(4, 3, 104), t.view(4, 3).cuda(), 100, beta=1.0, ref_log_probs=ref)
    (grad,) = torch.autograd.grad(r.loss, leaf)
    assert abs(r.loss.item() - 4e4) < 50 and torch.isfinite(grad).all()
    assert grad.view(4, 3, 104)[[0, 2]].any() and not grad.view(4, 3, 104)[[1, 3]].any()


def losses(x, t, old, adv, ref, vocab):
    leaf = x.detach().requires_grad_()
    logp, ent = softcap_log_probs(leaf, t, vocab, entropy=True)
    a = policy_loss(leaf, t, old, adv, vocab, ref_log_probs=ref, kl_coef=0.1)
    S = 4
    b = preference_loss(leaf.view(S, -1, x.shape[1]), t.view(S, -1), vocab)
    total = (logp * adv).sum() + 0.1 * ent.sum() + a.loss + b.loss
    return [logp, ent, *a, *b, *torch.autograd.grad(total, leaf)]


def test_losses_together_on_a_side_stream_and_replayed_from_a_graph():
    """The three operators on the same logits, eagerly, on another stream and captured: the same
    bits on every replay, with eager work and new inputs between the replays."""
    x, t, (old, adv, ref, _) = case(32, 1000, 1024, 9)
    args = [v.cuda() for v in (x, t, old - 6, adv, ref - 6)]
    want = losses(*args, 1000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = losses(*args, 1000)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    static = [v.clone() for v in args]
    with torch.cuda.graph(graph):
        out = losses(*static, 1000)
    for k in range(4):
        y = [v.cuda() for v in case(32, 1000, 1024, 20 + k)[:2]]
        static[0].copy_(y[0])
        static[1].copy_(y[1])
        graph.replay()
        torch.cuda.synchronize()
        eager = losses(y[0], y[1], *args[2:], 1000)
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k


@pytest.mark.parametrize("cols", [1024, 40000])
def test_two_captured_losses_take_turns(cols):
    """Two graphs of the same shapes, replayed on two streams: neither's workspaces are the other's."""
    sets = [[v.cuda() for v in (x, t, old - 6, adv, ref - 6)] for x, t, (old, adv, ref, _) in
            (case(32, 1000, cols, 40 + k) for k in range(2))]
    want = [[v.detach().clone() for v in losses(*a, 1000)] for a in sets]
    graphs, outs = [], []
    for a in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(losses(*a, 1000))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(3):
        for o in outs:
            for v in o:
                v.detach().zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w)), turn


@pytest.mark.parametrize("cols", [1024, 40000])
def test_policy_rows_of_weight_zero_are_not_read(cols):
    """In every form of the loss, NaN logits, advantages and old values of such rows reach nothing."""
    x, t, (old, adv, ref, w) = case(9, 1000, cols, 16, ignore_every=0)
    w = w.abs() + 0.1
    off = torch.tensor([0, 4, 8])
    w[off] = 0.0
    clean = [v.clone() for v in (x, old, adv, ref)]
    for v in (x, old, adv, ref):
        v[off] = float("nan")
    got, grads = [], []
    for values, expected in ((clean, 1.0), ((x, old, adv, ref), 1.0), ((x, old, adv, ref), None), ((x, old, adv, ref), 0.5)):
        leaf = values[0].cuda().requires_grad_()
        r = policy_loss(leaf, t.cuda(), values[1].cuda(), values[2].cuda(), 1000, ref_log_probs=values[3].cuda(), clip=1.0,
                        clip_high=9.0, kl_coef=0.1, weights=w.cuda(), expected_grad=expected)
        got.append(r)
        grads.append(torch.autograd.grad(r.loss, leaf)[0])
        with torch.no_grad():
            got.append(policy_loss(leaf, t.cuda(), values[1].cuda(), values[2].cuda(), 1000, ref_log_probs=values[3].cuda(),
                                   clip=1.0, clip_high=9.0, kl_coef=0.1, weights=w.cuda()))
    for r in got:
        assert not r.log_probs[off].any() and torch.isfinite(r.log_probs).all()
        # the same f64 terms, from sums of e^z in one order or another (EPS) and slopes of some e^9
        assert abs(r.loss.item() - got[0].loss.item()) <= 20 * eps_of(1000) * max(1.0, abs(got[0].loss.item()))
    for g in grads:
        assert not g[off].any() and torch.isfinite(g).all()
    assert torch.equal(grads[0], grads[1])


def test_entropy_gradient_of_a_target_outside_the_vocabulary():
    """Its log-probability is NaN; the row's entropy and the entropy's gradient are the row's own."""
    x, t, (_, _, _, h) = case(6, 1000, 1024, 14, ignore_every=0)
    t[2], t[4] = 1000, -7
    leaf = x.cuda().requires_grad_()
    logp, ent = softcap_log_probs(leaf, t.cuda(), 1000, entropy=True)
    assert torch.isnan(logp).tolist() == [False, False, True, False, True, False]
    (grad,) = torch.autograd.grad((ent * h.cuda()).sum(), leaf)
    inside = torch.where((t < 0) | (t >= 1000), 3, t)
    check_rows(logp[[0, 1, 3, 5]], None, x[[0, 1, 3, 5]], t[[0, 1, 3, 5]], 1000)
    check_grad(grad, x, inside, 1000, np.zeros(6), n(h))


@pytest.mark.parametrize("expected", [1.0, None])
def test_second_derivatives_are_refused(expected):
    """create_graph gives the same first gradient; differentiating it again is an error, not zero."""
    x, t, (old, adv, ref, _) = case(8, 1000, 1024, 17)
    leaf = x.cuda().requires_grad_()
    calls = [lambda: softcap_log_probs(leaf, t.cuda(), 1000).sum(),
             lambda: policy_loss(leaf, t.cuda(), old.cuda() - 8, adv.cuda(), 1000, expected_grad=expected).loss,
             lambda: preference_loss(leaf.view(4, 2, -1), t.cuda().view(4, 2), 1000).loss]
    for call in calls:
        (first,) = torch.autograd.grad(call(), leaf)
        (again,) = torch.autograd.grad(call(), leaf, create_graph=True)
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
            torch.autograd.grad(again.float().square().sum(), leaf)


def test_offsets_past_32_bits():
    """70000 rows of 32768 columns, 2.3e9 logits, with a few counted rows at both ends."""
    rows, vocab = 70000, 32768
    x, t, (old, adv, _, _) = case(8, vocab, vocab, 15, ignore_every=0)
    big = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 1, 2, 65535, 65536, 69997, 69998, 69999], device="cuda")
    big[some] = x.cuda()
    targets = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    targets[some] = t.cuda()
    leaf = big.requires_grad_()
    logp, ent = softcap_log_probs(leaf, targets, vocab, entropy=True)
    check_rows(logp[some], ent[some], x, t, vocab)
    (grad,) = torch.autograd.grad(logp.sum(), leaf)
    check_grad(grad[some], x, t, vocab, np.ones(8))
    grad[some] = 0
    assert not grad.any()
    del grad
    full = [torch.zeros(rows, device="cuda").index_put_((some,), v.cuda()) for v in (old - 10, adv)]
    out = policy_loss(leaf, targets, full[0], full[1], vocab, clip=1.0, clip_high=1e30)
    assert torch.equal(out.log_probs[some] != 0, torch.ones(8, dtype=torch.bool, device="cuda"))
    check_rows(out.log_probs[some], None, x, t, vocab)
    (grad,) = torch.autograd.grad(out.loss, leaf)
    e_logp = P.rows(n(x), t.tolist(), vocab, CAP)[0]
    # the slope's error: that of e^(logp - old), EPS and the roundings of logp and the difference
    slack = 4 * (eps_of(vocab) + 2.0 ** -23 * float(np.abs(e_logp).max() + 16))
    check_grad(grad[some], x, t, vocab, -np.exp(e_logp - n(old - 10)) * n(adv) / 8, slack=slack)
    grad[some] = 0
    assert not grad.any()


def test_decoder_trains_on_the_losses():
    """The decoder's own methods: loss values those of its logits, gradients those of the plain
    loss on them, for every parameter."""
    torch.manual_seed(0)
    m = GPT(GPTConfig(sequence_len=64, vocab_size=1000, n_layer=2, n_head=2, n_embd=128)).cuda()
    m.init_weights()
    torch.nn.init.normal_(m.lm_head.weight, 0.0, 0.3)
    for b in m.transformer.h:
        torch.nn.init.normal_(b.mlp.c_proj.weight, 0.0, 0.02)
        torch.nn.init.normal_(b.attn.o_proj.weight, 0.0, 0.02)
    idx = torch.randint(0, 1000, (4, 33), device="cuda")
    x, t = idx[:, :-1].contiguous(), idx[:, 1:].clone()
    t[:, :7] = -1
    adv = torch.randn(4, 32, device="cuda")
    with torch.no_grad():
        old = m.token_log_probs(x, t)
        want = torch.log_softmax(m(x).double(), -1).gather(2, t.clamp(min=0)[..., None])[..., 0] * (t >= 0)
    # bf16 logits both, f32 cap and softmax: EPS of the kernel and as much of torch's f32 logits
    assert (old - want).abs().max().item() <= 3 * eps_of(1000) + 2e-6

    params = list(m.parameters())

    def plain(kind):
        z = 15 * torch.tanh(m._logits(x)[..., :1000].float() / 15)
        q = torch.log_softmax(z, -1).gather(2, t.clamp(min=0)[..., None])[..., 0] * (t >= 0)
        if kind == "policy":
            return (-(q - old).exp() * adv * (t >= 0)).sum() / (t >= 0).sum()
        s = q.sum(1)
        return -torch.nn.functional.logsigmoid(0.3 * (s[:2] - s[2:])).mean()

    for kind, loss in (("policy", m.policy_loss(x, t, old, adv).loss), ("pref", m.preference_loss(x, t, beta=0.3).loss)):
        got = torch.autograd.grad(loss, params)
        ref = plain(kind)
        assert abs(loss.item() - ref.item()) <= 1e-4 * max(1.0, abs(ref.item()))
        for a, b in zip(got, torch.autograd.grad(ref, params)):
            # the same bf16 backward behind both, fed logit gradients that each are bf16 roundings
            # (2^-8) of the same values: a few such roundings' worth of the gradient's norm
            assert (a.double() - b.double()).norm() <= 0.02 * b.double().norm() + 1e-9
