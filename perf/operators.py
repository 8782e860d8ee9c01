"""The post-training operators whose speed counts: token log-probabilities, the two losses that
are built on them, and projections with low-rank adapters of many requests, each as a plain
form of elementary torch operations and as the call that a user of this package makes.

Every case is a dict with a ``kind``:

* ``logp``    ``softcap_log_probs``: scoring (``grad`` false) or with its gradient; ``entropy``
              adds the rows' entropies;
* ``policy``  ``policy_loss``: the clipped policy loss and its logit gradient, ``ref`` adds the KL
              term against a reference policy;
* ``pref``    ``preference_loss``: the paired loss and its logit gradient, over a padded batch or
              (``lens``) over packed sequences;
* ``lora``    ``lora_linear``: a shared projection with every request's own adapter, at inference
              or (``grad``) with the gradients of the input and of the adapters.
"""

from __future__ import annotations

import math

import torch

own = False

CAP = 15.0
IGNORE = -1
CLIP, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.05
BETA, SMOOTHING = 0.1, 0.05


def _logp(name, rows, vocab, stride, entropy=False, grad=False):
    c = {"kind": "logp", "rows": rows, "vocab": vocab, "stride": stride, "entropy": entropy, "grad": grad}
    return {"name": name, **c} if name else c


def _policy(name, rows, vocab, stride, ref=True):
    c = {"kind": "policy", "rows": rows, "vocab": vocab, "stride": stride, "ref": ref}
    return {"name": name, **c} if name else c


def _pref(name, pairs, T, vocab, stride, lens="", average=False):
    c = {"kind": "pref", "pairs": pairs, "T": T, "vocab": vocab, "stride": stride, "lens": lens, "average": average}
    return {"name": name, **c} if name else c


def _lora(name, B, T, K, N, R, n, grad=False, per_token=False):
    c = {"kind": "lora", "B": B, "T": T, "K": K, "N": N, "R": R, "n": n, "grad": grad, "per_token": per_token}
    return {"name": name, **c} if name else c


def listed():
    return [
        # scoring the few tokens of a short continuation under the trainer's vocabulary: latency
        _logp("logp_48x32768", 48, 32768, 32768),
        # scoring a batch of rollouts under the reference or the behaviour policy
        _logp("logp_8192x32768", 8192, 32768, 32768),
        # a training step on log-probabilities with an entropy bonus; a vocabulary with padding columns
        _logp("logp_grad_3001x50000", 3001, 50000, 50048, entropy=True, grad=True),
        # the policy step of a tiny model, a ragged vocabulary, no reference policy: launches count
        _policy("policy_500x8003", 500, 8003, 8064, ref=False),
        # the policy step over a micro-batch of the 6-layer trainer
        _policy("policy_8192x32768", 8192, 32768, 32768),
        # preference pairs of uneven lengths, packed, from a small vocabulary
        _pref("pref_packed_4x8192", 4, 0, 8192, 8192, lens="61,117,1,250,77,33,128,95"),
        # a micro-batch of 4 pairs of padded sequences under the trainer's vocabulary
        _pref("pref_4x1024x32768", 4, 1024, 32768, 32768),
        # one token for each of 8 requests through the decoder's MLP projection: latency
        _lora("lora_step_b8_384_1536_r16", 8, 1, 384, 1536, 16, 8),
        # one token for each of 64 requests, every one with an adapter of its own, a wider model
        _lora("lora_step_b64_2048_2048_r16", 64, 1, 2048, 2048, 16, 64),
        # prompts of 8 requests through the decoder's MLP projection
        _lora("lora_prompt_b8_t1024_384_1536_r16", 8, 1024, 384, 1536, 16, 8),
        # training two adapters on a micro-batch of the trainer, the MLP's second projection
        _lora("lora_train_b2_t4096_1536_384_r16", 2, 4096, 1536, 384, 16, 2, grad=True),
        # training adapters of a large rank in a wide model, sequences of an odd length
        _lora("lora_train_b7_t1111_4096_2048_r64", 7, 1111, 4096, 2048, 64, 3, grad=True),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# what the largest listed cases take: logits of one call, multiply-adds of one projection
MOST_LOGITS, MOST_PRODUCTS = 8192 * 32768, 7 * 1111 * 4096 * 2048


def _vocab(rng):
    vocab = rng.choice([_log(rng, 1000, 65000), 4096, 8192, 32000, 32768, 65536])
    return vocab, vocab + (-vocab) % rng.choice([8, 64])


def draw(rng):
    kind = rng.choice(["logp", "logp", "policy", "policy", "pref", "pref", "lora", "lora", "step", "train"])
    if kind in ("logp", "policy", "pref"):
        vocab, stride = _vocab(rng)
        most = MOST_LOGITS // stride
        if kind == "logp":
            return _logp("", _log(rng, 16, min(most, 16384)), vocab, stride, rng.random() < 0.5, rng.random() < 0.5)
        if kind == "policy":
            return _policy("", _log(rng, 16, min(most, 16384)), vocab, stride, rng.random() < 0.7)
        pairs = rng.randint(1, 8)
        if rng.random() < 0.5:
            lens = [_log(rng, 1, min(1500, most // (2 * pairs))) for _ in range(2 * pairs)]
            return _pref("", pairs, 0, vocab, stride, ",".join(map(str, lens)), rng.random() < 0.3)
        return _pref("", pairs, _log(rng, 8, min(2048, most // (2 * pairs))), vocab, stride, "", rng.random() < 0.3)
    R, n = rng.choice([8, 16, 16, 32, 64]), rng.randint(1, 16)
    K, N = (8 * _log(rng, 32, 512) for _ in range(2))
    if kind == "step":
        return _lora("", _log(rng, 1, 256), 1, K, N, R, rng.randint(1, 64))
    while True:
        B, T = rng.randint(1, 16), _log(rng, 2, 4096)
        if B * T * K * N <= MOST_PRODUCTS and B * T <= 16384:
            return _lora("", B, T, K, N, R, n, kind == "train", rng.random() < 0.3)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(c):
    """Tokens of every sequence of a preference case, chosen sequences first."""
    return [int(n) for n in c["lens"].split(",")] if c["lens"] else [c["T"]] * (2 * c["pairs"])


def _rows(c):
    return sum(_lens(c)) if c["kind"] == "pref" else c["rows"]


def _counted(c):
    """Rows with a target: one in eight is a prompt's or padding."""
    return _rows(c) - _rows(c) // 8


def _row_log_probs(logits, targets, vocab):
    """Row log-probabilities in 64 bits, a block of rows at a time (for inputs that go with them)."""
    out = []
    for i in range(0, logits.shape[0], 1024):
        z = CAP * torch.tanh(logits[i:i + 1024, :vocab].double() / CAP)
        t = targets[i:i + 1024]
        picked = z.gather(1, t.clamp(min=0)[:, None])[:, 0]
        out.append(torch.where(t == IGNORE, 0.0, picked - torch.logsumexp(z, 1)))
    return torch.cat(out)


def _prepare_loss(c, g):
    rows, vocab = _rows(c), c["vocab"]
    s = {"kind": c["kind"], "vocab": vocab}
    s["logits"] = (torch.randn(rows, c["stride"], device="cuda", generator=g) * 2.5).bfloat16()
    targets = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    targets[torch.randperm(rows, device="cuda", generator=g)[:rows // 8]] = IGNORE
    s["targets"] = targets
    noise = torch.randn(2, rows, device="cuda", generator=g, dtype=torch.float64)
    if c["kind"] == "logp":
        s["entropy"], s["grad"] = c["entropy"], c["grad"]
        s["g"], s["h"] = (noise / rows).float()
        return s
    logp = _row_log_probs(s["logits"], targets, vocab)
    if c["kind"] == "policy":
        # ratios around 1 as after a few updates on the same rollouts, some of them clipped; none within
        # 1e-3 of a clipping border, where the rounding of a log-probability would pick the side
        ratio = 0.15 * noise[0]
        for border in (math.log(1 - CLIP), math.log(1 + CLIP_HIGH)):
            ratio = torch.where((ratio - border).abs() < 1e-3, border + 2e-3, ratio)
        s["old"] = (logp - ratio).float()
        s["adv"] = torch.randn(rows, device="cuda", generator=g)
        s["ref"] = (logp + 0.3 * noise[1]).float() if c["ref"] else None
        return s
    lens = _lens(c)
    n = 2 * c["pairs"]
    s["average"], s["packed"] = c["average"], bool(c["lens"])
    s["starts"] = torch.tensor([0, *lens], device="cuda").cumsum(0).int()
    s["seq"] = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(lens, device="cuda"))
    s["beta"] = 2.0 if c["average"] else BETA
    sums = torch.zeros(n, device="cuda", dtype=torch.float64)
    count = torch.zeros_like(sums)
    sums = sums.index_add(0, s["seq"], logp)
    count = count.index_add(0, s["seq"], (targets != IGNORE).double())
    if c["average"]:
        sums = sums / count.clamp(min=1)
    # margins of 0.3 to 1.5 either way, as in the middle of a training run
    margin = 0.3 + 1.2 * torch.rand(c["pairs"], device="cuda", generator=g, dtype=torch.float64)
    margin = torch.where(torch.rand(c["pairs"], device="cuda", generator=g) < 0.5, -margin, margin)
    s["ref"] = (sums - torch.cat([margin, -margin]) / (2 * s["beta"])).float()
    if s["packed"]:
        return s
    s["logits"], s["targets"] = s["logits"].view(n, c["T"], -1), targets.view(n, c["T"])
    return s


def _prepare_lora(c, g):
    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    B, T, K, N, R, n = (c[k] for k in ("B", "T", "K", "N", "R", "n"))
    kind = torch.float32 if c["grad"] else torch.bfloat16  # trained adapters are f32 masters
    s = {"kind": "lora", "grad": c["grad"], "x": normal(B, T, K).bfloat16(), "w": (normal(N, K) * K ** -0.5).bfloat16(),
         "a": (normal(n, R, K) * K ** -0.5).to(kind), "b": (normal(n, N, R) * 0.5 * R ** -0.5).to(kind),
         "scale": 0.5 + torch.rand(n, device="cuda", generator=g), "dy": normal(B, T, N).bfloat16()}
    if c["per_token"]:  # several requests packed in a row: runs of tokens of one adapter
        cuts = torch.randint(0, T, (7,), device="cuda", generator=g).sort()[0]
        run = torch.searchsorted(cuts, torch.arange(T, device="cuda"), right=True)
        s["ids"] = torch.randint(-1, n, (B, 8), device="cuda", generator=g)[:, run].int()
    else:
        s["ids"] = torch.randint(-1, n, (B,), device="cuda", generator=g).int()
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_lora(case, g) if case["kind"] == "lora" else _prepare_loss(case, g)


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _plain_rows(logits, targets, vocab):
    """tanh, z and lse of every row, its target's log-probability (0 without a target), the mask."""
    t = torch.tanh(logits[:, :vocab].float() / CAP)
    z = CAP * t
    lse = z.exp().sum(1).log()
    keep = targets != IGNORE
    logp = torch.where(keep, z.gather(1, targets.clamp(min=0)[:, None])[:, 0] - lse, 0.0)
    return t, z, lse, logp, keep


def _plain_grad(t, z, lse, targets, keep, stride, g, h=None, entropy=None):
    """The logit gradient for the rows' upstream gradients g of logp and h of the entropy."""
    p = (z - lse[:, None]).exp()
    g = torch.where(keep, g, 0.0)
    d = -p * g[:, None]
    d = d.scatter_add(1, targets.clamp(min=0)[:, None], g[:, None])
    if h is not None:
        d = d - torch.where(keep, h, 0.0)[:, None] * p * (z - lse[:, None] + entropy[:, None])
    d = (d * (1 - t * t)).bfloat16()
    return torch.cat([d, d.new_zeros(d.shape[0], stride - d.shape[1])], 1)


def _plain_logp(s):
    targets, stride = s["targets"], s["logits"].shape[1]
    t, z, lse, logp, keep = _plain_rows(s["logits"], targets, s["vocab"])
    out = [logp]
    if s["entropy"]:
        out.append(torch.where(keep, lse - ((z - lse[:, None]).exp() * z).sum(1), 0.0))
    if s["grad"]:
        more = (s["h"], out[1]) if s["entropy"] else ()
        out.append(_plain_grad(t, z, lse, targets, keep, stride, s["g"], *more))
    return out


def _plain_policy(s):
    targets, stride = s["targets"], s["logits"].shape[1]
    t, z, lse, logp, keep = _plain_rows(s["logits"], targets, s["vocab"])
    w = keep.float() / keep.sum()
    adv = s["adv"]
    ratio = (logp - s["old"]).exp()
    free, held = ratio * adv, ratio.clamp(1 - CLIP, 1 + CLIP_HIGH) * adv
    clipped = held < free
    loss = -torch.minimum(free, held)
    g = torch.where(clipped, 0.0, -free)
    out = []
    if s["ref"] is not None:
        d = s["ref"] - logp
        kl = torch.expm1(d) - d
        loss = loss + KL_COEF * kl
        g = g - KL_COEF * torch.expm1(d)
        out.append((w * kl).sum())
    return [(w * loss).sum(), logp, (w * clipped).sum(), *out,
            _plain_grad(t, z, lse, targets, keep, stride, w * g)]


def _plain_pref(s):
    logits, targets = s["logits"].flatten(0, -2), s["targets"].flatten()
    t, z, lse, logp, keep = _plain_rows(logits, targets, s["vocab"])
    n = s["ref"].shape[0]
    member = torch.arange(n, device=logits.device)[:, None] == s["seq"][None]
    sums = torch.where(member, logp.double(), 0.0).sum(1)  # thousands of terms, and then differences of them
    per = 1.0 / (member & keep).sum(1).clamp(min=1) if s["average"] else torch.ones_like(sums)
    sums = sums * per
    gain = sums - s["ref"].double()
    margin = s["beta"] * (gain[:n // 2] - gain[n // 2:])
    up, down = torch.log1p((-margin).exp()), torch.log1p(margin.exp())
    loss = ((1 - SMOOTHING) * up + SMOOTHING * down).mean()
    dm = s["beta"] / margin.shape[0] * (SMOOTHING - torch.sigmoid(-margin))
    g = (torch.cat([dm, -dm]) * per)[s["seq"]].float()
    grad = _plain_grad(t, z, lse, targets, keep, logits.shape[1], g)
    return [loss.float(), sums.float(), margin.float(), grad.view(s["logits"].shape)]


def _plain_lora(s):
    x, w, dy = s["x"].flatten(0, 1).float(), s["w"].float(), s["dy"].flatten(0, 1).float()
    n, R, K = s["a"].shape
    M, N = dy.shape
    # the adapters of all requests side by side; f32 masters are used as the weights of Linear are, rounded to bf16
    a = s["a"].bfloat16().float().reshape(n * R, K)
    b = s["b"].bfloat16().float().transpose(1, 2).reshape(n * R, N)
    ids = s["ids"] if s["ids"].ndim == 2 else s["ids"][:, None].expand(s["x"].shape[:2])
    on = (ids.reshape(M, 1) == torch.arange(n, device=x.device)).float() * s["scale"]
    on = on[:, :, None].expand(M, n, R).reshape(M, n * R)
    u = (x @ a.t().contiguous()) * on
    y = (x @ w.t().contiguous() + u @ b).bfloat16().view(*s["x"].shape[:2], N)
    if not s["grad"]:
        return [y]
    t = (dy @ b.t().contiguous()) * on
    dx = (dy @ w + t @ a).bfloat16().view(s["x"].shape)
    da = (t.t().contiguous() @ x).view(n, R, K)
    db = (u.t().contiguous() @ dy).view(n, R, N).transpose(1, 2)
    return [y, dx, da, db]


# ---------------------------------------------------------------------------
# the package's calls
# ---------------------------------------------------------------------------

def _own_logp(s):
    from experiment_swa_kda_amd.model import softcap_log_probs

    logits = s["logits"].detach().requires_grad_(s["grad"])
    out = softcap_log_probs(logits, s["targets"], s["vocab"], CAP, IGNORE, entropy=s["entropy"])
    out = list(out) if s["entropy"] else [out]
    if s["grad"]:
        out += torch.autograd.grad(out, logits, [s["g"], s["h"]][:len(out)])
    return out


def _own_policy(s):
    from experiment_swa_kda_amd.model import policy_loss

    logits = s["logits"].detach().requires_grad_()
    r = policy_loss(logits, s["targets"], s["old"], s["adv"], s["vocab"], CAP, IGNORE, ref_log_probs=s["ref"],
                    clip=CLIP, clip_high=CLIP_HIGH, kl_coef=KL_COEF)
    kl = [] if s["ref"] is None else [r.kl]
    return [r.loss, r.log_probs, r.clip_fraction, *kl, *torch.autograd.grad(r.loss, logits)]


def _own_pref(s):
    from experiment_swa_kda_amd.model import preference_loss

    logits = s["logits"].detach().requires_grad_()
    r = preference_loss(logits, s["targets"], s["vocab"], CAP, IGNORE, beta=s["beta"], ref_log_probs=s["ref"],
                        label_smoothing=SMOOTHING, average=s["average"],
                        cu_seqlens=s["starts"] if s["packed"] else None)
    return [r.loss, r.log_probs, r.margins, *torch.autograd.grad(r.loss, logits)]


def _own_lora(s):
    from experiment_swa_kda_amd.kda import lora_linear

    if not s["grad"]:
        return [lora_linear(s["x"], s["w"], s["a"], s["b"], s["ids"], s["scale"])]
    leaves = [s[k].detach().requires_grad_() for k in ("x", "a", "b")]
    y = lora_linear(leaves[0], s["w"], leaves[1], leaves[2], s["ids"], s["scale"])
    return [y, *torch.autograd.grad(y, leaves, s["dy"])]


def run(state):
    if own:
        return {"logp": _own_logp, "policy": _own_policy, "pref": _own_pref, "lora": _own_lora}[state["kind"]](state)
    return {"logp": _plain_logp, "policy": _plain_policy, "pref": _plain_pref, "lora": _plain_lora}[state["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its exact outputs
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "lora":
        M, K, N, R = c["B"] * c["T"], c["K"], c["N"], c["R"]
        used = min(c["n"], c["B"] * (8 if c["per_token"] else 1))
        once = 2 * M * (N * K + R * (K + N))
        if not c["grad"]:
            return {"bytes": 2 * (M * (K + N) + N * K + used * R * (K + N)), "flops": once}
        # x, dy, w and the masters in; y, dx and the masters' gradients out; no gradient of the shared weight
        return {"bytes": 2 * (2 * M * (K + N) + N * K) + 8 * c["n"] * R * (K + N),
                "flops": 2 * once + 2 * M * R * (K + N)}
    rows, kept = _rows(c), _counted(c)
    grad = c["kind"] != "logp" or c["grad"]
    return {"bytes": 2 * kept * c["vocab"] + (2 * rows * c["stride"] if grad else 0) + 24 * rows,
            "flops": (20 if grad else 8) * kept * c["vocab"]}


def _exact_rows(logits, targets, vocab, of_row):
    """Rows in 64 bits, 512 at a time: (logp, entropy, gradients for of_row(first row, logp, entropy))."""
    parts = []
    for i in range(0, logits.shape[0], 512):
        l, y = logits[i:i + 512].double(), targets[i:i + 512]
        z = CAP * torch.tanh(l[:, :vocab] / CAP)
        q = torch.log_softmax(z, 1)
        keep = (y != IGNORE).double()
        y = y.clamp(min=0)[:, None]
        logp, ent = q.gather(1, y)[:, 0] * keep, -(q.exp() * q).sum(1) * keep
        grad = None
        if of_row is not None:
            g, h = of_row(slice(i, i + 512), logp, ent)
            grad = -q.exp() * ((g * keep)[:, None] + (h * keep)[:, None] * (q + ent[:, None]))
            grad.scatter_add_(1, y, (g * keep)[:, None])
            grad = grad * (1 - (z / CAP) ** 2)
            grad = torch.cat([grad, grad.new_zeros(len(grad), l.shape[1] - vocab)], 1).float()
        parts.append((logp, ent, grad))
    logp, ent, grad = zip(*parts)
    return torch.cat(logp), torch.cat(ent), None if of_row is None else torch.cat(grad)


def _exact_loss(s):
    logits, targets, vocab = s["logits"].flatten(0, -2), s["targets"].flatten(), s["vocab"]
    if s["kind"] == "logp":
        h = s["h"].double() if s["entropy"] else torch.zeros_like(s["g"]).double()
        logp, ent, grad = _exact_rows(logits, targets, vocab,
                                      (lambda at, q, e: (s["g"][at].double(), h[at])) if s["grad"] else None)
        return [logp, *([ent] if s["entropy"] else []), *([grad] if s["grad"] else [])]
    count = (targets != IGNORE).double()
    if s["kind"] == "policy":
        w = count / count.sum()

        def terms(at, q):
            r, a = (q - s["old"][at].double()).exp(), s["adv"][at].double()
            out = ((a > 0) & (r > 1 + CLIP_HIGH)) | ((a < 0) & (r < 1 - CLIP))
            loss = -a * torch.where(out, r.clamp(1 - CLIP, 1 + CLIP_HIGH), r)
            slope = torch.where(out, 0.0, -a * r)
            kl = torch.zeros_like(r)
            if s["ref"] is not None:
                d = s["ref"][at].double() - q
                kl = torch.expm1(d) - d
                slope = slope - KL_COEF * torch.expm1(d)
            return loss + KL_COEF * kl, slope, out.double(), kl

        logp, _, grad = _exact_rows(logits, targets, vocab, lambda at, q, e: (w[at] * terms(at, q)[1], 0 * q))
        loss, _, out, kl = terms(slice(None), logp)
        return [w @ loss, logp, w @ out, *([w @ kl] if s["ref"] is not None else []), grad]
    logp = _exact_rows(logits, targets, vocab, None)[0]
    at = s["starts"].tolist()
    sums, counts = (torch.stack([v[i:j].sum() for i, j in zip(at, at[1:])]) for v in (logp, count))
    counts = counts.clamp(min=1) if s["average"] else torch.ones_like(counts)
    gain = (sums / counts - s["ref"].double()).view(2, -1)
    margin = s["beta"] * (gain[0] - gain[1])
    sg = torch.nn.functional.logsigmoid
    loss = -((1 - SMOOTHING) * sg(margin) + SMOOTHING * sg(-margin)).mean()
    slope = s["beta"] / margin.numel() * (SMOOTHING * sg(margin).exp() - (1 - SMOOTHING) * sg(-margin).exp())
    per_row = torch.cat([torch.full((j - i,), float(v / n), device=logits.device, dtype=torch.float64)
                         for i, j, v, n in zip(at, at[1:], torch.cat([slope, -slope]), counts)])
    grad = _exact_rows(logits, targets, vocab, lambda at, q, e: (per_row[at], 0 * q))[2]
    return [loss, sums / counts, margin, grad.view(s["logits"].shape)]


def _exact_lora(s):
    x, w, dy = (s[k].flatten(0, -2).double() for k in ("x", "w", "dy"))
    y, dx = x @ w.t(), dy @ w
    ids = s["ids"] if s["ids"].ndim == 2 else s["ids"][:, None].expand(s["x"].shape[:2])
    ids = ids.reshape(-1)
    da, db = (torch.zeros_like(s[k], dtype=torch.float64) for k in ("a", "b"))
    for i in range(s["a"].shape[0]):
        rows = (ids == i).nonzero()[:, 0]
        a, b, c = s["a"][i].bfloat16().double(), s["b"][i].bfloat16().double(), s["scale"][i].double()
        y[rows] += c * (x[rows] @ a.t()) @ b.t()
        dx[rows] += c * (dy[rows] @ b) @ a
        da[i] = c * (dy[rows] @ b).t() @ x[rows]
        db[i] = c * dy[rows].t() @ (x[rows] @ a.t())
    y = y.view(*s["x"].shape[:2], -1)
    return [y, dx.view(s["x"].shape), da, db] if s["grad"] else [y]


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_lora(s) if case["kind"] == "lora" else _exact_loss(s)
