"""GPU parity of the low-rank adapters with the float64 oracle.

Tolerances.  Operands are bf16, their products are exact in f32, and a sum of J of them with f32
partial sums is off by at most J 2^-24 of the sum of magnitudes (far less in practice: several
accumulators).  y is the adapters' part, u = s A x in f32 split in two bf16 (16 bits) and rounded to
bf16, added to the projection and rounded once more: 2^-8 of |part| and of |y|.  The factors'
gradients are f32 throughout: (J + M + 64) 2^-24 of the sums of magnitudes.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import post_training as P

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from experiment_swa_kda_amd import KimiDeltaAttention, lora_linear, ops
    from experiment_swa_kda_amd.kda import Linear, LoraLinear
    from experiment_swa_kda_amd.model import GPT, Block, GPTConfig, GraphedUpdate, KVCache


def n64(t):
    return t.detach().double().cpu().numpy()


def case(B, T, K, N, R, n, seed, masters=False):
    g = torch.Generator().manual_seed(seed)

    def normal(*s, k=1.0):
        return torch.randn(*s, generator=g) * k

    d = dict(x=normal(B, T, K).bfloat16(), w=normal(N, K, k=K ** -0.5).bfloat16(), a=normal(n, R, K, k=K ** -0.5),
             b=normal(n, N, R, k=R ** -0.5), scale=torch.rand(n, generator=g) + 0.5, dy=normal(B, T, N).bfloat16())
    if not masters:
        d["a"], d["b"] = d["a"].bfloat16(), d["b"].bfloat16()
    ids = torch.randint(-1, n, (B,), generator=g).int()
    per_row = torch.randint(-1, n, (B, T), generator=g).int()
    return {k: v.cuda() for k, v in d.items()}, ids, per_row


def check(d, ids, y, dx=None, dw=None, da=None, db=None):
    B, T, K = d["x"].shape
    M, N, n, R = B * T, d["w"].shape[0], *d["a"].shape[:2]
    rows = (ids if ids.ndim == 2 else ids[:, None].expand(B, T)).flatten().tolist()
    x, dy = n64(d["x"]).reshape(M, K), n64(d["dy"]).reshape(M, N)
    w, a, b, s = n64(d["w"]), n64(d["a"].bfloat16()), n64(d["b"].bfloat16()), n64(d["scale"])
    e = P.lora(x, w, a, b, rows, s, dy)
    part = np.abs(e[0] - x @ w.T), np.abs(e[1] - dy @ w)
    # sums of magnitudes of every result
    m = P.lora(*map(np.abs, (x, w, a, b)), rows, s, np.abs(dy))
    f32 = (K + N + R + 64) * 2.0 ** -24
    for got, want, delta, size in ((y, e[0], part[0], m[0]), (dx, e[1], part[1], m[1])):
        if got is not None:
            off = np.abs(n64(got).reshape(want.shape) - want)
            assert np.all(off <= 1.01 * 2.0 ** -8 * (np.abs(want) + 2 * delta) + (f32 + 2.0 ** -16 * (delta > 0)) * size)
    f32 = (K + N + M + 64) * 2.0 ** -24
    for got, want, size, round_ in ((dw, e[2], m[2], d["w"].dtype), (da, e[3], m[3], d["a"].dtype), (db, e[4], m[4], d["b"].dtype)):
        if got is not None:
            half = 2.0 ** -8 if round_ == torch.bfloat16 else 0.0
            assert got.dtype == round_
            assert np.all(np.abs(n64(got) - want) <= f32 * size + 1.01 * half * np.abs(want))


SHAPES = [  # B, T, K, N, R, n
    (1, 1, 8, 8, 8, 1), (3, 1, 40, 24, 8, 2), (8, 1, 384, 1536, 16, 8), (64, 1, 264, 520, 16, 64),
    (17, 1, 2048, 72, 64, 3), (2, 5, 72, 136, 24, 3), (3, 33, 136, 264, 32, 2), (2, 300, 384, 200, 16, 5),
    (1, 513, 96, 1544, 40, 1), (5, 77, 520, 384, 128, 3), (2, 2100, 64, 72, 8, 4), (70, 3, 128, 128, 56, 9),
]


@pytest.mark.parametrize("B,T,K,N,R,n", SHAPES)
@pytest.mark.parametrize("per_row", [False, True])
def test_lora_matches_oracle(B, T, K, N, R, n, per_row):
    d, ids, row_ids = case(B, T, K, N, R, n, B + T + K, masters=per_row)
    ids = row_ids if per_row else ids
    print(f"lora B{B} T{T} K{K} N{N} R{R} n{n} per_row {per_row}", flush=True)
    leaves = [d[k].detach().requires_grad_() for k in ("x", "w", "a", "b")]
    y = lora_linear(*leaves, ids.cuda(), d["scale"])
    check(d, ids, y)
    check(d, ids, y, *torch.autograd.grad(y, leaves, d["dy"], retain_graph=True))
    with torch.no_grad():
        z = lora_linear(d["x"], d["w"], d["a"], d["b"], ids.cuda(), d["scale"])
    check(d, ids, z)
    some = torch.autograd.grad(y, leaves[3], d["dy"])  # one gradient alone
    check(d, ids, y, db=some[0])


def test_ids_out_of_range_strides_and_types():
    d, _, _ = case(4, 6, 64, 96, 16, 3, 5)
    want = [lora_linear(d["x"], d["w"], d["a"], d["b"], torch.tensor(i, dtype=torch.int32).cuda(), d["scale"])
            for i in ([2, -1, 0, -1],)][0]
    for ids in ([2, 3, 0, -5], [2, 2 ** 31 - 1, 0, -2 ** 31]):
        for kind in (torch.int32, torch.int64):
            got = lora_linear(d["x"], d["w"], d["a"], d["b"], torch.tensor(ids, dtype=kind).cuda(), d["scale"])
            assert torch.equal(got, want)
    far = torch.tensor([2, 2 ** 32 + 1, 0, -2 ** 40]).cuda()
    assert torch.equal(lora_linear(d["x"], d["w"], d["a"], d["b"], far, d["scale"]), want)
    # every operand a strided or unaligned view of the same values
    wide = torch.zeros(4, 6, 200, dtype=torch.bfloat16, device="cuda")
    wide[..., 4:68] = d["x"]
    ids = torch.tensor([2, 9, -1, 9, 0, 9, -1, 9], dtype=torch.int32).cuda()[::2]
    got = lora_linear(wide[..., 4:68], d["w"].t().contiguous().t(), d["a"].transpose(1, 2).contiguous().transpose(1, 2),
                      torch.cat([d["b"], d["b"]])[:3], ids, torch.stack([d["scale"], d["scale"]], 1)[:, 0])
    check(d, torch.tensor([2, -1, 0, -1]), got)


@pytest.mark.parametrize("T", [1, 40])
def test_another_requests_nan_and_an_unused_adapters_inf_stay_out(T):
    d, _, _ = case(6, T, 64, 96, 16, 4, 7, masters=True)
    ids = torch.tensor([0, 1, 0, -1, 2, 1], dtype=torch.int32)
    d["x"][1] = float("nan")
    d["dy"][1] = float("inf")
    d["x"][3] = float("inf")  # no adapter
    d["a"][3] = float("nan")
    d["b"][3] = float("inf")
    leaves = [d[k].detach().requires_grad_() for k in ("x", "a", "b")]
    y = lora_linear(leaves[0], d["w"], *leaves[1:], ids.cuda(), d["scale"])
    dx, da, db = torch.autograd.grad(y, leaves, d["dy"])
    keep = [0, 2, 4]
    assert all(torch.isfinite(v[keep]).all() for v in (y, dx))
    assert not torch.isfinite(y[[1, 5]]).all() or T == 0
    assert torch.isfinite(da[[0, 2]]).all() and torch.isfinite(db[[0, 2]]).all()
    assert not da[3].any() and not db[3].any()
    assert torch.isnan(da[1]).any() and torch.isfinite(y[5]).all()


# contraction, outputs and rows of every way a call takes: few rows, rows with ids of their own, whole
# sequences; one kernel for the projection or the adapters' part beside it, in either direction
WAYS = [(6, 1, 64, 96), (9, 7, 1032, 72), (40, 1, 520, 4096), (90, 1, 64, 96), (6, 40, 64, 96), (6, 40, 1608, 72), (6, 40, 72, 1608),
        (3, 90, 1600, 1544), (7, 190, 64, 200), (9, 60, 64, 200), (4, 75, 520, 4096)]


@pytest.mark.parametrize("B,T,K,N", WAYS)
@pytest.mark.parametrize("per_row", [False, True])
def test_every_way_matches_oracle(B, T, K, N, per_row):
    d, ids, row_ids = case(B, T, K, N, 24, 3, B + K, masters=True)
    ids = row_ids if per_row else ids
    leaves = [d[k].detach().requires_grad_() for k in ("x", "w", "a", "b")]
    y = lora_linear(*leaves, ids.cuda(), d["scale"])
    check(d, ids, y, *torch.autograd.grad(y, leaves, d["dy"]))


@pytest.mark.parametrize("B,T,K,N", WAYS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_broken_adapter_in_use_stays_with_its_requests(B, T, K, N, bad):
    d, _, ids = case(B, T, K, N, 16, 3, 11, masters=True)  # every row its own: tiles of all adapters
    d["a"][1, 3, 5] = bad
    d["b"][1, 7] = bad
    leaves = [d[k].detach().requires_grad_() for k in ("x", "a", "b")]
    y = lora_linear(leaves[0], d["w"], *leaves[1:], ids.cuda(), d["scale"])
    dx, da, db = torch.autograd.grad(y, leaves, d["dy"])
    broken = ids.cuda() == 1
    assert torch.isfinite(y[~broken]).all() and torch.isfinite(dx[~broken]).all()
    assert not torch.isfinite(y[broken]).all(-1).any() and not torch.isfinite(dx[broken]).all(-1).any()
    assert torch.isfinite(da[[0, 2]]).all() and torch.isfinite(db[[0, 2]]).all()


@pytest.mark.parametrize("B,T,K,N", WAYS)
def test_an_infinite_input_is_not_turned_to_nan(B, T, K, N):
    """x = (inf, 0, ..) and positive weights: every output is the infinity, not infinity - infinity."""
    d, _, _ = case(B, T, K, N, 8, 2, 12)
    d["x"].zero_()
    d["x"][..., 0] = float("inf")
    for k in ("w", "a", "b"):
        d[k] = d[k].abs() + 0.5
    ids = torch.zeros(B, dtype=torch.int32, device="cuda")
    y = lora_linear(d["x"], d["w"], d["a"], d["b"], ids, d["scale"])
    assert (y == float("inf")).all()


def test_gradient_ranges_of_several_windows():
    """Long ranges of rows (few ranges for many columns): factor gradients of 5000 rows by 32768 outputs."""
    g = torch.Generator().manual_seed(13)
    M, K, N, R, n = 5000, 8, 32768, 8, 3
    x, dy = (torch.randn(M, k, generator=g).bfloat16().cuda() for k in (K, N))
    w = torch.zeros(N, K, dtype=torch.bfloat16, device="cuda")
    a, b = (torch.randn(*s, generator=g).bfloat16().cuda() for s in ((n, R, K), (n, N, R)))
    scale = torch.ones(n, device="cuda")
    ids = torch.randint(-1, n, (M,), generator=g).int().cuda()
    ids[:2100] = 2  # the first steps hold no row of the others
    _, u = ops.lora_forward(x, w, a, b, ids, scale)
    _, _, db = ops.lora_backward(x, w, a, b, ids, scale, u, dy, False, False, True)
    for i in range(n):
        on = ids == i
        t = x[on].double() @ a[i].double().t()
        want, size = dy[on].double().t() @ t, dy[on].double().abs().t() @ (x[on].double().abs() @ a[i].double().abs().t())
        assert ((db[i] - want).abs() <= (K + M + 64) * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("K,N", [(4096, 64), (64, 4096)])
@pytest.mark.parametrize("per_row", [False, True])
def test_offsets_past_32_bits(K, N, per_row):
    """Inputs or outputs of more than 2^31 elements: the last rows, and the gradients of all."""
    B, T, R, n = 4, 131500, 8, 3
    g = torch.Generator().manual_seed(14)
    small = torch.randn(n, R, K, generator=g) * K ** -0.5, torch.randn(n, N, R, generator=g) * R ** -0.5
    w = (torch.randn(N, K, generator=g) * K ** -0.5).bfloat16().cuda()
    torch.manual_seed(14)
    x, dy = (torch.randn(B, T, k, device="cuda", dtype=torch.bfloat16) for k in (K, N))
    ids = torch.randint(-1, n, (B, T), generator=g).int() if per_row else torch.tensor([1, -1, 0, 2], dtype=torch.int32)
    leaves = [x.requires_grad_(), *(v.cuda().requires_grad_() for v in small)]
    scale = torch.tensor([0.5, 1.0, 1.5]).cuda()
    y = lora_linear(leaves[0], w, *leaves[1:], ids.cuda(), scale)
    dx, da, db = torch.autograd.grad(y, leaves, dy)
    last = slice(T - 96, T)
    d = dict(x=x[3:, last], dy=dy[3:, last], w=w, a=leaves[1], b=leaves[2], scale=scale)
    check(d, ids[3:, last] if per_row else ids[3:], y[3:, last], dx[3:, last])
    want = [[torch.zeros_like(v, dtype=torch.float64) for v in (da, db)] for _ in range(2)]  # and of magnitudes
    for b in range(B):
        for t0 in range(0, T, 32875):
            at = (b, slice(t0, t0 + 32875))
            row = (ids[at] if per_row else ids[b].expand(T)[at[1]]).cuda()
            for i in range(n):
                xi, gi = (v[at][row == i].detach().double() for v in (x, dy))
                f = [v[i].detach().bfloat16().double() for v in leaves[1:]]
                for (wa, wb), (X, G, A, F) in zip(want, ((xi, gi, *f), [v.abs() for v in (xi, gi, *f)])):
                    wa[i] += scale[i].double() * (G @ F).t() @ X
                    wb[i] += scale[i].double() * G.t() @ (X @ A.t())
    # a range of at most 32896 rows is a chain of 3 products for each 32 of them, its sum one of some
    # 32 more; the factor's row (K or N terms) is summed by eight waves or more
    bound = (3 * 32896 / 32 + 32 + 4096 / 8) * 2.0 ** -24
    for got, e, size in zip((da, db), *want):
        assert ((got - e).abs() <= bound * size).all()


def test_empty_and_single():
    d, _, _ = case(2, 3, 64, 96, 16, 2, 8, masters=True)
    for x, ids in ((d["x"][:0], torch.zeros(0)), (d["x"][:, :0], torch.zeros(2))):
        leaf = x.detach().requires_grad_()
        a, b = (d[k].detach().requires_grad_() for k in ("a", "b"))
        y = lora_linear(leaf, d["w"], a, b, ids.int().cuda(), d["scale"])
        assert y.shape == (*x.shape[:-1], 96)
        dx, da, db = torch.autograd.grad(y.sum(), [leaf, a, b])
        assert dx.shape == x.shape and not da.any() and not db.any()
    two = lora_linear(d["x"][:, 0], d["w"], d["a"], d["b"], torch.tensor([1, 0], dtype=torch.int32).cuda(), d["scale"])
    check({**d, "x": d["x"][:, :1]} | {"dy": d["dy"][:, :1]}, torch.tensor([1, 0]), two)


def test_second_derivatives_are_refused():
    d, ids, _ = case(3, 30, 64, 96, 16, 2, 18, masters=True)
    leaves = [d[k].detach().requires_grad_() for k in ("x", "a", "b")]
    y = lora_linear(leaves[0], d["w"], *leaves[1:], ids.cuda(), d["scale"])
    first = torch.autograd.grad(y, leaves, d["dy"], retain_graph=True)
    again = torch.autograd.grad(y, leaves, d["dy"], create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        torch.autograd.grad(again[1].sum(), leaves[2])


def test_gpu_refusals():
    d, ids, _ = case(2, 3, 64, 96, 16, 2, 8)
    cuda = ids.cuda()
    for change, words in ((dict(w=d["w"][:, :60], a=d["a"][..., :60], x=d["x"][..., :60]), "multiples of 8"),
                          (dict(a=d["a"][:, :12], b=d["b"][..., :12]), "rank"),
                          (dict(a=d["a"].cpu()), "device")):
        e = d | change
        with pytest.raises(RuntimeError, match=words):
            lora_linear(e["x"], e["w"], e["a"], e["b"], cuda, e["scale"])
    with pytest.raises(RuntimeError, match="same number of rows"):
        ops.lora_forward(d["x"].view(6, 64), d["w"], d["a"], d["b"], torch.zeros(4, dtype=torch.int32, device="cuda"), d["scale"])


def step(d, ids):
    leaves = [d[k].detach().requires_grad_() for k in ("x", "a", "b")]
    y = lora_linear(leaves[0], d["w"], *leaves[1:], ids, d["scale"])
    return [y, *torch.autograd.grad(y, leaves, d["dy"])]


def test_repeats_streams_and_replays_are_bitwise_equal():
    """Training and token calls, eagerly, on another stream and captured; replays follow the ids,
    inputs and adapters copied in, with eager work between them."""
    d, ids, _ = case(3, 50, 128, 160, 16, 4, 9, masters=True)
    tok, _, _ = case(5, 1, 128, 160, 16, 4, 10)
    ids, tok_ids = ids.cuda(), torch.tensor([3, -1, 0, 3, 2], dtype=torch.int32).cuda()

    def both():
        with torch.no_grad():
            t = lora_linear(tok["x"], tok["w"], tok["a"], tok["b"], tok_ids, tok["scale"])
        return [*step(d, ids), t]

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(4):
        new, i, _ = case(3, 50, 128, 160, 16, 4, 20 + k, masters=True)
        for name in ("x", "a", "b", "dy"):
            d[name].copy_(new[name])
        ids.copy_(i)
        tok_ids.copy_(tok_ids.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, both())), k


def test_two_captured_calls_take_turns():
    """Two graphs of the same shapes, replayed by turns and on two streams: neither's workspaces are the other's."""
    sets = [case(4, 70, 1600, 136, 16, 3, 30 + k, masters=True) for k in range(2)]
    graphs, outs = [], []
    ids = [s[1].cuda() for s in sets]
    want = [step(s[0], i) for s, i in zip(sets, ids)]
    want = [[t.detach().clone() for t in w] for w in want]
    for s, i in zip(sets, ids):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(s[0], i))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(3):
        for o in outs:
            for t in o:
                t.detach().zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, w)), turn


def small_gpt(seed=0):
    torch.manual_seed(seed)
    m = GPT(GPTConfig(sequence_len=64, vocab_size=500, n_layer=2, n_head=2, n_embd=128)).cuda()
    m.init_weights()
    torch.nn.init.normal_(m.lm_head.weight, 0.0, 0.3)
    for b in m.transformer.h:
        torch.nn.init.normal_(b.mlp.c_proj.weight, 0.0, 0.02)
        torch.nn.init.normal_(b.attn.o_proj.weight, 0.0, 0.02)
    return m


def test_decoder_serves_a_batch_of_requests_with_their_own_adapters():
    """Prompt and token steps of a mixed batch give every request what the model gives it alone
    with its adapter merged into the weights."""
    m = small_gpt()
    new = m.add_adapters(3, 16, alpha=32.0)
    with torch.no_grad():
        for p in new:
            p.normal_(0.0, 0.05)
    idx = torch.randint(0, 500, (4, 21), device="cuda")
    ids = torch.tensor([2, -1, 0, 2], dtype=torch.int32, device="cuda")

    def generate(model, tokens, adapters, cached):
        model.use_adapters(adapters) if adapters is not None else None
        cache = KVCache(len(tokens), 2, 64, 64, 2, "cuda", torch.bfloat16)
        if cached:
            model.cache_bf16_weights()
        with torch.no_grad():
            out = [model(tokens[:, :16], kv_cache=cache)[:, -1]]
            out += [model(tokens[:, k:k + 1], kv_cache=cache)[:, -1] for k in range(16, 21)]
        if cached:
            model.drop_bf16_weights()
        return torch.stack(out, 1)

    mixed = generate(m, idx, ids, False)
    assert torch.equal(generate(m, idx, ids, True), mixed)
    for row, a in enumerate(ids.tolist()):
        merged = small_gpt()
        if a >= 0:
            for lin, bank in ((p, q) for p, q in zip(merged.modules(), m.modules()) if isinstance(q, LoraLinear)):
                with torch.no_grad():
                    lin.weight += bank.scaling[a] * bank.lora_b[a].bfloat16().float() @ bank.lora_a[a].bfloat16().float()
        alone = generate(merged, idx[row:row + 1], None, False)
        # the merged weight is rounded to bf16 once, the adapter's path rounds its part: as far apart
        # as two bf16 forwards of 2 layers and a head are (logits of a few units)
        assert (alone[0] - mixed[row]).abs().max().item() < 0.25
        assert (alone[0] - mixed[row]).norm() < 0.03 * alone[0].norm()


def test_adapters_of_the_output_projection_alone_are_not_passed_over():
    """A block whose MLP is plain: its one-token step still adds the output projection's adapters."""
    m = small_gpt(4)
    for b in m.transformer.h:
        lin = LoraLinear(128, 128, 2, 8).cuda()
        lin.weight = b.attn.o_proj.weight
        torch.nn.init.normal_(lin.lora_b, 0.0, 0.1)
        b.attn.o_proj = lin
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    idx = torch.randint(0, 500, (3, 12), device="cuda")

    def generate(adapters):
        m.use_adapters(adapters)
        cache = KVCache(3, 2, 64, 64, 2, "cuda", torch.bfloat16)
        m.cache_bf16_weights()
        with torch.no_grad():
            out = [m(idx[:, :8], kv_cache=cache)[:, -1]] + [m(idx[:, k:k + 1], kv_cache=cache)[:, -1] for k in range(8, 12)]
        m.drop_bf16_weights()
        return torch.stack(out, 1)

    got, bare = generate(ids), generate(None)
    m.use_adapters(ids)
    with torch.no_grad():
        full = m(idx)[:, 7:]  # the whole sequence at once: no state, no token step
    # a step's activations and the prompt's are bf16 roundings of the same values, two layers of them
    assert (got - full).norm() <= 0.03 * full.norm()
    # without the one-token step that computes with a plain projection's weight: the same kernels, bit for bit
    kept = Block._token_ok
    try:
        Block._token_ok = lambda *args: False
        assert torch.equal(generate(ids), got)
    finally:
        Block._token_ok = kept
    # (a row's computation does not depend on the other rows: what differs from the bare model is the adapters')
    same = (got == bare).flatten(1).all(1).tolist()
    assert same == [False, True, False]


def test_adapter_gradients_beside_frozen_weights():
    """With the weights frozen the mixers' cores below run outside autograd: the adapters' gradients are
    those of the model that trains everything."""
    m = small_gpt(5)
    new = m.add_adapters(2, 8)
    with torch.no_grad():
        for p in new:
            p.normal_(0.0, 0.05)
    m.use_adapters(torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    idx = torch.randint(0, 500, (2, 40), device="cuda")
    want = torch.autograd.grad(m(idx[:, :-1], idx[:, 1:]), new)
    for p in m.parameters():
        p.requires_grad_(any(p is q for q in new))
    got = torch.autograd.grad(m(idx[:, :-1], idx[:, 1:]), new)
    for p, q in zip(got, want):
        assert q.any() and (p - q).norm() <= 0.02 * q.norm()  # (the same chain of bf16 roundings, 2^-8 each)


def test_decoder_trains_adapters_on_the_policy_loss():
    """The operators together: adapters of two policies trained in one batch, gradients against the
    same step with every adapter applied in plain torch."""
    m = small_gpt(1)
    new = m.add_adapters(3, 16)
    with torch.no_grad():
        for p in new:
            p.normal_(0.0, 0.05)
    ids = torch.tensor([1, 0, -1, 1], dtype=torch.int32, device="cuda")
    m.use_adapters(ids)
    idx = torch.randint(0, 500, (4, 33), device="cuda")
    t = idx[:, 1:].clone()
    t[:, :5] = -1
    adv = torch.randn(4, 32, device="cuda")
    with torch.no_grad():
        old = m.token_log_probs(idx[:, :-1], t)
    loss = m.policy_loss(idx[:, :-1], t, old, adv, ref_log_probs=old, kl_coef=0.1).loss
    got = torch.autograd.grad(loss, new)

    def plain(self, x, w16=None):
        y = x.float() @ self.weight.bfloat16().float().t()
        a, b = self.lora_a.bfloat16().float(), self.lora_b.bfloat16().float()
        on = (ids >= 0).float() * self.scaling[ids.clamp(min=0).long()]
        i = ids.clamp(min=0).long()
        u = torch.bmm(x.float(), a[i].transpose(1, 2).contiguous())
        return (y + torch.bmm(u, b[i].transpose(1, 2).contiguous()) * on[:, None, None]).bfloat16()

    kept = LoraLinear.forward
    try:
        LoraLinear.forward = plain
        ref = m.policy_loss(idx[:, :-1], t, old, adv, ref_log_probs=old, kl_coef=0.1).loss
        want = torch.autograd.grad(ref, new)
    finally:
        LoraLinear.forward = kept
    for p, q in zip(got, want):
        assert not p[2].any()  # an adapter that no sequence uses
        # both chains round activations and gradients to bf16 (2^-8) at some twenty places
        assert (p - q).norm() <= 0.05 * q.norm()


def test_graphed_update_of_adapters_is_the_eager_one():
    """Three captured updates of the adapters alone leave what three eager ones leave."""
    def trained(graphed):
        m = small_gpt(2)
        for p in m.parameters():
            p.requires_grad_(False)
        torch.manual_seed(3)
        new = m.add_adapters(3, 8)
        m.use_adapters(torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda"))
        batch = torch.randint(0, 500, (3, 34), device="cuda")
        opt = torch.optim.AdamW(new, lr=1e-2, fused=True, capturable=True)
        update = GraphedUpdate(m, opt, [batch]) if graphed else None
        for _ in range(3):
            if graphed:
                update()
            else:
                for p, g in zip(new, torch.autograd.grad(m(batch[:, :-1], batch[:, 1:]), new)):
                    p.grad = g
                opt.step()
        torch.cuda.synchronize()
        return [p.detach().clone() for p in new]

    for p, q in zip(trained(True), trained(False)):
        assert torch.equal(p, q)
