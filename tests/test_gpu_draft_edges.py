"""The drafted-token operators (fun_asr_gguf.ops) on the GPU where they can go wrong: many splits of narrow heads, infinities and
NaN among keys, weights far below the largest, float32 queries of any size, large vocabularies, what autograd sees. Plain 64-bit
forms: tests/draft_oracle.py; tolerances as in test_gpu_draft_ops.py unless a test says more."""
import numpy as np
import pytest
import torch  # noqa: F401  (before any engine: the library then shares torch's HIP runtime)

from draft_oracle import attention
from test_gpu_draft_ops import U, check, close, kind, ops, paged, sampled, t, tolerance, trees, wide  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------ joining splits
@pytest.mark.parametrize("ctx,N,H,KV,D,qn,cn,order", [
    ([8150], 1, 8, 8, 96, "f16", "f16", "hpd"), ([8180], 4, 16, 8, 80, "bf16", "bf16", "phd"),
    ([9000], 3, 2, 1, 192, "f32", "f16", "hpd"), ([2040, 700], 2, 2, 2, 8, "f16", "f16", "hpd"),
    ([40000], 1, 7, 1, 96, "bf16", "bf16", "hpd"), ([6000], 40, 4, 2, 40, "f16", "f16", "hpd"),
    ([8190], 1, 8, 8, 128, "f16", "f16", "hpd"), ([8190], 2, 8, 8, 64, "f32", "bf16", "hpd")])
def test_attention_splits_of_every_head_size(t, ops, ctx, N, H, KV, D, qn, cn, order):
    """One or two long sequences: up to 64 splits, more than a narrow head has lanes in the launch that joins them."""
    kc, vc, table = paged(t, ctx, N, 16, KV, D, cn, order, 5)
    q = (2 * t.randn(len(ctx), N, H, D, generator=t.Generator().manual_seed(6))).to(kind(t, qn)).cuda()
    check(t, ops, q, kc, vc, table, ctx, names=(qn, cn))


# ---------------------------------------------------------------------------------------- infinities and NaN, committed
@pytest.mark.parametrize("N", [1, 9, 40])
@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("D", [128, 96])
def test_attention_nonfinite_committed_values_reach_every_row(t, ops, name, N, D):
    """Wherever the key lies: tiles before the last, the tile that also holds the drafts, the last committed token."""
    ctx = [100]
    kc, vc, table = paged(t, ctx, N, 16, 2, D, name, "hpd", 8)
    q = t.randn(1, N, 4, D, generator=t.Generator().manual_seed(1)).to(kind(t, name)).cuda()
    mask = trees(t, 1, N, 9) if N > 1 else None
    lens = t.tensor(ctx, dtype=t.int32).cuda()
    run = lambda: ops.tree_attention(q, kc, vc, table, lens, mask=None if mask is None else mask.cuda())  # noqa: E731
    clean = check(t, ops, q, kc, vc, table, ctx, mask, names=(name, name))
    for p in (10, 63, 64, 95, 96, 99):
        at = int(table[0, p // 16]), slice(None), p % 16
        for what in (float("inf"), float("-inf"), float("nan")):
            for d in (3, 77):
                keep = vc[at].clone()
                vc[at[0], :, at[2], d] = what
                out = run()
                vc[at] = keep
                hit = out[..., d]
                assert (hit.isnan().all() if what != what else (hit == what).all()), (p, what, d)
                rest = [x for x in range(D) if x != d]
                assert t.equal(out[..., rest], clean[..., rest]), (p, what, d)


# --------------------------------------------------------------------------------------------- weights far below the largest
@pytest.mark.parametrize("keys,N,gap", [(8192, 1, 18.0), (40000, 1, 17.0), (40000, 1, 18.0), (8192, 40, 18.0), (3000, 2, 21.0)])
@pytest.mark.parametrize("qn,cn", [("f16", "f16"), ("f32", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
def test_attention_long_tails_below_one_large_weight(t, ops, keys, N, gap, qn, cn):
    """One key takes nearly all the weight and has a value of 0; the rest, e^-gap below it, make the output. Beside the
    tolerance of every test: over a float16 cache a weight is a float16 number (two, for a float32 query) of 2^15 at the largest,
    so its absolute step counts too: half of 2^-24, 2^-40 of the largest weight, for every key."""
    D = 64
    g = t.Generator().manual_seed(keys + N)
    ctx = [keys - N]
    pages = -(-keys // 64)
    kc = t.zeros(pages, 1, 64, D)
    vc = (1 + 0.25 * t.randn(pages, 1, 64, D, generator=g)).abs()
    kc[..., 0] = 4 + 0.02 * t.randn(pages, 1, 64, generator=g)
    one = keys // 3
    kc[one // 64, 0, one % 64, 0] = 4 + gap / 4
    vc[one // 64, 0, one % 64] = 0
    kc, vc = (c.to(kind(t, cn)).cuda() for c in (kc, vc))
    q = t.zeros(1, N, 2, D)
    q[..., 0] = 4
    q = q.to(kind(t, qn)).cuda()
    table = t.arange(pages, dtype=t.int32)[None].cuda()
    out = ops.tree_attention(q, kc, vc, table, t.tensor(ctx, dtype=t.int32).cuda(), scale=1.0)
    want, mass, reach = attention(wide(q), wide(kc), wide(vc), table.cpu().numpy(), ctx, [N], None, 1.0)
    assert want.max() < keys * np.exp(2 - gap)
    tol = tolerance(want, mass, reach, qn, cn, D)
    if cn == "f16":
        tol = tol + keys * 2.0 ** -40 * float(vc.max())
    close(out, want, tol)


@pytest.mark.parametrize("size,scale", [(1e5, 1e-6), (1e-4, 1e3), (1e30, 1e-31), (1e-30, 1e28), (None, 0.05)])
@pytest.mark.parametrize("D,N,cn", [(128, 3, "f16"), (64, 40, "f16"), (96, 2, "bf16"), (256, 20, "f16")])
def test_attention_float32_queries_of_any_size(t, ops, size, scale, D, N, cn):
    """Queries past float16's range, or under its steps, at scales that give ordinary scores. None: rows of many sizes in one
    call, and a row of zeros."""
    ctx = [130, 3]
    kc, vc, table = paged(t, ctx, N, 16, 2, D, cn, "hpd", 12)
    g = t.Generator().manual_seed(3)
    q = t.randn(2, N, 4, D, generator=g)
    if size is None:
        q *= 10 ** (4 * t.rand(2, N, 4, 1, generator=g) - 2)
        q[0, 0, 1] = 0
        q[1, 1, :, 1:] = 0
    else:
        q *= size
    check(t, ops, q.cuda(), kc, vc, table, ctx, names=("f32", cn), scale=scale)


def test_attention_infinite_float32_queries(t, ops):
    """An infinite query makes its own row NaN (a score of +inf somewhere) and leaves the others as they are."""
    ctx, N, D = [50], 4, 128
    kc, vc, table = paged(t, ctx, N, 16, 2, D, "f16", "hpd", 13)
    q = t.randn(1, N, 4, D, generator=t.Generator().manual_seed(4)).cuda()
    lens = t.tensor(ctx, dtype=t.int32).cuda()
    clean = ops.tree_attention(q, kc, vc, table, lens)
    for what in (float("inf"), float("-inf"), float("nan")):
        bad = q.clone()
        bad[0, 2, 1, 7] = what
        out = ops.tree_attention(bad, kc, vc, table, lens)
        assert out[0, 2, 1].isnan().all()
        out[0, 2, 1] = clean[0, 2, 1]
        assert t.equal(out, clean)


@pytest.mark.parametrize("D,N,qn,cn", [
    (96, 3, "f16", "f16"), (40, 40, "bf16", "bf16"), (80, 1, "bf16", "bf16"), (128, 4, "f16", "f16"),
    (128, 3, "f32", "f16"), (128, 3, "f32", "bf16"), (64, 40, "f32", "f16"), (96, 2, "f32", "f16"), (256, 5, "f32", "bf16")])
@pytest.mark.parametrize("whole", [False, True])
def test_attention_infinite_keys(t, ops, D, N, qn, cn, whole):
    """A score of -inf is a weight of 0, one of +inf a row of NaN, whatever lies beside the infinity in the products: the places
    behind a narrow head, or a float32 query's lower terms (`whole`: they are 0)."""
    ctx = [70]
    kc, vc, table = paged(t, ctx, N, 16, 2, D, cn, "hpd", 11)
    g = t.Generator().manual_seed(2)
    q = t.randint(1, 4, (1, N, 4, D), generator=g) * 0.5 if whole else t.randn(1, N, 4, D, generator=g).abs()
    q[:, :, 1::2] *= -1  # one head of each pair meets +inf, the other -inf
    q = q.to(kind(t, qn)).cuda()
    lens = t.tensor(ctx, dtype=t.int32).cuda()
    plain = lambda: attention(wide(q), np.where(np.isnan(wide(kc)), 0, wide(kc)), np.nan_to_num(wide(vc)),  # noqa: E731
                              table.cpu().numpy(), ctx, [N], None, D ** -0.5)
    _, mass, reach = plain()
    tol = tolerance(0, mass, reach, qn, cn, D)
    for p, d, what in ((10, 0, float("inf")), (10, D - 1, float("-inf")), (69, 1, float("inf")), (70, 5, float("-inf")),
                       (64, 33, float("inf"))):
        at = int(table[0, p // 16]), slice(None), p % 16
        keep = kc[at].clone()
        kc[at[0], :, at[2], d] = what
        out = wide(ops.tree_attention(q, kc, vc, table, lens))
        with np.errstate(invalid="ignore"):
            want, _, _ = plain()
        kc[at] = keep
        none = np.isnan(want)
        assert none.any() and not none.all()
        assert (np.isnan(out) == none).all(), (p, d, what)
        # (without the key the weights of the others grow, by no more than its share: the tolerance's mass does too)
        assert (np.abs(out - want)[~none] <= (4 * tol + U[qn] * np.abs(want))[~none]).all(), (p, d, what)


@pytest.mark.parametrize("cn", ["f16", "bf16"])
@pytest.mark.parametrize("D,N", [(128, 9), (96, 40)])
@pytest.mark.parametrize("what", [float("inf"), float("-inf"), float("nan")])
def test_attention_nonfinite_drafts_of_float32_queries(t, ops, cn, D, N, what):
    """A drafted token's infinity reaches the tokens below it alone, in its value as in its key; another draft's key, infinite
    too, is left out where its score is -inf."""
    ctx = [45]
    kc, vc, table = paged(t, ctx, N, 16, 2, D, cn, "hpd", 8)
    q = t.randn(1, N, 4, D, generator=t.Generator().manual_seed(5)).cuda()
    q[..., 3] = q[..., 3].abs() + 0.1
    mask = trees(t, 1, N, 9)
    mask[0, 8, 4] = True
    seers = mask[0, :, 4]
    lens = t.tensor(ctx, dtype=t.int32).cuda()
    run = lambda: ops.tree_attention(q, kc, vc, table, lens, mask=mask.cuda())  # noqa: E731
    check(t, ops, q, kc, vc, table, ctx, mask, names=("f32", cn))
    gone = [int(table[0, 50 // 16]), slice(None), 50 % 16]  # draft 5: a score of -inf for every row
    kc[(*gone, 3)] = float("-inf")
    clean = run()
    without = mask.clone()
    without[0, :, 5] = False
    assert t.equal(clean, ops.tree_attention(q, kc, vc, table, lens, mask=without.cuda()))  # (a weight of 0 either way)
    at = int(table[0, 49 // 16]), slice(None), 49 % 16
    for c, d in ((vc, 3), (vc, 77), (kc, 5)):
        keep = c[at].clone()
        c[(*at, d)] = what
        out = run()
        c[at] = keep
        assert t.equal(out[0, ~seers], clean[0, ~seers])
        if c is vc:
            hit = out[0, seers][..., d]
            assert hit.isnan().all() if what != what else (hit == what).all()
            rest = [x for x in range(D) if x != d]
            assert t.equal(out[0, seers][..., rest], clean[0, seers][..., rest])


def test_what_autograd_sees(t, ops):
    """Every tensor that a call writes has a new version, so a graph that saved it notices; what it reads keeps its own."""
    x = t.randn(1, 2, 4, 32, device="cuda", dtype=t.float16)
    c, n = t.zeros(1, 2, 8, 32, device="cuda", dtype=t.float16), t.zeros(1, device="cuda", dtype=t.int32)
    kc, vc, q, k = c.clone(), c.clone(), t.randn(4, 2, 32, device="cuda"), t.randn(4, 2, 32, device="cuda")
    oq, ok, oa = t.empty_like(q), t.empty_like(k), t.empty_like(x)
    tok, prob = t.zeros(2, device="cuda", dtype=t.int32), t.zeros(2, device="cuda")
    logits, u = t.randn(2, 50, device="cuda"), t.rand(2, device="cuda")
    written, read = [kc, vc, oq, ok, oa, tok, prob], [q, k, x, n, logits, u]
    was = [a._version for a in written], [a._version for a in read]
    ops.qk_norm_rope(q, k, None, None, None, out_q=oq, out_k=ok)
    ops.kv_append(k, k, kc, vc, t.arange(4, device="cuda"))
    ops.tree_attention(x, kc, vc, n.view(1, 1), n, out=oa)
    ops.sample_tokens(logits, u, out=tok, out_prob=prob)
    assert all(a._version > b for a, b in zip(written, was[0])) and [a._version for a in read] == was[1]
    y = t.ones_like(kc, requires_grad=True)
    z = (y * kc).sum()
    ops.kv_append(k, k, kc, vc, t.arange(4, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z.backward()
    with t.inference_mode():
        i = t.zeros(1, 2, 8, 32, device="cuda", dtype=t.float16)
        ops.kv_append(k, k, i, i.clone(), t.arange(4, device="cuda"))


# ----------------------------------------------------------------------------------------------------------- arguments
def test_arguments_that_would_be_ignored_are_refused(t, ops):
    k = t.randn(4, 2, 32, device="cuda")
    c, s, w = t.zeros(1, 2, 8, 32, device="cuda", dtype=t.float16), t.arange(4, device="cuda"), t.ones(32, device="cuda")
    with pytest.raises(ValueError, match="out_q"):
        ops.kv_append(k, k, c, c.clone(), s, out_q=t.empty_like(k))
    with pytest.raises(ValueError, match="q_weight"):
        ops.kv_append(k, k, c, c.clone(), s, q_weight=w)


def test_an_interleaved_that_is_neither_true_nor_false_raises_its_own_error(t, ops):
    k = t.randn(4, 2, 32, device="cuda")
    with pytest.raises(RuntimeError, match="Boolean value"):
        ops.qk_norm_rope(k, k, None, None, None, interleaved=t.zeros(2))
    with pytest.raises(ZeroDivisionError):
        ops.qk_norm_rope(k, k, None, None, None, interleaved=type("X", (), {"__bool__": lambda self: 1 // 0})())
    assert all(t.equal(x, k) for x in ops.qk_norm_rope(k, k, None, None, None, interleaved=1))


# ------------------------------------------------------------------------------------------------------------ sampling
@pytest.mark.parametrize("vocab", [151936, 200001, 262145, 2 ** 22])
@pytest.mark.parametrize("kw", [dict(temperature=0.4, top_k=50), dict(top_k=5000, top_p=0.9), dict(top_p=0.95), dict(),
                                dict(temperature=0.8, min_p=0.02), dict(temperature=0.0), dict(top_k=1000)])
def test_sample_large_vocabularies(t, ops, vocab, kw):
    """Up to the largest: more chunks than a wave has lanes, more maxima than k_finish holds in registers, a thread a chunk;
    random numbers at both ends, rows at an odd stride."""
    g = t.Generator(device="cuda").manual_seed(vocab)
    u = t.tensor([0.37, 1 - 2.0 ** -24] if vocab == 2 ** 22 else [0.0, 0.37, 1 - 2.0 ** -24]).cuda()
    big = t.randn(len(u), vocab + 5, device="cuda", generator=g) * 3
    sampled(t, ops, big[:, 5:], u, **kw)
    if vocab != 2 ** 22:
        sampled(t, ops, big[1:2, :vocab].contiguous(), u[1:2], **kw)  # 16-byte aligned
