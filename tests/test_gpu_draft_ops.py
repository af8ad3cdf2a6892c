"""The drafted-token operators (fun_asr_gguf.ops) on the GPU against plain 64-bit forms (tests/draft_oracle.py).

Tolerances, from arithmetic (u = half a step of the output's type relative to the value, 2^-24 for float32):
  * norm + rotation: the sum of up to 512 squares (16 a lane, then log2 lanes), its root, reciprocal and the products stay
    within 32 * 2^-24 of |a| + |b| of the pair; then one rounding u |y| (float16: never under 2^-25, its subnormal step).
  * attention: scores are off by at most (D + 8) 2^-24 sum |q| |k| scale (float32 accumulation) plus, with float32 q, the
    term that splitting it drops (2^-21 of the same sum); weights by twice that plus 2^-20 (exponential, sums), plus the
    rounding of the weights themselves to 16 bits (u of the cache's type; float32 q: 2^-21); all times sum p |v|; the
    output's own rounding u |y| last.
  * sampling: tokens equal unless u * total lies within 1e-9 of a border; probabilities to float32.
"""
import numpy as np
import pytest
import torch  # noqa: F401  (before any engine: the library then shares torch's HIP runtime)

from draft_oracle import attention, norm_rope, sample

pytestmark = pytest.mark.gpu
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def t():
    import torch
    return torch


@pytest.fixture(scope="module")
def ops():
    from fun_asr_gguf import ops
    return ops


def kind(t, name):
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16}[name]


def wide(x):
    return None if x is None else x.double().cpu().numpy()


def tables(t, n, rot):
    a = t.arange(n, dtype=t.float64)[:, None] * t.pow(t.tensor(1e4, dtype=t.float64), -t.arange(rot // 2) * 2.0 / rot)[None]
    return a.cos().float().cuda(), a.sin().float().cuda()


def close(got, want, tol):
    got = wide(got)
    off = np.abs(got - want) - tol
    assert np.isfinite(got).all() and off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


# ------------------------------------------------------------------------------------------------- norm and rotation
ROWS = [  # tokens, heads, kv, D, rot, types, interleaved, norm
    (1, 16, 8, 128, 128, "bf16", False, True), (7, 16, 8, 128, 128, "f32", False, True),
    (33, 3, 1, 80, 32, "f16", True, True), (5, 8, 8, 64, 64, "bf16", True, False), (130, 6, 2, 96, 48, "f32", False, True),
    (2, 1, 1, 16, 16, "f16", False, True), (9, 2, 2, 512, 512, "bf16", False, True), (3, 4, 1, 256, 16, "f32", True, True),
    (1000, 4, 2, 112, 112, "bf16", False, True)]


def rows(t, seed, T, heads, D, name, pad=0):
    g = t.Generator().manual_seed(seed)
    x = t.randn(T, heads * D + pad, generator=g) * (0.2 + 4 * t.rand(T, 1, generator=g))
    return x.to(kind(t, name)).cuda()


@pytest.mark.parametrize("case", ROWS)
@pytest.mark.parametrize("odd", [0, 5])
def test_norm_rope(t, ops, case, odd):
    """Views of one projection, aligned and at odd strides; positions repeated, at the table's ends, int32 and int64."""
    T, H, KV, D, R, name, inter, norm = case
    x = rows(t, T, T, H + KV, D, name, odd)
    q, k = x[:, odd:odd + H * D].view(T, H, D) if not odd else x[:, odd:].unflatten(1, (H + KV, D))[:, :H], None
    k = (x[:, H * D:].view(T, KV, D) if not odd else x[:, odd:].unflatten(1, (H + KV, D))[:, H:])
    qw, kw = ((1 + 0.1 * t.randn(D)).cuda() if norm else None for _ in range(2))
    cos, sin = tables(t, 300, R)
    pos = t.randint(0, 300, (T,), dtype=t.int64 if odd else t.int32)
    pos[0], pos[-1] = 0, 299
    before = x.clone()
    oq, ok = ops.qk_norm_rope(q, k, cos, sin, pos.cuda(), qw, kw, eps=1e-5, interleaved=inter)
    assert t.equal(before, x)
    for got, src, w in ((oq, q, qw), (ok, k, kw)):
        y, size = norm_rope(wide(src), wide(w), wide(cos), wide(sin), pos.numpy(), 1e-5, inter)
        close(got, y, 32 * U["f32"] * size + U[name] * np.abs(y) + (2.0 ** -25 if name == "f16" else 0))
    # in place
    ops.qk_norm_rope(q, k, cos, sin, pos.cuda(), qw, kw, eps=1e-5, interleaved=inter, out_q=q, out_k=k)
    assert t.equal(q, oq) and t.equal(k, ok)


def test_norm_rope_without_rotation_zero_rows_and_positions_outside(t, ops):
    q, k = rows(t, 1, 6, 4, 64, "f32").view(6, 4, 64), rows(t, 2, 6, 2, 64, "f32").view(6, 2, 64)
    q[2] = 0
    w = t.ones(64).cuda()
    oq, ok = ops.qk_norm_rope(q, k, None, None, None, w, None)
    y, size = norm_rope(wide(q), np.ones(64), None, None, None, 1e-6, False)
    close(oq, y, 32 * U["f32"] * size + U["f32"] * np.abs(y))
    assert t.equal(ok, k)  # neither norm nor rotation: a copy
    cos, sin = tables(t, 10, 64)
    out_q, out_k = t.full_like(q, 7.0), t.full_like(k, 7.0)
    pos = t.tensor([0, -1, 9, 10, 2 ** 31 - 1, 3], dtype=t.int64).cuda()
    ops.qk_norm_rope(q, k, cos, sin, pos, w, w, out_q=out_q, out_k=out_k)
    bad = t.tensor([False, True, False, True, True, False]).cuda()
    assert (out_q[bad] == 7).all() and (out_k[bad] == 7).all() and not (out_k[~bad] == 7).any()
    empty = ops.qk_norm_rope(q[:0], k[:0], cos, sin, pos[:0], w, w)
    assert empty[0].shape == (0, 4, 64)


# -------------------------------------------------------------------------------------------------------------- append
def cache(t, pages, KV, page, D, name, order, seed=0, fill=None):
    """order "hpd": [pages, KV, page, D] contiguous; "phd": slots before heads."""
    shape = (pages, KV, page, D) if order == "hpd" else (pages, page, KV, D)
    g = t.Generator().manual_seed(seed)
    x = (t.randn(shape, generator=g) if fill is None else t.full(shape, fill)).to(kind(t, name)).cuda()
    return x if order == "hpd" else x.permute(0, 2, 1, 3)


@pytest.mark.parametrize("T,H,KV,D,R,name,cname,page,order,with_q", [
    (1, 16, 8, 128, 128, "bf16", "bf16", 16, "hpd", True), (37, 4, 2, 64, 32, "f32", "f16", 7, "phd", True),
    (100, 8, 1, 96, 96, "f16", "f16", 1, "hpd", False), (64, 2, 2, 80, 80, "f32", "bf16", 24, "hpd", True),
    (300, 6, 3, 256, 128, "bf16", "f16", 128, "phd", False)])
@pytest.mark.parametrize("wide_slots", [False, True])
def test_append(t, ops, T, H, KV, D, R, name, cname, page, order, with_q, wide_slots):
    pages = T // page + 3
    kc, vc = cache(t, pages, KV, page, D, cname, order, 1), cache(t, pages, KV, page, D, cname, order, 2)
    k, v, q = (rows(t, s, T, n, D, name).view(T, n, D) for s, n in ((3, KV), (4, KV), (5, H)))
    w = (1 + 0.1 * t.randn(D)).cuda()
    cos, sin = tables(t, 500, R)
    pos = t.randint(0, 500, (T,), dtype=t.int32)
    slots = t.randperm(pages * page)[:T].to(t.int64 if wide_slots else t.int32)
    if T > 4:
        slots[1], slots[2], slots[3] = -1, pages * page, -2 ** 31  # not appended
        pos[4] = 500                                               # left out
    want_k, want_v = kc.clone(), vc.clone()
    got = ops.kv_append(k, v, kc, vc, slots.cuda(), cos=cos, sin=sin, positions=pos.cuda(), k_weight=w,
                        q=q if with_q else None, q_weight=w if with_q else None)
    ok = ((slots >= 0) & (slots < pages * page) & (pos < 500)).numpy()
    y, size = norm_rope(wide(k), wide(w), wide(cos), wide(sin), np.minimum(pos.numpy(), 499), 1e-6, False)
    tol = 32 * U["f32"] * size + U[cname] * np.abs(y) + (2.0 ** -25 if cname == "f16" else 0)
    s = slots.numpy()[ok]
    a, b = wide(kc)[s // page, :, s % page], wide(vc)[s // page, :, s % page]
    assert (np.abs(a - y[ok]) <= tol[ok]).all()
    assert (b == wide(v.to(kind(t, cname)))[ok]).all()
    # everything else as it was
    s = t.from_numpy(s).cuda().long()
    for c, was in ((kc, want_k), (vc, want_v)):
        c[s // page, :, s % page] = 0
        was[s // page, :, s % page] = 0
        assert t.equal(c, was)
    if with_q:
        y, size = norm_rope(wide(q), wide(w), wide(cos), wide(sin), np.minimum(pos.numpy(), 499), 1e-6, False)
        live = (pos < 500).numpy()
        assert (np.abs(wide(got) - y)[live] <= (32 * U["f32"] * size + U[name] * np.abs(y) + 2.0 ** -25)[live]).all()
    else:
        assert got is None


# ----------------------------------------------------------------------------------------------------------- attention
def trees(t, B, N, seed):
    rng = np.random.default_rng(seed)
    p = np.array([[-1 if j == 0 else rng.integers(-1, j) for j in range(N)] for _ in range(B)]).reshape(B, N)
    from fun_asr_gguf.ops import tree_mask
    return tree_mask(t.from_numpy(p))


def paged(t, ctx, N, page, KV, D, name, order, seed, spare=2, fill=float("nan")):
    """Caches whose only finite values are those that the sequences hold; a random page order."""
    B = len(ctx)
    need = [-(-(c + N) // page) for c in ctx]
    pages = sum(need) + spare
    ids = np.random.default_rng(seed).permutation(pages)
    table = np.full((B, max(max(need), 1)), ids[-1], np.int32)
    kc, vc = (cache(t, pages, KV, page, D, name, order, fill=fill) for _ in range(2))
    g = t.Generator().manual_seed(seed)
    at = 0
    for b in range(B):
        table[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]
        pos = t.arange(ctx[b] + N)
        where = t.from_numpy(table[b]).long()[pos // page].cuda(), slice(None), (pos % page).cuda()
        for c in (kc, vc):
            c[where] = t.randn(len(pos), KV, D, generator=g).to(c.dtype).cuda()
    return kc, vc, t.from_numpy(table).cuda()


def tolerance(want, mass, reach, qname, cname, D):
    split = qname == "f32"
    score = (D + 8) * 2.0 ** -24 * reach + (2.0 ** -21 * reach if split else 0)
    p = 2 * score + 2.0 ** -20 + (2.0 ** -21 if split else U[cname])
    return p * mass + U[qname] * np.abs(want) + (2.0 ** -24 if qname == "f16" else 1e-30)


def check(t, ops, q, kc, vc, table, ctx, mask=None, drafts=None, names=("f16", "f16"), **kw):
    B, N, H, D = q.shape
    out = t.full_like(q, 9.0)
    ops.tree_attention(q, kc, vc, table, t.tensor(ctx, dtype=t.int32).cuda(), mask=None if mask is None else mask.cuda(),
                       draft_lens=None if drafts is None else t.tensor(drafts, dtype=t.int32).cuda(), out=out, **kw)
    m = None if mask is None else np.broadcast_to(mask.numpy().astype(bool), (B, N, N))
    kn, vn = np.nan_to_num(wide(kc)), np.nan_to_num(wide(vc))
    want, mass, reach = attention(wide(q), kn, vn, table.cpu().numpy(), ctx, drafts or [N] * B, m, kw.get("scale") or D ** -0.5)
    left = np.isnan(want)
    assert (wide(out)[left] == 9.0).all()
    close(t.from_numpy(np.where(left, 0, wide(out))), np.where(left, 0, want),
          tolerance(np.where(left, 0, want), mass, reach, *names, D))
    return out


ATTN = [  # ctx, N, H, KV, D, q, cache, page, order, mask
    ([0], 1, 1, 1, 64, "f16", "f16", 16, "hpd", None), ([1, 31, 32, 33], 1, 16, 8, 128, "bf16", "bf16", 16, "hpd", None),
    ([204], 8, 16, 8, 128, "f32", "f16", 16, "hpd", "tree"), ([5, 700, 0], 16, 4, 2, 128, "bf16", "bf16", 24, "phd", "tree"),
    ([127, 128, 129], 3, 6, 2, 96, "f16", "f16", 7, "hpd", None), ([300, 4], 33, 7, 1, 64, "f32", "bf16", 1, "phd", "tree"),
    ([513], 64, 4, 2, 128, "f16", "f16", 64, "hpd", "tree"), ([77, 1000], 5, 4, 4, 256, "bf16", "bf16", 128, "hpd", "tree"),
    ([60], 20, 8, 1, 256, "f32", "f16", 16, "phd", None), ([2000, 9, 512], 2, 3, 1, 40, "f16", "f16", 32, "hpd", "tree"),
    ([100], 130, 2, 2, 64, "bf16", "bf16", 16, "hpd", None), ([90, 17], 12, 8, 2, 8, "f32", "bf16", 16, "hpd", "tree"),
    ([5000, 1], 9, 8, 2, 128, "bf16", "bf16", 256, "hpd", "tree"), ([3000], 40, 8, 1, 128, "f16", "f16", 48, "phd", "tree")]


@pytest.mark.parametrize("case", ATTN)
def test_attention(t, ops, case):
    """Against the formula; every value that no row may see is NaN."""
    ctx, N, H, KV, D, qn, cn, page, order, mk = case
    kc, vc, table = paged(t, ctx, N, page, KV, D, cn, order, 3)
    q = (2 * t.randn(len(ctx), N, H, D, generator=t.Generator().manual_seed(4))).to(kind(t, qn)).cuda()
    mask = trees(t, len(ctx), N, 5) if mk else None
    a = check(t, ops, q, kc, vc, table, ctx, mask, names=(qn, cn))
    assert t.equal(a, check(t, ops, q, kc, vc, table, ctx, mask, names=(qn, cn)))  # the same bits again
    # a bound on the context that is far too low, and a tight one: other splits, the same result
    check(t, ops, q, kc, vc, table, ctx, mask, names=(qn, cn), max_context=1)
    check(t, ops, q, kc, vc, table, ctx, mask, names=(qn, cn), max_context=max(max(ctx), 1), scale=0.3)


def test_attention_ragged_drafts_empty_rows_and_shared_mask(t, ops):
    ctx, N = [50, 0, 3, 400, 0], 6
    kc, vc, table = paged(t, ctx, N, 16, 2, 64, "bf16", "hpd", 7)
    q = t.randn(5, N, 4, 64).to(t.bfloat16).cuda()
    mask = t.zeros(N, N, dtype=t.bool)  # node 0 sees itself; 1 and 2 nothing; the others node 0
    mask[0, 0] = mask[3, 0] = mask[4, 0] = mask[5, 0] = True
    for drafts in ([6, 6, 6, 6, 6], [0, 3, 1, 6, -4], [9, 2, 0, 5, 1]):
        out = check(t, ops, q, kc, vc, table, ctx, mask, drafts, names=("bf16", "bf16"))
    assert (out[1, 1] == 0).all()  # no context, an empty mask row
    # strides: q and out as views with other orders, a byte mask of which only a part is used
    big = t.randn(N, 5, 4, 80).to(t.bfloat16).cuda()
    qv = big.permute(1, 0, 2, 3)[..., 3:67]
    bytes_ = t.zeros(5, 11, 13, dtype=t.uint8)
    bytes_[:, :N, :N] = t.eye(N, dtype=t.uint8) * 3
    want = check(t, ops, qv, kc, vc, table, ctx, t.eye(N, dtype=t.bool), names=("bf16", "bf16"))
    got = ops.tree_attention(qv, kc, vc, table, t.tensor(ctx, dtype=t.int32).cuda(), mask=bytes_.cuda()[:, :N, :N])
    assert t.equal(got, want)


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("what", [float("inf"), float("-inf"), float("nan")])
def test_attention_nonfinite_drafts_reach_only_those_that_see_them(t, ops, name, what):
    ctx, N, D = [45], 9, 128
    kc, vc, table = paged(t, ctx, N, 16, 2, D, name, "hpd", 8)
    q = t.randn(1, N, 4, D).to(kind(t, name)).cuda()
    mask = trees(t, 1, N, 9)
    mask[0, 8, 4] = True
    clean = check(t, ops, q, kc, vc, table, ctx, mask, names=(name, name))
    p = 45 + 4
    at = int(table[0, p // 16]), slice(None), p % 16
    seers = mask[0, :, 4]
    for c, d in ((vc, 3), (vc, 77), (kc, 5)):
        keep = c[at].clone()
        c[at[0], :, at[2], d] = what
        out = ops.tree_attention(q, kc, vc, table, t.tensor(ctx, dtype=t.int32).cuda(), mask=mask.cuda())
        assert t.equal(out[0, ~seers], clean[0, ~seers])
        if c is vc:
            hit = out[0, seers][..., d]
            assert (hit.isnan().all() if what != what else (hit == what).all())
            rest = [x for x in range(D) if x != d]
            assert t.equal(out[0, seers][..., rest], clean[0, seers][..., rest])
        c[at] = keep


def test_attention_bad_pages_lengths_and_tables(t, ops):
    """Page numbers outside the cache make their keys absent; lengths are cut to the table."""
    ctx, N = [100, 64, 200], 4
    kc, vc, table = paged(t, ctx, N, 16, 2, 64, "f16", "hpd", 10, fill=0.5)
    q = t.randn(3, N, 2, 64).half().cuda()
    table[0, 2], table[0, 6], table[1] = -1, kc.shape[0], 2 ** 31 - 1
    check(t, ops, q, kc, vc, table, ctx, names=("f16", "f16"))
    table[1] = table[2]
    check(t, ops, q, kc, vc, table, [10 ** 6, -5, 200], names=("f16", "f16"))
    out = ops.tree_attention(q[:0], kc, vc, table[:0], t.zeros(0, dtype=t.int32).cuda())
    assert out.shape == (0, N, 2, 64)
    assert ops.tree_attention(q[:, :0], kc, vc, table, t.zeros(3, dtype=t.int32).cuda()).shape == (3, 0, 2, 64)


def test_attention_and_append_behind_32_bit_offsets(t, ops):
    """A cache of more than 2^32 bytes and 2^31 elements: pages at both ends."""
    KV, page, D = 8, 64, 128
    pages = 2 ** 31 // (KV * page * D) + 40
    kc, vc = (t.empty(pages, KV, page, D, dtype=t.float16, device="cuda") for _ in range(2))
    ctx, N = 500, 3
    ids = t.cat([t.arange(pages - 5, pages), t.arange(4)])
    T = ctx + N
    slots = ids.repeat_interleave(page)[:T] * page + t.arange(T) % page
    k, v = t.randn(T, KV, D).half().cuda(), t.randn(T, KV, D).half().cuda()
    ops.kv_append(k, v, kc, vc, slots.cuda())
    at = (slots // page).cuda(), slice(None), (slots % page).cuda()
    assert t.equal(kc[at], k) and t.equal(vc[at], v)
    q = t.randn(1, N, 16, D).half().cuda()
    out = ops.tree_attention(q, kc, vc, ids[None].int().cuda(), t.tensor([ctx], dtype=t.int32).cuda())
    small = t.zeros(8, KV, page, D, dtype=t.float16, device="cuda"), t.zeros(8, KV, page, D, dtype=t.float16, device="cuda")
    for c, x in zip(small, (k, v)):
        pos = t.arange(T).cuda()
        c[pos // page, :, pos % page] = x
    table = t.arange(9, dtype=t.int32)[None].cuda().clamp(max=7)
    assert t.equal(out, ops.tree_attention(q, *small, table, t.tensor([ctx], dtype=t.int32).cuda()))


# ------------------------------------------------------------------------------------------------------------ sampling
def sampled(t, ops, x, u, check_prob=True, **kw):
    got, prob = ops.sample_tokens(x, u, **kw)
    rows = x.shape[0]
    per = {n: (wide(kw[n]) if isinstance(kw.get(n), t.Tensor) else np.full(rows, np.float32(kw.get(n, d))))
           for n, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))}
    xs, us = wide(x), wide(u)
    for r in range(rows):
        tok, p, gap = sample(xs[r], us[r], *(np.float32(per[n][r]) if n != "top_k" else int(per[n][r])
                                             for n in ("temperature", "top_k", "top_p", "min_p")))
        if gap > 1e-9:
            assert int(got[r]) == tok, (r, int(got[r]), tok, gap)
            assert abs(float(prob[r]) - p) <= 2.0 ** -23 * p + 1e-9
    return got


def logits(t, rows, vocab, name, spread, seed):
    g = t.Generator().manual_seed(seed)
    x = t.randn(rows, vocab, generator=g) * spread
    return x.to(kind(t, name)).cuda(), t.rand(rows, generator=g).cuda()


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 1000, 4097, 60515])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kw", [
    dict(), dict(temperature=0.4, top_k=50), dict(top_p=0.9), dict(temperature=0.7, top_k=900, top_p=0.5, min_p=0.01),
    dict(min_p=0.1, temperature=1.5), dict(temperature=0.0), dict(top_k=1), dict(top_k=5000, top_p=0.999),
    dict(top_p=0.0), dict(top_p=1e-6), dict(min_p=1.0, temperature=2.0)])
def test_sample(t, ops, vocab, name, kw):
    x, u = logits(t, 5, vocab, name, 3.0, vocab)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    sampled(t, ops, x, u, **kw)


@pytest.mark.parametrize("kw", [dict(top_k=7), dict(top_k=5000), dict(top_p=0.3), dict(top_k=20000, top_p=0.77),
                                dict(min_p=0.5), dict(), dict(temperature=0.0)])
@pytest.mark.parametrize("values", [1, 2, 5])
def test_sample_ties(t, ops, kw, values):
    """Rows of a few distinct values (one: all tokens equal): ties rank by id, and a border falls exactly on one."""
    vocab = 30000
    x = t.randint(0, values, (4, vocab), generator=t.Generator().manual_seed(values)).float().cuda()
    sampled(t, ops, x, t.tensor([0.0, 0.25, 0.5, 0.9]).cuda(), **kw)


def test_sample_infinities_nans_zeros_and_empty_rows(t, ops):
    inf, nan = float("inf"), float("nan")
    x = t.full((9, 5000), -inf)
    x[1, 77] = -3.4e38
    x[2, 5:900] = nan
    x[3] = nan
    x[3, 4000] = 1.0
    x[4, 10], x[4, 4000], x[4, 20] = inf, inf, 3.0
    x[5, ::2], x[5, 1::2] = 0.0, -0.0
    x[6] = t.linspace(-3e38, 3e38, 5000)
    x[7] = 1e-42 * t.arange(5000)
    x[8, 3000:] = -100.0
    x = x.cuda()
    u = t.tensor([.5, .5, .5, .5, .75, .999, .3, .6, .5]).cuda()
    for kw in (dict(), dict(top_k=2), dict(top_k=40, top_p=.6), dict(top_p=.5), dict(min_p=.5), dict(temperature=0.),
               dict(temperature=1e-30), dict(temperature=1e30, top_k=3000)):
        got = sampled(t, ops, x, u, **kw).tolist()
        assert got[0] == -1 and got[1] == 77 and got[2] == -1 and got[3] == 4000 and got[4] in (10, 4000)
    assert ops.sample_tokens(x[:0], u[:0])[0].shape == (0,)


def test_sample_settings_of_each_row_and_strides(t, ops):
    """Per-row settings equal one-row calls with numbers; rows at odd strides and offsets; no probabilities asked for."""
    x, u = logits(t, 24, 9001, "bf16", 2.5, 3)
    big = t.zeros(24, 9100, dtype=t.bfloat16).cuda()
    big[:, 13:9014] = x
    view = big[:, 13:9014]
    temp = t.tensor([0.0, 0.3, 1.0, 2.0] * 6).cuda()
    k = t.tensor([0, 1, 10, 2000, 9001, 50000] * 4, dtype=t.int32).cuda()
    p = t.tensor([1.0, 0.2, 0.95] * 8).cuda()
    m = t.tensor([0.0, 0.0, 0.0, 0.3, 0.01] * 5).cuda()[:24].contiguous()
    got = sampled(t, ops, view, u, temperature=temp, top_k=k, top_p=p, min_p=m)
    for r in range(24):
        one, _ = ops.sample_tokens(x[r:r + 1], u[r:r + 1], temperature=float(temp[r]), top_k=int(k[r]), top_p=float(p[r]),
                                   min_p=float(m[r]))
        assert int(one) == int(got[r])


def test_sample_follows_its_distribution(t, ops):
    """20 000 evenly spread numbers on one row: every token's share is its probability."""
    x = t.randn(1, 500, generator=t.Generator().manual_seed(1)).cuda() * 2
    n = 20000
    u = (t.arange(n) + 0.5).div(n).float().cuda()
    got, prob = ops.sample_tokens(x.expand(n, 500).contiguous(), u, temperature=0.8, top_k=30)
    w = t.softmax(x[0].double() / 0.8, 0)
    keep = x[0].topk(30).indices
    want = t.zeros(500, dtype=t.float64).cuda()
    want[keep] = w[keep] / w[keep].sum()
    share = t.bincount(got.long(), minlength=500).double() / n
    assert float((share - want).abs().max()) <= 1.5 / n
    assert float((prob.double() - want[got.long()]).abs().max()) <= 1e-6


# ------------------------------------------------------------------------------------------------------- as they are used
def step(t, ops, s):
    """One verifying step of a layer: append with norm and rotation, attend the tree, sample from a projection."""
    B, N, H, KV, D = s["dims"]
    q = ops.kv_append(s["k"], s["v"], s["kc"], s["vc"], s["slots"], cos=s["cos"], sin=s["sin"], positions=s["pos"],
                      k_weight=s["kw"], q=s["q"], q_weight=s["qw"])
    o = ops.tree_attention(q.view(B, N, H, D), s["kc"], s["vc"], s["table"], s["ctx"], mask=s["mask"])
    return (o, *ops.sample_tokens(o.reshape(B * N, H * D).float() @ s["w"], s["u"], temperature=0.7, top_k=40, top_p=0.9,
                                  min_p=0.02))


def make_step(t, seed):
    B, N, H, KV, D, page = 3, 7, 8, 2, 64, 16
    ctx = [40, 5, 90]
    kc, vc, table = paged(t, ctx, N, page, KV, D, "f16", "hpd", seed)
    g = t.Generator().manual_seed(seed)
    x = t.randn(B * N, (H + 2 * KV) * D, generator=g).half().cuda()
    mask = trees(t, B, N, seed)
    depth = mask.sum(-1) - 1
    c = t.tensor(ctx)
    pos = (c[:, None] + depth).flatten()
    at = (c[:, None] + t.arange(N)).flatten()
    row = t.arange(B).repeat_interleave(N)
    slots = table.cpu()[row, at // page].long() * page + at % page
    cos, sin = tables(t, 200, D)
    return dict(dims=(B, N, H, KV, D), q=x[:, :H * D].view(-1, H, D), k=x[:, H * D:(H + KV) * D].view(-1, KV, D),
                v=x[:, (H + KV) * D:].view(-1, KV, D), kc=kc, vc=vc, table=table, ctx=c.int().cuda(), mask=mask.cuda(),
                slots=slots.cuda(), pos=pos.cuda(), cos=cos, sin=sin, qw=(1 + .1 * t.randn(D, generator=g)).cuda(),
                kw=(1 + .1 * t.randn(D, generator=g)).cuda(), w=(t.randn(H * D, 3001, generator=g) * .3).cuda(),
                u=t.rand(B * N, generator=g).cuda())


def test_a_verifying_step(t, ops):
    s = make_step(t, 21)
    B, N, H, KV, D = s["dims"]
    kn, vn = np.nan_to_num(wide(s["kc"])), np.nan_to_num(wide(s["vc"]))
    o, tok, prob = step(t, ops, s)
    pos, slots = s["pos"].cpu().numpy(), s["slots"].cpu().numpy()
    q, _ = norm_rope(wide(s["q"]), wide(s["qw"]), wide(s["cos"]), wide(s["sin"]), pos, 1e-6, False)
    k, _ = norm_rope(wide(s["k"]), wide(s["kw"]), wide(s["cos"]), wide(s["sin"]), pos, 1e-6, False)
    kn[slots // 16, :, slots % 16] = k
    vn[slots // 16, :, slots % 16] = wide(s["v"])
    want, mass, reach = attention(q.reshape(B, N, H, D), kn, vn, s["table"].cpu().numpy(), s["ctx"].tolist(), [N] * B,
                                  s["mask"].cpu().numpy(), D ** -0.5)
    # q and k were rounded to float16 on the way: each score moves by up to 2 * 2^-11 of sum |q| |k|
    tol = tolerance(want, mass, reach, "f16", "f16", D) + 2 * (2 * 2.0 ** -11 * reach) * mass
    close(o, want, tol)
    x = o.reshape(B * N, H * D).float() @ s["w"]
    sampled(t, ops, x, s["u"], temperature=0.7, top_k=40, top_p=0.9, min_p=0.02)


def test_steps_in_graphs_on_streams_and_at_once(t, ops):
    """Two captured steps replayed between eager work, on streams of their own and at the same time: always the eager bits."""
    a, b = make_step(t, 31), make_step(t, 32)
    want = [[x.clone() for x in step(t, ops, s)] for s in (a, b)]
    graphs, outs = [], []
    for s in (a, b):
        side = t.cuda.Stream()
        side.wait_stream(t.cuda.current_stream())
        with t.cuda.stream(side):
            step(t, ops, s)
        t.cuda.current_stream().wait_stream(side)
        g = t.cuda.CUDAGraph()
        with t.cuda.graph(g):
            outs.append(step(t, ops, s))
        graphs.append(g)
    streams = [t.cuda.Stream(), t.cuda.Stream()]
    for turn in range(4):
        t.cuda.synchronize()
        for o in outs:
            for x in o:
                x.zero_()
        t.cuda.synchronize()
        if turn % 2:
            for g in graphs:
                g.replay()
        else:
            for g, st in zip(graphs, streams):
                with t.cuda.stream(st):
                    g.replay()
        t.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(t.equal(x, y) for x, y in zip(o, w))
        got = step(t, ops, a)  # eager work in between
        assert all(t.equal(x, y) for x, y in zip(got, want[0]))
    t.cuda.synchronize()
    res = []
    for s, st in zip((a, b), streams):
        with t.cuda.stream(st):
            res.append([step(t, ops, s) for _ in range(3)])
    t.cuda.synchronize()
    for group, w in zip(res, want):
        for o in group:
            assert all(t.equal(x, y) for x, y in zip(o, w))


@pytest.mark.parametrize("dim", [16, 32, 48, 112, 144, 176, 208, 336, 512])
def test_norm_rope_of_every_group(t, ops, dim):
    """Rows of 1 to 32 lanes, a wave's lanes used up or not, more rows than a block; a row of huge, one of tiny values."""
    g = t.Generator(device="cuda").manual_seed(dim)
    q = t.randn(67, 5, dim, device="cuda", generator=g)
    k = t.randn(67, 1, dim, device="cuda", generator=g)
    q[3, 1] *= 1e12
    q[4, 2] *= 1e-12
    w = t.rand(dim, device="cuda", generator=g) + 0.5
    ang = t.rand(80, 8, device="cuda", generator=g) * 6
    cos, sin = ang.cos(), ang.sin()
    pos = t.arange(67, device="cuda", dtype=t.int32)
    got = ops.qk_norm_rope(q, k, cos, sin, pos, w, None, eps=1e-30)
    for y, x, wt in zip(got, (q, k), (w, None)):
        ref, size = norm_rope(wide(x), None if wt is None else wide(wt), wide(cos), wide(sin), wide(pos).astype(int), 1e-30, False)
        err = np.abs(wide(y) - ref)
        assert (err <= 32 * 2.0 ** -24 * size + U["f32"] * np.abs(ref)).all(), (err / (size + 1e-300)).max()


def test_outputs_that_share_memory_gradients_and_negated_views_are_refused(t, ops):
    q = t.randn(4, 2, 32, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        ops.qk_norm_rope(q, q, None, None, None, out_q=t.zeros(1, 2, 32, device="cuda").expand(4, 2, 32))
    c = t.zeros(1, 2, 8, 32, device="cuda", dtype=t.float16)
    s = t.arange(4, device="cuda")
    for kw in [dict(k_cache=c.expand(3, 2, 8, 32), v_cache=c), dict(k_cache=c, v_cache=c[:, :1].expand(1, 2, 8, 32))]:
        with pytest.raises(ValueError):
            ops.kv_append(q, q, slots=s, **kw)
    x, n = t.randn(1, 2, 4, 32, device="cuda", dtype=t.float16), t.zeros(1, device="cuda", dtype=t.int32)
    kw = dict(k_cache=c, v_cache=c, block_table=n.view(1, 1), context_lens=n)
    with pytest.raises(ValueError, match="share memory"):
        ops.tree_attention(x, out=x[:, :1].clone().expand(1, 2, 4, 32), **kw)
    with pytest.raises(ValueError, match="gradient"):
        ops.tree_attention(x.clone().requires_grad_(), **kw)
    with t.no_grad():
        ops.tree_attention(x.clone().requires_grad_(), **kw)
    with pytest.raises(ValueError, match="negated"):
        ops.tree_attention(t._neg_view(x), **kw)
    with pytest.raises(ValueError, match="gradient"):
        ops.sample_tokens(t.zeros(2, 8, device="cuda"), t.zeros(2, device="cuda").requires_grad_())
