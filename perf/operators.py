"""What the drafted-token operators of the decoder are measured on: their cases, inputs, plain forms and 64-bit results.

A decoding step that verifies drafted tokens runs these one after the other:

* ``qk_norm_rope``: every head row of q and k divided by its root mean square, weighted, and rotated by its position;
* ``kv_append``: the same for k (and, where given, q) with k and v written into the pages of a cache on the way;
* ``tree_attention``: the drafted tokens' attention over the paged cache, each of them seeing the committed tokens and
  its own ancestors in the draft tree (one token a sequence: an ordinary decoding step);
* ``sample_tokens``: a token for every row of logits, from top-k, top-p, min-p, temperature and a given random number.

``own`` false: elementary torch operations in 32 bits (64 where a value lies next to a border). True: the framework's
entry points in ``fun_asr_gguf.ops``.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_ops = None


def _framework():
    global _ops
    if _ops is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fun-asr-gguf_amd"))
        from fun_asr_gguf import ops
        _ops = ops
    return _ops


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decoded token of the speech decoder's shape (16 query heads, 8 kv heads of 128): latency
        dict(name="norm_rope 1 token", op="qk_norm_rope", tokens=1, heads=16, kv_heads=8, dim=128, rot=128, inter=False,
             types="bf16", norm=True, table=2048),
        # the prompts of a 32-clip batch (32 x 204 rows), float32 rows as the engine's projections give them
        dict(name="norm_rope 32 prompts", op="qk_norm_rope", tokens=6528, heads=16, kv_heads=8, dim=128, rot=128,
             inter=False, types="f32", norm=True, table=2048),
        # a long prompt batch of another head layout: partial rotation of neighbouring pairs, odd length
        dict(name="norm_rope long, partial", op="qk_norm_rope", tokens=16381, heads=24, kv_heads=8, dim=80, rot=32,
             inter=True, types="f16", norm=True, table=8192),
        # a decoding step of 6 sequences, q in the same call
        dict(name="append 6 tokens + q", op="kv_append", tokens=6, heads=16, kv_heads=8, dim=128, rot=128, inter=False,
             types="bf16", cache="bf16", norm=True, table=2048, page=16, pages=192, pad=0),
        # the prompts of a 32-clip batch into a float16 cache, q in the same call, the last rows padding
        dict(name="append 32 prompts + q", op="kv_append", tokens=6528, heads=16, kv_heads=8, dim=128, rot=128,
             inter=False, types="f32", cache="f16", norm=True, table=2048, page=64, pages=160, pad=17),
        # keys and values of a long prompt, no norms, rotation only
        dict(name="append long prompt", op="kv_append", tokens=16384, heads=0, kv_heads=8, dim=64, rot=64, inter=False,
             types="bf16", cache="bf16", norm=False, table=32768, page=32, pages=1024, pad=0),
        # one clip: 8 drafted tokens behind a 204-row prompt, the engine's types (float32 rows, float16 cache)
        dict(name="tree 1 clip", op="tree_attention", seqs=1, nodes=8, heads=16, kv_heads=8, dim=128, ctx=204,
             ragged=False, q="f32", cache="f16", page=16, mask="tree"),
        # 32 clips of ragged lengths, 16 drafted tokens each
        dict(name="tree 32 clips", op="tree_attention", seqs=32, nodes=16, heads=16, kv_heads=8, dim=128, ctx=2032,
             ragged=True, q="bf16", cache="bf16", page=64, mask="tree"),
        # a few long transcripts with wide trees
        dict(name="tree long", op="tree_attention", seqs=4, nodes=63, heads=32, kv_heads=8, dim=128, ctx=32685,
             ragged=False, q="bf16", cache="bf16", page=256, mask="tree"),
        # ordinary decoding of many sequences: one token each
        dict(name="decode 48 sequences", op="tree_attention", seqs=48, nodes=1, heads=32, kv_heads=8, dim=128, ctx=8191,
             ragged=True, q="f16", cache="f16", page=16, mask="none"),
        # the sampler chain of one sequence at the decoder's vocabulary and the default settings
        dict(name="sample 1 row", op="sample", rows=1, vocab=151936, types="f32", temperature=0.4, top_k=50, top_p=1.0,
             min_p=0.0, per_row=False, spread=2.5),
        # a batch whose rows come with settings of their own, most without a top-k
        dict(name="sample 61 rows", op="sample", rows=61, vocab=151936, types="f32", temperature=0.9, top_k=0, top_p=0.95,
             min_p=0.0, per_row=True, spread=2.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["qk_norm_rope", "kv_append", "tree_attention", "tree_attention", "sample"])
    if op in ("qk_norm_rope", "kv_append"):
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([dim, dim, dim // 32 * 16])
        heads = kv * group
        tokens = _log(rng, 1, min(20000, 40_000_000 // ((heads + 2 * kv) * dim)))
        types = rng.choice(["f32", "f16", "bf16"])
        case = dict(op=op, tokens=tokens, heads=heads, kv_heads=kv, dim=dim, rot=rot, inter=rng.random() < 0.3,
                    types=types, norm=rng.random() < 0.8, table=max(2048, tokens))
        if op == "kv_append":
            page = rng.choice([16, 24, 64, 128, 256])
            case.update(heads=rng.choice([0, heads]), page=page, pages=tokens // page + rng.randint(2, 40),
                        cache=types if types != "f32" else rng.choice(["f16", "bf16"]),
                        pad=rng.randint(0, tokens // 4))
        return case
    if op == "tree_attention":
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 7, 8])
        dim = rng.choice([64, 96, 128, 256])
        nodes = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 2, 64)])
        seqs = _log(rng, 1, 64)
        most = min(40000, 100_000_000 // (seqs * kv * dim), 33_000_000_000 // (seqs * nodes * kv * group * dim))
        cache = rng.choice(["f16", "bf16"])
        return dict(op=op, seqs=seqs, nodes=nodes, heads=kv * group, kv_heads=kv, dim=dim, ctx=_log(rng, 1, max(64, most)),
                    ragged=rng.random() < 0.7, q=rng.choice([cache, cache, "f32"]), cache=cache,
                    page=rng.choice([16, 24, 64, 128, 256]), mask="none" if nodes == 1 else rng.choice(["tree", "none"]))
    vocab = _log(rng, 1000, 151936)
    return dict(op="sample", rows=_log(rng, 1, min(256, 9_000_000 // vocab)), vocab=vocab,
                types=rng.choice(["f32", "f32", "f16", "bf16"]), temperature=rng.choice([0.0, 0.4, 0.8, 1.0, 1.5]),
                top_k=rng.choice([0, 0, 1, 20, 50, 900, 5000]), top_p=rng.choice([1.0, 0.5, 0.9, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.2]), per_row=rng.random() < 0.4, spread=rng.choice([0.5, 1.5, 2.5, 4.0]))


def _lengths(case):
    """Committed tokens of each sequence: all of them ctx, or from ctx down to a quarter of it."""
    n, c = case["seqs"], case["ctx"]
    return [c - (3 * c * b) // (4 * n) if case["ragged"] else c for b in range(n)]


# --------------------------------------------------------------------------------------------------------------- inputs
def _tables(case):
    r, p = case["rot"], case["table"]
    a = torch.arange(p, device=DEV, dtype=torch.float64)[:, None] * \
        torch.pow(1e6, -2.0 * torch.arange(r // 2, device=DEV, dtype=torch.float64) / r)[None]
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=DEV) * scale

    s = dict(op=case["op"])
    if case["op"] in ("qk_norm_rope", "kv_append"):
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        # the rows of one projection, heads of q, then k, then v: the operators get strided views of it
        x = (normal(t, (h + 2 * kv) * d) * (0.5 + torch.rand(t, 1, generator=g, device=DEV) * 3)).to(TYPES[case["types"]])
        s["q"] = x[:, :h * d].view(t, h, d) if h else None
        s["k"] = x[:, h * d:(h + kv) * d].view(t, kv, d)
        s["v"] = x[:, (h + kv) * d:].view(t, kv, d)
        s["q_weight"] = 1 + normal(d, scale=0.1) if case["norm"] and h else None
        s["k_weight"] = 1 + normal(d, scale=0.1) if case["norm"] else None
        s["cos"], s["sin"] = _tables(case)
        s["positions"] = torch.randint(0, case["table"], (t,), generator=g, device=DEV, dtype=torch.int32)
        s["interleaved"], s["eps"] = case["inter"], 1e-6
        if case["op"] == "kv_append":
            page, pages = case["page"], case["pages"]
            shape = (pages + 1, kv, page, d)  # the last page belongs to nobody
            s["k_cache"], s["v_cache"] = (normal(*shape).to(TYPES[case["cache"]]) for _ in range(2))
            slots = torch.randperm(pages * page, generator=g, device=DEV)[:t]
            if case["pad"]:
                slots[t - case["pad"]:] = -1
            s["slots"] = slots
        return s
    if case["op"] == "tree_attention":
        b, n, h, kv, d, page = (case[k] for k in ("seqs", "nodes", "heads", "kv_heads", "dim", "page"))
        lens = _lengths(case)
        order = torch.randperm(b, generator=g, device=DEV).tolist()
        lens = [lens[i] for i in order]
        wide = -(-(case["ctx"] + n) // page)
        need = [-(-(c + n) // page) for c in lens]
        pages = sum(need)
        ids = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        table = torch.zeros(b, wide, dtype=torch.int32, device=DEV)
        at = 0
        for i in range(b):
            table[i, :need[i]] = ids[at:at + need[i]]
            at += need[i]
        s["k_cache"], s["v_cache"] = (normal(pages, kv, page, d).to(TYPES[case["cache"]]) for _ in range(2))
        s["q"] = normal(b, n, h, d, scale=2.0).to(TYPES[case["q"]])
        s["block_table"], s["context_lens"] = table, torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["max_context"] = case["ctx"]
        s["mask"] = None
        if case["mask"] == "tree":  # node 0 is the token sampled last, every other one hangs from an earlier one
            parent = torch.zeros(b, n, dtype=torch.int64)
            r = torch.rand(b, n, generator=g, device=DEV).cpu()
            for j in range(1, n):
                parent[:, j] = (r[:, j] * j).long()
            m = torch.zeros(b, n, n, dtype=torch.bool)
            for j in range(n):
                if j:
                    m[:, j] = m[torch.arange(b), parent[:, j]]
                m[:, j, j] = True
            s["mask"] = m.to(DEV)
        return s
    r, v = case["rows"], case["vocab"]
    # a body of unlikely tokens, a likely few that differ from row to row
    x = normal(r, v, scale=case["spread"])
    top = torch.randint(0, v, (r, 8), generator=g, device=DEV)
    x.scatter_add_(1, top, normal(r, 8).abs() * 2.0 * case["spread"] + case["spread"])
    s["logits"] = x.to(TYPES[case["types"]])
    s["u"] = torch.rand(r, generator=g, device=DEV)
    for k, kind in (("temperature", torch.float32), ("top_k", torch.int32), ("top_p", torch.float32), ("min_p", torch.float32)):
        s[k] = case[k]
        if case["per_row"]:  # every eighth row: greedy; another eighth: a top-k; another: a min-p; another: nothing but temperature
            t = torch.full((r,), case[k], dtype=kind, device=DEV)
            i = torch.arange(r, device=DEV) % 8
            if k == "temperature":
                t[i == 1] = 0.0
            if k == "top_k":
                t[i == 2] = 40
            if k == "min_p":
                t[i == 3] = 0.05
            if k == "top_p":
                t[i == 4] = 1.0
            s[k] = t
    return s


# ---------------------------------------------------------------------------------------------------------- plain forms
def _norm_rope(x, w, cos, sin, positions, eps, inter):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
    c, n = cos[positions.long()][:, None], sin[positions.long()][:, None]
    r = 2 * cos.shape[1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :r // 2], x[..., r // 2:r])
    y, z = a * c - b * n, a * n + b * c
    y = torch.stack((y, z), -1).flatten(-2) if inter else torch.cat((y, z), -1)
    return torch.cat((y, x[..., r:]), -1)


def _put(cache, slots, rows):
    page = cache.shape[2]
    pad = slots < 0  # padding goes, unchanged, to the page that belongs to nobody
    at = torch.where(pad, torch.full_like(slots, cache.shape[0] * page - 1), slots)
    p, o = at // page, at % page
    cache[p, :, o] = torch.where(pad[:, None, None], cache[p, :, o], rows.to(cache.dtype))


def _attention(s):
    q, mask = s["q"], s["mask"]
    b, n, h, d = q.shape
    kv, page = s["k_cache"].shape[1:3]
    g, length = h // kv, s["block_table"].shape[1] * page
    k, v = (c[s["block_table"].long()].permute(0, 2, 1, 3, 4).reshape(b, kv, length, d).float()
            for c in (s["k_cache"], s["v_cache"]))
    x = q.float().view(b, n, kv, g, d).permute(0, 2, 3, 1, 4).reshape(b, kv, g * n, d)
    x = torch.matmul(x, k.transpose(-1, -2)).view(b, kv, g, n, length) * (1.0 / math.sqrt(d))
    if mask is None:
        mask = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()[None]
    j = torch.arange(length, device=q.device)[None] - s["context_lens"][:, None]  # the draft's index of a key
    drafted = mask.expand(b, n, n).gather(2, j.clamp(0, n - 1)[:, None].expand(b, n, length))
    seen = torch.where((j < 0)[:, None], True, drafted & (j < n)[:, None])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = x.sum(-1, keepdim=True)
    x = torch.matmul(x.view(b, kv, g * n, length), v).view(b, kv, g, n, d) / torch.where(total == 0, 1.0, total)
    return x.permute(0, 3, 1, 2, 4).reshape(b, n, h, d).to(q.dtype)


def _column(x, like, kind):
    """A setting of every row: single precision where it is no whole number, as a tensor or as one number for all rows."""
    if not isinstance(x, torch.Tensor):
        x = torch.full((like.shape[0],), x, dtype=torch.int32 if kind == torch.int64 else torch.float32, device=like.device)
    return x.to(kind)[:, None]


def _sample(s):
    """In 64 bits throughout: sums over a vocabulary are compared with borders."""
    x = s["logits"].double()
    rows, v = x.shape
    temp, k, p, least = (_column(s[n], x, t) for n, t in (
        ("temperature", torch.float64), ("top_k", torch.int64), ("top_p", torch.float64), ("min_p", torch.float64)))
    x = torch.where(x.isnan(), -math.inf, x)
    x, order = torch.sort(x, dim=1, descending=True, stable=True)  # equal values: the lowest index first
    rank = torch.arange(v, device=x.device)[None]
    keep = (rank < torch.where((k > 0) & (k < v), k, v)) & (x > -math.inf)
    rel = x - x[:, :1]
    rel = torch.where(x == x[:, :1], 0.0, rel)
    w = torch.where(keep, torch.exp(rel), 0.0)
    before = torch.cumsum(w, 1) - w
    keep &= (p >= 1) | (before < p * w.sum(1, keepdim=True)) | (rank == 0)
    keep &= (least <= 0) | (rel >= torch.log(least)) | (rank == 0)
    keep &= (temp > 0) | (rank == 0)
    w = torch.where(keep, torch.exp(rel / torch.where(temp > 0, temp, 1.0)), 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)  # the draw goes through the tokens in their own order
    below = torch.cumsum(w, 1)
    target = s["u"].double()[:, None] * below[:, -1:]
    at = (below <= target).sum(1, keepdim=True)
    last = torch.where(w > 0, rank, -1).amax(1, keepdim=True)
    at = torch.minimum(at, last)
    prob = torch.where(at >= 0, w.gather(1, at.clamp(min=0)) / below[:, -1:], 0.0)
    return {"token": at[:, 0].to(torch.int32), "prob": prob[:, 0].float()}


# ------------------------------------------------------------------------------------------------------------------ run
def run(s):
    if own:
        ops = _framework()
        if s["op"] == "qk_norm_rope":
            q, k = ops.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], s["q_weight"], s["k_weight"],
                                    eps=s["eps"], interleaved=s["interleaved"])
            return {"q": q, "k": k}
        if s["op"] == "kv_append":
            q = ops.kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], cos=s["cos"], sin=s["sin"],
                              positions=s["positions"], k_weight=s["k_weight"], q=s["q"], q_weight=s["q_weight"],
                              eps=s["eps"], interleaved=s["interleaved"])
            return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": q}
        if s["op"] == "tree_attention":
            return ops.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["context_lens"],
                                      mask=s["mask"], max_context=s["max_context"])
        token, prob = ops.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                        top_p=s["top_p"], min_p=s["min_p"])
        return {"token": token, "prob": prob}
    if s["op"] == "tree_attention":
        return _attention(s)
    if s["op"] == "sample":
        return _sample(s)
    q = s["q"]
    if q is not None:
        q = _norm_rope(q, s["q_weight"], s["cos"], s["sin"], s["positions"], s["eps"], s["interleaved"]).to(q.dtype)
    k = _norm_rope(s["k"], s["k_weight"], s["cos"], s["sin"], s["positions"], s["eps"], s["interleaved"])
    if s["op"] == "qk_norm_rope":
        return {"q": q, "k": k.to(s["k"].dtype)}
    _put(s["k_cache"], s["slots"], k)
    _put(s["v_cache"], s["slots"], s["v"].float())
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "q": q}


def work(case):
    if case["op"] in ("qk_norm_rope", "kv_append"):
        t, h, kv, d, size = case["tokens"], case["heads"], case["kv_heads"], case["dim"], BYTES[case["types"]]
        live = t - case.get("pad", 0)
        # a row's angles once a token; weights once
        extra = min(t, case["table"]) * case["rot"] * 4 + t * 4 + (2 * d * 4 if case["norm"] else 0)
        if case["op"] == "qk_norm_rope":
            return {"bytes": 2 * t * (h + kv) * d * size + extra, "flops": 7 * t * (h + kv) * d}
        return {"bytes": 2 * t * h * d * size + 2 * live * kv * d * (size + BYTES[case["cache"]]) + extra + 8 * t,
                "flops": 7 * (t * h + live * kv) * d}
    if case["op"] == "tree_attention":
        n, h, kv, d, lens = case["nodes"], case["heads"], case["kv_heads"], case["dim"], _lengths(case)
        keys = sum(c + n for c in lens)
        return {"bytes": 2 * keys * kv * d * BYTES[case["cache"]] + 2 * case["seqs"] * n * h * d * BYTES[case["q"]] +
                (case["seqs"] * n * n if case["mask"] == "tree" else 0) + 4 * sum(-(-(c + n) // case["page"]) for c in lens),
                "flops": 4 * keys * n * h * d}
    return {"bytes": case["rows"] * (case["vocab"] * BYTES[case["types"]] + 12), "flops": 4 * case["rows"] * case["vocab"]}


# ---------------------------------------------------------------------------------------------------------------- exact
def _exact_rows(x, w, cos, sin, pos, eps, inter):
    """One array of head rows [T, heads, d], pair by pair."""
    x = x.copy()
    if w is not None:
        x *= w / np.sqrt(np.einsum("thd,thd->th", x, x)[..., None] / x.shape[-1] + eps)
    half = cos.shape[1]
    i = np.arange(half)
    first, second = (2 * i, 2 * i + 1) if inter else (i, i + half)
    z = (x[..., first] + 1j * x[..., second]) * (cos[pos] + 1j * sin[pos])[:, None, :]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda x: None if x is None else x.double().cpu().numpy()  # noqa: E731
    if case["op"] in ("qk_norm_rope", "kv_append"):
        pos = s["positions"].cpu().numpy()
        cos, sin = wide(s["cos"]), wide(s["sin"])
        q, k = (None if x is None else _exact_rows(wide(x), wide(w), cos, sin, pos, s["eps"], s["interleaved"])
                for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))
        if case["op"] == "qk_norm_rope":
            return {"q": torch.from_numpy(q), "k": torch.from_numpy(k)}
        slots, page = s["slots"].cpu().numpy(), case["page"]
        live = np.nonzero(slots >= 0)[0]
        kc, vc = wide(s["k_cache"]), wide(s["v_cache"])
        kc[slots[live] // page, :, slots[live] % page] = k[live]
        vc[slots[live] // page, :, slots[live] % page] = wide(s["v"])[live]
        return {"k_cache": torch.from_numpy(kc), "v_cache": torch.from_numpy(vc),
                "q": None if q is None else torch.from_numpy(q)}
    if case["op"] == "tree_attention":
        n, h, kv, d, page = case["nodes"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        out = torch.empty(case["seqs"], n, h, d, dtype=torch.float64)
        for b in range(case["seqs"]):
            c = int(s["context_lens"][b])
            used = s["block_table"][b, : -(-(c + n) // page)].long()
            bias = torch.zeros(n, c + n, dtype=torch.float64, device=DEV)
            m = s["mask"][b] if s["mask"] is not None else torch.ones(n, n, device=DEV).tril().bool()
            bias[:, c:][~m] = -math.inf
            for x in range(kv):
                k = s["k_cache"][used, x].reshape(-1, d)[: c + n].double()
                v = s["v_cache"][used, x].reshape(-1, d)[: c + n].double()
                for y in range(x * (h // kv), (x + 1) * (h // kv)):
                    out[b, :, y] = (torch.softmax(s["q"][b, :, y].double() @ k.T / math.sqrt(d) + bias, -1) @ v).cpu()
        return out
    logits, u = wide(s["logits"]), wide(s["u"])
    per = {n: (wide(s[n]) if isinstance(s[n], torch.Tensor) else np.full(len(u), np.float32(s[n]), np.float64))
           for n in ("temperature", "top_k", "top_p", "min_p")}
    token, prob = np.zeros(len(u), np.int32), np.zeros(len(u))
    for r, x in enumerate(logits):
        ids = np.lexsort((np.arange(len(x)), -x))
        if per["temperature"][r] <= 0:
            token[r], prob[r] = ids[0], 1.0
            continue
        if 0 < per["top_k"][r] < len(x):
            ids = ids[: int(per["top_k"][r])]
        e = np.exp(x[ids] - x[ids[0]])
        if per["top_p"][r] < 1:
            ids = ids[: 1 + int(np.searchsorted(np.cumsum(e), per["top_p"][r] * e.sum()))]
        if per["min_p"][r] > 0:
            ids = ids[x[ids] - x[ids[0]] >= np.log(per["min_p"][r])]
        ids = np.sort(ids)
        e = np.exp((x[ids] - x[ids].max()) / per["temperature"][r])
        at = min(int(np.searchsorted(np.cumsum(e), u[r] * e.sum(), side="right")), len(ids) - 1)
        token[r], prob[r] = ids[at], e[at] / e.sum()
    return {"token": torch.from_numpy(token), "prob": torch.from_numpy(prob)}
