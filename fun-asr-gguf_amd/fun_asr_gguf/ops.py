"""Drafted-token operators on torch tensors (include/funasr_hip.h, fa_qk_norm_rope ... fa_sample_tokens).

What a decoding step that verifies drafted tokens needs beside the engine: head norms with the rotation, a paged key / value
cache, attention of a tree of drafted tokens over it, and draws from given random numbers. The calls enqueue hand-written
gfx950 kernels on the current stream of their tensors' device, allocate nothing but outputs and workspaces (through torch's
allocator, on that stream), never synchronise, and can be captured into a graph. A tensor that was made on another stream is
ordered before the call by its user, as with any torch operation. Wrong shapes, types, strides or devices raise ValueError
before anything is enqueued; a refusal of the library raises RuntimeError with its message. There is no CPU fallback.
"""
import ctypes

import torch

from . import _native

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_HALF = (torch.float16, torch.bfloat16)
_INTS = (torch.int32, torch.int64)
_lib = None


def _library():
    global _lib
    if _lib is None:
        _lib = _native.load()
    return _lib


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _on(dev, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, not on {dev}")


def _run(call, what, args, dev):
    """call(args, stream) with the tensors' device current."""
    if dev.index == torch.cuda.current_device():
        rc = call(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = call(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    if rc != 0:
        _native._check(rc, what)


def _gpu(t, name):
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a tensor on the GPU")
    return t.device


def _head_args(k, cos, sin, positions, q, q_weight, k_weight, eps, interleaved):
    """What qk_norm_rope and kv_append share: checks, and their arguments filled in as far as they agree."""
    dev = _gpu(k, "k")
    _need(k.dtype in TYPES, f"k: type {k.dtype}")
    _need(k.dim() == 3 and (k.shape[2] == 1 or k.stride(2) == 1), "k must be [tokens, kv_heads, head_dim] with contiguous heads")
    tokens, kv_heads, dim = k.shape
    a = _native.HeadRowsArgs()
    _on(dev, q=q, cos=cos, sin=sin, positions=positions, q_weight=q_weight, k_weight=k_weight)
    if q is not None:
        _need(q.dim() == 3 and q.shape[0] == tokens and q.shape[2] == dim and q.dtype == k.dtype and
              (dim == 1 or q.stride(2) == 1), "q must be [tokens, heads, head_dim] of k's type with contiguous heads")
        a.q, a.q_token, a.q_head, a.heads = q.data_ptr(), q.stride(0), q.stride(1), q.shape[1]
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        _need(w is None or (w.dtype == torch.float32 and w.shape == (dim,) and w.is_contiguous()),
              f"{name} must be float32 [head_dim]")
    _need((cos is None) == (sin is None) and (cos is None) == (positions is None), "cos, sin and positions come together")
    if cos is not None:
        _need(cos.dtype == sin.dtype == torch.float32 and cos.dim() == 2 and cos.shape == sin.shape and
              cos.is_contiguous() and sin.is_contiguous(), "cos and sin must be float32 [table, rot_dim / 2]")
        _need(positions.dtype in _INTS and positions.shape == (tokens,) and (tokens < 2 or positions.stride(0) == 1),
              "positions must be int32 or int64 [tokens]")
        a.cos, a.sin, a.positions = cos.data_ptr(), sin.data_ptr(), positions.data_ptr()
        a.table_len, a.rot_dim, a.positions_64 = cos.shape[0], 2 * cos.shape[1], positions.dtype == torch.int64
    a.q_weight = None if q_weight is None else q_weight.data_ptr()
    a.k_weight = None if k_weight is None else k_weight.data_ptr()
    a.k, a.k_token, a.k_head = k.data_ptr(), k.stride(0), k.stride(1)
    a.tokens, a.kv_heads, a.head_dim, a.type = tokens, kv_heads, dim, TYPES[k.dtype]
    a.interleaved, a.eps = bool(interleaved), eps
    return a, dev


def _rows_out(x, out, name):
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _need(out.shape == x.shape and out.dtype == x.dtype and out.device == x.device and
          (x.shape[2] == 1 or out.stride(2) == 1), f"{name} must be like its input, with contiguous heads")
    return out


def qk_norm_rope(q, k, cos, sin, positions, q_weight=None, k_weight=None, *, eps=1e-6, interleaved=False, out_q=None,
                 out_k=None):
    """Head rows of q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] divided by their root mean square and
    weighted (a weight of None: no norm), then rotated by the token's angles cos / sin [table, rot_dim / 2] at positions
    [tokens] (all three None: no rotation), pairs (i, i + rot_dim / 2) or, interleaved, (2 i, 2 i + 1). 32-bit arithmetic,
    one rounding. out_q / out_k may be q / k themselves. A token whose position is outside the table is not written.
    -> (q, k)"""
    _need(q is not None, "q is missing (kv_append takes keys alone)")
    a, dev = _head_args(k, cos, sin, positions, q, q_weight, k_weight, eps, interleaved)
    out_q, out_k = _rows_out(q, out_q, "out_q"), _rows_out(k, out_k, "out_k")
    a.q_out, a.q_out_token, a.q_out_head = out_q.data_ptr(), out_q.stride(0), out_q.stride(1)
    a.k_out, a.k_out_token, a.k_out_head = out_k.data_ptr(), out_k.stride(0), out_k.stride(1)
    _run(_library().fa_qk_norm_rope, "fa_qk_norm_rope", a, dev)
    return out_q, out_k


def kv_append(k, v, k_cache, v_cache, slots, *, cos=None, sin=None, positions=None, k_weight=None, q=None, q_weight=None,
              eps=1e-6, interleaved=False, out_q=None):
    """k (normed and rotated as in qk_norm_rope) and v [tokens, kv_heads, head_dim] into the pages of a cache: k_cache /
    v_cache [pages, kv_heads, page_size, head_dim] of float16 or bfloat16 (any strides that keep rows 16-byte aligned), token
    t at slots[t] = page * page_size + offset. A token with a slot outside the cache (padding: -1) is not appended. The
    slots of one call are distinct. q: its rows are normed and rotated in the same launch. -> q's rows (None without q)"""
    a, dev = _head_args(k, cos, sin, positions, q, q_weight, k_weight, eps, interleaved)
    _on(dev, v=v, k_cache=k_cache, v_cache=v_cache, slots=slots)
    _need(v.shape == k.shape and v.dtype == k.dtype and (k.shape[2] == 1 or v.stride(2) == 1), "v must be like k")
    _need(k_cache.dtype in _HALF and v_cache.dtype == k_cache.dtype and k_cache.dim() == 4 and
          v_cache.shape == k_cache.shape and k_cache.shape[1] == k.shape[1] and k_cache.shape[3] == k.shape[2] and
          k_cache.stride(3) == 1 and v_cache.stride(3) == 1,
          "the caches must be float16 or bfloat16 [pages, kv_heads, page_size, head_dim] with contiguous rows")
    _need(slots.dtype in _INTS and slots.shape == (k.shape[0],) and (k.shape[0] < 2 or slots.stride(0) == 1),
          "slots must be int32 or int64 [tokens]")
    if q is not None:
        out_q = _rows_out(q, out_q, "out_q")
        a.q_out, a.q_out_token, a.q_out_head = out_q.data_ptr(), out_q.stride(0), out_q.stride(1)
    a.v, a.v_token, a.v_head = v.data_ptr(), v.stride(0), v.stride(1)
    a.k_out, a.v_out = k_cache.data_ptr(), v_cache.data_ptr()
    a.k_out_page, a.k_out_head, a.k_out_token, _ = k_cache.stride()
    a.v_out_page, a.v_out_head, a.v_out_token, _ = v_cache.stride()
    a.pages, a.page_size, a.cache_type = k_cache.shape[0], k_cache.shape[2], TYPES[k_cache.dtype]
    a.slots, a.slots_64 = slots.data_ptr(), slots.dtype == torch.int64
    _run(_library().fa_kv_append, "fa_kv_append", a, dev)
    return out_q


def tree_mask(parents):
    """The mask of draft trees for tree_attention: parents [.., nodes], each an earlier node or -1 (it hangs from the
    committed tokens) -> bool [.., nodes, nodes], row i true for i and its ancestors."""
    p = torch.as_tensor(parents).cpu()
    n = p.shape[-1]
    _need(bool((p < torch.arange(n)).all()) and bool((p >= -1).all()), "a node's parent must be an earlier node or -1")
    flat = p.reshape(-1, n).long()
    m = torch.zeros(flat.shape[0], n, n, dtype=torch.bool)
    for j in range(n):
        has = flat[:, j] >= 0
        m[has, j] = m[has, flat[has, j]]
        m[:, j, j] = True
    return m.reshape(*p.shape, n)


def tree_attention(q, k_cache, v_cache, block_table, context_lens, *, mask=None, draft_lens=None, scale=None,
                   max_context=None, out=None):
    """Attention of drafted tokens q [seqs, nodes, heads, head_dim] over a paged cache [pages, kv_heads, page_size,
    head_dim] of float16 or bfloat16 (q: the same type, or float32). Sequence b reads position p in page
    block_table[b, p // page_size] (int32 [seqs, width]); it has context_lens[b] (int32) committed tokens and behind them
    draft_lens[b] (int32; None: nodes) drafted ones, already appended. Drafted token i sees all committed tokens and the
    drafted tokens j with mask[.., i, j] (bool [nodes, nodes] or [seqs, nodes, nodes], see tree_mask; None: j <= i, so one
    node is an ordinary decoding step). A row that sees nothing is 0; rows behind draft_lens[b] are left as they were.
    max_context: the largest context length if the caller knows it (default: what the table holds); it shapes the launch,
    not the result's definition. scale: default head_dim ** -0.5. -> out, like q"""
    dev = _gpu(q, "q")
    _need(q.dim() == 4 and q.dtype in TYPES and (q.shape[3] == 1 or q.stride(3) == 1),
          "q must be [seqs, nodes, heads, head_dim] with contiguous heads")
    seqs, nodes, heads, dim = q.shape
    _on(dev, k_cache=k_cache, v_cache=v_cache, block_table=block_table, context_lens=context_lens, mask=mask,
        draft_lens=draft_lens, out=out)
    _need(k_cache.dtype in _HALF and v_cache.dtype == k_cache.dtype and k_cache.dim() == 4 and
          v_cache.shape == k_cache.shape and k_cache.shape[3] == dim and k_cache.stride(3) == 1 and v_cache.stride(3) == 1,
          "the caches must be float16 or bfloat16 [pages, kv_heads, page_size, head_dim] with contiguous rows")
    _need(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == seqs and
          (block_table.shape[1] < 2 or block_table.stride(1) == 1), "block_table must be int32 [seqs, width]")
    _need(context_lens.dtype == torch.int32 and context_lens.shape == (seqs,) and
          (seqs < 2 or context_lens.stride(0) == 1), "context_lens must be int32 [seqs]")
    _need(draft_lens is None or (draft_lens.dtype == torch.int32 and draft_lens.shape == (seqs,) and
                                 (seqs < 2 or draft_lens.stride(0) == 1)), "draft_lens must be int32 [seqs]")
    a = _native.TreeAttentionArgs()
    if mask is not None:
        _need(mask.dtype in (torch.bool, torch.uint8) and mask.dim() in (2, 3) and mask.shape[-2:] == (nodes, nodes) and
              (mask.dim() == 2 or mask.shape[0] == seqs) and (nodes < 2 or mask.stride(-1) == 1),
              "mask must be bool [nodes, nodes] or [seqs, nodes, nodes]")
        a.mask, a.mask_row, a.mask_seq = mask.data_ptr(), mask.stride(-2), mask.stride(0) if mask.dim() == 3 else 0
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and (dim == 1 or out.stride(3) == 1), "out must be like q")
    a.q, a.out, a.k_cache, a.v_cache = q.data_ptr(), out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.block_table, a.context_lens = block_table.data_ptr(), context_lens.data_ptr()
    a.draft_lens = None if draft_lens is None else draft_lens.data_ptr()
    a.q_seq, a.q_node, a.q_head, _ = q.stride()
    a.out_seq, a.out_node, a.out_head, _ = out.stride()
    a.k_page, a.k_head, a.k_slot, _ = k_cache.stride()
    a.v_page, a.v_head, a.v_slot, _ = v_cache.stride()
    a.table_seq, a.table_len = block_table.stride(0), block_table.shape[1]
    a.seqs, a.nodes, a.heads, a.kv_heads, a.head_dim = seqs, nodes, heads, k_cache.shape[1], dim
    a.q_type, a.cache_type = TYPES[q.dtype], TYPES[k_cache.dtype]
    a.pages, a.page_size, a.max_context = k_cache.shape[0], k_cache.shape[2], max_context or 0
    a.scale = dim ** -0.5 if scale is None else scale
    _with_workspace(a, "fa_tree_attention", dev)
    return out


def _with_workspace(a, what, dev):
    lib = _library()
    need = ctypes.c_int64()
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _with_workspace(a, what, dev)
    rc = getattr(lib, what + "_workspace")(ctypes.byref(a), ctypes.byref(need))
    if rc != 0:
        _native._check(rc, what)
    ws = None
    if need.value:
        ws = torch.empty(need.value, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
    _run(getattr(lib, what), what, a, dev)


def sample_tokens(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, out_prob=None):
    """One token for every row of logits [rows, vocab] (float32, float16 or bfloat16) from the random numbers u [rows]
    (float32 in [0, 1)): top_k -> top_p -> min_p -> temperature, then the first token in the vocabulary's order whose
    cumulative mass exceeds u times the whole. Settings: numbers, or tensors [rows] (float32; top_k int32). temperature <= 0
    is greedy; top_k <= 0, top_p >= 1 and min_p <= 0 switch a step off; equal logits rank by id; NaN counts as -inf; a row
    with nothing above -inf gives -1. -> (tokens int32 [rows], their probabilities float32 [rows])"""
    dev = _gpu(logits, "logits")
    _need(logits.dtype in TYPES and logits.dim() == 2 and (logits.shape[1] < 2 or logits.stride(1) == 1),
          "logits must be [rows, vocab] with contiguous rows")
    rows = logits.shape[0]
    a = _native.SampleArgs()
    _on(dev, u=u, out=out, out_prob=out_prob)

    def vector(t, kind):
        return t.dtype == kind and t.shape == (rows,) and (rows < 2 or t.stride(0) == 1)
    _need(vector(u, torch.float32), "u must be float32 [rows]")
    for name, x, kind in (("temperature", temperature, torch.float32), ("top_p", top_p, torch.float32),
                          ("min_p", min_p, torch.float32), ("top_k", top_k, torch.int32)):
        if isinstance(x, torch.Tensor):
            _on(dev, **{name: x})
            _need(vector(x, kind), f"{name} must be a number or {kind} [rows]")
            setattr(a, name + "s", x.data_ptr())
        else:
            setattr(a, name, x)
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=dev)
    if out_prob is None:
        out_prob = torch.empty(rows, dtype=torch.float32, device=dev)
    _need(vector(out, torch.int32) and vector(out_prob, torch.float32), "out must be int32 [rows], out_prob float32 [rows]")
    a.logits, a.u, a.token_out, a.prob_out = logits.data_ptr(), u.data_ptr(), out.data_ptr(), out_prob.data_ptr()
    a.rows, a.vocab, a.row_stride, a.type = rows, logits.shape[1], logits.stride(0) if rows > 1 else logits.shape[1], TYPES[logits.dtype]
    _with_workspace(a, "fa_sample_tokens", dev)
    return out, out_prob
