"""Drafted-token operators on torch tensors (include/funasr_hip.h, fa_qk_norm_rope ... fa_sample_tokens).

What a decoding step that verifies drafted tokens needs beside the engine: head norms with the rotation, a paged key / value
cache, attention of a tree of drafted tokens over it, and draws from given random numbers. The calls enqueue hand-written
gfx950 kernels on the current stream of their tensors' device, allocate nothing but outputs and workspaces (through torch's
allocator, on that stream), never synchronise, and can be captured into a graph. A tensor that was made on another stream is
ordered before the call by its user, as with any torch operation. Wrong shapes, types, strides or devices raise ValueError
before anything is enqueued; a refusal of the library raises RuntimeError with its message. There is no CPU fallback and no
gradient: a tensor that requires one is refused outside torch.no_grad(). Outputs overlap no input, but where it is said.

A program that also creates an Engine imports torch (or this module) before the first one: torch brings a HIP runtime of its
own, and the engine's library uses it where it is loaded already. The other way round the process holds two, and torch's
finds no device.

Tensors that a call writes (caches, out, out_q ...) get a new version, as by any in-place operation of torch. A tensor with a
forward-mode tangent is refused.
"""
import ctypes
import importlib.machinery
import importlib.util
import os
import sys
import warnings

from . import _native

if _native._lib is not None and "torch" not in sys.modules:
    warnings.warn("torch is imported after the engine's library has loaded another HIP runtime and will find no GPU: import "
                  "torch or fun_asr_gguf.ops before the first Engine", RuntimeWarning, stacklevel=2)
import torch  # noqa: E402

_BINDING = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lib", "draft_ops.so")
_module = None


def _ops():
    """The torch binding (csrc/ops_torch.cpp), bound to the loaded engine library."""
    global _module
    if _module is None:
        if not os.path.exists(_BINDING):
            raise RuntimeError(f"{_BINDING} not found: run __graft_entry__.build() first")
        lib = _native.load()
        loader = importlib.machinery.ExtensionFileLoader("draft_ops", _BINDING)
        m = importlib.util.module_from_spec(importlib.util.spec_from_file_location("draft_ops", _BINDING, loader=loader))
        loader.exec_module(m)
        m.bind(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in (
            "fa_qk_norm_rope", "fa_kv_append", "fa_tree_attention", "fa_tree_attention_workspace", "fa_sample_tokens",
            "fa_sample_tokens_workspace", "fa_last_error")))
        _module = m
    return _module


def qk_norm_rope(q, k, cos, sin, positions, q_weight=None, k_weight=None, *, eps=1e-6, interleaved=False, out_q=None,
                 out_k=None):
    """Head rows of q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] divided by their root mean square and
    weighted (a weight of None: no norm), then rotated by the token's angles cos / sin [table, rot_dim / 2] at positions
    [tokens] (all three None: no rotation), pairs (i, i + rot_dim / 2) or, interleaved, (2 i, 2 i + 1). 32-bit arithmetic,
    one rounding. out_q / out_k may be q / k themselves. A token whose position is outside the table is not written.
    -> (q, k)"""
    return (_module or _ops()).qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved, out_q, out_k)


def kv_append(k, v, k_cache, v_cache, slots, *, cos=None, sin=None, positions=None, k_weight=None, q=None, q_weight=None,
              eps=1e-6, interleaved=False, out_q=None):
    """k (normed and rotated as in qk_norm_rope) and v [tokens, kv_heads, head_dim] into the pages of a cache: k_cache /
    v_cache [pages, kv_heads, page_size, head_dim] of float16 or bfloat16 (any strides that keep rows 16-byte aligned), token
    t at slots[t] = page * page_size + offset. A token with a slot outside the cache (padding: -1) is not appended. The
    slots of one call are distinct. q: its rows are normed and rotated in the same launch (q_weight and out_q belong to it).
    -> q's rows (None without q)"""
    return (_module or _ops()).kv_append(k, v, k_cache, v_cache, slots, cos, sin, positions, k_weight, q, q_weight, eps, interleaved,
                                         out_q)


def tree_mask(parents):
    """The mask of draft trees for tree_attention: parents [.., nodes], each an earlier node or -1 (it hangs from the
    committed tokens) -> bool [.., nodes, nodes], row i true for i and its ancestors."""
    p = torch.as_tensor(parents).cpu()
    n = p.shape[-1]
    if not (bool((p < torch.arange(n)).all()) and bool((p >= -1).all())):
        raise ValueError("a node's parent must be an earlier node or -1")
    flat = p.reshape(p.shape[:-1].numel(), n).long()
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
    node is an ordinary decoding step). A row that sees nothing is 0; rows behind draft_lens[b] are left as they were. Weights
    are rounded to the cache's type for the second product; float32 q keeps them, and q itself, to 22 (float16 cache) or 24 bits.
    max_context: the largest context length if the caller knows it (default: what the table holds); it shapes the launch,
    not the result's definition. scale: default head_dim ** -0.5. -> out, like q"""
    return (_module or _ops()).tree_attention(q, k_cache, v_cache, block_table, context_lens, mask, draft_lens, scale, max_context,
                                              out)


def sample_tokens(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, out_prob=None):
    """One token for every row of logits [rows, vocab] (float32, float16 or bfloat16) from the random numbers u [rows]
    (float32 in [0, 1)): top_k -> top_p -> min_p -> temperature, then the first token in the vocabulary's order whose
    cumulative mass exceeds u times the whole. Settings: numbers, or tensors [rows] (float32; top_k int32). temperature <= 0
    is greedy; top_k <= 0, top_p >= 1 and min_p <= 0 switch a step off; equal logits rank by id; NaN counts as -inf; a row
    with nothing above -inf gives -1. -> (tokens int32 [rows], their probabilities float32 [rows])"""
    return (_module or _ops()).sample_tokens(logits, u, temperature, top_k, top_p, min_p, out, out_prob)
