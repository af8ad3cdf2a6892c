"""The drafted-token operators (fun_asr_gguf.ops) on the GPU where they can go wrong: many splits of narrow heads.
Plain 64-bit forms: tests/draft_oracle.py; tolerances as in test_gpu_draft_ops.py unless a test says more."""
import numpy as np
import pytest
import torch  # noqa: F401  (before any engine: the library then shares torch's HIP runtime)

from test_gpu_draft_ops import check, kind, ops, paged, t  # noqa: F401

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
