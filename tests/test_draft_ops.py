"""CPU checks of the drafted-token operators: what the library refuses before it touches a device (fa_qk_norm_rope ...
fa_sample_tokens with sizes, strides, types and pointers that do not fit), what fun_asr_gguf.ops refuses, and the plain
forms the GPU tests compare with."""
import ctypes

import os

import numpy as np
import pytest
import torch

from draft_oracle import attention, norm_rope, sample
from fun_asr_gguf import _native, ops

P = 0x10000  # never dereferenced: every call below is refused first


def head(**kw):
    a = _native.HeadRowsArgs(q=P, k=P, v=P, q_out=2 * P, k_out=3 * P, v_out=4 * P, cos=P, sin=P, positions=P, slots=P, q_token=1024,
                             q_head=128, k_token=1024, k_head=128, v_token=1024, v_head=128, q_out_token=1024, q_out_head=128,
                             k_out_token=128, k_out_head=2048, k_out_page=16384, v_out_token=128, v_out_head=2048,
                             v_out_page=16384, tokens=4, heads=8, kv_heads=8, head_dim=128, rot_dim=128, table_len=10, type=2,
                             cache_type=2, pages=3, page_size=16, eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(call, a, word, *more):
    lib = _native.load()
    assert getattr(lib, call)(ctypes.byref(a), *(more or (None,))) == -1
    assert word in lib.fa_last_error().decode(), lib.fa_last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(tokens=-1), "negative"), (dict(head_dim=24), "head_dim"), (dict(head_dim=528), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(type=3), "type"), (dict(rot_dim=130), "rot_dim"), (dict(rot_dim=24), "rot_dim"),
    (dict(rot_dim=144), "rot_dim"), (dict(cos=None), "together"), (dict(table_len=0), "table"),
    (dict(positions=None), "positions"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(q=None), "q and"),
    (dict(tokens=2 ** 30), "2^31")])
def test_head_rows_refusals(kw, word):
    refused("fa_qk_norm_rope", head(**kw), word)
    refused("fa_kv_append", head(**kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(cache_type=0), "cache"), (dict(kv_heads=0), "sizes"), (dict(page_size=0), "sizes"), (dict(pages=-1), "sizes"),
    (dict(pages=2 ** 20, page_size=2 ** 12), "slots"), (dict(k=None), "k, v"), (dict(v=None), "k, v"),
    (dict(slots=None), "k, v"), (dict(k_out=None), "caches"), (dict(k_out=3 * P + 8), "aligned"), (dict(v_out_token=132), "aligned"),
    (dict(k_out_page=16388), "aligned"), (dict(k_out_head=2052), "aligned")])
def test_append_refusals(kw, word):
    refused("fa_kv_append", head(**kw), word)


def test_norm_rope_in_place_with_other_strides_is_refused():
    refused("fa_qk_norm_rope", head(q_out=P, q_out_token=2048), "in place")
    refused("fa_qk_norm_rope", head(k_out=P, k_out_token=2048, k_out_head=128), "in place")


def tree(**kw):
    a = _native.TreeAttentionArgs(q=P, out=P, k_cache=P, v_cache=P, block_table=P, context_lens=P, q_seq=4096, q_node=1024,
                                  q_head=128, out_seq=4096, out_node=1024, out_head=128, k_page=16384, k_head=2048, k_slot=128,
                                  v_page=16384, v_head=2048, v_slot=128, table_seq=8, seqs=2, nodes=4, heads=8, kv_heads=8,
                                  head_dim=128, q_type=2, cache_type=2, pages=3, page_size=16, table_len=8, scale=0.1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(seqs=-1), "heads"), (dict(nodes=-1), "heads"), (dict(heads=0), "heads"), (dict(heads=12), "multiple"),
    (dict(kv_heads=0), "heads"), (dict(seqs=70000), "65535"), (dict(head_dim=12), "head_dim"), (dict(head_dim=264), "head_dim"),
    (dict(cache_type=0), "cache"), (dict(q_type=1), "q is"), (dict(q_type=7), "q is"), (dict(page_size=0), "pages"),
    (dict(pages=0), "pages"), (dict(table_len=0), "pages"), (dict(page_size=2 ** 28), "positions"), (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(nodes=65535, heads=16), "rows")])
def test_tree_attention_refusals(kw, word):
    refused("fa_tree_attention", tree(**kw), word)
    n = ctypes.c_int64()
    refused("fa_tree_attention_workspace", tree(**kw), word, ctypes.byref(n))
    refused("fa_tree_attention_workspace", tree(), "size", None)


def rows(**kw):
    a = _native.SampleArgs(logits=P, u=P, token_out=P, rows=2, vocab=100, row_stride=100, type=0, temperature=1.0, top_p=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(vocab=2 ** 24 + 1), "vocab"), (dict(type=5), "type"),
    (dict(row_stride=99), "overlap"), (dict(logits=None), "null"), (dict(u=None), "null"), (dict(token_out=None), "null")])
def test_sample_refusals(kw, word):
    refused("fa_sample_tokens", rows(**kw), word)


def test_null_arguments_are_refused():
    lib = _native.load()
    for f in ("fa_qk_norm_rope", "fa_kv_append", "fa_tree_attention", "fa_sample_tokens"):
        assert getattr(lib, f)(None, None) == -1


def test_python_refuses_tensors_off_the_gpu():
    x = torch.zeros(2, 4, 32)
    with pytest.raises(ValueError, match="GPU"):
        ops.qk_norm_rope(x, x, None, None, None)
    with pytest.raises(ValueError, match="GPU"):
        ops.kv_append(x, x, x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        ops.tree_attention(x[None], x, x, x, x)
    with pytest.raises(ValueError, match="GPU"):
        ops.sample_tokens(x[0], x[0, 0])


def test_tree_mask():
    m = ops.tree_mask([[-1, 0, 0, 2, -1], [-1, -1, 1, 2, 3]])
    assert m.shape == (2, 5, 5)
    assert m[0].int().tolist() == [[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 0, 1, 1, 0], [0, 0, 0, 0, 1]]
    assert m[1].int().tolist() == [[1, 0, 0, 0, 0], [0, 1, 0, 0, 0], [0, 1, 1, 0, 0], [0, 1, 1, 1, 0], [0, 1, 1, 1, 1]]
    assert ops.tree_mask([-1, 0, 1]).int().tolist() == torch.ones(3, 3).tril().int().tolist()
    for bad in ([0], [-1, 1], [-2], [-1, 0, 2]):
        with pytest.raises(ValueError):
            ops.tree_mask(bad)


def test_plain_forms():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 2, 32))
    a = np.arange(10)[:, None] * 0.3 ** np.arange(16)[None]
    y, _ = norm_rope(x, np.ones(32), np.cos(a), np.sin(a), np.array([0, 4, 9]), 0.0, False)
    assert np.allclose((y ** 2).mean(-1), 1)  # a rotation keeps the norm
    assert np.allclose(y[0], x[0] / np.sqrt((x[0] ** 2).mean(-1, keepdims=True)))
    q, k, v = rng.standard_normal((1, 2, 2, 8)), rng.standard_normal((4, 1, 2, 8)), rng.standard_normal((4, 1, 2, 8))
    out, _, _ = attention(q, k, v, np.array([[2, 0, 3]]), [3], [2], None, 0.5)
    keys, vals = (c[[2, 0, 3], 0].reshape(6, 8) for c in (k, v))
    for i in range(2):
        for h in range(2):
            s = torch.softmax(torch.from_numpy(keys[:4 + i] @ q[0, i, h] * 0.5), 0).numpy()
            assert np.allclose(out[0, i, h], s @ vals[:4 + i])
    z = np.log([0.5, 0.3, 0.15, 0.05])
    assert [sample(z, u, 1.0, 0, 1.0, 0.0)[0] for u in (0.0, 0.49, 0.51, 0.94, 0.99)] == [0, 0, 1, 2, 3]
    assert sample(z, 0.99, 1.0, 3, 1.0, 0.0)[0] == 2 and sample(z, 0.99, 1.0, 0, 0.79, 0.0)[0] == 1
    assert sample(z, 0.99, 1.0, 0, 1.0, 0.25)[0] == 2 and sample(z, 0.99, 0.0, 0, 1.0, 0.0)[:2] == (0, 1.0)
    assert sample([1.0, 2.0, 2.0, 2.0], 0.99, 1.0, 2, 1.0, 0.0)[0] == 2  # equal values: the lower ids


@pytest.mark.parametrize("first,warned", [("fun_asr_gguf._native as n; n.load()", True), ("torch", False)])
def test_import_order(first, warned):
    """torch behind the engine's library in one process would find no GPU: importing the operators says so."""
    import subprocess
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fun-asr-gguf_amd")
    prog = f"import sys; sys.path.insert(0, {pkg!r})\nimport {first}\nimport fun_asr_gguf._native as n; n.load()\nimport fun_asr_gguf.ops"
    r = subprocess.run([sys.executable, "-W", "always", "-c", prog], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert ("before the first Engine" in r.stderr) == warned


def test_tensors_that_require_a_gradient_are_refused():
    x, u = torch.zeros(2, 8, requires_grad=True), torch.zeros(2)
    with pytest.raises(ValueError, match="gradient"):
        ops.sample_tokens(x, u)
    with torch.no_grad(), pytest.raises(ValueError, match="on the GPU"):
        ops.sample_tokens(x, u)
    q = torch.zeros(2, 3, 32, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        ops.qk_norm_rope(q, q.detach(), None, None, None)


def test_lds_is_asked_for_on_every_device(tmp_path):
    """A kernel with more than 64 KB of LDS asks for it once on each device it runs on, and again where that failed. Four HIP
    calls are replaced: the machine has the devices that the test says."""
    import shutil
    import subprocess
    import sys
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    (tmp_path / "hip.c").write_text("""
        static int device, fail, asked[8], launched;
        void shim_set(int d, int f) { device = d; fail = f; }
        int shim_asked(int d) { return asked[d]; }
        int shim_launched(void) { return launched; }
        int hipGetDevice(int* d) { *d = device; return 0; }
        int hipDeviceGetAttribute(int* v) { *v = 256; return 0; }
        int hipFuncSetAttribute() { if (fail) return 1; ++asked[device]; return 0; }
        int hipLaunchKernel() { ++launched; return 0; }
    """)
    shim = str(tmp_path / "hip.so")
    subprocess.run(["gcc", "-w", "-shared", "-fPIC", str(tmp_path / "hip.c"), "-o", shim], check=True)
    here = os.path.dirname(os.path.abspath(__file__))
    prog = f"""
import ctypes, sys
sys.path[:0] = [{here!r}, {os.path.join(os.path.dirname(here), "fun-asr-gguf_amd")!r}]
from fun_asr_gguf import _native
from test_draft_ops import tree
lib, shim = _native.load(), ctypes.CDLL({shim!r})
call = lambda: lib.fa_tree_attention(ctypes.byref(tree(head_dim=256, q_head=256, out_head=256, k_slot=256, v_slot=256)), None)
for device in (0, 1):
    shim.shim_set(device, 0)
    assert call() == 0 and call() == 0, lib.fa_last_error()
    assert shim.shim_asked(device) == 1, device
shim.shim_set(2, 1)
assert call() != 0 and shim.shim_launched() == 4
shim.shim_set(2, 0)
assert call() == 0 and shim.shim_asked(2) == 1 and shim.shim_launched() == 5
print("fine")
"""
    env = dict(os.environ, LD_PRELOAD=":".join(x for x in (shim, os.environ.get("LD_PRELOAD")) if x))
    r = subprocess.run([sys.executable, "-c", prog], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr


def test_tensors_with_a_tangent_are_refused():
    import torch.autograd.forward_ad as fw
    x, u = torch.zeros(2, 8), torch.zeros(2)
    with fw.dual_level(), pytest.raises(ValueError, match="tangent"):
        ops.sample_tokens(fw.make_dual(x, torch.ones(2, 8)), u)
    q = torch.zeros(2, 3, 32)
    with fw.dual_level(), pytest.raises(ValueError, match="tangent"):
        ops.qk_norm_rope(fw.make_dual(q, q), q, None, None, None)


@pytest.mark.parametrize("heads,kv_heads", [(2 ** 31 - 1, 8), (8, 2 ** 31 - 1), (2 ** 30, 2 ** 30), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("tokens", [1, 3])
def test_head_counts_whose_sum_passes_32_bits_are_refused(heads, kv_heads, tokens):
    for call in ("fa_qk_norm_rope", "fa_kv_append"):
        refused(call, head(heads=heads, kv_heads=kv_heads, tokens=tokens), "2^31")


def test_tree_mask_of_no_nodes_and_of_more_dimensions():
    assert ops.tree_mask(torch.zeros(3, 0, dtype=torch.int32)).shape == (3, 0, 0)
    assert ops.tree_mask([]).shape == (0, 0)
    assert ops.tree_mask(torch.zeros(0, 4, dtype=torch.int64)).shape == (0, 4, 4)
    p = torch.tensor([[[-1, 0, 1], [-1, -1, 0]]])
    assert torch.equal(ops.tree_mask(p)[0, 1], ops.tree_mask([-1, -1, 0]))


def test_the_engine_builds_without_torch(tmp_path):
    """The binding of the operators is the one part that needs torch: without it the rest is built, and the engine's package
    imports; the operators' module says what it misses."""
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    prog = f"""
import sys
sys.path[:0] = [{root!r}]
sys.modules["torch"] = None  # (import torch raises ImportError)
import __graft_entry__ as g
assert g.build_ops() is None
g.build_native = g.build_llama_compat = g._build_oracle_c = lambda **kw: None
g.build()
import fun_asr_gguf
try:
    import fun_asr_gguf.ops
except ImportError as e:
    print("no operators:", e)
"""
    r = subprocess.run([sys.executable, "-c", prog], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "no operators" in r.stdout and "torch" in r.stderr, r.stdout + r.stderr


def test_vocabularies_end_at_2_22():
    """k_finish has a thread for every chunk up to there."""
    lib, n = _native.load(), ctypes.c_int64()
    refused("fa_sample_tokens", rows(vocab=2 ** 22 + 1, row_stride=2 ** 22 + 1), "2^22")
    refused("fa_sample_tokens_workspace", rows(vocab=2 ** 22 + 1, row_stride=2 ** 22 + 1), "2^22", ctypes.byref(n))
    assert lib.fa_sample_tokens_workspace(ctypes.byref(rows(vocab=2 ** 22, row_stride=2 ** 22)), ctypes.byref(n)) == 0
    assert n.value > 2 * 1024 * 4


def test_every_script_builds_device_code_with_the_library_s_flags():
    """A variant or a microbenchmark is compared with the library: no packed f32 instructions there either."""
    import glob
    import __graft_entry__ as g
    flags = " ".join(g.HIP_FLAGS)
    found = 0
    for path in glob.glob(os.path.join(g.ROOT, "scripts", "**", "*.sh"), recursive=True):
        text = open(path).read().replace("\\\n", " ")
        for line in text.splitlines():
            if "hipcc" not in line or line.lstrip().startswith("#"):
                continue
            for cmd in line.split("&&"):
                if "hipcc" in cmd and ".hip" in cmd.replace(".hip.o", ""):  # (a link of objects compiles nothing)
                    found += 1
                    assert flags in cmd or ("$F" in cmd and flags in text[:text.index("hipcc")]), (path, cmd)
    assert found > 10


def test_build_compiles_every_source_each_time(monkeypatch):
    """build() is the check that the tree builds: nothing is skipped because an older result is there."""
    import subprocess
    import __graft_entry__ as g
    if not os.path.exists(g.LIB):
        pytest.skip("nothing built")
    done = []

    def run(cmd, **kw):
        done.append(" ".join(map(str, cmd)))
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(g.subprocess, "run", run)
    g.build()
    for src in g.SOURCES + ["ops_torch.cpp", "llama_compat.cpp", "ggml_compat.c"]:
        assert any(os.path.join(g.CSRC, src) + " " in c for c in done), src
