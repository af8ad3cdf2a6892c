"""fa_llm_verify / Engine.llm_verify: a decode step that verifies a tree of drafted tokens on the engine's own cache.

Logits are compared with the CPU oracle's by the bound of teacher-forced decoding (cosine >= 0.9995: q8_0 activation
rounding differs); tokens are those of the engine's own logits, exactly."""
import ctypes

import numpy as np
import pytest

import draft_oracle
from oracle import qwen3 as oqw, synth

COS = 0.9995
N_CTX = 160


@pytest.fixture(scope="module")
def eng():
    from fun_asr_gguf import _native
    e = _native.Engine(synth.ENC_TINY, dict(synth.LLM_TINY, n_ctx=N_CTX, max_seqs=3), max_batch=1, max_samples=16000)
    e.synthetic_weights(0)
    yield e
    e.close()


@pytest.fixture(scope="module")
def oracle():
    return oqw.Qwen3Q8(synth.make_weights(synth.llm_tensors(synth.LLM_TINY)), synth.LLM_TINY, n_ctx=N_CTX)


def cos(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(a @ b / np.linalg.norm(a) / np.linalg.norm(b))


def start(eng, prompt, seq):
    eng.llm_reset(seq)
    return eng.llm_prefill(seq, eng.embd_rows(prompt))


def oracle_logits(oracle, prompt, tokens):
    """After the prompt and `tokens`: the last row's logits."""
    oracle.reset()
    lg = oracle.forward(oracle.embed_prompt(prompt), 0)
    if len(tokens):
        lg = oracle.forward(oracle.embed_tokens(np.asarray(tokens)), len(prompt))
    return lg


def right_path(eng, prompt, seq, where, tokens, parents, **samp):
    """tokens with those at `where` (a path below the root) replaced by what is drawn there, one depth a call; every call has
    the same shape, so its rows above are the same bits."""
    tokens, seen = list(tokens), []
    for depth in range(len(where) + 1):
        start(eng, prompt, seq)
        got, path = eng.llm_verify(seq, tokens, parents, **samp)
        assert got[:depth] == seen and path == list(where[:depth])
        assert len(got) == depth + 1
        seen = got
        if depth < len(where):
            tokens[where[depth]] = got[depth]
    return tokens, seen


# trees of drafts: (parents, the path that is accepted)
TREES = [([], []), ([-1], [0]), ([-1, 0, 1, 2], [0, 1, 2, 3]), ([-1, -1, 1, 0, 2, 4, 4], [1, 2, 4, 6]),
         ([-1] * 20, [17]), ([-1, -1, 0, 0, 1, 1, 2, 3, 4, 5, 7, 10, 11], [0, 3, 7, 10, 11, 12]),
         (list(range(-1, 62)), list(range(63)))]


def decoys(parents, vocab):
    """Drafts that are not what the model draws (were one, right_path would see a longer path)."""
    return [(1009 * (i + 3)) % vocab for i in range(len(parents))]


@pytest.mark.gpu
@pytest.mark.parametrize("parents,where", TREES)
@pytest.mark.parametrize("rows", [1, 37])
@pytest.mark.parametrize("temperature", [0.0, 2.0])
def test_accepted_path(eng, oracle, parents, where, rows, temperature):
    prompt = np.arange(rows) * 31 + 5
    seq = 1
    first = start(eng, prompt, seq)
    u = np.random.default_rng(len(parents)).random(len(parents) + 1).astype(np.float32)
    tokens, got = right_path(eng, prompt, seq, where, decoys(parents, 4096), parents, u=u, temperature=temperature, top_k=0)
    # the sequence holds the fed token and the accepted drafts; the next one is drawn from the last accepted row
    assert eng.llm_n_past(seq) == rows + len(got)
    lg = eng.llm_logits(seq)
    row = where[-1] + 1 if where else 0
    tok, _, gap = draft_oracle.sample(lg, u[row], np.float32(temperature), 0, np.float32(1), np.float32(0))
    assert tok == got[-1] or gap < 1e-9
    fed = [first] + got[:-1]
    assert cos(lg, oracle_logits(oracle, prompt, fed)) > COS
    # and goes on with the accepted rows' keys and values, step by step and by a chain of drafts
    eng.llm_set_token(seq, 77)
    nxt = int(eng.llm_generate([seq], 1)[0, 0])
    ref = oracle_logits(oracle, prompt, fed + [77])
    assert cos(eng.llm_logits(seq), ref) > COS
    if len(set(fed)) > 3:  # (the bound notices rows in the wrong order)
        assert cos(eng.llm_logits(seq), oracle_logits(oracle, prompt, fed[:1] + fed[:0:-1] + [77])) < COS
    eng.llm_set_token(seq, nxt)
    eng.llm_verify(seq, [])
    assert cos(eng.llm_logits(seq), oracle_logits(oracle, prompt, fed + [77, nxt])) > COS


@pytest.mark.gpu
def test_other_sequences_stay(eng):
    """A verifying step of one sequence leaves the others' rows as they were, and its own committed ones."""
    a, b = np.arange(11) * 17, np.arange(23) * 13
    start(eng, a, 0)
    want = eng.llm_generate([0], 6).tolist()
    last = eng.llm_logits(0)
    start(eng, a, 0)
    start(eng, b, 1)
    eng.llm_verify(1, decoys(range(40), 4096), [-1] * 40)
    start(eng, b, 2)
    eng.llm_verify(2, decoys(range(9), 4096))
    assert eng.llm_generate([0], 6).tolist() == want
    np.testing.assert_array_equal(eng.llm_logits(0), last)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature,top_k,top_p", [(0.9, 0, 1.0), (1.3, 40, 0.9), (1.0, 0, 0.5)])
def test_draws(eng, temperature, top_k, top_p):
    """Each row draws with its own random number; the last one's draw is the oracle's on the engine's logits."""
    parents, where = [-1, -1, 1, 0, 2, 4, 4], [1, 2, 4, 6]
    prompt = np.arange(19) * 23
    samp = dict(temperature=temperature, top_k=top_k, top_p=top_p)
    u = np.random.default_rng(5).random(8).astype(np.float32)
    _, got = right_path(eng, prompt, 0, where, decoys(parents, 4096), parents, u=u, **samp)
    f = np.float32
    tok, _, gap = draft_oracle.sample(eng.llm_logits(0), u[7], f(temperature), top_k, f(top_p), f(0))
    assert tok == got[-1] or gap < 1e-9


@pytest.mark.gpu
def test_duplicate_children_and_repeat(eng):
    """Of two children with the drawn token the first is followed; the same call on the same state gives the same."""
    prompt = np.arange(5) * 7
    start(eng, prompt, 0)
    (t,), _ = eng.llm_verify(0, [])
    runs = []
    for _ in range(2):
        start(eng, prompt, 0)
        runs.append(eng.llm_verify(0, [(t + 1) % 4096, t, t, 9, 9], [-1, -1, -1, 1, 2]) + (eng.llm_logits(0).tobytes(),))
    assert runs[0] == runs[1]
    assert runs[0][0][0] != t or runs[0][1][0] == 1


@pytest.mark.gpu
def test_refusals(eng):
    prompt = np.arange(100) * 3
    eng.llm_reset(0)
    with pytest.raises(RuntimeError, match="prefill first"):
        eng.llm_verify(0, [1])
    start(eng, prompt, 0)
    before = eng.llm_n_past(0)
    for kw, text in [(dict(tokens=[4096]), "token out of range"), (dict(tokens=[-1]), "token out of range"),
                     (dict(tokens=[1, 2], parents=[-1, 1]), "parent"), (dict(tokens=[1], parents=[-2]), "parent"),
                     (dict(tokens=[1] * 64), "63"), (dict(tokens=[1] * 60), "n_ctx"),
                     (dict(tokens=[1], temperature=1.0), "random numbers"),
                     (dict(tokens=[1], temperature=1.0, u=[0.5, 1.0]), "u lies in"),
                     (dict(tokens=[1], temperature=1.0, u=[0.5, float("nan")]), "u lies in"),
                     (dict(tokens=[1], temperature=float("nan"), u=[0.5, 0.5]), "NaN")]:
        with pytest.raises(RuntimeError, match=text):
            eng.llm_verify(0, **kw)
    for kw in [dict(tokens=[1, 2], parents=[-1]), dict(tokens=[1], u=[0.5]), dict(tokens=[[1]])]:
        with pytest.raises(ValueError):
            eng.llm_verify(0, **kw)
    for seq in (-1, 3):
        with pytest.raises(RuntimeError, match="seq out of range"):
            eng.llm_verify(seq, [1])
    eng.llm_generate_begin([0], 2)
    with pytest.raises(RuntimeError, match="in flight"):
        eng.llm_verify(0, [1])
    eng.llm_generate_end()
    assert eng.llm_n_past(0) == before + 2
    # up to the last row of the cache
    n = N_CTX - eng.llm_n_past(0) - 1
    eng.llm_verify(0, [1] * n, [-1] * n)


def test_entry_refuses_without_an_engine():
    from fun_asr_gguf import _native
    lib, n = _native.load(), ctypes.c_int32(-7)
    assert lib.fa_llm_verify(None, 0, None, None, 0, None, None, None, None, ctypes.byref(n)) == -1
    assert n.value == -7 and b"fa_llm_verify" in lib.fa_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("samp", [dict(temperature=0.0), dict(temperature=0.7, top_k=1)])
def test_greedy_is_that_of_the_generating_step_whatever_the_logits(samp):
    """A NaN logit ranks above every number in both, the lower id first; of logits that are all -inf or NaN one is taken."""
    from fun_asr_gguf import _native
    e = _native.Engine(synth.ENC_TINY, dict(synth.LLM_TINY, n_ctx=64, max_seqs=1), max_batch=1, max_samples=16000)
    try:
        e.synthetic_weights(0)
        V, E = 4096, synth.LLM_TINY["n_embd"]
        clean = e.get_tensor_q8_0("token_embd.weight", V * E)
        embd = e.embd_rows(np.arange(9) * 31 + 5)
        for bad in ([], [1234], [3000, 2999], range(V)):
            w = clean.copy().reshape(V, E // 32, 34)
            w[list(bad), 0, :2] = np.float16(np.nan).view(np.uint16).reshape(1).view(np.uint8)
            e.set_tensor_q8_0("token_embd.weight", w.reshape(-1))
            drafts = [7, 9, 11, 13, 15, 17, 19]
            picked = []
            for n in (None, 0, 1, 7):  # the generating step; one row, two, eight
                e.llm_reset(0)
                e.llm_prefill(0, embd)
                e.llm_set_token(0, 77)
                if n is None:
                    picked.append(int(e.llm_generate([0], 1, **samp)[0, 0]))
                else:
                    picked.append(e.llm_verify(0, drafts[:n], [-1] * n, u=np.full(n + 1, 0.5), **samp)[0][0])
            assert len(set(picked)) == 1, (list(bad)[:3], picked)
            if len(bad):
                assert picked[0] == min(bad)
    finally:
        e.close()
