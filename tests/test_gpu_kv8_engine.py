"""Engines with an 8-bit cache, and sequences that begin with the same pages, through the step function and the generation loop,
against the plain model (with its keys and values rounded as the cache rounds them)."""
import subprocess
import sys

import numpy as np
import pytest
import torch

import conftest
import goridra_models as gm
import helpers
import plain_llama
from helpers import TOL
from kv8_plain import quantise, to_bf16

pytestmark = pytest.mark.gpu
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def _engine(model_dirs, name="E", dtype="bfloat16", **kw):
    from oracle_engine_b200.engine.engine import Engine
    kw.setdefault("max_tokens", 4096)
    return Engine.from_pretrained(model_dirs[name], dtype=dtype, **kw)


@pytest.fixture
def rounded(monkeypatch):
    """The plain model reads keys and values as an 8-bit cache keeps them."""
    plain = plain_llama.causal_attention

    def use(kind):
        def attention(q, k, v, window=None):
            def kept(x):
                c, s = quantise(to_bf16(x), CODES[kind])
                return c * s[..., None]
            return plain(q, kept(k), kept(v), window)
        monkeypatch.setattr(plain_llama, "causal_attention", attention)
    return use


@pytest.fixture
def always_share(monkeypatch):
    """Steps read common pages apart however short they are."""
    from oracle_engine_b200.csrc import ops_kv8
    calls = []
    inner = ops_kv8.attention_shared
    monkeypatch.setattr(ops_kv8, "sharing_pays", lambda groups, eight: True)
    monkeypatch.setattr(ops_kv8, "attention_shared", lambda *a, **kw: (calls.append(1), inner(*a, **kw)))
    return calls


def _logits(engine, slot, tokens, portions):
    """Logits of every token, the tokens taken in portions of these sizes (the last size again and again)."""
    from oracle_engine_b200 import SequenceStep
    out, at, i = [], 0, 0
    while at < len(tokens):
        n = min(portions[min(i, len(portions) - 1)], len(tokens) - at)
        out.append(engine.step([SequenceStep(slot, tokens[at:at + n], list(range(n)))]).float().cpu().numpy().copy())
        at, i = at + n, i + 1
    engine.check_device_errors()
    return np.concatenate(out)


@pytest.mark.parametrize("kind", list(CODES))
def test_whole_in_portions_and_token_by_token(model_dirs, plain_models, rounded, kind):
    rounded(kind)
    tokens = helpers.random_tokens(300, 389, 1)
    want = plain_models["E"].logits(tokens).numpy()
    eng = _engine(model_dirs, cache_dtype=kind)
    assert eng.cache.groups[0].storage["codes"].dtype == CODES[kind]
    for portions in ([300], [130, 64, 7, 1, 1, 50], [200, 1]):
        slot = eng.alloc()
        got = _logits(eng, slot, tokens, portions)
        eng.free(slot)
        err = np.abs(got - want).max()
        assert err < TOL["bfloat16"], f"portions {portions}: {err}"
    eng.cache.check()


@pytest.mark.parametrize("kind", list(CODES))
@pytest.mark.parametrize("graphs", [True, False])
def test_ragged_batches_decode_beside_each_other(model_dirs, plain_models, rounded, kind, graphs):
    from oracle_engine_b200 import SequenceStep
    rounded(kind)
    eng = _engine(model_dirs, cache_dtype=kind, use_graphs=graphs)
    prompts = [helpers.random_tokens(n, 389, 10 + n) for n in (3, 70, 129, 260, 64)]
    want = [plain_models["E"].logits(p).numpy() for p in prompts]
    slots = [eng.alloc() for _ in prompts]
    eng.step([SequenceStep(s, p[:-2], []) for s, p in zip(slots, prompts)])
    for i in (2, 1):
        got = eng.step([SequenceStep(s, [p[-i]], [0]) for s, p in zip(slots, prompts)]).float().cpu().numpy()
        for b, w in enumerate(want):
            assert np.abs(got[b] - w[-i]).max() < TOL["bfloat16"]
    eng.check_device_errors()


@pytest.mark.parametrize("kind", list(CODES))
def test_chunks_and_layers_that_read_another_s_cache(tmp_path, kind):
    """The Goridra decoder's attention in chunks with heads of 64: whole prompts against single tokens, in one 8-bit cache."""
    from oracle_engine_b200.engine.engine import Engine
    raw = gm.config(150, 128, 1e-5, [gm.layer(gm.attention(4, 2, 64, 64, 0.125, 70, (24, 50000.0)), gm.dense(64)),
                                     gm.layer(gm.attention(4, 2, 64, 64, 0.2, 100, (24, 50000.0), 0), gm.dense(64)),
                                     gm.layer(gm.attention(2, 1, 64, 64, 0.125), gm.dense(64))])
    folder = gm.write(tmp_path, raw, 3)
    eng = Engine.from_pretrained(folder, dtype="bfloat16", max_tokens=2048, cache_dtype=kind)
    sixteen = Engine.from_pretrained(folder, dtype="bfloat16", max_tokens=2048)
    tokens = helpers.random_tokens(333, 150, 4)
    slot = eng.alloc()
    whole = _logits(eng, slot, tokens, [333])
    eng.free(slot)
    slot = eng.alloc()
    single = _logits(eng, slot, tokens, [20, 1])
    eng.free(slot)
    slot = sixteen.alloc()
    plain = _logits(sixteen, slot, tokens, [333])
    size = np.sqrt((plain ** 2).mean())
    assert np.sqrt(((whole - single) ** 2).mean()) / size < TOL["bfloat16"]
    # e4m3 keeps 4 bits of a value: 2^-4 of each at most, and a layer's output is an average of such values
    assert np.sqrt(((whole - plain) ** 2).mean()) / size < (TOL["bfloat16"] if kind == "int8" else 2.0 ** -4 + TOL["bfloat16"])
    eng.cache.check()


@pytest.mark.parametrize("dtype,kind", [("float32", None), ("bfloat16", None), ("bfloat16", "int8"), ("bfloat16", "fp8")])
@pytest.mark.parametrize("graphs", [True, False])
def test_forks_go_on_as_if_alone(model_dirs, plain_models, rounded, always_share, dtype, kind, graphs):
    """Two bases, forks of each, a fork of a fork and a sequence on its own decode in one step; forks come and go."""
    from oracle_engine_b200 import SequenceStep
    if kind:
        rounded(kind)
    plain = plain_models["E"]
    eng = _engine(model_dirs, dtype=dtype, cache_dtype=kind, use_graphs=graphs)
    base = [helpers.random_tokens(n, 389, 30 + n) for n in (128, 64)]
    slots = [eng.alloc() for _ in base]
    eng.step([SequenceStep(s, t, []) for s, t in zip(slots, base)])
    live = {}                                               # slot -> its tokens
    for k, n in ((0, 3), (1, 2)):
        for _ in range(n):
            live[eng.fork(slots[k])] = list(base[k])
    alone = eng.alloc()
    live[alone] = helpers.random_tokens(70, 389, 40)
    eng.step([SequenceStep(alone, live[alone], [])])
    eng.free(slots[0])                                      # its forks keep the pages
    live[slots[1]] = list(base[1])
    rng = np.random.default_rng(5)

    def decode(steps):
        for _ in range(steps):
            order = list(live)
            new = [int(t) for t in rng.integers(0, 389, len(order))]
            got = eng.step([SequenceStep(s, [t], [0]) for s, t in zip(order, new)]).float().cpu().numpy()
            for i, (s, t) in enumerate(zip(order, new)):
                live[s].append(t)
                want = plain.logits(live[s])[-1].numpy()
                assert np.abs(got[i] - want).max() < TOL[dtype], f"{len(live[s])} tokens"
    decode(3)
    some = next(s for s in live if len(live[s]) == 131)
    grow = helpers.random_tokens(192 - 131, 389, 41)        # to a whole number of pages, then fork the fork
    eng.step([SequenceStep(some, grow, [])])
    live[some] += grow
    live[eng.fork(some)] = list(live[some])
    decode(2)
    for s in list(live)[:2]:
        eng.free(s)
        del live[s]
    decode(2)
    eng.cache.check()
    for s in list(live):
        eng.free(s)
    eng.cache.check()
    eng.check_device_errors()
    assert all(g.pool.n_free == g.pool.n for g in eng.cache.groups)
    assert bool(always_share) == (dtype == "bfloat16")


def test_forks_of_recurrent_layers_take_their_state(tmp_path):
    import fuvipel_models as fm
    from oracle_engine_b200 import SequenceStep
    from oracle_engine_b200.engine.engine import Engine
    folder = fm.write(tmp_path, *fm.ALL["F1"])
    eng = Engine.from_pretrained(folder, dtype="float32", max_tokens=1024)
    tokens = helpers.random_tokens(64, 300, 6)
    a = eng.alloc()
    eng.step([SequenceStep(a, tokens, [])])
    b = eng.fork(a)
    for t in helpers.random_tokens(5, 300, 7):
        one = eng.step([SequenceStep(a, [t], [0])]).clone()
        two = eng.step([SequenceStep(b, [t], [0])]).clone()
        assert torch.equal(one, two)


@pytest.mark.parametrize("dtype,kind", [("float32", None), ("bfloat16", None), ("bfloat16", "int8"), ("bfloat16", "fp8")])
@pytest.mark.parametrize("portion", [None, 50])
def test_generation_with_common_beginnings(model_dirs, plain_models, rounded, always_share, dtype, kind, portion):
    from oracle_engine_b200 import GenParams
    if kind:
        rounded(kind)
    plain = plain_models["E"]
    eng = _engine(model_dirs, dtype=dtype, cache_dtype=kind)
    common = helpers.random_tokens(200, 389, 50)
    prompts = [common + helpers.random_tokens(3 + 30 * i, 389, 51 + i) for i in range(4)]
    prompts += [helpers.random_tokens(90, 389, 60), common[:130] + [1], common[:64] + helpers.random_tokens(5, 389, 61)]
    params = GenParams.greedy(6, ignore_eos=True)
    free = [g.pool.n_free for g in eng.cache.groups]
    got = eng.generate(prompts, params, max_step_tokens=portion, share_prefix=True)
    assert [g.pool.n_free for g in eng.cache.groups] == free
    eng.cache.check()
    for p, g in zip(prompts, got):
        assert len(g) == 6
        seq = list(p)
        for tok in g:
            lg = plain.logits(seq)[-1]
            assert lg.max().item() - lg[tok].item() <= 2 * TOL[dtype]
            seq.append(tok)
    if dtype == "float32":
        assert got == eng.generate(prompts, params, max_step_tokens=portion)


def test_refusals(model_dirs, tmp_path):
    from oracle_engine_b200 import SequenceStep
    from oracle_engine_b200.engine.engine import Engine
    import fuvipel_models as fm
    for kw in ({"dtype": "float32"}, {"tensor_cores": False}, {"cache_dtype": "int4"}):
        with pytest.raises(ValueError):
            _engine(model_dirs, **{"cache_dtype": "int8", **kw})
    with pytest.raises(ValueError, match="heads of"):
        _engine(model_dirs, "B", cache_dtype="int8")
    with pytest.raises(ValueError, match="no 8-bit cache"):
        Engine.from_pretrained(fm.write(tmp_path, *fm.ALL["F1"]), dtype="bfloat16", max_tokens=512, cache_dtype="fp8")
    eng = _engine(model_dirs)
    slot = eng.alloc()
    with pytest.raises(ValueError, match="whole pages"):
        eng.fork(slot)
    eng.step([SequenceStep(slot, [1] * 65, [])])
    with pytest.raises(ValueError, match="whole pages"):
        eng.fork(slot)
    eng.free(slot)
    with pytest.raises(ValueError, match="not held"):
        eng.fork(slot)


def test_command_lines(model_dirs, tmp_path):
    """bin/oracle and bin/trace_run take the cache's type; the former common beginnings."""
    common = ",".join(str(t) for t in helpers.random_tokens(70, 389, 70))
    cmd = [sys.executable, str(helpers.ROOT / "bin" / "oracle"), "-m", model_dirs["E"], "-n", "4", "--temp", "0", "--ignore-eos",
           "--tokens", common + ",5", "--tokens", common + ",6,7"]
    for more in ([], ["--cache-dtype", "int8", "--share-prefix"], ["--cache-dtype", "fp8"]):
        r = subprocess.run(cmd + more, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0 and [len(x.split()) for x in r.stdout.strip().splitlines()] == [4, 4], r.stderr
    r = subprocess.run(cmd + ["--cache-dtype", "int4"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 1 and "int8 or fp8" in r.stderr
    r = subprocess.run([sys.executable, str(helpers.ROOT / "bin" / "trace_run"), "--model", model_dirs["E"], "--dtype", "bfloat16", "--out",
                        str(tmp_path), "--max-tokens", "512", "--cache-dtype", "fp8"], capture_output=True, text=True, timeout=300,
                       input='{"step": 0, "entries": [{"id": "a", "tokens": [1, 2, 3], "want": [2]}], "end": ["a"]}\n')
    assert r.returncode == 0 and r.stdout.split() == ["done", "0"], r.stderr
