"""Engines whose requests start behind what their prompts have in common."""
import pytest

import helpers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("params", [dict(temperature=0.0), dict(temperature=0.8, top_k=30, repeat_penalty=1.2, seed=5)])
def test_as_many_slots_as_requests(model_dirs, params):
    """Tokens, random draws among them, are those of the batch without common beginnings."""
    from oracle_engine_b200 import GenParams
    from oracle_engine_b200.engine.engine import Engine
    eng = Engine.from_pretrained(model_dirs["E"], dtype="float32", max_tokens=2048, n_slots=4)
    common = helpers.random_tokens(150, 389, 1)
    prompts = [common + helpers.random_tokens(3 + 20 * i, 389, 2 + i) for i in range(4)]
    p = GenParams(n_predict=6, ignore_eos=True, **params)
    want = eng.generate(prompts, p)
    for _ in range(2):
        assert eng.generate(prompts, p, share_prefix=True) == want
        eng.cache.check()
    assert eng.cache.slots.n_free == 4


def test_recurrent_layers_in_the_common_tokens_own_slot(tmp_path):
    import fuvipel_models as fm
    from oracle_engine_b200 import GenParams
    from oracle_engine_b200.engine.engine import Engine
    eng = Engine.from_pretrained(fm.write(tmp_path, *fm.ALL["F1"]), dtype="float32", max_tokens=1024, n_slots=3)
    common = helpers.random_tokens(64, 300, 6)
    prompts = [common + helpers.random_tokens(4 + i, 300, 7 + i) for i in range(3)]
    p = GenParams.greedy(5, ignore_eos=True)
    alone = [eng.generate([q], p)[0] for q in prompts]
    shared = eng.generate(prompts, p, share_prefix=True)
    cut = [eng.generate([q], p, max_step_tokens=64)[0] for q in prompts]
    assert shared in (alone, cut)
    eng.cache.check()


def test_groups_within_a_group(model_dirs):
    """Prompts that are a tree of pages: some have more in common than all of them have."""
    from oracle_engine_b200 import GenParams
    from oracle_engine_b200.engine.engine import Engine
    eng = Engine.from_pretrained(model_dirs["E"], dtype="float32", max_tokens=4096, n_slots=8)
    text, docs = helpers.random_tokens(70, 389, 1), [helpers.random_tokens(n, 389, n) for n in (130, 200)]
    prompts = [text[:64] + docs[i % 2] + helpers.random_tokens(3 + i, 389, 20 + i) for i in range(6)]
    prompts += [text + [3], helpers.random_tokens(100, 389, 40)]
    p = GenParams.greedy(5, ignore_eos=True)
    want = eng.generate(prompts, p)
    for portion in (None, 100):
        assert eng.generate(prompts, p, share_prefix=True, max_step_tokens=portion) == want
        eng.cache.check()
    assert eng.cache.slots.n_free == 8


def test_captured_steps_of_many_shapes(model_dirs, monkeypatch):
    """More shapes of groups than graphs are kept for, each used until it is captured and replayed, and the first once more."""
    import numpy as np

    from oracle_engine_b200 import SequenceStep
    from oracle_engine_b200.csrc import ops_kv8
    from oracle_engine_b200.engine import step
    from oracle_engine_b200.engine.engine import Engine
    monkeypatch.setattr(ops_kv8, "sharing_pays", lambda *a: True)
    monkeypatch.setattr(step, "MAX_PREFIX_GRAPHS", 3)
    eng = Engine.from_pretrained(model_dirs["E"], dtype="bfloat16", max_tokens=8192)
    alone = Engine.from_pretrained(model_dirs["E"], dtype="bfloat16", max_tokens=8192)
    for n, pages in ((2, 1), (3, 1), (5, 2), (9, 1), (2, 5), (3, 1), (2, 1)):
        common = helpers.random_tokens(64 * pages, 389, 7 + pages)
        slots = []
        for e in (eng, alone):
            base = e.alloc()
            e.step([SequenceStep(base, common, [])])
            slots.append([e.fork(base) for _ in range(n)])
            e.free(base)
        alone.cache.prefix = [None] * alone.cache.n_slots
        for k in range(4):
            toks = helpers.random_tokens(n, 389, 100 * n + k)
            got, want = (e.step([SequenceStep(s, [t], [0]) for s, t in zip(sl, toks)]).float().cpu().numpy().copy()
                         for e, sl in zip((eng, alone), slots))
            assert np.abs(got - want).max() < helpers.TOL["bfloat16"]
        assert len(eng.stepper._prefix_graphs) <= 3 and not alone.stepper._prefix_graphs
        for e, sl in zip((eng, alone), slots):
            for s in sl:
                e.free(s)
    eng.check_device_errors()


def test_steps_that_read_no_page_apart_are_captured_once(model_dirs, monkeypatch):
    """A float32 engine's kernels do not look at the groups: their shapes are no part of what is captured."""
    from oracle_engine_b200 import SequenceStep
    from oracle_engine_b200.csrc import ops_kv8
    from oracle_engine_b200.engine.engine import Engine
    monkeypatch.setattr(ops_kv8, "sharing_pays", lambda *a: True)
    eng = Engine.from_pretrained(model_dirs["E"], dtype="float32", max_tokens=4096)
    for n in (5, 6, 7):
        base = eng.alloc()
        eng.step([SequenceStep(base, helpers.random_tokens(128, 389, 1), [])])
        slots = [eng.fork(base) for _ in range(n)] + [base]
        for _ in range(2):
            eng.step([SequenceStep(s, [7], [0]) for s in slots])
        for s in slots:
            eng.free(s)
    assert list(eng.stepper._graphs) == [(8, 0)] and not eng.stepper._prefix_graphs


@pytest.mark.parametrize("dtype,kind", [("float32", None), ("bfloat16", None), ("bfloat16", "int8")])
def test_forks_over_chunks_and_another_entry_s_cache(tmp_path, monkeypatch, dtype, kind):
    """Layers of chunks give their part of the common pages back one sequence at a time, beside a layer that keeps all of them."""
    import numpy as np

    import goridra_models as gm
    from oracle_engine_b200 import SequenceStep
    from oracle_engine_b200.csrc import ops_kv8
    from oracle_engine_b200.engine.engine import Engine
    monkeypatch.setattr(ops_kv8, "sharing_pays", lambda *a: True)
    raw = gm.config(150, 128, 1e-5, [gm.layer(gm.attention(4, 2, 64, 64, 0.125, 70, (24, 50000.0)), gm.dense(64)),
                                     gm.layer(gm.attention(4, 2, 64, 64, 0.2, 100, (24, 50000.0), 0), gm.dense(64)),
                                     gm.layer(gm.attention(2, 1, 64, 64, 0.125), gm.dense(64))])
    eng = Engine.from_pretrained(gm.write(tmp_path, raw, 3), dtype=dtype, max_tokens=4096, cache_dtype=kind)
    common = helpers.random_tokens(128, 150, 4)
    tails = [helpers.random_tokens(90, 150, 5 + i) for i in range(3)]

    def run(shared):
        if shared:
            base = eng.alloc()
            eng.step([SequenceStep(base, common, [])])
            slots = [eng.fork(base) for _ in tails]
            eng.free(base)
        else:
            slots = [eng.alloc() for _ in tails]
            for s in slots:
                eng.step([SequenceStep(s, common, [])])
        out = []
        for at, n in ((0, 40), (40, 1), (41, 1), (42, 40)) + tuple((82 + i, 1) for i in range(8)):
            got = eng.step([SequenceStep(s, t[at:at + n], [n - 1]) for s, t in zip(slots, tails)])
            out.append(got.float().cpu().numpy().copy())
            eng.cache.check()
        for s in slots:
            eng.free(s)
        return np.stack(out)
    alone, forked = run(False), run(True)
    if dtype == "float32":
        assert np.array_equal(alone, forked)
    assert np.sqrt(((alone - forked) ** 2).mean() / (alone ** 2).mean()) < helpers.TOL[dtype]
    eng.check_device_errors()
