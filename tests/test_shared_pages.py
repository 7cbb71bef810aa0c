"""Pages that several sequences hold, 8-bit caches' storage, and how the generation loop uses common beginnings (no GPU)."""
import random

import numpy as np
import pytest
import torch

from oracle_engine_b200 import GenParams
from oracle_engine_b200.cache.kv_cache import KVCache
from oracle_engine_b200.cache.slots import CacheFull, PagePool
from oracle_engine_b200.cache.state import StateStore
from oracle_engine_b200.engine.batch import shared_prefixes
from oracle_engine_b200.engine.engine import check_cache_form
from oracle_engine_b200.engine.generate import common_prefixes, run_generation
from oracle_engine_b200.engine.runtime import Runtime, parse_cache_dtype
from oracle_engine_b200.parts.spec import CacheNeed, StateNeed, attention_cache_need
from test_generate_loop import Scripted, ScriptedAhead

FULL, WIN = attention_cache_need(2, 16), attention_cache_need(2, 16, 100)


def grow(c, slot, n):
    c.reserve(slot, c.length(slot) + n)
    c.commit(slot, c.length(slot) + n)


def test_pool_keeps_a_page_until_its_last_holder():
    p = PagePool(4)
    a, b = p.alloc_many(2)
    p.share([a, b])
    p.share([a])
    p.check()
    assert [p.holders(x) for x in (a, b, 3)] == [3, 2, 0]
    p.release_all([a, b])
    p.release(a)
    p.check()
    assert p.holders(a) == p.holders(b) == 1 and p.n_free == 2
    p.release_all([a, b])
    p.check()
    assert p.n_free == 4
    for bad in ([a], [0, 0]):
        with pytest.raises(ValueError):
            p.share(bad)
    with pytest.raises(ValueError):
        p.release(a)


def test_fork_shares_whole_pages():
    c = KVCache([FULL, WIN, None, FULL], 64 * 20, 64 * 10, allocate=False, n_slots=5)
    base = c.alloc_slot()
    for n in (0, 1, 63):
        if n:
            grow(c, base, n)
            n = c.length(base)
        if n % 64 or n == 0:
            with pytest.raises(ValueError):
                c.fork(base)
    assert c.length(base) == 64
    grow(c, base, 64)
    free = [g.pool.n_free for g in c.groups]
    version = c.version
    kids = [c.fork(base) for _ in range(3)]
    assert c.version > version and [g.pool.n_free for g in c.groups] == free
    assert all(c.length(k) == 128 for k in kids) and len({c.prefix[s] for s in [base] + kids}) == 1
    for k in kids:
        grow(c, k, 70)
        c.check()
    for g in c.groups:
        assert len({tuple(g.tables[s][:2]) for s in [base] + kids}) == 1
        assert len({int(g.tables[s][2]) for s in kids}) == 3
    c.free_slot(base)
    c.check()
    for k in kids:
        grow(c, k, 200)                     # the window group gives its part of the common pages back
        c.check()
    c.free_slot(kids[0])
    again = c.alloc_slot()
    assert c.prefix[again] is None
    c.check()
    for s in (again, kids[1], kids[2]):
        c.free_slot(s)
    c.check()
    assert all(g.pool.n_free == g.pool.n for g in c.groups)


def test_a_page_reserved_beyond_the_length_is_not_shared():
    c = KVCache([FULL], 64 * 8, 64 * 8, allocate=False, n_slots=3)
    base = c.alloc_slot()
    grow(c, base, 64)
    c.reserve(base, 65)                     # a step that was not committed
    kid = c.fork(base)
    grow(c, kid, 1)
    grow(c, base, 1)
    c.check()
    assert c.groups[0].tables[base][1] != c.groups[0].tables[kid][1]


def test_what_others_hold_is_not_counted_as_room():
    """A window that moves on gives its pages back, but a page that another sequence holds too does not become free by that."""
    c = KVCache([attention_cache_need(1, 8, 64)], 64 * 4, 64 * 4, allocate=False, n_slots=3)
    base = c.alloc_slot()
    grow(c, base, 128)
    kid = c.fork(base)
    other = c.alloc_slot()
    grow(c, other, 128)                     # every page of the pool is in use
    before = (c.groups[0].tables.copy(), c.groups[0].pool.n_free, c.version)
    with pytest.raises(CacheFull):
        grow(c, kid, 64)
    assert (c.groups[0].tables == before[0]).all() and (c.groups[0].pool.n_free, c.version) == before[1:]
    c.check()
    c.free_slot(base)
    grow(c, kid, 64)
    c.check()


def test_marks_of_forks_at_other_lengths():
    c = KVCache([FULL], 64 * 30, 64 * 10, allocate=False, n_slots=8)
    base = c.alloc_slot()
    grow(c, base, 64)
    a, b = c.fork(base), c.fork(base)
    grow(c, base, 64)
    d = c.fork(base)
    assert c.prefix[a] == c.prefix[b] != c.prefix[d] == c.prefix[base] and c.prefix[d][1] == 2
    grow(c, a, 64)
    e = c.fork(a)
    assert c.prefix[e] == c.prefix[a] and c.prefix[e] not in (c.prefix[b], c.prefix[d])
    c.check()
    while True:
        try:
            c.fork(base)
        except CacheFull:
            break
    c.check()


def test_random_forks_lose_nothing():
    r = random.Random(5)
    c = KVCache([FULL, WIN, attention_cache_need(1, 8, -90)], 64 * 60, 64 * 12, allocate=False, n_slots=12)
    live = []
    for _ in range(600):
        what = r.random()
        try:
            if what < 0.2 or not live:
                live.append(c.alloc_slot())
            elif what < 0.35:
                s = r.choice(live)
                if c.length(s) and c.length(s) % 64 == 0:
                    live.append(c.fork(s))
            elif what < 0.5:
                c.free_slot(live.pop(r.randrange(len(live))))
            else:
                grow(c, r.choice(live), r.choice([1, 64, 64 - c.length(live[0]) % 64, r.randint(1, 100)]))
        except CacheFull:
            c.free_slot(live.pop(r.randrange(len(live))))
        c.check()


def test_state_rows_are_copied():
    s = StateStore(3, "cpu")
    a, b = s.add(0, "a", StateNeed((2, 3), torch.float32)), s.add(1, "b", StateNeed((), torch.int64))
    a[1], b[1] = 5.0, 7
    s.copy(1, 2)
    assert (a[2] == 5).all() and b[2] == 7 and (a[0] == 0).all()
    with pytest.raises(IndexError):
        s.copy(0, 3)


def test_storage_of_an_8_bit_cache():
    need = attention_cache_need(3, 64, 0, torch.int8)
    assert need.bytes_per_token(2) == 2 * 3 * (64 + 4) and attention_cache_need(3, 64).bytes_per_token(2) == 2 * 3 * 64 * 2
    c = KVCache([need, attention_cache_need(3, 64)], 64 * 4, 64 * 4, dtype=torch.bfloat16, device="cpu")
    st = c.storage_of(0)
    assert st["codes"].dtype == torch.int8 and tuple(st["codes"].shape) == (4, 2, 3, 64, 64)
    assert st["scales"].dtype == torch.float32 and tuple(st["scales"].shape) == (4, 2, 3, 64, 1)
    assert c.storage_of(1)["kv"].dtype == torch.bfloat16
    assert c.total_bytes(2) == 256 * (2 * 3 * 68 + 2 * 3 * 64 * 2)
    from oracle_engine_b200.cache.kv_cache import CacheView
    codes, scales = CacheView(st, None, 0).kv
    assert codes is st["codes"] and scales.is_contiguous() and tuple(scales.shape) == (4, 2, 3, 64)
    joined = attention_cache_need(3, 64, 100, torch.int8).joined(attention_cache_need(3, 64, 0, torch.int8))
    assert joined == need
    joined = attention_cache_need(3, 64, 100, torch.int8).joined(attention_cache_need(3, 64, 200, torch.int8))
    assert joined.dtypes == need.dtypes


def test_cache_types_by_name():
    assert parse_cache_dtype(None) is None and parse_cache_dtype("same") is None
    assert parse_cache_dtype("INT8") is torch.int8 and parse_cache_dtype("fp8") is torch.float8_e4m3fn
    assert parse_cache_dtype(torch.int8) is torch.int8
    for bad in ("int4", "bf16", torch.bfloat16):
        with pytest.raises(ValueError, match="int8 or fp8"):
            parse_cache_dtype(bad)


def test_models_without_an_8_bit_form_are_refused():
    from oracle_engine_b200.config.base import get_architecture
    from oracle_engine_b200.parts.model import DecoderModel
    import conftest
    import fuvipel_models as fm
    rt = Runtime(torch.bfloat16, torch.device("cpu"), True, torch.int8)

    def model(raw):
        arch = get_architecture(raw.get("architecture") or raw["architectures"][0])
        return DecoderModel(arch.build_spec(arch.config_cls.from_dict(raw), 256), rt)
    check_cache_form(model(conftest.TINY_E), rt)
    with pytest.raises(ValueError, match="heads of"):
        check_cache_form(model(conftest.TINY_B), rt)
    with pytest.raises(ValueError, match="no 8-bit cache"):
        check_cache_form(model(fm.F1), rt)


# ------------------------------------------------------------------------------------------------ steps and prompts
def test_when_sharing_pays():
    from oracle_engine_b200.csrc.ops_kv8 import sharing_pays
    assert not sharing_pays([], False) and not sharing_pays([(2, 1), (60, 1)], False)
    assert sharing_pays([(16, 64)], False) and sharing_pays([(64, 32)], False) and not sharing_pays([(16, 16)], False)
    assert sharing_pays([(64, 16)], True) and not sharing_pays([(2, 64)], True) and sharing_pays([(6, 64), (4, 64)], True)
    assert sharing_pays([(8, 64)], False) and not sharing_pays([(2, 300)], False) and not sharing_pays([(4, 128)], False)
    assert shared_prefixes([(1, 3)] * 8, 8) is None and shared_prefixes([(1, 300)] * 8, 8) is not None


def test_groups_of_a_step(monkeypatch):
    from oracle_engine_b200.csrc import ops_kv8
    monkeypatch.setattr(ops_kv8, "sharing_pays", lambda groups, eight: True)
    assert shared_prefixes([None, (1, 3), None], 4) is None and shared_prefixes([(1, 2), (2, 2)], 2) is None
    p = shared_prefixes([(1, 3), None, (2, 5), (1, 3), (3, 1), (2, 5), (1, 3)], 8)
    members, first, pages, seq_pages = p.arrays
    assert p.shape == (2, 8, 8)
    assert members[:5].tolist() == [0, 3, 6, 2, 5] and first.tolist() == [0, 3, 5] and pages.tolist() == [3, 5]
    assert seq_pages.tolist() == [3, 0, 5, 3, 0, 5, 3, 0]
    p = shared_prefixes([(g, 2) for g in range(3) for _ in range(2)], 6)
    assert p.n_groups == 4 and p.arrays[1].tolist() == [0, 2, 4, 6, 6] and p.arrays[2].tolist() == [2, 2, 2, 0]
    assert p.n_members == 6


def test_what_prompts_have_in_common():
    a, b = list(range(300)), list(range(1000, 1300))
    prompts = [a[:200] + [7], a[:250], b[:100], a[:64] + [1] * 64, b[:70], a[:64], [5], a[:200] + [9]]
    got = common_prefixes(prompts, list(range(len(prompts))))
    assert got == [([0, 1, 3, 7], 64), ([2, 4], 64)]
    assert common_prefixes(prompts, [0, 1, 7]) == [([0, 1, 7], 192)]
    assert common_prefixes([a[:128], a[:128]], [0, 1]) == [([0, 1], 64)]          # a token of each is left
    assert common_prefixes([a[:129], a[:129]], [0, 1]) == [([0, 1], 128)]
    assert common_prefixes(prompts, [2]) == [] and common_prefixes([a[:64], a[:64]], [0, 1]) == []
    r = random.Random(3)
    for _ in range(200):
        n = r.randint(2, 5)
        base = [r.randint(0, 1) for _ in range(400)]
        ps = []
        for _ in range(n):
            k = r.randint(60, 300)
            ps.append(base[:k] + [r.randint(0, 1) for _ in range(r.randint(1, 50))])
        for members, m in common_prefixes(ps, list(range(n))):
            assert m % 64 == 0 and m >= 64 and all(len(ps[i]) > m and ps[i][:m] == ps[members[0]][:m] for i in members)
            longer = [ps[i][:m + 64] for i in members]
            assert any(len(p) < m + 64 or p != longer[0] for p in longer) or min(len(ps[i]) for i in members) <= m + 64


class Sharing:
    def alloc_prefix(self):
        slot = self.free_slots.pop(0)
        self.owner[slot] = "prefix"
        return slot

    def alloc_behind(self, base, i, prompt, params):
        assert self.owner[base] == "prefix"
        self.events.append(("behind", i, base))
        return self.alloc(i, prompt, params)


class ScriptedSharing(Sharing, Scripted):
    pass


class ScriptedSharingAhead(Sharing, ScriptedAhead):
    pass


@pytest.mark.parametrize("backend", [ScriptedSharing, ScriptedSharingAhead])
@pytest.mark.parametrize("portion", [None, 100])
def test_the_common_part_goes_through_once(backend, portion):
    common = list(range(200))
    prompts = [common + [1, 2], [9, 8], common + [3], common[:192] + [4] * 10]
    b = backend([[5, 6, 7]] * 4, n_slots=5, max_seq_len=400)
    got = run_generation(b, prompts, GenParams.greedy(3), max_step_tokens=portion, share_prefix=True)
    assert [g.tokens for g in got] == [[5, 6, 7]] * 4
    first = [s for s in b.steps if s[0][0] == "prefix"]
    assert [x[0][1] for x in first] == ([common[:192]] if portion is None else [common[:100], common[100:192]])
    assert all(x[0][2] == [] for x in first)
    fed = {i: [] for i in range(4)}
    for s in b.steps:
        for who, toks, want in s:
            if who != "prefix" and toks[0] != "ahead":
                fed[who] += toks
    assert fed[0][:10] == prompts[0][192:] and fed[1][:2] == [9, 8] and fed[2][:9] == prompts[2][192:]
    assert sorted(b.free_slots) == list(range(5))


def test_a_common_part_that_cannot_be_held_gives_its_slots_back():
    common = list(range(100))
    b = ScriptedSharing([[5]] * 3, n_slots=3, max_seq_len=400)
    with pytest.raises(IndexError):
        run_generation(b, [common + [i] for i in range(3)], GenParams.greedy(1), share_prefix=True)
    assert sorted(b.free_slots) == [0, 1, 2]


def test_without_the_option_or_tokens_nothing_is_shared():
    common = list(range(100))
    b = ScriptedSharing([[5]] * 2, n_slots=2, max_seq_len=400)
    run_generation(b, [common + [i] for i in range(2)], GenParams.greedy(1))
    run_generation(b, [common + [i] for i in range(2)], GenParams.greedy(0), share_prefix=True)
    assert not [e for e in b.events if e[0] == "behind"]
