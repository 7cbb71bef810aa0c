"""How the generation loop starts requests behind what their prompts have in common: slots and steps (no GPU)."""
import pytest

from oracle_engine_b200 import GenParams
from oracle_engine_b200.engine.generate import run_generation
from test_generate_loop import Scripted, ScriptedAhead


class Taking:
    """A backend whose slots remember the tokens they hold; a request may go on in a prefix's slot."""

    def _note(self, slot, tokens):
        self.held[slot] = list(tokens)

    def alloc(self, i, prompt, params):
        slot = super().alloc(i, prompt, params)
        self._note(slot, [])
        return slot

    def step(self, seqs):
        for s in seqs:
            self.held[s.slot] += s.tokens
        return super().step(seqs)

    def alloc_prefix(self):
        slot = self.free_slots.pop(0)
        self.owner[slot] = "prefix"
        self._note(slot, [])
        return slot

    def alloc_behind(self, base, i, prompt, params):
        assert self.owner[base] == "prefix" and prompt[:len(self.held[base])] == self.held[base]
        slot = self.alloc(i, prompt, params)
        self._note(slot, self.held[base])
        return slot

    def take_prefix(self, base, i, prompt, params):
        assert self.owner[base] == "prefix" and prompt[:len(self.held[base])] == self.held[base]
        if i == self.fails:
            raise RuntimeError("no")
        self.owner[base], self.pos[i] = i, 0
        self.events.append(("taken", i, base))


class Plain(Taking, Scripted):
    fails = None

    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.held = {}

    def fed(self):
        """Per request the tokens of its prompt's own steps, and per step those of prefixes."""
        mine, prefix = {}, []
        for st in self.steps:
            for who, toks, _ in st:
                if who != "prefix":
                    mine.setdefault(who, []).extend(toks if toks[0] != "ahead" else [])
            prefix += [[toks for who, toks, _ in st if who == "prefix"]] if any(who == "prefix" for who, _, _ in st) else []
        return mine, prefix


class Ahead(Plain, ScriptedAhead):
    pass


@pytest.mark.parametrize("backend", [Plain, Ahead])
@pytest.mark.parametrize("portion", [None, 50])
def test_as_many_slots_as_requests(backend, portion):
    common = list(range(100))
    prompts = [common + [200 + i] for i in range(4)]
    for n in (2, 4):
        b = backend([[5, 6]] * n, n_slots=n, max_seq_len=400)
        got = run_generation(b, prompts[:n], GenParams.greedy(2), max_step_tokens=portion, share_prefix=True)
        assert [g.tokens for g in got] == [[5, 6]] * n
        mine, prefix = b.fed()
        assert sum(len(t) for p in prefix for t in p) == 64
        assert all(mine[i][:37] == prompts[i][64:] for i in range(n))
        assert sorted(b.free_slots) == list(range(n))


@pytest.mark.parametrize("fails", [None, 3])
def test_slots_go_back_when_a_request_cannot_start(fails):
    common = list(range(100))
    b = Plain([[5]] * 4, n_slots=4 if fails else 3, max_seq_len=400)
    b.fails = fails
    with pytest.raises(RuntimeError if fails else IndexError):
        run_generation(b, [common + [i] for i in range(4)], GenParams.greedy(1), share_prefix=True)
    assert sorted(b.free_slots) == list(range(4 if fails else 3))


class Tree(Plain):
    def fork_prefix(self, base):
        assert self.owner[base] == "prefix"
        slot = self.alloc_prefix()
        self._note(slot, self.held[base])
        return slot


def _tree(prompts, portion=None):
    n = len(prompts)
    b = Tree([[5, 6]] * n, n_slots=n, max_seq_len=10000)
    got = run_generation(b, prompts, GenParams.greedy(2), max_step_tokens=portion, share_prefix=True)
    assert [g.tokens for g in got] == [[5, 6]] * n
    mine, prefix = b.fed()
    assert sorted(b.free_slots) == list(range(n))
    for i, p in enumerate(prompts):
        own = mine[i][:-1]                       # (the last one is its first token)
        assert own and own == p[len(p) - len(own):]
    if portion is not None:
        assert all(sum(len(t) for t in st) <= portion for st in prefix)
    return {i: len(p) - len(mine[i]) + 1 for i, p in enumerate(prompts)}, prefix


@pytest.mark.parametrize("portion", [None, 100])
def test_one_request_that_shares_little_does_not_take_it_from_the_others(portion):
    long = list(range(1000))
    prompts = [long + [2000 + i] for i in range(5)] + [long[:64] + [1]]
    shared, prefix = _tree(prompts, portion)
    assert shared == {0: 960, 1: 960, 2: 960, 3: 960, 4: 960, 5: 64}
    assert sum(len(t) for st in prefix for t in st) == 960


def test_two_documents_behind_one_text():
    text, docs = list(range(128)), [list(range(1000, 1320)), list(range(2000, 2200))]
    prompts = [text + docs[i % 2] + [i] for i in range(6)]
    shared, prefix = _tree(prompts)
    assert shared == {i: 448 if i % 2 == 0 else 320 for i in range(6)}
    # the text in one step, what the documents' requests have in common in one more
    assert [sorted(len(t) for t in st) for st in prefix] == [[128], [192, 320]]


def test_every_prompt_goes_on_from_the_one_before():
    talk = list(range(64 * 6))
    shared, prefix = _tree([talk[:64 * k] + [9000 + k] for k in range(1, 7)])
    assert shared == {0: 64, 1: 128, 2: 192, 3: 256, 4: 320, 5: 320}
    assert sum(len(t) for st in prefix for t in st) == 320


def test_prompts_of_random_trees():
    import random
    r = random.Random(9)
    for _ in range(60):
        stems = [[r.randint(0, 3) for _ in range(r.randint(0, 3) * 64 + r.randint(0, 40))] for _ in range(3)]
        prompts = []
        for _ in range(r.randint(1, 9)):
            p = []
            for _ in range(r.randint(1, 3)):
                p = p + r.choice(stems)
            prompts.append(p + [r.randint(0, 3) for _ in range(r.randint(1, 5))])
        shared, prefix = _tree(prompts, r.choice([None, 30, 64, 1000]))
        # every page that two prompts have in common, a token of each left, is computed once
        pages = {}
        for p in prompts:
            for k in range(64, len(p), 64):
                pages.setdefault(tuple(p[:k]), []).append(1)
        assert sum(len(t) for st in prefix for t in st) == 64 * sum(1 for c in pages.values() if len(c) > 1)
        for i, p in enumerate(prompts):
            assert shared[i] == max([k for k in range(64, len(p), 64) if len(pages[tuple(p[:k])]) > 1], default=0)


def test_a_deep_group_that_cannot_be_held_gives_its_slots_back():
    a, b = list(range(100, 300)), list(range(1000, 1300))
    prompts = [a + [1], a + [2], a[:64] + b + [3], a[:64] + b + [4]]
    for n in (1, 2, 3):
        be = Tree([[5]] * 4, n_slots=n, max_seq_len=1000)
        with pytest.raises(IndexError):
            run_generation(be, prompts, GenParams.greedy(1), share_prefix=True)
        assert sorted(be.free_slots) == list(range(n))


def test_captured_steps_of_groups_that_come_and_go_are_bounded():
    """Only the shapes used last keep a graph; steps without groups, and shapes in use, keep theirs."""
    from types import SimpleNamespace

    import torch

    from oracle_engine_b200.engine import step
    from oracle_engine_b200.engine.batch import shared_prefixes
    st = object.__new__(step.Stepper)
    st._graphs, st._prefix_graphs = {}, {}
    st.cache, st.rt = SimpleNamespace(groups=[0], max_pages_per_seq=4), SimpleNamespace(device=torch.device("cpu"))
    plain = st._decode_graph(64, 0, None)
    often = shared_prefixes([(1, 300)] * 16, 64)
    kept = st._decode_graph(64, 0, often)
    made = set()
    for bucket in (64, 96, 128):
        for n in (16, 32, 60):
            for pages in (64, 128, 1000):
                p = shared_prefixes([(1, pages)] * n, bucket)
                made.add((bucket, 3) + p.shape)
                st._decode_graph(bucket, 3, p)
                assert len(st._prefix_graphs) <= step.MAX_PREFIX_GRAPHS
                assert st._decode_graph(64, 0, often) is kept
    assert len(made) > step.MAX_PREFIX_GRAPHS and st._decode_graph(64, 0, None) is plain
    last = st._decode_graph(128, 3, shared_prefixes([(1, 1000)] * 60, 128))
    assert st._decode_graph(128, 3, shared_prefixes([(7, 400)] * 60, 128)) is last       # (no form distinguishes the two)


def test_which_models_read_common_pages_apart():
    import conftest
    import fuvipel_models as fm
    import torch

    from oracle_engine_b200.config.base import get_architecture
    from oracle_engine_b200.engine.runtime import Runtime
    from oracle_engine_b200.parts.model import DecoderModel

    def reads(raw, dtype=torch.bfloat16, tensor_cores=True):
        arch = get_architecture(raw.get("architecture") or raw["architectures"][0])
        rt = Runtime(dtype, torch.device("cpu"), tensor_cores)
        return DecoderModel(arch.build_spec(arch.config_cls.from_dict(raw), 256), rt).reads_common_pages()
    assert reads(conftest.TINY_E)
    assert not reads(conftest.TINY_E, torch.float32) and not reads(conftest.TINY_E, tensor_cores=False)
    assert not reads(conftest.TINY_B)                    # heads of another size
    assert not reads(fm.F1)
    odd = dict(conftest.TINY_E)
    arch = get_architecture(odd["architectures"][0])
    model = DecoderModel(arch.build_spec(arch.config_cls.from_dict(odd), 256), Runtime(torch.bfloat16, torch.device("cpu"), True))
    for e in model.schedule:
        model.layers[e.layer].mixer.scale = -0.125       # the kernels of common beginnings take positive scales
    assert not model.reads_common_pages()
