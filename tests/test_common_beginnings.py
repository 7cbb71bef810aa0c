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
