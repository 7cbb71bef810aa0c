"""Steps whose numbers on the device leave what the tables hold: nothing is read or written there, and the other rows are as ever."""
import pytest
import torch

from kv8_plain import Step, close

pytestmark = pytest.mark.gpu
TYPES = [torch.int8, torch.float8_e4m3fn]


def _cut(s, positions, host):
    """Angles for the first positions only; host: what the step says of its longest sequence (None: nothing)."""
    s.cos, s.sin = s.cos[:positions].contiguous(), s.sin[:positions].contiguous()
    if host is None:
        del s.ctx.max_kvlen
    else:
        s.ctx.max_kvlen = host


def _untouched(s, before, places):
    """The cache's rows of (sequence, position) places are what they were."""
    for b, pos in places:
        for now, was in zip(s.cache if isinstance(s.cache, tuple) else (s.cache,), before):
            page = s.tables_list[b][pos // 64]
            assert torch.equal(now[page, :, :, pos % 64].contiguous().view(torch.uint8), was[page, :, :, pos % 64].contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("host", [None, 1])
@pytest.mark.parametrize("form", [None, (4, 2, 1), (4, 1, 3)])
def test_single_tokens_without_an_angle(dtype, host, form):
    s = Step([150, 20, 99, 100], [1] * 4, 6, 2, 64, dtype, seed=1)
    want, tol, _ = s.truth()
    _cut(s, 100, host)
    before = [t.clone() for t in s.cache]
    got = s.out(form=form)
    assert torch.isnan(got[[0, 3]]).all()
    close(got[1:3], want[1:3], tol[1:3])
    _untouched(s, before, [(0, 150), (3, 100)])
    assert not torch.isnan(s.cache[1][s.tables_list[1][0], :, :, 20]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("qlens,form", [([70, 3, 90], (1, 1)), ([70, 3, 90], (2, 1)), ([70, 3, 90], (2, 3)), ([2, 1, 2], None)])
def test_prompts_without_angles(dtype, qlens, form):
    s = Step([60, 98, 0], qlens, 6, 2, 64, dtype, seed=2)
    want, tol, _ = s.truth()
    _cut(s, 100, None)
    before = [t.clone() for t in s.cache]
    got = s.out(form=form)
    where = [(b, p) for b, (a, q) in enumerate(zip(s.starts, qlens)) for p in range(a, a + q)]
    there = torch.tensor([p < 100 for _, p in where])
    assert torch.isnan(got.cpu()[~there]).all()
    close(got.cpu()[there], want[there], tol[there])
    _untouched(s, before, [w for w in where if w[1] >= 100])


@pytest.mark.parametrize("dtype", [torch.bfloat16] + TYPES)
def test_common_beginnings_without_an_angle(dtype):
    s = Step([128, 200, 150, 64], [1] * 4, 6, 2, 64, dtype, seed=3, prefixes=[(0, 2)] * 3 + [None])
    want, tol, _ = s.truth()
    _cut(s, 180, 1)
    before = [t.clone() for t in (s.cache if isinstance(s.cache, tuple) else (s.cache,))]
    got = s.shared_out()
    assert torch.isnan(got[1]).all()
    close(got[[0, 2, 3]], want[[0, 2, 3]], tol[[0, 2, 3]])
    _untouched(s, before, [(1, 200)])


@pytest.mark.parametrize("dtype", [torch.bfloat16] + TYPES)
@pytest.mark.parametrize("number", [5, -1, 2 ** 31 - 1])
def test_members_that_are_no_sequences(dtype, number):
    """Its group's results are undefined then; the others' are not."""
    s = Step([128, 200, 150, 64, 90, 64], [1] * 6, 6, 2, 64, dtype, seed=4, prefixes=[(0, 2), (0, 2), (0, 2), (1, 1), (1, 1), None])
    want, tol, cache = s.truth()
    for at in (0, 1):
        s.prefix.members[0:3] = torch.tensor([0, 1, 2])
        s.prefix.members[at] = number if number != 5 else 6
        got = s.shared_out()
        close(got[3:], want[3:], tol[3:])
        s.check_cache(cache)


def test_refusals():
    from oracle_engine_b200.csrc.ops import KernelError
    s = Step([10], [1], 4, 2, 64, torch.int8, seed=5)
    _cut(s, 0, 0)
    with pytest.raises(KernelError):
        s.out()
