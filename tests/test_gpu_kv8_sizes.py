"""The 8-bit cache and common beginnings where numbers are large: caches of more than 2^32 bytes, many sequences, large groups."""
import pytest
import torch

from kv8_plain import Step, close

pytestmark = pytest.mark.gpu
TYPES = [torch.int8, torch.float8_e4m3fn]


def _far(s, n_pages):
    """The step over a cache of n_pages pages, its own pages at the end of it."""
    at = n_pages - s.n_pages
    tensors = s.cache if isinstance(s.cache, tuple) else (s.cache,)
    big = [torch.empty((n_pages,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in tensors]
    for b, t in zip(big, tensors):
        b[at:].copy_(t)
    s.tables = torch.where(s.tables >= 0, s.tables + at, s.tables)
    s.cache = tuple(big) if isinstance(s.cache, tuple) else big[0]
    return at


@pytest.mark.parametrize("dtype", [torch.bfloat16] + TYPES)
@pytest.mark.parametrize("kind", ["single", "prompt", "common"])
def test_pages_behind_the_first_4_gigabytes(dtype, kind):
    """The same bits as over a small cache."""
    if dtype == torch.bfloat16 and kind != "common":
        pytest.skip("the 16-bit cache's own kernels have tests of their own")
    args, kw = ([200, 140, 330], [80, 3, 1] if kind == "prompt" else [1] * 3, 16, 8, 128, dtype), {}
    if kind == "common":
        kw["prefixes"] = [(0, 2), (0, 2), None]
    run = lambda s: s.shared_out() if kind == "common" else s.out()          # noqa: E731
    near, far = Step(*args, seed=1, **kw), Step(*args, seed=1, **kw)
    want = run(near)
    pages = 2 ** 32 // (2 * 8 * 64 * 128 * (2 if dtype == torch.bfloat16 else 1)) + 1000
    at = _far(far, pages)
    assert torch.equal(run(far), want)
    for b, t in zip(far.cache if isinstance(far.cache, tuple) else (far.cache,), near.cache if isinstance(near.cache, tuple) else (near.cache,)):
        assert torch.equal(b[at:].contiguous().view(torch.uint8), t.view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,KVH", [(150, 4), (256, 2), (257, 2)])
def test_many_sequences_of_any_length(dtype, n, KVH):
    """More pairs of sequences and KV heads than there is room for at once: the longest go first, up to 256 of them."""
    from oracle_engine_b200.csrc import ops_kv8
    assert ops_kv8.many_pairs(n, KVH)
    starts = [(37 * i * i) % 190 for i in range(n)]
    s = Step(starts, [1] * n, 2 * KVH, KVH, 64, dtype, seed=2)
    want, tol, cache = s.truth()
    s.pad(3)
    got = s.out()
    close(got[:n], want, tol)
    assert (got[n:] == 7.0).all()
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", [torch.bfloat16] + TYPES)
@pytest.mark.parametrize("H,KVH", [(128, 1), (100, 1), (86, 2)])
def test_large_groups(dtype, H, KVH):
    """Up to 128 heads share a KV head: a tile of one token."""
    s = Step([130, 70, 200], [1] * 3, H, KVH, 64, dtype, seed=3, prefixes=[(0, 1)] * 3)
    want, tol, cache = s.truth()
    close(s.shared_out(), want, tol)
    s.check_cache(cache)
    if dtype != torch.bfloat16:
        for qlens in ([1, 1, 1], [20, 1, 3]):
            s = Step([130, 70, 200], qlens, H, KVH, 64, dtype, seed=4)
            want, tol, cache = s.truth()
            close(s.out(), want, tol)
            s.check_cache(cache)
