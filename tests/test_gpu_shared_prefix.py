"""Attention of sequences that begin with the same pages, against the definition in 64 bits."""
import pytest
import torch

from kv8_plain import Step, close

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KVH,hd", [(6, 2, 64), (24, 8, 128), (4, 4, 128), (32, 2, 64), (20, 1, 128)])
def test_one_group(H, KVH, hd, dtype):
    """Members that end right behind the prefix, inside the next page, and pages further."""
    s = Step([128, 129, 191, 192, 300, 128, 150], [1] * 7, H, KVH, hd, dtype, seed=1, prefixes=[(0, 2)] * 7)
    want, tol, cache = s.truth()
    close(s.shared_out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_groups_and_sequences_without_one(dtype):
    pre = [(0, 1), None, (1, 5), (0, 1), (2, 3), None, (1, 5), (1, 5), None]
    s = Step([64, 0, 400, 90, 192, 77, 320, 333, 511], [1] * 9, 8, 4, 128, dtype, seed=2, prefixes=pre, peaked=3.0)
    want, tol, cache = s.truth()
    close(s.shared_out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_members_and_a_long_prefix(dtype):
    n = 50
    s = Step([1280 + 3 * i for i in range(n)], [1] * n, 6, 2, 64, dtype, seed=3, prefixes=[(0, 20)] * n, peaked=2.0)
    want, tol, cache = s.truth()
    for ahead in (False, True):
        torch.cuda.synchronize()
        close(s.shared_out(ahead=ahead), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_rows_than_a_tile(dtype):
    """300 members of one head each, and a group of one member."""
    n = 300
    s = Step([64 + i % 7 for i in range(n)] + [200], [1] * (n + 1), 2, 2, 64, dtype, seed=4, prefixes=[(0, 1)] * n + [(1, 3)])
    want, tol, cache = s.truth()
    close(s.shared_out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_groups_and_with_bounds(dtype):
    """No group at all; and host numbers that are bounds: groups without members behind the real ones."""
    s = Step([0, 70, 150], [1] * 3, 8, 4, 64, dtype, seed=5)
    want, tol, cache = s.truth()
    close(s.shared_out(), want, tol)
    s = Step([64, 70, 150], [1] * 3, 8, 4, 64, dtype, seed=6, prefixes=[(0, 1), None, (0, 1)])
    s.prefix.n_groups, s.prefix.n_members, s.prefix.max_pages = 3, 3, 9
    s.prefix.first = torch.tensor([0, 2, 2, 2], dtype=torch.int32, device="cuda")
    s.prefix.pages = torch.tensor([1, 0, 0], dtype=torch.int32, device="cuda")
    want, tol, cache = s.truth()
    close(s.shared_out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tiles,splits,wide,cluster", [(1, 1, True, 1), (2, 1, False, 1), (2, 3, True, 2), (1, 7, False, 4), (2, 148, True, 8)])
@pytest.mark.parametrize("H,KVH,hd", [(6, 2, 64), (24, 8, 128)])
def test_forms(H, KVH, hd, tiles, splits, wide, cluster, dtype):
    n = 60
    s = Step([320 + i for i in range(n)] + [100, 0], [1] * (n + 2), H, KVH, hd, dtype, seed=11, peaked=2.0, prefixes=[(0, 5)] * n + [None] * 2)
    want, tol, cache = s.truth()
    warps = (12 if wide else 4) if dtype != torch.bfloat16 else (6 if wide else 3)
    close(s.shared_out(form=(tiles, splits, warps, cluster)), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_padding_rows_and_codes_that_are_no_numbers(dtype):
    s = Step([192, 200, 255, 80], [1] * 4, 6, 2, 64, dtype, seed=12, prefixes=[(0, 3)] * 3 + [None])
    if dtype == torch.float8_e4m3fn:
        s.spoil_codes()
    want, tol, cache = s.truth()
    s.pad(4)
    got = s.shared_out()
    close(got[:4], want, tol)
    assert (got[4:] == 7.0).all()
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_common_page_that_is_not_there(dtype):
    """It has no keys, whatever the cache's first page holds: as if read sequence by sequence."""
    got = []
    for spoilt in (False, True):
        s = Step([192, 200, 255], [1] * 3, 6, 2, 64, dtype, seed=13, prefixes=[(0, 3)] * 3)
        assert all(0 not in t for t in s.tables_list)
        s.tables[:, 1] = -1
        if spoilt and dtype == torch.float8_e4m3fn:
            s.spoil_codes()
        got.append(s.shared_out(form=(1, 2, 6 if dtype == torch.bfloat16 else 12, 1)))
    assert torch.equal(*got) and torch.isfinite(got[0].float()).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ahead", [False, True])
def test_tokens_one_after_the_other(dtype, ahead):
    """Every call reads what the call before wrote, with nothing between them; with ahead, another kernel."""
    n, H, KVH, hd = 40, 6, 2, 64
    s = Step([150 + n, 128 + n, 191 + n, 40 + n], [1] * 4, H, KVH, hd, dtype, seed=14, prefixes=[(0, 2)] * 3 + [None])
    first = [x - n for x in s.starts]
    g = torch.Generator().manual_seed(1)
    rows = torch.randn(n, *s.qkv.shape, generator=g).to(torch.bfloat16).cuda()
    starts = torch.tensor([[x + i for x in first] for i in range(n)], dtype=torch.int32, device="cuda")
    outs = []
    torch.cuda.synchronize()
    for i in range(n):
        s.qkv, s.ctx.seq_start = rows[i].clone() if ahead else rows[i], starts[i]
        outs.append(s.shared_out(ahead=ahead))
    for i in range(n):
        s.qkv, s.starts = rows[i], [x + i for x in first]
        want, tol, cache = s.truth()
        close(outs[i], want, tol)
        if dtype == torch.bfloat16:
            s.rows64 = cache
        else:
            s.codes64, s.scales64 = cache
            s.rows64 = s.codes64 * s.scales64[..., None]


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_only(dtype):
    s = Step([128, 140], [1, 1], 8, 4, 64, dtype, seed=7, prefixes=[(0, 2)] * 2, has_kv=False)
    want, tol, cache = s.truth()
    close(s.shared_out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_as_without_sharing(dtype):
    """The same step through the attention that reads every sequence's pages by themselves."""
    if dtype == torch.bfloat16:
        pytest.skip("the 16-bit cache's own kernels have tests of their own")
    args = ([640, 700, 655], [1] * 3, 24, 8, 128, dtype)
    one, two = Step(*args, seed=8, prefixes=[(0, 10)] * 3), Step(*args, seed=8, prefixes=[(0, 10)] * 3)
    want, tol, _ = one.truth()
    close(one.shared_out(), want, tol)
    close(two.out(), want, tol)
    assert torch.equal(one.cache[0].view(torch.uint8), two.cache[0].view(torch.uint8))


@pytest.mark.parametrize("dtype", TYPES)
def test_graph_and_another_stream(dtype):
    s = Step([256 + i for i in range(5)], [1] * 5, 6, 2, 64, dtype, seed=9, prefixes=[(0, 4)] * 5)
    want, tol, _ = s.truth()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.shared_out()
    torch.cuda.current_stream().wait_stream(side)
    close(got, want, tol)
    graphs = []
    for _ in range(2):                              # two graphs that are alive at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = s.shared_out()
        graphs.append((g, o))
    for _ in range(3):
        for g, o in graphs:
            o.zero_()
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, got) for _, o in graphs)


def test_refusals_on_the_device():
    from oracle_engine_b200.csrc.ops import KernelError
    for spoil in (lambda s: setattr(s.prefix, "members", s.prefix.members[:1]), lambda s: setattr(s.prefix, "first", s.prefix.first.long()),
                  lambda s: setattr(s.prefix, "seq_pages", s.prefix.seq_pages[:1]), lambda s: setattr(s.ctx, "all_decode", False),
                  lambda s: setattr(s, "cache", s.cache.float()), lambda s: setattr(s, "cache", s.cache[:, :1])):
        s = Step([64, 64], [1, 1], 4, 2, 64, torch.bfloat16, seed=10, prefixes=[(0, 1)] * 2)
        spoil(s)
        with pytest.raises(KernelError):
            s.shared_out()
