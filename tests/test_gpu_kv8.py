"""The 8-bit cache: what is written, and attention over it, against the definitions in 64 bits."""
import math

import pytest
import torch

from kv8_plain import PAGE, Step, close, quantise

pytestmark = pytest.mark.gpu
TYPES = [torch.int8, torch.float8_e4m3fn]
HEADS = [(6, 2, 64), (24, 8, 128), (4, 4, 128), (32, 2, 64), (20, 1, 128)]     # the last two: 16 and 20 heads share a KV head


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KVH,hd", HEADS[:3])
def test_write(H, KVH, hd, dtype):
    from oracle_engine_b200.csrc import ops_kv8
    s = Step([0, 63, 64, 1, 200], [1, 2, 65, 130, 7], H, KVH, hd, dtype, seed=1)
    before = s.qkv.clone()
    ops_kv8.kv8_write(s.qkv, s.cos, s.sin, s.cache, s.tables, s.ctx.tok_seq, s.ctx.tok_pos, H, KVH, hd)
    _, _, want = s.truth()
    s.check_cache(want)
    assert torch.equal(s.qkv, before)


@pytest.mark.parametrize("dtype", TYPES)
def test_write_of_unusual_rows(dtype):
    """Rows of zeros, of one value, of the largest and smallest magnitudes, on the borders between codes, infinite and undefined."""
    from oracle_engine_b200.csrc import ops_kv8
    H, KVH, hd = 2, 2, 64
    s = Step([5], [12], H, KVH, hd, dtype, seed=2, rotate=False)
    kv = s.qkv.view(12, H + 2 * KVH, hd)
    g = torch.Generator().manual_seed(3)
    kv[0] = 0
    kv[1] = 0
    kv[1, :, 3] = -2.5
    kv[2] *= 2.0 ** 126
    kv[2, :, 0] = torch.finfo(torch.bfloat16).max
    kv[3] *= 2.0 ** -120
    kv[4, :, 0] = 254.0                       # quotients on the border: x / 2
    kv[4, :, 1:] = torch.randint(-254, 255, (hd - 1,), generator=g).to(torch.bfloat16).cuda()
    kv[5, :, 0] = 448.0 * 2                   # borders of e4m3, among them those of its smallest codes
    kv[5, :, 1:] = (torch.randint(-255, 256, (hd - 1,), generator=g) * 2.0 ** torch.randint(-14, 2, (hd - 1,), generator=g)).to(torch.bfloat16).cuda()
    kv[6, :, 7] = math.inf
    kv[7, :, 8] = math.nan
    kv[8, :, 9] = -math.inf
    kv[9, :, :] = kv[9, :, :1]
    kv[10, :, 0] = -0.0
    want = quantise(kv[:, H:].reshape(12, 2, KVH, hd).cpu().double(), dtype)
    ops_kv8.kv8_write(s.qkv, None, None, s.cache, s.tables, s.ctx.tok_seq, s.ctx.tok_pos, H, KVH, hd)
    page = s.tables_list[0][0]
    codes, scales = s.cache[0].float()[page, :, :, 5:17].cpu().double(), s.cache[1][page, :, :, 5:17].cpu()
    assert torch.equal(codes, want[0].permute(1, 2, 0, 3))
    exp = want[1].permute(1, 2, 0).float()
    assert torch.equal(torch.isnan(scales), torch.isnan(exp))
    assert torch.equal(scales.nan_to_num(-1), exp.nan_to_num(-1))
    assert torch.isnan(scales[:, :, 6:9]).all() and not torch.isnan(scales[:, :, 9:]).any()


def test_write_leaves_padding_and_unmapped_pages_alone():
    from oracle_engine_b200.csrc import ops_kv8
    s = Step([0, 70], [4, 4], 4, 2, 64, torch.int8, seed=4)
    s.ctx.tok_seq[1] = -1
    s.tables[1, 1] = -1                       # sequence 1's page of positions 64..127
    s.tables[0, 0] = s.n_pages                # a number outside the cache
    codes, scales = s.cache[0].clone(), s.cache[1].clone()
    ops_kv8.kv8_write(s.qkv, s.cos, s.sin, s.cache, s.tables, s.ctx.tok_seq, s.ctx.tok_pos, 4, 2, 64)
    assert torch.equal(codes, s.cache[0]) and torch.equal(scales.nan_to_num(-1), s.cache[1].nan_to_num(-1))


def test_write_leaves_places_that_are_not_there_alone():
    """A sequence behind the page tables, a position behind the angles or before the first: the other tokens are written."""
    from oracle_engine_b200.csrc import ops_kv8
    s = Step([0], [6], 4, 2, 64, torch.int8, seed=3)
    s.ctx.tok_seq[1], s.ctx.tok_pos[2], s.ctx.tok_pos[3] = 1, 1000, -5
    ops_kv8.kv8_write(s.qkv, s.cos, s.sin, s.cache, s.tables, s.ctx.tok_seq, s.ctx.tok_pos, 4, 2, 64)
    page = s.tables_list[0][0]
    written = ~torch.isnan(s.cache[1]).cpu()
    assert written[page, :, :, [0, 4, 5]].all() and written.sum() == 3 * 2 * 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("window", [0, 1, 50, 64, -64, -100])
def test_single_tokens(H, KVH, hd, dtype, window):
    s = Step([0, 1, 31, 32, 63, 64, 65, 127, 128, 200, 333], [1] * 11, H, KVH, hd, dtype, seed=5 + window, window=window)
    want, tol, cache = s.truth()
    close(s.out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", [(4, 1, 1), (12, 1, 1), (4, 2, 1), (12, 4, 1), (4, 8, 1), (12, 8, 1), (4, 1, 7), (12, 1, 40)])
def test_single_tokens_of_long_sequences(dtype, form):
    s = Step([0, 3000, 1279, 2111], [1] * 4, 6, 2, 128, dtype, seed=6, peaked=3.0)
    want, tol, cache = s.truth()
    for ahead in (False, True):
        torch.cuda.synchronize()
        close(s.out(form=form, ahead=ahead), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,KVH,hd", HEADS)
@pytest.mark.parametrize("window", [0, 40, -64])
def test_prompts(H, KVH, hd, dtype, window):
    s = Step([0, 0, 5, 64, 130], [1, 97, 64, 3, 33], H, KVH, hd, dtype, seed=7 + window, window=window, pad_seqs=2)
    want, tol, cache = s.truth()
    close(s.out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_long_prompt(dtype):
    s = Step([0, 700], [400, 150], 6, 2, 128, dtype, seed=8, peaked=3.0)
    want, tol, cache = s.truth()
    close(s.out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("qlens", [[1, 1, 1], [3, 1, 70]])
def test_rows_of_another_layer_s_cache(dtype, qlens):
    """Queries only: the keys are in the cache already."""
    s = Step([0, 65, 130], qlens, 8, 4, 64, dtype, seed=9, has_kv=False)
    want, tol, cache = s.truth()
    close(s.out(), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_of_very_different_size(dtype):
    """Values that grow by 2^100 along a sequence, and shrink again: what O is relative to has to follow."""
    s = Step([300], [1], 2, 1, 64, dtype, seed=10)
    codes, scales = s.cache
    f = torch.exp2(100.0 * torch.sin(torch.arange(300) / 40.0)).float()
    for p in range(300):
        page = s.tables_list[0][p // PAGE]
        s.scales64[page, 1, :, p % PAGE] *= f[p].double()
        s.scales64 = s.scales64.float().double()
        s.rows64[page, 1, :, p % PAGE] = s.codes64[page, 1, :, p % PAGE] * s.scales64[page, 1, :, p % PAGE][..., None]
        scales[page, 1, :, p % PAGE] = s.scales64[page, 1, :, p % PAGE].float().cuda()
    want, tol, _ = s.truth()
    close(s.out(), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_of_any_size(dtype):
    """Rows of queries from 2^-60 to 2^60 of each other's size, and one of zeros (equal weights)."""
    s = Step([90, 90, 90, 90], [1] * 4, 4, 2, 64, dtype, seed=11)
    for b, f in enumerate([2.0 ** -60, 2.0 ** 4, 0.0, 2.0 ** -8]):
        s.qkv[b, :4 * 64] *= f
    want, tol, _ = s.truth()
    close(s.out(), want, tol)


@pytest.mark.parametrize("dtype", TYPES)
def test_undefined_rows_show_only_where_they_are_seen(dtype):
    s = Step([100, 100], [1, 1], 4, 2, 64, dtype, seed=12, window=32)
    s.cache[1][s.tables_list[0][0], :, :, 10] = math.nan           # outside sequence 0's window
    s.cache[1][s.tables_list[1][1], 1, 0, 90 - 64] = math.nan      # a value of sequence 1's KV head 0, inside
    want, tol, _ = s.truth()
    got = s.out()
    close(got[0], want[0], tol[0])
    assert torch.isnan(got[1, :2 * 64]).all()
    close(got[1, 2 * 64:], want[1, 2 * 64:], tol[1, 2 * 64:])


@pytest.mark.parametrize("starts,qlens,window,forms", [
    ([100, 0, 63, 700], [1] * 4, 0, [(4, 1, 1), (12, 2, 1), (4, 1, 5)]), ([100, 200, 65], [1] * 3, 40, [None]),
    ([30, 0], [2, 1], 0, [None]), ([0, 70, 300], [90, 3, 33], 0, [(1, 1), (2, 1), (2, 3)]), ([300], [100], 50, [None, (2, 2)])])
def test_codes_behind_the_last_token_that_are_no_numbers(starts, qlens, window, forms):
    for form in forms:
        s = Step(starts, qlens, 6, 2, 64, torch.float8_e4m3fn, seed=19, window=window)
        s.spoil_codes()
        want, tol, cache = s.truth()
        close(s.out(form=form), want, tol)
        s.check_cache(cache)


@pytest.mark.parametrize("qlens", [[1], [60]])
def test_a_page_that_is_not_there_has_no_codes(qlens):
    """Whatever the cache's first page holds."""
    got = []
    for spoilt in (False, True):
        s = Step([200], qlens, 4, 2, 64, torch.float8_e4m3fn, seed=21)
        assert 0 not in s.tables_list[0]
        s.tables[0, 1] = -1
        if spoilt:
            s.spoil_codes()
        got.append(s.out())
    assert torch.equal(*got) and torch.isfinite(got[0].float()).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", [(1, 1), (2, 1), (1, 3), (2, 4), (2, 16)])
@pytest.mark.parametrize("H,KVH,hd,window", [(6, 2, 128, 0), (10, 2, 64, 0), (4, 4, 64, 100), (6, 2, 64, -128)])
def test_forms_of_prompts(H, KVH, hd, window, form, dtype):
    s = Step([0, 600, 129, 64], [300, 70, 1, 129], H, KVH, hd, dtype, seed=21, window=window, peaked=2.0, pad_seqs=1)
    want, tol, cache = s.truth()
    close(s.out(form=form), want, tol)
    s.check_cache(cache)


@pytest.mark.parametrize("starts,qlens,form", [([70, 0, 900], [1] * 3, (4, 1, 1)), ([70, 0, 900], [1] * 3, (12, 4, 1)),
                                               ([70, 0, 900], [1] * 3, (4, 1, 7)), ([0, 100], [80, 50], (2, 1)), ([0, 100], [80, 50], (1, 3))])
def test_padding_rows_are_left_alone(starts, qlens, form):
    s = Step(starts, qlens, 6, 2, 64, torch.int8, seed=22)
    want, tol, cache = s.truth()
    n = s.qkv.shape[0]
    s.pad(5)
    got = s.out(form=form)
    close(got[:n], want, tol)
    assert (got[n:] == 7.0).all()
    s.check_cache(cache)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [0, 60])
@pytest.mark.parametrize("form", [(2, 1), (1, 2)])
def test_undefined_keys_and_values_of_a_prompt(dtype, window, form):
    """Tokens before an undefined one, and those whose window it has left, do not see it."""
    for which, value in ((1, math.inf), (2, math.nan)):
        s = Step([40], [200], 4, 1, 64, dtype, seed=23, window=window)
        sees = torch.zeros(200, dtype=torch.bool)
        for at in (77, 150):
            s.qkv[at, 4 * 64 + (which - 1) * 64 + 5] = value
            sees[at:at + window if window else None] = True
        want, tol, _ = s.truth()
        got = s.out(form=form).cpu()
        assert torch.isnan(got[sees]).all()
        close(got[~sees], want[~sees], tol[~sees])


def test_strided_rows_no_rotation_another_stream_and_a_graph():
    s = Step([70, 0, 200], [1, 1, 1], 6, 2, 64, torch.int8, seed=13, rotate=False, stride_pad=24)
    want, tol, cache = s.truth()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s.out()
    torch.cuda.current_stream().wait_stream(side)
    close(got, want, tol)
    s.check_cache(cache)
    first = got.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = s.out()
    for _ in range(3):
        captured.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, first)


def test_the_same_bits_every_time():
    s = Step([3000, 17, 900], [1, 1, 1], 24, 8, 128, torch.float8_e4m3fn, seed=14)
    got = [s.out(form=(12, 4, 1)) for _ in range(4)]
    assert all(torch.equal(got[0], o) for o in got)


def test_a_sequence_token_by_token():
    """Every call reads what the call before wrote, with nothing between them."""
    from oracle_engine_b200.csrc import ops_kv8
    n, H, KVH, hd = 150, 4, 2, 64
    whole = Step([0], [n], H, KVH, hd, torch.int8, seed=15)
    want, tol, cache = whole.truth()
    outs = []
    for p in range(n):
        one = Step([p], [1], H, KVH, hd, torch.int8, seed=16)
        one.qkv, one.cache, one.cos, one.sin = whole.qkv[p:p + 1], whole.cache, whole.cos, whole.sin
        one.tables = whole.tables
        outs.append(one.out())
    close(torch.cat(outs), want, tol)
    whole.check_cache(cache)


def test_pages_outside_the_cache_have_no_keys():
    s = Step([200], [1], 4, 2, 64, torch.int8, seed=17)
    page = s.tables_list[0][1]
    s.tables[0, 1] = -1
    want = s.out()
    s.tables[0, 1] = s.n_pages + 5
    assert torch.equal(s.out(), want) and torch.isfinite(want.float()).all()
    s.tables[0, 1] = page
    assert not torch.equal(s.out(), want)


def test_refusals_on_the_device():
    from oracle_engine_b200.csrc import ops_kv8
    from oracle_engine_b200.csrc.ops import KernelError
    s = Step([10], [1], 4, 2, 64, torch.int8, seed=18)
    bad = [lambda: setattr(s, "qkv", s.qkv.float()), lambda: setattr(s, "qkv", s.qkv[:, :-64]),
           lambda: setattr(s.ctx, "max_kvlen", 100000), lambda: setattr(s.ctx, "cu_q", s.ctx.cu_q.long()),
           lambda: setattr(s, "cos", s.cos.double()), lambda: setattr(s, "sin", None),
           lambda: setattr(s, "cache", (s.cache[0].cpu(), s.cache[1])), lambda: setattr(s, "tables", s.tables[:0])]
    for spoil in bad:
        s = Step([10], [1], 4, 2, 64, torch.int8, seed=18)
        spoil()
        with pytest.raises(KernelError):
            s.out()
    s = Step([10], [1], 4, 2, 64, torch.int8, seed=18)
    for form in ((4, 0, 1), (4, 3, 1), (12, 32, 1), (5, 1, 1), (4, 2, 2), (4, 1, 0)):
        with pytest.raises(KernelError):
            s.out(form=form)
    with pytest.raises(KernelError):
        ops_kv8.kv8_write(s.qkv, s.cos, s.sin, s.cache, s.tables, s.ctx.tok_seq[:0], s.ctx.tok_pos, 4, 2, 64)
