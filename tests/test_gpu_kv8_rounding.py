"""Codes of the 8-bit cache are the nearest ones for every pair of a value and a largest magnitude, and turned keys are rounded once."""
import pytest
import torch

from kv8_plain import PAGE, Step, quantise, to_bf16, turn

pytestmark = pytest.mark.gpu


def written(kv, dtype, cos=None, sin=None):
    """kv [T, 2, KVH, hd] bfloat16 through kv8_write, token t at position t of one sequence: (codes, scales) [T, 2, KVH, hd]."""
    from oracle_engine_b200.csrc import ops_kv8
    T, _, KVH, hd = kv.shape
    pages = -(-T // PAGE)
    cache = (torch.zeros(pages, 2, KVH, PAGE, hd, dtype=dtype, device="cuda"), torch.zeros(pages, 2, KVH, PAGE, device="cuda"))
    qkv = torch.cat([torch.zeros(T, KVH * hd, dtype=torch.bfloat16, device="cuda"), kv.reshape(T, -1)], 1).contiguous()
    i32 = dict(dtype=torch.int32, device="cuda")
    ops_kv8.kv8_write(qkv, cos, sin, cache, torch.arange(pages, **i32)[None].contiguous(), torch.zeros(T, **i32), torch.arange(T, **i32),
                      KVH, KVH, hd)
    codes = cache[0].float().permute(0, 3, 1, 2, 4).reshape(-1, 2, KVH, hd)[:T]
    return codes.double(), cache[1].permute(0, 3, 1, 2).reshape(-1, 2, KVH)[:T]


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("exponent", [0, 126, -60, -108])
def test_every_quotient(dtype, exponent):
    """All 128 largest magnitudes of a binade against the values of that and the 16 binades below it (the lowest are still normal numbers)."""
    hd = 64
    largest = torch.arange(128, 256, dtype=torch.float64, device="cuda") * 2.0 ** (exponent - 7)
    values = [torch.arange(128, 256, dtype=torch.float64, device="cuda") * 2.0 ** (exponent - 7 - k) for k in range(17)]
    values = torch.cat(values + [v * -1 for v in values])
    values = torch.cat([values, values.new_zeros(-len(values) % (hd - 1))]).view(-1, hd - 1)      # rows of hd - 1
    rows = torch.cat([largest[:, None, None].expand(-1, values.shape[0], 1), values[None].expand(128, -1, -1)], -1)
    over = rows.abs() > rows[..., :1]
    rows = torch.where(over, rows / 2, rows).reshape(-1, hd)
    rows = torch.cat([rows, rows.new_zeros(-len(rows) % 8, hd)]).view(-1, 2, 4, hd)
    kv = rows.to(torch.bfloat16)
    assert torch.equal(kv.double(), rows)
    got, scales = written(kv, dtype)
    want, want_scales = quantise(rows, dtype)
    assert torch.equal(got, want)
    assert torch.equal(scales, want_scales.float())


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_turned_keys(dtype):
    """Millions of turned values, among them ones whose two products nearly cancel and ones on the border of two bfloat16."""
    T, KVH, hd = 8192, 4, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn(T, 2, KVH, hd, generator=g, device="cuda")
    ang = torch.rand(T, hd // 2, generator=g, device="cuda", dtype=torch.float64) * 6.3
    ang[: T // 4] = torch.randint(0, 9, (T // 4, hd // 2), generator=g, device="cuda").double() * (torch.pi / 4)
    cos, sin = ang.cos().float(), ang.sin().float()
    cos[T // 4: T // 2] = (torch.randint(-16, 17, (T // 4, hd // 2), generator=g, device="cuda") / 16).float()       # exact products: borders
    sin[T // 4: T // 2] = (torch.randint(-16, 17, (T // 4, hd // 2), generator=g, device="cuda") / 16).float()
    near = kv[T // 2: 3 * T // 4, 0]                       # lo / hi = tan(angle), nearly: the turned lower half cancels
    near[..., :hd // 2] = near[..., hd // 2:] * ang[T // 2: 3 * T // 4, None].tan().float().clamp(-50, 50)
    kv = kv.to(torch.bfloat16)
    rows = kv.double()
    rows[:, 0] = to_bf16(turn(rows[:, 0], cos.double()[:, None], sin.double()[:, None]))
    got, scales = written(kv, dtype, cos.contiguous(), sin.contiguous())
    want, want_scales = quantise(rows, dtype)
    assert torch.equal(scales, want_scales.float())
    assert torch.equal(got, want)
