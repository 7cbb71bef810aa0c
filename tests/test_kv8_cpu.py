"""The 8-bit cache's entry points refuse what their kernels do not take, before anything is launched (no GPU needed)."""
from types import SimpleNamespace

import pytest
import torch

from kv8_plain import PAGE, quantise, to_bf16
from oracle_engine_b200.csrc import ops_kv8
from oracle_engine_b200.csrc.ops import KernelError


def entry(pages=2, KVH=2, hd=64, dtype=torch.int8):
    return torch.zeros(pages, 2, KVH, PAGE, hd, dtype=dtype), torch.zeros(pages, 2, KVH, PAGE)


def call(name, cache, H=4, KVH=2, hd=64, all_decode=True):
    qkv = torch.zeros(1, (H + 2 * KVH) * hd, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    ctx = SimpleNamespace(n_seqs=1, max_qlen=1, max_kvlen=1, all_decode=all_decode, context_class=0, cu_q=i, seq_start=i, seq_qlen=i,
                          tok_seq=i, tok_pos=i)
    tables = torch.zeros(1, 2, dtype=torch.int32)
    if name == "write":
        ops_kv8.kv8_write(qkv, None, None, cache, tables, i, i, H, KVH, hd)
    elif name == "attention":
        ops_kv8.attention_kv8(torch.zeros(1, H * hd), qkv, None, None, cache, tables, ctx, H, KVH, hd, 0, 1.0)
    else:
        pre = SimpleNamespace(n_groups=0, n_members=0, max_pages=0, members=i, first=i, pages=i, seq_pages=i)
        ops_kv8.attention_shared(torch.zeros(1, H * hd), qkv, None, None, cache, tables, ctx, pre, H, KVH, hd, 1.0)


CALLS = ["write", "attention", "shared"]


@pytest.mark.parametrize("name", CALLS)
def test_head_sizes_and_groups(name):
    for H, KVH, hd in ((4, 2, 96), (4, 2, 32), (5, 2, 64), (1, 2, 64)):
        with pytest.raises(KernelError, match="outside what the kernels take"):
            call(name, entry(KVH=KVH, hd=hd), H, KVH, hd)


@pytest.mark.parametrize("name", CALLS)
def test_caches_that_do_not_fit(name):
    codes, scales = entry()
    for bad in ((codes.float(), scales), (codes, None), (codes.to(torch.uint8), scales), (codes, scales.double()),
                (codes, scales[:1]), (codes[:, :1], scales[:, :1]), (codes.transpose(0, 1), scales),
                torch.zeros(2, 2, 2, PAGE, 64)):
        with pytest.raises(KernelError):
            call(name, bad)
    if name != "shared":
        with pytest.raises(KernelError, match="codes and scales expected"):
            call(name, torch.zeros(2, 2, 2, PAGE, 64, dtype=torch.bfloat16))


@pytest.mark.parametrize("name", CALLS)
def test_tensors_on_the_host(name):
    for dtype in (torch.int8, torch.float8_e4m3fn):
        with pytest.raises(KernelError, match="CUDA tensors"):
            call(name, entry(dtype=dtype))


def test_split_and_cluster_rules():
    for n in (1, 2, 7, 64, 500):
        for kvh in (1, 2, 8):
            for cls in range(4):
                warps, c, shares = ops_kv8.decode_form(n, kvh, cls, 0, 148)
                assert warps in (4, 12) and c in (1, 2, 4, 8) and shares >= 1 and (c == 1 or shares == 1)
                assert c * shares == 1 or n * kvh * c * shares * warps <= 12 * 148
                assert ops_kv8.decode_form(n, kvh, cls, 100, 148)[1:] == (1, 1)
            for pages in (1, 5, 500):
                for eight in (False, True):
                    mt, splits, warps, c = ops_kv8.shared_form(n, n, 1, 4, kvh, pages, eight, 148)
                    assert mt in (1, 2) and 1 <= splits <= min(pages, ops_kv8.MAX_SPLITS) and c in (1, 2)
                    assert warps in ((4, 12) if eight else (3, 6))
            for tokens in (1, 40, 5000):
                mt, splits = ops_kv8.prompt_form(tokens, n, 4, kvh, cls, 0, 148)
                assert mt in (1, 2) and 1 <= splits <= 16


def test_the_plain_rounding():
    """What the GPU tests compare with: one rounding to bfloat16, codes to the nearest with ties to even."""
    x = torch.tensor([1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -8, 1.0 + 2.0 ** -8 + 2.0 ** -40, -3.0, 0.0], dtype=torch.float64)
    assert to_bf16(x).tolist() == [1.0, 1.0 + 2.0 ** -6, 1.0 + 2.0 ** -7, -3.0, 0.0]
    row = torch.tensor([[254.0, 1.0, 3.0, -5.0, 0.0]], dtype=torch.float64)
    codes, scale = quantise(row, torch.int8)
    assert codes.tolist() == [[127.0, 0.0, 2.0, -2.0, 0.0]] and scale.item() == 2.0
    for v in (448.0, 1.0625, 2.0 ** -9, 3 * 2.0 ** -10, 0.3):
        row = torch.tensor([[448.0, v]], dtype=torch.float64)
        assert quantise(row, torch.float8_e4m3fn)[0][0, 1].item() == torch.tensor(v).to(torch.float8_e4m3fn).float().item()
