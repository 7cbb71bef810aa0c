"""Scales of the scores that the 8-bit cache's attention and that of common beginnings do not take (no GPU needed)."""
from types import SimpleNamespace

import pytest
import torch

from oracle_engine_b200.csrc import ops_kv8
from oracle_engine_b200.csrc.ops import KernelError
from test_kv8_cpu import entry


@pytest.mark.parametrize("scale", [0.0, 1e-9, -0.125, float("nan"), float("inf"), -float("inf")])
def test_scales_that_are_not_positive(scale):
    cache, i = entry(), torch.zeros(2, dtype=torch.int32)
    qkv, out = torch.zeros(1, 8 * 64, dtype=torch.bfloat16), torch.zeros(1, 4 * 64, dtype=torch.bfloat16)
    ctx = SimpleNamespace(n_seqs=1, max_qlen=1, max_kvlen=1, all_decode=True, context_class=0, cu_q=i, seq_start=i, seq_qlen=i, tok_seq=i, tok_pos=i)
    pre = SimpleNamespace(n_groups=0, n_members=0, max_pages=0, members=i, first=i, pages=i, seq_pages=i)
    tables = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(KernelError, match="scale must be a positive number"):
        ops_kv8.attention_kv8(out, qkv, None, None, cache, tables, ctx, 4, 2, 64, 0, scale)
    with pytest.raises(KernelError, match="scale must be a positive number"):
        ops_kv8.attention_shared(out, qkv, None, None, cache, tables, ctx, pre, 4, 2, 64, scale)
