"""The rules that choose forms of the 8-bit cache's kernels, at the ends of their range (no GPU needed)."""
import pytest

from oracle_engine_b200.csrc import ops_kv8


@pytest.mark.parametrize("n,kvh", [(1, 1), (1, 2), (2, 1), (3, 1), (1, 4), (1, 8), (2, 8), (1, 16), (18, 1)])
def test_ctas_that_leave_parts(n, kvh):
    """Few pairs of a sequence and a KV head: not more CTAs a pair than its keys have work for, as many as before where that was so."""
    warps, cluster, shares = ops_kv8.decode_form(n, kvh, 3, 0, 148)
    assert (warps, cluster) == (4, 1) and shares == min(2 * 148 // (n * kvh), 74)
