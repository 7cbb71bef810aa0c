"""Pages that are not in the cache, against the definition in 64 bits without their keys."""
import pytest
import torch

from kv8_plain import PAGE, Step, close

pytestmark = pytest.mark.gpu
TYPES = [torch.int8, torch.float8_e4m3fn]


def _without(s, missing):
    """What has to come out, and how far off it may be (kv8_plain.py: Step.truth), if page `missing` of every sequence has no keys."""
    H, KVH, hd, scale = s.H, s.KVH, s.hd, s.hd ** -0.5
    G, eight = H // KVH, s.dtype != torch.bfloat16
    _, _, cache = s.truth()
    rows = cache[0] * cache[1][..., None] if eight else cache
    heads = s.qkv.cpu().double().reshape(s.qkv.shape[0], -1, hd)
    cos, sin = s.cos.cpu().double(), s.sin.cpu().double()
    outs, tols, t = [], [], 0
    for b, (start, q) in enumerate(zip(s.starts, s.qlens)):
        for pos in range(start, start + q):
            there = torch.tensor([p for p in range(pos + 1) if p // PAGE != missing])
            pages = torch.tensor(s.tables_list[b])[there // PAGE]
            kv = rows[pages, :, :, there % PAGE].permute(1, 2, 0, 3)                       # [2, KVH, keys, hd]
            x = heads[t, :H]
            lo, hi, c, n = x[:, :hd // 2], x[:, hd // 2:], cos[pos], sin[pos]
            qh = torch.cat([lo * c - hi * n, lo * n + hi * c], -1).view(KVH, G, hd)
            p = torch.softmax(torch.einsum("kgd,knd->kgn", qh, kv[0]) * scale, -1)
            out = torch.einsum("kgn,knd->kgd", p, kv[1])
            size = (torch.einsum("kgd,knd->kgn", qh.abs(), kv[0].abs()) * scale).amax(-1)
            r = 2.0 ** -12 if eight else 2.0 ** -16
            off = 2 * ((r + 2.0 ** -17) * size + r + 2.0 ** -17)
            tol = 2.0 ** -8 * out.abs() + off[..., None] * 1.02 * torch.einsum("kgn,knd->kgd", p, kv[1].abs()) + 1e-30
            if eight:
                tol = tol + (2.0 ** -32 * cache[1][pages, 1, :, there % PAGE].amax(0)[:, None] * cache[0][pages, 1, :, there % PAGE].abs().sum(0))[:, None]
            outs.append(out.reshape(-1))
            tols.append(tol.reshape(-1))
            t += 1
    return torch.stack(outs), torch.stack(tols)


@pytest.mark.parametrize("dtype", [torch.bfloat16] + TYPES)
@pytest.mark.parametrize("missing", [0, 1, 2])
@pytest.mark.parametrize("form", [None, (1, 1), (1, 3), (2, 2)])
def test_common_pages(dtype, missing, form):
    """The group's first, second or last common page."""
    s = Step([192, 200, 255, 70], [1] * 4, 6, 2, 64, dtype, seed=13, prefixes=[(0, 3)] * 3 + [None])
    s.tables[:3, missing] = -1 if missing else s.n_pages
    got = s.shared_out(form=None if form is None else form + (6 if dtype == torch.bfloat16 else 12, 1))
    want, tol = _without(s, missing)
    close(got[:3], want[:3], tol[:3])
    want, tol, _ = s.truth()
    close(got[3:], want[3:], tol[3:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("missing", [0, 1])
@pytest.mark.parametrize("qlens,form", [([1, 1], None), ([1, 1], (4, 2, 1)), ([1, 1], (4, 1, 3)), ([2, 1], None), ([60, 70], (1, 1)), ([60, 70], (2, 1)),
                                        ([60, 70], (1, 2))])
def test_pages_of_a_sequence(dtype, missing, qlens, form):
    s = Step([200, 140], qlens, 6, 2, 64, dtype, seed=14)
    s.tables[:, missing] = -1
    got = s.out(form=form)
    close(got, *_without(s, missing))
