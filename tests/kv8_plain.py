"""The 8-bit cache and attention over it from their definitions, in 64 bits, and random steps to run them on."""
import math
import random
from types import SimpleNamespace

import torch

PAGE = 64
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def nearest(x, step):
    """x to a multiple of step, ties to the even one (float64)."""
    return torch.round(x / step) * step


def to_bf16(x):
    """float64 values rounded once to 8 significant bits (as float64)."""
    _, e = torch.frexp(x)
    return torch.ldexp(torch.round(torch.ldexp(x, 8 - e)), e - 8)


def turn(x, cos, sin):
    """x [..., hd] float64 turned by its position's cos and sin [..., hd/2]."""
    half = x.shape[-1] // 2
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)


def quantise(rows, dtype):
    """(codes, scales) of rows [..., hd] float64 whose values a bfloat16 holds: both float64."""
    c = LARGEST[dtype]
    a = rows.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(rows).all(-1, keepdim=True)
    x = torch.where(bad, torch.zeros_like(rows), rows * c / torch.where(a > 0, a, torch.ones_like(a)))
    if dtype == torch.int8:
        code = nearest(x, torch.ones_like(x))
    else:
        code = nearest(x, torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3))
    scale = torch.where(bad, torch.full_like(a, math.nan), a / c)
    return code, scale.float().double()[..., 0]


class Step:
    """A random step: `starts` cached tokens and `qlens` new ones per sequence, over pages in random order.  prefixes: per sequence
    (group, pages) or None.  Rows of the cache that no token has yet hold what would spoil a result that reads them."""

    def __init__(self, starts, qlens, H, KVH, hd, dtype, seed=0, prefixes=None, window=0, pad_seqs=0, rotate=True, has_kv=True,
                 peaked=1.0, extra_pages=3, stride_pad=0):
        r = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.H, self.KVH, self.hd, self.dtype, self.window, self.has_kv = H, KVH, hd, dtype, window, has_kv
        self.starts, self.qlens = list(starts), list(qlens)
        B = len(starts)
        self.prefixes = prefixes or [None] * B
        for b, p in enumerate(self.prefixes):
            assert p is None or p[1] * PAGE <= starts[b]
        n = sum(-(-(s + q) // PAGE) for s, q in zip(starts, qlens)) + extra_pages
        free = list(range(n))
        r.shuffle(free)
        common, self.tables_list = {}, []
        for b in range(B):
            need, row = -(-(starts[b] + qlens[b]) // PAGE), []
            if self.prefixes[b] is not None:
                k, pages = self.prefixes[b]
                row = list(common.setdefault(k, [free.pop() for _ in range(pages)]) if k not in common else common[k])
                assert len(row) == pages
            self.tables_list.append(row + [free.pop() for _ in range(need - len(row))])
        width = max(len(t) for t in self.tables_list) + 1
        self.n_pages = n
        rows = torch.randn(n, 2, KVH, PAGE, hd, generator=g).to(torch.bfloat16)
        rows[:, :1] *= torch.exp(torch.randn(1, 1, KVH, 1, hd, generator=g)).to(torch.bfloat16)
        rows[:, 1:] *= torch.exp(torch.randn(n, 1, KVH, PAGE, 1, generator=g)).to(torch.bfloat16)
        self.rows64 = rows.double()
        if dtype == torch.bfloat16:
            self.codes64, self.scales64 = None, None
        else:
            self.codes64, self.scales64 = quantise(self.rows64, dtype)
            self.rows64 = self.codes64 * self.scales64[..., None]
        # rows that hold a token
        live = torch.zeros(n, PAGE, dtype=torch.bool)
        for b in range(B):
            for p in range(0, starts[b] + (0 if has_kv else qlens[b])):
                live[self.tables_list[b][p // PAGE], p % PAGE] = True
        self.live = live
        dead = ~live[:, None, None, :].expand(n, 2, KVH, PAGE)
        T = sum(qlens)
        width_q = (H + (2 * KVH if has_kv else 0)) * hd
        buf = torch.randn(T, width_q + stride_pad, generator=g) * 1.0
        buf[:, :H * hd] *= peaked
        self.qkv = buf.to(torch.bfloat16).cuda()[:, :width_q]
        if dtype == torch.bfloat16:
            stored = rows.clone()
            stored[dead] = math.nan
            self.cache = stored.cuda()
        else:
            scales = self.scales64.float()
            scales[dead] = math.nan
            codes = self.codes64.to(torch.int8) if dtype == torch.int8 else self.codes64.float().to(dtype)
            self.cache = (codes.cuda().contiguous(), scales.cuda().contiguous())
        longest = max([s + q for s, q in zip(starts, qlens)] + [1])
        if rotate:
            ang = torch.arange(longest, dtype=torch.float64)[:, None] * \
                10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
            self.cos, self.sin = ang.cos().float().cuda(), ang.sin().float().cuda()
        else:
            self.cos = self.sin = None
        i32 = dict(dtype=torch.int32, device="cuda")
        Bp = B + pad_seqs
        cu = [0]
        for q in qlens:
            cu.append(cu[-1] + q)
        cu += [cu[-1]] * pad_seqs
        single = all(q == 1 for q in qlens) and not pad_seqs
        tabs = [t + [-1] * (width - len(t)) for t in self.tables_list] + [[-1] * width] * pad_seqs
        self.tables = torch.tensor(tabs, **i32)
        self.ctx = SimpleNamespace(
            n_tokens=T, n_seqs=Bp, max_qlen=max(list(qlens) + [1]), max_kvlen=longest,
            all_decode=single, context_class=sum(longest > t for t in (768, 1536, 4096)),
            cu_q=torch.tensor(cu, **i32), seq_start=torch.tensor(list(starts) + [0] * pad_seqs, **i32),
            seq_qlen=torch.tensor(list(qlens) + [0] * pad_seqs, **i32),
            tok_seq=torch.tensor([b for b, q in enumerate(qlens) for _ in range(q)], **i32),
            tok_pos=torch.tensor([s + i for s, q in zip(starts, qlens) for i in range(q)], **i32))
        groups = sorted({p[0] for p in self.prefixes if p is not None})
        members = [[b for b in range(B) if self.prefixes[b] is not None and self.prefixes[b][0] == k] for k in groups]
        ends = [0]
        for m in members:
            ends.append(ends[-1] + len(m))
        pages = [next(p[1] for p in self.prefixes if p is not None and p[0] == k) for k in groups]
        self.prefix = SimpleNamespace(
            n_groups=len(groups), n_members=ends[-1], max_pages=max(pages, default=0),
            members=torch.tensor(sum(members, []) + [b for b in range(B) if self.prefixes[b] is None], **i32),
            first=torch.tensor(ends, **i32), pages=torch.tensor(pages or [0], **i32),
            seq_pages=torch.tensor([p[1] if p is not None else 0 for p in self.prefixes], **i32))

    def pad(self, n):
        """n padding tokens, each a sequence without tokens, behind a step of single tokens, or behind the last sequence of others."""
        more = lambda t, v, k=n: torch.cat([t, torch.full((k,), v, dtype=t.dtype, device=t.device)])    # noqa: E731
        c = self.ctx
        self.qkv = torch.cat([self.qkv, torch.full((n, self.qkv.shape[1]), math.nan, dtype=self.qkv.dtype, device="cuda")])
        c.n_tokens += n
        c.tok_seq, c.tok_pos = more(c.tok_seq, -1), more(c.tok_pos, 0)
        if c.all_decode:
            c.n_seqs += n
            c.cu_q, c.seq_start, c.seq_qlen = more(c.cu_q, int(c.cu_q[-1])), more(c.seq_start, 0), more(c.seq_qlen, 0)
            self.tables = torch.cat([self.tables, torch.full((n, self.tables.shape[1]), -1, dtype=torch.int32, device="cuda")])
            self.prefix.seq_pages = more(self.prefix.seq_pages, 0)

    def spoil_codes(self):
        """Codes of rows that no token has yet become e4m3's codes that are no number."""
        codes = self.cache[0].view(torch.uint8)
        dead = ~self.live[:, None, None, :].expand(codes.shape[:4])
        codes[dead.to(codes.device)] = 0x7f

    # ---------------------------------------------------------------------------------------------- what has to come out
    def truth(self):
        """(out, tolerance) [T, H hd] float64, and the cache as it has to be afterwards (codes and scales, or rows)."""
        H, KVH, hd, scale = self.H, self.KVH, self.hd, self.hd ** -0.5
        T = self.qkv.shape[0]
        heads = self.qkv.cpu().double().reshape(T, -1, hd)
        cos = self.cos.cpu().double() if self.cos is not None else None
        sin = self.sin.cpu().double() if self.cos is not None else None
        rows = self.rows64.clone()
        codes, scales = (None, None) if self.codes64 is None else (self.codes64.clone(), self.scales64.clone())
        out = torch.zeros(T, H, hd, dtype=torch.float64)
        tol = torch.zeros(T, H, hd, dtype=torch.float64)
        eight = self.dtype != torch.bfloat16
        t = 0
        plan = []
        for b, (s0, q) in enumerate(zip(self.starts, self.qlens)):
            for i in range(q):
                pos = s0 + i
                qh = heads[t, :H]
                if cos is not None:
                    qh = turn(qh, cos[pos], sin[pos])
                if self.has_kv:
                    k, v = heads[t, H:H + KVH], heads[t, H + KVH:]
                    if cos is not None:
                        k = to_bf16(turn(k, cos[pos], sin[pos]))
                    kv = torch.stack([k, v])
                    page, slot = self.tables_list[b][pos // PAGE], pos % PAGE
                    if eight:
                        c, sc = quantise(kv, self.dtype)
                        codes[page, :, :, slot], scales[page, :, :, slot] = c, sc
                        kv = c * sc[..., None]
                    rows[page, :, :, slot] = kv
                plan.append((t, b, pos, qh))
                t += 1
        for t, b, pos, qh in plan:
            first = pos - self.window + 1 if self.window > 0 else pos - pos % -self.window if self.window < 0 else 0
            first = max(first, 0)
            kv = rows[self.tables_list[b][first // PAGE:pos // PAGE + 1]].permute(1, 2, 0, 3, 4).reshape(2, KVH, -1, hd)
            kv = kv[:, :, first % PAGE:first % PAGE + pos - first + 1]
            G = H // KVH
            qg = qh.view(KVH, G, hd)
            score = torch.einsum("kgd,knd->kgn", qg, kv[0]) * scale
            p = torch.softmax(score, -1)
            out[t] = torch.einsum("kgn,knd->kgd", p, kv[1]).reshape(H, hd)
            # the turned queries and the weights are rounded to 2^-12 of themselves (8-bit cache: float16) or 2^-16 (a sum of
            # two bfloat16); the turn itself, the float32 sums and exponentials are within 2^-17 of the magnitudes they add; a weight
            # relative to their sum is off by twice what a score or a weight is; the result is rounded to bfloat16 once
            size = (torch.einsum("kgd,knd->kgn", qg.abs(), kv[0].abs()) * scale).amax(-1)
            r = 2.0 ** -12 if eight else 2.0 ** -16
            off = 2 * ((r + 2.0 ** -17) * size + r + 2.0 ** -17)
            spread = torch.einsum("kgn,knd->kgd", p, kv[1].abs())
            bound = 2.0 ** -8 * out[t].view(KVH, G, hd).abs() + off[..., None] * 1.02 * spread + 1e-30
            if eight:
                # a weight times its value's scale is held in float16 times 2^8 / R, R at most twice the largest scale up to the
                # step's last token: off by half of float16's smallest number, 2^-25, hence by 2^-32 of that scale at most,
                # whatever its size; the row's largest weight is 1, so that the sum they are divided by is 1 or more
                held = self.tables_list[b][:-(-(self.starts[b] + self.qlens[b]) // PAGE)]
                sv = scales[held, 1].permute(1, 0, 2).reshape(KVH, -1)[:, :self.starts[b] + self.qlens[b]]
                most = torch.where(torch.isfinite(sv), sv, torch.zeros_like(sv)).amax(-1)
                seen = codes[self.tables_list[b][first // PAGE:pos // PAGE + 1], 1].permute(1, 0, 2, 3).reshape(KVH, -1, hd)
                seen = seen[:, first % PAGE:first % PAGE + pos - first + 1].abs().sum(1)
                bound = bound + (2.0 ** -32 * most[:, None] * seen)[:, None]
            tol[t] = bound.reshape(H, hd)
        return out.view(T, -1), tol.view(T, -1), (codes, scales) if eight else rows

    def check_cache(self, want):
        """Live rows and the step's own are as they have to be; no other row was touched."""
        touched = self.live.clone()
        if self.has_kv:
            for b, (s0, q) in enumerate(zip(self.starts, self.qlens)):
                for p in range(s0, s0 + q):
                    touched[self.tables_list[b][p // PAGE], p % PAGE] = True
        m = touched[:, None, None, :].expand(-1, 2, self.KVH, -1)
        if self.dtype == torch.bfloat16:
            got = self.cache.cpu().double()
            # a key turned in 32 bits may round to the other neighbour
            assert ((got[m] - want[m]).abs() <= 2.0 ** -7 * want[m].abs() + 1e-30).all()
            assert torch.isnan(got[~m]).all()
            return
        codes, scales = self.cache
        assert torch.equal(codes.float().cpu().double()[m], want[0][m])
        assert torch.equal(scales.cpu().double()[m].nan_to_num(-1), want[1].float().double()[m].nan_to_num(-1))
        assert torch.isnan(scales.cpu()[~m]).all()

    def shared_out(self, **kw):
        from oracle_engine_b200.csrc import ops_kv8
        out = torch.full((self.qkv.shape[0], self.H * self.hd), 7.0, dtype=torch.bfloat16, device="cuda")
        ops_kv8.attention_shared(out, self.qkv, self.cos, self.sin, self.cache, self.tables, self.ctx, self.prefix, self.H, self.KVH,
                                 self.hd, self.hd ** -0.5, has_kv=self.has_kv, **kw)
        return out

    def out(self, **kw):
        from oracle_engine_b200.csrc import ops_kv8
        out = torch.full((self.qkv.shape[0], self.H * self.hd), 7.0, dtype=torch.bfloat16, device="cuda")
        ops_kv8.attention_kv8(out, self.qkv, self.cos, self.sin, self.cache, self.tables, self.ctx, self.H, self.KVH, self.hd,
                              self.window, self.hd ** -0.5, has_kv=self.has_kv, **kw)
        return out


def close(got, want, tol):
    d = (got.cpu().double() - want).abs()
    worst = (d / tol).max().item() if d.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} times the tolerance"
