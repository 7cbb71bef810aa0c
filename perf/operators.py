"""The 8-bit cache and the attention over it, and the attention of sequences that begin with the same pages, as cases to be timed.

The paged cache of a grouped-query attention holds pages of 64 tokens.  In its 8-bit form a row (one token's key or value of one
KV head) is kept as codes, int8 or e4m3, and a float32 scale: with a = the row's largest magnitude and c = 127 (int8) or 448 (e4m3)
    code = row * c / a, rounded to the nearest code, ties to even;    scale = a / c;    the row reads as code * scale.
Keys are turned by their position first and rounded to bfloat16, which is what the 16-bit cache holds.  Four kinds of case:

  write    keys and values of a step's tokens into the cache (`kv8_write`)
  decode   a step of one token a sequence: rotation, write and attention over the 8-bit cache (`attention_kv8`)
  prompt   a step of prompts or of portions behind a cache, the same call
  shared   a step of one token a sequence, where the first pages of groups of sequences are the same pages (`attention_shared`),
           over the 16-bit or the 8-bit cache

Heads are those of the Llama shapes that the benchmark has: 24 over 8 KV heads of 128 (3B), 32 over 8 of 64 (1B) and of 128 (8B),
and drawn cases add single heads and larger groups.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

PAGE = 64
SHAPES = {"3b": (24, 8, 128), "1b": (32, 8, 64), "8b": (32, 8, 128), "one": (8, 8, 128), "wide": (32, 2, 64), "odd": (20, 4, 128)}
LARGEST = {"int8": 127.0, "fp8": 448.0}
TYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------- the cases
def _case(kind, shape, codes, batch, lo, hi, new=1, window=0, groups=0, prefix=0, alone=0):
    """batch sequences whose caches hold lo to hi tokens before the step, `new` tokens each at most (the last sequence's; the others
    bring fewer where `new` is above 1).  window: 0 every key, n the last n, -n the chunk of n.  shared: `groups` groups of
    sequences with a prefix of `prefix` tokens (the g-th group's is shorter by g eighths), `alone` sequences in none; lo to hi
    are then what each holds behind its prefix."""
    return {"kind": kind, "shape": shape, "codes": codes, "batch": batch, "lo": lo, "hi": hi, "new": new, "window": window,
            "groups": groups, "prefix": prefix, "alone": alone}


def listed():
    return [
        # one user's next token: the write alone, a call where only latency counts
        {"name": "write-1", **_case("write", "3b", "int8", 1, 130, 130)},
        # a full server's step, one token of each of 64 sequences
        {"name": "write-64", **_case("write", "8b", "fp8", 64, 33, 4019)},
        # prompts of a batch that start together
        {"name": "write-prompts", **_case("write", "3b", "int8", 5, 0, 0, new=2047)},
        # a short question continued
        {"name": "decode-1", **_case("decode", "3b", "int8", 1, 137, 137)},
        # one user behind a long document
        {"name": "decode-1-long", **_case("decode", "8b", "fp8", 1, 32000, 32000)},
        # a full server, contexts of unequal length
        {"name": "decode-64", **_case("decode", "3b", "int8", 64, 144, 4019)},
        # layers with a window
        {"name": "decode-16-window", **_case("decode", "1b", "fp8", 16, 300, 6001, window=1024)},
        # a prompt of 2,048 tokens into an empty cache
        {"name": "prompt-2048", **_case("prompt", "3b", "int8", 1, 0, 0, new=2048)},
        # a portion of a prompt behind a long document
        {"name": "portion-192", **_case("prompt", "8b", "fp8", 1, 12005, 12005, new=192)},
        # eight requests behind one instruction text
        {"name": "shared-8", **_case("shared", "3b", "bf16", 8, 20, 512, groups=1, prefix=2048)},
        # a full server of requests about one long document
        {"name": "shared-64", **_case("shared", "8b", "int8", 64, 20, 480, groups=1, prefix=8192)},
        # three instruction texts at once, some requests with none
        {"name": "shared-groups", **_case("shared", "1b", "bf16", 48, 20, 700, groups=3, prefix=4096, alone=6)},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "decode", "decode", "prompt", "shared", "shared"])
    shape = rng.choice(list(SHAPES))
    codes = rng.choice(["int8", "fp8"] if kind != "shared" else ["bf16", "int8", "fp8"])
    if kind == "write":
        new = rng.choice([1, _log(rng, 2, 2048)])
        batch = _log(rng, 1, 64) if new == 1 else _log(rng, 1, max(1, min(64, 10000 // new)))
        hi = _log(rng, 1, 4000)
        return _case(kind, shape, codes, batch, rng.randint(0, hi), hi, new=new)
    if kind == "decode":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 1, min(32000, 250000 // batch))
        window = rng.choice([0, 0, 0, _log(rng, 1, 4096), -_log(rng, 64, 4096)])
        return _case(kind, shape, codes, batch, rng.randint(0, hi), hi, window=window)
    if kind == "prompt":
        batch = _log(rng, 1, 8)
        new = _log(rng, 2, 2048 // batch)
        hi = rng.choice([0, _log(rng, 1, max(2, min(12000, 2400000 // (new * batch))))])
        window = rng.choice([0, 0, 0, _log(rng, 1, 4096), -_log(rng, 64, 4096)])
        return _case(kind, shape, codes, batch, rng.randint(0, hi), hi, new=new, window=window)
    batch = _log(rng, 2, 64)
    groups = rng.randint(1, max(1, min(4, batch // 2)))
    hi = _log(rng, 1, 700)
    return _case(kind, shape, codes, batch, rng.randint(0, hi), hi, groups=groups, prefix=_log(rng, 64, 8192) // 64 * 64,
                 alone=rng.randint(0, batch - 2 * groups) // 3)


# ------------------------------------------------------------------------------------------------------- inputs
def _plan(case):
    """Per sequence (prefix pages, its group or -1, tokens held before the step, new tokens): of the case alone."""
    B, lo, hi, new = (case[k] for k in ("batch", "lo", "hi", "new"))
    seqs = []
    for i in range(B):
        at = (i + 1) * 0.6180339887498949 % 1.0 if i + 1 < B else 1.0          # the last one has the most
        group = -1 if case["groups"] == 0 or i < case["alone"] else (i - case["alone"]) % case["groups"]
        pages = max(1, case["prefix"] // PAGE * (8 - group) // 8) if group >= 0 else 0
        seqs.append((pages, group, pages * PAGE + lo + int((hi - lo) * at), max(1, int(new * (0.25 + 0.75 * at))) if new > 1 else 1))
    return seqs


def _quantise(rows, codes):
    """Codes and scales of rows whose values a bfloat16 holds.  The product and the quotient in 64 bits: the quotient of such values
    lies on the border between two codes or far from it in 32 bits' terms."""
    c = LARGEST[codes]
    a = rows.double().abs().amax(-1, keepdim=True)
    x = rows.double() * c / torch.where(a > 0, a, torch.ones_like(a))
    code = torch.round(x).to(torch.int8) if codes == "int8" else x.float().to(torch.float8_e4m3fn)
    return code, (a / c).float()[..., 0]


def prepare(case, seed):
    H, KVH, hd = SHAPES[case["shape"]]
    codes, B = case["codes"], case["batch"]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    seqs = _plan(case)
    # page tables: a group's prefix pages are its members', the other pages each sequence's own, all in any order
    first, tables, n_pages = {}, [], 0
    for pages, group, held, new in seqs:
        if group >= 0 and group not in first:
            first[group] = (n_pages, pages)
            n_pages += pages
    for pages, group, held, new in seqs:
        own_pages = -(-(held + new) // PAGE) - pages
        row = list(range(first[group][0], first[group][0] + pages)) if group >= 0 else []
        tables.append(row + list(range(n_pages, n_pages + own_pages)))
        n_pages += own_pages
    width = max(len(t) for t in tables)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    flat = torch.tensor([t + [-1] * (width - len(t)) for t in tables], dtype=torch.int64, device="cuda")
    tables = torch.where(flat >= 0, order[flat.clamp(min=0)], torch.full_like(order[:1], -1)).contiguous()

    # what the cache holds: keys with a few large channels, values of unequal size from token to token
    loud = torch.exp(0.7 * torch.randn(1, 1, KVH, 1, hd, generator=g, device="cuda"))
    kv = torch.empty(n_pages, 2, KVH, PAGE, hd, dtype=torch.bfloat16, device="cuda")
    for p in range(0, n_pages, 512):
        x = torch.randn(min(512, n_pages - p), 2, KVH, PAGE, hd, generator=g, device="cuda")
        x[:, :1] *= loud
        x[:, 1:] *= torch.exp(0.5 * torch.randn(x.shape[0], 1, KVH, PAGE, 1, generator=g, device="cuda"))
        kv[p:p + 512] = x.to(torch.bfloat16)
    s = {"case": dict(case)}
    if codes == "bf16":
        s["cache"] = kv
    else:
        s["codes"] = torch.empty(kv.shape, dtype=TYPES[codes], device="cuda")
        s["scales"] = torch.empty(kv.shape[:-1], dtype=torch.float32, device="cuda")
        for p in range(0, n_pages, 512):
            s["codes"][p:p + 512], s["scales"][p:p + 512] = _quantise(kv[p:p + 512], codes)

    # the step: the projections of its tokens and what says where they belong
    qlen = [n for _, _, _, n in seqs]
    start = [h for _, _, h, _ in seqs]
    T = sum(qlen)
    qkv = torch.randn(T, (H + 2 * KVH) * hd, generator=g, device="cuda")
    qkv[:, H * hd:(H + KVH) * hd] *= loud.view(1, KVH, 1, hd).expand(1, KVH, 1, hd).reshape(1, KVH * hd)
    s["qkv"] = qkv.to(torch.bfloat16)
    i32 = dict(dtype=torch.int32, device="cuda")
    cu = [0]
    for n in qlen:
        cu.append(cu[-1] + n)
    longest = max(h + n for h, n in zip(start, qlen))
    s["step"] = SimpleNamespace(
        n_tokens=T, n_seqs=B, max_qlen=max(qlen), max_kvlen=longest, all_decode=max(qlen) == 1,
        context_class=sum(longest > t for t in (768, 1536, 4096)), cu_q=torch.tensor(cu, **i32), seq_start=torch.tensor(start, **i32),
        seq_qlen=torch.tensor(qlen, **i32),
        tok_seq=torch.tensor([b for b, n in enumerate(qlen) for _ in range(n)], **i32),
        tok_pos=torch.tensor([h + i for h, n in zip(start, qlen) for i in range(n)], **i32))
    if case["kind"] == "shared":
        members = [[b for b, q in enumerate(seqs) if q[1] == k] for k in range(case["groups"])]
        ends = [0]
        for m in members:
            ends.append(ends[-1] + len(m))
        s["prefix"] = SimpleNamespace(
            n_groups=case["groups"], n_members=ends[-1], max_pages=max(first[k][1] for k in first),
            members=torch.tensor(sum(members, []) + [b for b, q in enumerate(seqs) if q[1] < 0], **i32),
            first=torch.tensor(ends, **i32), pages=torch.tensor([first[k][1] for k in range(case["groups"])], **i32),
            seq_pages=torch.tensor([q[0] for q in seqs], **i32))
    s["tables"] = tables
    angle = torch.arange(longest, dtype=torch.float64, device="cuda")[:, None] * \
        500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
    s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    return s


# ------------------------------------------------------------------------------------------------------- the plain form
def _turn(x, cos, sin):
    half = x.shape[-1] // 2
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)


def _to_bf16_once(x):
    """float64 to the nearest bfloat16 in one rounding (a cast would go through 32 bits)."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 256.0), e - 8).to(torch.bfloat16)


def _plain(s):
    case, step = s["case"], s["step"]
    H, KVH, hd = SHAPES[case["shape"]]
    T, G = step.n_tokens, H // KVH
    seq, pos = step.tok_seq.long(), step.tok_pos.long()
    qkv = s["qkv"].view(T, H + 2 * KVH, hd)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    k = _to_bf16_once(_turn(qkv[:, H:H + KVH].double(), cos.double(), sin.double()))         # values next to a border
    kv = torch.stack([k, qkv[:, H + KVH:]], 1)                                               # [T, 2, KVH, hd]
    page, row = s["tables"][seq, pos // PAGE].long(), pos % PAGE
    if case["codes"] == "bf16":
        s["cache"][page, :, :, row] = kv
        kept = {"cache": s["cache"]}
    else:
        code, scale = _quantise(kv, case["codes"])
        s["codes"].view(torch.uint8)[page, :, :, row] = code.view(torch.uint8)
        s["scales"][page, :, :, row] = scale
        kept = {"codes": s["codes"], "scales": s["scales"]}
    if case["kind"] == "write":
        return kept

    # the sequences' rows side by side, padded to the longest
    B, Q, at = step.n_seqs, step.max_qlen, s["tables"].clamp(min=0).long()
    N = at.shape[1] * PAGE
    if case["codes"] == "bf16":
        rows = s["cache"][at].float()
    else:
        rows = s["codes"].view(torch.uint8)[at].view(TYPES[case["codes"]]).float() * s["scales"][at][..., None]
    rows = rows.permute(2, 0, 3, 1, 4, 5).reshape(2, B, KVH, N, hd)
    index = torch.arange(T, device="cuda") - step.cu_q[seq].long()
    q = torch.zeros(B, Q, H, hd, device="cuda")
    q[seq, index] = _turn(qkv[:, :H].float(), cos, sin)
    where = torch.zeros(B, Q, dtype=torch.int64, device="cuda")
    where[seq, index] = pos
    q = q.view(B, Q, KVH, G, hd).permute(0, 2, 1, 3, 4).reshape(B, KVH, Q * G, hd)
    scores = (q @ rows[0].transpose(-1, -2)).view(B, KVH, Q, G, N) * hd ** -0.5
    keys, w = torch.arange(N, device="cuda"), case["window"]
    lowest = where - w + 1 if w > 0 else where - where % -w if w < 0 else torch.zeros_like(where)
    seen = (keys <= where[..., None]) & (keys >= lowest[..., None])
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, KVH, Q * G, N)
    out = (p @ rows[1]).view(B, KVH, Q, G, hd).permute(0, 2, 1, 3, 4).reshape(B, Q, H * hd)
    return {"out": out[seq, index].to(torch.bfloat16), **kept}


def run(s):
    if not own:
        return _plain(s)
    from oracle_engine_b200.csrc import ops_kv8
    case, step = s["case"], s["step"]
    H, KVH, hd = SHAPES[case["shape"]]
    if case["codes"] == "bf16":
        cache, kept = s["cache"], {"cache": s["cache"]}
    else:
        cache, kept = (s["codes"], s["scales"]), {"codes": s["codes"], "scales": s["scales"]}
    if case["kind"] == "write":
        ops_kv8.kv8_write(s["qkv"], s["cos"], s["sin"], cache, s["tables"], step.tok_seq, step.tok_pos, H, KVH, hd)
        return kept
    out = torch.empty(step.n_tokens, H * hd, dtype=torch.bfloat16, device="cuda")
    if case["kind"] == "shared":
        ops_kv8.attention_shared(out, s["qkv"], s["cos"], s["sin"], cache, s["tables"], step, s["prefix"], H, KVH, hd, hd ** -0.5)
    else:
        ops_kv8.attention_kv8(out, s["qkv"], s["cos"], s["sin"], cache, s["tables"], step, H, KVH, hd, case["window"], hd ** -0.5)
    return {"out": out, **kept}


# ------------------------------------------------------------------------------------------------------- work and truth
def work(case):
    H, KVH, hd = SHAPES[case["shape"]]
    seqs, w = _plan(case), case["window"]
    row = hd * 2 if case["codes"] == "bf16" else hd + 4
    T = sum(n for _, _, _, n in seqs)
    written = T * 2 * KVH * (2 * hd + row)                    # read as projected, written to the cache
    if case["kind"] == "write":
        return {"bytes": written, "flops": 6.0 * T * KVH * hd}
    read, pairs, prefixes = 0, 0, {}
    for pages, group, held, new in seqs:
        def first(p):
            return max(0, p - w + 1) if w > 0 else p - p % -w if w < 0 else 0
        pairs += sum(p - first(p) + 1 for p in range(held, held + new))
        read += max(0, held - max(first(held), pages * PAGE))           # what earlier steps left; a prefix is read once
        if group >= 0:
            prefixes[group] = pages * PAGE
    read += sum(prefixes.values())
    return {"bytes": read * 2 * KVH * row + written + T * 2 * H * hd * 2, "flops": 4.0 * H * hd * pairs}


def _nearest(x, step):
    """x to the nearest multiple of step, ties to the even one, in 64 bits."""
    y = x / step
    down = torch.floor(y)
    up = (y - down > 0.5) | ((y - down == 0.5) & (down.remainder(2) == 1))
    return (down + up.double()) * step


def exact(case, seed):
    s = prepare(case, seed)
    H, KVH, hd = SHAPES[case["shape"]]
    T = s["step"].n_tokens
    half, c = hd // 2, LARGEST.get(case["codes"])
    heads = s["qkv"].view(T, H + 2 * KVH, hd).double()
    turned = heads.clone()
    angles = torch.complex(s["cos"].double(), s["sin"].double())[s["step"].tok_pos.long()][:, None]
    z = torch.complex(heads[:, :H + KVH, :half], heads[:, :H + KVH, half:]) * angles
    turned[:, :H + KVH, :half], turned[:, :H + KVH, half:] = z.real, z.imag
    new = turned[:, H:].reshape(T, 2, KVH, hd)
    new = _nearest(new, torch.exp2(torch.floor(torch.log2(new.abs().clamp(min=1e-300))) - 7))    # 8 significant bits
    if case["codes"] == "bf16":
        rows = s["cache"].double()
        kept = {"cache": rows}
    else:
        codes, scales = s["codes"].double(), s["scales"].double()
        kept = {"codes": codes, "scales": scales}
        a = new.abs().amax(-1, keepdim=True)
        x = new * c / a.clamp(min=1e-300)
        x = _nearest(x, 1.0 if case["codes"] == "int8" else torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3))
    at = [(int(t), int(p)) for t, p in zip(s["step"].tok_seq.tolist(), s["step"].tok_pos.tolist())]
    tables = s["tables"].tolist()
    page = torch.tensor([tables[b][p // PAGE] for b, p in at], device="cuda")
    slot = torch.tensor([p % PAGE for _, p in at], device="cuda")
    if case["codes"] == "bf16":
        rows[page, :, :, slot] = new
    else:
        codes[page, :, :, slot] = x
        scales[page, :, :, slot] = (a / c)[..., 0]
        if case["codes"] == "int8":
            kept["codes"] = codes.to(torch.int8)
    if case["kind"] == "write":
        return kept
    out = torch.zeros(T, H, hd, dtype=torch.float64, device="cuda")
    t0 = 0
    for b, (_, _, held, n) in enumerate(_plan(case)):
        mine = torch.tensor(tables[b][:-(-(held + n) // PAGE)], device="cuda")
        kv = rows[mine] if case["codes"] == "bf16" else codes[mine] * scales[mine][..., None]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(2, KVH, -1, hd)[:, :, :held + n]
        p = torch.arange(held, held + n, device="cuda")[:, None]
        key = torch.arange(held + n, device="cuda")[None]
        w = case["window"]
        hidden = key > p
        if w > 0:
            hidden |= p - key >= w
        if w < 0:
            hidden |= key // -w != p // -w
        for h in range(H):
            score = turned[t0:t0 + n, h] @ kv[0, h // (H // KVH)].T / math.sqrt(hd)
            score[hidden] = -math.inf
            out[t0:t0 + n, h] = torch.softmax(score, -1) @ kv[1, h // (H // KVH)]
        t0 += n
    return {"out": out.view(T, H * hd), **kept}
