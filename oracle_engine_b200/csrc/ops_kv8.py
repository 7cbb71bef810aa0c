"""The 8-bit paged cache and the attention that reads it, and the attention of sequences that begin with the same pages
(csrc/attention_kv8.cu: the write, and few rows; csrc/attention_rows.cu: many; one library of each per head size).

A `cache` argument is one cache entry: a pair (codes [pages, 2, KVH, PAGE, hd] int8 or float8_e4m3fn, scales float32 [pages, 2, KVH,
PAGE]), or, where a function says so, the 16-bit entry [pages, 2, KVH, PAGE, hd] bfloat16.  A row (one token's key or value of one KV
head) reads as code * scale: with a the row's largest magnitude and c = 127 or 448, code = row * c / a to the nearest code (ties to
even) and scale = a / c.  Keys are turned by their position and rounded to bfloat16 before that.  A row with an infinite or
undefined value reads as undefined.

`ahead`: the caller knows that whatever wrote the cache's earlier rows has ended when the kernel before this call starts; the call's kernel
then asks for those rows while the kernel before it still runs.  A copy between the two is enough, or a kernel that is launched without
programmatic serialization, as torch's are; one of this package's is not, since most of them let their successor start before they
have waited for their predecessor.  A model's steps have such a copy: that of their integers.
"""
from __future__ import annotations

import struct
from ctypes import c_char_p, c_int

import torch

from . import build as _build
from . import ops
from .ops import PAGE, KernelError

HEAD_DIMS = (64, 128)
MAX_SPLITS = 148     # of a prefix; with a cluster's CTAs at most MAX_JOINED of attention_kv8.cu
FEW_ROWS = 16        # rows of a tile of attention_kv8.cu
MAX_RUNS = 16        # that a tile's pages are cut into
TILE_ROWS = 128      # rows (a token's or member's heads of one KV head) of a tile of attention_rows.cu; must equal its BM
CODE_TYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32
_KINDS = {torch.bfloat16: 0, torch.int8: 1, torch.float8_e4m3fn: 2}
_libs: dict = {}


_CALL = struct.Struct("<21q21if")        # Kv8Call of kv8.cuh


def _lib(head_dim: int):
    lib = _libs.get(head_dim)
    if lib is None:
        if head_dim not in HEAD_DIMS:
            raise KernelError(f"the 8-bit cache's kernels take heads of {HEAD_DIMS}, not {head_dim}")
        lib = _build.load("attention_kv8", {"OE_HD": head_dim})
        lib.oe_kv8_write.argtypes = lib.oe_attn_kv8.argtypes = [c_char_p]
        lib.oe_kv8_write.restype = lib.oe_attn_kv8.restype = c_int
        _libs[head_dim] = lib
    return lib


def _rows_lib(head_dim: int):
    lib = _libs.get(("rows", head_dim))
    if lib is None:
        lib = _build.load("attention_rows", {"OE_HD": head_dim})
        lib.oe_attn_rows.argtypes = lib.oe_attn_rows_prefix.argtypes = lib.oe_join_parts.argtypes = [c_char_p]
        lib.oe_attn_rows_error.argtypes = []
        lib.oe_attn_rows.restype = lib.oe_attn_rows_prefix.restype = lib.oe_join_parts.restype = lib.oe_attn_rows_error.restype = c_int
        _libs[("rows", head_dim)] = lib
    return lib


def _packed(out, qkv, cos, sin, rows, scales, tables, ctx, part, part_rows: int, parts: int, head_dim: int, dev: int, kind: int, write: int,
            max_qlen: int, n_heads: int, n_kv_heads: int, window: int, scale: float, ahead: bool, warps: int = 0, cluster: int = 0, ordered: int = 0,
            shares: int = 1, mt: int = 0, splits: int = 1, prefix=None) -> bytes:
    """The argument of an attention's entry points; part: room for `parts` parts of `part_rows` rows, or None."""
    T, max_pages, n_pages = qkv.shape[0], tables.shape[1], rows.shape[0]
    part_o = 0 if part is None else part.data_ptr()
    if prefix is None:
        lists, n_groups, n_members = (0, 0, 0, 0), 0, 0
    else:
        lists = (prefix.members.data_ptr(), prefix.first.data_ptr(), prefix.pages.data_ptr(), prefix.seq_pages.data_ptr())
        n_groups, n_members = prefix.n_groups, prefix.n_members
    return _CALL.pack(
        out.data_ptr(), qkv.data_ptr(), qkv.stride(0), 0 if cos is None else cos.data_ptr(), 0 if sin is None else sin.data_ptr(),
        rows.data_ptr(), 0 if scales is None else scales.data_ptr(), n_pages, tables.data_ptr(), ctx.cu_q.data_ptr(), ctx.seq_start.data_ptr(),
        ctx.seq_qlen.data_ptr(), 0, 0, *lists,
        part_o, part_o + 4 * part_rows * parts * head_dim if part_o else 0, _stream(dev),
        _CALL.size, kind, write, max_pages, ctx.n_seqs, T, max_qlen, n_heads, n_kv_heads, window, warps, cluster, ordered, shares, mt, splits,
        n_groups, n_members, ahead, 2 ** 31 - 1 if cos is None else cos.shape[0], tables.shape[0], scale)


def _stream(dev: int) -> int:
    return ops._raw_stream(dev) if ops._raw_stream is not None else ops._stream()


def _sms(dev: int) -> int:
    return ops._sms.get(dev) or ops.sm_count()


def device_error() -> int:
    """The code of a bounded wait that ran out since the last call (0: none).  Synchronises the device."""
    code = 0
    for key, lib in list(_libs.items()):
        if isinstance(key, tuple):
            code = code or int(lib.oe_attn_rows_error())
    return code


def supported(head_dim: int, n_heads: int, n_kv_heads: int) -> bool:
    return head_dim in HEAD_DIMS and n_kv_heads >= 1 and n_heads % n_kv_heads == 0 and 1 <= n_heads // n_kv_heads <= TILE_ROWS


def _cache_args(what: str, cache, n_kv_heads: int, head_dim: int, allow_16: bool) -> tuple:
    """(kind, rows, scales or None) of a cache entry."""
    rows, scales = (cache, None) if isinstance(cache, torch.Tensor) else cache
    kind = _KINDS.get(rows.dtype)
    if kind is None or (scales is None) != (kind == 0):
        raise KernelError(f"{what}: a cache entry is (codes, scales) with int8 or float8_e4m3fn codes, or a bfloat16 tensor")
    if scales is None and not allow_16:
        raise KernelError(f"{what}: codes and scales expected")
    shape = rows.shape
    if shape[1:] != (2, n_kv_heads, PAGE, head_dim) or not rows.is_contiguous():
        raise KernelError(f"{what}: cache entry must be contiguous [pages, 2, KVH, PAGE, head_dim]")
    if scales is not None and (scales.dtype is not _F32 or not scales.is_contiguous() or scales.shape != shape[:4]):
        raise KernelError(f"{what}: scales must be contiguous float32 [pages, 2, KVH, PAGE]")
    return kind, rows, scales


def _check_heads(what: str, n_heads: int, n_kv_heads: int, head_dim: int) -> None:
    if not supported(head_dim, n_heads, n_kv_heads):
        raise KernelError(f"{what}: {n_heads} heads over {n_kv_heads} KV heads of {head_dim} are outside what the kernels take "
                          f"(head sizes {HEAD_DIMS}, heads a multiple of the KV heads)")


def _check_scale(what: str, scale: float) -> None:
    """The kernels take a row's largest score times the scale for its largest weight's exponent; with the factor of a row of queries of
    zeros, 2^-126, the scale has to stay a number that is not 0."""
    if not 1e-6 <= scale < float("inf"):
        raise KernelError(f"{what}: the scores' scale must be a positive number, 1e-6 at least, not {scale}")


def _check_rows(what: str, qkv, cos, sin, width: int, head_dim: int) -> None:
    shape, stride = qkv.shape, qkv.stride()
    if qkv.dtype is not _BF16 or len(shape) != 2 or shape[1] != width or stride[1] != 1 or stride[0] % 8 or qkv.data_ptr() % 16:
        raise KernelError(f"{what}: qkv must be bfloat16 [T, {width}] with rows of multiples of 16 bytes")
    if cos is None and sin is None:
        return
    for t in (cos, sin):
        if t is None or t.dtype is not _F32 or t.dim() != 2 or t.shape[1] != head_dim // 2 or not t.is_contiguous() or t.data_ptr() % 16:
            raise KernelError(f"{what}: cos/sin must be contiguous float32 [max_pos, head_dim/2]")
    if cos.shape != sin.shape:
        raise KernelError(f"{what}: cos and sin must have equally many rows")


def _check_ints(what: str, names: tuple, tensors: tuple) -> None:
    for t, name in zip(tensors, names):
        if t.dtype is not _I32 or not t.is_contiguous():
            raise KernelError(f"{what}: {name} must be a contiguous int32 tensor")


def _here(what: str, *tensors) -> int:
    """The current device, on whose stream the kernel is launched; every tensor is on it."""
    if tensors[0].get_device() < 0:
        ops._dev(*tensors)
    dev = torch._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            ops._dev(t)
            raise KernelError(f"{what}: a tensor is on {t.device}, the current device is cuda:{dev}")
    return dev


def _check_step(what: str, out, qkv, cos, tables, ctx, n_heads: int, head_dim: int) -> None:
    n, longest = ctx.n_seqs, getattr(ctx, "max_kvlen", 0)
    cu_q, start, qlen = ctx.cu_q, ctx.seq_start, ctx.seq_qlen
    _check_ints(what, ("tables", "cu_q", "seq_start", "seq_qlen"), (tables, cu_q, start, qlen))
    if out.dtype is not _BF16 or out.shape != (qkv.shape[0], n_heads * head_dim) or not out.is_contiguous() or out.data_ptr() % 16:
        raise KernelError(f"{what}: out must be contiguous bfloat16 [T, {n_heads * head_dim}]")
    table = tables.shape
    if len(table) != 2 or table[0] < n or cu_q.numel() <= n or start.numel() < n or qlen.numel() < n:
        raise KernelError(f"{what}: the step's tables are shorter than its {n} sequences")
    if longest > table[1] * PAGE or cos is not None and max(longest, 1) > cos.shape[0]:
        raise KernelError(f"{what}: a sequence of {longest} tokens is longer than its page table or the position tables")


def kv8_write(qkv, cos, sin, cache, tables, tok_seq, tok_pos, n_heads: int, n_kv_heads: int, head_dim: int) -> None:
    """Keys (turned at each token's position; cos/sin float32 [max_pos, hd/2] or None) and values of the step's tokens into the
    8-bit cache.  qkv [T, (H + 2 KVH) hd] is left as it is; tok_seq < 0: a padding row; a sequence without a table, a
    position without an angle or a page outside the cache: nothing is written.  No two tokens of a call have the same place."""
    what = "kv8_write"
    _check_heads(what, n_heads, n_kv_heads, head_dim)
    kind, codes, scales = _cache_args(what, cache, n_kv_heads, head_dim, False)
    dev = _here(what, qkv, cos, sin, codes, scales, tables, tok_seq, tok_pos)
    _check_rows(what, qkv, cos, sin, (n_heads + 2 * n_kv_heads) * head_dim, head_dim)
    _write(what, dev, kind, qkv, cos, sin, codes, scales, tables, tok_seq, tok_pos, n_heads, n_kv_heads, head_dim)


def _write(what: str, dev: int, kind: int, qkv, cos, sin, codes, scales, tables, tok_seq, tok_pos, n_heads: int, n_kv_heads: int, head_dim: int) -> None:
    """kv8_write of rows and a cache that have been checked."""
    _check_ints(what, ("tables", "tok_seq", "tok_pos"), (tables, tok_seq, tok_pos))
    T, table = qkv.shape[0], tables.shape
    if len(table) != 2 or tok_seq.numel() < T or tok_pos.numel() < T:
        raise KernelError(f"{what}: fewer places than the {T} tokens")
    if T == 0:
        return
    ops._check(_lib(head_dim).oe_kv8_write(_CALL.pack(
        0, qkv.data_ptr(), qkv.stride(0), 0 if cos is None else cos.data_ptr(), 0 if sin is None else sin.data_ptr(), codes.data_ptr(),
        scales.data_ptr(), codes.shape[0], tables.data_ptr(), 0, 0, 0, tok_seq.data_ptr(), tok_pos.data_ptr(), 0, 0, 0, 0, 0, 0, _stream(dev),
        _CALL.size, kind, 1, table[1], 0, T, 0, n_heads, n_kv_heads, 0, 0, 0, 0, 1, 0, 1, 0, 0, 0,
        2 ** 31 - 1 if cos is None else cos.shape[0], table[0], 0.0)), "kv8_write")


def many_pairs(n_seqs: int, n_kv_heads: int, sm_count: int | None = None) -> bool:
    """More than three (sequence, KV head) pairs for each SM, of which two to five are resident at once: the longest sequences go first."""
    return n_seqs * n_kv_heads > 3 * (sm_count or ops.sm_count())


def decode_form(n_seqs: int, n_kv_heads: int, context_class: int, window: int = 0, sm_count: int | None = None) -> tuple:
    """(warps of a CTA, CTAs (a thread-block cluster) that share the keys of one (sequence, KV head), or CTAs that do so without being
    a cluster) of a step of few rows.

    Short contexts: a CTA a pair, of twelve warps, which fill an SM's shared memory, while the pairs have an SM each, else of four.
    Longer ones: CTAs of four warps, which leave room on their SMs for the products that overlap them; up to 8 of a cluster, and
    for very long ones as many as fill the SMs twice and leave parts for another kernel.  ms a decode step of the 28-layer model with 24
    heads over 8 KV heads of 128, int8:  1 sequence of 2,000 keys 12x1 1.83, 12x4 1.63, 12x8 1.58, 4x8 1.64; of 8,000 12x8 1.78,
    12x1x18 2.39, 4x1x18 1.74; of 32,000 12x8 2.46, 12x1x18 2.74, 4x1x18 2.30, 4x1x37 2.05;  4 of 2,000 12x2 1.79, 12x4 2.47, 4x4
    1.79, of 8,000 12x2 2.43, 4x4 2.40;  8 of 512 12x1 1.66, 4x1 1.77, of 2,000 12x1 2.10, 12x2 2.46, 4x2 2.03, 4x4 1.90, of 8,000 12x1
    3.40, 12x2 3.15, 4x4 2.52;  16 of 2,000 12x1 2.39, 4x1 2.64, 4x2 2.32;  32 of 1,000 12x1 2.94, 4x1 2.78.
    A pair's parts are joined by one warp a row, and a CTA of 8,000 keys split over 296 has no tile for most warps: no more than half as many
    as there are SMs (us a call, one sequence of 8,000, 32,000, 120,000 keys: 16 heads over 1 of 128 with 37 CTAs 15.5, 24.2, 56.1, 74 18.0,
    23.5, 39.7, 296 39.7, 41.8, 47.4; 16 over 2 with 37 12.6, 19.6, 45.1, 74 15.8, 19.9, 32.4, 148 23.7, 26.5, 37.3).  Heads do not enter
    otherwise: with heads of 64, calls alone are faster with twelve warps than by this rule (32 over 8 heads, 8 of 8,000 keys 27 instead
    of 38, 16 of 2,000 15 instead of 21), with heads of 128 it is within 20 % of the fastest form for 8 and 16 KV heads."""
    sms = sm_count or ops.sm_count()
    pairs = n_seqs * n_kv_heads
    if window and abs(window) <= 1536:             # no more than the second class of contexts is seen
        context_class = min(context_class, 1 if abs(window) > 768 else 0)
    if context_class >= 3 and pairs * 8 <= sms:
        return 4, 1, min(2 * sms // pairs, sms // 2)
    if context_class >= 1:
        if pairs * 16 <= sms:
            return 12, 8, 1
        for cr in (8, 4):
            if pairs * cr <= sms * (1 if cr == 8 else 2):
                return 4, cr, 1
        if context_class >= 2 and pairs <= sms:
            return 4, 2, 1
    return (12 if pairs <= sms else 4), 1, 1


def attention_kv8(out, qkv, cos, sin, cache, tables, ctx, n_heads: int, n_kv_heads: int, head_dim: int, window: int, scale: float,
                  has_kv: bool = True, ahead: bool = False, form: tuple | None = None) -> None:
    """Rotation, cache write (has_kv) and attention of the step's tokens over the 8-bit cache: out[t] is the attention of token t's
    query heads over its sequence's keys up to its own position (window 0: all of them, n > 0: the last n, -n: those of the
    chunk of n positions it lies in), as the cache keeps them, the step's own among them.

    qkv bfloat16 [T, (H + 2 KVH) hd] (or [T, H hd] when has_kv is false: the rows are in the cache) before rotation, left as it
    is; out bfloat16 [T, H hd]; ctx: the step (StepContext: cu_q, seq_start, seq_qlen, tok_seq, tok_pos, n_seqs, max_qlen,
    all_decode; max_kvlen, where it is there, is checked against the tables).  A token at a position without an angle comes out
    undefined and is not written; pages that are not in the cache, or behind the page table, have no keys.  A step of one token a sequence is one launch, any other a write and an attention.  form: the kernel's
    form (decode_form where a sequence has few rows, prompt_form else); None: by those rules."""
    what = "attention_kv8"
    _check_heads(what, n_heads, n_kv_heads, head_dim)
    _check_scale(what, scale)
    kind, codes, scales = _cache_args(what, cache, n_kv_heads, head_dim, False)
    dev = _here(what, out, qkv, cos, sin, codes, scales, tables, ctx.cu_q, ctx.seq_start, ctx.seq_qlen)
    _check_rows(what, qkv, cos, sin, (n_heads + (2 * n_kv_heads if has_kv else 0)) * head_dim, head_dim)
    _check_step(what, out, qkv, cos, tables, ctx, n_heads, head_dim)
    T, n_seqs, sms, window = qkv.shape[0], ctx.n_seqs, _sms(dev), int(window)
    if T == 0 or n_seqs == 0:
        return
    single = bool(ctx.all_decode) and T == n_seqs
    if has_kv and not single:
        _here(what, out, ctx.tok_seq, ctx.tok_pos)
        _write(what, dev, kind, qkv, cos, sin, codes, scales, tables, ctx.tok_seq, ctx.tok_pos, n_heads, n_kv_heads, head_dim)
    group, context_class, max_qlen = n_heads // n_kv_heads, getattr(ctx, "context_class", 0), 1 if single else max(1, ctx.max_qlen)
    if single or max_qlen * group <= FEW_ROWS:
        warps, cluster, shares = form or decode_form(n_seqs, n_kv_heads, context_class, window, sms)
        part = _parts(T * n_heads, shares, head_dim, out.device) if shares > 1 else None
        call = _packed(out, qkv, cos, sin, codes, scales, tables, ctx, part, T * n_heads, shares, head_dim, dev, kind, has_kv and single, max_qlen,
                       n_heads, n_kv_heads, window, scale, ahead, warps, cluster, many_pairs(n_seqs, n_kv_heads, sms), shares)
        ops._check(_lib(head_dim).oe_attn_kv8(call), what, {"warps": warps, "cluster": cluster, "shares": shares})
        if shares > 1:
            ops._check(_rows_lib(head_dim).oe_join_parts(call), "join_parts")
        return
    mt, splits = form or prompt_form(T, n_seqs, group, n_kv_heads, context_class, window, sms, ctx.max_qlen)
    part = _parts(T * n_heads, splits, head_dim, out.device) if splits > 1 else None
    call = _packed(out, qkv, cos, sin, codes, scales, tables, ctx, part, T * n_heads, splits, head_dim, dev, kind, 0, max_qlen, n_heads, n_kv_heads,
                   window, scale, ahead, mt=mt, splits=splits)
    ops._check(_rows_lib(head_dim).oe_attn_rows(call), what, {"tiles": mt, "splits": splits})
    if splits > 1:
        ops.LAUNCHES[0] += 1


def _parts(rows: int, splits: int, head_dim: int, device):
    """Room for the parts of `rows` rows: their sums, then maxima and sums of weights."""
    return torch.empty(rows * splits * (head_dim + 2), dtype=torch.float32, device=device)


def prompt_form(n_tokens: int, n_seqs: int, group: int, n_kv_heads: int, context_class: int, window: int, sm_count: int | None = None,
                max_qlen: int | None = None) -> tuple:
    """(tiles of 128 rows a CTA has, runs that a tile's pages are cut into) of a step of prompts: those of the lowest estimate.

    A CTA takes about 10 us to start and end and 1.0 us a page with one tile, 13 and 1.4 with two; CTAs beyond one an SM queue; runs
    cost their parts' traffic, and the kernel that joins them 3 us.  How long the contexts are is known by class only.  us with 32
    heads over 8 KV heads of 128 in int8, (tiles, runs):  64 tokens (1,1) 11, (1,3) 15, (2,1) 14, (2,3) 18; 300 16, 26, 20, 23; 600 22, 48,
    27, 41; 2,048 (1,1) 95, (2,1) 74, (2,2) 126; 4 of 500 42, 38, 73; 64 of 30 38, 47, 88; 192 tokens behind 12,000 (1,1) 201, (1,3) 81,
    (2,4) 89, (2,6) 68, (2,12) 81; 512 behind 4,000 (1,1) 82, (2,1) 113, (2,2) 78, (2,4) 85; 32 behind 12,000 (1,8) 37, (1,16) 29, (2,16) 33,
    (1,24) 38; 4 of 64 behind 8,000 (1,2) 80, (2,3) 81, (2,4) 67, (2,8) 76; 4 of 192 behind 2,000 (1,1) 85, (2,1) 65, (2,2) 80.
    With 24 heads over 8 and 16 over 16, 2 and 1 of 128, and 32 over 8 of 64, the choice is within 9 % of the fastest form, but for 2,048 tokens of
    16 heads: over 16, 2, 1 KV heads (2,1) 70, 61, 61 where (1,1) takes 56, 49, 49."""
    sms, pages, best = sm_count or ops.sm_count(), (6, 18, 44, 128)[context_class], None
    if window:
        pages = min(pages, abs(window) // PAGE + 2)
    for mt in (1, 2):
        tokens = TILE_ROWS // group * mt                       # of a CTA
        ctas = min(n_seqs * -(-(max_qlen or n_tokens) // tokens), n_tokens // tokens + n_seqs) * n_kv_heads
        for runs in {1, max(1, min(sms // ctas, pages // 4, MAX_RUNS))}:
            full = ctas * runs / sms                            # (the CTAs that queue end together less well)
            us = (full + 0.3 if full > 1 else 1.0) * (10 + pages / runs if mt == 1 else 13 + 1.4 * pages / runs)
            if runs > 1:
                us += 3 + runs * n_tokens * group * n_kv_heads * 2.5e-4
            if best is None or us < best[0]:
                best = us, mt, runs
    return best[1:]


def sharing_pays(groups: list, eight: bool) -> bool:
    """Whether a step's groups, (members, pages in common) each, are read faster by attention_shared than sequence by sequence, where
    the common pages come out of the L2 for all but the first.  Measured with 24 heads over 8 KV heads of 128, 100 keys behind the prefix: ms
    a decode step of 28 layers, shared / apart, prefixes of 1,024, 2,048, 4,096, 8,192 tokens.  16-bit cache: 2 members 2.21/1.56,
    2.28/1.61, 2.42/1.74, 2.65/1.96; 4 2.22/1.63, 2.30/1.74, 2.44/1.97, 2.64/2.41; 8 2.03/1.77, 2.13/2.00, 2.27/2.46, 2.47/3.29; 16 2.00/2.04,
    2.06/2.27, 2.17/2.71, 2.37/3.56; 32 2.73/2.62, 2.78/3.01, 2.83/3.79.  int8: 2 1.73/1.62, 1.79/1.68, 1.92/1.73, 2.12/1.85; 4 1.77/1.67,
    1.83/1.78, 1.93/2.01, 2.14/2.45; 8 1.86/1.78, 1.91/1.89, 2.02/2.12, 2.22/2.56; 16 2.00/2.08, 2.06/2.32, 2.17/2.76, 2.37/3.61; 32
    2.69/2.75, 2.72/3.19, 2.77/4.05.
    The rule does not look at heads.  Other shapes (16 layers, us a layer of a step, shared / apart; S: the rule shares).  16-bit cache, 32
    heads over 8 of 64, 4 members behind 1,024, 2,048, 8,192 tokens 44/44, 46/48, 55/70; 8 46/49, 48/56, 57/97 S; 64 behind 1,024 83/80 S;
    32 over 8 of 128, 8 103/103, 105/111, 116/157 S; 64 behind 1,024 165/152 S; 16 over 16 of 128, 4 59/50, 63/58, 88/104; 8 55/60,
    59/67, 87/115 S; 64 behind 1,024 119/132 S; 32 over 2 of 64, 8 48/48, 51/49, 55/62 S; 64 behind 1,024 76/74 S; 16 over 2 of 128, 8 50/48,
    53/50, 59/63 S.  int8, 32 over 8 of 64, 4 45/52, 47/57, 57/91 S; 8 46/56, 49/60 S, 59/94 S; 16 over 16 of 128, 4 52/50, 56/54, 81/77 S;
    8 52/62, 56/62 S, 81/109 S; 32 over 2 of 64, 4 46/45, 48/46, 50/51 S; 16 over 2 of 128, 4 46/45, 48/46, 52/51 S.  Near its border it costs
    up to 9 % of a layer where it shares, and where it does not it leaves up to a fifth with heads of 64."""
    less, base = (1, 256) if eight else (3, 768)
    return sum((members - less) * (pages * PAGE - base) for members, pages in groups if members > less and pages * PAGE > base) >= 11500


def shared_form(n_seqs: int, n_members: int, n_groups: int, group: int, n_kv_heads: int, max_pages: int, eight: bool,
                sm_count: int | None = None) -> tuple:
    """(tiles of 128 rows a CTA has, runs that a prefix's pages are cut into; warps of a CTA and CTAs of a cluster for the keys behind
    the prefixes).  One tile, so that there are fewer parts to join, unless the tiles alone outnumber the SMs (us, 64 members of 32
    heads behind 8,192 tokens in 8 bits: two tiles and 18 runs 54.0, one tile and 9 runs 53.1; behind 2,048 44.0 / 39.8).  The two kernels
    run beside each other: as many runs as give half of the SMs a CTA while there are at most three of the own keys' CTAs for each SM of the
    other half, else as many as give every SM one (us, 24 heads, runs of half / of all SMs: 8 members behind 2,048 tokens 14.8 / 21.4, in 8 bits 14.2 / 21.3; 16 behind
    4,096 21.7 / 25.6, 18.1 / 23.7; 32 in 8 bits 30.9 / 28.1).  Own keys: CTAs of all an SM has room for while they have an SM each, no clusters
    (8 members, 9 runs, 6 / 3 warps 14.8 / 15.9; 16 24.9 / 21.7)."""
    sms = sm_count or ops.sm_count()
    tiles = -(-n_members // (TILE_ROWS // group))
    mt = 2 if tiles * n_kv_heads > sms else 1
    ctas = max(-(-tiles // mt), n_groups) * n_kv_heads          # (groups of equal size)
    pairs, few = n_seqs * n_kv_heads, 4 if eight else 3
    half = sms // 2
    beside = pairs <= 3 * half and ctas <= half
    warps = few if pairs > (half if beside else sms) else 12 if eight else 6
    return mt, max(1, min(max_pages, (half if beside else sms) // ctas, MAX_SPLITS)), warps, 1


def attention_shared(out, qkv, cos, sin, cache, tables, ctx, prefix, n_heads: int, n_kv_heads: int, head_dim: int, scale: float,
                     has_kv: bool = True, ahead: bool = False, form: tuple | None = None) -> None:
    """A step of one token a sequence in which groups of sequences begin with the same pages: rotation, cache write (has_kv) and
    attention over all keys, as attention_kv8 with window 0, but a group's common pages are read once for all of its members.
    cache: the 8-bit pair or the 16-bit entry.

    prefix: n_groups and n_members (host numbers, or bounds for them: what first and members hold beyond the real ones are
    groups without members), max_pages (the most pages a group has in common), and int32 tensors members (sequences in the order of
    their groups), first [n_groups + 1] (where each group's members begin), pages [n_groups] (full pages that the group's
    tables begin with, whose tokens are all earlier than the step's), seq_pages [n_seqs] (those of the sequence's group, 0 for a sequence in none).
    A group with a member that is no sequence of the step has undefined results.
    form: the kernels' form; None: by shared_form."""
    what = "attention_shared"
    _check_heads(what, n_heads, n_kv_heads, head_dim)
    _check_scale(what, scale)
    kind, rows, scales = _cache_args(what, cache, n_kv_heads, head_dim, True)
    lists = (prefix.members, prefix.first, prefix.pages, prefix.seq_pages)
    dev = _here(what, out, qkv, cos, sin, rows, scales, tables, ctx.cu_q, ctx.seq_start, ctx.seq_qlen, *lists)
    _check_rows(what, qkv, cos, sin, (n_heads + (2 * n_kv_heads if has_kv else 0)) * head_dim, head_dim)
    _check_step(what, out, qkv, cos, tables, ctx, n_heads, head_dim)
    B, n_groups, n_members, sms = ctx.n_seqs, prefix.n_groups, prefix.n_members, _sms(dev)
    if not ctx.all_decode or qkv.shape[0] != B:
        raise KernelError(f"{what}: one token a sequence expected")
    names = ("members", "first", "pages", "seq_pages")
    _check_ints(what, names, lists)
    for t, n, least in zip(lists, names, (n_members, n_groups + 1, n_groups, B)):
        if t.numel() < least:
            raise KernelError(f"{what}: {n} holds {t.numel()} numbers, {least} are needed")
    if B == 0:
        return
    mt, splits, warps, cluster = form or shared_form(
        B, max(1, n_members), max(1, n_groups), n_heads // n_kv_heads, n_kv_heads, max(1, prefix.max_pages), scales is not None, sms)
    part = _parts(B * n_heads, splits, head_dim, out.device)
    call = _packed(out, qkv, cos, sin, rows, scales, tables, ctx, part, B * n_heads, splits, head_dim, dev, kind, has_kv, 1, n_heads, n_kv_heads, 0,
                   scale, ahead, warps, cluster, many_pairs(B, n_kv_heads, sms), 1, mt, splits, prefix)
    if n_groups > 0 and n_members > 0:
        ops._check(_rows_lib(head_dim).oe_attn_rows_prefix(call), "attention_shared_prefix", {"tiles": mt, "splits": splits})
    ops._check(_lib(head_dim).oe_attn_kv8(call), what)
