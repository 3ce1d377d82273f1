"""Paged KV cache in e4m3: half the bytes of the bf16 cache of `ops.paged`, with a power of two for every page and KV head.

`PagesE4M3` holds the pages of one layer.  `kv_append_e4m3` stores new tokens, `paged_attention_decode_e4m3` is the attention of single tokens over
the pages (and can keep the attention weight that every cached token has had), `kv_read_e4m3` gives whole sequences back as rows, as later
portions of prompts attend over them, and `kv_evict_e4m3` drops the tokens with the least attention weight and closes the gaps.

A number of a page is code * 2^exponent.  The exponent of a page's keys (values) for a head is the least in -100 .. 119 under which their largest
finite number is at most 448, the largest code; infinities are held as that code, NaN stays NaN.  Block tables and lengths are those of the
bf16 cache: int32 [batch, width] and int32 [batch], tokens in the cache with the new ones.  On a GPU attention and eviction take up to 65535
sequences a call.
"""
from __future__ import annotations

import functools
import math
import struct
from dataclasses import dataclass

import torch

from .. import _native as N

C = N.C
LEAST_EXPONENT, MOST_EXPONENT, LARGEST_CODE = -100, 119, 448.0
MOST_BLOCK, MOST_TOKENS = 1 << 20, (1 << 30) - 1        # on a GPU: of a page, of a table's row
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


# The argument blocks of csrc/kernels/paged_e4m3.h, packed: a ctypes structure of 25 fields takes 2 us to fill, a fifth of a small call.
_PAGES = "6P3i0q"                                                     # k, v, exponents, weights, blocks; block size, KV heads, head size
_APPEND = struct.Struct("@" + _PAGES + "5P2q4i")                      # k, v, tables, lengths, starts; pitches; rows, batch, width, type
_READ = struct.Struct("@" + _PAGES + "5P2q4i")                        # the same
_DECODE = struct.Struct("@" + _PAGES + "5P2q5if")                     # q, out, tables, lengths, scratch; pitches; batch, width, heads, type, accumulate; scale
_EVICT = struct.Struct("@" + _PAGES + "5P6i")                         # tables, lengths, out tables, kept, lengths out; batch, widths, keep, recent, first

for _name in ("append", "read", "decode", "evict"):
    N.optional_sig("rb_e4m3_" + _name, [C.c_char_p, N.c_void_p])
N.optional_sig("rb_e4m3_decode_scratch_floats", [N.c_int] * 7, N.c_ll)
N._LAUNCHES["rb_e4m3_decode"] = 2
N._LAUNCHES["rb_e4m3_evict"] = 2


@dataclass
class PagesE4M3:
    """The pages of one layer: codes `k`, `v` (float8_e4m3fn [num_blocks, kv_heads, block_size, head_dim]), exponents `k_exp`, `v_exp` (int8
    [num_blocks, kv_heads]) and, where attention weights are kept, `weight` (fp32 [num_blocks, kv_heads, block_size]).  On a GPU block_size is a
    multiple of 16, at most 2^20, head_dim 64 or 128, and a table's row has room for fewer than 2^30 tokens."""
    k: torch.Tensor
    v: torch.Tensor
    k_exp: torch.Tensor
    v_exp: torch.Tensor
    weight: torch.Tensor | None = None

    @classmethod
    def zeros(cls, num_blocks: int, block_size: int, kv_heads: int, head_dim: int, device="cpu", weights: bool = False) -> "PagesE4M3":
        codes = lambda: torch.zeros((num_blocks, kv_heads, block_size, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)  # noqa: E731
        exps = lambda: torch.zeros((num_blocks, kv_heads), dtype=torch.int8, device=device)  # noqa: E731
        return cls(codes(), codes(), exps(), exps(),
                   torch.zeros((num_blocks, kv_heads, block_size), dtype=torch.float32, device=device) if weights else None)

    @property
    def block_size(self) -> int:
        return self.k.shape[2]

    def memory_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_exp, self.v_exp, self.weight) if t is not None)


def _check(what: str, pages: PagesE4M3, block_tables, context_lens, *others) -> tuple:
    """(blocks, KV heads, block size, head size, sequences, table width) of pages and tables that a kernel can take; `others`: further tensors of the
    call.  (Every look at a tensor counts here: the attributes are read once, and shapes before anything else.)"""
    k, v, ke, ve, w = pages.k, pages.v, pages.k_exp, pages.v_exp, pages.weight
    shape, dev = k.shape, k.get_device()
    nb, G, bs, D = shape
    if not (k.dtype is v.dtype is torch.float8_e4m3fn and ke.dtype is ve.dtype is torch.int8 and v.shape == shape and ke.shape == ve.shape == (nb, G) and
            k.is_contiguous() and v.is_contiguous() and ke.is_contiguous() and ve.is_contiguous()):
        raise TypeError(f"{what}: pages are contiguous e4m3 codes [blocks, kv_heads, block_size, head_dim] with int8 exponents [blocks, kv_heads]")
    if w is not None and not (w.dtype is torch.float32 and w.shape == (nb, G, bs) and w.is_contiguous()):
        raise TypeError(f"{what}: weights are contiguous fp32 [blocks, kv_heads, block_size]")
    table, batch = block_tables.shape, context_lens.shape
    if not (block_tables.dtype is context_lens.dtype is torch.int32 and len(table) == 2 and len(batch) == 1 and table[0] == batch[0] and
            block_tables.is_contiguous() and context_lens.is_contiguous()):
        raise TypeError(f"{what}: a contiguous int32 table row and an int32 length per sequence are required")
    if not (v.get_device() == ke.get_device() == ve.get_device() == block_tables.get_device() == context_lens.get_device() == dev and
            (w is None or w.get_device() == dev)):
        raise ValueError(f"{what}: pages, tables and lengths are on one device")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what}: tensors on {k.device} and {t.device}")
    if dev >= 0:
        if bs & 15 or bs > MOST_BLOCK or (D != 64 and D != 128):
            raise ValueError(f"{what}: pages of a multiple of 16 tokens, at most 2^20, and heads of 64 or 128 are required, not {bs} and {D}")
        if table[1] * bs > MOST_TOKENS:
            raise ValueError(f"{what}: a table's row has room for fewer than 2^30 tokens, not {table[1]} pages of {bs}")
        if dev != torch._C._cuda_getDevice():
            raise ValueError(f"{what}: the pages are on {k.device}, which is not the current device")
    return nb, G, bs, D, table[0], table[1]


def _native(p: PagesE4M3, shape) -> tuple:
    w = p.weight
    return (p.k.data_ptr(), p.v.data_ptr(), p.k_exp.data_ptr(), p.v_exp.data_ptr(), 0 if w is None else w.data_ptr(), shape[0], shape[2], shape[1], shape[3])


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


@functools.lru_cache(4096)
def _scratch_floats(dev, *sizes) -> int:                             # (work is cut by the number of SMs of the device, which is the current one)
    return N.kernels().rb_e4m3_decode_scratch_floats(*sizes)


def _pitch(t: torch.Tensor) -> int:
    """The pitch of the rows of `t`, 0 where the kernels cannot read or write them 16 bytes at a time."""
    pitch, step = t.stride()
    return 0 if step != 1 or (t.data_ptr() | pitch * t.element_size()) & 15 else pitch


def _starts(what: str, row_starts, batch: int):
    if row_starts.dtype is not torch.int32 or row_starts.shape != (batch + 1,) or not row_starts.is_contiguous():
        raise TypeError(f"{what}: row_starts is int32 [batch + 1], the first row of every sequence and the end")


# ---- the same on the host ----------------------------------------------------------------------------------------------------------------
def exponent_e4m3(most: torch.Tensor) -> torch.Tensor:
    """The exponents of pages whose largest finite magnitudes are `most`."""
    m, x = torch.frexp(most.float())                                  # 448 = 0.875 * 2^9
    return torch.where(most > 0, x - 9 + (m > 0.875).to(x.dtype), LEAST_EXPONENT).clamp(LEAST_EXPONENT, MOST_EXPONENT)


def _encode(x: torch.Tensor, exp: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(x.double(), -exp.double()).clamp(-LARGEST_CODE, LARGEST_CODE).float().to(torch.float8_e4m3fn)


def _page(tables, num_blocks: int, b: int, i: int) -> int:
    """Page `i` of sequence b, -1 where the table has none or names one that is not there."""
    p = int(tables[b, i]) if i < tables.shape[1] else -1
    return p if 0 <= p < num_blocks else -1


def _put(codes, index, new) -> None:
    codes.view(torch.uint8)[index] = new.view(torch.uint8)


def _append_cpu(pages, k_new, v_new, tables, lens, starts) -> None:
    nb, G, bs, D = pages.k.shape
    for b in range(tables.shape[0]):
        first, last = (b, b + 1) if starts is None else (int(starts[b]), min(int(starts[b + 1]), k_new.shape[0]))
        pos0 = int(lens[b]) - ((b + 1 if starts is None else int(starts[b + 1])) - first)
        r = first + max(0, -pos0)
        while r < last:
            pos = pos0 + r - first
            off, i = pos % bs, pos // bs
            n = min(bs - off, last - r)
            page = _page(tables, nb, b, i)
            if page >= 0:
                for codes, exps, new in ((pages.k, pages.k_exp, k_new), (pages.v, pages.v_exp, v_new)):
                    x = new[r:r + n].float().reshape(n, G, D).transpose(0, 1)                       # [G, n, D]
                    e = exponent_e4m3(torch.where(x.isfinite(), x.abs(), 0.0).amax((1, 2)))
                    if off:
                        had = exps[page].int()
                        e = torch.maximum(e, had)
                        _put(codes, (page, slice(None), slice(0, off)), _encode(codes[page, :, :off].float(), (e - had)[:, None, None]))
                    _put(codes, (page, slice(None), slice(off, off + n)), _encode(x, e[:, None, None]))
                    exps[page] = e.to(torch.int8)
                if pages.weight is not None:
                    pages.weight[page, :, off:off + n] = 0.0
            r += n


def _values_cpu(codes, exps, tables, b: int, n: int) -> torch.Tensor:
    """Numbers [n, kv_heads, head_dim] of the first n tokens of sequence b; pages that are not there count as page 0."""
    bs = codes.shape[2]
    table = torch.tensor([max(_page(tables, codes.shape[0], b, i), 0) for i in range((n + bs - 1) // bs)], dtype=torch.long)
    x = torch.ldexp(codes.view(torch.uint8)[table].view(codes.dtype).float(), exps[table].float()[:, :, None, None])
    return x.transpose(1, 2).reshape(-1, codes.shape[1], codes.shape[3])[:n]


def _held(pages, tables, lens, b: int) -> int:
    return max(0, min(int(lens[b]), tables.shape[1] * pages.k.shape[2]))


# ---- the operators -------------------------------------------------------------------------------------------------------------------------
def kv_append_e4m3(pages: PagesE4M3, k_new, v_new, block_tables, context_lens, row_starts=None) -> None:
    """Stores new tokens.  k_new / v_new [rows, kv_heads * head_dim] (row-strided views allowed; bf16, fp16 or fp32): the last tokens of every
    sequence, of sequence b rows row_starts[b] to row_starts[b + 1] (int32 [batch + 1]; None: one row each).  `context_lens` counts them.

    A page whose first slot gets a token forgets what it held and takes its exponents from this call; in any other page an exponent grows if a
    new token asks for it, and the codes in front are rounded to it (exactly, but for those that become subnormal).  Rows whose position has no
    page are not stored.  The new tokens' weights become 0.  No two sequences of a call store into the same page."""
    shape = _check("kv_append_e4m3", pages, block_tables, context_lens, k_new, v_new, row_starts)
    batch, width = shape[4:]
    given, kind = k_new.shape, k_new.dtype
    rows = given[0]
    if kind not in _TYPES or v_new.dtype is not kind or given != (rows, shape[1] * shape[3]) or v_new.shape != given:
        raise TypeError("kv_append_e4m3: keys and values are [rows, kv_heads * head_dim] in bf16, fp16 or fp32")
    if row_starts is not None:
        _starts("kv_append_e4m3", row_starts, batch)
    elif rows != batch:
        raise ValueError(f"kv_append_e4m3: {rows} rows for {batch} sequences need row_starts")
    if not k_new.is_cuda:
        return _append_cpu(pages, k_new, v_new, block_tables, context_lens, row_starts)
    if rows == 0 or batch == 0 or width == 0:
        return
    ld_k, ld_v = _pitch(k_new), _pitch(v_new)
    if not ld_k:
        k_new, ld_k = k_new.clone(memory_format=torch.contiguous_format), given[1]
    if not ld_v:
        v_new, ld_v = v_new.clone(memory_format=torch.contiguous_format), given[1]
    a = _APPEND.pack(*_native(pages, shape), k_new.data_ptr(), v_new.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), _ptr(row_starts),
                     ld_k, ld_v, rows, batch, width, _TYPES[kind])
    N.check(N.kernels().rb_e4m3_append(a, N.stream_ptr()), "rb_e4m3_append")


def kv_read_e4m3(pages: PagesE4M3, block_tables, context_lens, row_starts, rows: int, dtype=torch.bfloat16, out=None):
    """Keys and values of whole sequences, (k, v) of [rows, kv_heads * head_dim] each: position i of sequence b in row row_starts[b] + i.
    bf16 and fp32 hold every number of a page exactly (fp16: those in its range).  `out`: a pair that receives them; rows that no position has
    stay as they are (in a pair made here: undefined)."""
    shape = _check("kv_read_e4m3", pages, block_tables, context_lens, row_starts, *(out or ()))
    nb, G, bs, D, batch, width = shape
    _starts("kv_read_e4m3", row_starts, batch)
    ld_k = ld_v = G * D
    if out is None:
        if dtype not in _TYPES:
            raise TypeError("kv_read_e4m3: rows in bf16, fp16 or fp32")
        k = pages.k.new_empty((rows, ld_k), dtype=dtype)
        v = torch.empty_like(k)
    else:
        k, v = out
        dtype = k.dtype
        if dtype not in _TYPES or v.dtype is not dtype or k.shape != (rows, ld_k) or v.shape != (rows, ld_k):
            raise TypeError("kv_read_e4m3: out is a pair of [rows, kv_heads * head_dim] in bf16, fp16 or fp32")
    if not k.is_cuda:
        for b in range(batch):
            first = int(row_starts[b])
            n = max(0, min(_held(pages, block_tables, context_lens, b), int(row_starts[b + 1]) - first, rows - first))
            there = [_page(block_tables, nb, b, i // bs) >= 0 for i in range(n)]
            for to, codes, exps in ((k, pages.k, pages.k_exp), (v, pages.v, pages.v_exp)):
                x = _values_cpu(codes, exps, block_tables, b, n).reshape(n, G * D).to(to.dtype)
                to[first:first + n][there] = x[there]
        return k, v
    if rows == 0 or batch == 0 or width == 0:
        return k, v
    if out is not None:
        ld_k, ld_v = _pitch(k), _pitch(v)
        if not (ld_k and ld_v):
            raise ValueError("kv_read_e4m3: rows of out start at multiples of 16 bytes")
    a = _READ.pack(*_native(pages, shape), k.data_ptr(), v.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), row_starts.data_ptr(),
                   ld_k, ld_v, rows, batch, width, _TYPES[dtype])
    N.check(N.kernels().rb_e4m3_read(a, N.stream_ptr()), "rb_e4m3_read")
    return k, v


def paged_attention_decode_e4m3(q, pages: PagesE4M3, block_tables, context_lens, scale: float | None = None, out=None, accumulate: bool = False):
    """Attention of one token per sequence over its pages; the token's own key is in them already.  q [batch, heads * head_dim] (row-strided
    views allowed; on a GPU bf16 or fp16), the same out.  A sequence of length 0 gets zeros.  With `accumulate` the weight of every cached token
    (`pages.weight`) grows by its softmax weights, summed over the query heads of its KV head; sequences that share a page must then not be in
    one call."""
    shape = _check("paged_attention_decode_e4m3", pages, block_tables, context_lens, q, out)
    nb, G, bs, D, B, width = shape
    given, kind = q.shape, q.dtype
    row = given[-1] if len(given) == 2 else 0
    if row == 0 or given[0] != B or row % (G * D):
        raise TypeError("paged_attention_decode_e4m3: q is [batch, heads * head_dim], a multiple of the KV heads")
    if accumulate and pages.weight is None:
        raise ValueError("paged_attention_decode_e4m3: these pages keep no weights")
    heads = row // D
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((B, row))
    elif out.dtype is not kind or out.shape != given or out.stride(1) != 1:
        raise TypeError("paged_attention_decode_e4m3: out is like q, with contiguous rows")
    if not q.is_cuda:
        for b in range(B):
            n = _held(pages, block_tables, context_lens, b)
            k = _values_cpu(pages.k, pages.k_exp, block_tables, b, n)
            v = _values_cpu(pages.v, pages.v_exp, block_tables, b, n)
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[b].float().view(G, heads // G, D), k) * scale, -1)
            out[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(-1)
            if accumulate:
                for i in range((n + bs - 1) // bs):
                    page = _page(block_tables, nb, b, i)
                    if page >= 0:
                        w = p[:, :, i * bs:(i + 1) * bs].sum(1)
                        pages.weight[page, :, :w.shape[1]] += w
        return out
    if kind is not torch.bfloat16 and kind is not torch.float16:
        raise TypeError("paged_attention_decode_e4m3: CUDA queries are bf16 or fp16")
    if B == 0:
        return out
    ld_q, step = q.stride()
    if step != 1:
        q, ld_q = q.contiguous(), row
    if width == 0:
        return out.zero_()
    floats = _scratch_floats(pages.k.get_device(), B, heads, G, D, width, bs, accumulate)
    scratch = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    a = _DECODE.pack(*_native(pages, shape), q.data_ptr(), out.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), _ptr(scratch),
                     ld_q, out.stride(0), B, width, heads, _TYPES[kind], accumulate, scale)
    N.check(N.kernels().rb_e4m3_decode(a, N.stream_ptr()), "rb_e4m3_decode")
    return out


def kv_evict_e4m3(pages: PagesE4M3, block_tables, context_lens, keep: int, recent: int = 0, keep_first: int = 0, out_tables=None):
    """Brings every sequence down to `keep` tokens.  A longer one keeps, for each KV head, its first `keep_first` tokens, its last `recent` and,
    of the others, those with the largest weights (`pages.weight`; of equal ones the earlier, NaN counts as largest).  They move, in their order and
    with their weights, to the front of the sequence's pages; what lies behind is free.  With `out_tables` (int32 [batch, width], pages that no
    sequence of `block_tables` has) every sequence moves there instead, also one that is short enough, and the old pages stay as they are; only
    then may sequences share pages.

    Returns (lengths int32 [batch], kept int32 [batch, kv_heads, keep]): the place that each token came from, -1 behind the last.

    A page's exponent becomes the largest of those that its tokens had; codes from smaller ones are rounded to it.  Attention does not ask for
    positions (keys are stored rotated), but a sequence's next position is no longer its length."""
    shape = _check("kv_evict_e4m3", pages, block_tables, context_lens, out_tables)
    _, G, bs, _, B, width = shape
    if pages.weight is None:
        raise ValueError("kv_evict_e4m3: these pages keep no weights")
    if keep < 1 or recent < 0 or keep_first < 0 or recent + keep_first > keep:
        raise ValueError("kv_evict_e4m3: keep must be at least 1 and at least recent + keep_first")
    out_width = 0
    if out_tables is not None:
        if not (out_tables.dtype is torch.int32 and out_tables.dim() == 2 and out_tables.shape[0] == B and out_tables.is_contiguous()):
            raise TypeError("kv_evict_e4m3: out_tables is a contiguous int32 table row per sequence")
        out_width = out_tables.shape[1]
        if out_width * bs < min(keep, width * bs):
            raise ValueError("kv_evict_e4m3: out_tables has no room for the tokens that may be kept")
    lens, kept = torch.empty_like(context_lens), context_lens.new_empty((B, G, keep))
    if not pages.k.is_cuda:
        _evict_cpu(pages, block_tables, context_lens, keep, recent, keep_first, out_tables, lens, kept)
        return lens, kept
    if B == 0:
        return lens, kept
    if width == 0:
        return lens.zero_(), kept.fill_(-1)
    a = _EVICT.pack(*_native(pages, shape), block_tables.data_ptr(), context_lens.data_ptr(), _ptr(out_tables), kept.data_ptr(), lens.data_ptr(),
                    B, width, out_width, keep, recent, keep_first)
    N.check(N.kernels().rb_e4m3_evict(a, N.stream_ptr()), "rb_e4m3_evict")
    return lens, kept


def _evict_cpu(pages, tables, context_lens, keep, recent, first, out_tables, lens, kept) -> None:
    nb, G, bs, D = pages.k.shape
    for b in range(tables.shape[0]):
        n = _held(pages, tables, context_lens, b)
        m = min(n, keep)
        lens[b], kept[b] = m, -1
        table = torch.tensor([max(_page(tables, nb, b, i), 0) for i in range((n + bs - 1) // bs)], dtype=torch.long)
        for h in range(G):
            places = torch.arange(m)
            if n > keep:
                order = torch.sort(pages.weight[table, h].reshape(-1)[first:n - recent], descending=True, stable=True).indices + first
                places = torch.cat([torch.arange(first), order[:m - first - recent].sort().values, torch.arange(n - recent, n)])
            kept[b, h, :m] = places
            if n <= keep and out_tables is None:
                continue
            page, off = table[places // bs], places % bs
            w = pages.weight[page, h, off]
            moved = [(codes, exps, codes.view(torch.uint8)[page, h, off].view(codes.dtype).float(), exps[page, h].int())
                     for codes, exps in ((pages.k, pages.k_exp), (pages.v, pages.v_exp))]
            for i in range(0, m, bs):
                to = _page(tables if out_tables is None else out_tables, nb, b, i // bs)
                if to < 0:
                    continue
                c = min(bs, m - i)
                for codes, exps, x, e in moved:
                    top = e[i:i + c].max()
                    _put(codes, (to, h, slice(0, c)), _encode(x[i:i + c], (top - e[i:i + c])[:, None]))
                    exps[to, h] = int(top)
                pages.weight[to, h, :c] = w[i:i + c]
