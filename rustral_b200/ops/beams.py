"""Several continuations of one prompt: selection of beams, states in the order of the selected, copied blocks of a cache, attention over what they share.

`beam_select` chooses the best continuations over beams and vocabulary.  What the chosen beams inherit moves in one of two ways: dense states (caches
[batch, ...], recurrent cells) take the selection's order in place with `reorder_rows_`; sequences of a paged cache share their full pages
(`serve.kv_cache.PagedCache.fork`) and only the page that is still filling is copied, in all layers by one `copy_blocks_`.  `paged_attention_shared` is
decode attention for sequences that share their first tokens, whose keys and values are then read once for all of them.
"""
from __future__ import annotations

import functools
import math
import struct
from array import array

import torch

from .. import _native as N

C = N.C
MOST_COUNT, MOST_BEAMS, MOST_GROUP, MOST_SEQUENCES = 128, 256, 256, 4096
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}

# The argument blocks of csrc/kernels/beam.h, move_rows.h and shared_prefix.h, packed
_SELECT = struct.Struct("@7Pq6i")                # logits, scores, ended, out scores, rows, tokens, scratch; pitch; groups, beams, vocab, count, type, end token
_MOVE = struct.Struct("@P4q2i")                  # base; outer, row and segment stride, segment bytes; outer, segments
_SHARED = struct.Struct("@10P3q9if")             # q, out, caches, tables, lengths, shared, group of, span of, scratch; pitches, blocks; sizes; scale

N.optional_sig("rb_beam_select", [C.c_char_p, N.c_void_p])
N.optional_sig("rb_beam_select_scratch_bytes", [N.c_int] * 5, N.c_ll)
N.optional_sig("rb_move_blocks", [C.c_char_p, N.c_int, N.c_void_p, N.c_void_p, N.c_int, N.c_int, N.c_void_p])
N.optional_sig("rb_move_reorder", [C.c_char_p, N.c_int, N.c_void_p, N.c_int, N.c_int, N.c_void_p])
N.optional_sig("rb_shared_prefix", [C.c_char_p, N.c_void_p])
N.optional_sig("rb_shared_prefix_scratch_bytes", [N.c_int] * 7, N.c_ll)
N._LAUNCHES["rb_beam_select"] = 2
N._LAUNCHES["rb_shared_prefix"] = 2


def _here(what: str, dev: int, *tensors) -> None:
    """All tensors are on the device `dev`, which on a GPU is the current one."""
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what}: tensors on different devices")
    if dev >= 0 and dev != torch._C._cuda_getDevice():
        raise ValueError(f"{what}: the tensors are not on the current device")


# ---- selection ---------------------------------------------------------------------------------------------------------------------------
@functools.lru_cache(4096)
def _select_bytes(dev, *sizes) -> int:                               # (work is cut by the number of SMs of the device, which is the current one)
    return N.kernels().rb_beam_select_scratch_bytes(*sizes)


def beam_select(logits, scores, count: int, ended=None, end_token: int = 0):
    """The `count` best continuations of every group of beams.  logits [groups * beams, vocab] (bf16, fp16 or fp32; row-strided views allowed, such as the
    real columns of a padded vocabulary), scores fp32 [groups, beams]: the sums of the beams' logarithmic probabilities.  Continuing row r by token t gives
    scores[r] + log_softmax(logits[r])[t].  Where `ended` (bool [groups, beams]) is true a beam has one continuation, `end_token` at its own score.

    Returns (scores fp32, rows int64, tokens int64), each [groups, count] in descending order of the scores; rows index `logits`.  Equal scores go to the lowest row,
    then the lowest token.  Sums are compared in 64 bits and rounded once.  Minus infinity is a token that is not allowed (or a beam that is not there), and NaN
    counts as that; plus infinity counts as the largest fp32 number.  Fewer continuations than `count`: the remaining places have minus infinity and the group's first
    (row, token) pairs that are not among the continuations.  A row's logits are compared as they are: of two so close that their 64-bit sums are equal either
    may come first.  A sum is as exact as its row's sum of exponentials, which is formed in 32 bits.  On a GPU: up to 256 beams and a count of up to 128."""
    # (Every look at a tensor counts in a small call: attributes are read once.)
    shape, each, kind = logits.shape, scores.shape, _TYPES.get(logits.dtype)
    if len(shape) != 2 or len(each) != 2 or kind is None or scores.dtype is not torch.float32 or not scores.is_contiguous():
        raise TypeError("beam_select: logits [groups * beams, vocab] in bf16, fp16 or fp32 and contiguous fp32 scores [groups, beams] are required")
    (rows, vocab), (groups, beams) = shape, each
    if rows != groups * beams or beams < 1 or vocab < 1:
        raise ValueError(f"beam_select: {rows} rows of {vocab} logits for {groups} groups of {beams} beams")
    if not 1 <= count <= beams * vocab:
        raise ValueError(f"beam_select: {count} of {beams} x {vocab} continuations")
    if ended is not None:
        if ended.dtype is not torch.bool or ended.shape != each or not ended.is_contiguous():
            raise TypeError("beam_select: ended is a contiguous bool tensor of the scores' shape")
        if not 0 <= end_token < vocab:
            raise ValueError(f"beam_select: no token {end_token} in a vocabulary of {vocab}")
    dev = logits.get_device()
    _here("beam_select", dev, scores, ended)
    if dev < 0:
        return _select_cpu(logits, scores, count, ended, end_token)
    if beams > MOST_BEAMS or count > MOST_COUNT or vocab > 1 << 26:
        raise ValueError(f"beam_select: up to {MOST_BEAMS} beams, a count of up to {MOST_COUNT} and 2^26 tokens are served")
    pitch, step = logits.stride()
    if step != 1 or pitch < vocab:
        logits, pitch = logits.contiguous(), vocab
    out_scores = scores.new_empty((groups, count))
    out_rows = scores.new_empty((groups, count), dtype=torch.int64)
    out_tokens = torch.empty_like(out_rows)
    scratch = scores.new_empty(_select_bytes(dev, groups, beams, vocab, count, kind), dtype=torch.uint8)
    N.check(N.kernels().rb_beam_select(
        _SELECT.pack(logits.data_ptr(), scores.data_ptr(), 0 if ended is None else ended.data_ptr(), out_scores.data_ptr(), out_rows.data_ptr(), out_tokens.data_ptr(),
                     scratch.data_ptr(), pitch, groups, beams, vocab, count, kind, end_token), N.stream_ptr()), "rb_beam_select")
    return out_scores, out_rows, out_tokens


def _clean(x):
    x = x.double()
    return torch.where(x.isnan(), -math.inf, x.clamp(max=torch.finfo(torch.float32).max))


def _select_cpu(logits, scores, count, ended, end_token):
    groups, beams = scores.shape
    x, s = _clean(logits), _clean(scores)
    most = x.amax(1, keepdim=True)
    x = x - torch.where(most == -math.inf, 0.0, most)
    total = s[..., None] + (x - x.exp().sum(1, keepdim=True).log()).view(groups, beams, logits.shape[1])
    total = torch.where(total.isnan(), -math.inf, total)               # rows without a token that is allowed
    if ended is not None:
        total = total.masked_fill(ended[..., None], -math.inf)
        total[:, :, end_token] = torch.where(ended, s, total[:, :, end_token])
    best = torch.sort(total.view(groups, beams * logits.shape[1]), dim=1, descending=True, stable=True)
    at, vocab = best.indices[:, :count], logits.shape[1]
    return best.values[:, :count].float(), torch.arange(groups)[:, None] * beams + at // vocab, at % vocab


# ---- moves -----------------------------------------------------------------------------------------------------------------------------------
def _row(what: str, t, dim: int) -> tuple:
    """(rows, and how they lie in memory: outer stride, row stride, segment stride, segment bytes, outer, segments) of the rows of `t` along `dim`, the bytes from the
    first to the last, and the same in runs (bytes of one, then (number, distance) from the widest distance down)."""
    shape, size = t.shape, t.element_size()
    if not 0 <= dim < len(shape):
        raise ValueError(f"{what}: a tensor of shape {tuple(shape)} has no rows along dimension {dim}")
    rows = shape[dim]
    if t.is_contiguous():
        row = math.prod(shape[dim + 1:]) * size
        n = math.prod(shape[:dim])
        return rows, (rows * row, row, 0, row, n, 1), n * rows * row, (n * rows * row, ())
    stride = t.stride()

    def merged(dims):
        """(length, stride) of these dimensions, neighbours that lie behind one another made one."""
        out = []
        for d in dims:
            if shape[d] == 1:
                continue
            if out and out[-1][1] == stride[d] * shape[d]:
                out[-1] = (out[-1][0] * shape[d], stride[d])
            else:
                out.append((shape[d], stride[d]))
        return out

    outer, inner = merged(range(dim)), merged(range(dim + 1, len(shape)))
    if inner and inner[-1][1] == 1:
        piece, inner = inner[-1][0], inner[:-1]
    else:
        piece = 1
    if len(outer) > 1 or len(inner) > 1 or any(s <= 0 for _, s in outer + inner) or (rows > 1 and stride[dim] <= 0):
        raise ValueError(f"{what}: the rows of a tensor of shape {tuple(shape)} and strides {tuple(stride)} are not pieces at equal distances")
    n, far = outer[0] if outer else (1, 0)
    segs, apart = inner[0] if inner else (1, 0)
    end, runs = piece, []
    for length, apart_ in sorted([(n, far), (rows, stride[dim] if rows > 1 else 0), (segs, apart)], key=lambda x: x[1]):
        if length > 1:
            runs.insert(0, (length, apart_ * size))
        if length > 1 and apart_ < end:
            raise ValueError(f"{what}: the rows of a tensor of shape {tuple(shape)} and strides {tuple(stride)} share memory")
        end += max(length - 1, 0) * apart_
    return rows, (far * size, (stride[dim] if rows > 1 else 0) * size, apart * size, piece * size, n, segs), end * size, (piece * size, tuple(runs))


def _meet(gap: int, run: int, many: tuple, run2: int, many2: tuple, looks: list) -> bool:
    """Whether two tensors share a byte, the second `gap` bytes behind the first: runs of `run` bytes, in turn repeated as `many` (number, distance) says from the widest down.
    Only repetitions whose extents meet are looked at; more than `looks` of them count as meeting."""
    far, far2 = (r + sum((n - 1) * s for n, s in m) for r, m in ((run, many), (run2, many2)))
    if gap >= far or -gap >= far2:
        return False
    if not many and not many2:
        return True
    looks[0] -= 1
    if looks[0] < 0:
        return True
    if many and many2 and many[0][1] == many2[0][1]:              # both go on at one distance: by the difference of the two numbers
        (n, s), (n2, _) = many[0], many2[0]
        near, near2 = far - (n - 1) * s, far2 - (n2 - 1) * s
        return any(_meet(gap + k * s, run, many[1:], run2, many2[1:], looks) for k in range(max(1 - n, -((near2 + gap - 1) // s)), min(n2 - 1, (near - gap - 1) // s) + 1))
    if not many or (many2 and many2[0][1] > many[0][1]):
        return _meet(-gap, run2, many2, run, many, looks)
    n, s = many[0]
    near = far - (n - 1) * s
    return any(_meet(gap - i * s, run, many[1:], run2, many2, looks) for i in range(max(0, -((near - gap - 1) // s)), min(n - 1, (gap + far2 - 1) // s) + 1))


def _apart(what: str, spans: list) -> None:
    """Refuses tensors that share memory.  spans: (first address, behind the last, runs) of each."""
    spans.sort()
    behind = 0
    for at, end, _ in spans:
        if at < behind:
            break
        behind = end
    else:
        return
    together, behind = [], 0                                      # those whose extents meet
    for span in spans:
        if span[0] >= behind:
            together.append([])
        together[-1].append(span)
        behind = max(behind, span[1])
    for some in together:
        wide = {many[0][1] if many else 0 for _, _, (_, many) in some}
        if len(wide) == 1 and 0 not in wide:                      # parts of one tensor's rows, as a rule: their places within a row do not meet
            s = wide.pop()
            places = sorted((at % s, at % s + end - at - (many[0][0] - 1) * s) for at, end, (_, many) in some)
            if all(a[1] <= b[0] for a, b in zip(places, places[1:])) and places[-1][1] <= places[0][0] + s:
                continue
        for i, (at, end, (run, many)) in enumerate(some):
            for at2, _, (run2, many2) in some[i + 1:]:
                if at2 >= end:
                    break
                if _meet(at2 - at, run, many, run2, many2, [4096]):
                    raise ValueError(f"{what}: tensors that share memory")


def _listed(what: str, tensors) -> tuple:
    if isinstance(tensors, torch.Tensor):
        raise TypeError(f"{what}: a list of tensors is required")
    return tuple(tensors)


def _rows(what: str, tensors, dim: int, index=None) -> tuple:
    """(device, rows, packed descriptions, how many) of the tensors of a call; those without elements are left out."""
    dev = rows = None
    packed, spans, behind, ascending = [], [], 0, True            # (tensors made one after the other lie so, as a rule)
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled() and (t.is_leaf or t._base is not None and t._base.is_leaf):
            raise ValueError(f"{what}: a leaf that requires a gradient is not written in place")
        d = t.get_device()
        n, lies, extent, runs = _row(what, t, dim)
        if dev is None:
            dev, rows = d, n
        elif dev != d:
            raise ValueError(f"{what}: tensors on different devices")
        elif rows != n:
            raise ValueError(f"{what}: tensors of {rows} and of {n} rows")
        if n and lies[3] and lies[4]:
            at = t.data_ptr()
            end = at + extent
            ascending &= at >= behind
            behind = end
            spans.append((at, end, runs))
            packed.append(_MOVE.pack(at, *lies))
    if index is not None:
        at, size = index.data_ptr(), index.numel() * index.element_size()
        ascending &= at >= behind or (bool(spans) and at + size <= spans[0][0])
        spans.append((at, at + size, (size, ())))
    if not ascending:
        _apart(what, spans)
    if dev is not None and dev >= 0 and dev != torch._C._cuda_getDevice():
        raise ValueError(f"{what}: the tensors are not on the current device")
    return dev, rows, b"".join(packed), len(packed)


def copy_blocks_(tensors, src, dst, dim: int = 0) -> None:
    """Copies blocks in place: t[dst[i]] <- t[src[i]] along dimension `dim` of every tensor (one number of blocks for all of them; other sizes, types and strides may
    differ).  src and dst are numbers on the host (lists or the like); the call refuses blocks that are not there, a destination twice, and a destination that is a source
    too, tensors that share memory, and (where gradients are recorded) leaves that require one, before it copies anything.  No gradient follows the rows.  A CUDA graph keeps the numbers that it was captured with."""
    tensors = _listed("copy_blocks_", tensors)
    if isinstance(src, (bytes, bytearray)) or isinstance(dst, (bytes, bytearray)):          # their bytes would be taken for those of the numbers
        raise ValueError("copy_blocks_: src and dst are lists of block numbers")
    try:
        src, dst = array("i", src), array("i", dst)
    except (TypeError, OverflowError) as e:
        raise ValueError("copy_blocks_: src and dst are lists of block numbers") from e
    if len(src) != len(dst):
        raise ValueError(f"copy_blocks_: {len(src)} sources and {len(dst)} destinations")
    dev, rows, packed, count = _rows("copy_blocks_", tensors, dim)
    if rows is None:
        return
    if dev >= 0:
        code = N.kernels().rb_move_blocks(packed, count, src.buffer_info()[0], dst.buffer_info()[0], len(src), rows, N.stream_ptr())
    else:
        code = -2 if src and not (0 <= min(src) and max(src) < rows and 0 <= min(dst) and max(dst) < rows) else \
            -3 if len(set(dst)) != len(dst) else 0 if set(dst).isdisjoint(src) else -4
    if code in _BLOCKS_REFUSED:
        raise ValueError("copy_blocks_: " + _BLOCKS_REFUSED[code])
    if dev >= 0:
        N.check(code, "rb_move_blocks")
    elif src:
        of, to = torch.tensor(src, dtype=torch.int64), torch.tensor(dst, dtype=torch.int64)
        for t in tensors:
            bits = _bits(t)
            bits.index_copy_(dim, to, bits.index_select(dim, of))


_BLOCKS_REFUSED = {-2: "a block that is not there", -3: "a destination twice", -4: "a destination that is a source too"}


def _bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 and t.dtype is not torch.bool else t


def reorder_rows_(tensors, index, dim: int = 0, group: int | None = None) -> None:
    """Rows in a new order, in place: t[i] <- what t[index[i]] was, along dimension `dim` of every tensor (one number of rows for all; other sizes, types and strides
    may differ).  index: int64 [rows] on the tensors' device, any map.  `group`: rows come in groups of that many, as the beams of several prompts do, and indices stay
    in their row's group (None: all rows are one); an index that does not leaves its row as it is.  On a GPU a group has up to 256 rows.  Tensors that share
    memory, with the index too, are refused, and so are leaves that require a gradient where gradients are recorded; no gradient follows the rows."""
    tensors = _listed("reorder_rows_", tensors)
    dev, rows, packed, count = _rows("reorder_rows_", tensors, dim, index)
    if rows is None:
        return
    if index.dtype is not torch.int64 or index.dim() != 1 or not index.is_contiguous():
        raise TypeError("reorder_rows_: index is a contiguous int64 vector")
    if index.shape[0] != rows:
        raise ValueError(f"reorder_rows_: {index.shape[0]} indices for {rows} rows")
    group = max(rows, 1) if group is None else group
    if group < 1 or rows % group:
        raise ValueError(f"reorder_rows_: {rows} rows in groups of {group}")
    if index.get_device() != dev:
        raise ValueError("reorder_rows_: tensors on different devices")
    if dev < 0:
        first = torch.arange(rows) // group * group
        safe = torch.where((index >= first) & (index < first + group), index, torch.arange(rows))
        for t in tensors:
            bits = _bits(t)
            bits.copy_(bits.index_select(dim, safe))
        return
    if group > MOST_GROUP:
        raise ValueError(f"reorder_rows_: groups of up to {MOST_GROUP} rows are served")
    if rows and count:
        N.check(N.kernels().rb_move_reorder(packed, count, index.data_ptr(), rows, group, N.stream_ptr()), "rb_move_reorder")


# ---- attention over a shared prefix ------------------------------------------------------------------------------------------------------------
class PrefixGroups:
    """Which sequences of a batch share their first tokens: group i is the next `sizes[i]` sequences.  A program keeps one for as long as the batch is made up
    like this; the lengths are tensors of the calls."""

    def __init__(self, sizes, device="cpu"):
        self.sizes = tuple(int(n) for n in sizes)
        if any(n < 1 for n in self.sizes):
            raise ValueError("PrefixGroups: every group has a sequence")
        self.batch, self.most = sum(self.sizes), max(self.sizes, default=0)
        starts = [0]
        for n in self.sizes:
            starts.append(starts[-1] + n)
        span_of = [x for g, n in enumerate(self.sizes) for x in (starts[g], starts[g + 1]) * n]
        both = torch.tensor(span_of + [g for g, n in enumerate(self.sizes) for _ in range(n)], dtype=torch.int32).to(device)
        self.span_of, self.group_of = both[:2 * self.batch], both[2 * self.batch:]
        self.at = (self.group_of.data_ptr(), self.span_of.data_ptr())

    def __len__(self) -> int:
        return len(self.sizes)


@functools.lru_cache(4096)
def _shared_bytes(dev, *sizes) -> int:                               # (as for _select_bytes)
    return N.kernels().rb_shared_prefix_scratch_bytes(*sizes)


def shared_supported(q, k_cache, v_cache) -> bool:
    """Whether `paged_attention_shared` takes these operands (q [batch, heads * head_dim])."""
    if not q.is_cuda:
        return True
    return q.dtype in (torch.bfloat16, torch.float16) and q.dtype is k_cache.dtype is v_cache.dtype and k_cache.shape == v_cache.shape and \
        k_cache.shape[3] in (64, 128) and k_cache.is_contiguous() and v_cache.is_contiguous() and q.shape[0] <= MOST_SEQUENCES


def shared_pays(groups: PrefixGroups, shared_lens, row_bytes: int) -> bool:
    """Whether reading the shared tokens once saves more than the further launches cost.  `row_bytes`: of a token's keys and values."""
    return row_bytes * sum((n - 1) * p for n, p in zip(groups.sizes, shared_lens)) >= SHARED_PAYS


# Bytes that are not read again.  One B200, attention of a layer, us, every sequence's own reading / one for the group: 4 beams over 300 tokens (12 KV heads of 64; 3 MB) 7.6 / 11.3,
# 4 over 1000 (8 KV heads of 128; 12 MB) 7.5 / 15.2, 8 over 1000 (29 MB) 12.4 / 18.9, 4 over 4000 (49 MB) 21.4 / 17.9, 4 times 4 over 1000 (49 MB) 20.2 / 17.7, 16 over 1000
# (61 MB) 21.5 / 19.9, 2 over 16000 (66 MB) 43.7 / 22.3, 8 over 4000 (115 MB) 38.1 / 21.1, 32 over 2000 (254 MB) 59.8 / 22.5.
SHARED_PAYS = 48_000_000


def paged_attention_shared(q, k_cache, v_cache, groups: PrefixGroups, shared_lens, block_tables, context_lens, scale=None, out=None):
    """Decode attention for sequences that share their first tokens.  q [batch, heads * head_dim] (row-strided views allowed); caches
    [blocks, block_size, kv_heads, head_dim]; block_tables int32 [batch, width], context_lens int32 [batch] as for decode attention; shared_lens int32
    [groups]: the first tokens of a group's sequences that are the same.  Those are read once for the whole group, through the table of its first sequence, what follows through
    each sequence's own.  Where the shortest sequence of a group has fewer tokens (those without any aside) only that many count as shared.  A sequence without tokens
    gets zeros.  Returns [batch, heads * head_dim].

    On a GPU: bf16 or fp16, heads of 64 or 128, up to 4096 sequences (a batch of more than 704, pages that neither divide 128
    tokens nor hold a whole number of 128, and scales that are not positive go to the kernel for few rows: 478 us for a group of 705 where 704 take 137).  Where less than SHARED_PAYS bytes are saved, decode attention over every sequence's tokens is the faster call (`shared_pays`).  A sequence's result depends, within rounding, on the batch it is in; the same call gives the
    same bits."""
    qs, ks, dtype = q.shape, k_cache.shape, q.dtype
    if len(qs) != 2 or len(ks) != 4 or ks != v_cache.shape or not dtype is k_cache.dtype is v_cache.dtype or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise TypeError("paged_attention_shared: q [batch, heads * head_dim] and contiguous caches [blocks, block_size, kv_heads, head_dim] of its type are required")
    nb, bs, hk, d = ks
    batch, width = qs
    heads, n_groups = width // d, len(groups.sizes)
    if batch != groups.batch or width != heads * d or heads % hk or heads == 0:
        raise ValueError(f"paged_attention_shared: q of {tuple(qs)} for {groups.batch} sequences and {hk} KV heads of {d}")
    table = block_tables.shape
    if not (block_tables.dtype is context_lens.dtype is shared_lens.dtype is torch.int32 and len(table) == 2 and block_tables.is_contiguous() and
            context_lens.is_contiguous() and shared_lens.is_contiguous()) or \
            not (table[0] == batch and context_lens.shape == (batch,) and shared_lens.shape == (n_groups,)):
        raise TypeError("paged_attention_shared: contiguous int32 tables and lengths of every sequence and shared lengths of every group are required")
    if out is not None and (out.dtype is not dtype or out.shape != qs):
        raise TypeError("paged_attention_shared: out has the shape and type of q")
    if out is not None and batch > 1 and out.stride(1) in (0, 1) and out.stride(0) < width:
        raise ValueError("paged_attention_shared: the rows of out share memory")
    dev = q.get_device()
    _here("paged_attention_shared", dev, k_cache, v_cache, groups.group_of, shared_lens, block_tables, context_lens, out)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    if dev < 0:
        r = _shared_cpu(q, k_cache, v_cache, groups, shared_lens, block_tables, context_lens, scale)
        return r if out is None else out.copy_(r)
    kind = _TYPES.get(dtype, 3)
    if kind > 1 or d not in (64, 128) or batch > MOST_SEQUENCES:
        raise ValueError(f"paged_attention_shared: bf16 or fp16, heads of 64 or 128 and up to {MOST_SEQUENCES} sequences are served, not {dtype}, {d} and {batch}")
    if batch == 0 or table[1] == 0 or nb == 0 or bs == 0:
        return torch.zeros_like(q) if out is None else out.zero_()
    if nb * bs > 2 ** 31 - 1 or table[1] * bs > 1 << 30:
        raise ValueError("paged_attention_shared: caches of fewer than 2^31 tokens and tables of up to 2^30 are served")
    at, (pitch, step) = q.data_ptr(), q.stride()
    if step != 1 or pitch < width or pitch & 7 or at & 15:           # (rows that overlap, as of an expanded one, are nothing that a tensor map describes)
        q = q.clone(memory_format=torch.contiguous_format)
        at, pitch = q.data_ptr(), width
    res = out
    if out is None or out.stride(1) != 1 or out.stride(0) & 7 or out.data_ptr() & 15:
        res = q.new_empty((batch, width))
    scratch = q.new_empty(_shared_bytes(dev, batch, n_groups, heads, hk, d, bs, groups.most), dtype=torch.uint8)
    N.check(N.kernels().rb_shared_prefix(
        _SHARED.pack(at, res.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), shared_lens.data_ptr(), groups.at[0], groups.at[1],
                     scratch.data_ptr(), pitch, res.stride(0), nb, batch, n_groups, table[1], bs, heads, hk, d, kind, groups.most, scale), N.stream_ptr()), "rb_shared_prefix")
    return res if out is None or res is out else out.copy_(res)


def _shared_cpu(q, k_cache, v_cache, groups, shared_lens, block_tables, context_lens, scale):
    nb, bs, hk, d = k_cache.shape
    batch, heads = q.shape[0], q.shape[1] // d
    out = torch.zeros(batch, heads * d)
    cap, first = block_tables.shape[1] * bs, 0
    for g, size in enumerate(groups.sizes):
        lens = [min(max(int(n), 0), cap) for n in context_lens[first:first + size]]
        shared = min([max(int(shared_lens[g]), 0)] + [n for n in lens if n])
        for b, n in enumerate(lens, first):
            if n == 0:
                continue
            at = torch.arange(n)
            pages = torch.where(at < shared, block_tables[first, at // bs], block_tables[b, at // bs]).long()
            pages = torch.where((pages >= 0) & (pages < nb), pages, 0)
            k, v = (t[pages, at % bs].float() for t in (k_cache, v_cache))          # [n, kv heads, d]
            s = torch.einsum("hgd,nhd->hgn", q[b].float().view(hk, -1, d), k) * scale
            out[b] = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(-1)
        first += size
    return out.to(q.dtype)
