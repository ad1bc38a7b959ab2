"""A paged cache that holds keys and values in 4 bits: append with norms and rotation, read back, attention.

Rows of a head are held in groups of 32 elements: ``m`` (the smallest) and ``s`` (a fifteenth of the range) in bfloat16 and a
4-bit code each, value = m + s * code: 5 bits an element, 3.2 times as many positions in the same memory as bfloat16 holds.  One
layer's pages are uint8 [pages, 2 (keys, values), kv heads, page_size / 8, 160 * head_dim / 32] (csrc/kv4.h has the layout).

``store``   the tail of a q/k/v projection: norm and rotation of q and k, queries out, keys and values into the pages
``read``    rows of requests as ordinary pages of bfloat16 or float32
``attend``  causal attention of a step's tokens over the pages, which hold the step's own keys and values already

Queries and outputs are bfloat16 or float32; head sizes 32, 64, ..., 256; page sizes of a multiple of 8.  Like everything in this
package the functions launch on torch's current stream, on the current device, and return without waiting.
"""
from __future__ import annotations

import functools
from ctypes import c_char_p, c_int
from struct import Struct
from typing import NamedTuple

import numpy as np
import torch

from . import attention_f32, attention_mma, attention_tc, build, ops, tuning
from .ops import F32, KernelError, _check, _need, dtype_code

GROUP = 32
MOST_DIM = 256
PLAN_KEY = "kv4_attention"        # the step planner whose arrays ``attend`` reads (``describe_segments`` makes them)
#: Rows (tokens of a segment times query heads of a kv head) up to which the kernel that walks the codes takes more than one token; of
#: more the rows are read back once and attended to as 16-bit pages.  Measured (us, this kernel / the other one; 4 heads of 128 a kv head; of
#: 2, 4, 8, 12, 16 tokens): 8 segments behind 4000 20 / 74, 35 / 74, 59 / 75, 61 / 76, 102 / 77; one 11 / 26, 14 / 26, 18 / 26, 19 / 27, 23 / 27; 8
#: behind 500 8 / 21, 13 / 21, 17 / 21, 18 / 21, 23 / 23; 4 behind 16000 32 / 134, 61 / 134, 87 / 135, 117 / 135, 151 / 135.
FEW_ROWS = 48
#: Tokens of a segment up to which the 32-bit path takes them one by one.
FEW_TOKENS = 8
#: Positions per page of rows that are read back for a portion, and the most of them at a time (of several portions; a single
#: one may be longer): 8 heads of 128 in bfloat16 take 4 KB a position.
READ_PAGE, MOST_READ = 64, 1 << 16
#: The last position that the kernels count to: a tile behind it is a 32-bit number yet.
MOST_POSITION = 2**31 - 1 - 1024
#: Bytes that the memory for those rows grows by at most beyond what is asked for.
MOST_GROWTH = 256 << 20

SOURCES, DEPENDS = ["kv4_store.cu", "kv4_attention.cu"], ["kv4.h"]
_lib = None
_few_libs: dict = {}


# The C entries' arguments, packed: pointers, then 32-bit numbers (the structs beside the entries), padded to whole pointers.
_STORE, _READ, _SPREAD, _SINGLES, _FEW = (Struct(f"@{form}0P") for form in ("Pq10P2f17i", "5P11i", "8P11i", "9Pf10i", "9Pf13i"))


def _entry(lib, name, struct, size):
    """A C entry that takes ``struct``."""
    if size != struct.size:
        raise KernelError(f"{name} takes {size} bytes of arguments, not {struct.size}")
    entry = getattr(lib, name)
    entry.argtypes = [c_char_p]


def few_library_name(head_dim):
    """(name, defines) of the tensor-core library for heads of ``head_dim``."""
    return f"qil_kv4_d{head_dim}", {"QIL_HEAD_DIM": head_dim}


def few_library(head_dim):
    """(the library, its most spans, blocks an SM takes by tiles of rows) for heads of ``head_dim``."""
    held = _few_libs.get(head_dim)
    if held is None:
        name, defines = few_library_name(head_dim)
        lib = build.load(name, ["kv4_attention_mma.cu"], defines, depends=DEPENDS)
        if lib.qil_kv4_few_head_dim() != head_dim:
            raise KernelError("the 4-bit attention library was built for another head size")
        _entry(lib, "qil_kv4_few", _FEW, lib.qil_kv4_few_call_bytes())
        held = _few_libs[head_dim] = (lib, lib.qil_kv4_few_most_spans(), {nt: lib.qil_kv4_few_blocks_a_sm(c_int(nt)) for nt in (1, 2)})
    return held


def library():
    global _lib
    if _lib is None:
        lib = build.load("qil_kv4", SOURCES, depends=DEPENDS)
        for which, (name, struct) in enumerate((("qil_kv4_store", _STORE), ("qil_kv4_read", _READ), ("qil_kv4_spread", _SPREAD))):
            _entry(lib, name, struct, lib.qil_kv4_call_bytes(which))
        _entry(lib, "qil_kv4_singles", _SINGLES, lib.qil_kv4_singles_call_bytes())
        _lib = lib
    return _lib


def _at(tensor):
    return tensor.data_ptr() if tensor is not None else 0


_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)        # of a device


def _take(tensor, name, dtype, ndim, device):
    """``ops._need`` with what every call here asks, and the device: quick where all is well."""
    try:
        if tensor.dtype is dtype and tensor.get_device() == device and tensor.dim() == ndim and tensor.is_contiguous():
            return
    except AttributeError:
        pass
    _need(tensor, name, dtype, ndim)
    raise KernelError(f"{name} is on {tensor.device} while the current device is cuda:{device}")


def _device_of(tensor, name):
    """The current device, which ``tensor`` is on: a launch goes to its stream."""
    if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
        _need(tensor, name)
    device = tensor.get_device()
    if device != torch._C._cuda_getDevice():
        raise KernelError(f"{name} is on {tensor.device} while the current device is cuda:{torch._C._cuda_getDevice()}")
    return device


def supports(head_dim, page_size) -> bool:
    return head_dim % GROUP == 0 and 0 < head_dim <= MOST_DIM and page_size % 8 == 0 and page_size > 0


def page_shape(n_kv_heads, head_dim, page_size) -> tuple:
    """The shape of one page: multiply it out for its bytes."""
    if not supports(head_dim, page_size):
        raise KernelError(f"4-bit pages take head sizes 32, 64, ..., {MOST_DIM} and a multiple of 8 positions, not heads of {head_dim} "
                          f"and {page_size} positions")
    return (2, int(n_kv_heads), page_size // 8, 160 * (head_dim // GROUP))


def _check_pages(pages, n_kv_heads, head_dim, page_size, what, device):
    _take(pages, "pages", torch.uint8, 5, device)
    if pages.shape[1:] != page_shape(n_kv_heads, head_dim, page_size):
        raise KernelError(f"{what}: cache layout {tuple(pages.shape)} for {n_kv_heads} heads of {head_dim}, pages of {page_size}")
    if pages.data_ptr() % 16:
        raise KernelError(f"{what}: pages must start on a 16-byte boundary")


def store(proj, columns, q_out, pages, positions, token_row, block_table, n_q_heads, n_kv_heads, head_dim, page_size, *,
          q_norm_w=None, k_norm_w=None, eps=0.0, unit_heads=False, table=None, freq=None, rot_dims=0, layout=0, gain=1.0):
    """The tail of a q/k/v projection into 4-bit pages.

    ``proj`` [N, width] holds q, k, v from the columns ``columns`` = (q, k, v) on.  With ``q_norm_w`` and ``k_norm_w`` [head_dim] every q
    and k head is divided by its root mean square and multiplied by the weight; ``unit_heads``: divided by it after the turn, without
    a weight.  The first ``rot_dims`` dimensions of q and k heads are turned, paired by ``layout`` (``ops.ROTARY_HALVES`` or
    ``ops.ROTARY_INTERLEAVED``), by ``table`` float32 [positions, rot_dims] (cosines, then sines; a position beyond it turns as its
    last) or by ``freq`` float32 [rot_dims / 2]: angle = position * freq, in 64 bits, cosines and sines times ``gain``.  Queries go to
    ``q_out`` [N, n_q_heads * head_dim], rounded once; keys (64-bit arithmetic until they are coded) and values go to the token's page.  A
    token whose position has no page writes none.  Two tokens of one call must not share a position of a request.  With n_kv_heads ==
    0 only queries are processed (``pages`` and ``block_table`` may be None)."""
    device = _device_of(proj, "proj")
    dtype = proj.dtype
    act = dtype_code(dtype)
    _take(proj, "proj", dtype, 2, device); _take(q_out, "q_out", dtype, 2, device)
    _take(positions, "positions", torch.int32, 1, device); _take(token_row, "token_row", torch.int32, 1, device)
    n, width = proj.shape
    q_at, k_at, v_at = columns
    if n_q_heads < 1 or n_kv_heads < 0 or not supports(head_dim, page_size):
        raise KernelError(f"kv4.store: {n_q_heads} and {n_kv_heads} heads of {head_dim}, pages of {page_size}")
    q_width, k_width = n_q_heads * head_dim, n_kv_heads * head_dim
    if min(q_at, k_at, v_at) < 0 or q_out.shape != (n, q_width) or positions.shape[0] < n or token_row.shape[0] < n \
            or max(q_at + q_width, k_at + k_width, v_at + k_width) > width:
        raise KernelError("kv4.store: shapes do not match the head counts")
    table_height = table_width = num_pages = table_rows = 0
    if n_kv_heads:
        _check_pages(pages, n_kv_heads, head_dim, page_size, "kv4.store", device)
        _take(block_table, "block_table", torch.int32, 2, device)
        num_pages, (table_height, table_width) = pages.shape[0], block_table.shape
    else:
        pages = block_table = None
    norm, norm_code = 0, F32
    if q_norm_w is not None or k_norm_w is not None:
        if unit_heads:
            raise KernelError("kv4.store: heads of unit size have no norm weights")
        if not isinstance(q_norm_w, torch.Tensor):
            _need(q_norm_w, "q_norm_w")
        norm, norm_code = 1, dtype_code(q_norm_w.dtype)
        for weight, name in ((q_norm_w, "q_norm_w"), (k_norm_w, "k_norm_w")):
            _take(weight, name, q_norm_w.dtype, 1, device)
            if weight.shape[0] != head_dim:
                raise KernelError("kv4.store: norm weights must have head_dim elements")
    elif unit_heads:
        norm = 2
    if rot_dims % 2 or not 0 <= rot_dims <= head_dim or layout not in (ops.ROTARY_HALVES, ops.ROTARY_INTERLEAVED):
        raise KernelError(f"kv4.store: {rot_dims} rotated dimensions of {head_dim}, layout {layout}")
    if rot_dims:
        if (table is None) == (freq is None):
            raise KernelError("kv4.store: a rotation comes from a table or from frequencies")
        if table is not None:
            _take(table, "table", torch.float32, 2, device)
            table_rows = table.shape[0]
            if table.shape[1] != rot_dims or table_rows < 1 or gain != 1.0:
                raise KernelError("kv4.store: a table holds rot_dims columns, a gain included")
        else:
            _take(freq, "freq", torch.float32, 1, device)
            if freq.shape[0] != rot_dims // 2:
                raise KernelError("kv4.store: one frequency per rotated pair")
    else:
        table = freq = None
    if n == 0:
        return q_out
    lib = library()
    _check(lib, lib.qil_kv4_store(_STORE.pack(
        proj.data_ptr(), width, q_out.data_ptr(), _at(pages), _at(q_norm_w), _at(k_norm_w), _at(table), _at(freq), positions.data_ptr(),
        token_row.data_ptr(), _at(block_table), _stream(device), eps, gain, q_at, k_at, v_at, norm, table_rows, rot_dims, layout, table_height,
        table_width, n, n_q_heads, n_kv_heads, head_dim, page_size, num_pages, act, norm_code)), "kv4.store")
    return q_out


def read(pages, block_table, info, segments, longest, out, n_kv_heads, head_dim, page_size):
    """The values that rows of 4-bit pages stand for, as ordinary pages ``out`` [pages, 2, kv heads, positions a page, head_dim] of
    bfloat16 or float32 (positions a page need not be ``page_size``).

    ``info`` int32 [segments * 4]: (block-table row, first position, positions, first page of ``out``) a segment; ``longest``: no segment
    has more positions.  Position first + i goes to slot i % (positions a page) of page i // (positions a page) after the segment's
    first.  Positions without a page are read as zeros; slots behind a segment's last position are left as they are."""
    device = _device_of(pages, "pages")
    _check_pages(pages, n_kv_heads, head_dim, page_size, "kv4.read", device)
    _take(block_table, "block_table", torch.int32, 2, device); _take(info, "info", torch.int32, 1, device)
    if not isinstance(out, torch.Tensor):
        _need(out, "out")
    act = dtype_code(out.dtype)
    _take(out, "out", out.dtype, 5, device)
    if info.shape[0] < 4 * segments or segments < 0 or info.data_ptr() % 16:
        raise KernelError("kv4.read: four numbers a segment, from a 16-byte boundary on")
    out_pages, planes, heads, out_page_size, dim = out.shape
    if planes != 2 or heads != n_kv_heads or dim != head_dim or out.data_ptr() % 16:
        raise KernelError(f"kv4.read: output {tuple(out.shape)} for {n_kv_heads} heads of {head_dim}")
    if segments == 0 or longest <= 0 or out_pages * out_page_size == 0:
        return out
    lib = library()
    _check(lib, lib.qil_kv4_read(_READ.pack(
        pages.data_ptr(), block_table.data_ptr(), info.data_ptr(), out.data_ptr(), _stream(device), *block_table.shape, segments, longest, out_pages,
        out_page_size, n_kv_heads, head_dim, page_size, pages.shape[0], act)), "kv4.read")
    return out


# ------------------------------------------------------------------ the plan of a step
def _one_by_one(first, starts, lens, rows, indices):
    """The tokens of the segments ``indices``, four ints each: (token, its position, block-table row, the longest context among these)."""
    if not len(indices):
        return np.zeros(0, dtype=np.int64)
    of = np.repeat(indices, lens[indices])
    offset = np.arange(len(of)) - np.repeat(np.cumsum(lens[indices]) - lens[indices], lens[indices])
    return np.stack([first[of] + offset, starts[of] + offset, rows[of], np.full_like(of, (starts + lens)[indices].max())], axis=1).reshape(-1)


def describe_segments(first, starts, lens, rows, portion_tokens=True) -> dict:
    """A step's segments as ``attend`` wants them (numpy int64 arrays in, one entry per segment: first token in the flat batch,
    its absolute position, tokens, block-table row).

    ``singles``, ``few``, ``multi``  the segments of one token, of 2 to FEW_ROWS and of any more than one: eight ints each, (first token, its
                        position, tokens, block-table row, tokens of the segments before in this array, the longest context among these, 0, 0)
    ``single_tokens``, ``few_tokens``, ``portion_tokens``  the segments of one token, of 2 to FEW_TOKENS and the others token by token
                        (``_one_by_one``); the last are read by float32 attention with heads that the tile kernel does not take only, and are
                        left out where ``portion_tokens`` is False
    ``b0.spread`` ...   the segments of more than one token in batches whose contexts are read back together: (block-table row, first position,
                        end, first page); ``kv4.read``'s info of those beyond FEW_TOKENS; the block table of the pages they are read to; the
                        segments, and tiles of 64 of their tokens beyond FEW_TOKENS, over that table: (first token, its position, tokens, row of it)
    """
    lens, starts = np.asarray(lens, dtype=np.int64), np.asarray(starts, dtype=np.int64)
    first, rows = np.asarray(first, dtype=np.int64), np.asarray(rows, dtype=np.int64)
    ends = starts + lens

    def segments(indices):
        if not len(indices):
            return np.zeros(0, dtype=np.int64)
        before = np.cumsum(lens[indices]) - lens[indices]
        none = np.zeros_like(before)
        return np.stack([first[indices], starts[indices], lens[indices], rows[indices], before, none + ends[indices].max(), none, none], axis=1).reshape(-1)

    arrays = {}
    for name, some in (("singles", lens == 1), ("few", (lens > 1) & (lens <= FEW_ROWS)), ("multi", lens > 1)):
        arrays[name] = segments(np.nonzero(some)[0])
    for name, some in (("single_tokens", lens == 1), ("few_tokens", (lens > 1) & (lens <= FEW_TOKENS)), ("portion_tokens", lens > FEW_TOKENS)):
        if portion_tokens or name != "portion_tokens":
            arrays[name] = _one_by_one(first, starts, lens, rows, np.nonzero(some)[0])
    for batch, taken in enumerate(portion_batches(starts, lens)):
        width = -(-int(ends[taken[0]]) // READ_PAGE)               # pages a segment: of the longest, so that segment i's begin at i * width
        local = np.arange(len(taken), dtype=np.int64)
        counts = np.where(lens[taken] > FEW_TOKENS, ends[taken], 0)
        arrays[f"b{batch}.read"] = np.stack([rows[taken], np.zeros_like(local), counts, local * width], axis=1).reshape(-1)
        arrays[f"b{batch}.spread"] = np.stack([rows[taken], starts[taken], ends[taken], local * width], axis=1).reshape(-1)
        arrays[f"b{batch}.segments"] = np.stack([first[taken], starts[taken], lens[taken], local], axis=1).reshape(-1)
        arrays[f"b{batch}.table"] = np.arange(len(taken) * width, dtype=np.int64)
        tile = attention_mma.QUERY_TILE
        found = [(first[i] + off, starts[i] + off, min(tile, lens[i] - off), j) for j, i in enumerate(taken) if lens[i] > FEW_TOKENS
                 for off in range(0, int(lens[i]), tile)]
        found.sort(key=lambda t: -(t[1] + t[2]))                    # the longest contexts first: the short ones fill the gaps
        arrays[f"b{batch}.tiles"] = np.array(found, dtype=np.int64).reshape(-1)
    return arrays


def most_ints(tokens, requests, context) -> int:
    """A bound on the ints of ``describe_segments`` without ``portion_tokens``, every array rounded up to a multiple of 4 and at least 4, for
    up to so many tokens of so many requests with contexts of up to ``context``: 12 a single token; of a longer segment 16 in ``few`` and ``multi``, 12 in
    its batch, 8 for tiles that are not full, 20 where the batch is its own, and its pages; 4 a token one by one."""
    requests = min(requests, tokens)
    longer = min(requests, tokens // 2)
    return 12 * requests + longer * (56 + -(-context // READ_PAGE)) + 4 * tokens + 4 * -(-tokens // attention_mma.QUERY_TILE) + 64


def portion_batches(starts, lens) -> list:
    """The segments of more than one token in batches whose contexts are read back together, as arrays of their indices, the longest
    contexts first."""
    portions = np.nonzero(lens > 1)[0]
    ends = starts + lens
    order, batches = portions[np.argsort(-ends[portions], kind="stable")], []
    while len(order):
        width = -(-int(ends[order[0]]) // READ_PAGE)
        taken = max(1, MOST_READ // (width * READ_PAGE))
        batches.append(order[:taken])
        order = order[taken:]
    return batches


def refresh_single_tokens(arrays, starts) -> None:
    """``describe_segments`` of a step of single tokens whose rows are those of the step before: only the positions change."""
    n, longest = len(starts), int(starts.max()) + 1
    for info, width, last in ((arrays["singles"], 8, 5), (arrays["single_tokens"], 4, 3)):
        info[1:width * n:width] = starts
        info[last:width * n:width] = longest


def recorded_fill(ends) -> float:
    """How full a recorded step of single tokens takes its contexts ``ends`` to be, as a part of the longest: all of it, or half.  Two
    values, so that a number of requests has two recordings a bucket of the longest context, and a step's is one that was made for steps
    like it.  Measured (us, spans for full ones / for half of it; 32 heads of 128 over 8; contexts all of the longest, spread evenly up to it, all but one a
    sixteenth of it): 48 requests, 16384 221 / 221, 151 / 139, 73 / 53; 64, 8192 166 / 170, 142 / 106, 87 / 27; 16, 8192 49 / 54, 48 / 38, 29 / 21; 128, 2048
    79 / 111, 62 / 72, 28 / 20."""
    return 1.0 if 4 * float(ends.mean()) >= 3 * float(ends.max()) else 0.5


class Reach(NamedTuple):
    """Contexts that a launch walks: the longest of them, the shortest that the longest may be, their mean as a part of the longest."""
    max_context: int
    min_context: int
    fill: float

    @classmethod
    def of(cls, ends, most=0, least=0):
        """``most``: of a recorded step, the longest context of those that it is replayed for; ``least``: their shortest longest one."""
        if most:
            return cls(most, least, recorded_fill(ends))
        longest = int(ends.max(initial=1))
        return cls(longest, least, round(16 * float(ends.mean()) / longest) / 16 if len(ends) else 1.0)


class StepPlan:
    """A step's segments on the device, as ``attend`` reads them.  ``max_context``: the longest context; of a recorded step the
    longest of the steps it is replayed for, ``min_context`` then the shortest of these steps' longest (these, the tokens and ``recorded_fill`` are
    all that a recorded step goes by).  ``settled``: no kernel right
    before an ``attend`` writes these arrays or the block table, so that it may read them while that one finishes."""

    def __init__(self, array, count, first, starts, lens, rows, max_context, min_context=0, settled=False):
        """``first``, ``starts``, ``lens`` and ``rows``: the segments' on the host (numpy)."""
        self.array, self.count = array, count
        self._segments = first, starts, lens, rows
        batches = portion_batches(starts, lens)
        self.portion_lens = [lens[taken] for taken in batches]          # of the batches' segments
        self.portion_ends = [(starts + lens)[taken] for taken in batches]
        self.multi_lens = lens[lens > 1]
        self.tokens = int(lens.sum())
        self.max_context, self.min_context, self.settled = int(max_context), int(min_context), int(settled)
        ends = starts + lens
        # the contexts of single tokens and of longer segments; of recorded steps (single tokens) the longest is a bound
        self.singles = Reach.of(ends[lens == 1], self.max_context if min_context else 0, self.min_context)
        self.multi = Reach.of(ends[lens > 1])
        # ... and of those that share an array: ``few``, ``few_tokens``, ``portion_tokens``
        some = lens[lens > 1]
        self.few, self.few_tokens, self.long = (self.multi if of.all() else Reach.of(ends[lens > 1][of])
                                                for of in (some <= FEW_ROWS, some <= FEW_TOKENS, some > FEW_TOKENS))

    @classmethod
    def of_segments(cls, rows, starts, lens, device):
        """Of a flat batch of segments one after another: their block-table rows, the absolute position of each one's first token and
        its tokens (host sequences)."""
        rows, starts, lens = (np.asarray(list(v), dtype=np.int64) for v in (rows, starts, lens))
        if not len(rows) == len(starts) == len(lens) or (lens < 1).any() or (starts < 0).any() or (rows < 0).any():
            raise KernelError("kv4.StepPlan: a row, a start and at least one token a segment")
        if max((starts + lens).max(initial=0), rows.max(initial=0), lens.sum()) > MOST_POSITION:
            raise KernelError(f"kv4.StepPlan: rows, positions and tokens are 32-bit numbers of up to {MOST_POSITION}")
        arrays = describe_segments(np.cumsum(lens) - lens, starts, lens, rows)
        # one upload, every array from a 16-byte boundary on
        at = np.cumsum([0] + [-(-len(values) // 4) * 4 for values in arrays.values()])
        packed = np.zeros(int(at[-1]), dtype=np.int32)
        for begin, values in zip(at, arrays.values()):
            packed[begin:begin + len(values)] = values
        there = torch.from_numpy(packed).to(device)
        array = {name: there[begin:begin + len(values)] for begin, (name, values) in zip(at.tolist(), arrays.items())}
        return cls(array, {name: len(values) for name, values in arrays.items()}, np.cumsum(lens) - lens, starts, lens, rows,
                   int((starts + lens).max(initial=0)))

    @classmethod
    def of_step(cls, ctx):
        """Of the step in flight, from the arrays that the planner made for it: the step's ``store`` comes after they are there."""
        view = ctx.plans[PLAN_KEY]
        return cls(view.array, view.count, ctx.h_seg_start, ctx.h_seg_pos0, ctx.h_seg_len, ctx.h_seg_row, ctx.max_context, ctx.min_context,
                   settled=True)

    def portion_tokens(self):
        """(array, tokens) of the portions' tokens one by one.  A step's description leaves them out: few steps need them."""
        if "portion_tokens" not in self.array:
            tokens = _one_by_one(*self._segments, np.nonzero(self._segments[2] > FEW_TOKENS)[0]).astype(np.int32)
            self.array["portion_tokens"] = torch.from_numpy(tokens).pin_memory().to(self.array["singles"].device, non_blocking=True)
        array = self.array["portion_tokens"]
        return array, array.shape[0] // 4


# ------------------------------------------------------------------ attention
#: Keys that a block of the span kernels takes at a time: a tile of 32 for each of its four warps.
STEP = 128
#: What a step takes, in us, with that many blocks on an SM: of the tensor-core kernel for heads of 128 by its tiles of rows (one B200, a
#: recorded chain of the kernel; up to 4 rows 1.11, 1.46, 2.37, 2.46, of 8 1.25, 1.63, 2.51, 2.59, of 16 1.57, 2.02, 3.05, 4.3, which choose
#: other spans for few calls, better and worse ones; a step of another head size takes (0.4 + 0.15 G) of it by G = head_dim / 32), and of the other kernel.
STEP_US = {1: (1.18, 1.58, 2.5, 2.6), 2: (1.65, 2.9, 4.0, 4.6)}
SINGLES_STEP_US = (2.0, 2.4, 3.0)
#: ... a launch and a block's start, and what a join of spans costs at all and for every span: by tiles of rows through memory, the last
#: block to arrive, and as a cluster of blocks.  Measured (us, memory / cluster): one request of 2 tokens behind 2043 and 2, 4, 8, 16 spans 18.3 /
#: 15.4, 14.7 / 10.6, 11.0 / 8.6, 10.2 / 8.8, of 4 tokens 26.8 / 21.3, 21.8 / 14.7, 17.2 / 11.9, 16.8 / 11.9; 8 requests of one token behind 8191
#: and 8 spans 29.2 / 28.4.
START_US, JOIN_US, SPAN_US = tuning.KV4_START_US, tuning.KV4_JOIN_US, tuning.KV4_SPAN_US
JOINS_US = {1: (JOIN_US, SPAN_US), 2: (5.0, 0.2)}
CLUSTER_SPAN_US = 0.14
#: Spans that are a cluster where all of them run at the same time, by tiles of rows.  Clusters of other sizes are placed badly (8 requests behind 8191,
#: 9 spans: 28.1 through memory, 37.0 as clusters; one request and 16 spans 10.9 / 12.7), and so are clusters of a second wave (24
#: requests behind 4095 and 3 spans 37.2 / 45.9).  16 blocks have to fit into one group of SMs, which leaves places empty: of one request of 12 tokens behind 4000
#: (24 clusters of 16, 3 blocks an SM) some come second, 27.6 as 16 spans and 18.8 as 8; of 5 tokens (16 clusters) 17.2 and 17.7.
CLUSTERS = {1: (2, 4, 8), 2: (2, 4, 8, 16)}
SMS, SMS_FOR_16 = 148, 100


def _clustered(n, blocks_per_span, step_us, clusters) -> bool:
    return n in clusters and blocks_per_span * n <= (SMS_FOR_16 if n == 16 else SMS) * len(step_us)


@functools.lru_cache(maxsize=4096)
def _plan(blocks_per_span, step_us, size, lo, hi, most, join, clusters, fill) -> int:
    """The number of spans that costs least per step of keys at both ends of [lo, hi] steps of longest context, of which the contexts have
    ``fill`` on the average: half a span more than that share of the spans holds something (48 requests spread evenly up to 16384: 3 spans 151 us, 10 137)."""
    full = SMS * len(step_us)

    def cost(steps, n):
        clustered = _clustered(n, blocks_per_span, step_us, clusters)
        each = -(-steps // n)
        n = -(-steps // each)                           # spans that hold anything
        waves, rest = divmod(int(blocks_per_span * min(n, fill * n + 0.5)), full)
        time = each * size * (waves * step_us[-1] + (step_us[-(-rest // SMS) - 1] if rest else 0.0)) + START_US * (waves + (rest > 0))
        return (time + (CLUSTER_SPAN_US * n if clustered else join[0] + join[1] * n if n > 1 else 0.0)) / steps
    return min(range(1, min(hi, most) + 1), key=lambda n: cost(hi, n) + (cost(lo, min(n, lo)) if lo != hi else 0.0))


def _spans(blocks_per_span, step_us, size, reach, window, most, join=(JOIN_US, SPAN_US), clusters=()) -> int:
    """Parts to cut the contexts into."""
    hi, lo = reach.max_context, reach.min_context or reach.max_context
    if window:
        hi, lo = min(hi, window + STEP), min(lo, window + STEP)
    hi = max(1, -(-hi // STEP))
    return _plan(blocks_per_span, step_us, size, max(1, min(hi, -(-lo // STEP))), hi, max(1, most), join, clusters, 1.0 if window else reach.fill)


def _capturing() -> bool:
    return torch._C._cuda_isCurrentStreamCapturing()


def _keep(extras, tensors) -> None:
    """What a recorded graph points to stays for as long as ``extras`` does, whatever other calls replace there."""
    kept = extras.setdefault("kv4_recorded", [])
    if not any(held is tensors for held in kept):
        kept.append(tensors)


def _replaced(old) -> None:
    """Memory that goes back to the stream it came from may still be in use on the current one."""
    for tensor in old or ():
        if tensor.is_cuda:
            tensor.record_stream(torch.cuda.current_stream())


def _scratch(extras, device, tokens, n_q_heads, n_spans, head_dim):
    """Partial sums, their (maximum, sum) pairs and the counters of the blocks that are done, which are zero between launches.  One
    span needs no partial sums."""
    if n_spans == 1:
        tokens, n_q_heads = 1, 1
    key = ("kv4_scratch", device)
    held, slots, heads = extras.get(key), tokens * n_q_heads * n_spans, tokens * n_q_heads
    if held is None or held[0].numel() < slots * head_dim or held[1].numel() < 2 * slots or held[2].numel() < heads:
        room = [2 * t.numel() for t in held] if held else [0, 0, 0]
        new = (torch.empty(max(slots * head_dim, min(room[0], attention_f32.MOST_SCRATCH // 4)), dtype=torch.float32, device=device),
               torch.empty(max(2 * slots, room[1]), dtype=torch.float32, device=device),
               torch.zeros(max(heads, room[2]), dtype=torch.int32, device=device))
        if _capturing():            # the counters are zeroed when the graph runs: no other call may count on it
            _keep(extras, new)
            return new
        _replaced(held)
        held = extras[key] = new
    elif _capturing():
        _keep(extras, held)
    return held


def _rows(extras, device, nbytes):
    """Memory for the rows of portions.  It grows to twice what it was, by MOST_GROWTH at most: a prompt that comes in chunks asks for a page
    more every 64 positions, and as much as it asks for would leave the allocator a block that is too small behind every time (chunks of 64
    behind up to 32768: 10 allocations instead of 512)."""
    key = ("kv4_rows", device)
    held = extras.get(key)
    if held is None or held[0].numel() < nbytes:
        had = held[0].numel() if held else 0
        _replaced(held)
        held = None
        extras.pop(key, None)           # given back before the larger one is asked for, unless a recorded graph points to it
        held = extras[key] = (torch.empty(max(nbytes, min(2 * had, had + MOST_GROWTH)), dtype=torch.uint8, device=device),)
    if _capturing():
        _keep(extras, held)
    return held[0]


def _few(info, n, tokens, most_tokens, plan, reach, q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, scale, window, extras):
    lib, most, blocks_a_sm = few_library(head_dim)
    rows = most_tokens * (n_q_heads // n_kv_heads)
    nt = 1 if rows <= 8 else 2
    blocks = n * n_kv_heads * -(-rows // (8 * nt))
    # the partial sums of all spans: fewer spans where they would outgrow their limit
    most = min(most, attention_f32.MOST_SCRATCH // (4 * tokens * n_q_heads * head_dim))
    step_us = STEP_US[nt][:blocks_a_sm[nt]]
    n_spans = _spans(blocks, step_us, 0.4 + 0.15 * (head_dim // GROUP), reach, window, most, JOINS_US[nt], CLUSTERS[nt])
    clustered = _clustered(n_spans, blocks, step_us, CLUSTERS[nt])
    device = q.get_device()
    part_o, part_ml, tickets = _scratch(extras, device, tokens, n_q_heads, 1 if clustered else n_spans, head_dim)
    _check(lib, lib.qil_kv4_few(_FEW.pack(
        q.data_ptr(), pages.data_ptr(), out.data_ptr(), info.data_ptr(), part_o.data_ptr(), part_ml.data_ptr(), tickets.data_ptr(),
        block_table.data_ptr(), _stream(device), scale, n, most_tokens, nt, n_spans, *block_table.shape, n_q_heads, n_kv_heads, page_size,
        pages.shape[0], window, clustered, plan.settled)), "kv4.attend (few tokens)")


def _singles(info, n, reach, q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, scale, window, extras):
    lib = library()
    chunks = -(-(n_q_heads // n_kv_heads) // lib.qil_kv4_singles_heads(n_q_heads // n_kv_heads))
    for begin in range(0, n, 65535):                       # a grid's third size
        some = min(65535, n - begin)
        most = attention_f32.MOST_SCRATCH // (4 * some * n_q_heads * head_dim)
        n_spans = _spans(some * n_kv_heads * chunks, SINGLES_STEP_US, 1.0, reach, window, most)
        device = q.get_device()
        part_o, part_ml, tickets = _scratch(extras, device, some, n_q_heads, n_spans, head_dim)
        _check(lib, lib.qil_kv4_singles(_SINGLES.pack(
            q.data_ptr(), pages.data_ptr(), out.data_ptr(), info.data_ptr() + 16 * begin, part_o.data_ptr(), part_ml.data_ptr(), tickets.data_ptr(),
            block_table.data_ptr(), _stream(device), scale, some, n_spans, *block_table.shape, n_q_heads, n_kv_heads, head_dim, page_size,
            pages.shape[0], window)), "kv4.attend (single tokens)")


def _portions(plan, batch, least, beside, q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, scale, window, extras):
    """A batch of portions of at least ``least`` tokens: their contexts' rows as pages of 64 positions, then the attention over those.
    ``beside``: the launch before this is ``_few``'s of the same step."""
    array, count = plan.array, plan.count
    segments, n_pages = count[f"b{batch}.read"] // 4, count[f"b{batch}.table"]
    table = array[f"b{batch}.table"][:n_pages].view(segments, n_pages // segments)
    lens = plan.portion_lens[batch]
    most = -(-int(plan.portion_ends[batch][lens >= least].max(initial=0)) // READ_PAGE)          # pages of the longest context of those that are meant
    if not most:
        return
    size = n_pages * 2 * n_kv_heads * READ_PAGE * head_dim
    if q.dtype == torch.float32:
        rows = _rows(extras, q.get_device(), 4 * size)[:4 * size].view(torch.float32).view(n_pages, 2, n_kv_heads, READ_PAGE, head_dim)
        read(pages, block_table, array[f"b{batch}.read"], segments, most * READ_PAGE, rows, n_kv_heads, head_dim, page_size)
        attention_f32.tiles(q, rows, out, array[f"b{batch}.tiles"], count[f"b{batch}.tiles"] // 4, table, n_q_heads, n_kv_heads, head_dim, READ_PAGE,
                            window, scale)
        return
    pack = attention_tc.keys16_pack(n_q_heads, n_kv_heads)
    groups, n_tiles = n_q_heads // pack, int((-(-lens[lens >= least] // (attention_tc.TILE // pack))).sum())
    splits = attention_tc.keys16_splits(n_tiles * groups, min(most, -(-window // READ_PAGE) + 1) if window else most)
    # rows, what goes with them and partial outputs, in one buffer: every part from a 128-byte boundary on
    heads, parts = n_pages * n_kv_heads, n_tiles * groups * splits * attention_tc.TILE if splits > 1 else 0
    at, total = [], 0
    for nbytes in (2 * size, 8 * heads, 4 * heads, heads * READ_PAGE, 4 * parts * head_dim, 16 * parts):
        at.append(total)
        total += -(-nbytes // 128) * 128
    base = _rows(extras, q.get_device(), total).data_ptr()
    rows, factors, value_marks, marks, part_o, part_ml = (base + offset for offset in at)
    lib = library()
    _check(lib, lib.qil_kv4_spread(_SPREAD.pack(
        pages.data_ptr(), block_table.data_ptr(), array[f"b{batch}.spread"].data_ptr(), rows, factors, value_marks, marks, _stream(q.get_device()),
        *block_table.shape, segments, most, n_kv_heads, head_dim, page_size, pages.shape[0], window, least, beside)), "kv4.attend (rows of portions)")
    attention_tc.prefill_keys16(q, rows, factors, value_marks, marks, part_o, part_ml, out, array[f"b{batch}.segments"], segments, least, n_tiles,
                                table, n_pages, n_q_heads, n_kv_heads, head_dim, scale, window, pack, splits)


def attend(plan, q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, scale, *, window=0, extras):
    """Causal attention of the tokens of ``plan`` (a :class:`StepPlan`) over 4-bit pages that hold their own keys and values already.

    q and out [N, n_q_heads * head_dim], bfloat16 or float32, the plan's tokens' rows of the flat batch; rows of other tokens are left as they
    are.  A token at position p sees the positions up to p, with ``window`` > 0 the last ``window`` of them.  Segments of up to FEW_TOKENS
    tokens (bfloat16: of up to FEW_ROWS tokens times heads on a kv head) do not see positions whose page the block table does not have, and a
    token that sees none gets zeros; longer ones need the pages of all that they see.  A value that is NaN reaches the tokens that see it and no others.  ``extras``: a dict that the caller keeps from call
    to call for the scratch memory, and for as long as a graph that recorded the call; calls that may run at the same time (other
    streams, recorded graphs too) need one each."""
    device = _device_of(q, "q")
    dtype_code(q.dtype)
    _take(q, "q", q.dtype, 2, device); _take(out, "out", q.dtype, 2, device); _take(block_table, "block_table", torch.int32, 2, device)
    _check_pages(pages, n_kv_heads, head_dim, page_size, "kv4.attend", device)
    if n_kv_heads < 1 or n_q_heads < 1 or n_q_heads % n_kv_heads:
        raise KernelError(f"kv4.attend: {n_q_heads} query heads do not divide into {n_kv_heads} kv heads")
    if q.shape[1] != n_q_heads * head_dim or out.shape != q.shape:
        raise KernelError(f"kv4.attend: queries {tuple(q.shape)}, output {tuple(out.shape)}")
    if window < 0 or not scale > 0:
        raise KernelError("kv4.attend: a window cannot be negative, and a scale is a positive number")
    if plan.array["singles"].get_device() != device or q.shape[0] < plan.tokens:
        raise KernelError(f"kv4.attend: a plan of {plan.tokens} tokens on {plan.array['singles'].device} for queries {tuple(q.shape)}")
    if window >= plan.max_context:            # everybody sees all
        window = 0
    shape = (q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, float(scale), int(window), extras)
    count, array = plan.count, plan.array
    if q.dtype == torch.float32:
        for name, reach in (("single_tokens", plan.singles), ("few_tokens", plan.few_tokens)):
            if count[name]:
                _singles(array[name], count[name] // 4, reach, *shape)
        if (plan.multi_lens > FEW_TOKENS).any():
            if attention_f32.supports(q, q, head_dim, head_dim, n_q_heads, n_kv_heads):
                for batch in range(len(plan.portion_lens)):
                    _portions(plan, batch, FEW_TOKENS + 1, False, *shape)
            else:       # heads of a size that the tile kernel does not take: token by token
                _singles(*plan.portion_tokens(), plan.long, *shape)
        return out
    if count["singles"]:
        _few(array["singles"], count["singles"] // 8, count["singles"] // 8, 1, plan, plan.singles, *shape)
    if len(plan.multi_lens):
        if not attention_tc.supports(head_dim, READ_PAGE, window):          # heads beyond 128
            _few(array["multi"], len(plan.multi_lens), int(plan.multi_lens.sum()), int(plan.multi_lens.max()), plan, plan.multi, *shape)
            return out
        most = FEW_ROWS // (n_q_heads // n_kv_heads)           # tokens
        few = plan.multi_lens[plan.multi_lens <= most]
        if len(few):
            _few(array["few"], count["few"] // 8, int(plan.multi_lens[plan.multi_lens <= FEW_ROWS].sum()), int(few.max()), plan, plan.few, *shape)
        if len(few) < len(plan.multi_lens):
            for batch in range(len(plan.portion_lens)):
                _portions(plan, batch, max(most, 1) + 1, batch == 0 and bool(count["singles"] or len(few)), *shape)
    return out
