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
from ctypes import c_float, c_int, c_longlong
from types import SimpleNamespace

import numpy as np
import torch

from . import attention_f32, attention_mma, attention_tc, build, ops, tuning
from .ops import F32, KernelError, _check, _need, _p, _stream, dtype_code

GROUP = 32
MOST_DIM = 256
PLAN_KEY = "kv4_attention"        # the step planner whose arrays ``attend`` reads (``describe_segments`` makes them)
#: Tokens of a segment up to which the kernels that walk the codes take it; longer portions' rows are read back once and attended to
#: as ordinary pages.
FEW_TOKENS = 8
#: Positions per page of rows that are read back for a portion, and the most of them at a time (of several portions; a single
#: one may be longer): 8 heads of 128 in bfloat16 take 4 KB a position.
READ_PAGE, MOST_READ = 64, 1 << 16

SOURCES, DEPENDS = ["kv4_store.cu", "kv4_attention.cu"], ["kv4.h"]
_lib = None
_few_libs: dict = {}


def few_library_name(head_dim):
    """(name, defines) of the tensor-core library for heads of ``head_dim``."""
    return f"qil_kv4_d{head_dim}", {"QIL_HEAD_DIM": head_dim}


def few_library(head_dim):
    lib = _few_libs.get(head_dim)
    if lib is None:
        name, defines = few_library_name(head_dim)
        lib = build.load(name, ["kv4_attention_mma.cu"], defines, depends=DEPENDS)
        if lib.qil_kv4_few_head_dim() != head_dim:
            raise KernelError("the 4-bit attention library was built for another head size")
        _few_libs[head_dim] = lib
    return lib


def library():
    global _lib
    if _lib is None:
        _lib = build.load("qil_kv4", SOURCES, depends=DEPENDS)
    return _lib


def supports(head_dim, page_size) -> bool:
    return head_dim % GROUP == 0 and 0 < head_dim <= MOST_DIM and page_size % 8 == 0 and page_size > 0


def page_shape(n_kv_heads, head_dim, page_size) -> tuple:
    """The shape of one page: multiply it out for its bytes."""
    if not supports(head_dim, page_size):
        raise KernelError(f"4-bit pages take head sizes 32, 64, ..., {MOST_DIM} and a multiple of 8 positions, not heads of {head_dim} "
                          f"and {page_size} positions")
    return (2, int(n_kv_heads), page_size // 8, 160 * (head_dim // GROUP))


def _check_pages(pages, n_kv_heads, head_dim, page_size, what):
    _need(pages, "pages", torch.uint8)
    if tuple(pages.shape[1:]) != page_shape(n_kv_heads, head_dim, page_size):
        raise KernelError(f"{what}: cache layout {tuple(pages.shape)} for {n_kv_heads} heads of {head_dim}, pages of {page_size}")
    if pages.data_ptr() % 16:
        raise KernelError(f"{what}: pages must start on a 16-byte boundary")


def _here(what, *tensors):
    """All on the current device: a launch goes to its stream."""
    current = torch.cuda.current_device()
    for tensor in tensors:
        if tensor is not None and tensor.device.index != current:
            raise KernelError(f"{what}: a tensor on {tensor.device} while the current device is cuda:{current}")


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
    _need(proj, "proj", ndim=2); _need(q_out, "q_out", proj.dtype, 2)
    _need(positions, "positions", torch.int32, 1); _need(token_row, "token_row", torch.int32, 1)
    n, width = proj.shape
    q_at, k_at, v_at = (int(c) for c in columns)
    if not supports(head_dim, page_size):
        page_shape(n_kv_heads, head_dim, page_size)
    if n_q_heads < 1 or n_kv_heads < 0:
        raise KernelError("kv4.store: head counts")
    if min(q_at, k_at, v_at) < 0 or q_out.shape != (n, n_q_heads * head_dim) or positions.shape[0] < n or token_row.shape[0] < n \
            or max(q_at + n_q_heads * head_dim, k_at + n_kv_heads * head_dim, v_at + n_kv_heads * head_dim) > width:
        raise KernelError("kv4.store: shapes do not match the head counts")
    if n_kv_heads:
        _check_pages(pages, n_kv_heads, head_dim, page_size, "kv4.store"); _need(block_table, "block_table", torch.int32, 2)
    norm, norm_code = 0, F32
    if q_norm_w is not None or k_norm_w is not None:
        if unit_heads:
            raise KernelError("kv4.store: heads of unit size have no norm weights")
        _need(q_norm_w, "q_norm_w", ndim=1); _need(k_norm_w, "k_norm_w", q_norm_w.dtype, 1)
        if q_norm_w.shape[0] != head_dim or k_norm_w.shape[0] != head_dim:
            raise KernelError("kv4.store: norm weights must have head_dim elements")
        norm, norm_code = 1, dtype_code(q_norm_w.dtype)
    elif unit_heads:
        norm = 2
    if rot_dims % 2 or not 0 <= rot_dims <= head_dim or layout not in (ops.ROTARY_HALVES, ops.ROTARY_INTERLEAVED):
        raise KernelError(f"kv4.store: {rot_dims} rotated dimensions of {head_dim}, layout {layout}")
    if rot_dims:
        if (table is None) == (freq is None):
            raise KernelError("kv4.store: a rotation comes from a table or from frequencies")
        if table is not None:
            _need(table, "table", torch.float32, 2)
            if table.shape[1] != rot_dims or table.shape[0] < 1 or gain != 1.0:
                raise KernelError("kv4.store: a table holds rot_dims columns, a gain included")
        else:
            _need(freq, "freq", torch.float32, 1)
            if freq.shape[0] != rot_dims // 2:
                raise KernelError("kv4.store: one frequency per rotated pair")
    _here("kv4.store", proj, q_out, pages if n_kv_heads else None, positions, token_row, block_table if n_kv_heads else None, q_norm_w,
          k_norm_w, table, freq)
    if n == 0:
        return q_out
    lib = library()
    _check(lib, lib.qil_kv4_store(
        _p(proj), c_longlong(width), c_int(q_at), c_int(k_at), c_int(v_at), _p(q_out), _p(pages if n_kv_heads else None), _p(q_norm_w),
        _p(k_norm_w), c_float(float(eps)), c_int(norm), _p(table if rot_dims else None), c_int(table.shape[0] if table is not None else 0),
        _p(freq if rot_dims else None), c_float(float(gain)), c_int(rot_dims), c_int(layout), _p(positions), _p(token_row),
        _p(block_table if n_kv_heads else None), c_int(block_table.shape[1] if n_kv_heads else 0), c_int(n), c_int(n_q_heads), c_int(n_kv_heads),
        c_int(head_dim), c_int(page_size), c_int(pages.shape[0] if n_kv_heads else 0), c_int(dtype_code(proj.dtype)), c_int(norm_code), _stream()),
        "kv4.store")
    return q_out


def read(pages, block_table, info, segments, longest, out, n_kv_heads, head_dim, page_size):
    """The values that rows of 4-bit pages stand for, as ordinary pages ``out`` [pages, 2, kv heads, positions a page, head_dim] of
    bfloat16 or float32 (positions a page need not be ``page_size``).

    ``info`` int32 [segments * 4]: (block-table row, first position, positions, first page of ``out``) a segment; ``longest``: no segment
    has more positions.  Position first + i goes to slot i % (positions a page) of page i // (positions a page) after the segment's
    first.  Positions without a page are read as zeros; slots behind a segment's last position are left as they are."""
    _check_pages(pages, n_kv_heads, head_dim, page_size, "kv4.read")
    _need(block_table, "block_table", torch.int32, 2); _need(info, "info", torch.int32, 1); _need(out, "out", ndim=5)
    if info.shape[0] < 4 * segments or segments < 0:
        raise KernelError("kv4.read: four numbers a segment")
    if out.shape[1] != 2 or out.shape[2] != n_kv_heads or out.shape[4] != head_dim or out.data_ptr() % 16:
        raise KernelError(f"kv4.read: output {tuple(out.shape)} for {n_kv_heads} heads of {head_dim}")
    _here("kv4.read", pages, block_table, info, out)
    if segments == 0 or longest <= 0 or out.numel() == 0:
        return out
    lib = library()
    _check(lib, lib.qil_kv4_read(_p(pages), _p(block_table), c_int(block_table.shape[1]), _p(info), c_int(segments), c_int(int(longest)),
                                 _p(out), c_int(out.shape[0]), c_int(out.shape[3]), c_int(n_kv_heads), c_int(head_dim), c_int(page_size),
                                 c_int(pages.shape[0]), c_int(dtype_code(out.dtype)), _stream()), "kv4.read")
    return out


# ------------------------------------------------------------------ the plan of a step
def describe_segments(first, starts, lens, rows) -> dict:
    """A step's segments as ``attend`` wants them (numpy int64 arrays in, one entry per segment: first token in the flat batch,
    its absolute position, tokens, block-table row).

    ``singles``, ``few``, ``portions``  the segments of one token, of up to FEW_TOKENS and the others: eight ints each, (first token, its
                        position, tokens, block-table row, tokens of the segments before in this array, the longest context among these, 0, 0)
    ``single_tokens``, ``few_tokens``, ``portion_tokens``  the same token by token, four ints each, (token, its position, block-table row, the
                        longest context among these)
    ``b0.read`` ...     the portions in batches whose contexts are read back together: ``kv4.read``'s info, the block table of the
                        pages they are read to, and their query tiles over that table (``attention_mma.describe_segments``)
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

    def one_by_one(indices):
        if not len(indices):
            return np.zeros(0, dtype=np.int64)
        of = np.repeat(indices, lens[indices])
        offset = np.arange(len(of)) - np.repeat(np.cumsum(lens[indices]) - lens[indices], lens[indices])
        return np.stack([first[of] + offset, starts[of] + offset, rows[of], np.full_like(of, ends[indices].max())], axis=1).reshape(-1)

    arrays = {}
    for name, tokens, some in (("singles", "single_tokens", lens == 1), ("few", "few_tokens", (lens > 1) & (lens <= FEW_TOKENS)),
                               ("portions", "portion_tokens", lens > FEW_TOKENS)):
        indices = np.nonzero(some)[0]
        arrays[name], arrays[tokens] = segments(indices), one_by_one(indices)
    portions = np.nonzero(lens > FEW_TOKENS)[0]
    order = portions[np.argsort(-ends[portions], kind="stable")]
    batch = 0
    while len(order):
        width = -(-int(ends[order[0]]) // READ_PAGE)               # pages a segment: of the longest, so that segment i's begin at i * width
        taken = order[:max(1, MOST_READ // (width * READ_PAGE))]
        order = order[len(taken):]
        local = np.arange(len(taken), dtype=np.int64)
        tiles = attention_mma.describe_segments(first[taken], starts[taken], lens[taken], local)
        arrays[f"b{batch}.read"] = np.stack([rows[taken], np.zeros_like(local), ends[taken], local * width], axis=1).reshape(-1)
        arrays[f"b{batch}.table"] = np.arange(len(taken) * width, dtype=np.int64)
        for name in ("tile_info", "big_tile_info", "rest_tile_info"):
            arrays[f"b{batch}.{name}"] = tiles[name]
        batch += 1
    return arrays


def refresh_single_tokens(arrays, starts) -> None:
    """``describe_segments`` of a step of single tokens whose rows are those of the step before: only the positions change."""
    n, longest = len(starts), int(starts.max()) + 1
    for info, width, last in ((arrays["singles"], 8, 5), (arrays["single_tokens"], 4, 3)):
        info[1:width * n:width] = starts
        info[last:width * n:width] = longest


class StepPlan:
    """A step's segments on the device, as ``attend`` reads them.  ``max_context``: the longest context; of a recorded step the
    longest of the steps it is replayed for, ``min_context`` then the shortest of these steps' longest."""

    def __init__(self, array, count, max_context, min_context=0, most_tokens=0):
        self.array, self.count = array, count
        self.most_tokens = int(most_tokens)          # of a segment
        self.max_context, self.min_context = int(max_context), int(min_context)
        self.batches = 0
        while f"b{self.batches}.read" in count:
            self.batches += 1

    @classmethod
    def of_segments(cls, rows, starts, lens, device):
        """Of a flat batch of segments one after another: their block-table rows, the absolute position of each one's first token and
        its tokens (host sequences)."""
        rows, starts, lens = (np.asarray(list(v), dtype=np.int64) for v in (rows, starts, lens))
        if not len(rows) == len(starts) == len(lens) or (lens < 1).any() or (starts < 0).any() or (rows < 0).any():
            raise KernelError("kv4.StepPlan: a row, a start and at least one token a segment")
        arrays = describe_segments(np.cumsum(lens) - lens, starts, lens, rows)
        array = {name: torch.from_numpy(values.astype(np.int32)).to(device) for name, values in arrays.items()}
        return cls(array, {name: len(values) for name, values in arrays.items()}, int((starts + lens).max(initial=0)),
                   most_tokens=lens.max(initial=0))

    @classmethod
    def of_step(cls, ctx):
        """Of the step in flight, from the arrays that the planner made for it."""
        view = ctx.plans[PLAN_KEY]
        return cls(view.array, view.count, ctx.max_context, ctx.min_context, most_tokens=max(ctx.h_seg_len))


# ------------------------------------------------------------------ attention
_sms = None


def _slots(blocks_per_sm) -> int:
    global _sms
    if _sms is None:
        _sms = torch.cuda.get_device_properties(torch.cuda.current_device()).multi_processor_count if torch.cuda.is_available() else 148
    return _sms * blocks_per_sm


#: Keys that a block of the span kernels takes at a time: a tile of 32 for each of its four warps.
STEP = 128


@functools.lru_cache(maxsize=4096)
def _plan(blocks_per_span, slots, lo, hi, most) -> int:
    """The number of spans with the lowest cost per step of keys at both ends of [lo, hi] steps of longest context.  A wave of blocks takes
    the steps of a span and a start-up; every span costs the join something."""
    def cost(steps, n):
        each = -(-steps // n)
        n = -(-steps // each)
        return (-(-blocks_per_span * n // slots) * (each + tuning.KV4_SPAN_STARTUP) + tuning.KV4_SPAN_JOIN * n) / steps
    return min(range(1, min(hi, most) + 1), key=lambda n: cost(hi, n) + (cost(lo, min(n, lo)) if lo != hi else 0.0))


def _spans(blocks_per_span, slots, plan, window, most) -> int:
    """Parts to cut the contexts into."""
    reach = lambda context: min(context, window + STEP) if window else context
    hi = max(1, -(-reach(plan.max_context) // STEP))
    lo = max(1, min(hi, -(-reach(plan.min_context or plan.max_context) // STEP)))
    return _plan(blocks_per_span, slots, lo, hi, max(1, most))


def _scratch(extras, device, tokens, n_q_heads, n_spans, head_dim):
    return attention_mma.decode_scratch(SimpleNamespace(extras=extras, device=device), tokens, n_q_heads, n_spans, head_dim,
                                        most=attention_f32.MOST_SCRATCH)


def _few(info, n, tokens, most_tokens, plan, q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, scale, window, extras):
    lib = few_library(head_dim)
    rows = most_tokens * (n_q_heads // n_kv_heads)
    nt = 1 if rows <= 8 else 2 if rows <= 16 or head_dim > 128 else 4
    blocks = n * n_kv_heads * -(-rows // (8 * nt))
    # the partial sums of all spans: fewer spans where they would outgrow their limit
    most = min(lib.qil_kv4_few_most_spans(), attention_f32.MOST_SCRATCH // (4 * tokens * n_q_heads * head_dim))
    n_spans = _spans(blocks, _slots(lib.qil_kv4_few_blocks_a_sm(c_int(nt))), plan, window, most)
    part_o, part_ml, tickets = _scratch(extras, q.device, tokens, n_q_heads, n_spans, head_dim)
    _check(lib, lib.qil_kv4_few(_p(q), _p(pages), _p(out), _p(info), c_int(n), c_int(most_tokens), c_int(nt), _p(part_o), _p(part_ml), _p(tickets),
                                c_int(n_spans), _p(block_table), c_int(block_table.shape[1]), c_int(n_q_heads), c_int(n_kv_heads), c_int(page_size),
                                c_int(pages.shape[0]), c_int(window), c_float(scale), _stream()), "kv4.attend (few tokens)")


def _singles(info, n, plan, q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, scale, window, extras):
    lib = library()
    share = n_q_heads // n_kv_heads
    chunks = -(-share // lib.qil_kv4_singles_heads(c_int(share)))
    most = attention_f32.MOST_SCRATCH // (4 * n * n_q_heads * head_dim)
    n_spans = _spans(n * n_kv_heads * chunks, _slots(3), plan, window, most)
    part_o, part_ml, tickets = _scratch(extras, q.device, n, n_q_heads, n_spans, head_dim)
    _check(lib, lib.qil_kv4_singles(_p(q), _p(pages), _p(out), _p(info), c_int(n), _p(part_o), _p(part_ml), _p(tickets), c_int(n_spans),
                                    _p(block_table), c_int(block_table.shape[1]), c_int(n_q_heads), c_int(n_kv_heads), c_int(head_dim),
                                    c_int(page_size), c_int(pages.shape[0]), c_int(window), c_float(scale), c_int(dtype_code(q.dtype)), _stream()),
           "kv4.attend (single tokens)")


def _portions(plan, batch, q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, scale, window, extras):
    """A batch of portions: their contexts' rows as ordinary pages, then the attention over those."""
    array = {name: plan.array[f"b{batch}.{name}"] for name in ("read", "table", "tile_info", "big_tile_info", "rest_tile_info")}
    count = {name: plan.count[f"b{batch}.{name}"] for name in array}
    segments = count["read"] // 4
    width = count["table"] // segments
    shape = (count["table"], 2, n_kv_heads, READ_PAGE, head_dim)
    held = extras.get(("kv4_rows", q.dtype))
    size = count["table"] * 2 * n_kv_heads * READ_PAGE * head_dim
    if held is None or held.numel() < size:
        held = extras[("kv4_rows", q.dtype)] = torch.empty(size, dtype=q.dtype, device=q.device)
    rows = held[:size].view(shape)
    read(pages, block_table, array["read"], segments, width * READ_PAGE, rows, n_kv_heads, head_dim, page_size)
    table = array["table"][:count["table"]].view(segments, width)
    if q.dtype == torch.bfloat16:
        array["decode_info"], count["decode_info"] = None, 0
        ctx = SimpleNamespace(plans={attention_mma.PLAN_KEY: SimpleNamespace(array=array, count=count)}, max_context=plan.max_context, min_context=0,
                              extras=extras, device=q.device)
        view = SimpleNamespace(pages=rows, block_table=table, page_size=READ_PAGE, window=window)
        attention_mma.attend(ctx, q, view, out, n_q_heads, n_kv_heads, head_dim, window, scale)
    else:
        attention_f32.tiles(q, rows, out, array["tile_info"], count["tile_info"] // 4, table, n_q_heads, n_kv_heads, head_dim, READ_PAGE,
                            window, scale)


def attend(plan, q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, scale, *, window=0, extras):
    """Causal attention of the tokens of ``plan`` (a :class:`StepPlan`) over 4-bit pages that hold their own keys and values already.

    q and out [N, n_q_heads * head_dim], bfloat16 or float32, the plan's tokens' rows of the flat batch; rows of other tokens are left as they
    are.  A token at position p sees the positions up to p, with ``window`` > 0 the last ``window`` of them.  Positions whose page the block
    table does not have are not seen; a token that sees none gets zeros.  ``extras``: a dict that the caller keeps from call to call
    for the scratch memory; calls that may run at the same time (other streams) need one each."""
    _need(q, "q", ndim=2); _need(out, "out", q.dtype, 2); _need(block_table, "block_table", torch.int32, 2)
    dtype_code(q.dtype)
    _check_pages(pages, n_kv_heads, head_dim, page_size, "kv4.attend")
    if n_kv_heads < 1 or n_q_heads < 1 or n_q_heads % n_kv_heads:
        raise KernelError(f"kv4.attend: {n_q_heads} query heads do not divide into {n_kv_heads} kv heads")
    if q.shape[1] != n_q_heads * head_dim or out.shape != q.shape:
        raise KernelError(f"kv4.attend: queries {tuple(q.shape)}, output {tuple(out.shape)}")
    if window < 0:
        raise KernelError("kv4.attend: a window cannot be negative")
    _here("kv4.attend", q, pages, out, block_table, plan.array["singles"])
    shape = (q, pages, out, block_table, n_q_heads, n_kv_heads, head_dim, page_size, float(scale), int(window), extras)
    count, array = plan.count, plan.array
    if q.dtype == torch.float32:
        for name in ("single_tokens", "few_tokens"):
            if count[name]:
                _singles(array[name], count[name] // 4, plan, *shape)
        if count["portion_tokens"]:
            if attention_f32.supports(q, q, head_dim, head_dim, n_q_heads, n_kv_heads):
                for batch in range(plan.batches):
                    _portions(plan, batch, *shape)
            else:       # heads of a size that the tile kernel does not take: token by token
                _singles(array["portion_tokens"], count["portion_tokens"] // 4, plan, *shape)
        return out
    if count["singles"]:
        _few(array["singles"], count["singles"] // 8, count["singles"] // 8, 1, plan, *shape)
    if count["few"]:
        _few(array["few"], count["few"] // 8, count["few_tokens"] // 4, FEW_TOKENS, plan, *shape)
    if count["portions"]:
        if attention_tc.supports(head_dim, READ_PAGE, window):
            for batch in range(plan.batches):
                _portions(plan, batch, *shape)
        else:           # heads beyond 128
            _few(array["portions"], count["portions"] // 8, count["portion_tokens"] // 4, plan.most_tokens, plan, *shape)
    return out
