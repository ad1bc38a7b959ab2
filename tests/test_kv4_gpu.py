"""The cache of 4 bits, kernel by kernel, against its definition in 64 bits."""
import math

import pytest
import torch

from tests.plain import kv4_plain as plain

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-6


def kv4():
    from qwen_inference_lab_b200.kernels import kv4 as module
    return module


def refused(call, *args, **kwargs):
    from qwen_inference_lab_b200.kernels.ops import KernelError
    with pytest.raises(KernelError):
        call(*args, **kwargs)


# ------------------------------------------------------------------ store
STORES = [  # hq, hkv, dim, page, norm, rotary, rot, layout, gain, first positions of the requests, tokens of each
    (1, 1, 32, 8, "none", None, 0, 0, 1.0, [0], [1]),
    (4, 2, 64, 8, "heads", "table", 64, 0, 1.0, [5, 0], [11, 1]),
    (32, 8, 128, 16, "heads", "table", 128, 0, 1.0, [1000, 7, 16], [3, 1, 17]),
    (6, 3, 96, 24, "unit", "freq", 32, 1, 1.25, [70001, 23], [2, 30]),
    (5, 1, 256, 64, "heads", "freq", 256, 1, 1.0, [399990, 0], [9, 65]),
    (7, 7, 160, 8, "none", "freq", 50, 0, 0.5, [3], [20]),
    (2, 2, 128, 32, "heads", "table", 64, 1, 1.0, [31], [4]),
]


def store_case(hq, hkv, dim, page, norm, rotary, rot, layout, gain, starts, lens, dtype, weight_dtype=None, extra_columns=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = sum(lens)
    width = (hq + 2 * hkv) * dim + extra_columns
    case = dict(hq=hq, hkv=hkv, dim=dim, page=page, norm=norm, rot=rot, layout=layout, gain=gain, dtype=dtype)
    case["proj"] = (torch.randn(n, width, generator=g) * 2).to(dtype)
    case["columns"] = (extra_columns, extra_columns + hq * dim, extra_columns + (hq + hkv) * dim)
    case["positions"] = torch.cat([torch.arange(s, s + k) for s, k in zip(starts, lens)]).int()
    case["token_row"] = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).int()
    needed = [-(-(s + k) // page) for s, k in zip(starts, lens)]
    order = torch.randperm(sum(k // page + 2 for k in lens) + 2, generator=g).int()
    table = torch.full((len(lens), max(needed) + 1), -1, dtype=torch.int32)
    begin = 0
    for i, (s, k) in enumerate(zip(starts, lens)):
        for index in range(s // page, needed[i]):
            table[i, index] = order[begin]
            begin += 1
    case["table"], case["n_pages"] = table, len(order)
    if norm == "heads":
        case["weights"] = [(1 + 0.1 * torch.randn(dim, generator=g)).to(weight_dtype or dtype) for _ in range(2)]
    else:
        case["weights"] = [None, None]
    case["rope"] = case["freq"] = None
    if rotary == "table":
        inverse = 1.0 / 1e6 ** (torch.arange(0, rot, 2).double() / rot)
        angles = torch.arange(max(s + k for s, k in zip(starts, lens))).double()[:, None] * inverse
        case["rope"] = torch.cat((angles.cos(), angles.sin()), -1).float().to(dtype).float()
    elif rotary == "freq":
        case["freq"] = (1e4 ** (-torch.arange(0, rot, 2).double() / rot)).float()
    return case


def store_plain(case):
    hq, hkv, dim, rot = (case[k] for k in ("hq", "hkv", "dim", "rot"))
    n = len(case["proj"])
    q, k, v = (case["proj"][:, c:c + h * dim].double().view(n, h, dim) for c, h in zip(case["columns"], (hq, hkv, hkv)))
    pos = case["positions"].long()

    def tail(x, weight):
        if case["norm"] == "heads":
            x = plain.normed(x, weight, EPS)
        if rot:
            angles = None if case["freq"] is None else pos.double()[:, None] * case["freq"].double()
            x = plain.turned(x, angles, rot, case["layout"], case["gain"], None if case["rope"] is None else case["rope"][pos])
        return plain.normed(x, None, EPS) if case["norm"] == "unit" else x

    return tail(q, case["weights"][0]), tail(k, case["weights"][1]), v


def store_run(case, pages, q_out=None):
    up = lambda t: None if t is None else t.cuda()
    n = len(case["proj"])
    q_out = torch.empty(n, case["hq"] * case["dim"], dtype=case["dtype"], device="cuda") if q_out is None else q_out
    kv4().store(case["proj"].cuda(), case["columns"], q_out, pages, case["positions"].cuda(), case["token_row"].cuda(),
                case["table"].cuda(), case["hq"], case["hkv"], case["dim"], case["page"], q_norm_w=up(case["weights"][0]),
                k_norm_w=up(case["weights"][1]), eps=EPS, unit_heads=case["norm"] == "unit", table=up(case["rope"]),
                freq=up(case["freq"]), rot_dims=case["rot"], layout=case["layout"], gain=case["gain"])
    return q_out


def check_store(case):
    pages = torch.full((case["n_pages"], *kv4().page_shape(case["hkv"], case["dim"], case["page"])), 0xA5, dtype=torch.uint8, device="cuda")
    q_out = store_run(case, pages)
    q, k, v = store_plain(case)
    # queries: 32-bit arithmetic (the norm's sum, a handful of roundings of values up to |turned head|) and one rounding
    unit = 2.0 ** -8 if case["dtype"] == BF16 else 0.0
    got = q_out.cpu().double().view(q.shape)
    size = q.abs().amax(-1, keepdim=True)
    assert ((got - q).abs() <= unit * q.abs() + 16 * 2.0 ** -24 * size).all()
    # keys and values: the very bytes; all others untouched
    expected = torch.full(pages.shape, 0xA5, dtype=torch.uint8)
    for token in range(len(k)):
        pos, row = int(case["positions"][token]), int(case["token_row"][token])
        page = int(case["table"][row, pos // case["page"]])
        if page < 0:
            continue
        for plane, rows in enumerate((k, v)):
            codes, pairs = plain.coded(rows[token])
            for head in range(case["hkv"]):
                plain.put(expected, page, plane, head, pos % case["page"], codes[head], pairs[head])
    assert torch.equal(pages.cpu(), expected)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("case", STORES, ids=[f"{c[0]}_{c[1]}x{c[2]}_{c[4]}_{c[5]}" for c in STORES])
def test_store(case, dtype):
    check_store(store_case(*case, dtype))


def test_store_float32_weights_and_odd_columns():
    check_store(store_case(4, 2, 64, 8, "heads", "table", 64, 0, 1.0, [5, 0], [11, 1], BF16, weight_dtype=F32, extra_columns=3))
    check_store(store_case(4, 2, 64, 8, "heads", "freq", 64, 0, 1.0, [5, 0], [11, 1], F32, weight_dtype=BF16, extra_columns=1))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_store_rows_at_the_edges(dtype):
    """Zeros, one value everywhere, ties between two codes, NaN and infinities, the largest and the smallest numbers; a token
    without a page."""
    case = store_case(1, 1, 64, 8, "none", None, 0, 0, 1.0, [0], [12], dtype)
    rows = case["proj"].view(12, 3, 64)
    rows[0] = 0.0
    rows[1] = -3.5
    rows[2, 1:] = torch.arange(64).float() % 16 / 2           # s = 0.5: every code exact
    rows[3, 1:] = torch.cat((torch.tensor([0.0, 15.0]), torch.arange(62).float() % 15 + 0.5))     # s = 1: halves
    rows[4, 1:, 5] = math.nan
    rows[5, 1:, 40] = math.inf
    rows[6, 1:, 3] = -math.inf
    big = torch.finfo(dtype).max
    rows[7, 1:, 0], rows[7, 1:, 1] = big, -big
    rows[8, 1:] = 1e-38 * torch.randn(64)
    rows[9, 1:] = 1e30 * torch.randn(64)
    rows[10, 1:] = 1000 + torch.randn(64)
    case["table"][0, 1] = -1                                  # positions 8 .. 11 have no page
    check_store(case)


def test_store_queries_only_and_no_tokens():
    case = store_case(4, 2, 64, 8, "heads", "table", 64, 0, 1.0, [5], [3], BF16)
    n = 3
    q_out = torch.empty(n, 4 * 64, dtype=BF16, device="cuda")
    up = lambda t: t.cuda()
    args = (case["columns"], q_out, None, up(case["positions"]), up(case["token_row"]), None, 4, 0, 64, 8)
    kv4().store(up(case["proj"]), *args, q_norm_w=up(case["weights"][0]), k_norm_w=up(case["weights"][1]), eps=EPS, table=up(case["rope"]), rot_dims=64)
    whole = torch.zeros((case["n_pages"], *kv4().page_shape(2, 64, 8)), dtype=torch.uint8, device="cuda")
    assert torch.equal(q_out, store_run(case, whole))
    empty = torch.empty(0, case["proj"].shape[1], dtype=BF16, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    kv4().store(empty, case["columns"], q_out[:0], whole, none, none, up(case["table"]), 4, 2, 64, 8)


# ------------------------------------------------------------------ read
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("heads,dim,page,out_page", [(1, 32, 8, 1), (3, 96, 16, 64), (8, 128, 32, 5), (2, 256, 8, 64)])
def test_read(dtype, heads, dim, page, out_page):
    torch.manual_seed(3)
    lens = [1, page, 3 * page + 5, 131]
    keys = [torch.randn(n, heads, dim) for n in lens]
    values = [torch.randn(n, heads, dim) * 3 for n in lens]
    pages, table, held = plain.build(keys, values, lens, page)
    table[3, 2] = -1                                          # a page given back
    segments, at = [], 0
    for i, n in enumerate(lens):
        first = min(n // 3, 7)
        segments.append((i, first, n - first, at))
        at += -(-(n - first) // out_page)
    out = torch.full((at + 1, 2, heads, out_page, dim), 7.0, dtype=dtype, device="cuda")
    info = torch.tensor(segments, dtype=torch.int32).view(-1).cuda()
    kv4().read(pages.cuda(), table.cuda(), info, len(segments), max(s[2] for s in segments), out, heads, dim, page)
    expected = torch.full(out.shape, 7.0, dtype=dtype)
    for i, first, count, at in segments:
        for t in range(count):
            absent = table[i, (first + t) // page] < 0
            for plane in (0, 1):
                row = torch.zeros(heads, dim) if absent else held[i][plane][first + t].float()
                expected[at + t // out_page, plane, :, t % out_page] = row.to(dtype)
    assert torch.equal(out.cpu(), expected)


# ------------------------------------------------------------------ attend
def attend_case(hq, hkv, dim, page, starts, lens, dtype, seed=0, loud=1.0):
    g = torch.Generator().manual_seed(seed)
    total = [s + n for s, n in zip(starts, lens)]
    keys = [torch.randn(t, hkv, dim, generator=g) * loud for t in total]
    values = [torch.randn(t, hkv, dim, generator=g) for t in total]
    pages, table, held = plain.build(keys, values, total, page, seed=seed)
    q = torch.randn(sum(lens), hq * dim, generator=g).to(dtype)
    return dict(hq=hq, hkv=hkv, dim=dim, page=page, starts=starts, lens=lens, pages=pages, table=table, held=held, q=q, dtype=dtype)


def attend_run(case, window=0, scale=None, extras=None, plan=None, out=None):
    module = kv4()
    device = "cuda"
    plan = plan or module.StepPlan.of_segments(range(len(case["lens"])), case["starts"], case["lens"], device)
    out = torch.full(case["q"].shape, math.nan, dtype=case["dtype"], device=device) if out is None else out
    module.attend(plan, case["q"].cuda(), case["pages"].cuda(), out, case["table"].cuda(), case["hq"], case["hkv"], case["dim"], case["page"],
                  case["dim"] ** -0.5 if scale is None else scale, window=window, extras={} if extras is None else extras)
    return out


def attend_check(case, out, window=0, scale=None):
    """Against 64 bits.  A relative error e of every weight p moves a result by e sum p |v| at most, and of the sum that divides it by as much.
    A weight's error is twice that of its score at most: float32 sums of dim terms are off by dim 2^-24 scale sum |q k|, keys in 11 bits
    (long portions) by 2^-11 of it.  For bfloat16 queries the kernels round p once (2^-8) and its product with a step once more, which moves
    the result by 2^-8 sum p (v - m), or the values that it weighs; then the result."""
    scale = case["dim"] ** -0.5 if scale is None else scale
    first = 0
    got = out.cpu().double().view(len(out), case["hq"], case["dim"])
    for i, (start, n) in enumerate(zip(case["starts"], case["lens"])):
        q = case["q"][first:first + n].view(n, case["hq"], case["dim"]).double()
        keys = case["held"][i][0].repeat_interleave(case["hq"] // case["hkv"], dim=1)
        exact, size = plain.attention(q, *case["held"][i], torch.arange(start, start + n), scale, window)
        off = (got[first:first + n] - exact).abs()
        most = scale * torch.einsum("nhd,thd->nht", q.abs(), keys.abs()).amax(-1, keepdim=True)      # of the terms of a score
        if case["dtype"] == BF16:
            groups = case["held"][i][1].unflatten(-1, (-1, 32))
            _, above = plain.attention(q, case["held"][i][0], (groups - groups.amin(-1, keepdim=True)).flatten(-2), torch.arange(start, start + n), scale, window)
            bar = 2.0 ** -8 * exact.abs() + (4 * 2.0 ** -8 + 2 * 2.0 ** -11 * most) * size + 2.0 ** -8 * above
        else:
            bar = 2.0 ** -24 * (start + n + 64 + 2 * case["dim"] * most) * size
        assert torch.isfinite(got[first:first + n]).all() and (off <= bar).all(), (i, float((off / bar).max()))
        if case["dtype"] == BF16 and n * case["hq"] * case["dim"] >= 512:      # rounding errors are random: the whole is much nearer
            spread = scale * torch.einsum("nhd,thd->nht", q.square(), keys.square()).amax().sqrt()
            assert off.norm() <= (4e-3 + 2.0 ** -11 * spread) * exact.norm(), (i, float(off.norm() / exact.norm()))
        first += n


ATTENDS = [  # hq, hkv, dim, page, starts, lens, window
    (1, 1, 32, 8, [0], [1], 0),                               # one key
    (4, 4, 64, 16, [0, 1, 31, 32, 33], [1, 1, 1, 1, 1], 0),   # a head of its own each; borders of a tile
    (32, 8, 128, 16, [700, 0, 5, 2049], [1, 1, 1, 1], 0),
    (12, 4, 64, 8, [100, 40, 0], [1, 1, 1], 33),              # windows that begin inside a page and before the first position
    (5, 1, 96, 8, [64, 9], [1, 3], 0),
    (16, 1, 256, 32, [300], [2], 0),                          # 16 heads share a key
    (20, 1, 128, 16, [77, 3], [1, 5], 50),
    (16, 8, 128, 16, [400, 3, 0], [5, 8, 2], 0),              # a few tokens
    (6, 2, 128, 16, [0, 130, 65], [9, 40, 200], 0),           # portions
    (8, 2, 64, 64, [513, 0], [129, 64], 100),
    (3, 1, 32, 8, [1], [130], 0),
    (4, 1, 256, 8, [50], [70], 0),
    (8, 8, 96, 16, [0, 20, 500], [300, 1, 17], 0),            # all kinds at once
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("case", ATTENDS, ids=[f"{c[0]}_{c[1]}x{c[2]}_{i}" for i, c in enumerate(ATTENDS)])
def test_attend(case, dtype):
    *sizes, window = case
    built = attend_case(*sizes, dtype)
    attend_check(built, attend_run(built, window), window)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_attend_peaked_scores_and_other_scales(dtype):
    built = attend_case(8, 2, 128, 16, [900, 300], [1, 6], dtype, loud=4.0)
    attend_check(built, attend_run(built, scale=0.25), scale=0.25)


def test_attend_spans_agree_with_one():
    """A context cut over many blocks gives what one block gives, to the sums' rounding, twice the same bits."""
    built = attend_case(8, 2, 128, 16, [5000], [1], F32)
    a, b = attend_run(built), attend_run(built)
    assert torch.equal(a, b)
    attend_check(built, a)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_attend_nan_goes_to_those_who_see_it(dtype):
    built = attend_case(4, 2, 64, 8, [40, 40, 40, 0], [1, 1, 4, 30], dtype)
    key = built["table"]
    plane_bytes = built["pages"]
    # request 0: the key at position 3 of head 0 is NaN; request 1: the value at position 3 of head 1; request 3: the value at position 20
    for row, plane, head, pos in ((0, 0, 0, 3), (1, 1, 1, 3), (3, 1, 0, 20)):
        codes, pairs = plain.get(plane_bytes, int(key[row, pos // 8]), plane, head, pos % 8)
        pairs[0] = math.nan
        plain.put(plane_bytes, int(key[row, pos // 8]), plane, head, pos % 8, codes, pairs)
    out = attend_run(built).float().cpu().view(-1, 4, 64)
    assert out[0, :2].isnan().all() and out[0, 2:].isfinite().all()
    assert out[1, 2:, :32].isnan().all() and out[1, 2:, 32:].isfinite().all() and out[1, :2].isfinite().all()
    assert out[2:6].isfinite().all()
    portion = out[6:]
    assert portion[20:, :2, :32].isnan().all() and portion[20:, :2, 32:].isfinite().all() and portion[:, 2:].isfinite().all()
    assert portion[:20].isfinite().all()
    # a window that has passed position 3 does not see it
    assert attend_run(built, window=20).float().cpu().view(-1, 4, 64)[:6].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_attend_pages_given_back_are_not_seen(dtype):
    """Of a context whose first pages are gone a token sees the rest; of one with no page at all, nothing: zeros."""
    built = attend_case(4, 2, 64, 8, [63, 5], [1, 1], dtype)
    built["table"][0, :3] = -1
    built["table"][1, :] = -1
    out = attend_run(built)
    keys, values = built["held"][0]
    q = built["q"][:1].view(1, 4, 64)
    exact, size = plain.attention(q, keys[24:], values[24:], torch.tensor([39]), 64 ** -0.5)
    off = (out[:1].cpu().double().view(1, 4, 64) - exact).abs()
    assert (off <= (6 * 2.0 ** -8 if dtype == BF16 else 1e-5) * size).all()
    assert (out[1] == 0).all()


def test_attend_leaves_other_rows_alone():
    built = attend_case(4, 2, 64, 8, [10, 12], [2, 40], BF16)
    out = torch.full((50, 4 * 64), 9.0, dtype=BF16, device="cuda")
    built["q"] = torch.cat((built["q"], torch.zeros(8, 4 * 64, dtype=BF16)))
    attend_run(built, out=out)
    assert (out[42:] == 9.0).all() and not (out[:42] == 9.0).all(-1).any()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_store_attend_recorded_and_replayed(dtype):
    """A token's store, attention and read as they follow one another in a step, recorded once and replayed with other inputs, on another
    stream than the default one."""
    module = kv4()
    torch.manual_seed(5)
    hq, hkv, dim, page = 8, 2, 128, 16
    built = attend_case(hq, hkv, dim, page, [200, 33], [1, 1], dtype)
    pages, table = built["pages"].cuda(), built["table"].cuda()
    proj = torch.randn(2, (hq + 2 * hkv) * dim).to(dtype).cuda()
    positions, rows = torch.tensor([200, 33], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda()
    freq = (1e6 ** (-torch.arange(0, dim, 2).double() / dim)).float().cuda()
    plan, extras = module.StepPlan.of_segments([0, 1], [200, 33], [1, 1], "cuda"), {}
    q = torch.empty(2, hq * dim, dtype=dtype, device="cuda")
    out = torch.empty_like(q)

    def step(pages, q, out, extras):
        module.store(proj, (0, hq * dim, (hq + hkv) * dim), q, pages, positions, rows, table, hq, hkv, dim, page, freq=freq, rot_dims=dim, unit_heads=True, eps=EPS)
        module.attend(plan, q, pages, out, table, hq, hkv, dim, page, dim ** -0.5, extras=extras)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(pages, q, out, extras)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(pages, q, out, extras)
        for turn in range(3):
            proj.copy_(torch.randn(proj.shape).to(dtype))
            graph.replay()
            other_pages, other_q, other = pages.clone(), torch.empty_like(q), torch.empty_like(out)
            step(other_pages, other_q, other, {})
            assert torch.equal(other, out) and torch.equal(other_q, q) and torch.equal(other_pages, pages)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    # and the last turn is right
    hold = module.read(pages, table, torch.tensor([0, 0, 201, 0, 1, 0, 34, 4], dtype=torch.int32, device="cuda"), 2, 201,
                       torch.zeros(5, 2, hkv, 64, dim, dtype=F32, device="cuda"), hkv, dim, page).cpu().double()
    for i, (at, n) in enumerate(((0, 201), (4, 34))):
        keys, values = (hold[at:at + 4, plane].transpose(1, 2).reshape(-1, hkv, dim)[:n] for plane in (0, 1))
        exact, size = plain.attention(q[i:i + 1].cpu().view(1, hq, dim), keys, values, torch.tensor([n - 1]), dim ** -0.5)
        off = (out[i].cpu().double().view(1, hq, dim) - exact).abs()
        assert (off <= (6 * 2.0 ** -8 if dtype == BF16 else 1e-5) * size).all()


def test_scratch_grows_with_the_work():
    """One dict for calls of all sizes: small, large, small again."""
    extras = {}
    for case in (ATTENDS[0], ATTENDS[2], ATTENDS[8], ATTENDS[11], ATTENDS[2]):
        *sizes, window = case
        for dtype in (BF16, F32):
            built = attend_case(*sizes, dtype)
            attend_check(built, attend_run(built, window, extras=extras), window)


# ------------------------------------------------------------------ refusals
def test_refusals():
    module = kv4()
    z = lambda *shape, dtype=BF16: torch.zeros(shape, dtype=dtype, device="cuda")
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    pages = z(4, 2, 2, 2, 320, dtype=torch.uint8)
    good = dict(proj=z(3, 8 * 64), columns=(0, 256, 384), q_out=z(3, 256), pages=pages, positions=ints(3), token_row=ints(3), block_table=ints(1, 4),
                n_q_heads=4, n_kv_heads=2, head_dim=64, page_size=16)
    module.store(**good)
    for wrong in (dict(proj=z(3, 8 * 64, dtype=torch.float16)), dict(q_out=z(3, 256, dtype=F32)), dict(q_out=z(2, 256)), dict(columns=(0, 256, 400)),
                  dict(columns=(-1, 256, 384)), dict(pages=z(4, 2, 2, 2, 160, dtype=torch.uint8)), dict(pages=z(4, 2, 2, 2, 320)), dict(pages=pages.cpu()),
                  dict(page_size=12), dict(page_size=8), dict(head_dim=48), dict(positions=ints(2)), dict(token_row=torch.zeros(3, device="cuda")),
                  dict(block_table=ints(4)), dict(rot_dims=3), dict(rot_dims=66), dict(rot_dims=64), dict(rot_dims=64, table=z(9, 32, dtype=F32)),
                  dict(rot_dims=64, freq=z(16, dtype=F32)), dict(rot_dims=64, freq=z(32, dtype=F32), table=z(9, 64, dtype=F32)), dict(layout=2),
                  dict(q_norm_w=z(64)), dict(q_norm_w=z(32), k_norm_w=z(32)), dict(q_norm_w=z(64), k_norm_w=z(64), unit_heads=True),
                  dict(q_norm_w=z(64), k_norm_w=z(64, dtype=F32)), dict(proj=z(3, 16 * 64)[:, ::2]), dict(n_kv_heads=3), dict(n_q_heads=0)):
        refused(module.store, **{**good, **wrong})
    info = torch.tensor([0, 0, 5, 0], dtype=torch.int32, device="cuda")
    good = dict(pages=pages, block_table=ints(1, 4), info=info, segments=1, longest=5, out=z(1, 2, 2, 8, 64), n_kv_heads=2, head_dim=64, page_size=16)
    module.read(**good)
    for wrong in (dict(out=z(1, 2, 2, 8, 32)), dict(out=z(1, 1, 2, 8, 64)), dict(out=z(1, 2, 2, 8, 64, dtype=torch.float16)), dict(info=info[:3]),
                  dict(segments=2), dict(pages=pages[:, :1]), dict(info=info.long()), dict(page_size=32)):
        refused(module.read, **{**good, **wrong})
    plan = module.StepPlan.of_segments([0], [3], [2], "cuda")
    good = dict(plan=plan, q=z(2, 256), pages=pages, out=z(2, 256), block_table=ints(1, 4), n_q_heads=4, n_kv_heads=2, head_dim=64, page_size=16, scale=0.125, extras={})
    module.attend(**good)
    for wrong in (dict(q=z(2, 256, dtype=F32)), dict(q=z(2, 256, dtype=torch.float16), out=z(2, 256, dtype=torch.float16)), dict(out=z(1, 256)), dict(n_q_heads=3),
                  dict(n_kv_heads=4), dict(window=-1), dict(page_size=8), dict(pages=pages.cpu()), dict(block_table=ints(4)), dict(q=z(2, 512)[:, ::2])):
        refused(module.attend, **{**good, **wrong})
    refused(module.StepPlan.of_segments, [0], [3], [0], "cuda")
    refused(module.StepPlan.of_segments, [0, 1], [3], [1], "cuda")
    refused(module.StepPlan.of_segments, [0], [-1], [1], "cuda")


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 256])
def test_attend_queries_of_any_size(dtype, dim):
    """Zero and tiny queries weigh all they see alike; one that is 10^30 times a key sees that key only.  Single tokens, a few and a portion."""
    case = attend_case(4, 2, dim, 16, [90, 70, 40], [1, 3, 60], dtype, seed=5)
    q, first = case["q"].view(-1, 4, dim), 0
    q[:, 0], q[:, 1] = 0.0, 1e-30 * q[:, 1]
    for i, n in enumerate(case["lens"]):
        q[first:first + n, 2:] = (1e30 * case["held"][i][0][7, 1].to(q.dtype)).to(dtype)
        first += n
    got, first = attend_run(case).cpu().double().view(-1, 4, dim), 0
    for i, (start, n) in enumerate(zip(case["starts"], case["lens"])):
        values = case["held"][i][1]
        for t in range(n):
            seen = values[:start + t + 1, 0]
            # p rounded (2^-8), its product with a step once more: 2^-8 of what is weighed each; the result once; float32 sums
            bar = (3 * 2.0 ** -8 if dtype == BF16 else 2.0 ** -18) * seen.abs().amax(0)
            assert ((got[first + t, :2] - seen.mean(0)).abs() <= bar).all()
            one = values[7, 1]
            bar = (4 * 2.0 ** -8 if dtype == BF16 else 2.0 ** -18) * values[:start + t + 1, 1].abs().amax()
            assert ((got[first + t, 2:] - one).abs() <= bar).all()
        first += n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("case", [
    (40, 1, 64, 16, [70, 5, 0], [1, 2, 33]),                  # more heads on a key than few tokens have rows
    (14, 2, 160, 8, [40, 3], [1, 6]),                         # a head size that no model here has
    (2, 2, 224, 64, [0, 65], [70, 1]),
    (33, 3, 32, 8, [300], [12]),
], ids=["40_1x64", "14_2x160", "2_2x224", "33_3x32"])
def test_attend_unusual_shapes(case, dtype):
    built = attend_case(*case, dtype, seed=11)
    attend_check(built, attend_run(built))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_attend_nothing_and_windows_that_hide_nothing(dtype):
    module = kv4()
    built = attend_case(8, 2, 64, 16, [100, 20], [1, 40], dtype, seed=3)
    open_out = attend_run(built)
    for window in (141, 1 << 31, 1 << 40):
        assert torch.equal(attend_run(built, window), open_out)
    out = torch.full((3, 512), 7.0, dtype=dtype, device="cuda")
    empty = module.StepPlan.of_segments([], [], [], "cuda")
    module.attend(empty, torch.zeros_like(out), built["pages"].cuda(), out, built["table"].cuda(), 8, 2, 64, 16, 0.125, extras={})
    assert (out == 7.0).all()


def test_rows_outside_the_table_are_rows_without_pages():
    """A plan may name a row that the table does not have: nothing is seen there, nothing is written."""
    module = kv4()
    built = attend_case(4, 2, 64, 16, [20], [1], BF16, seed=4)
    plan = module.StepPlan.of_segments([7], [20], [1], "cuda")
    assert (attend_run(built, plan=plan) == 0).all()
    case = dict(built, q=built["q"].float(), dtype=F32)
    assert (attend_run(case, plan=plan) == 0).all()
    info = torch.tensor([9, 0, 16, 0], dtype=torch.int32, device="cuda")
    back = torch.full((1, 2, 2, 16, 64), 5.0, device="cuda")
    module.read(built["pages"].cuda(), built["table"].cuda(), info, 1, 16, back, 2, 64, 16)
    assert (back == 0).all()
    pages, proj = built["pages"].cuda(), torch.randn(1, 512, device="cuda")
    one = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")
    for row, position in ((9, 0), (-1, 0), (0, -1), (0, 1 << 30)):
        module.store(proj, (0, 256, 384), torch.empty(1, 256, device="cuda"), pages, one(position), one(row), built["table"].cuda(), 4, 2, 64, 16)
    assert torch.equal(pages.cpu(), built["pages"])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
def test_a_table_written_right_before(dtype):
    """The block table, the queries and the scratch are the previous kernel's: a plan of the caller's is read after it."""
    module = kv4()
    built = attend_case(8, 2, 128, 16, [600, 33, 1], [1, 1, 4], dtype, seed=8)
    plan = module.StepPlan.of_segments(range(3), built["starts"], built["lens"], "cuda")
    right, q, pages = built["table"].cuda(), built["q"].cuda(), built["pages"].cuda()
    expected, extras = attend_run(built), {}
    table, out = torch.empty_like(right), torch.empty_like(q)
    for _ in range(20):
        table.fill_(-1)
        out.fill_(math.nan)
        torch.add(right, 0, out=table)
        module.attend(plan, q, pages, out, table, 8, 2, 128, 16, 128 ** -0.5, extras=extras)
        assert torch.equal(out, expected)


def test_another_stream():
    """Work queued on a stream of the caller's: store, attend and read there, in order."""
    module = kv4()
    built = attend_case(8, 2, 64, 16, [50, 9], [1, 30], BF16, seed=6)
    expected, stream = attend_run(built), torch.cuda.Stream()
    plan = module.StepPlan.of_segments(range(2), built["starts"], built["lens"], "cuda")
    q, pages, table, extras = built["q"].cuda(), built["pages"].cuda(), built["table"].cuda(), {}
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        outs = []
        for _ in range(5):
            outs.append(torch.empty_like(q))
            module.attend(plan, q, pages, outs[-1], table, 8, 2, 64, 16, 0.125, extras=extras)
    other = torch.empty_like(q)
    module.attend(plan, q, pages, other, table, 8, 2, 64, 16, 0.125, extras={})            # beside it, scratch of its own
    torch.cuda.synchronize()
    assert all(torch.equal(out, expected) for out in (*outs, other))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("clusters", [True, False], ids=["clusters", "memory"])
def test_two_graphs_and_a_call_share_scratch(dtype, clusters, monkeypatch):
    """Recorded before any other call with the dict, replayed one after another in any order, calls in between, after larger ones replaced
    the scratch."""
    module = kv4()
    if not clusters:
        monkeypatch.setattr(module, "CLUSTERS", {1: (), 2: ()})
    built = attend_case(8, 2, 64, 16, [2000, 700], [1, 1], dtype, seed=9)
    large = attend_case(8, 2, 64, 16, [900] * 9 + [10], [1] * 9 + [90], dtype, seed=10)
    expected, expected_large = attend_run(built), attend_run(large)
    plan = module.StepPlan.of_segments(range(2), built["starts"], built["lens"], "cuda")
    q, pages, table, extras, graphs = built["q"].cuda(), built["pages"].cuda(), built["table"].cuda(), {}, []
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(2):
            out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                module.attend(plan, q, pages, out, table, 8, 2, 64, 16, 0.125, extras=extras)
            graphs.append((graph, out))
        for turn, which in enumerate((1, 0, 1, 1, 0, 0)):
            if turn in (1, 3):
                assert torch.equal(attend_run(large, extras=extras), expected_large)
            assert torch.equal(attend_run(built, extras=extras), expected)
            graph, out = graphs[which]
            out.fill_(math.nan)
            graph.replay()
            assert torch.equal(out, expected)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("lens", [[1, 4], [150, 40]], ids=["few", "portions"])
def test_attend_values_of_all_sizes(lens, window, dtype):
    """Pages whose values are 10^-20 beside pages of 10^6 and of zeros: rows that see the small ones only have them as exactly as others."""
    starts = [700 - n for n in lens]
    built = attend_case(8, 2, 64, 16, starts, lens, dtype, seed=12)
    sizes = torch.tensor([1e-20, 1e3, 0.0, 1e-3, 1.0, 1e-12, 30.0, 1e6, 0.0, 1e-20, 1e-20, 5.0])[:, None, None]
    keys = [held[0] for held in built["held"]]
    values = [held[1].float() * sizes.repeat_interleave(64, dim=0)[:700] for held in built["held"]]
    pages, table, held = plain.build(keys, values, [700, 700], 16, seed=1)
    built.update(pages=pages, table=table, held=held)
    attend_check(built, attend_run(built, window), window)


@pytest.mark.parametrize("lens", [[1, 4], [150, 40]], ids=["few", "portions"])
def test_attend_groups_of_other_sizes(lens):
    """A head whose groups of values are up to 2^10 apart, and one of zeros: every group as exact as if it were alone."""
    starts = [300 - n for n in lens]
    built = attend_case(8, 2, 128, 16, starts, lens, BF16, seed=14)
    sizes = torch.tensor([1.0, 2.0 ** -10, 0.0, 2.0 ** -5]).repeat_interleave(32)
    keys, values = [held[0].float() for held in built["held"]], [held[1].float() * sizes for held in built["held"]]
    pages, table, held = plain.build(keys, values, [300, 300], 16, seed=2)
    built.update(pages=pages, table=table, held=held)
    attend_check(built, attend_run(built))


@pytest.mark.parametrize("size", [1e-30, 3e-5, 1e25])
@pytest.mark.parametrize("lens", [[1, 4], [150, 40]], ids=["few", "portions"])
def test_attend_values_all_of_one_size(lens, size):
    starts = [300 - n for n in lens]
    built = attend_case(8, 2, 64, 16, starts, lens, BF16, seed=13)
    keys, values = ([held[i].float() * (size if i else 1.0) for held in built["held"]] for i in (0, 1))
    pages, table, held = plain.build(keys, values, [300, 300], 16, seed=2)
    built.update(pages=pages, table=table, held=held)
    attend_check(built, attend_run(built))
