"""The operators of a paged cache that holds keys and values in 4 bits, as cases that can be timed and compared.

A row of a head (a key after its norm and rotation, a value as projected) is held in groups of 32 neighbouring elements:
``m`` = the smallest element and ``s`` = a fifteenth of the range, both in bfloat16, and for each element the 4-bit code
``rint((y - m) / s)`` within 0 .. 15; the value held is ``m + s * code``.  A page is uint8
[2 (keys, values), kv heads, page size / 8, 160 * groups]: of every run of 8 slots first the codes [groups, 8, 16] (element i
of a group in byte i // 2, the even ones in the low half), then the pairs (s, m) [8, groups, 2].

``op``        ``store``: the tail of a q/k/v projection: norms, rotates, queries out, keys and values into the pages; the rows that were
              written are read back as the values they stand for.  ``read``: the rows of requests as ordinary pages.
              ``attend``: attention of single tokens and of prompt portions over the pages
``hq hkv dim``    query heads, kv heads, head size;  ``page``: cache positions per page
``norm``      ``heads``: every q and k head by its root mean square, times a weight; ``unit``: without a weight; ``none``
``rotary``    ``table``: cosines and sines of every position in a table; ``halves`` or ``interleaved``: from frequencies
              (``rot`` dimensions, the rest unturned), stretched by YaRN's ramp where ``gain`` is not 1
``decodes``   requests that bring one token each behind ``context`` cached ones; ``prompts`` requests that bring ``portion`` tokens
              each behind ``prefix`` cached ones; ``ragged``: lengths in eight levels; ``window``: positions seen (0: all)
"""
import math

import torch

own = False
GROUP = 32
EPS = 1e-6
LEVELS = 8
READ_PAGE = 64


def _case(name, op, dtype, hq, hkv, dim, *, page=16, norm="heads", rotary="table", rot=0, gain=1.0, decodes=0, context=0,
          prompts=0, portion=0, prefix=0, ragged=False, window=0):
    case = dict(op=op, dtype=dtype, hq=hq, hkv=hkv, dim=dim, page=page, norm=norm, rotary=rotary, rot=rot or dim, gain=gain,
                decodes=decodes, context=context, prompts=prompts, portion=portion, prefix=prefix, ragged=ragged,
                window=window)
    return dict(name=name, **case) if name else case


def listed():
    big, small = (32, 8, 128), (16, 8, 128)      # heads of the 8b and 0.6b models of the benchmark
    return [
        # what every decoded token of a single user pays in each layer: latency
        _case("store_1", "store", "bfloat16", *big, decodes=1, context=8192),
        # a serving batch far into long contexts: frequencies stretched by a ramp, neighbours paired, half of the head turned, 32 bits
        _case("store_40_f32_far", "store", "float32", 16, 2, 64, norm="unit", rotary="interleaved", rot=32, gain=1.2,
              decodes=40, context=120011, ragged=True, page=32),
        # the benchmark's prompt
        _case("store_2048", "store", "bfloat16", *big, prompts=1, portion=2048),
        # a long request's rows for somebody who wants them in 16 bits, and odd lengths of odd heads in 32 bits
        _case("read_8192", "read", "bfloat16", *big, prompts=1, portion=1, prefix=8191),
        _case("read_7_f32_ragged", "read", "float32", 6, 2, 96, prompts=7, portion=3, prefix=1007, ragged=True, page=8),
        # one user behind a long chat; the benchmark's decode point; a serving batch of all lengths
        _case("decode_1", "attend", "bfloat16", *big, decodes=1, context=8191),
        _case("decode_8", "attend", "bfloat16", *big, decodes=8, context=8191),
        _case("decode_48_ragged", "attend", "bfloat16", *big, decodes=48, context=16383, ragged=True),
        # the true 32-bit path with a sliding window
        _case("decode_5_f32_window", "attend", "float32", 12, 4, 64, decodes=5, context=3001, ragged=True, window=1000, page=8),
        # a few tokens at a time behind a context: guesses to verify, or what is left of a prompt
        _case("draft_8_of_5", "attend", "bfloat16", *small, prompts=8, portion=5, prefix=4001),
        # chunked prefill: the last portion of a long prompt beside requests that already run
        _case("chunk_beside_decode", "attend", "bfloat16", *big, prompts=1, portion=509, prefix=6001, decodes=12,
              context=3000, ragged=True),
        # the benchmark's prompt
        _case("prompt_2048", "attend", "bfloat16", *big, prompts=1, portion=2048),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choices(("store", "read", "attend"), (5, 3, 10))[0]
    dim = rng.choices((32, 64, 96, 128, 256), (1, 4, 2, 9, 1))[0]
    hkv = rng.choice((1, 2, 4, 8) if dim <= 128 else (1, 2, 4))
    hq = hkv * rng.choice((1, 2, 3, 4, 5, 7, 8, 16) if hkv <= 4 else (1, 2, 4, 5))
    dtype = rng.choices(("bfloat16", "float32"), (3, 1))[0]
    case = dict(page=rng.choice((8, 16, 16, 32, 64)), ragged=rng.random() < 0.6)
    if op == "store":
        case.update(norm=rng.choice(("heads", "heads", "unit", "none")), rotary=rng.choice(("table", "halves", "interleaved")),
                    rot=rng.choice((dim, dim, dim // 2)), gain=1.0)
        if case["rotary"] != "table" and rng.random() < 0.4:
            case["gain"] = 1.0 + 0.1 * math.log(rng.choice((4, 16, 40)))
        far = 30000 if case["rotary"] == "table" else 400000
        if rng.random() < 0.5:
            case.update(decodes=_log_uniform(rng, 1, 200), context=_log_uniform(rng, 1, far))
        else:
            prompts = rng.choice((1, 1, 2, 3))
            case.update(prompts=prompts, portion=_log_uniform(rng, 2, 2048 // prompts), prefix=_log_uniform(rng, 1, far))
        return _case(None, op, dtype, hq, hkv, dim, **case)
    rows = 8 * 128 * 8192 // (hkv * dim)                # cached positions of all requests: as much as decode_8 reads
    if op == "read":
        prompts = _log_uniform(rng, 1, 12)
        case.update(prompts=prompts, portion=rng.randint(1, 9), prefix=_log_uniform(rng, 1, min(rows // prompts, 40000)))
        return _case(None, op, dtype, hq, hkv, dim, **case)
    kind = rng.choices(("decode", "portions", "mixed"), (6, 5, 4))[0]
    rows = min(rows, 40000) if dtype == "float32" or kind != "decode" else rows
    case["window"] = rng.choice((0, 0, 0, _log_uniform(rng, 16, 4000)))
    if kind != "portions":
        decodes = _log_uniform(rng, 1, 64)
        case.update(decodes=decodes, context=_log_uniform(rng, 1, min(40000, max(1, rows // decodes))))
    if kind != "decode":
        prompts = rng.choice((1, 1, 2, 5, 8))
        portion = _log_uniform(rng, 2, (1024 if dtype == "bfloat16" else 256) // prompts)
        case.update(prompts=prompts, portion=portion, prefix=_log_uniform(rng, 1, min(8000, rows // prompts)))
        if rng.random() < 0.3:
            case["prefix"] = 0
    return _case(None, op, dtype, hq, hkv, dim, **case)


# ------------------------------------------------------------------ the batch
def _segments(case):
    """(cached positions, new tokens) of every request, those with a single token first."""
    def level(value, i):
        return value - (i % LEVELS) * (value // (LEVELS + 1)) if case["ragged"] else value
    return [(level(case["context"], i), 1) for i in range(case["decodes"])] \
        + [(level(case["prefix"], i), level(case["portion"], i)) for i in range(case["prompts"])]


def _flat(case, device):
    """Absolute position and request of every token of the flat batch."""
    segments = _segments(case)
    positions = torch.cat([torch.arange(cached, cached + new) for cached, new in segments])
    rows = torch.repeat_interleave(torch.arange(len(segments)), torch.tensor([new for _, new in segments]))
    return positions.to(torch.int32).to(device), rows.to(torch.int32).to(device)


def _to_be_read(case):
    """(request, first position, positions, first page of the output) of what ``read`` returns, the positions in a page of it, and the pages."""
    segments, found, pages = _segments(case), [], 0
    per_page = 1 if case["op"] == "store" and all(new == 1 for _, new in segments) else READ_PAGE
    for i, (cached, new) in enumerate(segments):
        first, count = (cached, new) if case["op"] == "store" else (0, cached + new)
        found.append((i, first, count, pages))
        pages += -(-count // per_page)
    return found, per_page, pages


def _frequencies(case):
    """Of every turned pair, float32: base 1e6, or with a gain stretched by YaRN's ramp (factor e^(10 (gain - 1)) over 32768 positions)."""
    dims, base = case["rot"], 1e6
    values = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if case["gain"] != 1.0:
        factor = math.exp(10.0 * (case["gain"] - 1.0))
        pair = lambda turns: dims * math.log(32768 / (2.0 * math.pi * turns)) / (2.0 * math.log(base))
        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), dims - 1)
        for i, f in enumerate(values):
            slowed = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            values[i] = f / factor * slowed + f * (1.0 - slowed)
    return torch.tensor(values, dtype=torch.float64).float()


# ------------------------------------------------------------------ inputs
def _packed(rows):
    """[n, 2, kv heads, slots, dim] in 32 bits -> pages (in 64 bits: which code an element gets)."""
    n, planes, heads, slots, dim = rows.shape
    y = rows.double().view(n, planes, heads, slots, dim // GROUP, GROUP)
    m = y.amin(-1).float().bfloat16()
    s = ((y.amax(-1) - y.amin(-1)) / 15.0).float().bfloat16()
    wide = s.double()[..., None]
    code = torch.where(wide > 0, (y - m.double()[..., None]) / wide, torch.zeros_like(y)).round().clamp(0, 15)
    good = (torch.isfinite(m) & torch.isfinite(s) & torch.isfinite(y).all(-1))[..., None]
    code = torch.where(good, code, torch.zeros_like(code)).to(torch.uint8)
    pairs = torch.where(good, torch.stack((s, m), -1), torch.full_like(s, math.nan)[..., None])
    codes = (code[..., 0::2] | code[..., 1::2] << 4).view(n, planes, heads, slots // 8, 8, dim // GROUP, 16)
    codes = codes.transpose(-2, -3).reshape(n, planes, heads, slots // 8, -1)
    return torch.cat((codes, pairs.reshape(n, planes, heads, slots // 8, -1).view(torch.uint8)), -1)


def _held(case, pages):
    """The float32 values that pages [n, 2, kv heads, runs of 8, bytes] stand for: [n, 2, kv heads, slots, dim]."""
    groups = case["dim"] // GROUP
    n, planes, heads, runs, _ = pages.shape
    codes = pages[..., :128 * groups].reshape(n, planes, heads, runs, groups, 8, 16)
    pairs = pages[..., 128 * groups:].contiguous().view(torch.bfloat16).view(n, planes, heads, runs, 8, groups, 2).float()
    code = torch.stack((codes & 15, codes >> 4), -1).view(n, planes, heads, runs, groups, 8, GROUP).transpose(4, 5)
    return (pairs[..., 1:] + pairs[..., :1] * code.float()).reshape(n, planes, heads, runs * 8, case["dim"])


def _inputs(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device).manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    segments = _segments(case)
    positions, rows = _flat(case, device)
    n = len(positions)
    normal = lambda *shape: torch.randn(shape, generator=g, device=device)
    # a few channels of the keys are several times as large as the others, as in trained models
    loud = 1.0 + 3.0 * (torch.rand((hkv, 1, dim), generator=g, device=device) < 0.06).float()
    needed = [-(-(cached + new) // page) for cached, new in segments]
    held = [(new + cached % page + page - 1) // page for cached, new in segments] if case["op"] == "store" else needed
    # pages in no order; of a store case only those that are written exist
    order = torch.randperm(sum(held), generator=g, device=device).to(torch.int32)
    table = torch.full((len(segments), max(needed)), -1, dtype=torch.int32, device=device)
    begin = 0
    for i, (whole, some) in enumerate(zip(needed, held)):
        table[i, whole - some:whole] = order[begin:begin + some]
        begin += some
    state = dict(case=case, positions=positions, rows=rows, table=table, segments=segments)
    runs = page // 8
    if case["op"] == "store":
        projected = normal(n, (hq + 2 * hkv) * dim)
        projected[:, hq * dim:(hq + hkv) * dim] *= loud.view(1, -1)
        state.update(proj=projected.to(dtype), q_out=torch.zeros((n, hq * dim), dtype=dtype, device=device),
                     pages=torch.zeros((sum(held), 2, hkv, runs, 5 * dim), dtype=torch.uint8, device=device))
        if case["norm"] == "heads":
            state.update(q_norm=(1.0 + 0.05 * normal(dim)).to(dtype), k_norm=(1.0 + 0.05 * normal(dim)).to(dtype))
        if case["rotary"] == "table":       # as a model makes it: angles in 32 bits, cosines and sines rounded to its type
            inverse = 1.0 / (1e6 ** (torch.arange(0, case["rot"], 2, dtype=torch.float32) / case["rot"]))
            angles = torch.arange(int(positions.max()) + 1).float()[:, None] * inverse[None, :]
            state["rotary"] = torch.cat((angles.cos(), angles.sin()), -1).to(dtype).float().to(device)
        else:
            state["rotary"] = _frequencies(case).to(device)
    else:
        pages = torch.empty((sum(held), 2, hkv, runs, 5 * dim), dtype=torch.uint8, device=device)
        at_once = max(1, (1 << 25) // (2 * hkv * page * dim))
        for first in range(0, len(pages), at_once):
            some = normal(min(at_once, len(pages) - first), 2, hkv, page, dim)
            some[:, 0] *= loud
            pages[first:first + at_once] = _packed(some)
        state["pages"] = pages
        if case["op"] == "attend":
            state["q"] = (1.5 * normal(n, hq * dim)).to(dtype)
            state["out"] = torch.zeros((n, hq * dim), dtype=dtype, device=device)
    if case["op"] != "attend":
        wanted, per_page, count = _to_be_read(case)
        state.update(wanted=wanted, back=torch.zeros((count, 2, hkv, per_page, dim), dtype=dtype, device=device))
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        from qwen_inference_lab_b200.kernels import kv4
        device = state["table"].device
        if case["op"] == "attend":          # what the engine uploads with a step, and what its runner keeps between steps
            starts, lens = zip(*state["segments"])
            state["plan"] = kv4.StepPlan.of_segments(range(len(starts)), starts, lens, device)
            state["extras"] = {}
        else:
            state["info"] = torch.tensor(state["wanted"], dtype=torch.int32).view(-1).to(device)
            state["longest"] = max(count for _, _, count, _ in state["wanted"])
    return state


# ------------------------------------------------------------------ one pass
def _turned(case, x, cosines, sines):
    """The first ``rot`` dimensions of every row of x [n, heads, dim] turned; cosines, sines [n, 1, rot / 2]."""
    rot = case["rot"]
    if case["rotary"] == "interleaved":
        u, v = x[..., 0:rot:2], x[..., 1:rot:2]
        front = torch.stack((u * cosines - v * sines, v * cosines + u * sines), -1).flatten(-2)
    else:
        u, v = x[..., :rot // 2], x[..., rot // 2:rot]
        front = torch.cat((u * cosines - v * sines, v * cosines + u * sines), -1)
    return torch.cat((front, x[..., rot:]), -1)


def _normed(case, x, weight):
    if case["norm"] == "none":
        return x
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x if weight is None else x * weight.to(x.dtype)


def _store(state):
    case = state["case"]
    n, hq, hkv, dim, page = len(state["positions"]), case["hq"], case["hkv"], case["dim"], case["page"]
    positions, rot = state["positions"].long(), case["rot"]
    if case["rotary"] == "table":
        cosines, sines = state["rotary"][positions].double().split(rot // 2, -1)
    else:                                   # angles of far positions: 64 bits
        angles = positions.double()[:, None] * state["rotary"].double()[None, :]
        cosines, sines = case["gain"] * angles.cos(), case["gain"] * angles.sin()
    cosines, sines = cosines[:, None], sines[:, None]
    q, k, v = (part.view(n, -1, dim) for part in state["proj"].split((hq * dim, hkv * dim, hkv * dim), -1))
    unit = case["norm"] == "unit"           # heads of unit size are those of the turned heads
    after = lambda x: _normed(case, x, None) if unit else x
    before = lambda x, weight: x if unit else _normed(case, x, weight)
    q = after(_turned(case, before(q.float(), state.get("q_norm")), cosines.float(), sines.float()))
    state["q_out"].copy_(q.reshape(n, -1))
    # 64 bits decide which code an element gets where it lies between two
    k = after(_turned(case, before(k.double(), state.get("k_norm")), cosines, sines))
    both = torch.stack((k, v.double()), 1)[:, :, :, None].expand(-1, -1, -1, 8, -1)
    run = _packed(both)[:, :, :, 0]         # [n, 2, heads, bytes] of runs whose 8 slots hold the same row
    groups = dim // GROUP
    where = state["table"][state["rows"].long(), positions // page].long()
    into = state["pages"][..., :128 * groups].unflatten(-1, (groups, 8, 16))
    into[where, :, :, positions % page // 8, :, positions % 8] = run[..., :128 * groups].unflatten(-1, (groups, 8, 16))[..., 0, :]
    into = state["pages"][..., 128 * groups:].unflatten(-1, (8, groups * 4))
    into[where, :, :, positions % page // 8, positions % 8] = run[..., 128 * groups:].unflatten(-1, (8, groups * 4))[..., 0, :]


def _rows_held(state, request, first, count):
    """float32 [2, kv heads, count, dim]: the values of a request's positions."""
    case, page = state["case"], state["case"]["page"]
    begin, end = first // page, -(-(first + count) // page)
    held = _held(case, state["pages"][state["table"][request, begin:end].long()])
    held = held.permute(1, 2, 0, 3, 4).reshape(2, case["hkv"], -1, case["dim"])
    return held[:, :, first - begin * page:first - begin * page + count]


def _read(state):
    back = state["back"]
    per_page = back.shape[3]
    for request, first, count, at in state["wanted"]:
        rows = _rows_held(state, request, first, count)
        for begin in range(0, count, per_page):
            some = rows[:, :, begin:begin + per_page]
            back[at + begin // per_page, :, :, :some.shape[2]] = some.to(back.dtype)


def _attend(state):
    case, out = state["case"], state["out"]
    hq, hkv, dim, window = case["hq"], case["hkv"], case["dim"], case["window"]
    first = 0
    for request, (cached, new) in enumerate(state["segments"]):
        keys, values = _rows_held(state, request, 0, cached + new)
        at_once = max(1, (1 << 28) // (hq * (cached + new)))
        for begin in range(0, new, at_once):
            some = min(at_once, new - begin)
            rows = slice(first + begin, first + begin + some)
            q = state["q"][rows].float().view(some, hkv, hq // hkv, dim).permute(1, 2, 0, 3).reshape(hkv, -1, dim)
            scores = (q @ keys.transpose(1, 2)).view(hkv, hq // hkv, some, -1) * dim ** -0.5
            if some > 1 or window:
                at = torch.arange(cached + begin, cached + begin + some, device=q.device)[:, None]
                key = torch.arange(cached + new, device=q.device)[None, :]
                hidden = key > at
                if window:
                    hidden = hidden | (key <= at - window)
                scores = torch.where(hidden, torch.full_like(scores[:1, :1, :1, :1], -math.inf), scores)
            elif begin + some < new:
                scores = scores[..., :cached + begin + 1]
            weights = (scores - scores.amax(-1, keepdim=True)).exp()
            weights = weights / weights.sum(-1, keepdim=True)
            got = weights.view(hkv, -1, weights.shape[-1]) @ values[:, :weights.shape[-1]]
            out[rows] = got.view(hkv, hq // hkv, some, dim).permute(2, 0, 1, 3).reshape(some, -1).to(out.dtype)
        first += new


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "attend":
            _attend(state)
            return state["out"]
        if case["op"] == "store":
            _store(state)
        _read(state)
        return [state["q_out"], state["back"]] if case["op"] == "store" else state["back"]
    from qwen_inference_lab_b200.kernels import kv4
    hq, hkv, dim, page = case["hq"], case["hkv"], case["dim"], case["page"]
    if case["op"] == "attend":
        return kv4.attend(state["plan"], state["q"], state["pages"], state["out"], state["table"], hq, hkv, dim, page,
                          dim ** -0.5, window=case["window"], extras=state["extras"])
    if case["op"] == "store":
        table = case["rotary"] == "table"
        kv4.store(state["proj"], (0, hq * dim, (hq + hkv) * dim), state["q_out"], state["pages"], state["positions"],
                  state["rows"], state["table"], hq, hkv, dim, page, q_norm_w=state.get("q_norm"),
                  k_norm_w=state.get("k_norm"), eps=EPS, unit_heads=case["norm"] == "unit",
                  table=state["rotary"] if table else None, freq=None if table else state["rotary"], rot_dims=case["rot"],
                  layout=1 if case["rotary"] == "interleaved" else 0, gain=case["gain"])
    kv4.read(state["pages"], state["table"], state["info"], len(state["wanted"]), state["longest"], state["back"], hkv, dim, page)
    return [state["q_out"], state["back"]] if case["op"] == "store" else state["back"]


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    hq, hkv, dim, segments = case["hq"], case["hkv"], case["dim"], _segments(case)
    tokens = sum(new for _, new in segments)
    held = 2 * hkv * dim * 5 // 8                      # bytes of a cached position: 4 bits an element, 4 bytes a group of 32
    if case["op"] == "store":
        # the projection in, the queries and the cached rows out; those rows in again and their values out
        moved = tokens * ((2 * hq + 2 * hkv) * dim * size + 2 * held + 2 * hkv * dim * size)
        return {"bytes": moved, "flops": tokens * (hq + hkv) * dim * 8.0 + tokens * 2 * hkv * dim * 8.0}
    if case["op"] == "read":
        rows = sum(cached + new for cached, new in segments)
        return {"bytes": rows * (held + 2 * hkv * dim * size), "flops": rows * 2 * hkv * dim * 2.0}
    window = case["window"] or 1 << 60
    rows = sum(min(cached + new, window + new - 1) for cached, new in segments)
    pairs = 0
    for cached, new in segments:
        whole = max(0, min(new, window - cached))      # queries that see everything up to themselves
        pairs += whole * cached + whole * (whole + 1) // 2 + (new - whole) * min(window, cached + new)
    return {"bytes": rows * held + 2 * tokens * hq * dim * size, "flops": 4.0 * hq * dim * pairs}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_group(y):
    """The values that the last axis, 32 exact numbers, is held as."""
    low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
    base = low.to(torch.float32).to(torch.bfloat16).double()
    step = ((high - low) / 15).to(torch.float32).to(torch.bfloat16).double()
    code = torch.clamp(torch.round((y - base) / torch.where(step == 0, torch.ones_like(step), step)), 0, 15)
    return base + step * torch.where(step == 0, torch.zeros_like(code), code)


def _exact_rows(case, state, request, first, count):
    """float64 [2, kv heads, count, dim], position by position out of the bytes."""
    groups, page = case["dim"] // GROUP, case["page"]
    at = torch.arange(first, first + count, device=state["table"].device)
    physical = state["table"][request].long()[at // page]
    run, slot = at % page // 8, at % 8
    blob = state["pages"][physical, :, :, run].long()                      # [count, 2, heads, 160 groups]
    element = torch.arange(case["dim"], device=at.device)
    byte = (element // GROUP * 128 + element % GROUP // 2)[None, :] + (slot * 16)[:, None]
    byte = byte[:, None, None].expand(-1, 2, case["hkv"], -1)
    code = (blob.gather(-1, byte) >> (4 * (element % 2))) & 15

    def number(offset):     # a bfloat16 from its two bytes
        place = (128 * groups + element // GROUP * 4 + offset)[None, :] + (slot * 4 * groups)[:, None]
        place = place[:, None, None].expand(-1, 2, case["hkv"], -1)
        bits = blob.gather(-1, place) << 16 | blob.gather(-1, place + 1) << 24
        return torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32).view(torch.float32).double()

    return (number(2) + number(0) * code).permute(1, 2, 0, 3)


def _exact_store(case, state):
    hq, hkv, dim, rot = case["hq"], case["hkv"], case["dim"], case["rot"]
    rows = state["proj"].double().view(-1, hq + 2 * hkv, dim)
    n = len(rows)
    at = state["positions"].long()
    if case["rotary"] == "table":
        complexes = torch.complex(state["rotary"][at, :rot // 2].double(), state["rotary"][at, rot // 2:].double())
    else:
        angle = at.double()[:, None] * state["rotary"].double()
        complexes = case["gain"] * torch.polar(torch.ones_like(angle), angle)
    head = rows[:, :hq + hkv].clone()
    if case["norm"] == "heads":
        head *= torch.rsqrt(head.square().sum(-1, keepdim=True) / dim + EPS)
        head[:, :hq] *= state["q_norm"].double()
        head[:, hq:] *= state["k_norm"].double()
    if case["rotary"] == "interleaved":
        one, other = torch.arange(0, rot, 2), torch.arange(1, rot, 2)
    else:
        one, other = torch.arange(rot // 2), torch.arange(rot // 2, rot)
    one, other = one.to(head.device), other.to(head.device)
    pair = torch.complex(head[..., one], head[..., other]) * complexes[:, None]
    head[..., one], head[..., other] = pair.real, pair.imag
    if case["norm"] == "unit":
        head *= torch.rsqrt(head.square().sum(-1, keepdim=True) / dim + EPS)
    kept = torch.stack((head[:, hq:], rows[:, hq + hkv:]), 1)              # [n, 2, kv heads, dim]
    kept = _exact_group(kept.view(n, 2, hkv, dim // GROUP, GROUP)).view(n, 2, hkv, dim)
    back = torch.zeros(state["back"].shape, dtype=torch.float64, device=head.device)
    token = 0
    for _, _, count, page in state["wanted"]:
        for i in range(0, count, back.shape[3]):
            some = kept[token + i:token + min(count, i + back.shape[3])]
            back[page + i // back.shape[3], :, :, :len(some)] = some.permute(1, 2, 0, 3)
        token += count
    return [head[:, :hq].reshape(n, -1), back]


def exact(case, seed):
    state = _inputs(case, seed)
    if case["op"] == "store":
        return _exact_store(case, state)
    if case["op"] == "read":
        back = torch.zeros(state["back"].shape, dtype=torch.float64, device=state["back"].device)
        for request, first, count, page in state["wanted"]:
            rows = _exact_rows(case, state, request, first, count)
            for i in range(0, count, back.shape[3]):
                some = rows[:, :, i:i + back.shape[3]]
                back[page + i // back.shape[3], :, :, :some.shape[2]] = some
        return back
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    out, first = torch.empty(state["q"].shape, dtype=torch.float64, device=state["q"].device), 0
    for request, (cached, new) in enumerate(state["segments"]):
        rows = _exact_rows(case, state, request, 0, cached + new)
        for begin in range(0, new, 128):
            end = min(new, begin + 128)
            query = state["q"][first + begin:first + end].double().view(end - begin, hq, dim)
            low = max(0, cached + begin + 1 - case["window"]) if case["window"] else 0
            high = cached + end
            key = torch.arange(low, high, device=query.device)
            at = torch.arange(cached + begin, high, device=query.device)[:, None]
            seen = key <= at
            if case["window"]:
                seen &= key > at - case["window"]
            for head in range(hq):
                k, v = rows[0, head // (hq // hkv), low:high], rows[1, head // (hq // hkv), low:high]
                chances = (query[:, head] @ k.t() / math.sqrt(dim)).masked_fill(~seen, -math.inf).softmax(-1)
                out[first + begin:first + end, head * dim:(head + 1) * dim] = chances @ v
        first += new
    return out
