"""Measured cases of the operators for pages with images and for many readers
of one page: rotary positions on several axes (alone, and on the way into the
paged 8-bit cache), attention over a sliding window and a few first positions
that stay visible, for single rows and for prompts, and attention of sequences
that share a long beginning, which is read once for all of them.

Every case runs in two forms on the same prepared tensors: the plain one
(elementary torch operations in FP32) and, with ``own`` set, the calls of
``fo_cuda`` that a serving program makes.  ``exact`` states the same results in
64 bits, written apart from the plain form.

The cache: codes [pages][kv heads][page size][head dim] of int8 or FP8 (e4m3)
for keys and for values, one FP32 scale per (page, kv head) of each; a
sequence's pages are listed in a page table, and ``lens`` counts a sequence's
positions with the rows of the call included.  A row's place in the cache is
``len - rows + r``; where it stands in the rotation is given for each axis.
"""

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
THETA = 10000.0
QMAX = {"i8": 127.0, "e4m3": 448.0}
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _fo():
    path = os.path.join(ROOT, "falcon-ocr-cpu_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fo_cuda
    return fo_cuda


# ------------------------------------------------------------------ the cases
def listed():
    rope = dict(op="rope", rot=64, layout="half", axes="sections", image=0, inverse=False, fused_row=False)
    append = dict(op="append", rot=64, layout="half", axes="sections", image=0, ragged=False, groups=0,
                  table_positions=16384)
    window = dict(op="window", rows=1, ragged=False, sinks=True, lse=False, groups=0)
    prefix = dict(op="prefix", rows=1, ragged=False, groups=1, sinks=True, lse=False, window=0, first=0)
    return [
        # The 16 query and 8 key heads of eight sequences' newest tokens, the temporal half of each head turned on
        # three axes, in place of a decode step's rows: the smallest call, where only latency counts.
        dict(rope, name="rope axes step", rows=8, heads=24, dim=64, rot=32, dtype="bf16", table_positions=16384,
             fused_row=True),
        # Gradient of the rotation over frames of 64 x 64 patches and the text after them: wide heads, the axes
        # taking turns over the pairs, an odd number of rows.
        dict(rope, name="rope axes video gradient", rows=32771, heads=40, dim=128, rot=128, dtype="bf16",
             axes="turns", image=28672, inverse=True, table_positions=65536),
        # A page's whole prompt after its prefill, 4,096 tokens of its image and 2,448 of text, FP32 rows as the
        # prefill takes them, into 64-token pages.
        dict(append, name="append axes page", seqs=1, rows=6544, min_len=6544, max_len=6544, heads=16, kv_heads=8,
             dim=64, page=64, fmt="i8", dtype="f32", image=4096),
        # One short sequence, one row, small pages: the latency of a call.
        dict(window, name="window one short", seqs=1, min_len=777, max_len=777, heads=16, kv_heads=8, dim=64, page=16,
             fmt="i8", dtype="bf16", window=256, first=4),
        # 64 long pages being decoded at once, each row with the newest 4,096 positions and the first 16.
        dict(window, name="window 64 pages", seqs=64, min_len=6545, max_len=20001, heads=16, kv_heads=8, dim=64,
             page=64, fmt="i8", dtype="bf16", window=4096, first=16),
        # A whole page's 6,544 rows over their own positions, read in windows of 1,024 with the first 64 in sight.
        dict(window, name="window page prompt", seqs=1, rows=6544, min_len=6544, max_len=6544, heads=16, kv_heads=8,
             dim=64, page=64, fmt="i8", dtype="bf16", window=1024, first=64),
        # Prompts of very different lengths with wide heads and FP8 codes, some continuing a cached beginning.
        dict(window, name="window ragged prompts", seqs=16, rows=4096, ragged=True, min_len=4097, max_len=9001,
             heads=32, kv_heads=8, dim=128, page=128, fmt="e4m3", dtype="bf16", window=2048, first=128, lse=True),
        # Eight readings of one page (6,544 positions), some tokens in: two query heads to a key head.
        dict(prefix, name="prefix eight readings", seqs=8, prefix_min=6544, prefix_max=6544, own_max=200, heads=16,
             kv_heads=8, dim=64, page=64, fmt="i8", dtype="bf16"),
        # 64 continuations of one long document, up to 1,024 tokens in.
        dict(prefix, name="prefix 64 continuations", seqs=64, prefix_min=16384, prefix_max=16384, own_max=1024,
             heads=16, kv_heads=8, dim=64, page=64, fmt="e4m3", dtype="bf16"),
        # Four documents of different lengths, twelve questions of up to 96 tokens to each, wide heads.
        dict(prefix, name="prefix questions", seqs=48, groups=4, rows=96, ragged=True, prefix_min=3001,
             prefix_max=9001, own_max=300, heads=32, kv_heads=8, dim=128, page=128, fmt="e4m3", dtype="bf16",
             lse=True),
        # Speculative verify of 32 continuations of one page, five FP32 rows each.
        dict(prefix, name="prefix verify", seqs=32, rows=5, prefix_min=12000, prefix_max=12000, own_max=400, heads=16,
             kv_heads=8, dim=64, page=32, fmt="i8", dtype="f32"),
        # A whole serving step of 16 readings of two pages: turn and append the new rows, then attend with them.
        dict(prefix, op="step", name="prefix serving step", seqs=16, groups=2, prefix_min=6000, prefix_max=9000,
             own_max=700, heads=16, kv_heads=8, dim=64, page=64, fmt="e4m3", dtype="bf16", rot=64, layout="half",
             axes="sections", image=0, table_positions=16384),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "append", "window", "window", "window", "prefix", "prefix", "step"])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    turn = dict(layout=rng.choice(["interleaved", "half"]), rot=rng.choice([dim, dim, dim // 2, 32, 24]),
                axes=rng.choice(["sections", "turns", "grid"]))
    if op == "rope":
        rows = _log(rng, 1, 30000)
        return dict(turn, op=op, rows=rows, heads=rng.choice([1, 3, 8, 24, 40]), dim=dim,
                    image=rng.choice([0, rows // 2, rows]), inverse=rng.random() < 0.4, dtype=dtype,
                    fused_row=rng.random() < 0.5, table_positions=rng.choice([16384, 65536]))
    kv_heads = rng.choice([1, 2, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    page, fmt = rng.choice([16, 32, 64, 128]), rng.choice(["i8", "e4m3"])
    base = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=page, fmt=fmt, dtype=dtype, groups=0)
    if op == "append":
        rows = _log(rng, 1, 6000)
        seqs = max(1, min(_log(rng, 1, 128), 40000 // rows))
        return dict(base, **turn, seqs=seqs, rows=rows, ragged=rng.random() < 0.5 and rows > 1, min_len=rows,
                    max_len=rows + _log(rng, 1, 8000), image=rng.choice([0, rows // 2]), table_positions=16384)
    attend = dict(base, sinks=rng.random() < 0.5, lse=rng.random() < 0.3)
    if op == "window":
        rows = rng.choice([1, 1, 2, 5, _log(rng, 1, 4000), _log(rng, 1, 4000)])
        window, first = rng.choice([1, 100, 1024, 2048, 4096, 0]), rng.choice([0, 1, 4, 16, 100, 300])
        max_len = _log(rng, rows, max(20000, rows)) if rows > 1 else _log(rng, 8, 32768)
        if not window:
            max_len = max(rows, min(max_len, int(2.5e11 / (rows * heads * dim))))
        seqs = max(1, min(_log(rng, 1, 128), int(400e6 / (max_len * kv_heads * dim * 2)),
                          int(2.5e11 / (rows * heads * min(max_len, window or max_len) * dim))))
        return dict(attend, seqs=seqs, rows=rows, ragged=rng.random() < 0.4 and rows > 1, window=window, first=first,
                    min_len=min(_log(rng, 1, max_len), max_len), max_len=max_len)
    rows = rng.choice([1, 1, 2, 5, 8, _log(rng, 9, 100)]) if op == "prefix" else rng.choice([1, 1, 2, 5])
    groups = rng.choice([1, 1, 2, 5])
    longest = _log(rng, 16, 16384 if op == "prefix" else 12000)
    seqs = max(groups, min(_log(rng, 1, 96), int(2.5e11 / (rows * heads * longest * dim))))
    case = dict(attend, seqs=seqs, rows=rows, ragged=rng.random() < 0.4 and rows > 1,
                groups=groups, prefix_min=_log(rng, 8, longest), prefix_max=longest, own_max=rows + _log(rng, 1, 1500),
                window=0, first=0)
    if op == "step":
        case.update(turn, image=0, table_positions=16384)
    return case


def _rows_of(case):
    """Rows of each sequence: the same for all, or anything from one to that many."""
    if not case["ragged"]:
        return [case["rows"]] * case["seqs"]
    r = random.Random("rows %d %d" % (case["seqs"], case["rows"]))
    return [case["rows"] if b == 0 else r.randint(1, case["rows"]) for b in range(case["seqs"])]


def _groups_of(case):
    """The first sequence of each group and the end of the last, and the length of each one's beginning."""
    n, seqs = case["groups"], case["seqs"]
    r = random.Random("groups %d %d %d" % (n, case["prefix_min"], case["prefix_max"]))
    starts = [g * seqs // n for g in range(n + 1)]
    lens = [case["prefix_max"] if g == 0 else r.randint(case["prefix_min"], case["prefix_max"]) for g in range(n)]
    return starts, lens


def _prefix_of(case):
    """The length of each sequence's shared beginning."""
    if not case["groups"]:
        return [0] * case["seqs"]
    starts, lens = _groups_of(case)
    return [n for g, n in enumerate(lens) for _ in range(starts[g + 1] - starts[g])]


def _lens_of(case):
    """Positions of each sequence, the rows of the call included."""
    rows = _rows_of(case)
    if case["groups"]:
        r = random.Random("own %d %d" % (case["seqs"], case["own_max"]))
        return [p + (case["own_max"] if b == 0 else r.randint(m, max(m, case["own_max"])))
                for b, (p, m) in enumerate(zip(_prefix_of(case), rows))]
    r = random.Random("lens %d %d %d" % (case["seqs"], case["min_len"], case["max_len"]))
    lens = [case["max_len"] if b == 0 else r.randint(case["min_len"], case["max_len"]) for b in range(case["seqs"])]
    return [max(n, m) for n, m in zip(lens, rows)]


# ------------------------------------------------------------- inputs and state
def _pair_axes(kind, pairs):
    """The axis of each rotated pair: time, height and width in sections of a quarter and the rest, or in turns; or
    height and width alone, half of the pairs each."""
    if kind == "turns":
        return [i % 3 for i in range(pairs)]
    if kind == "grid":
        return [0 if i < pairs // 2 else 1 for i in range(pairs)]
    t = max(1, pairs // 4)
    h = (pairs - t + 1) // 2
    return [0] * t + [1] * h + [2] * (pairs - t - h)


def _table(case, device):
    """{cos, sin} of each position and rotated pair, [positions][rot / 2][2], the table that a program keeps."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=device)
    freq = THETA ** (-2.0 * i / case["rot"])
    angle = torch.arange(case["table_positions"], dtype=torch.float64, device=device)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), dim=-1).float().contiguous()


def _axis_positions(case, rows, g, device):
    """Where each row stands on each axis, [axes][rows]: the first `image` rows are patches of 64 x 64 frames, the
    others text, which stands at one place on all axes."""
    axes = 2 if case["axes"] == "grid" else 3
    n = case["table_positions"]
    at = torch.arange(rows, device=device)
    base = int(torch.randint(0, n // 4, (1,), device=device, generator=g).item())
    frame = torch.stack((base + at // 4096, base + at % 4096 // 64, base + at % 64))[3 - axes:]
    if case["image"] == 0 and rows <= 4096:  # rows of different sequences
        text = torch.randint(0, n, (rows,), device=device, generator=g)
    else:
        text = (base + 64 + at - case["image"]).clamp(0, n - 1)
    return torch.where(at < case["image"], frame, text.expand(axes, rows)).to(torch.int32).contiguous()


def _rows(g, rows, heads, dim, dtype, fused, device):
    """Rows [rows][heads][dim]; with `fused` the leading heads of wider rows, as a projection writes them."""
    wide = heads + (8 if fused else 0)
    x = torch.randn(rows, wide, dim, device=device, generator=g, dtype=torch.float32).to(dtype)
    return x[:, :heads]


def _codes(g, pages, case, device):
    """Codes of normal values against a scale that their page's largest one set."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    if case["fmt"] == "i8":
        out = torch.empty(shape, dtype=torch.int8, device=device)
    else:
        out = torch.empty(shape, dtype=torch.float8_e4m3fn, device=device)
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for p in range(0, pages, step):
        x = torch.randn((min(step, pages - p),) + shape[1:], device=device, generator=g)
        if case["fmt"] == "i8":
            out[p:p + step] = (x * (127.0 / 4.0)).round().clamp(-127.0, 127.0).to(torch.int8)
        else:
            out[p:p + step] = (x * (448.0 / 4.0)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return out


def _scales(g, pages, case, device):
    spread = torch.rand(pages, case["kv_heads"], device=device, generator=g) * 0.6 + 0.7
    return spread * (4.0 / QMAX[case["fmt"]])


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    s = {"case": case}
    dtype = DTYPES[case["dtype"]]
    if case["op"] in ("rope", "append", "step"):
        s["table"] = _table(case, device)
        s["pair_axes"] = _pair_axes(case["axes"], case["rot"] // 2)
        if own:
            s["rope"] = _fo().RopeAxes(s["table"], s["pair_axes"], layout=case["layout"])
    if case["op"] == "rope":
        s["x"] = _rows(g, case["rows"], case["heads"], case["dim"], dtype, case["fused_row"], device)
        s["positions"] = _axis_positions(case, case["rows"], g, device)
        s["out"] = torch.empty(case["rows"], case["heads"], case["dim"], dtype=dtype, device=device)
        return s

    rows, lens, page, seqs = _rows_of(case), _lens_of(case), case["page"], case["seqs"]
    total, shared = sum(rows), _prefix_of(case)
    per_seq = -(-max(lens) // page)
    # Pages are handed out in any order.  An append touches a sequence's last pages alone, so only those are its own
    # there; an attention reads them all, and the pages that a group's beginning fills are the same for its
    # sequences, each of which has a page of its own from where the beginning ends.
    if case["op"] == "append":
        first = [(n - m) // page for n, m in zip(lens, rows)]
    else:
        first = [p // page for p in shared]
    starts = _groups_of(case)[0] if case["groups"] else []
    common = [shared[b] // page for b in starts[:-1]] if starts else []
    used = sum(-(-n // page) - f for n, f in zip(lens, first)) + sum(common)
    pages = used + 3
    order = torch.randperm(pages, device=device, generator=g).to(torch.int32).cpu().tolist()
    table, at = [[0] * per_seq for _ in range(seqs)], 0
    for i, n in enumerate(common):
        for b in range(starts[i], starts[i + 1]):
            table[b][:n] = order[at:at + n]
        at += n
    for b in range(seqs):
        n = -(-lens[b] // page) - first[b]
        table[b][first[b]:first[b] + n] = order[at:at + n]
        at += n
    s["page_table"] = torch.tensor(table, dtype=torch.int32, device=device)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=device)
    s["row_start"] = None
    if case["ragged"]:
        begin = [0]
        for n in rows:
            begin.append(begin[-1] + n)
        s["row_start"] = torch.tensor(begin, dtype=torch.int32, device=device)
    s["k_codes"], s["v_codes"] = _codes(g, pages, case, device), _codes(g, pages, case, device)
    s["k_scales"], s["v_scales"] = _scales(g, pages, case, device), _scales(g, pages, case, device)
    s["q"] = _rows(g, total, case["heads"], case["dim"], dtype, True, device)
    if case["op"] in ("append", "step"):
        s["positions"] = _axis_positions(case, total, g, device)
        s["k"] = _rows(g, total, case["kv_heads"], case["dim"], dtype, True, device)
        s["v"] = _rows(g, total, case["kv_heads"], case["dim"], dtype, True, device)
        s["q_out"] = torch.empty(total, case["heads"], case["dim"], dtype=dtype, device=device)
    if case["op"] != "append":
        s["sinks"] = torch.randn(case["heads"], device=device, generator=g) if case["sinks"] else None
        s["out"] = torch.empty(total, case["heads"], case["dim"], dtype=dtype, device=device)
        s["lse"] = torch.empty(total, case["heads"], device=device) if case["lse"] else None
    if case["groups"]:
        s["group_start"] = torch.tensor(starts, dtype=torch.int32, device=device)
        s["group_lens"] = torch.tensor(_groups_of(case)[1], dtype=torch.int32, device=device)
    if own:
        F = _fo()
        s["kv"] = F.PagedKv(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
        s["batch"] = F.PagedBatch(s["page_table"], s["lens"], rows=case["rows"], row_start=s["row_start"])
        if case["groups"]:
            s["groups"] = F.PagedGroups(s["group_start"], s["group_lens"])
    return s


# ------------------------------------------------------------- the plain form
def _rotate(x, cos_sin, layout, inverse=False):
    """FP32 rows [rows][heads][dim] rotated by [rows][pairs][2]."""
    pairs = cos_sin.shape[1]
    c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    s = -s if inverse else s
    y = x.clone()
    if layout == "interleaved":
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        y[..., 0:2 * pairs:2] = a * c - b * s
        y[..., 1:2 * pairs:2] = b * c + a * s
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        y[..., :pairs] = a * c - b * s
        y[..., pairs:2 * pairs] = b * c + a * s
    return y


def _entries(s):
    """{cos, sin} of each row and pair, [rows][pairs][2]."""
    axis = torch.tensor(s["pair_axes"], device="cuda")
    pair = torch.arange(axis.numel(), device="cuda")
    return s["table"][s["positions"].long()[axis].t(), pair]


def _row_places(s):
    """Sequence, number within it, and place in the cache of every row."""
    case, lens = s["case"], s["lens"].long()
    seqs = case["seqs"]
    if s["row_start"] is None:
        count = torch.full((seqs,), case["rows"], device=lens.device)
        total = seqs * case["rows"]
        begin = torch.arange(seqs, device=lens.device) * case["rows"]
    else:
        count, begin = (s["row_start"][1:] - s["row_start"][:-1]).long(), s["row_start"][:-1].long()
        total = s["q"].shape[0]
    at = torch.arange(total, device=lens.device)
    b = torch.repeat_interleave(torch.arange(seqs, device=lens.device), count, output_size=total)
    r = at - begin[b]
    return b, r, lens[b] - count[b] + r


def _round(y, fmt):
    y = y.round() if fmt == "i8" else y
    y = y.clamp(-QMAX[fmt], QMAX[fmt])
    return y.to(torch.int8) if fmt == "i8" else y.to(torch.float8_e4m3fn).view(torch.int8)


def _encode(x, scale, fmt):
    """x / scale as codes; a scale of zero has only zeros."""
    y = torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x))
    return _round(y, fmt)


def _store(codes, scales, x, page_id, offset, fmt):
    """Rows x [rows][kv heads][dim] into their pages, whose scales grow where they have to."""
    pages, _, page, _ = codes.shape
    heads = x.shape[1]
    raw = codes.view(torch.int8)
    top = torch.zeros(pages, heads, device=x.device)
    top.scatter_reduce_(0, page_id[:, None].expand(-1, heads), x.abs().amax(dim=-1), "amax")
    begin = torch.full((pages,), page, device=x.device)
    begin.scatter_reduce_(0, page_id, offset, "amin")
    needed = top / torch.full_like(top, QMAX[fmt])
    old = torch.where((begin > 0)[:, None], scales, torch.zeros_like(scales))
    new = torch.where((begin < page)[:, None], torch.maximum(old, needed), scales)
    # The tokens that a page already held, against its new scale.
    grown = (begin < page)[:, None] & (new > old)
    ratio = old / torch.where(new > 0, new, torch.ones_like(new))
    held = torch.arange(page, device=x.device)[None, :] < begin[:, None]
    again = _round(codes.float() * ratio[:, :, None, None], fmt)
    change = grown[:, :, None, None] & held[:, None, :, None]
    raw.copy_(torch.where(change, again, raw))
    scales.copy_(new)
    raw[page_id, :, offset] = _encode(x, new[page_id][:, :, None].expand_as(x), fmt)


def _append(s):
    case = s["case"]
    b, _, place = _row_places(s)
    cos_sin = _entries(s)
    page_id = s["page_table"][b, place // case["page"]].long()
    offset = place % case["page"]
    q = _rotate(s["q"].float(), cos_sin, case["layout"])
    k = _rotate(s["k"].float(), cos_sin, case["layout"])
    _store(s["k_codes"], s["k_scales"], k, page_id, offset, case["fmt"])
    _store(s["v_codes"], s["v_scales"], s["v"].float(), page_id, offset, case["fmt"])
    s["q_out"].copy_(q)


def _at(codes, scales, table, b, places):
    """FP32 [n][kv heads][places][dim] of the places [n][places] of sequences b [n]."""
    page = codes.shape[2]
    ids = table[b[:, None], places // page]
    x = codes.view(torch.int8)[ids, :, places % page].view(codes.dtype).float() * scales[ids][..., None]
    return x.transpose(1, 2)


def _softmax_parts(parts, sinks):
    """Joins parts (scores [.., n], values [.., n, dim], -infinity what is not seen): out and the log of the sum.
    `sinks` has the scores' shape without the last dimension."""
    top = parts[0][0].amax(dim=-1)
    for score, _ in parts[1:]:
        top = torch.maximum(top, score.amax(dim=-1))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    below, o = 0, 0
    for score, v in parts:
        p = torch.exp(score - top[..., None])
        below = below + p.sum(dim=-1)
        o = o + torch.matmul(p, v)
    total = below if sinks is None else below + torch.exp(sinks - top)
    o = torch.where(below[..., None] > 0, o / torch.where(below > 0, total, torch.ones_like(total))[..., None],
                    torch.zeros_like(o))
    return o, top + torch.log(below)


def _window(s):
    """Pieces of at most 256 rows of a sequence, as many at a time as there is room for their scores."""
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, rows, device = heads // kv_heads, min(case["rows"], 256), s["q"].device
    b, r, place = _row_places(s)
    piece_of = torch.nn.functional.pad(((r[1:] % 256 == 0) | (b[1:] != b[:-1])).long().cumsum(0), (1, 0))
    begins = torch.nonzero(r % 256 == 0)[:, 0]
    window = case["window"] or case["max_len"]
    first = min(case["first"], case["max_len"])
    near = min(window + rows - 1, max(case["max_len"], case["rows"]))
    step = max(1, (1 << 28) // (heads * rows * (first + near)))
    n = sum(-(-m // 256) for m in _rows_of(case))
    sinks = s["sinks"]
    if sinks is not None:
        sinks = sinks.view(1, kv_heads, 1, group).expand(1, kv_heads, rows, group).reshape(1, kv_heads, -1)
    for i in range(0, n, step):
        m = min(step, n - i)
        mine = (piece_of >= i) & (piece_of < i + m)
        where = torch.nonzero(mine)[:, 0]
        at = (piece_of[where] - i, r[where] % 256)
        q = torch.zeros(m, rows, heads, dim, device=device)
        q[at] = s["q"][where].float()
        seen = torch.full((m, rows), -1, dtype=torch.long, device=device)
        seen[at] = place[where]
        seqs = b[begins[i:i + m]]
        low = (place[begins[i:i + m]] - window + 1).clamp(min=0)
        places = low[:, None] + torch.arange(near, device=device)
        places = torch.cat((torch.arange(first, device=device).expand(m, first), places), dim=1)
        inside = places < s["lens"][seqs].long()[:, None]
        kept = torch.where(inside, places, torch.zeros_like(places))
        k = _at(s["k_codes"], s["k_scales"], s["page_table"].long(), seqs, kept)
        v = _at(s["v_codes"], s["v_scales"], s["page_table"].long(), seqs, kept)
        # A place is counted once: among the first ones, or in the window behind them.
        early = torch.arange(first + near, device=device) < first
        visible = inside[:, None] & (places[:, None] <= seen[:, :, None]) & (
            early | ((places >= first)[:, None] & (places[:, None] > seen[:, :, None] - window)))
        qg = q.view(m, rows, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(m, kv_heads, rows * group, dim)
        score = torch.matmul(qg, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
        visible = visible[:, None, :, None].expand(m, kv_heads, rows, group, first + near).reshape(score.shape)
        o, lse = _softmax_parts([(score.masked_fill(~visible, -math.inf), v)], sinks)
        o = o.view(m, kv_heads, rows, group, dim).permute(0, 2, 1, 3, 4).reshape(m, rows, heads, dim)
        s["out"][where] = o[at].to(s["out"].dtype)
        if s["lse"] is not None:
            s["lse"][where] = lse.view(m, kv_heads, rows, group).permute(0, 2, 1, 3).reshape(m, rows, heads)[at]


def _prefix(s, q):
    """A group's beginning against all rows of the group, and each sequence's own positions against its rows."""
    case = s["case"]
    heads, kv_heads, dim, rows = case["heads"], case["kv_heads"], case["dim"], case["rows"]
    group, device = heads // kv_heads, q.device
    b, r, place = _row_places(s)
    table = s["page_table"].long()
    starts, shared = _groups_of(case)
    counts, lens = _rows_of(case), _lens_of(case)
    for g, n in enumerate(shared):
        b0, b1 = starts[g], starts[g + 1]
        r0 = sum(counts[:b0])
        where = torch.arange(r0, r0 + sum(counts[b0:b1]), device=device)
        m, at = b1 - b0, (b[where] - b0, r[where])
        padded = torch.zeros(m, rows, heads, dim, device=device)
        padded[at] = q[where].float()
        seen = torch.full((m, rows), -1, dtype=torch.long, device=device)
        seen[at] = place[where]
        qg = padded.view(m, rows, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(m, kv_heads, rows * group, dim)
        every = torch.arange(n, device=device)[None]
        k0 = _at(s["k_codes"], s["k_scales"], table, torch.full((1,), b0, device=device), every)
        v0 = _at(s["v_codes"], s["v_scales"], table, torch.full((1,), b0, device=device), every)
        sinks = s["sinks"]
        if sinks is not None:
            sinks = sinks.view(1, kv_heads, 1, group).expand(1, kv_heads, rows, group).reshape(1, kv_heads, -1)
        step = max(1, (1 << 28) // (heads * rows * n))
        own_n = max(lens[b0:b1]) - n
        for i in range(0, m, step):
            seqs = torch.arange(b0 + i, min(b0 + i + step, b1), device=device)
            places = (n + torch.arange(own_n, device=device)).expand(seqs.numel(), own_n)
            kept = torch.minimum(places, s["lens"][seqs].long()[:, None] - 1)
            k1 = _at(s["k_codes"], s["k_scales"], table, seqs, kept)
            v1 = _at(s["v_codes"], s["v_scales"], table, seqs, kept)
            x = qg[i:i + step] * (1.0 / math.sqrt(dim))
            visible = (places[:, None] <= seen[i:i + step, :, None])[:, None, :, None]
            visible = visible.expand(-1, kv_heads, rows, group, own_n).reshape(-1, kv_heads, rows * group, own_n)
            near = torch.matmul(x, k1.transpose(2, 3)).masked_fill(~visible, -math.inf)
            # All rows of the group in one product with the beginning.
            flat = x.transpose(0, 1).reshape(1, kv_heads, -1, dim)
            far = torch.matmul(flat, k0.transpose(2, 3)).view(kv_heads, -1, rows * group, n).transpose(0, 1)
            o, lse = _softmax_parts([(far, v0), (near, v1)], sinks)
            o = o.view(-1, kv_heads, rows, group, dim).permute(0, 2, 1, 3, 4).reshape(-1, rows, heads, dim)
            mine = (at[0] >= i) & (at[0] < i + step)
            to = where[mine]
            s["out"][to] = o[at[0][mine] - i, at[1][mine]].to(s["out"].dtype)
            if s["lse"] is not None:
                lse = lse.view(-1, kv_heads, rows, group).permute(0, 2, 1, 3).reshape(-1, rows, heads)
                s["lse"][to] = lse[at[0][mine] - i, at[1][mine]]


# ------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        F = _fo()
        if op == "rope":
            F.rope(s["x"], s["out"], s["rope"], positions=s["positions"], inverse=case["inverse"])
        if op in ("append", "step"):
            F.paged_append(s["kv"], s["batch"], s["k"], s["v"], rope=s["rope"], positions=s["positions"], q=s["q"],
                           q_out=s["q_out"])
        if op == "window":
            F.paged_window_attention(s["kv"], s["batch"], s["q"], s["out"], window=case["window"], first=case["first"],
                                     sinks=s["sinks"], lse=s["lse"])
        if op in ("prefix", "step"):
            F.paged_prefix_attention(s["kv"], s["batch"], s["groups"], s["q_out"] if op == "step" else s["q"],
                                     s["out"], sinks=s["sinks"], lse=s["lse"])
    else:
        if op == "rope":
            s["out"].copy_(_rotate(s["x"].float(), _entries(s), case["layout"], case["inverse"]))
        if op in ("append", "step"):
            _append(s)
        if op == "window":
            _window(s)
        if op in ("prefix", "step"):
            _prefix(s, s["q_out"] if op == "step" else s["q"])
    return _outputs(s)


def _outputs(s):
    """Whole outputs.  An append's are the rotated queries and the cache: FP8 codes as the numbers that they are,
    int8 codes as whole numbers (held to equality, which is stricter than any bound on code times scale), and the
    scales beside them."""
    op = s["case"]["op"]
    got = {}
    if op != "append":
        got["out"] = s["out"]
    if op in ("append", "step"):
        got.update(q=s["q_out"], k_codes=s["k_codes"], v_codes=s["v_codes"], k_scales=s["k_scales"],
                   v_scales=s["v_scales"])
    if s.get("lse") is not None:
        got["lse"] = s["lse"]
    return got


def work(case):
    """Every input read once, every output written once: of a cache, what a row of the call sees, a shared beginning
    once for its group."""
    wide = 4 if case["dtype"] == "f32" else 2
    dim = case["dim"]
    axes = 2 if case.get("axes") == "grid" else 3
    if case["op"] == "rope":
        moved = case["rows"] * case["heads"] * dim * wide * 2
        return {"bytes": moved + case["rows"] * (4 * axes + case["rot"] * 4),
                "flops": case["rows"] * case["heads"] * case["rot"] * 3}
    rows, lens, shared = _rows_of(case), _lens_of(case), _prefix_of(case)
    total, kv_heads, heads = sum(rows), case["kv_heads"], case["heads"]
    b, f = 0, 0
    if case["op"] in ("append", "step"):
        b += total * (2 * kv_heads * dim * (wide + 1) + 2 * heads * dim * wide + case["rot"] * 4 + 4 * axes)
        f += total * (heads + kv_heads) * case["rot"] * 3 + total * 2 * kv_heads * dim * 3
    if case["op"] != "append":
        places = sum(_groups_of(case)[1]) if case["groups"] else 0
        pairs = 0
        for n, m, p in zip(lens, rows, shared):
            if case["op"] == "window":
                window, first = case["window"] or n, case["first"]
                low = max(0, n - m + 1 - window)
                places += n - low + min(first, low)
                for seen in range(n - m + 1, n + 1):
                    pairs += min(seen, window) + min(first, max(0, seen - window))
            else:
                places += n - p
                pairs += m * n - m * (m - 1) // 2
        b += places * kv_heads * dim * 2 + places // case["page"] * kv_heads * 8
        b += total * heads * dim * wide * 2 + (total * heads * 4 if case["lse"] else 0)
        f += pairs * heads * dim * 4
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------- the same in 64 bits
def _exact_rope(x, s, inverse):
    """Complex multiplication of each pair by the {cos, sin} of its axis's position."""
    case, pos = s["case"], s["positions"].long()
    t = torch.stack([s["table"][pos[a], i] for i, a in enumerate(s["pair_axes"])], dim=1).double()
    turn = torch.complex(t[..., 0], -t[..., 1] if inverse else t[..., 1])[:, None, :]
    pairs = turn.shape[-1]
    y = x.double().clone()
    head = y[..., :2 * pairs]
    if case["layout"] == "interleaved":
        z = torch.complex(head[..., 0::2].contiguous(), head[..., 1::2].contiguous()) * turn
        y[..., :2 * pairs] = torch.stack((z.real, z.imag), dim=-1).flatten(-2)
    else:
        z = torch.complex(head[..., :pairs].contiguous(), head[..., pairs:].contiguous()) * turn
        y[..., :2 * pairs] = torch.cat((z.real, z.imag), dim=-1)
    return y


def _exact_e4m3(x):
    """Nearest e4m3 number, ties to the even one: steps of 2^(exponent - 3), exponents from -6 up."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -30))
    step = torch.exp2((e.double() - 1.0).clamp(min=-6.0) - 3.0)
    return ((x / step).round() * step).clamp(-448.0, 448.0)


def _exact_store(codes, scales, x, rows, lens, table, case):
    """One sequence's page after another; codes as FP64 numbers."""
    top, page, at = QMAX[case["fmt"]], case["page"], 0

    def nearest(y):
        return y.round().clamp(-127.0, 127.0) if case["fmt"] == "i8" else _exact_e4m3(y)

    for n, m, pages in zip(lens, rows, table):
        position = n - m
        while position < n:
            begin = position % page
            stop = min(n, position - begin + page)
            part = x[at:at + stop - position].transpose(0, 1)  # [kv heads][rows][dim]
            p = pages[position // page]
            old = scales[p] if begin else torch.zeros_like(scales[p])
            new = torch.maximum(old, part.abs().amax(dim=(1, 2)) / top)
            held = codes[p, :, :begin]
            grown = (new > old)[:, None, None]
            safe = torch.where(new > 0, new, torch.ones_like(new))[:, None, None]
            codes[p, :, :begin] = torch.where(grown, nearest(held * (old[:, None, None] / safe)), held)
            codes[p, :, begin:begin + stop - position] = nearest(part / safe)
            scales[p] = new
            at += stop - position
            position = stop


def _exact_attend(s, q, k_codes, v_codes, k_scales, v_scales):
    """Sequence by sequence, 128 rows at a time, over the range that these see and the first positions before it."""
    case = s["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group, device = heads // kv_heads, q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=device)
    table, at = s["page_table"].long(), 0
    leader = list(range(case["seqs"]))
    if case["groups"]:
        starts = _groups_of(case)[0]
        leader = [b0 for b0, b1 in zip(starts, starts[1:]) for _ in range(b0, b1)]

    def values(codes, scales, b, j, shared):
        ids = torch.where(j < shared, table[leader[b], j // page], table[b, j // page])
        raw = codes.view(torch.int8)[ids, :, j % page].view(codes.dtype) if codes.element_size() == 1 else \
            codes[ids, :, j % page]
        return (raw.double() * scales[ids].double()[..., None]).transpose(0, 1)

    for b, (n, m, shared) in enumerate(zip(_lens_of(case), _rows_of(case), _prefix_of(case))):
        step = 128 if m * n < 1 << 26 else 64
        for r0 in range(0, m, step):
            p = n - m + torch.arange(r0, min(r0 + step, m), device=device)
            high = int(n - m + min(r0 + step, m))
            low = max(0, n - m + r0 + 1 - case["window"]) if case["window"] else 0
            j = torch.cat((torch.arange(min(case["first"], low), device=device), torch.arange(low, high, device=device)))
            seen = j[None] <= p[:, None]
            if case["window"]:
                seen &= (j[None] > p[:, None] - case["window"]) | (j[None] < case["first"])
            k, v = values(k_codes, k_scales, b, j, shared), values(v_codes, v_scales, b, j, shared)
            rows = slice(at + r0, at + r0 + p.numel())
            x = q[rows].double().view(-1, kv_heads, group, dim)
            score = torch.einsum("rhgd,hnd->hgrn", x, k) / math.sqrt(dim)
            score = torch.where(seen, score, torch.full_like(score, -math.inf))
            z = torch.logsumexp(score, dim=-1)
            o = torch.einsum("hgrn,hnd->hgrd", torch.exp(score - z[..., None]), v)
            if s["sinks"] is not None:
                o = o * torch.sigmoid(z - s["sinks"].double().view(kv_heads, group)[..., None])[..., None]
            out[rows] = o.permute(2, 0, 1, 3).reshape(-1, heads, dim)
            lse[rows] = z.permute(2, 0, 1).reshape(-1, heads)
        at += m
    return out, lse


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "rope":
        return {"out": _exact_rope(s["x"], s, case["inverse"])}
    rows, lens = _rows_of(case), _lens_of(case)
    got, q = {}, s["q"]
    caches = [s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"]]
    if case["op"] in ("append", "step"):
        table = s["page_table"].cpu().tolist()
        q, k = _exact_rope(s["q"], s, False), _exact_rope(s["k"], s, False)
        caches = [c.double() for c in caches]
        _exact_store(caches[0], caches[2], k, rows, lens, table, case)
        _exact_store(caches[1], caches[3], s["v"].double(), rows, lens, table, case)
        whole = case["fmt"] == "i8"
        got.update(q=q, k_codes=None if whole else caches[0], v_codes=None if whole else caches[1],
                   k_scales=caches[2], v_scales=caches[3])
    if case["op"] != "append":
        out, lse = _exact_attend(s, q, *caches)
        got["out"] = out
        if case["lse"]:
            got["lse"] = lse
    return got
