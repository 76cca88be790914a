"""Measured cases of the paged 8-bit KV cache operators: rotary positions,
appending rotated keys and values to the paged cache, and the attention that
reads it.

Every case runs in two forms on the same prepared tensors: the plain one
(elementary torch operations in FP32) and, with ``own`` set, the calls of
``fo_cuda`` that a serving program makes.  ``exact`` states the same results in
64 bits, written apart from the plain form.

The cache: codes [pages][kv heads][page size][head dim] of int8 or FP8 (e4m3)
for keys and for values, one FP32 scale per (page, kv head) of each; a
sequence's pages are listed in a page table, and ``lens`` counts a sequence's
positions with the rows of the call included.  A row's position is
``len - rows + r``.
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
    rope = dict(op="rope", rot=64, layout="interleaved", scaling="none", factor=1.0, inverse=False, fused_row=False)
    append = dict(op="append", rot=64, layout="interleaved", ragged=False, table_positions=16384)
    attn = dict(op="attend", rows=1, ragged=False, window=0, sinks=True, lse=False)
    return [
        # The 16 query and 8 key heads of eight sequences' newest tokens, the temporal half of each head rotated,
        # in place of a decode step's rows: the smallest call, where only latency counts.
        dict(rope, name="rope step", rows=8, heads=24, dim=64, rot=32, dtype="bf16", table_positions=16384,
             fused_row=True),
        # One full page of 6,544 tokens (4,096 of its image, 2,448 of text), FP32 as the fused rows hold it.
        dict(rope, name="rope page", rows=6544, heads=24, dim=64, dtype="f32", table_positions=8192),
        # Gradient of the rotation over a long document's rows: wide heads, half layout, positions stretched
        # eightfold by parts, an odd number of rows.
        dict(rope, name="rope long gradient", rows=32771, heads=40, dim=128, rot=128, dtype="bf16", layout="half",
             scaling="yarn", factor=8.0, inverse=True, table_positions=131072),
        # A decode step of 64 pages being read at once: one new row each, with its queries rotated.
        dict(append, name="append step", seqs=64, rows=1, min_len=6545, max_len=8592, heads=16, kv_heads=8, dim=64,
             page=64, fmt="i8", dtype="bf16"),
        # A page's whole prompt after its prefill, FP32 rows as the prefill takes them, into 64-token pages.
        dict(append, name="append page", seqs=1, rows=6544, min_len=6544, max_len=6544, heads=16, kv_heads=8, dim=64,
             page=64, fmt="i8", dtype="f32"),
        # Prompts of very different lengths, some of them continuing a cached beginning, with wide heads and FP8 codes.
        dict(append, name="append ragged prompts", seqs=24, rows=4096, ragged=True, min_len=4097, max_len=9001,
             heads=32, kv_heads=8, dim=128, rot=128, layout="half", page=128, fmt="e4m3", dtype="bf16"),
        # One short sequence, one row, small pages: the latency of a call.
        dict(attn, name="attend one short", seqs=1, min_len=777, max_len=777, heads=16, kv_heads=8, dim=64, page=16,
             fmt="i8", dtype="bf16"),
        # Speculative verify of one long page: five FP32 rows against 16,384 positions.
        dict(attn, name="attend verify", seqs=1, rows=5, min_len=16384, max_len=16384, heads=16, kv_heads=8, dim=64,
             page=64, fmt="i8", dtype="f32"),
        # 64 pages being decoded at once, between 6,545 and 8,592 positions each.
        dict(attn, name="attend 64 pages", seqs=64, min_len=6545, max_len=8592, heads=16, kv_heads=8, dim=64, page=64,
             fmt="i8", dtype="bf16"),
        # Long documents with wide heads and FP8 codes, uneven lengths.
        dict(attn, name="attend long", seqs=16, min_len=1000, max_len=32768, heads=32, kv_heads=8, dim=128, page=128,
             fmt="e4m3", dtype="bf16", sinks=False),
        # Verify rows of different numbers over a sliding window of 4,096, eight query heads to a key head.
        dict(attn, name="attend window", seqs=48, rows=5, ragged=True, min_len=1, max_len=20001, heads=64, kv_heads=8,
             dim=128, page=32, fmt="i8", dtype="bf16", window=4096, lse=True),
        # A whole serving step of eight pages: rotate and append the new rows, then attend with them.
        dict(append, op="step", name="serving step", seqs=8, rows=1, min_len=9000, max_len=12000, heads=16, kv_heads=8,
             dim=64, page=64, fmt="e4m3", dtype="bf16", window=0, sinks=True, lse=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend", "step"])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    layout = rng.choice(["interleaved", "half"])
    rot = rng.choice([dim, dim, dim // 2, 32, 24])
    if op == "rope":
        rows, heads = _log(rng, 1, 30000), rng.choice([1, 3, 8, 24, 40])
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return dict(op=op, rows=rows, heads=heads, dim=dim, rot=rot, layout=layout, scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 5.5, 8.0]), inverse=rng.random() < 0.4,
                    dtype=dtype, fused_row=rng.random() < 0.5, table_positions=rng.choice([16384, 65536, 131072]))
    kv_heads = rng.choice([1, 2, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    page, fmt = rng.choice([16, 32, 64, 128]), rng.choice(["i8", "e4m3"])
    base = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=page, fmt=fmt, dtype=dtype)
    if op == "append":
        rows = _log(rng, 1, 6000)
        seqs = max(1, min(_log(rng, 1, 128), 40000 // rows))
        start = _log(rng, 1, 8000)
        return dict(base, seqs=seqs, rows=rows, ragged=rng.random() < 0.5 and rows > 1, min_len=rows,
                    max_len=rows + start, rot=rot, layout=layout, table_positions=16384)
    rows = rng.choice([1, 1, 1, 2, 4, 5, 8])
    max_len = _log(rng, 8, 32768)
    row_bytes = kv_heads * dim * 2
    seqs = max(1, min(_log(rng, 1, 128), int(400e6 / (max_len * row_bytes))))
    min_len = max(rows, _log(rng, 8, max_len)) if op == "step" else _log(rng, 1, max_len)
    attend = dict(base, seqs=seqs, rows=rows, ragged=rng.random() < 0.3 and rows > 1, min_len=min(min_len, max_len),
                  max_len=max_len, window=rng.choice([0, 0, 0, 1, 100, 4096]), sinks=rng.random() < 0.5,
                  lse=rng.random() < 0.3)
    if op == "step":
        attend.update(rot=rot, layout=layout, table_positions=32768 + 16)
    return attend


def _rows_of(case):
    """Rows of each sequence: the same for all, or anything from one to that many."""
    if not case["ragged"]:
        return [case["rows"]] * case["seqs"]
    r = random.Random("rows %d %d" % (case["seqs"], case["rows"]))
    return [case["rows"] if b == 0 else r.randint(1, case["rows"]) for b in range(case["seqs"])]


def _lens_of(case):
    """Positions of each sequence, the rows of the call included."""
    r = random.Random("lens %d %d %d" % (case["seqs"], case["min_len"], case["max_len"]))
    lens = [case["max_len"] if b == 0 else r.randint(case["min_len"], case["max_len"]) for b in range(case["seqs"])]
    if case["op"] != "attend":  # what is appended has a place
        lens = [max(n, m) for n, m in zip(lens, _rows_of(case))]
    return lens


# ------------------------------------------------------------- inputs and state
def _table(case, device):
    """{cos, sin} of each position and rotated pair, [positions][rot / 2][2], the table that a program keeps."""
    rot, n, factor = case["rot"], case["table_positions"], case.get("factor", 1.0)
    scaling = case.get("scaling", "none")
    theta = THETA * factor ** (rot / (rot - 2)) if scaling == "ntk" else THETA
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    freq = theta ** (-2.0 * i / rot)
    mscale = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        original = n / factor

        def turn(beta):
            return rot * math.log(original / (beta * 2.0 * math.pi)) / (2.0 * math.log(theta))

        low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rot - 1)
        keep = 1.0 - ((i - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq / factor * (1.0 - keep) + freq * keep
        mscale = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(n, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.stack((angle.cos(), angle.sin()), dim=-1) * mscale).float().contiguous()


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
    if case["op"] == "rope":
        s["table"] = _table(case, device)
        s["x"] = _rows(g, case["rows"], case["heads"], case["dim"], dtype, case["fused_row"], device)
        s["positions"] = torch.randint(0, case["table_positions"], (case["rows"],), device=device, generator=g,
                                       dtype=torch.int32)
        s["out"] = torch.empty(case["rows"], case["heads"], case["dim"], dtype=dtype, device=device)
        if own:
            s["rope"] = _fo().Rope(s["table"], layout=case["layout"])
        return s

    rows, lens, page = _rows_of(case), _lens_of(case), case["page"]
    total, seqs = sum(rows), case["seqs"]
    per_seq = -(-max(lens) // page)
    # Pages are handed out in any order.  An append touches a sequence's last pages alone, so only those are its own
    # there; an attention reads them all.
    if case["op"] == "append":
        first = [(n - m) // page for n, m in zip(lens, rows)]
    else:
        first = [0] * seqs
    used = sum(-(-n // page) - f for n, f in zip(lens, first))
    pages = used + 3
    order = torch.randperm(pages, device=device, generator=g).to(torch.int32).cpu().tolist()
    table, at = [[0] * per_seq for _ in range(seqs)], 0
    for b in range(seqs):
        for j in range(first[b], -(-lens[b] // page)):
            table[b][j] = order[at]
            at += 1
    s["page_table"] = torch.tensor(table, dtype=torch.int32, device=device)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=device)
    s["row_start"] = None
    if case["ragged"]:
        starts = [0]
        for n in rows:
            starts.append(starts[-1] + n)
        s["row_start"] = torch.tensor(starts, dtype=torch.int32, device=device)
    s["k_codes"], s["v_codes"] = _codes(g, pages, case, device), _codes(g, pages, case, device)
    s["k_scales"], s["v_scales"] = _scales(g, pages, case, device), _scales(g, pages, case, device)
    s["q"] = _rows(g, total, case["heads"], case["dim"], dtype, True, device)
    if case["op"] != "attend":
        s["table"] = _table(case, device)
        s["k"] = _rows(g, total, case["kv_heads"], case["dim"], dtype, True, device)
        s["v"] = _rows(g, total, case["kv_heads"], case["dim"], dtype, True, device)
        s["q_out"] = torch.empty(total, case["heads"], case["dim"], dtype=dtype, device=device)
    if case["op"] != "append":
        s["sinks"] = torch.randn(case["heads"], device=device, generator=g) if case["sinks"] else None
        s["out"] = torch.empty(total, case["heads"], case["dim"], dtype=dtype, device=device)
        s["lse"] = torch.empty(total, case["heads"], device=device) if case["lse"] else None
    if own:
        F = _fo()
        s["kv"] = F.PagedKv(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
        s["batch"] = F.PagedBatch(s["page_table"], s["lens"], rows=case["rows"], row_start=s["row_start"])
        if case["op"] != "attend":
            s["rope"] = F.Rope(s["table"], layout=case["layout"])
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


def _row_places(s):
    """Sequence, number within it, and position of every row."""
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


def _encode(x, scale, fmt):
    """x / scale as codes; a scale of zero has only zeros."""
    y = torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x))
    return _round(y, fmt)


def _round(y, fmt):
    y = y.round() if fmt == "i8" else y
    y = y.clamp(-QMAX[fmt], QMAX[fmt])
    return y.to(torch.int8) if fmt == "i8" else y.to(torch.float8_e4m3fn).view(torch.int8)


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
    b, _, position = _row_places(s)
    cos_sin = s["table"][position]
    page_id = s["page_table"][b, position // case["page"]].long()
    offset = position % case["page"]
    q = _rotate(s["q"].float(), cos_sin, case["layout"])
    k = _rotate(s["k"].float(), cos_sin, case["layout"])
    _store(s["k_codes"], s["k_scales"], k, page_id, offset, case["fmt"])
    _store(s["v_codes"], s["v_scales"], s["v"].float(), page_id, offset, case["fmt"])
    s["q_out"].copy_(q)


def _gathered(codes, scales, table):
    """[seqs][kv heads][positions][dim] FP32 of all pages that the table names."""
    x = codes.view(torch.int8)[table].view(codes.dtype).float() * scales[table][..., None, None]
    seqs, n, heads, page, dim = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(seqs, heads, n * page, dim)


def _attend(s, q):
    case = s["case"]
    heads, kv_heads, dim, rows, seqs = case["heads"], case["kv_heads"], case["dim"], case["rows"], case["seqs"]
    group = heads // kv_heads
    b, r, position = _row_places(s)
    padded = torch.zeros(seqs, rows, heads, dim, device=q.device)
    padded[b, r] = q.float()
    seen = torch.full((seqs, rows), -1, dtype=torch.long, device=q.device)
    seen[b, r] = position
    table = s["page_table"].long()
    k = _gathered(s["k_codes"], s["k_scales"], table)
    qg = padded.view(seqs, rows, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, rows * group, dim)
    score = torch.matmul(qg, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    del k
    j = torch.arange(score.shape[-1], device=q.device)
    visible = j <= seen[:, :, None]
    if case["window"]:
        visible &= j > seen[:, :, None] - case["window"]
    score = score.view(seqs, kv_heads, rows, group, -1).masked_fill(~visible[:, None, :, None, :], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    below = p.sum(dim=-1)
    lse = top[..., 0] + torch.log(below)
    total = below
    if s["sinks"] is not None:
        total = below + torch.exp(s["sinks"].view(1, kv_heads, 1, group) - top[..., 0])
    v = _gathered(s["v_codes"], s["v_scales"], table)
    o = torch.matmul(p.view(seqs, kv_heads, rows * group, -1), v).view(seqs, kv_heads, rows, group, dim)
    o = torch.where(total[..., None] > 0, o / torch.where(total > 0, total, torch.ones_like(total))[..., None],
                    torch.zeros_like(o))
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs, rows, heads, dim)
    s["out"].copy_(o[b, r])
    if s["lse"] is not None:
        s["lse"].copy_(lse.permute(0, 2, 1, 3).reshape(seqs, rows, heads)[b, r])


# ------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        F = _fo()
        if op == "rope":
            F.rope(s["x"], s["out"], s["rope"], positions=s["positions"], inverse=case["inverse"])
        q = s.get("q")
        if op in ("append", "step"):
            F.paged_append(s["kv"], s["batch"], s["k"], s["v"], rope=s["rope"], q=q, q_out=s["q_out"])
            q = s["q_out"]
        if op in ("attend", "step"):
            F.paged_attention(s["kv"], s["batch"], q, s["out"], sinks=s["sinks"], window=case["window"], lse=s["lse"])
    else:
        if op == "rope":
            x = _rotate(s["x"].float(), s["table"][s["positions"].long()], case["layout"], case["inverse"])
            s["out"].copy_(x)
        q = s.get("q")
        if op in ("append", "step"):
            _append(s)
            q = s["q_out"]
        if op in ("attend", "step"):
            _attend(s, q)
    return _outputs(s)


def _outputs(s):
    """Whole outputs.  An append's are the rotated queries and the cache: FP8 codes as the numbers that they are,
    int8 codes as whole numbers (held to equality, which is stricter than any bound on code times scale), and the
    scales beside them."""
    op = s["case"]["op"]
    got = {}
    if op in ("rope", "attend", "step"):
        got["out"] = s["out"]
    if op in ("append", "step"):
        got.update(q=s["q_out"], k_codes=s["k_codes"], v_codes=s["v_codes"], k_scales=s["k_scales"],
                   v_scales=s["v_scales"])
    if op in ("attend", "step") and s["lse"] is not None:
        got["lse"] = s["lse"]
    return got


def work(case):
    """Every input read once, every output written once."""
    wide = 4 if case["dtype"] == "f32" else 2
    dim = case["dim"]
    if case["op"] == "rope":
        moved = case["rows"] * case["heads"] * dim * wide * 2
        return {"bytes": moved + case["rows"] * (4 + case["rot"] * 4),
                "flops": case["rows"] * case["heads"] * case["rot"] * 3}
    rows, lens = _rows_of(case), _lens_of(case)
    total, kv_heads, heads = sum(rows), case["kv_heads"], case["heads"]
    b, f = 0, 0
    if case["op"] in ("append", "step"):
        b += total * (2 * kv_heads * dim * (wide + 1) + 2 * heads * dim * wide + case["rot"] * 4)
        f += total * (heads + kv_heads) * case["rot"] * 3 + total * 2 * kv_heads * dim * 3
    if case["op"] in ("attend", "step"):
        for n, m in zip(lens, rows):
            low = max(0, n - m + 1 - case["window"]) if case["window"] else 0
            b += (n - low) * kv_heads * dim * 2 + (n - low) // case["page"] * kv_heads * 8
            for r in range(m):
                p = n - m + r + 1
                f += max(0, min(p, case["window"]) if case["window"] else p) * heads * dim * 4
        b += total * heads * dim * wide * 2
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------- the same in 64 bits
def _exact_rope(x, table, positions, layout, inverse):
    """Complex multiplication of each pair by its {cos, sin}."""
    t = table.double()[positions.long()]
    turn = torch.complex(t[..., 0], -t[..., 1] if inverse else t[..., 1])[:, None, :]
    pairs = turn.shape[-1]
    y = x.double().clone()
    head = y[..., :2 * pairs]
    if layout == "interleaved":
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
    case = s["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = heads // kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    at = 0
    for n, m, pages in zip(_lens_of(case), _rows_of(case), s["page_table"].long()):
        low = max(0, n - m + 1 - case["window"]) if case["window"] else 0
        ids = pages[low // page:-(-n // page)]
        base = low // page * page

        def values(codes, scales):
            x = codes.view(torch.int8)[ids].view(codes.dtype) if codes.element_size() == 1 else codes[ids]
            x = x.double() * scales[ids].double()[:, :, None, None]
            return x.transpose(0, 1).reshape(kv_heads, -1, dim)

        k, v = values(k_codes, k_scales), values(v_codes, v_scales)
        for r in range(m):
            p = n - m + r
            if p < 0:
                continue
            first = max(0, p + 1 - case["window"]) if case["window"] else 0
            kk, vv = k[:, first - base:p + 1 - base], v[:, first - base:p + 1 - base]
            score = torch.einsum("hgd,hnd->hgn", q[at + r].double().view(kv_heads, group, dim), kk) / math.sqrt(dim)
            z = torch.logsumexp(score, dim=-1)
            weight = torch.exp(score - z[..., None])
            o = torch.einsum("hgn,hnd->hgd", weight, vv)
            if s["sinks"] is not None:
                o = o * torch.sigmoid(z - s["sinks"].double().view(kv_heads, group))[..., None]
            out[at + r], lse[at + r] = o.reshape(heads, dim), z.reshape(heads)
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
        return {"out": _exact_rope(s["x"], s["table"], s["positions"], case["layout"], case["inverse"])}
    rows, lens = _rows_of(case), _lens_of(case)
    got, q = {}, s["q"]
    caches = [s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"]]
    if case["op"] in ("append", "step"):
        at = torch.tensor([n - m + r for n, m in zip(lens, rows) for r in range(m)], device=q.device)
        table = s["page_table"].cpu().tolist()
        q = _exact_rope(s["q"], s["table"], at, case["layout"], False)
        k = _exact_rope(s["k"], s["table"], at, case["layout"], False)
        caches = [c.double() for c in caches]
        _exact_store(caches[0], caches[2], k, rows, lens, table, case)
        _exact_store(caches[1], caches[3], s["v"].double(), rows, lens, table, case)
        whole = case["fmt"] == "i8"
        got.update(q=q, k_codes=None if whole else caches[0], v_codes=None if whole else caches[1],
                   k_scales=caches[2], v_scales=caches[3])
    if case["op"] in ("attend", "step"):
        out, lse = _exact_attend(s, q, *caches)
        got["out"] = out
        if case["lse"]:
            got["lse"] = lse
    return got
