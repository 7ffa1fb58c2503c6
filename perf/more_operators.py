"""Measured calls of the operators for audio without an end: attention with a sliding window and sinks, over whole
segments and over the 4-bit cache; the cache's tables made on the GPU; and how sure a recognizer is of its tokens.

Frame t of a segment or stream attends the frames

    A(t) = { j : j <= t + right, and j >= t - left or j < sinks }

that it has: a window that slides with it, and a few first frames that stay visible (sinks). Its scores are the encoder's,

    s(t, j) = ((q_t + u) . k_j + (q_t + w) . p_(center - min(t - j, left))) / sqrt(dk)

or q_t . k_j / sqrt(dk) alone, a sink behind the window taking the position of distance left; then a softmax and the
weighted values. Over the cache, a frame whose page the stream does not hold is not attended.

The plan of a step is made from what each stream brings: its rows in the call, the pages that the window has left (but the
sinks') put behind the pool's queue of free ones, and pages for new frames taken from its front.

A row of logits gives the log probabilities of given tokens, its distribution's entropy, and its most probable tokens.
"""
import itertools
import math
import random

import torch

own = False

PAGE = 64
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a microphone's segment of 30.72 s, the encoder's limited context of ten seconds each way
        {"name": "window_1x384_segment", "kind": "window", "B": 1, "T": 384, "T_lo": 384, "H": 8, "G": 8, "dk": 128,
         "positions": True, "left": 128, "right": 128, "sinks": 4, "lengths": 1},
        # a batch of sentences of all lengths, look-ahead of about a second
        {"name": "window_16x750_ragged", "kind": "window", "B": 16, "T": 750, "T_lo": 20, "H": 8, "G": 8, "dk": 128,
         "positions": True, "left": 70, "right": 13, "sinks": 1, "lengths": 2},
        # causal, content scores alone, heads of 64 dimensions, four queries' heads to one
        {"name": "window_4x3000_shared", "kind": "window", "B": 4, "T": 3000, "T_lo": 2001, "H": 16, "G": 4, "dk": 64,
         "positions": False, "left": 511, "right": 0, "sinks": 8, "lengths": 3},
        # an hour of audio in one piece
        {"name": "window_1x45000_hour", "kind": "window", "B": 1, "T": 45000, "T_lo": 45000, "H": 8, "G": 8, "dk": 128,
         "positions": True, "left": 128, "right": 128, "sinks": 16, "lengths": 4},
        # one live microphone, a frame at a time, an hour into it
        {"name": "sinks_1x1_live", "kind": "sinks", "B": 1, "T": 1, "T_lo": 1, "len_lo": 44999, "len_hi": 44999,
         "H": 8, "G": 8, "dk": 128, "positions": True, "left": 70, "right": 0, "sinks": 4, "lengths": 5},
        # 16 streams served together in chunks of about a second, heads of 64 dimensions shared
        {"name": "sinks_16x14_shared", "kind": "sinks", "B": 16, "T": 14, "T_lo": 5, "len_lo": 0, "len_hi": 9000,
         "H": 16, "G": 4, "dk": 64, "positions": False, "left": 1000, "right": 13, "sinks": 16, "lengths": 6},
        # a full machine: 256 meetings of up to an hour, a frame each, a minute behind it
        {"name": "sinks_256x1_meetings", "kind": "sinks", "B": 256, "T": 1, "T_lo": 1, "len_lo": 3000, "len_hi": 45000,
         "H": 8, "G": 8, "dk": 128, "positions": True, "left": 750, "right": 0, "sinks": 64, "lengths": 7},
        # the step of 256 streams of one or two frames each
        {"name": "plan_256x2", "kind": "plan", "B": 256, "T": 2, "T_lo": 1, "columns": 2048, "len_lo": 0, "len_hi": 9000,
         "left": 750, "sinks": 16, "fresh": 0.0, "lengths": 8},
        # 48 requests of 20 to 30 s that take the places of others
        {"name": "plan_48_requests", "kind": "plan", "B": 48, "T": 384, "T_lo": 250, "columns": 64, "len_lo": 300,
         "len_hi": 3000, "left": -1, "sinks": 0, "fresh": 1.0, "lengths": 9},
        # the joint's token just taken, as each step of a live decoder asks
        {"name": "answer_1x1025", "kind": "answer", "rows": 1, "cols": 1025, "stride": 1040, "given": 1, "top": 4},
        # all frames of an hour's audio, with the alternatives that a lattice keeps
        {"name": "answer_45000x1025", "kind": "answer", "rows": 45000, "cols": 1025, "stride": 1040, "given": 1, "top": 8},
        # rows of a large vocabulary
        {"name": "answer_64x131072", "kind": "answer", "rows": 64, "cols": 131072, "stride": 131072, "given": 2, "top": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "window", "sinks", "sinks", "plan", "answer", "answer"])
    if kind == "answer":
        cols = _log(rng, 2, 200000)
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(100000, 40000000 // cols))), "cols": cols,
                "stride": cols + rng.choice([0, 0, rng.randint(1, 40)]), "given": rng.randint(1, 4),
                "top": rng.randint(0, min(20, cols))}
    if kind == "plan":
        B = _log(rng, 1, 512)
        far = _log(rng, 16, 45000)
        T = _log(rng, 1, min(750, max(1, 60000 // B)))
        return {"kind": kind, "B": B, "T": T, "T_lo": rng.randint(0, T), "columns": -(-far // PAGE) + rng.randint(8, 512),
                "len_lo": rng.randint(0, far), "len_hi": far, "left": rng.choice([-1, _log(rng, 1, 3000)]),
                "sinks": rng.choice([0, rng.randint(1, 200)]), "fresh": rng.choice([0.0, 0.1, 1.0]),
                "lengths": rng.randrange(1 << 30)}
    H, G, dk = rng.choice([(8, 8, 128), (8, 8, 128), (8, 8, 64), (16, 4, 64), (8, 2, 128), (4, 4, 32), (6, 3, 96)])
    B = _log(rng, 1, 64 if kind == "window" else 256)
    T = _log(rng, 1, max(1, (20000 if kind == "window" else min(750 * B, 2000)) // B))
    left = rng.choice([-1, _log(rng, 1, 600), _log(rng, 1, 600)])
    if left < 0 and (kind == "sinks" or T > 1500):
        left = rng.randint(0, 1000)
    case = {"kind": kind, "B": B, "T": T, "T_lo": rng.randint(1, T), "H": H, "G": G, "dk": dk,
            "positions": rng.random() < 0.7, "left": left, "right": rng.choice([0, rng.randint(0, 200), rng.randint(0, T)]),
            "sinks": rng.choice([0, rng.randint(1, 16), rng.randint(1, 150)]), "lengths": rng.randrange(1 << 30)}
    if kind == "window":
        case["right"] = min(case["right"], 600)
    else:
        far = _log(rng, 16, 45000)
        case |= {"len_lo": rng.randint(0, far), "len_hi": far}
    return case


# ---------------------------------------------------------------- inputs --

def _record(dk):
    return PAGE * dk + 4 * PAGE


def _lengths(case):
    """Each stream's frames before the call, and its frames in the call."""
    r = random.Random(case["lengths"])
    pairs = [(r.randint(case.get("len_lo", 0), case.get("len_hi", 0)), r.randint(case["T_lo"], case["T"]))
             for _ in range(case["B"])]
    return [a for a, _ in pairs], [t for _, t in pairs]


def _reach(case, before, rows):
    """How far back and ahead a frame attends at most, but to sinks."""
    most_left = max(b + t - 1 for b, t in zip(before, rows))
    return (most_left if case["left"] < 0 else min(case["left"], most_left)), min(case["right"], max(rows) - 1)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=g.device)


def _offsets(rows, dev):
    return torch.tensor([0] + list(itertools.accumulate(rows)), dtype=torch.int32, device=dev)


def _kept(g, pages, G, dk):
    """A pool as writes of normal values leave it: half bytes with the levels' shares, scales around their mean."""
    r = torch.rand(pages, G, PAGE * dk, 2, generator=g, device=g.device)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=g.device) * (2.75 / 6)
    magnitude = torch.bucketize((2 * r - 1).abs().contiguous(), torch.erf(edges / math.sqrt(2.0)))
    half = torch.where((r > 0.5) & (magnitude > 0), magnitude + 8, magnitude)
    data = torch.empty(1, pages, G, _record(dk), dtype=torch.uint8, device=g.device)
    data[0, :, :, :PAGE * dk] = (half[..., 0] | (half[..., 1] << 4)).to(torch.uint8)
    d = 0.46 * (0.7 + 0.6 * torch.rand(pages, G, 2 * PAGE, generator=g, device=g.device))
    data[0, :, :, PAGE * dk:] = d.to(torch.bfloat16).view(torch.uint8)
    return data


def _held(case, before, rows, dev):
    """Which columns of each stream's table are held: those its window may yet reach, the sinks', to its last frame."""
    columns = case.get("columns") or max(-(-(b + t) // PAGE) for b, t in zip(before, rows))
    col = torch.arange(columns, device=dev)
    b, t = (torch.tensor(x, device=dev)[:, None] for x in (before, rows))
    gone = torch.zeros_like(b) if case["left"] < 0 else (b - case["left"]).clamp_min(0) // PAGE
    return ((col >= gone) | (col < -(-case["sinks"] // PAGE))) & (col < -(-(b + t) // PAGE)), gone[:, 0]


def _dealt(g, mark, pages):
    """A table whose marked entries are pages of the pool in a random order, the others holes, and the pages left."""
    order = torch.randperm(pages, generator=g, device=g.device).to(torch.int32)
    rank = torch.cumsum(mark.flatten(), 0).reshape(mark.shape) - 1
    n = int(mark.sum())
    return torch.where(mark, order[rank.clamp_min(0)], -1).contiguous(), order[n:]


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "answer":    # a recognizer's logits: one token stands out, by much or by little
        n, cols = case["rows"], case["cols"]
        s["logits"] = 2.0 * _normal(g, n, case["stride"])
        best = torch.randint(0, cols, (n, 1), generator=g, device=dev)
        s["logits"].scatter_add_(1, best, 14.0 * torch.rand(n, 1, generator=g, device=dev))
        other = torch.randint(0, cols, (n, case["given"]), generator=g, device=dev)
        taken = torch.rand(n, case["given"], generator=g, device=dev) < 0.8
        s["tokens"] = torch.where(taken, best, other).to(torch.int32)
        return s
    before, rows = _lengths(case)
    if case["kind"] == "plan":
        B, columns = case["B"], case["columns"]
        r = torch.rand(B, generator=g, device=dev)
        s["fresh"] = (r < case["fresh"]).to(torch.int32)
        mark, gone = _held(case, before, [0] * B, dev)
        grow = 2 + -(-case["T"] // PAGE)
        pages = int(mark.sum()) + B * grow + 5
        s["table"], free = _dealt(g, mark, pages)
        s["state"] = torch.stack([torch.tensor(before, device=dev), gone], 1).to(torch.int32).contiguous()
        head = 3 if pages > 3 else 0        # the queue of free pages lies in a ring
        ring = torch.full((pages,), -1, dtype=torch.int32, device=dev)
        ring[(head + torch.arange(len(free), device=dev)) % pages] = free
        s["pool"] = torch.cat([torch.tensor([head, len(free)], dtype=torch.int32, device=dev), ring])
        s["add"] = torch.tensor(rows, dtype=torch.int32, device=dev)
        s["rows"], s["T"] = B * case["T"], case["T"]
        return s
    H, G, dk, N = case["H"], case["G"], case["dk"], sum(rows)
    s["row0"], s["N"], s["T"] = _offsets(rows, dev), N, max(rows)
    s["q"] = 1.5 * _normal(g, N, H * dk)
    if case["kind"] == "window":
        s["k"], s["v"] = _normal(g, N, G * dk), _normal(g, N, G * dk)
    else:
        mark, _ = _held(case, before, rows, dev)
        pages = int(mark.sum()) + 3
        s["table"], _ = _dealt(g, mark, pages)
        s["data"] = _kept(g, pages, G, dk)
        s["before"] = torch.tensor(before, dtype=torch.int32, device=dev)
    left, right = _reach(case, before, rows)
    s["left"], s["right"] = (None if case["left"] < 0 else case["left"]), case["right"]
    s["p"] = None
    if case["positions"]:
        s["p"], s["center"] = _normal(g, left + right + 1, H * dk), left
        s["u"], s["w"] = 0.1 * _normal(g, H * dk), 0.1 * _normal(g, H * dk)
        s["right"] = right
        s["left"] = left
    return s


# ------------------------------------------------------- the plain forms --

def _softmax_values(parts):
    """The weighted values over pairs (scores, -infinity where not attended; values) together: zeros where nothing is."""
    top = torch.stack([a.amax(-1) for a, _ in parts]).amax(0)[..., None]
    top = torch.where(top > -math.inf, top, 0.0)
    es = [torch.exp(a - top) for a, _ in parts]
    total = torch.stack([e.sum(-1) for e in es]).sum(0)[..., None]
    o = torch.stack([e @ v for e, (_, v) in zip(es, parts)]).sum(0)
    return o / torch.where(total > 0, total, 1.0)


def _by_heads(x, G):
    """[..., K, G * dk] to [..., G, K, dk]"""
    return x.reshape(*x.shape[:-1], G, -1).transpose(-2, -3)


def _queries(s, q, C):
    """Queries with the biases of content and place, as [..., G, H / G * C, dk]."""
    case = s["case"]
    G, Hg, dk = case["G"], case["H"] // case["G"], case["dk"]
    lead = q.shape[:-2]

    def laid(x):
        return x.reshape(*lead, C, G, Hg, dk).movedim(-4, -2).reshape(*lead, G, Hg * C, dk)
    return (laid(q), None) if s["p"] is None else (laid(q + s["u"]), laid(q + s["w"]))


def _place(s, place, C, m):
    """Position scores of m [..., C, K]'s rows of the table, as [..., G, H / G * C, K]."""
    case = s["case"]
    G, Hg, dk = case["G"], case["H"] // case["G"], case["dk"]
    lead = place.shape[:-3]
    p = s["p"].reshape(-1, G, Hg, dk).permute(1, 2, 3, 0)               # [G, Hg, dk, n]
    every = place.reshape(*lead, G, Hg, C, dk) @ p
    m = m.clamp(0, p.shape[-1] - 1)[..., None, None, :, :].expand(*lead, G, Hg, C, m.shape[-1])
    return torch.gather(every, -1, m).reshape(*lead, G, Hg * C, m.shape[-1])


def _scores(s, content, place, k, C, m, seen):
    score = content @ k.transpose(-1, -2)
    if place is not None:
        score = score + _place(s, place, C, m)
    score = score / math.sqrt(s["case"]["dk"])
    Hg = s["case"]["H"] // s["case"]["G"]
    seen = seen[..., None, None, :, :].expand(*score.shape[:-2], Hg, *seen.shape[-2:]).reshape(score.shape)
    return torch.where(seen, score, -math.inf)


def _plain_window(s):
    """Blocks of C queries of a segment, each with the frames that its window can reach, and the sinks."""
    case = s["case"]
    G, B, T, N, sinks = case["G"], case["B"], s["T"], s["N"], min(case["sinks"], s["T"])
    dev, row0 = s["q"].device, s["row0"].long()
    count = (row0[1:] - row0[:-1])[:, None, None]
    left = T - 1 if s["left"] is None else min(s["left"], T - 1)
    right = min(s["right"], T - 1)
    C = min(256, T)
    nb = -(-T // C)
    t = torch.arange(nb * C, device=dev).reshape(nb, C)
    j = t[:, :1] - left + torch.arange(left + C + right, device=dev)     # a block's frames
    first = row0[:-1, None, None]
    q = s["q"][(first + t).clamp_max(N - 1)]                            # [B, nb, C, H dk]
    content, place = _queries(s, q, C)
    k, v = (_by_heads(s[n][(first + j).clamp(0, N - 1)], G) for n in ("k", "v"))
    t, j = t[..., None], j[:, None]
    seen = (j >= t - left) & (j <= t + right) & (j >= 0) & (j < count[..., None])
    center = s.get("center", 0)
    m = (center - t + j)[None].expand(B, -1, -1, -1)
    parts = [(_scores(s, content, place, k, C, m, seen), v)]
    if sinks:
        f = torch.arange(sinks, device=dev)
        sk, sv = (_by_heads(s[n][(row0[:-1, None] + f).clamp_max(N - 1)], G)[:, None] for n in ("k", "v"))
        seen = ((f < t - left) & (f < count[..., None])).expand(B, nb, C, sinks)
        m = torch.full_like(seen, center - left, dtype=torch.int64)
        parts.append((_scores(s, content, place, sk, C, m, seen), sv.expand(B, nb, G, sinks, -1)))
    o = _softmax_values(parts)                                          # [B, nb, G, Hg C, dk]
    o = o.reshape(B, nb, G, -1, C, case["dk"]).movedim(4, 2).reshape(B, nb * C, -1)
    return o[torch.arange(nb * C, device=dev) < count[:, 0]]


def _values(record, dk):
    """The keys and values that records [..., bytes] of the cache stand for: two of [..., 64, dk]."""
    byte = torch.arange(256, device=record.device)
    half = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=record.device)
    pair = torch.stack([half[byte & 15], half[byte >> 4]], -1)
    lead, ns, n = record.shape[:-1], dk // 32, record.dim() - 1
    k = pair[record[..., :PAGE * dk // 2].long()].reshape(*lead, PAGE, dk)
    v = pair[record[..., PAGE * dk // 2:PAGE * dk].long()]      # [c // 32][w][c % 16][c // 16 % 2][g][h][r // 2][r % 2]
    v = v.reshape(*lead, ns, 4, 16, 2, 2, 2, 2, 2)
    v = v.permute(*range(n), n + 4, n + 5, n + 1, n + 6, n + 7, n, n + 3, n + 2).reshape(*lead, PAGE, dk)
    d = record[..., PAGE * dk:].contiguous().view(torch.bfloat16).float()
    return k * d[..., :PAGE, None], v * d[..., PAGE:, None]


def _plain_sinks(s):
    """The pages that a stream's window can reach, behind those of its sinks."""
    case = s["case"]
    G, dk, B, T, N = case["G"], case["dk"], case["B"], s["T"], s["N"]
    dev, before, row0 = s["q"].device, s["before"].long()[:, None], s["row0"].long()
    count = (row0[1:] - row0[:-1])[:, None]
    columns = s["table"].shape[1]
    left = columns * PAGE if s["left"] is None else s["left"]
    first = (before - left).clamp_min(0) // PAGE                        # the window's first page
    ns, nw = min(columns, -(-case["sinks"] // PAGE)), min(columns, (left + T + PAGE - 2) // PAGE + 1)
    window = first + torch.arange(nw, device=dev)
    col = torch.cat([torch.arange(ns, device=dev).expand(B, ns), window], 1)
    page = torch.gather(s["table"].long(), 1, col.clamp_max(columns - 1))
    there = (page >= 0) & (col < columns) & ((torch.arange(ns + nw, device=dev) >= ns) | (col < first))
    k, v = _values(s["data"][0][page.clamp_min(0)], dk)                 # [B, pages, G, 64, dk]
    k, v = (x.transpose(1, 2).reshape(B, G, -1, dk) for x in (k, v))
    j = (col[..., None] * PAGE + torch.arange(PAGE, device=dev)).reshape(B, 1, -1)
    i = torch.arange(T, device=dev)
    q = s["q"][(row0[:-1, None] + i).clamp_max(N - 1)]
    content, place = _queries(s, q, T)
    t = (before + i)[..., None]
    seen = there.repeat_interleave(PAGE, 1)[:, None] & (j < (before + count)[..., None]) & (j <= t + s["right"])
    seen = seen & ((j >= t - left) | (j < case["sinks"]))
    m = s.get("center", 0) - (t - j).clamp_max(left)
    o = _softmax_values([(_scores(s, content, place, k, T, m, seen), v)])
    o = o.reshape(B, G, -1, T, dk).movedim(3, 1).reshape(B, T, -1)
    return o[i < count]


def _plain_plan(s):
    case, table, pool = s["case"], s["table"], s["pool"]
    dev, columns = table.device, table.shape[1]
    pages, cap = len(pool) - 2, PAGE * table.shape[1]
    fresh = s["fresh"] != 0
    had, gone = s["state"][:, 0].clamp(0, cap).long(), s["state"][:, 1].long()
    start = torch.where(fresh, 0, had)
    most = (cap - start).clamp_max(s["T"])
    row0 = torch.cat([start.new_zeros(1), torch.minimum(s["add"].long(), most).clamp_min(0).cumsum(0)]).clamp_max(s["rows"])
    T = row0[1:] - row0[:-1]
    behind = torch.zeros_like(start) if case["left"] < 0 else (start - case["left"]).clamp_min(0) // PAGE
    from_ = gone.clamp_min(-(-case["sinks"] // PAGE))
    c = torch.arange(columns, device=dev)
    back = torch.where(fresh[:, None], c < (-(-had // PAGE))[:, None], (c >= from_[:, None]) & (c < behind[:, None]))
    given = back & (table >= 0) & (table < pages)
    head, free = pool[0].long(), pool[1].long()
    rank = torch.cumsum(given.flatten(), 0).reshape(given.shape)
    ring = torch.cat([pool[2:], pool.new_zeros(1)])                     # one place more, for what is not given back
    ring[torch.where(given, (head + free + rank - 1) % pages, pages)] = table
    free = free + rank[-1, -1]
    need = (c >= (-(-start // PAGE))[:, None]) & (c < (-(-(start + T) // PAGE))[:, None])
    rank = torch.cumsum(need.flatten(), 0).reshape(need.shape)
    taken = torch.minimum(rank[-1, -1], free)
    id_ = torch.where(rank <= free, ring[(head + rank - 1) % pages], -1)
    table.copy_(torch.where(need, id_, torch.where(back, -1, table)))
    s["state"].copy_(torch.stack([start + T, torch.where(fresh, 0, torch.maximum(gone, behind))], 1))
    pool[2:] = ring[:pages]
    pool[0], pool[1] = (head + taken) % pages, free - taken
    r = torch.arange(s["rows"], device=dev)
    b = torch.searchsorted(row0[1:].contiguous(), r, right=True).clamp_max(case["B"] - 1)
    f = (start[b] + r - row0[b]).clamp(0, cap - 1)
    page = table[b, f // PAGE].long()
    slot = torch.where((r < row0[-1]) & (page >= 0) & (page < pages), PAGE * page + f % PAGE, -1)
    told = torch.stack([row0[-1], s["add"].long().clamp_min(0).sum() - row0[-1], rank[-1, -1] - taken, free - taken])
    return [table, s["state"], pool] + [x.to(torch.int32) for x in (start, row0, slot, told)]


def _plain_answer(s):
    case = s["case"]
    logits = s["logits"][:, :case["cols"]]
    most = logits.amax(1, keepdim=True)
    x = logits - most
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    given = torch.gather(x, 1, s["tokens"].long()) - torch.log(total)
    entropy = torch.log(total[:, 0]) - (e * x).sum(1) / total[:, 0]
    if not case["top"]:
        return [given, entropy]
    best, at = (y[:, :case["top"]] for y in torch.sort(logits, dim=1, descending=True, stable=True))
    return [given, entropy, at.to(torch.int32), best - most - torch.log(total)]


# ------------------------------------------------------------------ runs --

def _handles(s):
    """What a program keeps between calls: descriptors, workspaces and outputs."""
    import libpktito_amd as pk
    s["pk"], case = pk, s["case"]
    if case["kind"] == "answer":
        x, k = s["logits"], case["top"]
        s["out"] = [torch.empty_like(s["tokens"], dtype=torch.float32), torch.empty_like(x[:, 0])]
        if k:
            s["out"] += [torch.empty(len(x), k, dtype=torch.int32, device=x.device),
                         torch.empty(len(x), k, device=x.device)]
        need = pk.logprobs_workspace(case["rows"], case["cols"], k)
        s["ws"] = torch.empty(need, dtype=torch.uint8, device=x.device)
        return
    if case["kind"] == "plan":
        slot = torch.empty(s["rows"], dtype=torch.int32, device=s["table"].device)
        s["plan"] = pk.CachePlan(s["table"], s["state"], s["pool"], s["rows"], s["T"], slot)
        return
    s["o"] = torch.empty_like(s["q"])
    s["at"] = None if s["p"] is None else (s["p"], s["center"], s["u"], s["w"])
    if case["kind"] == "window":
        s["segments"] = pk.Segments(s["row0"], s["N"], s["T"])
        return
    s["cache"] = pk.DeviceCache(s["data"], *s["data"].shape[:3], case["dk"])
    s["streams"] = pk.CacheStreams(s["table"], s["before"], s["row0"], s["N"], s["T"])
    need = s["cache"].attention_workspace(s["streams"], case["H"], s["at"], s["left"], s["right"], case["sinks"])
    s["ws"] = torch.empty(need, dtype=torch.uint8, device=s["q"].device)


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if own:
        if "pk" not in s:
            _handles(s)
        if kind == "answer":
            s["pk"].logprobs_dev(s["logits"][:, :case["cols"]], s["tokens"], *s["out"], ws=s["ws"])
            return s["out"]
        if kind == "plan":
            plan = s["plan"]
            plan.step(s["add"], s["fresh"], None if case["left"] < 0 else case["left"], case["sinks"])
            return [s["table"], s["state"], s["pool"], plan.streams.len, plan.streams.row0, plan.slot, plan.told]
        if kind == "window":
            s["pk"].attention_window_dev(s["o"], s["q"], s["k"], s["v"], s["segments"], case["H"], case["dk"], s["at"],
                                         s["left"], s["right"], case["sinks"])
        else:
            s["cache"].attention(s["o"], 0, s["q"], s["streams"], case["H"], s["ws"], s["at"], s["left"], s["right"],
                                 sinks=case["sinks"])
        return s["o"]
    if kind == "answer":
        return _plain_answer(s)
    if kind == "plan":
        return _plain_plan(s)
    return _plain_window(s) if kind == "window" else _plain_sinks(s)


def work(case):
    if case["kind"] == "answer":
        n = case["rows"]
        return {"bytes": 4 * n * case["cols"] + 4 * n * (2 * case["given"] + 1 + 2 * case["top"]), "flops": 0}
    before, rows = _lengths(case)
    if case["kind"] == "plan":      # what streams bring, their state, offsets and slots; a page's entry given or taken twice
        moved = sum(-(-(b + t) // PAGE) - -(-b // PAGE) for b, t in zip(before, rows))
        if case["fresh"] == 1.0:
            moved = sum(-(-t // PAGE) + -(-b // PAGE) for b, t in zip(before, rows))
        return {"bytes": case["B"] * (4 + 4 + 16 + 4 + 4) + 4 * case["B"] * case["T"] + 8 * moved, "flops": 0}
    G, dk, N, H = case["G"], case["dk"], sum(rows), case["H"]
    left, right = _reach(case, before, rows)
    pairs = frames = 0
    for b, t in zip(before, rows):
        frames += b + t - max(0, b - left) + max(0, min(case["sinks"], b - left))
        for i in range(b, b + t):
            pairs += min(b + t - 1, i + right) - max(0, i - left) + 1 + max(0, min(case["sinks"], i - left))
    flops = 2 * pairs * H * dk * (3 if case["positions"] else 2)
    places = left + right + 1 if case["positions"] else 0
    kept = 8 * N * G * dk if case["kind"] == "window" else frames * G * (dk + 4)
    return {"bytes": kept + 4 * places * H * dk + 8 * N * H * dk, "flops": flops}


# ----------------------------------------------------------- 64-bit values --

def _exact_values(head, dk):
    """Keys and values of one head's records [held, bytes], by their places."""
    level = torch.tensor(LEVELS, dtype=torch.float64, device=head.device)
    c = torch.arange(dk, device=head.device)
    f = torch.arange(PAGE, device=head.device)

    def taken(at, high):
        b = (head[:, at.reshape(-1)].long() >> (4 * high.expand(PAGE, dk).reshape(-1))) & 15
        return (torch.where(b >= 8, -1.0, 1.0).double() * level[b & 7]).reshape(-1, dk)

    k = taken(f[:, None] * (dk // 2) + c // 2, c % 2)
    g, h, w, r = f // 32, f // 16 % 2, f // 4 % 4, f % 4
    at = 1024 * (c // 32) + 16 * (c % 16) + 8 * (c // 16 % 2) + (256 * w + 4 * g + 2 * h + r // 2)[:, None]
    v = taken(PAGE * dk // 2 + at, (r % 2)[:, None])
    d = head[:, PAGE * dk:].contiguous().view(torch.bfloat16).double()
    return k * d[:, :PAGE].reshape(-1, 1), v * d[:, PAGE:].reshape(-1, 1)


def _exact_rows(s, out, r0, pos, frames, total, k, v, kept):
    """One head's kept frames (numbers `frames` of a stream of `total`) attended by rows r0 on, at positions pos."""
    case = s["case"]
    dk, Hg = case["dk"], case["H"] // case["G"]
    left = 1 << 40 if s["left"] is None else s["left"]
    dist = pos[:, None] - frames
    seen = (dist >= -s["right"]) & ((dist <= left) | (frames < case["sinks"])) & (frames < total)
    rows = slice(r0, r0 + len(pos))
    for h in range(kept * Hg, (kept + 1) * Hg):
        c = slice(h * dk, (h + 1) * dk)
        q = s["q"][rows, c].double()
        if s["p"] is None:
            score = q @ k.T.contiguous()
        else:
            at = (q + s["w"][c].double()) @ s["p"][:, c].double().T.contiguous()
            m = s["center"] - dist.clamp_max(left)
            score = (q + s["u"][c].double()) @ k.T.contiguous() + torch.gather(at, 1, m.clamp(0, at.shape[1] - 1))
        score = torch.where(seen, score / math.sqrt(dk), -math.inf)
        out[rows, c] = torch.softmax(score, 1) @ v


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    if case["kind"] == "answer":
        lp, entropy, best = [], [], []
        for x, tokens in zip(s["logits"][:, :case["cols"]].split(2048), s["tokens"].split(2048)):
            y = torch.log_softmax(x.double(), 1)
            lp.append(y[torch.arange(len(y), device=y.device)[:, None], tokens.long()])
            entropy.append(-(torch.exp(y) * y).sum(1))
            best.append(torch.topk(y, case["top"], 1)[0])
        got = [torch.cat(lp), torch.cat(entropy)]
        return got + [None, torch.cat(best)] if case["top"] else got
    before, rows = _lengths(case)
    dk, G, dev = case["dk"], case["G"], s["q"].device
    out = torch.zeros(s["N"], case["H"] * dk, dtype=torch.float64, device=dev)
    left = 1 << 40 if s["left"] is None else s["left"]
    r0 = 0
    for b, (len_b, t) in enumerate(zip(before, rows)):
        total = len_b + t
        for i0 in range(0, t, 2048):
            pos = len_b + torch.arange(i0, min(t, i0 + 2048), device=dev)
            lo, hi = max(0, len_b + i0 - left), min(total, len_b + min(t, i0 + 2048) + s["right"])
            if case["kind"] == "window":
                frames = torch.cat([torch.arange(min(lo, case["sinks"]), device=dev), torch.arange(lo, hi, device=dev)])
                at = r0 + frames
                for kept in range(G):
                    c = slice(kept * dk, (kept + 1) * dk)
                    _exact_rows(s, out, r0 + i0, pos, frames, total, s["k"][at, c].double(), s["v"][at, c].double(), kept)
                continue
            lo = lo // PAGE
            col = torch.cat([torch.arange(min(lo, -(-case["sinks"] // PAGE)), device=dev),
                             torch.arange(lo, -(-total // PAGE), device=dev)])
            record = s["data"][0, s["table"][b, col].long()]
            frames = (col[:, None] * PAGE + torch.arange(PAGE, device=dev)).reshape(-1)
            for kept in range(G):
                k, v = _exact_values(record[:, kept], dk)
                _exact_rows(s, out, r0 + i0, pos, frames, total, k, v, kept)
        r0 += t
    return out
