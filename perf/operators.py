"""Measured calls of the live-audio operators: keys and values kept in 4 bits between chunks of audio.

A recognizer that hears audio as it comes runs its encoder over a chunk of a few frames at a time (a frame is 80 ms) and
attends to the frames before it, whose keys and values it keeps. They are kept in pages of 64 frames in 4 bits, and
three operators work on them: the write of a chunk's keys and values, the attention of a chunk's frames to everything
kept, and the move of pages (a stream forked, a pool compacted). Many streams run in one call, each with its own length.

A page holds, for each layer and head of dk dimensions (32, 64, 96 or 128), a record of 64 dk + 256 bytes:

    keys    64 rows of dk / 2 bytes, dimension 2 b in byte b's low half, 2 b + 1 in its high half
    values  dimension c of frame 32 g + 16 h + 4 w + r (g, h < 2; w, r < 4) in half byte 4 h + r of the four bytes at
            1024 (c // 32) + 16 (16 w + c % 16) + 8 (c // 16 % 2) + 4 g
    scales  64 bfloat16 of the keys, 64 of the values

A half byte is a sign (8) and one of the eight levels 0, 1/2, 1, 3/2, 2, 3, 4, 6, times the scale of its frame and head:
the least bfloat16 whose six-fold is no less than the largest magnitude. The nearest level is taken, of two as near the
one with the even code. A head that holds a NaN or anything of 2^127 or more, or nothing of 2^-121 or more, is kept as
zeros.

The attention is the encoder's: frame i at position pos_i scores frame j by

    ((q_i + u) . k_j + (q_i + w) . p_(center - pos_i + j)) / sqrt(dk)

or by q_i . k_j / sqrt(dk) alone, over the frames from pos_i - left to pos_i + right that its stream has.
"""
import math
import random

import torch

own = False

PAGE = 64
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# halfway between neighbouring levels, and whether the value halfway goes up (to the even code)
HALFWAY = ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False))
LAYERS = 24


def listed():
    return [
        # one live microphone, a frame at a time, 70 frames (5.6 s) of left context: the smallest call
        {"name": "attend_1x1_left70", "kind": "attend", "B": 1, "T": 1, "T_lo": 1, "len_lo": 300, "len_hi": 300,
         "H": 8, "G": 8, "dk": 128, "positions": True, "left": 70, "right": 0, "lengths": 1},
        # 64 calls served together, two frames a step, up to a minute behind each
        {"name": "attend_64x2_minute", "kind": "attend", "B": 64, "T": 2, "T_lo": 2, "len_lo": 100, "len_hi": 750,
         "H": 8, "G": 8, "dk": 128, "positions": True, "left": -1, "right": -1, "lengths": 2},
        # chunks of about a second with look-ahead inside the chunk, ragged
        {"name": "attend_16x14_ragged", "kind": "attend", "B": 16, "T": 14, "T_lo": 5, "len_lo": 0, "len_hi": 1500,
         "H": 8, "G": 8, "dk": 128, "positions": True, "left": 1000, "right": 13, "lengths": 3},
        # a full machine: 256 meetings, a frame each, four to six minutes behind it
        {"name": "attend_256x1_meetings", "kind": "attend", "B": 256, "T": 1, "T_lo": 1, "len_lo": 3000, "len_hi": 4500,
         "H": 8, "G": 8, "dk": 128, "positions": True, "left": -1, "right": 0, "lengths": 4},
        # one frame against an hour of audio, content scores alone
        {"name": "attend_1x1_hour", "kind": "attend", "B": 1, "T": 1, "T_lo": 1, "len_lo": 44999, "len_hi": 44999,
         "H": 8, "G": 8, "dk": 128, "positions": False, "left": -1, "right": -1, "lengths": 5},
        # the longest segment in one piece, its cache just written: the whole attention of 30.72 s
        {"name": "attend_1x384_segment", "kind": "attend", "B": 1, "T": 384, "T_lo": 384, "len_lo": 0, "len_hi": 0,
         "H": 8, "G": 8, "dk": 128, "positions": True, "left": -1, "right": -1, "lengths": 6},
        # four files catching up, up to a minute a step after three to four minutes
        {"name": "attend_4x750_catch_up", "kind": "attend", "B": 4, "T": 750, "T_lo": 500, "len_lo": 2200,
         "len_hi": 3000, "H": 8, "G": 8, "dk": 128, "positions": True, "left": -1, "right": -1, "lengths": 7},
        # heads of 64 dimensions, four queries' heads to one kept head, causal
        {"name": "attend_8x3_shared_heads", "kind": "attend", "B": 8, "T": 3, "T_lo": 1, "len_lo": 2000, "len_hi": 9000,
         "H": 16, "G": 4, "dk": 64, "positions": False, "left": -1, "right": 0, "lengths": 8},
        # the write of the 64 calls' step
        {"name": "write_64x2", "kind": "write", "B": 64, "T": 2, "T_lo": 2, "len_lo": 100, "len_hi": 750,
         "H": 8, "G": 8, "dk": 128, "lengths": 9},
        # the write of whole segments: 48 of 20 to 30 s
        {"name": "write_48_segments", "kind": "write", "B": 48, "T": 384, "T_lo": 250, "len_lo": 0, "len_hi": 50,
         "H": 8, "G": 8, "dk": 128, "lengths": 10},
        # a stream forked: its last page copied in every layer
        {"name": "fork_2_pages", "kind": "move", "pages": 64, "pairs": 2, "layers": LAYERS, "G": 8, "dk": 128,
         "B": 0, "columns": 0},
        # a pool compacted: 300 pages moved down in every layer, the tables of 128 streams following
        {"name": "compact_300_pages", "kind": "move", "pages": 1200, "pairs": 300, "layers": LAYERS, "G": 8, "dk": 128,
         "B": 128, "columns": 9},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "attend", "attend", "write", "write", "move"])
    H, G, dk = rng.choice([(8, 8, 128), (8, 8, 128), (8, 8, 64), (16, 4, 64), (8, 2, 128), (4, 4, 32), (6, 3, 96)])
    if kind == "move":
        B = rng.choice([0, _log(rng, 1, 256)])
        return {"kind": kind, "pages": _log(rng, 40, 1200), "pairs": rng.randint(1, 20) if B == 0 else _log(rng, 4, 19),
                "layers": rng.choice([1, 17, LAYERS]), "G": G, "dk": dk, "B": B, "columns": rng.randint(1, 40) if B else 0}
    B = _log(rng, 1, 256)
    T = _log(rng, 1, max(1, min(750, (3000 if kind == "attend" else 16000) // B)))
    far = _log(rng, 16, max(16, min(45000, 900000 // B, 9000000 // (B * T))))
    case = {"kind": kind, "B": B, "T": T, "T_lo": rng.randint(1, T), "len_lo": rng.randint(0, far), "len_hi": far,
            "H": H, "G": G, "dk": dk, "lengths": rng.randrange(1 << 30)}
    if kind == "attend":
        case |= {"positions": rng.random() < 0.7, "left": rng.choice([-1, -1, _log(rng, 1, 2000)]),
                 "right": rng.choice([-1, 0, rng.randint(0, T)])}
        if case["positions"] and case["left"] < 0 and far > 6000:
            case["left"] = rng.randint(1000, 6000)
    return case


# ---------------------------------------------------------------- inputs --

def _record(dk):
    return PAGE * dk + 4 * PAGE


def _lengths(case):
    """Each stream's frames before the call, and its frames in the call."""
    r = random.Random(case["lengths"])
    pairs = [(r.randint(case["len_lo"], case["len_hi"]), r.randint(case["T_lo"], case["T"])) for _ in range(case["B"])]
    return [a for a, _ in pairs], [t for _, t in pairs]


def _reach(case, before, rows):
    """How far back and ahead a frame of the call attends at most."""
    most_left = max(b + t - 1 for b, t in zip(before, rows))
    most_right = max(rows) - 1
    left = most_left if case["left"] < 0 else min(case["left"], most_left)
    return left, most_right if case["right"] < 0 else min(case["right"], most_right)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=g.device)


def _kept(g, layers, pages, G, dk):
    """A pool as writes of normal values leave it: half bytes drawn with the levels' shares (a largest magnitude of
    2.75 deviations), scales around it."""
    data = torch.empty(layers, pages, G, _record(dk), dtype=torch.uint8, device=g.device)
    edges = torch.tensor([h for h, _ in HALFWAY], dtype=torch.float64) * (2.75 / 6)
    share = torch.erf(edges / math.sqrt(2.0))
    magnitude = torch.bucketize((torch.arange(2048, dtype=torch.float64) + 0.5) / 2048, share)
    half = torch.cat([magnitude, torch.where(magnitude > 0, magnitude + 8, magnitude)]).to(torch.uint8).to(g.device)
    flat = data.view(-1, _record(dk))
    step = max(1, (1 << 27) // _record(dk))
    for a in range(0, flat.shape[0], step):     # in parts, for the memory that the drawing takes
        part = flat[a:a + step]
        r = torch.randint(0, 1 << 24, (part.shape[0], PAGE * dk), generator=g, device=g.device, dtype=torch.int32)
        part[:, :PAGE * dk] = half[r & 4095] | (half[r >> 12] << 4)
        d = 0.46 * (0.7 + 0.6 * torch.rand(part.shape[0], 2 * PAGE, generator=g, device=g.device))
        part[:, PAGE * dk:] = d.to(torch.bfloat16).view(torch.uint8)
    return data


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    G, dk = case["G"], case["dk"]
    if case["kind"] == "move":
        data = torch.randint(0, 256, (case["layers"], case["pages"], G, _record(dk)), generator=g, device=dev,
                             dtype=torch.uint8)
        r = random.Random(seed)
        ids = r.sample(range(case["pages"]), 2 * case["pairs"])
        s = {"case": case, "data": data, "pairs": list(zip(ids[:case["pairs"]], ids[case["pairs"]:])), "table": None}
        if case["B"]:       # a table's entries: pages of the pool (never a page that is moved onto), some places empty
            live = torch.tensor(sorted(set(range(case["pages"])) - set(ids[case["pairs"]:])), device=dev)
            t = live[torch.randint(0, len(live), (case["B"], case["columns"]), generator=g, device=dev)]
            hole = torch.rand(case["B"], case["columns"], generator=g, device=dev) < 0.1
            s["table"] = torch.where(hole, -1, t).to(torch.int32)
        return s
    before, rows = _lengths(case)
    B, N, H = case["B"], sum(rows), case["H"]
    held = [-(-(b + t) // PAGE) for b, t in zip(before, rows)]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    column = torch.arange(max(held), device=dev)
    count = torch.tensor(held, device=dev)
    first = torch.cumsum(count, 0) - count
    table = order[(first[:, None] + column).clamp_max(pages - 1)]
    table = torch.where(column < count[:, None], table, -1).contiguous()
    row0 = [0]
    for t in rows:
        row0.append(row0[-1] + t)
    s = {"case": case, "table": table, "before": torch.tensor(before, dtype=torch.int32, device=dev),
         "row0": torch.tensor(row0, dtype=torch.int32, device=dev), "N": N, "T": max(rows)}
    if case["kind"] == "write":
        s["data"] = torch.zeros(1, pages, G, _record(dk), dtype=torch.uint8, device=dev)
        s["k"], s["v"] = _normal(g, N, G * dk), _normal(g, N, G * dk)
        return s
    s["data"] = _kept(g, 1, pages, G, dk)
    s["q"] = 1.5 * _normal(g, N, H * dk)
    left, right = _reach(case, before, rows)
    s["left"], s["right"] = (None if case[n] < 0 else case[n] for n in ("left", "right"))
    s["p"] = None
    if case["positions"]:
        s["p"], s["center"] = _normal(g, left + right + 1, H * dk), left
        s["u"], s["w"] = 0.1 * _normal(g, H * dk), 0.1 * _normal(g, H * dk)
    return s


# ------------------------------------------------------- the plain forms --

def _values(record, dk):
    """The keys and values that records [..., bytes] stand for: two of [..., 64, dk]."""
    byte = torch.arange(256, device=record.device)
    half = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=record.device)
    pair = torch.stack([half[byte & 15], half[byte >> 4]], -1)
    lead, ns = record.shape[:-1], dk // 32
    k = pair[record[..., :PAGE * dk // 2].long()].reshape(*lead, PAGE, dk)
    v = pair[record[..., PAGE * dk // 2:PAGE * dk].long()]      # [c // 32][w][c % 16][c // 16 % 2][g][h][r // 2][r % 2]
    n = len(lead)
    v = v.reshape(*lead, ns, 4, 16, 2, 2, 2, 2, 2)
    v = v.permute(*range(n), n + 4, n + 5, n + 1, n + 6, n + 7, n, n + 3, n + 2).reshape(*lead, PAGE, dk)
    d = record[..., PAGE * dk:].contiguous().view(torch.bfloat16).float()
    return k * d[..., :PAGE, None], v * d[..., PAGE:, None]


def _rounded(x, dk):
    """The values that x's heads of dk are kept as."""
    a = x.reshape(x.shape[0], -1, dk)
    top = a.abs().amax(-1, keepdim=True)
    fine = (top >= 2.0 ** -121) & (top < 2.0 ** 127)
    top = torch.where(fine, top, 1.0)
    d = (top / 6).view(torch.int32) & -65536        # a bfloat16 no more than a step from the scale; the least that holds
    d = torch.where(6 * d.view(torch.float32) >= top, d - 65536, d)
    d = torch.where(6 * d.view(torch.float32) >= top, d, d + 65536).view(torch.float32)
    code = sum(((a.abs() >= t * d) if up else (a.abs() > t * d)).int() for t, up in HALFWAY)
    value = torch.tensor(LEVELS, device=x.device)[code.long()] * d
    return torch.where(fine, torch.where(a < 0, -value, value), 0.0).reshape(x.shape)


def _plain_attend(s):
    case = s["case"]
    H, G, dk, B, T = case["H"], case["G"], case["dk"], case["B"], s["T"]
    dev, before, row0 = s["q"].device, s["before"].long(), s["row0"].long()
    count = row0[1:] - row0[:-1]
    record = s["data"][0][s["table"].long().clamp_min(0)]               # [B, held, G, bytes]
    k, v = _values(record, dk)
    K = record.shape[1] * PAGE
    k = k.permute(0, 2, 1, 3, 4).reshape(B, G, K, dk)
    v = v.permute(0, 2, 1, 3, 4).reshape(B, G, K, dk)
    i = torch.arange(T, device=dev)
    at = (row0[:-1, None] + i).clamp_max(s["N"] - 1)
    q = s["q"].reshape(s["N"], G, H // G, dk)[at]                       # [B, T, G, H / G, dk]
    content, place = (q, None) if s["p"] is None else (q + s["u"].reshape(G, -1, dk), q + s["w"].reshape(G, -1, dk))
    content = content.permute(0, 2, 3, 1, 4).reshape(B, G, H // G * T, dk)
    score = (content @ k.transpose(-1, -2)).reshape(B, H, T, K)
    j, pos = torch.arange(K, device=dev), before[:, None] + i
    if s["p"] is not None:
        p = s["p"].reshape(-1, H, dk).permute(1, 2, 0)                  # [H, dk, P]
        place = place.reshape(B * T, H, dk).transpose(0, 1)
        place = (place @ p).reshape(H, B, T, -1).transpose(0, 1)
        m = (s["center"] - pos[..., None] + j).clamp(0, p.shape[-1] - 1)
        score = score + torch.gather(place, 3, m[:, None].expand(B, H, T, K))
    score = score / math.sqrt(dk)
    seen = (j < (before + count)[:, None, None]) & (s["table"] >= 0).repeat_interleave(PAGE, 1)[:, None]
    seen = seen.expand(B, T, K)
    if s["left"] is not None:
        seen = seen & (j >= pos[..., None] - s["left"])
    if s["right"] is not None:
        seen = seen & (j <= pos[..., None] + s["right"])
    score = torch.where(seen[:, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    o = (e.reshape(B, G, H // G * T, K) @ v).reshape(B, H, T, dk) / torch.where(total > 0, total, 1.0)
    o = o.transpose(1, 2).reshape(B, T, H * dk)
    return o[(i < count[:, None])]


# ------------------------------------------------------------------ runs --

def _handles(s):
    """What a program keeps between steps: the cache, the streams' descriptor, the workspace and the outputs."""
    import libpktito_amd as pk
    case, data = s["case"], s["data"]
    s["cache"] = pk.DeviceCache(data, *data.shape[:3], case["dk"])
    if case["kind"] != "move":
        s["streams"] = pk.CacheStreams(s["table"], s["before"], s["row0"], s["N"], s["T"])
    if case["kind"] == "write":
        s["ko"], s["vo"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    if case["kind"] == "attend":
        s["at"] = None if s["p"] is None else (s["p"], s["center"], s["u"], s["w"])
        need = s["cache"].attention_workspace(s["streams"], case["H"], s["at"] is not None, s["left"], s["right"])
        s["ws"] = torch.empty(need, dtype=torch.uint8, device=data.device)
        s["o"] = torch.empty_like(s["q"])


def run(state):
    s, case = state, state["case"]
    kind = case["kind"]
    if own:
        if "cache" not in s:
            _handles(s)
        if kind == "write":     # the chunk into the cache, and what it keeps of it
            s["cache"].append(0, s["k"], s["v"], s["streams"])
            s["cache"].read(0, s["ko"], s["vo"], s["streams"])
            return [s["ko"], s["vo"]]
        if kind == "move":
            s["cache"].move(s["pairs"], s["table"])
            return [s["data"]] if s["table"] is None else [s["data"], s["table"]]
        s["cache"].attention(s["o"], 0, s["q"], s["streams"], case["H"], s["ws"], s["at"], s["left"], s["right"])
        return s["o"]
    if kind == "write":
        return [_rounded(s["k"], case["dk"]), _rounded(s["v"], case["dk"])]
    if kind == "move":
        src, dst = torch.tensor(s["pairs"], device=s["data"].device).T
        words = s["data"].view(torch.int64)
        words[:, dst] = words[:, src]
        if s["table"] is None:
            return [s["data"]]
        to = torch.arange(case["pages"], device=src.device, dtype=torch.int32)
        to[src] = dst.int()
        s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp_min(0).long()], s["table"]))
        return [s["data"], s["table"]]
    return _plain_attend(s)


def work(case):
    G, dk = case["G"], case["dk"]
    if case["kind"] == "move":
        return {"bytes": 2 * case["pairs"] * case["layers"] * G * _record(dk) + 8 * case["B"] * case["columns"], "flops": 0}
    before, rows = _lengths(case)
    N, H = sum(rows), case["H"]
    if case["kind"] == "write":     # read, kept, and read back
        return {"bytes": 2 * N * G * (4 * dk + (dk // 2 + 2) + 4 * dk), "flops": 0}
    left, right = _reach(case, before, rows)
    pairs = frames = 0
    for b, t in zip(before, rows):
        frames += b + t - max(0, b - left)
        pairs += sum(min(b + t - 1, b + i + right) - max(0, b + i - left) + 1 for i in range(t))
    places = left + right + 1 if case["positions"] else 0
    return {"bytes": frames * G * (dk + 4) + 4 * places * H * dk + 8 * N * H * dk,
            "flops": 2 * pairs * H * dk * (3 if case["positions"] else 2)}


# ----------------------------------------------------------- 64-bit values --

def _exact_values(head, frames, dk):
    """Keys and values of `frames` of one head, by their places: head [held, bytes] in frame order."""
    f = torch.arange(frames, device=head.device)
    level = torch.tensor(LEVELS, dtype=torch.float64, device=head.device)
    c = torch.arange(dk, device=head.device)

    def taken(at, high):
        b = torch.gather(head, 1, at.reshape(head.shape[0], -1)).long().reshape(-1, dk)
        h = (b >> (4 * high)) & 15
        return torch.where(h >= 8, -1.0, 1.0).double() * level[h & 7]

    f = torch.arange(head.shape[0] * PAGE, device=head.device) % PAGE
    k = taken(f[:, None] * (dk // 2) + c // 2, c % 2)
    g, h, w, r = f // 32, f // 16 % 2, f // 4 % 4, f % 4
    at = 1024 * (c // 32) + 16 * (c % 16) + 8 * (c // 16 % 2) + (256 * w + 4 * g + 2 * h + r // 2)[:, None]
    v = taken(PAGE * dk // 2 + at, (r % 2)[:, None])
    d = head[:, PAGE * dk:].contiguous().view(torch.bfloat16).double()
    return (k * d[:, :PAGE].reshape(-1, 1))[:frames], (v * d[:, PAGE:].reshape(-1, 1))[:frames]


def _exact_rounded(x, dk):
    a = x.double().reshape(-1, dk)
    top = a.abs().amax(1)
    whole = torch.floor(torch.log2(top / 6)) - 7        # a bfloat16's last place
    place = torch.exp2(whole)
    d = torch.ceil(top / 6 / place) * place
    d = torch.where(6 * (d - place) >= top, d - place, d)[:, None]
    level = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    even = torch.tensor([0, 1, 0, 1, 0, 1, 0, 1], dtype=torch.float64, device=x.device)
    off = (a.abs()[..., None] / d[..., None] - level).abs()
    near = off.amin(-1, keepdim=True)
    code = torch.where(off == near, even, 2.0).argmin(-1)
    return (torch.sign(a) * level[code] * d).reshape(x.shape)


def exact(case, seed):
    if case["kind"] == "move":
        return None
    s = prepare(case, seed)
    dk, G, H = case["dk"], case["G"], case["H"]
    if case["kind"] == "write":
        return [torch.cat([_exact_rounded(part, dk) for part in s[n].split(2048)]) for n in ("k", "v")]
    before, rows = _lengths(case)
    out = torch.zeros(s["N"], H * dk, dtype=torch.float64, device=s["q"].device)
    r0 = 0
    for b, (len_b, t) in enumerate(zip(before, rows)):
        total = len_b + t
        held = -(-total // PAGE)
        record = s["data"][0, s["table"][b, :held].long()]
        pos, j = len_b + torch.arange(t, device=out.device)[:, None], torch.arange(total, device=out.device)
        seen = torch.ones(t, total, dtype=torch.bool, device=out.device)
        if case["left"] >= 0:
            seen &= pos - j <= case["left"]
        if case["right"] >= 0:
            seen &= j - pos <= case["right"]
        for kept in range(G):
            k, v = _exact_values(record[:, kept].contiguous(), total, dk)
            for h in range(kept * (H // G), (kept + 1) * (H // G)):
                c = slice(h * dk, (h + 1) * dk)
                q = s["q"][r0:r0 + t, c].double()
                if s["p"] is None:
                    score = q @ k.T.contiguous()
                else:
                    score = (q + s["u"][c].double()) @ k.T.contiguous()
                    place = (q + s["w"][c].double()) @ s["p"][:, c].double().T.contiguous()
                    m = s["center"] - pos + j
                    score += torch.gather(place, 1, m.clamp(0, place.shape[1] - 1))
                score = torch.where(seen, score / math.sqrt(dk), -math.inf)
                out[r0:r0 + t, c] = torch.softmax(score, 1) @ v
        r0 += t
    return out
