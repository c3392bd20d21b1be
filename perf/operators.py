"""Operators over the paged KV cache, as cases that can be timed and checked
against their plain forms.

A case is a dict of plain values.  Its "kind":

    write    new rows quantised into the cache's pages and read back from them
             (what the cache rounds them to)
    read     whole sequences gathered from their pages
    attend   attention of each sequence's newest rows over its pages; with
             "window", over the last `window` positions and the first `sinks`

The cache holds f32, f16 (a power-of-two scale per position and head) or i8
codes (a scale per position and head).  `seqs` sequences hold up to `held`
positions and get up to `rows` new ones; "spread" says how both vary between
them ("same", "ragged", or "mixed": most get one row, some a chunk).
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
F32_TINY = 2.0 ** -126


# ---- the cases ---------------------------------------------------------------

def listed():
    big = {"n_head": 32, "n_kv_head": 8, "head_dim": 128}
    small = {"n_head": 14, "n_kv_head": 2, "head_dim": 64}
    return [
        # Prompts of several conversations written together, in a serving pass
        # that reads them in chunks: the widest writes.
        dict(big, name="write_i8_prompts", kind="write", precision="i8", page=64, seqs=5, held=1500, rows=1400,
             spread="ragged", window=0, sinks=0),
        # A token of each of 48 conversations: the write of every decode step,
        # a call of a few microseconds per layer.
        dict(small, name="write_f16_tokens", kind="write", precision="f16", page=32, seqs=48, held=1000, rows=1,
             spread="ragged", window=0, sinks=0),
        # A long document's cache read back whole: to move or park it.
        dict(big, name="read_i8_long", kind="read", precision="i8", page=64, seqs=1, held=20001, rows=0,
             spread="same", window=0, sinks=0),
        # A few short conversations read back in full precision.
        dict(small, name="read_f32_short", kind="read", precision="f32", page=32, seqs=3, held=301, rows=0,
             spread="ragged", window=0, sinks=0),
        # 64 conversations decoded together at an 8B decoder's geometry.
        dict(big, name="decode_i8_64seq", kind="attend", precision="i8", page=64, seqs=64, held=4000, rows=1,
             spread="ragged", window=0, sinks=0),
        # One conversation over a long document, a half-billion decoder.
        dict(small, name="decode_f16_long", kind="attend", precision="f16", page=128, seqs=1, held=32767, rows=1,
             spread="same", window=0, sinks=0),
        # A prompt's pass of 512 tokens behind 8000 held ones.
        dict(big, name="chunk_f16", kind="attend", precision="f16", page=64, seqs=1, held=8000, rows=512,
             spread="same", window=0, sinks=0),
        # A whole prompt of no even length, the cache kept in f32.
        dict(small, name="prompt_f32", kind="attend", precision="f32", page=32, seqs=1, held=0, rows=1001,
             spread="same", window=0, sinks=0),
        # Decoding conversations and two prompts' chunks in one call.
        {"name": "mixed_i8", "kind": "attend", "n_head": 12, "n_kv_head": 2, "head_dim": 128, "precision": "i8",
         "page": 64, "seqs": 17, "held": 3001, "rows": 200, "spread": "mixed", "window": 0, "sinks": 0},
        # Long conversations decoded through a window: the pages in between
        # are not read.
        dict(big, name="window_decode_i8", kind="attend", precision="i8", page=64, seqs=32, held=16000, rows=1,
             spread="ragged", window=1024, sinks=4),
        # A long prompt through a window, the largest call.
        dict(big, name="window_prompt_f16", kind="attend", precision="f16", page=64, seqs=1, held=0, rows=6000,
             spread="same", window=1024, sinks=4),
        # A few drafted tokens checked at once, as many KV heads as heads.
        {"name": "window_draft_f32", "kind": "attend", "n_head": 16, "n_kv_head": 16, "head_dim": 128,
         "precision": "f32", "page": 32, "seqs": 3, "held": 900, "rows": 5, "spread": "same", "window": 500,
         "sinks": 1},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of lo .. hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


GEOMETRIES = [(14, 2, 64), (32, 8, 128), (32, 8, 64), (16, 16, 128), (12, 2, 128), (32, 4, 64), (8, 1, 96)]


def draw(rng):
    while True:
        n_head, n_kv_head, head_dim = rng.choice(GEOMETRIES)
        c = {"kind": rng.choice(["write", "read", "attend", "attend", "attend", "attend"]), "n_head": n_head,
             "n_kv_head": n_kv_head, "head_dim": head_dim, "precision": rng.choice(["f32", "f16", "i8", "i8"]),
             "page": rng.choice([32, 64, 128]), "seqs": _log(rng, 1, 64), "held": _log(rng, 1, 20000) - 1,
             "rows": rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 2000)]),
             "spread": rng.choice(["same", "ragged", "mixed"]), "window": 0, "sinks": 0}
        if c["kind"] == "read":
            c["held"], c["rows"] = c["held"] + 1, 0
        if c["kind"] == "attend" and rng.random() < 0.4:
            c["window"], c["sinks"] = _log(rng, 16, 4000), rng.choice([0, 1, 4, 40])
        length = c["held"] + c["rows"]
        cells = c["seqs"] * length * n_kv_head * head_dim
        if cells <= 64 * 4000 * 1024 and c["seqs"] * max(c["rows"], 1) * length * n_head <= 400_000_000:
            return c


def layout(case):
    """Per sequence the positions it holds and how many of them are new, from
    the case alone."""
    rng = random.Random(repr([case[k] for k in sorted(case) if k != "name"]))
    lens, news = [], []
    for s in range(case["seqs"]):
        held, rows = case["held"], case["rows"]
        if s and case["spread"] != "same":
            held = rng.randint(held // 3, held)
            if case["spread"] == "ragged" and rows:
                rows = rng.randint(max(1, rows // 3), rows)
            elif case["spread"] == "mixed" and rows:
                rows = rng.randint(1, rows) if s == case["seqs"] // 2 else 1
        new = rows if case["kind"] != "read" else max(held, 1)
        lens.append(held + rows if case["kind"] != "read" else max(held, 1))
        news.append(new)
    return lens, news


ES = {"f32": 4, "f16": 2, "i8": 1}


def visible(case, p):
    """How many positions a row at position p sees."""
    w, sinks = case["window"], case["sinks"]
    if not w or p + 1 <= w:
        return p + 1
    return w + min(sinks, p + 1 - w)


def work(case):
    lens, news = layout(case)
    H, kv, hd, es = case["n_head"], case["n_kv_head"], case["head_dim"], ES[case["precision"]]
    stored = kv * (2 * hd * es + 8)
    f32 = 2 * kv * hd * 4
    rows = sum(news)
    tables = sum(4 * -(-n // case["page"]) + 8 for n in lens)
    if case["kind"] == "write":
        return {"bytes": rows * (2 * f32 + 2 * stored) + tables, "flops": 0}
    if case["kind"] == "read":
        return {"bytes": rows * (f32 + stored) + tables, "flops": 0}
    held, pairs = 0, 0
    for n, m in zip(lens, news):
        w, sinks = case["window"], case["sinks"]
        first = max(0, n - m - w + 1) if w else 0  # of the window of the first new row
        held += n - first + min(sinks if w else 0, first)
        pairs += sum(visible(case, p) for p in range(n - m, n))
    return {"bytes": held * stored + 2 * rows * H * hd * 4 + tables, "flops": 4 * hd * H * pairs}


# ---- inputs ------------------------------------------------------------------

def data(case, seed):
    """Keys and values of every position of every sequence, one sequence after
    the other, [positions][heads][dims], and the new rows' queries.  Some
    channels of the keys are several times the others; the scores spread as
    trained heads' do (a standard deviation of about 2)."""
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 4242)
    lens, news = layout(case)
    total, rows = sum(lens), sum(news)
    H, kv, hd = case["n_head"], case["n_kv_head"], case["head_dim"]
    channels = torch.exp(0.5 * torch.randn(kv, hd, device=DEV, generator=g))
    k = torch.randn(total, kv, hd, device=DEV, generator=g) * channels
    v = torch.randn(total, kv, hd, device=DEV, generator=g)
    q = torch.randn(rows, H, hd, device=DEV, generator=g) if case["kind"] == "attend" else None
    if q is not None:
        q = q * (2.0 / channels.square().mean().sqrt())
    return lens, news, k, v, q


def quantised(case, x):
    """What the cache holds for x [..., dims]: codes and a scale a row."""
    amax = x.abs().amax(-1, keepdim=True).double()
    if case["precision"] == "i8":
        scale = (amax / 127.0).float()
        scale = torch.where(scale < F32_TINY, torch.zeros_like(scale), scale)
        inv = torch.where(scale > 0, (1.0 / scale.double()).float(), torch.zeros_like(scale))
        t = (x.double() * inv.double()).float().double()  # the product, rounded to 32 bits
        code = torch.sign(t) * torch.floor(t.abs() + 0.5)
        return code.clamp(-127, 127).to(torch.int8), scale
    if case["precision"] == "f16":
        scale = torch.ldexp(torch.ones_like(amax), (torch.frexp(amax)[1] - 15).clamp(min=-126))
        return (x.double() / scale).half(), scale.float()
    return x, torch.ones_like(amax).float()


def prepare(case, seed):
    lens, news, k, v, q = data(case, seed)
    P, S = case["page"], case["seqs"]
    counts = [-(-n // P) for n in lens]
    # the pages of a pool in use for a while: in no order, a few of them free
    g = torch.Generator().manual_seed(int(seed) + 99)
    n_pages = sum(counts) + 3
    order = torch.randperm(n_pages, generator=g)
    table = torch.full((S, max(counts)), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c]
        at += c
    cum = lambda v: torch.cumsum(torch.tensor([0] + v), 0)  # noqa: E731
    t_len, t_new = torch.tensor(lens), torch.tensor(news)
    st = {"case": case, "pages": table.to(DEV), "len": t_len.to(torch.int32).to(DEV), "q": q, "max_len": max(lens),
          "max_new": max(news), "row_start": cum(news).to(torch.int32).to(DEV), "new": t_new.to(torch.int32).to(DEV)}
    new = torch.cat([torch.arange(e - m, e) for e, m in zip(cum(lens)[1:].tolist(), news)]).to(DEV)
    st["k"], st["v"] = k[new].contiguous(), v[new].contiguous()
    if case["kind"] == "write":  # the new rows are not in the cache yet
        k[new], v[new] = 0.0, 0.0
    kv, hd = case["n_kv_head"], case["head_dim"]
    outs = 1 if case["kind"] == "attend" else 2
    st["out"] = [torch.empty(len(new), case["n_head"] if outs == 1 else kv, hd, device=DEV) for _ in range(outs)]
    # every position's place in the pool, sequence after sequence
    pos = torch.cat([torch.arange(n) for n in lens])
    seq = torch.repeat_interleave(torch.arange(S), t_len)
    slot = (table[seq, pos // P].long() * P + pos % P).to(DEV)
    if own:
        import kvad_amd as K

        ctx = _context()
        st["cache"] = K.PagedCache(ctx, 1, kv, hd, n_pages, page_size=P,
                                   precision={"f32": K.F32, "f16": K.F16, "i8": K.I8}[case["precision"]])
        # row_start is left out where every sequence has as many new rows
        same = len(set(news)) == 1
        st["batch"] = K.Batch(S, len(new), st["len"].data_ptr(), st["pages"].data_ptr(), table.shape[1],
                              row_start=None if same else st["row_start"].data_ptr(), max_len=max(lens))
        starts = cum(lens).to(torch.int32).to(DEV)
        whole = K.Batch(S, sum(lens), st["len"].data_ptr(), st["pages"].data_ptr(), table.shape[1],
                        row_start=starts.data_ptr(), max_len=max(lens))
        torch.cuda.synchronize()
        st["cache"].push_dev(0, whole, k.data_ptr(), v.data_ptr())
        ctx.synchronize()
    else:
        for name, x in (("k", k), ("v", v)):
            codes, scale = quantised(case, x)
            pool = torch.zeros(n_pages * P, kv, hd, dtype=codes.dtype, device=DEV)
            scales = torch.zeros(n_pages * P, kv, 1, device=DEV)
            pool[slot], scales[slot] = codes, scale
            st[name + "_pool"], st[name + "_scale"] = pool, scales
    return st


_ctx = None


def _context():
    """One context for the process: a device and a stream."""
    global _ctx
    if _ctx is None:
        import kvad_amd as K

        _ctx = K.Context(0)
    return _ctx


# ---- the operators -----------------------------------------------------------

def run(st):
    case = st["case"]
    if own:
        cache, batch, out = st["cache"], st["batch"], st["out"]
        if case["kind"] == "attend":
            cache.attend_dev(0, batch, case["n_head"], st["q"].data_ptr(), out[0].data_ptr(), window=case["window"],
                             sinks=case["sinks"])
            return out[0]
        if case["kind"] == "write":
            cache.push_dev(0, batch, st["k"].data_ptr(), st["v"].data_ptr())
        cache.read_dev(0, batch, out[0].data_ptr(), out[1].data_ptr())
        return {"k": out[0], "v": out[1]}
    if case["kind"] == "attend":
        return plain_attend(st)
    slots = row_slots(st)
    if case["kind"] == "write":
        for name in ("k", "v"):
            codes, scale = quantised(case, st[name])
            st[name + "_pool"][slots], st[name + "_scale"][slots] = codes, scale
    return {name: held(st, name, slots) for name in ("k", "v")}


def row_places(st):
    """Each new row's sequence and position."""
    n_rows, rs = st["k"].shape[0], st["row_start"].long()
    row = torch.arange(n_rows, device=DEV)
    seq = torch.searchsorted(rs, row, right=True) - 1
    return seq, (st["len"] - st["new"]).long()[seq] + row - rs[seq]


def row_slots(st):
    seq, pos = row_places(st)
    P = st["case"]["page"]
    return st["pages"].long()[seq, pos // P] * P + pos % P


def held(st, name, slots):
    return st[name + "_pool"][slots].float() * st[name + "_scale"][slots]


def plain_attend(st):
    """Sequences padded to the longest, scores of every new row against the
    positions that some new row sees, a softmax over the visible ones."""
    case, P = st["case"], st["case"]["page"]
    S, L, R = case["seqs"], st["max_len"], st["max_new"]
    H, kv, hd = case["n_head"], case["n_kv_head"], case["head_dim"]
    G, window, sinks = H // kv, case["window"], min(case["sinks"], L)
    first = (st["len"] - st["new"]).long()[:, None]                         # [S, 1]: a sequence's first new position
    # the windows' positions, behind them the sinks in front of them
    start = (first - window + 1).clamp(min=0) if window else torch.zeros_like(first)
    t = start + torch.arange(min(L, window + R - 1) if window else L, device=DEV)
    keep = torch.ones_like(t, dtype=torch.bool)
    if window and sinks:
        front = torch.arange(sinks, device=DEV).expand(S, sinks)
        t, keep = torch.cat([t, front], 1), torch.cat([keep, front < start], 1)
    at = t.clamp(max=L - 1)
    slots = st["pages"].long().gather(1, at // P).clamp(min=0) * P + at % P  # [S, positions]
    keys = held(st, "k", slots).permute(0, 2, 3, 1).contiguous()             # [S, kv, hd, positions]
    values = held(st, "v", slots).permute(0, 2, 1, 3).contiguous()           # [S, kv, positions, hd]
    j = torch.arange(R, device=DEV)
    rows = (st["row_start"].long()[:-1, None] + j).clamp(max=st["k"].shape[0] - 1)
    q = st["q"][rows].reshape(S, R, kv, G, hd).permute(0, 2, 1, 3, 4).reshape(S, kv, R * G, hd)
    scores = torch.matmul(q, keys).reshape(S, kv, R, G, -1) * (1.0 / math.sqrt(hd))
    pos = (first + j)[:, :, None]                                            # [S, R, 1]
    t = t[:, None, :]
    seen = keep[:, None, :] & (t <= pos)
    if window:
        seen = seen & ((t > pos - window) | (t < sinks))
    scores = scores.masked_fill(~seen[:, None, :, None, :], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e.reshape(S, kv, R * G, -1), values).reshape(S, kv, R, G, hd)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 2, 1, 3, 4).reshape(S * R, H, hd)
    seq, place = row_places(st)
    return out[seq * R + place - first[seq, 0]]


# ---- the definition in 64 bits -------------------------------------------------

def rounded(case, x):
    """The values the cache holds for rows x, from the definition."""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    if case["precision"] == "f32":
        return x
    if case["precision"] == "f16":
        # eleven significant bits under the row's power of two, in steps of
        # at least 2^-24 of it
        unit = torch.exp2(torch.floor(torch.log2(amax.clamp(min=1e-300))) + 1 - 15).clamp(min=2.0 ** -126)
        y = x / unit
        step = torch.exp2((torch.frexp(y)[1] - 11).clamp(min=-24).double())
        return torch.round(y / step) * step * unit
    scale = (amax / 127.0).to(torch.float32).double()
    ok = scale >= F32_TINY
    inv = (1.0 / torch.where(ok, scale, torch.ones_like(scale))).to(torch.float32).double()
    y = (x * inv).to(torch.float32).double()
    code = torch.where(y < 0, torch.ceil(y - 0.5), torch.floor(y + 0.5)).clamp(-127, 127)
    return torch.where(ok, code * scale, torch.zeros_like(code))


def exact(case, seed):
    lens, news, k, v, q = data(case, seed)
    ends = torch.cumsum(torch.tensor(lens), 0).tolist()
    if case["kind"] != "attend":
        pick = lambda x: torch.cat([rounded(case, x[e - m:e]) for e, m in zip(ends, news)])  # noqa: E731
        return {"k": pick(k), "v": pick(v)}
    H, kv, hd = case["n_head"], case["n_kv_head"], case["head_dim"]
    out = torch.zeros(sum(news), H, hd, dtype=torch.float64, device=DEV)
    row = 0
    for n, m, e in zip(lens, news, ends):
        ks, vs = rounded(case, k[e - n:e]), rounded(case, v[e - n:e])
        i = torch.arange(n - m, n, device=DEV)[:, None]
        t = torch.arange(n, device=DEV)[None, :]
        hidden = t > i
        if case["window"]:
            hidden = hidden | ((i - t >= case["window"]) & (t >= case["sinks"]))
        for h in range(H):
            kh, vh = ks[:, h * kv // H].contiguous(), vs[:, h * kv // H].contiguous()
            s = q[row:row + m, h].double() @ kh.T.contiguous() / math.sqrt(hd)
            s.masked_fill_(hidden, float("-inf"))
            out[row:row + m, h] = torch.softmax(s, -1) @ vh
        row += m
    return out
