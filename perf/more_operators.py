"""More operators of a serving step over the paged KV cache, as cases that can
be timed and checked against their plain forms.

A case is a dict of plain values.  Its "kind":

    write    new rows quantised into a cache of 4-bit rows and read back from it
    attend   attention of each sequence's newest rows over such a cache; with
             "window", over the last `window` positions and the first `sinks`
    pages    pages of sequences given back, and pages, positions and slots
             given to each sequence's new rows
    rope     rows rotated at positions of their own: queries and keys in one
             row of a joint projection
    norm     the end of a block: y (normed, with "post") times a gate and a
             scale added to the residual x, and that normed for the next

The 4-bit rows: 32 dims of a head's row share a power of two 2^e, with
3.5 2^e <= amax < 7 2^e, and hold the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6
times it, with a sign.  `seqs` sequences hold up to `held` positions and get up
to `rows` new ones; "spread" says how both vary between them ("same", "ragged",
or "mixed": most get one row, some a chunk).
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
GROUP = 32


# ---- the cases ---------------------------------------------------------------

def listed():
    big = {"n_head": 32, "n_kv_head": 8, "head_dim": 128}
    small = {"n_head": 14, "n_kv_head": 2, "head_dim": 64}
    none = {"window": 0, "sinks": 0}
    return [
        # A token of each of 48 conversations: the write of every decode step,
        # a call of a few microseconds per layer.
        dict(small, **none, name="write_tokens", kind="write", page=32, seqs=48, held=1000, rows=1, spread="ragged"),
        # Prompts of several conversations written together, in a serving pass
        # that reads them in chunks.
        dict(big, **none, name="write_prompts", kind="write", page=64, seqs=5, held=1500, rows=1400, spread="ragged"),
        # 64 conversations decoded together at an 8B decoder's geometry.
        dict(big, **none, name="decode_64seq", kind="attend", page=64, seqs=64, held=4000, rows=1, spread="ragged"),
        # One conversation over a long document, a half-billion decoder.
        dict(small, **none, name="decode_long", kind="attend", page=128, seqs=1, held=32767, rows=1, spread="same"),
        # A prompt's pass of 512 tokens behind 8000 held ones, the largest call.
        dict(big, **none, name="chunk", kind="attend", page=64, seqs=1, held=8000, rows=512, spread="same"),
        # Decoding conversations and a prompt's chunk in one call, through a window.
        {"name": "window_mixed", "kind": "attend", "n_head": 12, "n_kv_head": 2, "head_dim": 128, "page": 64,
         "seqs": 17, "held": 3001, "rows": 200, "spread": "mixed", "window": 1024, "sinks": 4},
        # A decode step of 64 conversations: last step's drafted token is taken
        # back and another given its place.
        {"name": "pages_tokens", "kind": "pages", "page": 64, "seqs": 64, "held": 4000, "rows": 1, "spread": "ragged"},
        # Conversations that ended give their pages back and new prompts of up
        # to 6000 tokens take them, a pool of small pages.
        {"name": "pages_prompts", "kind": "pages", "page": 32, "seqs": 33, "held": 0, "rows": 6000, "spread": "ragged"},
        # The queries and keys of a decode step's tokens, in the joint row of a projection.
        dict(small, name="rope_tokens", kind="rope", page=32, seqs=48, held=1000, rows=1, spread="ragged",
             interleaved=False),
        # The same of prompts read together at an 8B decoder's geometry, pairs side by side.
        dict(big, name="rope_prompts", kind="rope", page=64, seqs=5, held=1500, rows=1400, spread="ragged",
             interleaved=True),
        # Between two sub-blocks of a decode step: the residual add and the next norm.
        {"name": "norm_tokens", "kind": "norm", "m": 48, "n": 896, "post": False, "gate": "none", "pre": True},
        # A prompt's pass at an 8B decoder's width, norms on both sides and a gate for each token.
        {"name": "norm_prompts", "kind": "norm", "m": 2050, "n": 4096, "post": True, "gate": "each", "pre": True},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of lo .. hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


GEOMETRIES = [(14, 2, 64), (32, 8, 128), (32, 8, 64), (16, 16, 128), (12, 2, 128), (32, 4, 64), (8, 1, 96), (8, 4, 256),
              (10, 5, 80)]


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "attend", "attend", "pages", "rope", "norm"])
    while True:
        if kind == "norm":
            c = {"kind": kind, "m": _log(rng, 1, 8000), "n": rng.choice([896, 1536, 2048, 4096, _log(rng, 33, 9000)]),
                 "post": rng.random() < 0.5, "gate": rng.choice(["none", "all", "each"]), "pre": rng.random() < 0.8}
            if c["m"] * c["n"] <= 2050 * 4096:
                return c
            continue
        n_head, n_kv_head, head_dim = rng.choice(GEOMETRIES)
        c = {"kind": kind, "page": rng.choice([32, 64, 128]), "seqs": _log(rng, 1, 64), "held": _log(rng, 1, 20000) - 1,
             "rows": rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 2000)]),
             "spread": rng.choice(["same", "ragged", "mixed"])}
        if kind == "pages":
            c["seqs"] = _log(rng, 1, 1000)
            if c["seqs"] * (c["held"] + c["rows"]) <= 4_000_000 and c["seqs"] * c["rows"] <= 33 * 6000:
                return c
            continue
        c.update(n_head=n_head, n_kv_head=n_kv_head, head_dim=head_dim)
        if kind == "rope":
            c["interleaved"] = rng.random() < 0.5
            if c["seqs"] * c["rows"] * (n_head + n_kv_head) * head_dim <= 7000 * 5120:
                return c
            continue
        c["window"], c["sinks"] = 0, 0
        if kind == "attend" and rng.random() < 0.4:
            c["window"], c["sinks"] = _log(rng, 16, 4000), rng.choice([0, 1, 4, 40])
        length = c["held"] + c["rows"]
        cells = c["seqs"] * length * n_kv_head * head_dim
        if kind == "write" and c["seqs"] * c["rows"] * n_kv_head * head_dim > 7000 * 1024:
            continue
        if cells <= 64 * 4000 * 1024 and c["seqs"] * c["rows"] * length * n_head * head_dim <= 512 * 8512 * 32 * 128:
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
            if case["spread"] == "ragged":
                rows = rng.randint(max(1, rows // 3), rows)
            else:
                rows = rng.randint(1, rows) if s == case["seqs"] // 2 else 1
        lens.append(held + rows)
        news.append(rows)
    return lens, news


def visible(case, p):
    """How many positions a row at position p sees."""
    w, sinks = case["window"], case["sinks"]
    if not w or p + 1 <= w:
        return p + 1
    return w + min(sinks, p + 1 - w)


def work(case):
    if case["kind"] == "norm":
        m, n = case["m"], case["n"]
        gate = {"none": 0, "all": n, "each": m * n}[case["gate"]]
        weights = n * (case["post"] + case["pre"])
        return {"bytes": 4 * (m * n * (3 + case["pre"]) + gate + weights),
                "flops": m * n * (2 + 4 * case["post"] + 4 * case["pre"] + (case["gate"] != "none"))}
    lens, news = layout(case)
    rows, S, P = sum(news), case["seqs"], case["page"]
    if case["kind"] == "pages":
        given = sum(-(-n // P) - -(-(n - m) // P) for n, m in zip(lens, news))
        # keep, rows and lengths in, lengths and first rows out; a page leaves
        # the table for the stack and comes back; a position and a slot a row
        return {"bytes": 20 * S + 20 * given + 12 * rows, "flops": 0}
    H, kv, hd = case["n_head"], case["n_kv_head"], case["head_dim"]
    if case["kind"] == "rope":
        places = len(set().union(*[range(n - m, n) for n, m in zip(lens, news)]))
        return {"bytes": 8 * rows * (H + kv) * hd + 4 * places * hd + 4 * rows, "flops": 3 * rows * (H + kv) * hd}
    groups = -(-hd // GROUP)
    stored = 2 * kv * (hd / 2 + groups)
    tables = sum(4 * -(-n // P) + 8 for n in lens)
    if case["kind"] == "write":
        return {"bytes": int(rows * (16 * kv * hd + 2 * stored)) + tables, "flops": 0}
    held, pairs = 0, 0
    for n, m in zip(lens, news):
        w, sinks = case["window"], case["sinks"]
        first = max(0, n - m - w + 1) if w else 0  # of the window of the first new row
        held += n - first + min(sinks if w else 0, first)
        pairs += sum(visible(case, p) for p in range(n - m, n))
    return {"bytes": int(held * stored) + 2 * rows * H * hd * 4 + tables, "flops": 4 * hd * H * pairs}


# ---- inputs ------------------------------------------------------------------

def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 777)
    return g


def data(case, seed):
    """Keys and values of every position of every sequence, one sequence after
    the other, [positions][heads][dims], and the new rows' queries.  Some
    channels of the keys are several times the others; the scores spread as
    trained heads' do (a standard deviation of about 2)."""
    g = generator(seed)
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


def tables(case, seed):
    """Page tables of a pool in use for a while, in no order: the sequences'
    rows, the free pages as a stack, and how many those are."""
    lens, _ = layout(case)
    P = case["page"]
    counts = [-(-n // P) for n in lens]
    g = torch.Generator().manual_seed(int(seed) + 99)
    n_pages = sum(counts) + 5
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    width = max(counts)
    column = torch.arange(width)
    table = torch.full((case["seqs"], width), -1, dtype=torch.int32)
    table[column[None, :] < torch.tensor(counts)[:, None]] = order[:sum(counts)]
    free = torch.full((n_pages,), -1, dtype=torch.int32)
    free[:5] = order[sum(counts):]
    return table, free, 5


def norm_data(case, seed):
    g = generator(seed)
    m, n = case["m"], case["n"]
    # a residual stream with a few large channels, and a block's output beside it
    big = 1.0 + 30.0 * (torch.rand(n, device=DEV, generator=g) < 0.01)
    x = torch.randn(m, n, device=DEV, generator=g) * big
    y = torch.randn(m, n, device=DEV, generator=g) * 0.3
    post = 1.0 + 0.2 * torch.randn(n, device=DEV, generator=g)
    pre = 1.0 + 0.2 * torch.randn(n, device=DEV, generator=g)
    gate = torch.sigmoid(torch.randn(m if case["gate"] == "each" else 1, n, device=DEV, generator=g))
    return {"x": x, "y": y, "post": post if case["post"] else None, "pre": pre if case["pre"] else None,
            "gate": None if case["gate"] == "none" else gate, "eps": 1e-6, "scale": 0.22}


def rope_data(case, seed):
    """Joint rows of queries, keys and values, their positions, and the
    rotation's tables."""
    g = generator(seed)
    lens, news = layout(case)
    H, kv, hd = case["n_head"], case["n_kv_head"], case["head_dim"]
    x = torch.randn(sum(news), (H + 2 * kv) * hd, device=DEV, generator=g)
    position = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, news)]).to(torch.int32).to(DEV)
    max_pos = max(lens)
    freq = 1e6 ** (-torch.arange(hd // 2, dtype=torch.float64, device=DEV) * 2.0 / hd)
    angle = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * freq
    return {"x": x, "position": position, "cos": torch.cos(angle).float(), "sin": torch.sin(angle).float()}


# E2M1's magnitudes; code 8 + i is minus code i
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantised(x):
    """What the cache holds for x [..., dims]: codes, padded to whole groups,
    and each group's exponent."""
    hd = x.shape[-1]
    groups = -(-hd // GROUP)
    x = torch.nn.functional.pad(x, (0, groups * GROUP - hd)).unflatten(-1, (groups, GROUP))
    amax = x.abs().amax(-1)
    # the exponent field, one more from 1.75 times a power of two on
    e = ((amax.view(torch.int32) + 0x200000) >> 23) - 129
    e = e.clamp(min=-128)
    e = torch.maximum(e, ((e.amax(-1, keepdim=True) - 12).clamp(min=-126) - 14))
    y = (x.double() * torch.exp2(-e.double())[..., None]).abs()
    # one up at each midpoint passed; those between an odd and an even code at the midpoint itself
    code = sum((y >= t if at else y > t).to(torch.uint8)
               for t, at in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)))
    code = code + 8 * (x < 0).to(torch.uint8)
    return code, e.to(torch.int16)


def packed(code):
    """Two codes a byte, the even dim's in the low half."""
    code = code.flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4


_ctx = None


def _context():
    """One context for the process: a device and a stream."""
    global _ctx
    if _ctx is None:
        import kvad_amd as K

        _ctx = K.Context(0)
    return _ctx


def prepare(case, seed):
    if case["kind"] == "norm":
        st = dict(norm_data(case, seed), case=case)
        st["x_out"], st["out"] = torch.empty_like(st["x"]), torch.empty_like(st["x"])
        if own:
            st["ctx"] = _context()
            torch.cuda.synchronize()
        return st
    if case["kind"] == "rope":
        st = dict(rope_data(case, seed), case=case)
        vectors = case["n_head"] + case["n_kv_head"]
        st["out"] = torch.empty(st["x"].shape[0], vectors, case["head_dim"], device=DEV)
        if own:
            st["ctx"] = _context()
            torch.cuda.synchronize()
        return st
    lens, news = layout(case)
    S, P = case["seqs"], case["page"]
    table, free, n_free = tables(case, seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    st = {"case": case, "pages": table.to(DEV), "len": i32(lens), "max_len": max(lens), "max_new": max(news),
          "new": i32(news), "row_start": i32([0] + list(torch.cumsum(torch.tensor(news), 0)))}
    if case["kind"] == "pages":
        n_pages = free.numel()
        st.update(free=free.to(DEV), n_free=i32([n_free]), keep=i32([n - m for n, m in zip(lens, news)]),
                  status=i32([0] * 4), position=i32([-1] * sum(news)),
                  slot=torch.full((sum(news),), -1, dtype=torch.int64, device=DEV))
        if own:
            import kvad_amd as K

            st["ctx"] = _context()
            st["table"] = K.PageTable(S, table.shape[1], P, n_pages, st["len"].data_ptr(), st["pages"].data_ptr(),
                                      st["row_start"].data_ptr(), st["free"].data_ptr(), st["n_free"].data_ptr(),
                                      st["status"].data_ptr())
            torch.cuda.synchronize()
        return st
    _, _, k, v, q = data(case, seed)
    kv, hd = case["n_kv_head"], case["head_dim"]
    cum = lambda v: torch.cumsum(torch.tensor([0] + v), 0)  # noqa: E731
    new = torch.cat([torch.arange(e - m, e) for e, m in zip(cum(lens)[1:].tolist(), news)]).to(DEV)
    st["q"], st["k"], st["v"] = q, k[new].contiguous(), v[new].contiguous()
    if case["kind"] == "write":  # the new rows are not in the cache yet
        k[new], v[new] = 0.0, 0.0
    outs = 1 if case["kind"] == "attend" else 2
    st["out"] = [torch.empty(len(new), case["n_head"] if outs == 1 else kv, hd, device=DEV) for _ in range(outs)]
    n_pages = free.numel()
    if own:
        import kvad_amd as K

        ctx = _context()
        st["cache"] = K.PagedCache(ctx, 1, kv, hd, n_pages, page_size=P, precision=K.MXFP4)
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
        # every position's place in the pool, sequence after sequence
        pos = torch.cat([torch.arange(n) for n in lens])
        seq = torch.repeat_interleave(torch.arange(S), torch.tensor(lens))
        slot = (table[seq, pos // P].long() * P + pos % P).to(DEV)
        groups = -(-hd // GROUP)
        for name, x in (("k", k), ("v", v)):
            pool = torch.zeros(n_pages * P, kv, groups * GROUP // 2, dtype=torch.uint8, device=DEV)
            exps = torch.zeros(n_pages * P, kv, groups, dtype=torch.int16, device=DEV)
            for at in range(0, len(slot), 16384):
                part = slice(at, at + 16384)
                code, e = quantised(x[part])
                pool[slot[part]], exps[slot[part]] = packed(code), e
            st[name + "_pool"], st[name + "_exps"] = pool, exps
        st["values"] = torch.tensor(VALUES + [-x for x in VALUES], device=DEV)
    return st


# ---- the operators -----------------------------------------------------------

def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        if kind == "norm":
            import kvad_amd as K

            m, n = case["m"], case["n"]
            ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
            K.norm_residual_dev(st["ctx"], st["x"].data_ptr(), st["y"].data_ptr(), m, n, st["eps"],
                                st["x_out"].data_ptr(), post_ptr=ptr(st["post"]), gate_ptr=ptr(st["gate"]),
                                gate_stride=n if case["gate"] == "each" else 0, scale=st["scale"],
                                pre_ptr=ptr(st["pre"]), out_ptr=st["out"].data_ptr() if case["pre"] else None)
            return {"x": st["x_out"], "out": st["out"]} if case["pre"] else {"x": st["x_out"]}
        if kind == "rope":
            import kvad_amd as K

            K.rope_rows_dev(st["ctx"], st["cos"].data_ptr(), st["sin"].data_ptr(), case["head_dim"] // 2,
                            st["cos"].shape[0], st["x"].data_ptr(), st["position"].data_ptr(), st["x"].shape[0],
                            case["n_head"] + case["n_kv_head"], st["out"].data_ptr(), case["interleaved"],
                            x_stride=st["x"].shape[1])
            return st["out"]
        if kind == "pages":
            table = st["table"]
            table.release_dev(st["ctx"], st["keep"].data_ptr())
            table.step_dev(st["ctx"], st["new"].data_ptr(), st["slot"].numel(), st["position"].data_ptr(),
                           st["slot"].data_ptr())
            return pages_out(st)
        cache, batch, out = st["cache"], st["batch"], st["out"]
        if kind == "attend":
            cache.attend_dev(0, batch, case["n_head"], st["q"].data_ptr(), out[0].data_ptr(), window=case["window"],
                             sinks=case["sinks"])
            return out[0]
        cache.push_dev(0, batch, st["k"].data_ptr(), st["v"].data_ptr())
        cache.read_dev(0, batch, out[0].data_ptr(), out[1].data_ptr())
        return {"k": out[0], "v": out[1]}
    if kind == "norm":
        return plain_norm(st)
    if kind == "rope":
        return plain_rope(st)
    if kind == "pages":
        plain_release(st)
        plain_step(st)
        return pages_out(st)
    if kind == "attend":
        return plain_attend(st)
    slots = row_slots(st)
    for name in ("k", "v"):
        code, st[name + "_exps"][slots] = quantised(st[name])
        st[name + "_pool"][slots] = packed(code)
    return {name: held(st, name, slots) for name in ("k", "v")}


def plain_norm(st):
    eps, x, t = st["eps"], st["x"], st["y"]
    rms = lambda a: a / torch.sqrt((a * a).mean(-1, keepdim=True) + eps)  # noqa: E731
    if st["post"] is not None:
        t = rms(t) * st["post"]
    if st["gate"] is not None:
        t = t * st["gate"]
    x = x + st["scale"] * t
    if st["pre"] is None:
        return {"x": x}
    return {"x": x, "out": rms(x) * st["pre"]}


def plain_rope(st):
    case, x = st["case"], st["x"]
    vectors, hd = case["n_head"] + case["n_kv_head"], case["head_dim"]
    x = x[:, :vectors * hd].reshape(-1, vectors, hd)
    at = st["position"].long()
    c, s = st["cos"][at][:, None, :], st["sin"][at][:, None, :]
    if case["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def pages_out(st):
    return {name: st[name] for name in ("pages", "len", "row_start", "free", "n_free", "position", "slot")}


def plain_release(st):
    """Pages behind the first `keep` positions go back on the stack, the last
    sequence's last page first."""
    P, pages, length = st["case"]["page"], st["pages"], st["len"]
    keep = torch.where(st["keep"] < 0, length, torch.minimum(st["keep"], length))
    column = torch.arange(pages.shape[1], device=DEV)
    gone = (column >= ((keep + P - 1) // P)[:, None]) & (column < ((length + P - 1) // P)[:, None])
    back = pages[gone].flip(0)
    st["free"][st["n_free"] + torch.arange(back.numel(), device=DEV)] = back
    st["n_free"] += back.numel()
    pages[gone] = -1
    length.copy_(keep)


def plain_step(st):
    """Each sequence's new rows: pages from the stack's top where they need
    them, in the sequences' order, a position and a slot each."""
    P, pages, length, new = st["case"]["page"], st["pages"], st["len"], st["new"]
    after = length + new
    column = torch.arange(pages.shape[1], device=DEV)
    more = (column >= ((length + P - 1) // P)[:, None]) & (column < ((after + P - 1) // P)[:, None])
    count = int(more.sum())
    pages[more] = st["free"][st["n_free"] - 1 - torch.arange(count, device=DEV)]
    st["n_free"] -= count
    start = torch.cumsum(new, 0)
    st["row_start"][1:] = start
    row = torch.arange(st["slot"].numel(), device=DEV)
    seq = torch.searchsorted(start, row, right=True)
    position = length[seq] + (row - st["row_start"][seq])
    st["position"].copy_(position)
    st["slot"].copy_(pages[seq, position // P].long() * P + position % P)
    length.copy_(after)


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
    byte = st[name + "_pool"][slots]
    code = torch.stack([byte & 15, byte >> 4], -1).flatten(-2)
    x = st["values"][code.int()].unflatten(-1, (-1, GROUP))
    scale = torch.exp2(st[name + "_exps"][slots].float())[..., None]
    return (x * scale).flatten(-2)[..., :st["case"]["head_dim"]]


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


# ---- the definitions in 64 bits ------------------------------------------------

def rounded(x):
    """The values the cache holds for rows x, from the definition: the nearest
    of E2M1's values, of two as near the one whose code is even."""
    x = x.double()
    hd = x.shape[-1]
    out = torch.zeros_like(x)
    tops = [x[..., a:a + GROUP].abs().amax(-1, keepdim=True) for a in range(0, hd, GROUP)]
    exps = []
    for amax in tops:
        e = torch.floor(torch.log2(amax.clamp(min=1e-300) / 3.5))
        # log2 rounds: the power of two that the definition asks for
        e = e + (amax >= 7.0 * torch.exp2(e)).double() - (amax < 3.5 * torch.exp2(e)).double()
        exps.append(e.clamp(min=-128.0))
    low = (torch.stack(exps).amax(0) - 12.0).clamp(min=-126.0) - 14.0
    for i, a in enumerate(range(0, hd, GROUP)):
        unit = torch.exp2(torch.maximum(exps[i], low))
        y = x[..., a:a + GROUP] / unit
        # steps of 0.5 up to 2, of 1 up to 4, of 2 beyond; torch rounds ties to even
        step = torch.where(y.abs() < 2.0, 0.5, torch.where(y.abs() < 4.0, 1.0, 2.0))
        out[..., a:a + GROUP] = (torch.round(y / step) * step).clamp(-6.0, 6.0) * unit
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "norm":
        d = {k: v.double() if torch.is_tensor(v) else v for k, v in norm_data(case, seed).items()}
        normed = lambda a, w: a * torch.rsqrt(a.square().sum(-1, keepdim=True) / case["n"] + d["eps"]) * w  # noqa: E731
        add = d["y"] if d["post"] is None else normed(d["y"], d["post"])
        x = d["x"] + d["scale"] * (add if d["gate"] is None else add * d["gate"])
        return {"x": x, "out": normed(x, d["pre"])} if case["pre"] else {"x": x}
    if kind == "rope":
        d = rope_data(case, seed)
        vectors, hd = case["n_head"] + case["n_kv_head"], case["head_dim"]
        turn = torch.complex(d["cos"].double(), d["sin"].double())[d["position"].long()][:, None, :]
        x = d["x"][:, :vectors * hd].double().reshape(-1, vectors, hd)
        if case["interleaved"]:
            return torch.view_as_real(torch.view_as_complex(x.reshape(-1, vectors, hd // 2, 2)) * turn).reshape(x.shape)
        z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)
    if kind == "pages":
        return exact_pages(case, seed)
    lens, news, k, v, q = data(case, seed)
    ends = torch.cumsum(torch.tensor(lens), 0).tolist()
    if kind == "write":
        pick = lambda x: torch.cat([rounded(x[e - m:e]) for e, m in zip(ends, news)])  # noqa: E731
        return {"k": pick(k), "v": pick(v)}
    H, kv, hd = case["n_head"], case["n_kv_head"], case["head_dim"]
    out = torch.zeros(sum(news), H, hd, dtype=torch.float64, device=DEV)
    row = 0
    for n, m, e in zip(lens, news, ends):
        ks, vs = rounded(k[e - n:e]), rounded(v[e - n:e])
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


def exact_pages(case, seed):
    """One page and one row at a time."""
    lens, news = layout(case)
    table, free, n_free = tables(case, seed)
    P, rows, stack = case["page"], table.tolist(), free.tolist()
    for s in reversed(range(case["seqs"])):
        used = -(-lens[s] // P)
        kept = -(-(lens[s] - news[s]) // P)
        for j in reversed(range(kept, used)):
            stack[n_free] = rows[s][j]
            n_free += 1
            rows[s][j] = -1
    position, slot, start = [], [], [0]
    for s in range(case["seqs"]):
        for p in range(lens[s] - news[s], lens[s]):
            if rows[s][p // P] < 0:
                n_free -= 1
                rows[s][p // P] = stack[n_free]
            position.append(p)
            slot.append(rows[s][p // P] * P + p % P)
        start.append(len(position))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"pages": i32(rows), "len": i32(lens), "row_start": i32(start), "free": i32(stack), "n_free": i32([n_free]),
            "position": i32(position), "slot": torch.tensor(slot, dtype=torch.int64, device=DEV)}
