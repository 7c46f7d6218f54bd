"""Performance cases of the operators around paged attention: the tables of an engine step, rotary positions with
several axes, and cross attention to an encoder's states.

Each case is a plain dict.  ``listed()`` gives the named ones, ``draw(rng)`` another of the same ranges,
``prepare(case, seed)`` what the program holds before the call, ``run(state)`` one pass -- through the framework's entry
points where ``own`` is true, in elementary torch operations otherwise --, ``work(case)`` the bytes and operations a pass
cannot do without and ``exact(case, seed)`` its result in 64 bits.

Kinds:
  tables   ops.step_tables: block tables, slots and positions of a step, from the requests' lengths and a free list
  write    ops.rope_axes_cache_write: Q rotated, rotated K and V written to their slots of the paged cache
  rope     ops.rope_axes: Q and K rotated into new tensors
  remap    ops.rope_remap_axes: recalled K re-rotated in its pages
  cross    ops.cross_attention: each sequence's tokens over its own encoder states
"""
from __future__ import annotations

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp16": 2, "fp32": 4}

_MAX_WORK = 1.3e12  # operations of a drawn case, the largest listed one's at most
_MAX_BYTES = 2.5e9


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # A decode step of 24 conversations, its tables padded to 32 token rows: the smallest call, all latency.
        dict(name="tables_decode", kind="tables", decode=24, prompts=0, chunk=0, prior=0, ctx=16384, page=16, rows=32),
        # A busy server's step: 960 decoding requests and 64 prompt chunks.
        dict(name="tables_mixed", kind="tables", decode=960, prompts=64, chunk=1111, prior=700, ctx=32768, page=16, rows=24576),
        # The same decode step's Q, K and V on three axes (time, height, width).
        dict(name="write_decode", kind="write", dtype="bf16", tokens=24, hq=32, hkv=8, d=128, rotary=128, sections="16,24,24",
             interleaved=False, adjacent=False, page=16, layout="block_kv", theta=500000.0, far=131072),
        # Prompts of images and text, 16,411 tokens in one step, axes dealt out in turn.
        dict(name="write_prompts", kind="write", dtype="bf16", tokens=16411, hq=32, hkv=8, d=128, rotary=128, sections="24,20,20",
             interleaved=True, adjacent=False, page=16, layout="block_kv", theta=500000.0, far=131072),
        # An image encoder's Q and K: two axes (height, width), neighbouring pairs, head_dim 64.
        dict(name="rope_image", kind="rope", dtype="fp16", tokens=9005, hq=16, hkv=16, d=64, rotary=64, sections="16,16",
             interleaved=False, adjacent=True, theta=10000.0, far=512),
        # Recalled K re-rotated in its pages, on three axes.
        dict(name="remap_65k", kind="remap", dtype="bf16", tokens=65536, hkv=8, d=128, rotary=128, sections="16,24,24",
             interleaved=False, adjacent=False, page=16, layout="native", theta=500000.0, far=1000000),
        # Speech decoding: 32 sequences, one token each, over 1,500 encoder states (K and V of one projection).
        dict(name="cross_decode", kind="cross", dtype="fp16", batch=32, hq=16, hkv=16, d=64, queries=1, spread=1.0, states=1500,
             kv_spread=1.0, masked=0.0, empty=False),
        # One token each over long video: 16 sequences of up to 25,600 states, eight query heads a kv head.
        dict(name="cross_decode_long", kind="cross", dtype="bf16", batch=16, hq=64, hkv=8, d=128, queries=1, spread=1.0,
             states=25600, kv_spread=0.25, masked=0.0, empty=False),
        # Forced decoding of transcripts: 8 texts of up to 448 tokens over 1,500 states.
        dict(name="cross_texts", kind="cross", dtype="fp16", batch=8, hq=16, hkv=16, d=64, queries=448, spread=0.3, states=1500,
             kv_spread=1.0, masked=0.0, empty=False),
        # A chunk of 4,096 tokens over the 16,384 states of a set of images.
        dict(name="cross_images", kind="cross", dtype="bf16", batch=1, hq=32, hkv=8, d=128, queries=4096, spread=1.0,
             states=16384, kv_spread=1.0, masked=0.0, empty=False),
        # A ragged batch with padded states: 13 texts of 21 to 701 tokens, up to 6,404 states, a tenth of them hidden,
        # one text without states.
        dict(name="cross_ragged", kind="cross", dtype="bf16", batch=13, hq=32, hkv=8, d=128, queries=701, spread=0.03,
             states=6404, kv_spread=0.1, masked=0.1, empty=True),
        # The same operator in fp32, at the size of a small caption model.
        dict(name="cross_fp32", kind="cross", dtype="fp32", batch=4, hq=12, hkv=12, d=64, queries=101, spread=0.5, states=577,
             kv_spread=1.0, masked=0.0, empty=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "write", "rope", "remap", "cross", "cross", "cross"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    hq, hkv, d = rng.choice([(32, 8, 128), (16, 16, 64), (64, 8, 128), (32, 4, 128), (24, 8, 128), (12, 12, 64), (8, 8, 128), (32, 8, 64)])
    while True:
        if kind == "tables":
            prompts = rng.choice([0, 1, 5, 64])
            c = dict(kind=kind, decode=_log(rng, 1, 2048), prompts=prompts, chunk=_log(rng, 2, 2048) if prompts else 0,
                     prior=rng.choice([0, _log(rng, 1, 4096)]), ctx=_log(rng, 64, 65536), page=rng.choice([16, 16, 32, 64]), rows=0)
            c["rows"] = sum(n for _, n in _requests(c)) + rng.choice([0, 7, 64])
        elif kind in ("write", "rope", "remap"):
            rotary = rng.choice([d, d, d // 2])
            half = rotary // 2
            axes = rng.choice([1, 2, 3, 3])
            s = [half // axes] * axes
            s[0] = half - sum(s[1:])
            c = dict(kind=kind, dtype=dtype, tokens=_log(rng, 1, 40000), hq=hq, hkv=hkv, d=d, rotary=rotary,
                     sections=",".join(map(str, s)), interleaved=rng.random() < 0.4, adjacent=rng.random() < 0.25, page=rng.choice([16, 16, 32]),
                     layout=rng.choice(["native", "kv_first", "block_kv"]), theta=rng.choice([10000.0, 500000.0]), far=_log(rng, 100, 1000000))
            if kind == "remap":
                del c["hq"]
            if kind == "rope":
                del c["page"], c["layout"]
        else:
            c = dict(kind=kind, dtype=dtype, batch=_log(rng, 1, 48), hq=hq, hkv=hkv, d=d, queries=rng.choice([1, _log(rng, 2, 4096)]),
                     spread=round(rng.choice([1.0, rng.uniform(0.02, 1.0)]), 3), states=_log(rng, 1, 32768),
                     kv_spread=round(rng.choice([1.0, rng.uniform(0.05, 1.0)]), 3), masked=rng.choice([0.0, 0.0, 0.2]), empty=False)
            c["empty"] = c["batch"] > 2 and rng.random() < 0.2
            if dtype == "fp32" and work(c)["flops"] > 1e11:
                continue
        w = work(c)
        pairs = c.get("batch", 0) * c.get("queries", 0) * c.get("states", 0) * c.get("hq", 0)
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= _MAX_WORK and pairs <= 2.2e9:  # (the plain form holds the padded scores)
            return c


# ---------------------------------------------------------------------------
# Sizes
# ---------------------------------------------------------------------------
def _lens(n, longest, spread):
    """n lengths from longest * spread to longest (spaced evenly over their logarithm), in a mixed order."""
    lo = max(1, int(longest * spread))
    if n == 1 or lo >= longest:
        return [longest] * n
    v = [int(round(math.exp(math.log(lo) + (math.log(longest) - math.log(lo)) * i / (n - 1)))) for i in range(n)]
    return [v[(i * 7 + 3) % n] if math.gcd(7, n) == 1 else v[i] for i in range(n)]


def _requests(case):
    """(tokens in the cache, new tokens) of each request: decoding ones, then prompt chunks, every other one fresh."""
    rows = [(n - 1, 1) for n in _lens(case["decode"], case["ctx"], 0.03)]
    for i, n in enumerate(_lens(case["prompts"], case["chunk"], 0.02) if case["prompts"] else []):
        rows.append((case["prior"] if i % 2 == 0 else 0, n))
    return rows


def _pages(tokens, page):
    return -(-tokens // page)


def _sequences(case):
    """(queries, states) of each sequence."""
    c = _lens(case["batch"], case["queries"], case["spread"])
    n = _lens(case["batch"], case["states"], case["kv_spread"])[::-1]
    if case["empty"]:
        n[len(n) // 2] = 0
    return list(zip(c, n))


def work(case):
    k = case["kind"]
    if k == "tables":
        rows, p = _requests(case), case["page"]
        new = sum(_pages(c + n, p) - _pages(c, p) for c, n in rows)
        # lengths and deltas read, offsets and lengths written; slots and positions; table entries of pages already
        # held that take new tokens; new pages read, and written to the table, the flags and the pages' positions
        held = sum(1 for c, n in rows if c % p and n)
        return {"bytes": 20 * len(rows) + 12 * case["rows"] + 4 * held + 13 * new, "flops": 0}
    if k in ("write", "rope", "remap"):
        t, es, axes = case["tokens"], _ES[case["dtype"]], len(case["sections"].split(","))
        if k == "remap":
            return {"bytes": t * (2 * case["hkv"] * case["rotary"] * es + 8 * axes), "flops": 0}
        heads = 2 * case["hq"] + 2 * case["hkv"] + (2 * case["hkv"] if k == "write" else 0)
        return {"bytes": t * (heads * case["d"] * es + 4 * axes + (8 if k == "write" else 0)), "flops": 0}
    es, d, hq, hkv = _ES[case["dtype"]], case["d"], case["hq"], case["hkv"]
    seqs = _sequences(case)
    return {"bytes": sum(2 * c * hq * d * es + n * (2 * hkv * d * es + (1 if case["masked"] else 0)) for c, n in seqs),
            "flops": 4 * d * hq * sum(c * n for c, n in seqs)}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _pool(g, pages, case, dtype):
    p, h, d = case["page"], case["hkv"], case["d"]
    shape = {"native": (pages, p, 2, h, d), "kv_first": (2, pages, p, h, d), "block_kv": (pages, 2, p, h, d)}[case["layout"]]
    return _randn(g, shape, dtype)


def _positions(g, case, far):
    """[axes, T]: text tokens (one number for all axes) with grids of 24 x 24 patches among them."""
    t = torch.arange(case["tokens"], device="cuda")
    axes = len(case["sections"].split(","))
    start = torch.randint(0, max(1, far - 1), (1,), generator=g, device="cuda")
    image = (t // 576) % 2 == 1
    rows = [torch.where(image, t // 576 * 576 + (0 if a == 0 and axes == 3 else (t % 576 // 24 if a == axes - 2 else t % 24)), t) for a in range(axes)]
    return ((torch.stack(rows) + start) % far).to(torch.int32)


def _axis_map(case):
    """The axis of each pair, as a list: sections one after the other, or dealt out in turn until a section is used up."""
    s = [int(x) for x in case["sections"].split(",")]
    n, half = len(s), sum(s)
    if not case["interleaved"]:
        return [a for a, c in enumerate(s) for _ in range(c)]
    return [j % n if j < n * s[j % n] else 0 for j in range(half)]


def prepare(case, seed):
    g = _gen(seed)
    k = case["kind"]
    if k == "tables":
        rows, p = _requests(case), case["page"]
        b, width = len(rows), max(_pages(c + n, p) for c, n in rows) + 3
        held = [_pages(c, p) for c, _ in rows]
        need = sum(_pages(c + n, p) for c, n in rows) - sum(held)
        pages = sum(held) + need + 40
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        col = torch.arange(width, device="cuda")
        h = torch.tensor(held, device="cuda")
        first = torch.cumsum(h, 0) - h
        table = torch.where(col < h[:, None], perm[(first[:, None] + col).clamp(max=pages - 1)], -1)
        free = torch.full((need + 64,), -1, dtype=torch.int32, device="cuda")
        free[:need + 40] = perm[sum(held):]
        i32 = dict(dtype=torch.int32, device="cuda")
        valid = torch.zeros(pages, dtype=torch.int8, device="cuda")
        valid[perm[:sum(held)].long()] = 1
        return dict(case=case, table=table.to(torch.int32).contiguous(), computed=torch.tensor([c for c, _ in rows], **i32),
                    new=torch.tensor([n for _, n in rows], **i32), delta=torch.randint(-500, 500, (b,), generator=g, **i32),
                    free=free, count=torch.tensor([need + 40], **i32), valid=valid,
                    where=torch.randint(0, 1 << 20, (pages,), generator=g, **i32),
                    out=(torch.empty(b + 1, **i32), torch.empty(b, **i32), torch.empty(case["rows"], dtype=torch.int64, device="cuda"),
                         torch.empty(case["rows"], **i32), torch.empty(1, **i32)))
    if k in ("write", "rope", "remap"):
        dt, t, half = _DT[case["dtype"]], case["tokens"], case["rotary"] // 2
        inv = 1.0 / (case["theta"] ** (torch.arange(half, dtype=torch.float32) / half))
        s = dict(case=case, inv=inv.cuda(), sections=[int(x) for x in case["sections"].split(",")], pos=_positions(g, case, case["far"]),
                 axis=torch.tensor(_axis_map(case), device="cuda"))
        hkv, d = case["hkv"], case["d"]
        if k == "remap":
            n = _pages(t, case["page"])
            s["pages"] = torch.randperm(n + 9, generator=g, device="cuda")[:n].to(torch.int32)
            s["pool"] = _pool(g, n + 9, case, dt)
            s["to"] = (s["pos"][:1] * 0 + torch.arange(t, device="cuda") + 1234).to(torch.int32).expand(s["pos"].shape[0], t).contiguous()
            return s
        # q, k and v are slices of one projection's output, as a model has them.
        hq = case["hq"]
        qkv = _randn(g, (t, hq + 2 * hkv, d), dt)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["q_out"] = torch.empty(t, hq, d, dtype=dt, device="cuda")
        if k == "rope":
            s["k_out"] = torch.empty(t, hkv, d, dtype=dt, device="cuda")
            return s
        n = _pages(t, case["page"]) + 9
        s["pool"] = _pool(g, n, case, dt)
        s["slots"] = torch.randperm(n * case["page"], generator=g, device="cuda")[:t].contiguous()
        s["slots"][5::97] = -1  # padded rows
        return s
    dt, d, hq, hkv = _DT[case["dtype"]], case["d"], case["hq"], case["hkv"]
    seqs = _sequences(case)
    c, n = torch.tensor([x for x, _ in seqs]), torch.tensor([x for _, x in seqs])
    nt = max(1, int(n.sum()))
    kv = _randn(g, (nt, 2, hkv, d), dt)  # one projection's output
    i32 = dict(dtype=torch.int32, device="cuda")
    mask = torch.rand(nt, generator=g, device="cuda") >= case["masked"] if case["masked"] else None
    return dict(case=case, q=_randn(g, (int(c.sum()), hq, d), dt), k=kv[:, 0], v=kv[:, 1], mask=mask,
                starts=torch.tensor([0] + torch.cumsum(c, 0).tolist(), **i32), kv_start=torch.tensor((torch.cumsum(n, 0) - n).tolist(), **i32),
                kv_lens=torch.tensor(n.tolist(), **i32), most_q=int(c.max()), most_kv=int(n.max()),
                out=torch.empty(int(c.sum()), hq, d, dtype=dt, device="cuda"))


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from kessie_amd import ops

    c = s["case"]
    k = c["kind"]
    if k == "tables":
        r = ops.step_tables(s["table"], s["computed"], s["new"], c["page"], c["rows"], s["free"], s["count"], position_delta=s["delta"],
                            page_valid=s["valid"], page_positions=s["where"], out=s["out"])
        return [*r, s["table"], s["valid"], s["where"]]
    if k == "cross":
        return ops.cross_attention(s["q"], s["k"], s["v"], s["starts"], s["most_q"], s["kv_start"], s["kv_lens"], s["most_kv"],
                                   key_mask=s["mask"], out=s["out"])
    kind = dict(interleaved=c["interleaved"], adjacent=c["adjacent"])
    if k == "write":
        q = ops.rope_axes_cache_write(s["q"], s["k"], s["v"], s["pos"], s["pool"], s["slots"], s["inv"], s["sections"], q_out=s["q_out"],
                                      layout=c["layout"], **kind)
        return [q, s["pool"]]
    if k == "rope":
        return list(ops.rope_axes(s["q"], s["k"], s["pos"], s["inv"], s["sections"], q_out=s["q_out"], k_out=s["k_out"], **kind))
    ops.rope_remap_axes(s["pool"], s["pos"], s["to"], s["inv"], s["sections"], page_list=s["pages"], layout=c["layout"], **kind)
    return s["pool"]


def _run_plain(s):
    c = s["case"]
    k = c["kind"]
    if k == "tables":
        return _plain_tables(s)
    if k == "cross":
        return _plain_cross(s)
    half = c["rotary"] // 2
    kp = vp = None
    if k != "rope":
        # K and V as [pages, P, H, D] views of the pool
        kp, vp = {"native": lambda x: (x[:, :, 0], x[:, :, 1]), "kv_first": lambda x: (x[0], x[1]),
                  "block_kv": lambda x: (x[:, 0], x[:, 1])}[c["layout"]](s["pool"])
    if k == "remap":
        t = torch.arange(c["tokens"], device="cuda")
        page, at = s["pages"].long()[t // c["page"]], t % c["page"]
        cos, sin = _plain_angles(s, s["to"].long() - s["pos"].long())
        kp[page, at] = _plain_rotate(kp[page, at], cos, sin, half, c["adjacent"])
        return s["pool"]
    cos, sin = _plain_angles(s, s["pos"].long())
    s["q_out"].copy_(_plain_rotate(s["q"], cos, sin, half, c["adjacent"]))
    key = _plain_rotate(s["k"], cos, sin, half, c["adjacent"])
    if k == "rope":
        s["k_out"].copy_(key)
        return [s["q_out"], s["k_out"]]
    # (Rows without a slot repeat row 0, which has one.)
    ok = s["slots"] >= 0
    row = torch.where(ok, torch.arange(c["tokens"], device="cuda"), 0)
    slot = s["slots"][row]
    kp[slot // c["page"], slot % c["page"]] = key[row]
    vp[slot // c["page"], slot % c["page"]] = s["v"][row]
    return [s["q_out"], s["pool"]]


def _plain_angles(s, pos):
    """cos, sin [T, 1, R/2] of pos[axis(j), t] * inv_freq[j], in 64 bits and rounded once."""
    ang = pos[s["axis"]].double().t() * s["inv"].double()
    return torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]


def _plain_rotate(x, cos, sin, half, adjacent):
    y = x.float()
    if adjacent:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([r, y[..., 2 * half:]], -1).to(x.dtype)


def _plain_tables(s):
    c = s["case"]
    p, rows, width = c["page"], c["rows"], s["table"].shape[1]
    n, have = s["new"].long(), s["computed"].long()
    end = torch.cumsum(n, 0)
    start = end - n
    held, total = (have + p - 1) // p, (have + n + p - 1) // p
    fits = total <= width
    need = torch.where(fits, total - held, 0)
    upto = torch.cumsum(need, 0)
    some = need > 0
    grant = fits & (end <= rows) & (~some | (upto <= s["count"]))
    start_loc, lens, slots, positions, taken = s["out"]
    start_loc[:1] = 0
    start_loc[1:] = end
    lens.copy_(torch.where(grant, have + n, have))
    taken.copy_(torch.where(grant & some, upto, 0).max())
    t = torch.arange(rows, device="cuda")
    live = t < end[-1]
    b = torch.searchsorted(end, t, right=True).clamp(max=n.numel() - 1)
    pos = have[b] + t - start[b]
    i = pos // p
    ok = live & grant[b]
    fresh = i >= held[b]
    old = s["table"].view(-1)[b * width + i.clamp(max=width - 1)]
    new = s["free"][(upto[b] - need[b] + i - held[b]).clamp(0, s["free"].numel() - 1)]
    page = torch.where(fresh, new, old).long()
    slots.copy_(torch.where(ok & (page >= 0), page * p + pos % p, -1))
    positions.copy_(torch.where(live, pos + s["delta"][b], 0))
    # A new page's first token writes its table entry, its flag and its position; the others write past the end.
    head = ok & fresh & (pos % p == 0)
    for to, at, value in ((s["table"], b * width + i, page), (s["valid"], page, torch.ones_like(page)), (s["where"], page, pos + s["delta"][b])):
        more = torch.cat([to.view(-1), to.view(-1)[:1]])
        more[torch.where(head, at, to.numel())] = value.to(to.dtype)
        to.view(-1).copy_(more[:-1])
    return [*s["out"], s["table"], s["valid"], s["where"]]


def _plain_cross(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    b, mq, mk = c["batch"], s["most_q"], s["most_kv"]
    counts = (s["starts"][1:] - s["starts"][:-1]).long()
    i, j = torch.arange(mq, device="cuda"), torch.arange(mk, device="cuda")
    qi = (s["starts"][:-1].long()[:, None] + i).clamp(max=s["q"].shape[0] - 1)
    kj = (s["kv_start"].long()[:, None] + j).clamp(max=s["k"].shape[0] - 1)
    seen = j < s["kv_lens"].long()[:, None]
    if s["mask"] is not None:
        seen = seen & s["mask"][kj]
    g = hq // hkv
    q = s["q"].float()[qi].view(b, mq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * mq, d)
    k = s["k"][kj].float().permute(0, 2, 3, 1).contiguous()  # [B, Hkv, D, mk]
    v = s["v"][kj].float().permute(0, 2, 1, 3).contiguous()
    x = torch.matmul(q * d ** -0.5, k).masked_fill_(~seen[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True) if mk else x.new_full((b, hkv, g * mq, 1), float("-inf"))
    x.sub_(torch.where(torch.isinf(m), 0.0, m)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v) / torch.where(total > 0, total, 1.0)
    o = o.view(b, hkv, g, mq, d).permute(0, 3, 1, 2, 4).reshape(b * mq, hq, d).to(s["q"].dtype)
    # (A row past its sequence's end repeats the sequence's last one.)
    src = torch.arange(b, device="cuda")[:, None] * mq + torch.minimum(i, counts[:, None] - 1)
    dst = s["starts"][:-1].long()[:, None] + torch.minimum(i, counts[:, None] - 1)
    s["out"][dst.view(-1)] = o[src.view(-1)]
    return s["out"]


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    k = case["kind"]
    if k == "tables":
        return None
    if k == "cross":
        return _exact_cross(s, case)
    delta = s["to"].double() - s["pos"].double() if k == "remap" else s["pos"].double()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       (delta[_axis_map(case)] * s["inv"].double()[:, None]).t()[:, None, :])  # [T, 1, R/2]
    r, half = case["rotary"], case["rotary"] // 2

    def rotate(x):
        x = x.double().clone()
        a = slice(0, r, 2) if case["adjacent"] else slice(0, half)
        b = slice(1, r, 2) if case["adjacent"] else slice(half, r)
        z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
        x[..., a], x[..., b] = z.real, z.imag
        return x

    if k == "rope":
        return [rotate(s["q"]), rotate(s["k"])]
    pool = s["pool"].double()
    order = {"native": (0, 1, 2, 3, 4), "kv_first": (1, 2, 0, 3, 4), "block_kv": (0, 2, 1, 3, 4)}[case["layout"]]
    flat = pool.permute(order)  # [pages, P, 2, H, D]
    p = case["page"]
    if k == "remap":
        slot = (s["pages"].long()[:, None] * p + torch.arange(p, device="cuda")).view(-1)[:case["tokens"]]
        flat[slot // p, slot % p, 0] = rotate(flat[slot // p, slot % p, 0])
        return pool
    keep = s["slots"] >= 0
    slot = s["slots"][keep]
    flat[slot // p, slot % p, 0] = rotate(s["k"])[keep]
    flat[slot // p, slot % p, 1] = s["v"].double()[keep]
    return [rotate(s["q"]), pool]


def _exact_cross(s, case):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["hq"] // case["hkv"]
    at = kv = 0
    for count, states in _sequences(case):
        keep = torch.ones(states, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"][kv:kv + states]
        if bool(keep.any()):
            for h in range(case["hq"]):
                key, value = (t[kv:kv + states, h // group][keep].double() for t in (s["k"], s["v"]))
                w = torch.softmax(s["q"][at:at + count, h].double() @ key.t() / math.sqrt(case["d"]), -1)
                out[at:at + count, h] = w @ value
        at, kv = at + count, kv + states
    return out
