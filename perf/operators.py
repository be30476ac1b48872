"""Cases of the 8-bit KV cache's operators: block tables and slot maps built on the GPU, appending to the cache,
reading it back, attention over it, and a whole step of them.

The cache holds int8 with one fp32 scale for each block of 16 positions, head, and K or V, in pages of 64 positions:
pages [n_pages][kv_heads][2][64][head_dim], scales [n_pages][kv_heads][2][4].  Plain forms are elementary torch
operations in 32 bits (64 where a rounding border decides an integer).
"""
import math
import random

import torch

own = False

PAGE, BLOCK = 64, 16
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one conversation takes its next token: the smallest call of the table builder
        _case("tables 1 seq", "tables", 1, 1, 1, 64, "bf16", 1087, 1087, 1, 1),
        # a full serving batch between two steps: some prompts arrive in chunks, every seventh sequence has ended
        _case("tables 4096 seqs", "tables", 4096, 1, 1, 64, "bf16", 0, 2040, 1, 31, released=7),
        # the next token of 64 sequences, K and V straight from the projection's fp32 epilogue
        _case("append 64 x 1 f32", "append", 64, 10, 1, 64, "f32", 256, 1535, 1, 1),
        # ragged prompt chunks of the default model, bf16 rows
        _case("append prompts", "append", 16, 10, 1, 64, "bf16", 0, 100, 129, 799),
        # large heads, few sequences, blocks half full: grouped-query layout
        _case("append 4 x 2001 hd128", "append", 4, 8, 4, 128, "f32", 7, 1000, 2001, 2001),
        # batch 1 at the end of the default context, fp32 queries and outputs: latency
        _case("decode 1 f32", "attn", 1, 10, 1, 64, "f32", 2047, 2047, 1, 1),
        # 512 ragged sequences, the throughput job of the default model
        _case("decode 512", "attn", 512, 10, 1, 64, "bf16", 256, 2047, 1, 1),
        # few long documents, grouped heads of 128
        _case("decode 4 long gqa", "attn", 4, 8, 4, 128, "bf16", 60001, 131071, 1, 1),
        # a chunk of ragged prompts of the default model
        _case("prompts", "attn", 12, 10, 1, 64, "bf16", 0, 64, 101, 1137),
        # further turns behind long histories, grouped heads of 128
        _case("turns gqa", "attn", 4, 8, 4, 128, "bf16", 2000, 6001, 513, 1025),
        # a whole step: tables, append, attention for 64 sequences, in lists padded as a captured step has them
        _case("step 64", "step", 64, 10, 1, 64, "bf16", 256, 1919, 1, 1),
        # a step that mixes prompt chunks with running sequences, grouped heads
        _case("step mixed gqa", "step", 24, 2, 4, 128, "bf16", 0, 4000, 1, 257),
    ]


def _case(name, op, seqs, kv_heads, group, head_dim, dtype, held_lo, held_hi, new_lo, new_hi, released=0):
    return {"name": name, "op": op, "seqs": seqs, "kv_heads": kv_heads, "group": group, "head_dim": head_dim, "dtype": dtype,
            "held_lo": held_lo, "held_hi": held_hi, "new_lo": new_lo, "new_hi": new_hi, "released": released}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(10, 1, 64), (4, 1, 32), (24, 1, 64), (8, 4, 128), (2, 4, 128), (2, 8, 64), (1, 16, 128), (3, 1, 16), (12, 1, 128), (6, 2, 32), (5, 3, 64)]


def draw(rng):
    op = rng.choice(["tables", "append", "attn", "attn", "attn", "step"])
    h, g, d = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    while True:
        n = _log(rng, 1, 4096 if op == "tables" else 512)
        if rng.random() < 0.5:          # one to four new tokens behind what is held
            new_lo, new_hi = 1, rng.choice([1, 1, 1, 2, 4])
            hi = _log(rng, 1, 131071)
            lo = _log(rng, 1, hi)
        else:                           # prompts and further turns
            new_hi = _log(rng, 2, 2048)
            new_lo = _log(rng, 1, new_hi)
            hi = 0 if rng.random() < 0.3 else _log(rng, 1, 8191)
            lo = rng.randint(0, hi)
        c = _case("", op, n, h, g, d, dtype, lo, hi, new_lo, new_hi, rng.choice([0, 0, 3]) if op == "tables" else 0)
        del c["name"]
        if _fits(c):
            return c


def _fits(c):
    """No dearer than the largest listed cases, padded plain form included."""
    before, after = _lengths(c)
    new = sum(max(0, a - b) for a, b in zip(after, before))
    pairs = c["seqs"] * c["new_hi"] * max(after) * c["kv_heads"] * c["group"]
    held = c["seqs"] * max(after) * c["kv_heads"] * c["head_dim"]
    if c["op"] == "tables":
        return sum(before) < 8 << 20 and new <= 1 << 16
    if new > 8192 or held > 600 << 20:
        return False
    if c["op"] == "append":
        return new * c["kv_heads"] * c["head_dim"] <= 8 << 20
    w = work(c)
    return pairs <= 1 << 30 and w["bytes"] <= 780e6 and w["flops"] <= 200e9


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lengths(c):
    """Lengths before and after the step.  Their order among the sequences is the seed's."""
    n = c["seqs"]
    before = _spread(c["held_lo"], c["held_hi"], n)
    new = _spread(c["new_lo"], c["new_hi"], n)[::-1]
    after = [b + a for b, a in zip(before, new)]
    if c["released"]:
        after = [0 if i % c["released"] == 1 else a for i, a in enumerate(after)]
    return before, after


def _ceil(a, b):
    return -(-a // b)


def _cache(c, n_pages, g):
    """A cache of quantised normal rows; K has louder channels, as behind a rotation."""
    h, d = c["kv_heads"], c["head_dim"]
    pages = torch.empty(n_pages, h, 2, PAGE, d, dtype=torch.int8, device="cuda")
    scales = torch.empty(n_pages, h, 2, PAGE // BLOCK, device="cuda")
    loud = torch.exp(0.4 * torch.randn(2, 1, d, device="cuda", generator=g))
    loud[1] = 1.0
    step = max(1, (64 << 20) // (h * 2 * PAGE * d))
    for a in range(0, n_pages, step):
        x = torch.randn(min(step, n_pages - a), h, 2, PAGE, d, device="cuda", generator=g) * loud
        x = x.view(-1, h, 2, PAGE // BLOCK, BLOCK * d)
        s = x.abs().amax(-1) / 127
        scales[a:a + step] = s
        pages[a:a + step] = torch.round(x / s[..., None]).to(torch.int8).view(-1, h, 2, PAGE, d)
    return pages, scales


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    before, after = _lengths(case)
    order = list(range(case["seqs"]))
    random.Random(seed).shuffle(order)
    before, after = [before[i] for i in order], [after[i] for i in order]
    n, op = case["seqs"], case["op"]
    h, grp, d, t = case["kv_heads"], case["group"], case["head_dim"], TYPES[case["dtype"]]
    have = [_ceil(b, PAGE) for b in before]
    need = [_ceil(a, PAGE) for a in after]
    width = max(max(have), max(need)) + 1
    used = sum(max(x, y) for x, y in zip(have, need))
    n_pages = used + used // 8 + 3
    pool = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    held = torch.tensor(have if op in ("tables", "step") else need, device="cuda")
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None] < held[:, None]
    n_held = int(held.sum())
    table[at] = pool[:n_held]
    head = seed % n_pages
    ring = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    ring[(head + torch.arange(n_pages - n_held, device="cuda")) % n_pages] = pool[n_held:]
    new = [max(0, a - b) for a, b in zip(after, before)]
    total = sum(new)
    room = _ceil(total, 64) * 64 if op in ("tables", "step") else total
    s = {"op": op, "table": table, "ring": ring, "scale": d ** -0.5, "max_new": max(new), "max_len": max(max(after), 1),
         "before": torch.tensor(before, dtype=torch.int32, device="cuda"), "after": torch.tensor(after, dtype=torch.int32, device="cuda"),
         "pool_in": torch.tensor([head, n_pages - n_held, 0, 0], device="cuda"), "pool_out": torch.zeros(4, dtype=torch.int64, device="cuda"),
         "cu_tok": torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
         "tok_seq": torch.zeros(room, dtype=torch.int32, device="cuda"), "tok_pos": torch.zeros(room, dtype=torch.int32, device="cuda"),
         "slot_map": torch.zeros(room, dtype=torch.int64, device="cuda")}
    if op == "tables":
        return s
    s["pages"], s["scales"] = _cache(case, n_pages, g)
    if op in ("append", "attn"):        # their lists are there already
        cnt = torch.tensor(new, device="cuda")
        s["cu_tok"][1:] = cnt.cumsum(0)
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), cnt)
        pos = torch.arange(total, device="cuda") - s["cu_tok"][seq] + s["before"][seq]
        s["tok_seq"], s["tok_pos"] = seq.to(torch.int32), pos.to(torch.int32)
        s["slot_map"] = table[seq, pos // PAGE].long() * PAGE + pos % PAGE
    if op == "append":                  # every position of the blocks that the new rows fall into
        first = s["before"].long() // BLOCK * BLOCK
        cnt = s["after"].long() - first
        seq = torch.repeat_interleave(torch.arange(n, device="cuda"), cnt)
        pos = torch.arange(len(seq), device="cuda") - (cnt.cumsum(0) - cnt)[seq] + first[seq]
        s["read"] = table[seq, pos // PAGE].long() * PAGE + pos % PAGE
    # one fused projection's output: query heads, key heads, value heads
    qkv = torch.randn(room, (h * grp + 2 * h) * d, device="cuda", generator=g)
    qkv[:, :h * grp * d] *= 1.5
    qkv = qkv.to(t).view(room, h * grp + 2 * h, d)
    s["q"], s["k"], s["v"] = qkv[:, :h * grp], qkv[:, h * grp:h * grp + h], qkv[:, h * grp + h:]
    s["out"] = torch.zeros(room, h * grp, d, dtype=t, device="cuda")
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------

def _tables(s):
    b, a, table, ring = s["before"].long(), s["after"].long(), s["table"], s["ring"]
    n, width = table.shape
    n_pages, room = ring.numel(), s["tok_seq"].numel()
    dev = table.device
    head, free = s["pool_in"][0], s["pool_in"][1]
    have, need = (b + PAGE - 1) // PAGE, (a + PAGE - 1) // PAGE
    grow, drop, new = (need - have).clamp(min=0), (have - need).clamp(min=0), (a - b).clamp(min=0)
    grow_x, drop_x = grow.cumsum(0) - grow, drop.cumsum(0) - drop
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    bad = ((b < 0) | (a < 0) | (a > width * PAGE) | (b > width * PAGE)).any() | (free + drop.sum() > n_pages)
    full = (grow.sum() > free) | (cu[-1] > room)
    code = torch.where(bad, 1, torch.where(full, 4, 0))
    ok = code == 0
    col = torch.arange(width, device=dev)[None]
    taken = ring[(head + grow_x[:, None] + col - have[:, None]) % n_pages]
    opened = ok & (col >= have[:, None]) & (col < need[:, None])
    closed = ok & (col >= need[:, None]) & (col < have[:, None])
    place = torch.where(closed, (head + free + drop_x[:, None] + col - need[:, None]) % n_pages, n_pages)
    old = torch.where(closed, table, 0)
    table.copy_(torch.where(opened, taken, table))
    wide = torch.cat([ring, ring.new_zeros(1)]).index_put((place.reshape(-1),), old.reshape(-1))
    ring.copy_(wide[:n_pages])
    t = torch.arange(room, device=dev)
    live = ok & (t < cu[-1])
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=n - 1)
    pos = torch.where(live, t - cu[seq] + b[seq], 0)
    slot = table[seq, pos // PAGE].long() * PAGE + pos % PAGE
    s["cu_tok"].copy_(torch.where(ok, cu, 0))
    s["tok_seq"].copy_(torch.where(live, seq, -1))
    s["tok_pos"].copy_(torch.where(live, pos, -1))
    s["slot_map"].copy_(torch.where(live, slot, -1))
    s["pool_out"].copy_(torch.stack([torch.where(ok, (head + grow.sum()) % n_pages, head), torch.where(ok, free - grow.sum() + drop.sum(), free),
                                     torch.where(ok, cu[-1], 0), code]))


def _append(s):
    """Blocks are gathered whole, requantised and written back; a block that no row of this call opens keeps its scale or gets a larger one."""
    pages, scales, slot = s["pages"], s["scales"], s["slot_map"]
    n_pages, h, _, _, d = pages.shape
    live = slot >= 0
    # a row that follows on the one before it, inside the same block, belongs to the run that the first such row leads
    follows = torch.cat([live.new_zeros(1), (slot[1:] == slot[:-1] + 1) & (slot[1:] % BLOCK != 0)])
    lead = live & ~follows
    run = lead.long().cumsum(0) - 1
    blocks = slot[lead] // BLOCK
    first = slot[lead] % BLOCK
    m = blocks.numel()
    run, at = run[live], slot[live] % BLOCK
    x = torch.stack([s["k"][live], s["v"][live]], 2).float().double()            # [rows][h][2][d]
    rows = torch.zeros(m, BLOCK, h, 2, d, dtype=torch.float64, device=x.device)
    rows[run, at] = x
    fresh = torch.zeros(m, BLOCK, dtype=torch.bool, device=x.device)
    fresh[run, at] = True
    page, quarter = blocks // 4, blocks % 4
    old = pages.view(n_pages, h, 2, 4, BLOCK, d)[page, :, :, quarter].permute(0, 3, 1, 2, 4)   # [m][16][h][2][d]
    s_old = torch.where((first == 0)[:, None, None], 0.0, scales[page, :, :, quarter])          # [m][h][2]
    top = rows.abs().amax((1, 4)).float()
    s_new = top / torch.full_like(top, 127)                                     # a tensor: a plain number would be multiplied by 1 / 127
    s_new = torch.where(top > 0, s_new.clamp(min=2.0 ** -126), s_new)
    s_new = torch.where(torch.isfinite(rows).all(4).all(1), torch.maximum(s_new, s_old), math.nan)
    div = torch.where(s_new > 0, s_new, 1.0).double()[:, None, :, :, None]
    grown = (s_new != s_old)[:, None, :, :, None]
    was = torch.where(grown, torch.round(old.double() * s_old.double()[:, None, :, :, None] / div), old.double())
    held = (torch.arange(BLOCK, device=x.device)[None] < first[:, None])[:, :, None, None, None]
    q = torch.where(fresh[:, :, None, None, None], torch.round(rows / div), torch.where(held, was, old.double()))
    q = torch.where(torch.isnan(s_new)[:, None, :, :, None], 0.0, q).to(torch.int8)
    pages.view(n_pages, h, 2, 4, BLOCK, d)[page, :, :, quarter] = q.permute(0, 2, 3, 1, 4)
    scales[page, :, :, quarter] = s_new


def _read(s, slot):
    pages, scales = s["pages"], s["scales"]
    page, at = slot // PAGE, slot % PAGE
    x = pages[page, :, :, at].float() * scales[page, :, :, at // BLOCK][..., None]      # [rows][h][2][d]
    return x[:, :, 0], x[:, :, 1]


def _attention(s):
    pages, scales, table, q = s["pages"], s["scales"], s["table"].long(), s["q"]
    n, width = table.shape
    h, d = pages.shape[1], pages.shape[4]
    grp, t_max = q.shape[1] // h, s["max_new"]
    span = min(width, (s["max_len"] + PAGE - 1) // PAGE)
    live = s["tok_seq"] >= 0
    seq = torch.where(live, s["tok_seq"], 0).long()
    j = torch.arange(q.shape[0], device=q.device) - s["cu_tok"][seq].long()
    j = torch.where(live, j, t_max)                                             # dead rows go to a row of their own
    qp = torch.zeros(n, t_max + 1, h, grp, d, device=q.device)
    qp[seq, j] = q.float().view(-1, h, grp, d)
    pos = torch.full((n, t_max + 1), -1, dtype=torch.long, device=q.device)
    pos[seq, j] = torch.where(live, s["tok_pos"], -1).long()
    at = table[:, :span].clamp(min=0)
    kv = pages[at].view(n, span, h, 2, 4, BLOCK, d).float() * scales[at][..., None, None]
    kv = kv.permute(3, 0, 2, 1, 4, 5, 6).reshape(2, n, h, span * PAGE, d)
    qp = qp.permute(0, 2, 1, 3, 4).reshape(n, h, (t_max + 1) * grp, d) * s["scale"]
    w = torch.matmul(qp, kv[0].transpose(2, 3)).view(n, h, t_max + 1, grp, span * PAGE)
    seen = torch.arange(span * PAGE, device=q.device)[None, None] <= pos[..., None]
    w = torch.where(seen[:, None, :, None], w, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-3e38))
    total = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(n, h, (t_max + 1) * grp, -1), kv[1]).view(n, h, t_max + 1, grp, d) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(n, t_max + 1, h * grp, d)[seq, j]
    s["out"].copy_(torch.where(live[:, None, None], o.to(q.dtype), s["out"]))
    return s["out"]


def run(state):
    s = state
    if own:
        from small_llm_b200 import kv8

        def tables():
            kv8.block_tables(s["before"], s["after"], s["table"], s["ring"], s["pool_in"], s["pool_out"], s["cu_tok"], s["tok_seq"], s["tok_pos"], s["slot_map"])

        def append():
            kv8.append(s["k"], s["v"], s["slot_map"], s["pages"], s["scales"])

        def read(slot):
            return kv8.read(slot, s["pages"], s["scales"])

        def attention():
            return kv8.attention(s["q"], s["pages"], s["scales"], s["table"], s["tok_seq"], s["tok_pos"], s["cu_tok"], max_new=s["max_new"],
                                 max_len=s["max_len"], scale=s["scale"], out=s["out"])
    else:
        def tables():
            _tables(s)

        def append():
            _append(s)

        def read(slot):
            return _read(s, slot)

        def attention():
            return _attention(s)
    if s["op"] == "tables":
        tables()
        return {k: s[k] for k in ("table", "ring", "pool_out", "cu_tok", "tok_seq", "tok_pos", "slot_map")}
    if s["op"] == "append":
        append()
        k, v = read(s["read"])
        return {"k": k, "v": v}
    if s["op"] == "attn":
        return {"out": attention()}
    tables()
    append()
    out = attention()
    k, v = read(s["slot_map"].clamp(min=0))
    return {"out": out, "table": s["table"], "slot_map": s["slot_map"], "k": k, "v": v}


def work(case):
    before, after = _lengths(case)
    op, h, grp, d = case["op"], case["kv_heads"], case["group"], case["head_dim"]
    size = 2 if case["dtype"] == "bf16" else 4
    new = sum(max(0, a - b) for a, b in zip(after, before))
    moved = sum(abs(_ceil(a, PAGE) - _ceil(b, PAGE)) for a, b in zip(after, before))
    first = sum(a - b // BLOCK * BLOCK for a, b in zip(after, before) if a > b)
    nbytes = flops = 0
    if op in ("tables", "step"):
        nbytes += case["seqs"] * 12 + new * 16 + moved * 8 + 64
    if op in ("append", "step"):        # rows in, 8-bit rows out, and the same rows read back
        nbytes += new * 2 * h * d * (size + 1) + new * 8
        nbytes += (first if op == "append" else new) * 2 * h * d * (1 + 4)
    if op in ("attn", "step"):
        keys = sum(a * h * (2 * d + 2) for a in after)
        nbytes += keys + 2 * new * h * grp * d * size
        flops += sum(4 * d * h * grp * sum(range(b + 1, a + 1)) for a, b in zip(after, before))
    return {"bytes": nbytes, "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------

def _exact_append(s, slots, map_):
    """Block by block: the scale is the largest magnitude over 127 (or what the block had, if that is larger), values are whole multiples of it."""
    n_pages, h, _, _, d = s["pages"].shape
    blocks = {}
    for t, slot in enumerate(map_.tolist()):
        if slot >= 0:
            blocks.setdefault(slot // BLOCK, []).append((t, slot % BLOCK))
    ids = sorted(blocks)
    where = {b: i for i, b in enumerate(ids)}
    rank = torch.tensor(ids, device="cuda")
    flat = s["pages"].reshape(n_pages, h, 2, 4, BLOCK, d).permute(0, 3, 4, 1, 2, 5).reshape(n_pages * 4, BLOCK, h, 2, d)
    had = s["scales"].permute(0, 3, 1, 2).reshape(n_pages * 4, h, 2)[rank].double()
    val = flat[rank].double() * had[:, None, :, :, None]
    started = torch.tensor([min(o for _, o in blocks[b]) == 0 for b in ids], device="cuda")
    had = torch.where(started[:, None, None], torch.zeros_like(had), had)
    i = torch.tensor([where[b] for b in ids for _ in blocks[b]], device="cuda")
    t, o = (torch.tensor([p[k] for b in ids for p in blocks[b]], device="cuda") for k in (0, 1))
    x = torch.stack([s["k"], s["v"]], 2).double()[t]
    big = torch.zeros(len(ids), h, 2, dtype=torch.float64, device="cuda").index_reduce_(0, i, x.abs().amax(-1), "amax")
    step = torch.maximum((big / 127).float().double(), had)     # a scale is held in 32 bits
    unit = step.clamp(min=1e-300)[:, None, :, :, None]
    keep = torch.round(val / unit) * unit
    keep[i, o] = torch.round(x / unit[i][:, 0]) * unit[i][:, 0]
    # the slots asked for all lie in blocks of this call
    slots = slots.tolist()
    b = torch.tensor([where.get(v // BLOCK, 0) for v in slots], device="cuda")
    r = keep[b, torch.tensor([v % BLOCK for v in slots], device="cuda")]
    return r[:, :, 0], r[:, :, 1], (rank, keep)


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "tables":
        return None
    if op == "append":
        k, v, _ = _exact_append(s, s["read"], s["slot_map"])
        return {"k": k, "v": v}
    h, d = case["kv_heads"], case["head_dim"]
    before, after = s["before"].tolist(), s["after"].tolist()
    values = None
    if op == "step":                    # pages are taken from the ring in the order of the sequences
        at = int(s["pool_in"][0])
        ring, slots = s["ring"].tolist(), []
        for i, (b, a) in enumerate(zip(before, after)):
            for p in range(_ceil(b, PAGE), _ceil(a, PAGE)):
                s["table"][i, p] = ring[at % len(ring)]
                at += 1
            row = s["table"][i].tolist()
            slots += [row[p // PAGE] * PAGE + p % PAGE for p in range(b, a)]
        room = s["out"].shape[0]
        slot_map = torch.tensor(slots + [-1] * (room - len(slots)))
        k, v, values = _exact_append(s, slot_map[:len(slots)], slot_map)
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    t = 0
    for i, (b, a) in enumerate(zip(before, after)):
        row = s["table"][i, :_ceil(a, PAGE)].long()
        kv = s["pages"][row].double().view(-1, h, 2, 4, BLOCK, d) * s["scales"][row].double()[..., None, None]
        if values is not None:          # blocks that the append has changed
            ids, kept = values
            mine = (row[:, None] * 4 + torch.arange(4, device="cuda")).view(-1)
            place = torch.searchsorted(ids, mine).clamp(max=len(ids) - 1)
            hit = ids[place] == mine
            kv = kv.permute(0, 3, 4, 1, 2, 5).reshape(-1, BLOCK, h, 2, d)
            kv[hit] = kept[place[hit]]
            kv = kv.view(-1, h, 2, d).permute(1, 2, 0, 3)
        else:
            kv = kv.permute(1, 2, 0, 3, 4, 5).reshape(h, 2, -1, d)
        q = s["q"][t:t + a - b].double().view(a - b, h, -1, d)
        for j in range(h):
            for at in range(0, a - b, 256):
                z = torch.einsum("tgd,kd->tgk", q[at:at + 256, j], kv[j, 0, :a]) * s["scale"]
                last = torch.arange(b + at, min(b + at + 256, a), device="cuda")
                z = z.masked_fill(torch.arange(a, device="cuda")[None, None] > last[:, None, None], -math.inf)
                p = torch.softmax(z, -1)
                g = q.shape[2]
                out[t + at:t + at + len(last), j * g:(j + 1) * g] = torch.einsum("tgk,kd->tgd", p, kv[j, 1, :a])
        t += a - b
    if op == "attn":
        return {"out": out}
    # rows behind the last sequence are read at slot 0: its value is the cache's own there
    rest = room - len(slots)
    first = s["pages"][0, :, :, 0].double() * s["scales"][0, :, :, 0].double()[..., None]
    ids, kept = values
    if rest and bool((ids == 0).any()):
        first = kept[0, 0]
    pad = first[None].expand(rest, -1, -1, -1)
    return {"out": out, "table": None, "slot_map": None, "k": torch.cat([k, pad[:, :, 0]]), "v": torch.cat([v, pad[:, :, 1]])}
