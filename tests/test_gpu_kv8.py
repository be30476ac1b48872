"""The 8-bit KV cache's operators against plain implementations in 64 bits (small sizes, edge cases, refusals).

Tolerances.  Integers, scales and lists are compared exactly.  Attention in fp32 is held to `_tol`, from the arithmetic: a score in
units of log2 carries a relative error of about 4 half steps (the split query and three products) plus the accumulation of
head_dim terms, and as an exponent turns it into a relative error of its weight; weights add the exponential's 2 units in the
last place and the split's 2^-22; sums of n terms add n half steps at most.  The sum is over weights that add up to one, so all of
it is relative to the largest value.  bf16 adds half a step of its own, eps / 2 = 2^-8 of the value; and its form for prompts rounds
each weight to fp16 before the product with V: half a step, eps / 2 = 2^-11 of the weight, where the denominator keeps the
unrounded one.  sum_j 2^-11 p_j |v_j| / sum_j p_j is at most 2^-11 of the largest value.  (Weights below fp16's normal range are
off by 2^-25 absolutely, with the largest at 1 or more: the sums' term covers that.)
"""
import itertools
import math

import numpy as np
import pytest
import torch

from small_llm_b200 import kv8

pytestmark = pytest.mark.gpu
PAGE, BLOCK = 64, 16
HEADS = [(2, 1, 64), (3, 1, 16), (2, 2, 32), (2, 4, 128), (1, 8, 64), (1, 12, 64), (1, 3, 128), (5, 5, 32)]
TYPES = [torch.float32, torch.bfloat16]


def ceil(a, b):
    return -(-a // b)


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


# ---- tables --------------------------------------------------------------------------------------------------------

def plain_tables(before, after, table, ring, pool_in, room):
    """The definition, sequence by sequence."""
    n, width = len(before), len(table[0])
    head, free = pool_in
    give_at, take, give, entries = 0, 0, 0, []
    table, ring, old_ring = [list(r) for r in table], list(ring), list(ring)
    for b, a in zip(before, after):
        if b < 0 or a < 0 or max(a, b) > width * PAGE:
            return None, 1
        take += max(0, ceil(a, PAGE) - ceil(b, PAGE))
        give += max(0, ceil(b, PAGE) - ceil(a, PAGE))
    if not 0 <= head < len(ring) or not 0 <= free <= len(ring) or free + give > len(ring):
        return None, 1
    if take > free or sum(max(0, a - b) for b, a in zip(before, after)) > room:
        return None, 4
    taken, cu = 0, [0]
    for i, (b, a) in enumerate(zip(before, after)):
        for p in range(ceil(b, PAGE), ceil(a, PAGE)):
            table[i][p] = old_ring[(head + taken) % len(ring)]
            taken += 1
        for p in range(ceil(a, PAGE), ceil(b, PAGE)):
            ring[(head + free + give_at) % len(ring)] = table[i][p]
            give_at += 1
        entries += [(i, p, table[i][p // PAGE] * PAGE + p % PAGE) for p in range(b, a)]
        cu.append(len(entries))
    return (table, ring, [(head + taken) % len(ring), free - taken + give, len(entries), 0], cu, entries), 0


class Tables:
    def __init__(self, n, width, n_pages, room, head=0):
        d = dict(dtype=torch.int32, device="cuda")
        self.table = torch.full((n, width), -7, **d)
        self.ring = torch.randperm(n_pages, device="cuda", generator=gen(n_pages)).to(torch.int32)
        self.pool = [torch.tensor([head, n_pages, 0, 0], device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")]
        self.cu, self.seq, self.pos = (torch.full((k,), 99, **d) for k in (n + 1, room, room))
        self.slot = torch.full((room,), 99, dtype=torch.int64, device="cuda")

    def step(self, before, after):
        b, a = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (before, after))
        want, code = plain_tables(before, after, self.table.tolist(), self.ring.tolist(), self.pool[0].tolist()[:2], self.seq.numel())
        had = self.table.clone(), self.ring.clone()
        kv8.block_tables(b, a, self.table, self.ring, *self.pool, self.cu, self.seq, self.pos, self.slot)
        room = self.seq.numel()
        if code:
            assert self.pool[1].tolist() == self.pool[0].tolist()[:2] + [0, code]
            assert torch.equal(self.table, had[0]) and torch.equal(self.ring, had[1])
            assert self.cu.tolist() == [0] * (len(before) + 1)
            entries = []
        else:
            table, ring, pool, cu, entries = want
            assert self.pool[1].tolist() == pool and self.cu.tolist() == cu
            assert self.table.tolist() == table and self.ring.tolist() == ring
        entries = entries + [(-1, -1, -1)] * (room - len(entries))
        assert list(zip(self.seq.tolist(), self.pos.tolist(), self.slot.tolist())) == entries
        self.pool.reverse()
        return code


@pytest.mark.parametrize("n,width,n_pages,room,most", [(1, 4, 5, 64, 200), (7, 9, 40, 300, 500), (33, 5, 90, 2100, 250), (300, 3, 500, 3000, 150), (1500, 2, 2500, 4000, 100),
                                                      (300, 3, 900, 30000, 150), (1500, 2, 2500, 90000, 100)])
def test_tables_over_many_steps(n, width, n_pages, room, most):
    """Growth, truncation, release, reuse of pages round the ring, refused steps in between: every step against the definition."""
    r = np.random.RandomState(n)
    t = Tables(n, width, n_pages, room, head=n_pages - 1)
    lens, codes = [0] * n, set()
    for step in range(14):
        kind = r.randint(0, 5, n)
        after = [min(width * PAGE, [x + 1, x, x + r.randint(0, most), r.randint(0, x + 1), 0][k]) for x, k in zip(lens, kind)]
        if step == 6:
            after[-1] = width * PAGE + 1
        if step == 9:
            after[0] = -1
        code = t.step(lens, after)
        codes.add(code)
        if code == 0:
            lens = after
        else:
            assert step in (6, 9) or code == 4
    assert 1 in codes and (0 in codes or room < n * most // 5)


@pytest.mark.parametrize("before,after,code", [
    ([0], [0], 0), ([0], [1], 0), ([63], [64], 0), ([64], [65], 0), ([0], [256], 0), ([0], [257], 1), ([64], [0], 0), ([65], [64], 0), ([1], [63], 0),
    ([0, 0, 0], [0, 5, 0], 0), ([0, 70, 0], [0, 70, 0], 0), ([100, 0], [0, 256], 0), ([0, 0], [256, 256], 4), ([0, 0], [150, 151], 4)])
def test_tables_at_the_borders(before, after, code):
    t = Tables(len(before), 4, 7, 300)
    if any(before):
        assert t.step([0] * len(before), before) == 0
    assert t.step(before, after) == code


def test_tables_at_the_largest_counts():
    n = kv8.MAX_SEQS
    t = Tables(n, 2, 2 * n, 1024)
    assert t.step([0] * n, [1 if i % 8 == 0 else 0 for i in range(n)]) == 0
    assert t.step([1 if i % 8 == 0 else 0 for i in range(n)], [0] * n) == 0
    t = Tables(2, 40, 100, 0)                      # no room for entries: only what needs none
    assert t.step([0, 0], [0, 0]) == 0 and t.step([0, 0], [1, 0]) == 4
    long = Tables(2, 1600, 1700, 70000)
    assert long.step([0, 0], [65536, 17]) == 0 and long.step([65536, 17], [65537, 0]) == 0


def test_tables_with_contradicting_counters():
    for pool in ([-1, 3], [8, 3], [0, 9], [0, -1]):
        t = Tables(1, 4, 8, 64)
        t.pool[0][:2] = torch.tensor(pool)
        assert t.step([0], [10]) == 1
    t = Tables(1, 4, 8, 64)                        # more pages given back than the pool can hold
    t.table[:] = 0
    assert t.step([200], [0]) == 1


# ---- append and read -----------------------------------------------------------------------------------------------

def plain_append(pages, scales, k, v, slots):
    """The definition in 64 bits, block by block, on copies in host memory."""
    pages, scales = pages.cpu().numpy().copy(), scales.cpu().numpy().copy()
    x = np.stack([k.double().cpu().numpy(), v.double().cpu().numpy()], 2)        # [n][H][2][hd]
    runs = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages.shape[0] * PAGE:
            runs.setdefault(s // BLOCK, []).append((t, s % BLOCK))
    for b, rows in runs.items():
        page, at = b // 4, (b % 4) * BLOCK
        off = rows[0][1]
        assert [o for _, o in rows] == list(range(off, off + len(rows)))
        for h in range(pages.shape[1]):
            for w in range(2):
                new = x[[t for t, _ in rows], h, w]
                old = scales[page, h, w, b % 4] if off else np.float32(0)
                top = np.float32(np.abs(new).max())
                s = np.float32(top / np.float32(127))
                if top > 0:
                    s = max(s, np.float32(2.0 ** -126))
                s = np.float32(np.nan) if np.isnan(old) or not np.isfinite(new).all() else max(s, old)
                blk = pages[page, h, w, at:at + BLOCK]
                if off and s != old:
                    blk[:off] = 0 if np.isnan(s) else np.rint(blk[:off].astype(np.float64) * np.float64(old) / np.float64(s))
                blk[off:off + len(rows)] = 0 if np.isnan(s) else np.rint(new / np.float64(s)) if s > 0 else 0
                scales[page, h, w, b % 4] = s
    return pages, scales


def check_append(k, v, slots, pages, scales):
    wp, ws = plain_append(pages, scales, k, v, slots)
    kv8.append(k, v, slots, pages, scales)
    assert np.array_equal(scales.cpu().numpy(), ws, equal_nan=True)
    assert np.array_equal(pages.cpu().numpy(), wp)
    kk, vv = kv8.read(slots, pages, scales)
    live = ((slots >= 0) & (slots < pages.shape[0] * PAGE)).cpu().numpy()
    s = np.where(live, slots.cpu().numpy(), 0)
    deq = wp[s // PAGE, :, :, s % PAGE].astype(np.float32) * ws[s // PAGE, :, :, s % PAGE // BLOCK][..., None]
    deq[~live] = 0
    assert np.array_equal(kk.cpu().numpy(), deq[:, :, 0], equal_nan=True) and np.array_equal(vv.cpu().numpy(), deq[:, :, 1], equal_nan=True)
    k16, v16 = kv8.read(slots, pages, scales, dtype=torch.bfloat16)
    assert torch.equal(k16.nan_to_num(7), kk.to(torch.bfloat16).nan_to_num(7)) and torch.equal(v16.nan_to_num(7), vv.to(torch.bfloat16).nan_to_num(7))


def random_cache(n_pages, h, d, seed):
    """Arbitrary integers and scales: what recycled pages hold."""
    g = gen(seed)
    return (torch.randint(-127, 128, (n_pages, h, 2, PAGE, d), device="cuda", generator=g, dtype=torch.int8),
            torch.rand(n_pages, h, 2, 4, device="cuda", generator=g) * 0.04)


@pytest.mark.parametrize("h,d", [(1, 16), (3, 32), (2, 64), (5, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_append_ragged_runs(h, d, dtype):
    """Runs of every length from every offset, blocks and pages crossed, dead entries in between, rows in a fused projection."""
    r = np.random.RandomState(d)
    pages, scales = random_cache(40, h, d, d)
    for step in range(4):
        slots, page = [], iter(r.permutation(40).tolist())
        for off, m in [(0, 1), (15, 1), (7, 1), (3, 13), (0, 64), (17, 47), (60, 4), (16, 16), (1, 33), (0, 16), (31, 2)]:
            p = next(page)
            slots += [p * PAGE + off + j for j in range(m)] + [-1] * r.randint(0, 3)
        slots += [40 * PAGE, -5, 10 ** 12]
        qkv = torch.randn(len(slots), 3 * h * d + 8, device="cuda", generator=gen(step)) * 10.0 ** (step - 2)
        qkv = qkv.to(dtype)[:, step * 2:step * 2 + 3 * h * d]               # steps 1, 3: bases that are not 16-byte aligned
        qkv = qkv.unflatten(1, (3 * h, d))
        check_append(qkv[:, h:2 * h], qkv[:, 2 * h:], torch.tensor(slots, device="cuda"), pages, scales)


def test_append_one_at_a_time_equals_growing_scales():
    """A decode run: each token in turn, scales growing, the earlier integers moved to the new scale each time."""
    pages, scales = random_cache(3, 2, 64, 5)
    x = torch.randn(2, 40, 2, 64, device="cuda", generator=gen(6)) * torch.logspace(-3, 3, 40, device="cuda")[:, None, None]
    for t in range(40):
        check_append(x[0, t:t + 1], x[1, t:t + 1], torch.tensor([PAGE + t], device="cuda"), pages, scales)


def test_append_rounds_exactly():
    """Quotients at and next to ties: x = (n + 1/2) s and its neighbours, for scales of many mantissas."""
    pages, scales = random_cache(8, 1, 64, 7)
    rows = []
    for i in range(32):
        s = np.float32(1 + i / 37) * np.float32(2.0) ** ((i % 9) * 25 - 100)
        top = np.float32(127) * s
        n = np.arange(-63, 63, 2, dtype=np.float32)
        x = ((n + np.float32(0.5)) * (top / np.float32(127))).astype(np.float32)
        x = np.concatenate([x[:63], [top]])
        rows.append(np.nextafter(x, np.float32(np.inf if i % 3 == 1 else -np.inf)) if i % 3 else x)
    k = torch.tensor(np.stack(rows), device="cuda")[:, None]
    slots = torch.arange(32, device="cuda") // 1 * 16 % (8 * PAGE)          # a block of its own for each row
    check_append(k, -k, slots, pages, scales)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_append_values_that_are_not_finite(value):
    pages, scales = random_cache(2, 2, 32, 9)
    k = torch.randn(20, 2, 32, device="cuda", generator=gen(1))
    k[5, 1, 3] = value
    slots = torch.arange(20, device="cuda") + 8
    check_append(k, k.clone().nan_to_num(0, 0, 0), slots, pages, scales)
    assert torch.isnan(scales[0, 1, 0, 0]) and torch.isfinite(scales[0, 0]).all() and torch.isfinite(scales[0, 1, 1]).all()
    check_append(k[:1], k[:1], torch.tensor([14], device="cuda"), pages, scales)      # stays until the block starts anew
    check_append(k[:1], k[:1], torch.tensor([0], device="cuda"), pages, scales)
    assert torch.isfinite(scales).all()


def test_append_extreme_magnitudes():
    pages, scales = random_cache(4, 1, 16, 11)
    for i, m in enumerate([0.0, 1e-45, 1e-38, 1.2e-38, 3.4e38, 1e-30]):
        k = torch.full((3, 1, 16), m, device="cuda") * torch.tensor([1.0, -0.5, 0.25], device="cuda")[:, None, None]
        check_append(k, -k, torch.arange(3, device="cuda") + i * 16, pages, scales)


# ---- attention -----------------------------------------------------------------------------------------------------

def setup_attention(lens_before, new, h, grp, d, dtype, seed, extra_rows=0, width_more=1, sharp=1.5):
    g = gen(seed)
    need = [ceil(b + n, PAGE) for b, n in zip(lens_before, new)]
    n_pages = sum(need) + 2
    pages, scales = random_cache(n_pages, h, d, seed)
    table = torch.full((len(need), max(need) + width_more), -1, dtype=torch.int32)
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    for i, k in enumerate(need):
        for j in range(k):
            table[i, j] = ids.pop()
    seq = [i for i, n in enumerate(new) for _ in range(n)] + [-1] * extra_rows
    pos = [b + j for b, n in zip(lens_before, new) for j in range(n)] + [-1] * extra_rows
    cu = list(itertools.accumulate(new, initial=0))
    i32 = dict(dtype=torch.int32, device="cuda")
    # scales are up to 0.04, integers up to 127: values of about 1.5
    q = (torch.randn(len(seq), h * grp, d, device="cuda", generator=g) * sharp).to(dtype)
    # what stands behind the last position is another owner's: scales there may be anything
    for i, (b, n) in enumerate(zip(lens_before, new)):
        for blk in range(ceil(b + n, BLOCK), need[i] * 4):
            scales[int(table[i, blk // 4]), :, :, blk % 4] = math.nan if blk % 2 else math.inf
    return q, pages, scales, table.cuda(), torch.tensor(seq, **i32), torch.tensor(pos, **i32), torch.tensor(cu, **i32)


def plain_attention(q, pages, scales, table, seq, pos, scale):
    n, heads, d = q.shape
    h = pages.shape[1]
    out = torch.zeros(n, heads, d, dtype=torch.float64, device="cuda")
    top = torch.zeros(n, heads, device="cuda", dtype=torch.float64)
    smax = 0.0
    for t, (s, p) in enumerate(zip(seq.tolist(), pos.tolist())):
        if s < 0 or p < 0:
            continue
        row = table[s, :p // PAGE + 1].long()
        ok = ((row >= 0) & (row < pages.shape[0])).repeat_interleave(PAGE)[:p + 1]
        row = row.clamp(0, pages.shape[0] - 1)
        x = pages[row].double().view(len(row), h, 2, 4, BLOCK, d) * scales[row].double()[..., None, None]
        x = x.permute(1, 2, 0, 3, 4, 5).reshape(h, 2, -1, d)[:, :, :p + 1][:, :, ok]
        if x.shape[2] == 0:
            continue
        z = torch.einsum("hgd,hkd->hgk", q[t].double().view(h, -1, d), x[:, 0]) * scale
        smax = max(smax, float(z.nan_to_num(0).abs().max()))
        out[t] = torch.einsum("hgk,hkd->hgd", torch.softmax(z, -1), x[:, 1]).reshape(heads, d)
        top[t] = x[:, 1].abs().amax((1, 2)).repeat_interleave(heads // h)
    return out, top[..., None], smax


def _tol(want, top, smax, keys, d, dtype):
    u = 2.0 ** -24
    weight = smax * 1.4427 * (8 + d) * u + 2 * 2.0 ** -22 + 2.0 ** -22      # scores (exponent), exponential, split
    tol = top * (2 * weight + 2 * keys * u)                                  # numerator and denominator
    return tol + (want.abs() * 2.0 ** -8 + top * 2.0 ** -11 if dtype == torch.bfloat16 else want.abs() * u)


def check_attention(args, dtype, scale=None, keys=None, **kw):
    q, pages, scales, table, seq, pos, cu = args
    sc = scale or q.shape[2] ** -0.5
    want, top, smax = plain_attention(q, pages, scales, table, seq, pos, sc)
    mark = torch.full(q.shape, 5.0, dtype=dtype, device="cuda")
    got = kv8.attention(q, pages, scales, table, seq, pos, scale=scale, out=mark, **kw)
    assert got is mark
    live = seq >= 0
    assert torch.equal(got[~live], torch.full_like(got[~live], 5.0))        # left as they were
    keys = keys or max(1, int(pos.max()) + 1)
    err = (got[live].double() - want[live]).abs()
    tol = _tol(want, top, smax, keys, q.shape[2], dtype)[live]
    assert bool((err <= tol).all()), (float((err / tol.clamp(min=1e-300)).max()), float(err.max()))
    return got


@pytest.mark.parametrize("h,grp,d", HEADS)
@pytest.mark.parametrize("dtype", TYPES)
def test_decode(h, grp, d, dtype):
    """Single tokens at every kind of length: ends of blocks, units, pages; one key; rows that attend nothing; padded rows."""
    before = [0, 1, 14, 15, 16, 30, 31, 32, 47, 62, 63, 64, 127, 128, 191, 300, 511, 512, 777]
    a = setup_attention(before, [1] * len(before), h, grp, d, dtype, seed=d + grp, extra_rows=3)
    q, pages, scales, table, seq, pos, cu = a
    check_attention(a, dtype, max_new=1, max_len=778)
    check_attention(a, dtype, max_new=1, max_len=0, cu_tok=cu)
    check_attention(a, dtype, max_new=1, max_len=33)                         # a wrong bound costs time, not results
    check_attention(a, dtype, max_new=0, max_len=1 << 20, cu_tok=cu)
    pos[4] = -1                                                              # attends nothing: zeros
    got = check_attention(a, dtype, max_new=1, max_len=778)
    assert float(got[4].abs().max()) == 0.0


@pytest.mark.parametrize("h,grp,d", HEADS)
@pytest.mark.parametrize("dtype", TYPES)
def test_prompts_and_drafts(h, grp, d, dtype):
    """Runs of one to a few hundred tokens of several sequences in one list, from position 0 and behind a history, some empty."""
    before = [0, 5, 0, 64, 200, 33, 0, 1000]
    new = [1, 3, 129, 0, 70, 8, 2, 17]
    a = setup_attention(before, new, h, grp, d, dtype, seed=d + 7 * grp, extra_rows=5)
    check_attention(a, dtype, max_new=129, max_len=1017, cu_tok=a[6])
    check_attention(a, dtype, cu_tok=a[6])
    check_attention(a, dtype)                                                # no offsets: each token alone
    check_attention(a, dtype, max_new=2, max_len=10, cu_tok=a[6], scale=0.31)


@pytest.mark.parametrize("h,grp,d", [(1, 1, 64), (2, 4, 128), (1, 1, 16)])
@pytest.mark.parametrize("dtype", TYPES)
def test_long_rows_in_chunks(h, grp, d, dtype):
    a = setup_attention([9000, 4095, 10, 6500], [1, 1, 1, 1], h, grp, d, dtype, seed=3)
    check_attention(a, dtype, max_new=1, max_len=9001)
    b = setup_attention([5000, 130], [3, 5], h, grp, d, dtype, seed=4)
    check_attention(b, dtype, max_new=5, max_len=5003, cu_tok=b[6])


@pytest.mark.parametrize("h,grp,d", [(1, 1, 64), (2, 4, 128), (1, 8, 64), (1, 5, 128), (1, 20, 64), (2, 1, 128)])
def test_long_prompts(h, grp, d):
    """Several tiles of query rows and steps of keys: from position 0, behind histories, ends on and off every border."""
    a = setup_attention([0, 640, 1, 127], [300, 257, 128, 70], h, grp, d, torch.bfloat16, seed=d + grp)
    check_attention(a, torch.bfloat16, max_new=300, max_len=897, cu_tok=a[6])
    b = setup_attention([0, 3000], [64, 90], h, grp, d, torch.bfloat16, seed=d - grp, sharp=6.0)
    check_attention(b, torch.bfloat16, max_new=90, max_len=3090, cu_tok=b[6], scale=-0.2)


@pytest.mark.parametrize("n,grp,d", [(64, 16, 64), (65, 16, 128), (300, 32, 64), (1100, 64, 64)])
def test_prompts_of_many_sequences(n, grp, d):
    """Each way in which a block finds its tile: sorted, in a copy of the offsets, in the offsets themselves; empty sequences among them."""
    r = np.random.RandomState(n)
    new = [int(x) for x in r.choice([0, 1, 3, 5, 9] if n < 500 else [0, 0, 1, 2], n)]
    a = setup_attention([int(x) for x in r.randint(0, 200, n)], new, 1, grp, d, torch.bfloat16, seed=n)
    assert sum(new) * grp >= 40 * n                                          # enough rows for the tensor-core form
    check_attention(a, torch.bfloat16, max_new=9, max_len=210, cu_tok=a[6])


@pytest.mark.parametrize("h,grp,d", [(1, 1, 64), (2, 4, 128), (1, 3, 64)])
def test_prompts_behind_long_histories_in_chunks(h, grp, d):
    """Few query rows and many keys: the keys of a tile in chunks, of which short sequences have one and some rows attend none."""
    a = setup_attention([9000, 3, 2500, 1023, 1024], [70, 64, 130, 1, 66], h, grp, d, torch.bfloat16, seed=d + 3 * grp, extra_rows=2)
    for max_len in (9070, 0, 1500):
        check_attention(a, torch.bfloat16, max_new=130, max_len=max_len, cu_tok=a[6])
    q, pages, scales, table, seq, pos, cu = a
    pos[3], pos[10], pos[80] = -1, 20, -1
    scales[int(table[0, 30]), 0, 0, 1] = math.nan                            # shows from its first key on
    got = kv8.attention(q, pages, scales, table, seq, pos, cu, max_new=130, max_len=9070, out=torch.zeros_like(q))
    bad = torch.isnan(got).any(-1)[:, :grp].all(1).cpu()
    assert bad.tolist() == [i < 70 and i not in (3, 10) for i in range(len(seq))]
    assert float(got[3].abs().max()) == 0.0 and float(got[80].abs().max()) == 0.0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("order", [1, -1])
def test_prompts_with_scales_of_many_magnitudes(d, order):
    """Scales that grow, or fall, by 2^24 along the sequence, zeros among them: the running references move many times."""
    q, pages, scales, table, seq, pos, cu = setup_attention([100, 0], [200, 260], 2, 2, d, torch.bfloat16, seed=77)
    for i in range(2):
        for p in range(5):
            f = 2.0 ** (order * (6 * p - 12))
            scales[int(table[i, p])] = torch.rand(2, 2, 4, device="cuda", generator=gen(p)) * 0.02 * torch.tensor([1.0, f], device="cuda")[:, None]
    scales[int(table[0, 1]), 0] = 0.0
    scales[int(table[1, 0]), 1, 1] = 0.0
    for rows in (torch.bfloat16, torch.float32):
        check_attention((q.to(rows), pages, scales, table, seq, pos, cu), rows, max_new=260, max_len=300, cu_tok=cu)
        check_attention((q.to(rows), pages, scales, table, seq, pos, cu), rows, max_new=1, max_len=300)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_loud_values_that_nothing_attends(d):
    """Keys whose weight is next to nothing hold values 2^14 times the others': the result keeps the precision of what is attended."""
    for dtype, kw in ((torch.bfloat16, dict(max_new=1)), (torch.float32, dict(max_new=1)), (torch.bfloat16, dict(max_new=64, cu_tok=True))):
        q, pages, scales, table, seq, pos, cu = setup_attention([300, 300], [64, 64], 1, 2, d, dtype, seed=91)
        sign = torch.sign(q[:1, :1].float())
        q = (q.float().abs() * sign).to(dtype)                               # all rows point one way
        row = table[:, 1].long()
        pages[row, 0, 0] = (-90 * sign[0, 0]).to(torch.int8)                 # keys 64 .. 127 the other way
        scales[row, 0, 0] = 0.04
        scales[row, 0, 1] = 0.04 * 2.0 ** 14
        if kw.get("cu_tok") is not None:
            kw["cu_tok"] = cu
        want, _, _ = plain_attention(q, pages, scales, table, seq, pos, d ** -0.5)
        got = kv8.attention(q, pages, scales, table, seq, pos, max_len=364, **kw).double()
        assert float(want.abs().max()) < 20                                  # the loud ones are not heard
        # half a step of bf16 of the value, and 2^-9 of the attended values (at most 127 * 0.04) for the roundings of q, p and vs
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + 127 * 0.04 * 2.0 ** -9).all()), (dtype, kw.keys(), float((got - want).abs().max()))


def test_prompts_with_bad_pages_and_values_that_are_not_finite():
    q, pages, scales, table, seq, pos, cu = setup_attention([0, 0], [260, 150], 2, 2, 64, torch.bfloat16, seed=78)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    kw = dict(max_new=260, max_len=260)
    clean = kv8.attention(q, pages, scales, table, seq, pos, cu, **kw)
    scales[int(table[0, 3]), 1, 0, 1] = math.nan                             # keys 208 .. 223, kv head 1
    q2 = q.clone()
    q2[300, 2, 7] = math.nan
    q2[301, 0, 7] = math.inf
    got = kv8.attention(q2, pages, scales, table, seq, pos, cu, status=status, **kw)
    want = torch.zeros(410, 4, dtype=torch.bool)
    want[208:260, 2:] = True
    want[300, 2] = want[301, 0] = True
    assert torch.equal(torch.isnan(got).any(-1).cpu(), want) and torch.equal(got[~want.cuda()], clean[~want.cuda()]) and int(status) == 0
    scales[int(table[0, 3]), 1, 0, 1] = 0.01
    table[0, 1], table[1, 0] = -1, 1 << 30
    pos[5], pos[399] = -1, -7
    got = check_attention((q, pages, scales, table, seq, pos, cu), torch.bfloat16, cu_tok=cu, status=status, **kw)
    assert int(status) == 1 and float(got[5].abs().max()) == 0.0 and float(got[265].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_unaligned_rows(dtype):
    before, new = [70, 0, 130], [1, 40, 2]
    q, *rest = setup_attention(before, new, 2, 3, 64, dtype, seed=12)
    for shift in (0, 1, 8):
        wide = torch.zeros(q.shape[0], 6 * 64 + 130, dtype=dtype, device="cuda")
        view = wide[:, shift:shift + 384].unflatten(1, (6, 64))
        view.copy_(q)
        want = kv8.attention(q, *rest[:5], rest[5], max_new=40, max_len=132)
        into = torch.zeros(q.shape[0], 6 * 64 + 9, dtype=dtype, device="cuda")[:, shift:shift + 384].unflatten(1, (6, 64))
        got = kv8.attention(view, *rest[:5], rest[5], max_new=40, max_len=132, out=into)
        assert torch.equal(got, want)


def test_peaked_and_extreme_scores():
    """One key takes everything; scores of hundreds; query magnitudes from 1e-30 to 1e30 (with the softmax scale undoing them)."""
    for m in (1e-30, 1.0, 1e30):
        a = setup_attention([200, 700], [1, 1], 2, 1, 64, torch.float32, seed=21, sharp=8.0)
        q = a[0] * m
        check_attention((q,) + a[1:], torch.float32, max_new=1, max_len=701, scale=1.0 / m)


@pytest.mark.parametrize("d", [16, 64, 128])
def test_values_of_extreme_magnitude(d):
    """V scaled by a power of two scales the result by it, whatever the form; a block of zeros among them."""
    for dtype, kw in ((torch.float32, dict(max_new=1)), (torch.bfloat16, dict(max_new=1)), (torch.bfloat16, dict())):
        q, pages, scales, table, seq, pos, cu = setup_attention([300, 40], [60, 60], 1, 2, d, dtype, seed=23)
        scales[int(table[0, 1]), 0, 1, 2] = 0.0
        kw = dict(kw, max_len=360, **({} if kw else dict(cu_tok=cu)))
        base = kv8.attention(q, pages, scales, table, seq, pos, **kw).double()
        for e in (-104, -60, 60, 104):
            loud = scales.clone()
            loud[:, :, 1] *= 2.0 ** e
            got = kv8.attention(q, pages, loud, table, seq, pos, **kw).double() * 2.0 ** -e
            top = base.abs().amax(-1, keepdim=True)
            assert bool(((got - base).abs() <= top * (2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -18)).all()), (dtype, e)


def test_values_that_are_not_finite():
    """A NaN scale shows in the rows that attend its block and in no other; a NaN query in its own row."""
    a = setup_attention([100, 100, 15], [1, 1, 1], 2, 2, 64, torch.float32, seed=8)
    q, pages, scales, table, seq, pos, cu = a
    clean = kv8.attention(q, pages, scales, table, seq, pos, max_new=1, max_len=101)
    assert torch.isfinite(clean).all()
    scales[int(table[1, 0]), 1, 0, 2] = math.nan
    q2 = q.clone()
    q2[2, 3, 5] = math.nan
    for kw in (dict(max_new=1), dict(cu_tok=cu)):
        got = kv8.attention(q2, pages, scales, table, seq, pos, max_len=101, **kw)
        bad = torch.isnan(got).all(-1)
        want = torch.zeros(3, 4, dtype=torch.bool)
        want[1, 2:] = True                                                   # query heads 2, 3 attend kv head 1
        want[2, 3] = True
        assert torch.equal(bad.cpu(), want) and torch.equal(got[~bad], clean[~bad])
    scales[int(table[1, 0]), 1, 0, 2] = 0.01
    scales[int(table[1, 0]), 1, 1, 2] = math.nan
    assert torch.equal(torch.isnan(kv8.attention(q, pages, scales, table, seq, pos, max_len=101, max_new=1)).all(-1).any(0).cpu(), torch.tensor([False, False, True, True]))


def test_pages_outside_the_pool_are_not_attended():
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for grp, kw in ((1, dict(max_new=1)), (2, dict())):
        a = setup_attention([300, 150, 63], [1, 1, 1], 1, grp, 64, torch.float32, seed=30)
        q, pages, scales, table, seq, pos, cu = a
        check_attention(a, torch.float32, max_len=301, status=status, **kw)
        assert int(status) == 0
        table[0, 2], table[1, 0], table[2, 0] = -1, pages.shape[0], 1 << 30
        got = check_attention(a, torch.float32, max_len=301, status=status, **kw)
        assert int(status) == 1 and float(got[2].abs().max()) == 0.0
        status.zero_()
        seq[0] = 3                                                           # no such sequence: skipped
        mark = torch.full_like(q, 2.0)
        kv8.attention(q, pages, scales, table, seq, pos, out=mark, **kw)
        assert torch.equal(mark[0], torch.full_like(mark[0], 2.0))
        pos[1] = 1 << 30                                                     # behind the table's width: all of it
        kv8.attention(q, pages, scales, table, seq, pos, out=mark, **kw)
        assert torch.isfinite(mark[2]).all()


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes, with the pages in use at its end."""
    h, d = 8, 128
    per = h * 2 * PAGE * d
    n_pages = (1 << 32) // per + 20
    pages = torch.zeros(n_pages, h, 2, PAGE, d, dtype=torch.int8, device="cuda")
    scales = torch.zeros(n_pages, h, 2, 4, device="cuda")
    small_p, small_s = kv8.empty_cache(20, h, d)
    g = gen(44)
    k, v = torch.randn(2, 200, h, d, device="cuda", generator=g)
    slots = torch.arange(200, device="cuda")
    at = (n_pages - 20) * PAGE
    kv8.append(k, v, slots, small_p, small_s)
    kv8.append(k, v, slots + at, pages, scales)
    for x, y in zip(kv8.read(slots, small_p, small_s), kv8.read(slots + at, pages, scales)):
        assert torch.equal(x, y)
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(3, 2 * h, d, device="cuda", generator=g)
    seq = torch.zeros(3, dtype=torch.int32, device="cuda")
    pos = torch.tensor([199, 64, 0], dtype=torch.int32, device="cuda")
    for t in (torch.float32, torch.bfloat16):
        assert torch.equal(kv8.attention(q.to(t), small_p, small_s, table, seq, pos), kv8.attention(q.to(t), pages, scales, table + (n_pages - 20), seq, pos))


def test_results_do_not_depend_on_the_run():
    a = setup_attention([4000, 100, 2500], [1, 4, 70], 2, 2, 64, torch.bfloat16, seed=50)
    q, *rest, cu = a
    first = kv8.attention(q, *rest, cu, max_new=70, max_len=4001)
    for _ in range(5):
        assert torch.equal(first, kv8.attention(q, *rest, cu, max_new=70, max_len=4001))


# ---- a step ---------------------------------------------------------------------------------------------------------

class Step:
    """Tables, append, attention over one layer, as a serving loop keeps them."""

    def __init__(self, n, h, grp, d, dtype, width, n_pages, room):
        self.t = Tables(n, width, n_pages, room)
        self.h, self.grp, self.d, self.dtype = h, grp, d, dtype
        self.pages, self.scales = random_cache(n_pages, h, d, 1)
        self.scales.fill_(math.nan)                                          # nothing of a recycled page counts
        self.qkv = torch.zeros(room, h * grp + 2 * h, d, dtype=dtype, device="cuda")
        self.before = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.after = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.out = torch.zeros(room, h * grp, d, dtype=dtype, device="cuda")

    def launch(self, max_new, max_len):
        t, hq = self.t, self.h * self.grp
        kv8.block_tables(self.before, self.after, t.table, t.ring, *t.pool, t.cu, t.seq, t.pos, t.slot)
        kv8.append(self.qkv[:, hq:hq + self.h], self.qkv[:, hq + self.h:], t.slot, self.pages, self.scales)
        kv8.attention(self.qkv[:, :hq], self.pages, self.scales, t.table, t.seq, t.pos, t.cu, max_new=max_new, max_len=max_len, out=self.out)

    def check(self):
        t = self.t
        want, top, smax = plain_attention(self.qkv[:, :self.h * self.grp], self.pages, self.scales, t.table, t.seq, t.pos, self.d ** -0.5)
        live = t.seq >= 0
        err = (self.out[live].double() - want[live]).abs()
        assert bool((err <= _tol(want, top, smax, int(self.after.max()), self.d, self.dtype)[live]).all())


@pytest.mark.parametrize("h,grp,d,dtype", [(2, 1, 64, torch.bfloat16), (1, 4, 128, torch.bfloat16), (3, 1, 32, torch.float32)])
def test_steps_of_a_serving_loop(h, grp, d, dtype):
    """Prompts, decode, a truncation, a release and a new sequence in its place; pages come round the ring, and the attention of
    every step is that of rows read back from the cache."""
    r = np.random.RandomState(3)
    s = Step(5, h, grp, d, dtype, width=8, n_pages=26, room=512)
    lens = [0] * 5
    for step in range(12):
        after = [min(500, x + n) for x, n in zip(lens, [[130, 70, 1, 0, 17], [1] * 5, [1, 1, 60, 200, 1], [1] * 5][step % 4])]
        if step % 5 == 4:
            after[step % 3] = 0
        if step == 6:
            after[3] = max(0, lens[3] - 33)
        s.before.copy_(torch.tensor(lens))
        s.after.copy_(torch.tensor(after))
        s.qkv.copy_(torch.randn(s.qkv.shape, device="cuda", generator=gen(step)))
        s.launch(max_new=1 if step % 4 % 2 else 200, max_len=512)
        assert int(s.t.pool[1][3]) == 0
        s.check()
        s.t.pool.reverse()
        lens = after
        held = [p for i, x in enumerate(lens) for p in s.t.table[i, :ceil(x, PAGE)].tolist()]
        assert len(set(held)) == len(held) and len(held) + int(s.t.pool[0][1]) == 26


def test_captured_step_replayed_for_other_lengths_and_beside_another():
    """Two captured steps replayed at the same time on two streams, several times, with other lengths than at the capture, while
    eager calls run on a third."""
    steps = [Step(6, 2, 2, 64, torch.bfloat16, width=40, n_pages=260, room=96) for _ in range(3)]
    graphs = []
    for s in steps[:2]:
        s.launch(16, 2560)                                                   # warm-up: kernels are loaded before the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.launch(16, 2560)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    lens = [[0] * 6 for _ in steps]
    for rnd in range(8):
        for i, s in enumerate(steps):
            after = [x + 1 + (rnd * 7 + i * 3 + j) % 16 for j, x in enumerate(lens[i])]
            s.before.copy_(torch.tensor(lens[i]))
            s.after.copy_(torch.tensor(after))
            s.qkv.copy_(torch.randn(s.qkv.shape, device="cuda", generator=gen(100 * rnd + i)))
            lens[i] = after
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay() if i < 2 else steps[2].launch(16, 2560)
        torch.cuda.synchronize()
        for s in steps:
            assert int(s.t.pool[1][3]) == 0
            s.check()
            s.t.pool[0].copy_(s.t.pool[1])                                   # the captured call reads and writes the same two buffers


@pytest.mark.parametrize("captured", [False, True])
def test_paged_cache(captured):
    """Two layers through PagedCache, step by step or as one captured graph: every step's attention is that of fp64 over the rows
    that the cache stands for, refused steps change nothing, and all pages come back."""
    L, n, h, grp, d, room = 2, 4, 2, 2, 64, 160
    cache = kv8.PagedCache(L, n, 14, h, d, max_len=400, max_tok=room)
    after = torch.zeros(n, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(L, room, h * grp + 2 * h, d, dtype=torch.bfloat16, device="cuda")
    outs = [torch.zeros(room, h * grp, d, dtype=torch.bfloat16, device="cuda") for _ in range(L)]
    split = lambda x: (x[:, :h * grp], x[:, h * grp:h * grp + h], x[:, h * grp + h:])  # noqa: E731

    def step():
        cache.step(after)
        for i in range(L):
            q, k, v = split(qkv[i])
            cache.append(i, k, v)
            cache.attention(i, q, out=outs[i])

    graph = None
    if captured:
        step()                                                               # lengths are all zero: nothing happens but the loading of kernels
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
    lens = [0] * n
    for i, (want, code) in enumerate([([100, 1, 0, 30], 0), ([101, 2, 1, 31], 0), ([102, 3, 120, 0], 0), ([102, 3, 281, 1], 4), ([103, 4, 121, 401], 4), ([103, 4, 121, 449], 1),
                                      ([64, 4, 200, 60], 0),
                                      ([65, 150, 201, 0], 0), ([400, 150, 201, 0], 4), ([66, 151, 202, 90], 0), ([0, 0, 0, 0], 0)]):
        after.copy_(torch.tensor(want))
        qkv.copy_(torch.randn(qkv.shape, device="cuda", generator=gen(i)))
        graph.replay() if captured else step()
        assert cache.status() == code
        lens = want if code == 0 else lens
        assert cache.lens.tolist() == lens and cache.free_pages() == 14 - sum(ceil(x, PAGE) for x in lens)
        live = cache.tok_seq >= 0
        assert code == 0 or not bool(live.any())
        for j in range(L):
            q = split(qkv[j])[0]
            ref, top, smax = plain_attention(q, *cache.layers[j], cache.table, cache.tok_seq, cache.tok_pos, d ** -0.5)
            err = (outs[j][live].double() - ref[live]).abs()
            assert bool((err <= _tol(ref, top, smax, 400, d, torch.bfloat16)[live]).all())
    assert sorted(cache.ring.tolist()) == list(range(14))
    extra = cache.attention(0, split(qkv[0])[0])
    assert float(extra.float().abs().max()) == 0.0                           # an empty list


# ---- refusals ---------------------------------------------------------------------------------------------------------

def test_refusals():
    pages, scales = kv8.empty_cache(3, 2, 64)
    k = torch.zeros(4, 2, 64, device="cuda")
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    table, seq = torch.zeros(1, 2, **i32), torch.zeros(4, **i32)
    with pytest.raises(ValueError, match="both be"):
        kv8.append(k.half(), k.half(), slots, pages, scales)
    with pytest.raises(ValueError, match="both be"):
        kv8.append(k, k.bfloat16(), slots, pages, scales)
    with pytest.raises(ValueError, match="must be"):
        kv8.append(k[:, :1], k, slots, pages, scales)
    with pytest.raises(ValueError, match="contiguous"):
        kv8.append(k.transpose(0, 1).contiguous().transpose(0, 1), k, slots, pages, scales)
    with pytest.raises(ValueError, match="contiguous"):
        kv8.append(k[:1].expand(4, 2, 64), k, slots, pages, scales)
    with pytest.raises(ValueError, match="slot_map"):
        kv8.append(k, k, slots.int(), pages, scales)
    with pytest.raises(ValueError, match="scales"):
        kv8.append(k, k, slots, pages, scales[:2])
    with pytest.raises(ValueError, match="on cuda"):
        kv8.append(k.cpu(), k, slots, pages, scales)
    with pytest.raises(ValueError, match="pages"):
        kv8.read(slots, pages.float(), scales)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        kv8.attention(torch.zeros(4, 3, 64, device="cuda"), pages, scales, table, seq, seq)
    with pytest.raises(ValueError, match="q must be"):
        kv8.attention(torch.zeros(4, 2, 32, device="cuda"), pages, scales, table, seq, seq)
    with pytest.raises(ValueError, match="overlap"):
        kv8.attention(k, pages, scales, table, seq, seq, out=k)
    with pytest.raises(ValueError, match="cu_tok"):
        kv8.attention(k, pages, scales, table, seq, seq, seq[:1])
    with pytest.raises(ValueError, match="scale"):
        kv8.attention(k, pages, scales, table, seq, seq, scale=0.0)
    for fn in (lambda: kv8.append(k[:0], k[:0], slots[:0], pages, scales), lambda: kv8.read(slots[:0], pages, scales),
               lambda: kv8.attention(k[:0], pages, scales, table, seq[:0], seq[:0])):
        fn()                                                                 # nothing to do is not an error
    # the C entry itself: host memory and missing workspaces
    import ctypes as C
    lib, host = kv8._lib(), torch.zeros(4, 2, 64)
    c = kv8._layer(pages, scales)[0]
    r = kv8._pack_rows(host.data_ptr(), k.data_ptr(), slots.data_ptr(), 128, 128, 4, 1)
    assert lib.sllm_k_kv8_append(c, r, None) == 1 and b"current device" in lib.sllm_last_error(None)
    long = torch.zeros(1, 4000, **i32)
    a = kv8._pack_attn(k.data_ptr(), torch.empty_like(k).data_ptr(), 128, 128, long.data_ptr(), seq.data_ptr(), seq.data_ptr(), 0, 0, 4, 1, 4000, 2, 1, 0, 1, 0.0)
    need = C.c_uint64()
    assert lib.sllm_k_attn_kv8_workspace(c, a, C.byref(need)) == 0 and need.value > 0
    assert lib.sllm_k_attn_kv8(c, a, None, 0, None) == 1 and b"workspace" in lib.sllm_last_error(None)
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    assert lib.sllm_k_attn_kv8(c, a, ws.data_ptr(), need.value - 1, None) == 1
