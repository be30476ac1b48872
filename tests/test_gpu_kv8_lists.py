"""Lists that say nothing to do, or that contradict one another, in every form of the 8-bit cache's attention: rows alone, rows
of a cluster's chunks, chunks by way of the workspace, the prompt form whole and in chunks."""
import pytest
import torch

from small_llm_b200 import kv8

from .test_gpu_kv8 import BLOCK, PAGE, TYPES, check_attention, gen, setup_attention

pytestmark = pytest.mark.gpu
LOWEST = -2 ** 31


@pytest.mark.parametrize("far", [-2, LOWEST, LOWEST + 1, LOWEST + 5000])
@pytest.mark.parametrize("h,grp,d", [(1, 8, 64), (1, 1, 64), (2, 4, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_positions_far_below_zero(dtype, h, grp, d, far):
    """Rows that attend nothing get zeros however far below zero their position is, in full tiles (8 heads) and beside other rows."""
    a = setup_attention([9000, 4095, 10, 6500], [1, 1, 1, 1], h, grp, d, dtype, seed=3)
    a[5][0], a[5][2] = far, far
    for max_len in (9001, 1000):
        got = check_attention(a, dtype, max_new=1, max_len=max_len, keys=9001)
        assert float(got[0].abs().max()) == 0.0 and float(got[2].abs().max()) == 0.0
    b = setup_attention([9000, 3, 2500, 1023], [70, 64, 130, 8], h, grp, d, dtype, seed=5, extra_rows=2)
    b[5][:16] = far                                                          # whole tiles of the general form
    b[5][40], b[5][200] = far, far
    for kw in (dict(max_new=130, max_len=9070), dict(max_new=130, max_len=1500), dict()):
        got = check_attention(b, dtype, cu_tok=b[6], keys=9070, **kw)
        assert float(got[:16].abs().max()) == 0.0 and float(got[40].abs().max()) == 0.0
    b[5][70:264] = far                                                       # all rows of two sequences
    got = check_attention(b, dtype, cu_tok=b[6], keys=9070, max_new=130, max_len=9070)
    assert float(got[70:264].abs().max()) == 0.0


@pytest.mark.parametrize("h,grp,d", [(2, 1, 32), (2, 2, 64), (1, 4, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_tables_of_many_pages(dtype, h, grp, d):
    """A table wider than 8192 pages, most of it not in use, with lengths known and not known; integers down to -128."""
    a = setup_attention([700, 20, 4000], [1, 3, 40], h, grp, d, dtype, seed=d, width_more=9000)
    q, pages, scales, table, seq, pos, cu = a
    pages.masked_fill_(pages == -127, -128)
    assert table.shape[1] > 8192
    for kw in (dict(max_new=1, max_len=4040), dict(max_new=1), dict(cu_tok=cu, max_new=40, max_len=4040), dict(cu_tok=cu)):
        check_attention(a, dtype, keys=4040, **kw)


@pytest.mark.parametrize("h,grp,d", [(1, 1, 64), (2, 4, 128), (1, 8, 64), (1, 2, 16)])
@pytest.mark.parametrize("dtype", TYPES)
def test_entries_of_no_sequence_inside_a_run(dtype, h, grp, d):
    """With cu_tok too an entry whose tok_seq names no sequence, or another than the one in whose run it stands, is skipped and its row left
    as it was, however the keys are cut; the others are as if it attended nothing."""
    for before, new, lens in (([700, 0], [12, 5], (712, 0, 50)), ([9000, 3], [70, 64], (9070, 1500)), ([300, 20, 0], [140, 2, 200], (440,)), ([2000], [3], (2003,))):
        a = setup_attention(before, new, h, grp, d, dtype, seed=6)
        q, pages, scales, table, seq, pos, cu = a
        odd = {1: -1, 2: len(new), 5: -2 ** 31, 11: 1 if len(new) > 1 else -1, new[0] - 1: 2 ** 31 - 1}
        for max_len in lens:
            for max_new in (max(new), 2, 0):
                mixed = seq.clone()
                for t, s in odd.items():
                    if t < new[0]:
                        mixed[t] = s
                gone = mixed != seq
                want = kv8.attention(q, pages, scales, table, seq, pos.masked_fill(gone, -1), cu, max_new=max_new, max_len=max_len)
                got = kv8.attention(q, pages, scales, table, mixed, pos, cu, max_new=max_new, max_len=max_len, out=torch.full_like(q, 3.0))
                assert bool((got[gone] == 3.0).all())
                assert torch.equal(got[~gone], want[~gone])


def test_paged_cache_says_what_attention_found():
    cache = kv8.PagedCache(1, 2, 8, 2, 64, max_len=200, max_tok=130)
    cache.step(torch.tensor([100, 30], dtype=torch.int32, device="cuda"))
    x = torch.randn(130, 2, 64, device="cuda")
    cache.append(0, x, x)
    cache.attention(0, x)
    assert cache.status() == 0
    cache.table[0, 0] = 8                                                    # no such page
    cache.attention(0, x)
    assert cache.status() == 1 and cache.status() == 0                       # said once
    mine = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.attention(0, x, status=mine)
    assert int(mine) == 1 and cache.status() == 0


@pytest.mark.parametrize("scale", [0.0, 1e-46, -1e-60, 1e39, float("inf"), float("-inf"), float("nan")])
def test_softmax_scales_that_fp32_does_not_have(scale):
    """One that fp32 rounds to 0 would stand for the default scale."""
    q, pages, scales, table, seq, pos, cu = setup_attention([40], [1], 1, 1, 64, torch.float32, seed=9)
    with pytest.raises(ValueError, match="scale"):
        kv8.attention(q, pages, scales, table, seq, pos, scale=scale)
    tiny = kv8.attention(q, pages, scales, table, seq, pos, scale=1e-44)      # the smallest ones count: all keys alike
    assert float((tiny - kv8.attention(q * 0, pages, scales, table, seq, pos)).abs().max()) < 1e-5


def test_tokens_appended_one_at_a_time():
    """What a decode loop's cache stands for, against the rows themselves: each rounding of a row, under its first scale and under every
    scale that the block grew to while it held it, is off by half a step at most; and over many rows the root of the mean square is no
    more than that many independent roundings would leave."""
    n, h, d = 32 * BLOCK, 2, 64
    k, v = torch.randn(2, n, h, d, device="cuda", generator=gen(41))
    slots = torch.arange(n, device="cuda")
    pages, scales = kv8.empty_cache(n // PAGE, h, d)
    seen = torch.zeros(2, n, h, dtype=torch.float64, device="cuda")          # sum over the roundings of a row: half a step
    square = torch.zeros_like(seen)                                          # the same of step^2 / 12
    block = lambda t: scales[t // PAGE, :, :, t % PAGE // BLOCK].double().T  # noqa: E731
    for t in range(n):
        first = t % BLOCK == 0
        was = block(t).clone()
        kv8.append(k[t:t + 1], v[t:t + 1], slots[t:t + 1], pages, scales)
        now = block(t)
        assert first or bool((now >= was).all())
        for i in range(t // BLOCK * BLOCK, t + 1):
            moved = torch.ones_like(now) if i == t else (now != was).double()
            seen[:, i] += moved * now / 2
            square[:, i] += moved * now ** 2 / 12
    got = torch.stack(kv8.read(slots, pages, scales))
    err = got.double() - torch.stack([k, v]).double()
    assert bool((err.abs() <= seen[..., None] * (1 + 2.0 ** -20)).all())
    # 2 x 512 x 2 x 64 errors, nearly independent: the mean of their squares is known to better than 2 %
    assert float((err ** 2).mean()) <= 1.05 * float(square.mean())
    whole_p, whole_s = kv8.empty_cache(n // PAGE, h, d)                      # one call for all: rounded once
    kv8.append(k, v, slots, whole_p, whole_s)
    assert torch.equal(whole_s, scales)                                      # the scales do not depend on the cut, the integers do
    assert not torch.equal(whole_p, pages)
