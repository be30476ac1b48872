"""Scales of the 8-bit cache that are NaN or infinite: they show in the rows that attend their block and in no other."""
import math

import pytest
import torch

from small_llm_b200 import kv8

from .test_gpu_kv8 import BLOCK, setup_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
def test_prompts_with_a_block_that_is_not_finite(d, which):
    """A NaN scale shows in the rows that attend its block and in no other, whichever of K and V it belongs to."""
    q, pages, scales, table, seq, pos, cu = setup_attention([0, 0], [260, 150], 2, 2, d, torch.bfloat16, seed=78)
    kw = dict(max_new=260, max_len=260)
    clean = kv8.attention(q, pages, scales, table, seq, pos, cu, **kw)
    scales[int(table[0, 3]), 1, which, 1] = math.nan                         # keys 208 .. 223, kv head 1
    want = torch.zeros(410, 4, dtype=torch.bool, device="cuda")
    want[208:260, 2:] = True
    for form in (kw, dict(max_new=1, max_len=260)):
        base = clean if form is kw else None
        got = kv8.attention(q, pages, scales, table, seq, pos, cu, **form)
        assert torch.equal(torch.isnan(got).any(-1), want)
        if base is not None:
            assert torch.equal(got[~want], base[~want])


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [2, 13])
def test_rows_before_a_block_that_is_infinite(d, which, at):
    """An infinite scale (which append never writes, but a caller may) does not touch the rows that stand before its block."""
    q, pages, scales, table, seq, pos, cu = setup_attention([0, 0], [260, 150], 2, 2, d, torch.bfloat16, seed=79)
    for kw in (dict(max_new=260, max_len=260), dict(max_new=1, max_len=260)):
        clean = kv8.attention(q, pages, scales, table, seq, pos, cu, **kw)
        loud = scales.clone()
        loud[int(table[0, at // 4]), 0, which, at % 4] = math.inf
        got = kv8.attention(q, pages, loud, table, seq, pos, cu, **kw)
        same = torch.ones_like(got, dtype=torch.bool)
        same[at * BLOCK:260, :2] = False
        assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("h,grp,d", [(1, 1, 64), (2, 4, 128), (1, 3, 64)])
def test_prompts_in_chunks_with_a_block_that_is_not_finite(h, grp, d, which):
    q, pages, scales, table, seq, pos, cu = setup_attention([9000, 3, 2500, 1023, 1024], [70, 64, 130, 1, 66], h, grp, d, torch.bfloat16, seed=d + 3 * grp)
    pos[3], pos[10], pos[80] = -1, 20, -1
    scales[int(table[0, 30]), 0, which, 1] = math.nan
    for kw in (dict(max_new=130, max_len=9070), dict(max_new=130, max_len=1500), dict(max_new=1, max_len=9070)):
        got = kv8.attention(q, pages, scales, table, seq, pos, cu, **kw)
        bad = torch.isnan(got).any(-1)[:, :grp].all(1).cpu()
        assert bad.tolist() == [i < 70 and i not in (3, 10) for i in range(len(seq))]
        assert float(got[3].abs().max()) == 0.0 and float(got[80].abs().max()) == 0.0


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dtype,d,kw", [(torch.float32, 64, dict(max_new=1)), (torch.bfloat16, 64, dict(max_new=1)), (torch.bfloat16, 16, dict(max_new=1)), (torch.bfloat16, 128, dict()),
                                        (torch.float32, 128, dict())])
def test_infinite_values_show_where_they_are_attended(dtype, d, kw, which):
    q, pages, scales, table, seq, pos, cu = setup_attention([0], [150], 2, 2, d, dtype, seed=80)
    scales[int(table[0, 1]), 1, which, 2] = math.inf                         # keys 96 .. 111, kv head 1
    got = kv8.attention(q, pages, scales, table, seq, pos, None if kw else cu, max_len=150, **kw)
    odd = ~torch.isfinite(got).all(-1)
    assert not bool(odd[:96].any()) and not bool(odd[:, :2].any())
    # K: scores without end of both signs, of which one takes everything; all of one sign downwards may leave the rest
    assert bool(odd[111:, 2:].all()) if which else float(odd[111:, 2:].float().mean()) > 0.9
