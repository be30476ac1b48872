"""Attention over the 8-bit cache where a softmax has a strong first key and a long tail.

A first key far above many others (an attention sink), whose value is next to nothing, leaves the result to a tail of weights that
are each below any fixed step relative to the largest, and that matter together.  Tolerances do not grow with the number of
keys; `_bounds` derives them from the weights themselves.
"""
import ctypes as C

import pytest
import torch

from small_llm_b200 import kv8

from .test_gpu_kv8 import BLOCK, PAGE, ceil, check_attention, gen, setup_attention

pytestmark = pytest.mark.gpu
UNIT = 32                                        # keys whose weights the general form takes relative to their own largest
PARTS = {torch.bfloat16: 2.0 ** -16, torch.float32: 2.0 ** -36}


def sink_cache(keys, h, d, gap, spread, seed):
    """One sequence's cache and a query of ones: key 0 stands `gap` nats above the others (deviation `spread` among them), its
    value is 0, and the others' values have mean 0.5 and deviation 1."""
    g = gen(seed)
    n = ceil(keys, PAGE)
    ks = gap / (100 * d ** 0.5)                  # a score is ks * (mean integer) * sqrt(d)
    k = torch.full((n * PAGE, d), -50.0, device="cuda") + torch.randn(n * PAGE, 1, device="cuda", generator=g) * spread / (ks * d ** 0.5)
    k[0] = 50.0
    v = 0.5 + torch.randn(n * PAGE, d, device="cuda", generator=g)
    v[0] = 0.0
    vs = float(v.abs().max()) / 127
    pages = torch.stack([k.round().clamp(-127, 127), (v / vs).round()]).to(torch.int8).view(2, n, PAGE, d).transpose(0, 1)
    pages = pages[:, None].expand(n, h, 2, PAGE, d).contiguous()
    scales = torch.empty(n, h, 2, PAGE // BLOCK, device="cuda")
    scales[:, :, 0], scales[:, :, 1] = ks, vs
    return pages, scales


def _bounds(q, pages, scales, pos, dtype, prompt):
    """The definition in 64 bits for a sequence in pages 0, 1, ..., query row by query row, and what a row may be off by.

    scores: a score z carries at most (4 + d) half steps of fp32 of the sum of its terms' magnitudes (the query's split, the products,
    their sum), the same relative error of its weight, and as much again in the denominator; ex2 adds 2^-22 to each.
    weights of the product with V: the general form holds 32 of them as multiples of PARTS times the largest of the 32 (half a multiple
    off), the prompt form as fp16, 2^-11 of the weight, or 2^-32 of the largest weight of the row (half a step of fp16's smallest, 2^-25, with
    the largest at 2^7 or more).
    sums: fp32, 32 to 64 keys at a time, then chunk by chunk: a random walk of at most keys / 32 roundings, of which no more than
    64 half steps are granted."""
    h, d = pages.shape[1], pages.shape[4]
    x = pages.double().view(-1, h, 2, 4, BLOCK, d) * scales.double()[..., None, None]
    x = x.permute(1, 2, 0, 3, 4, 5).reshape(h, 2, -1, d)
    want, tol = [], []
    for t, p in enumerate(pos.tolist()):
        k, v = x[:, 0, :p + 1], x[:, 1, :p + 1]
        qt = q[t].double().view(h, -1, d)
        z = torch.einsum("hgd,hkd->hgk", qt, k) * d ** -0.5
        mag = torch.einsum("hgd,hkd->hgk", qt.abs(), k.abs()) * d ** -0.5
        w = torch.softmax(z, -1)
        o = torch.einsum("hgk,hkd->hgd", w, v)
        top = v.abs().amax((1, 2))[:, None]
        u = 2.0 ** -24
        rel = float(mag.max()) * (4 + d) * u + 2.0 ** -22 + 64 * u
        heard = torch.einsum("hgk,hkd->hgd", w, v.abs())
        if prompt:
            part = 2.0 ** -11 * heard + (p + 1) * 2.0 ** -32 * w.amax(-1, keepdim=True) * top[..., None]
        else:
            pad = torch.nn.functional.pad(w, (0, -(p + 1) % UNIT)).unflatten(-1, (-1, UNIT))
            part = (pad.amax(-1) * UNIT).sum(-1, keepdim=True) * PARTS[dtype] * top[..., None]
        tol.append(2 * rel * heard + part + o.abs() * (2.0 ** -8 if dtype == torch.bfloat16 else u))
        want.append(o)
    return torch.stack(want).flatten(1, 2), torch.stack(tol).flatten(1, 2)


def workspace(q, pages, scales, table, seq, pos, cu, max_new, max_len):
    need = C.c_uint64()
    n, heads, d = q.shape
    a = kv8._pack_attn(q.data_ptr(), torch.empty_like(q).data_ptr(), heads * d, heads * d, table.data_ptr(), seq.data_ptr(), pos.data_ptr(), cu.data_ptr() if cu is not None else 0, 0,
                       n, *table.shape, heads, max_new, max_len, kv8._ROWS[q.dtype], 0.0)
    assert kv8._lib().sllm_k_attn_kv8_workspace(kv8._layer(pages, scales)[0], a, C.byref(need)) == 0
    return need.value


@pytest.mark.parametrize("gap", [7.0, 10.6, 14.0, 17.0])
@pytest.mark.parametrize("keys,spread", [(2048, 0.0), (8192, 1.0), (32768, 0.0), (32768, 0.5)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_with_a_strong_first_key(dtype, d, keys, spread, gap):
    """Enough sequences (of the same pages) that the keys of a row are not cut, and a few, which are."""
    h = 2
    pages, scales = sink_cache(keys, h, d, gap, spread, seed=keys)
    i32 = dict(dtype=torch.int32, device="cuda")
    for n in (600, 3):
        table = torch.arange(pages.shape[0], **i32)[None].expand(n, -1).contiguous()
        seq = torch.arange(n, **i32)
        pos = keys - 1 - (torch.arange(n, **i32) % 3) * 17
        q = torch.ones(n, h, d, dtype=dtype, device="cuda")
        if n > 3:
            assert workspace(q, pages, scales, table, seq, pos, None, 1, keys) == 0
        got = kv8.attention(q, pages, scales, table, seq, pos, max_new=1, max_len=keys)
        want, tol = _bounds(q[:3], pages, scales, pos[:3], dtype, False)
        err = (got[:3].double() - want).abs()
        assert bool((err <= tol).all()), (n, float((err / tol).max()), float((err / want.abs().clamp(min=1e-3)).max()))
        for i in range(3):                                                   # rows of one length are one result
            same = got[i::3]
            assert torch.equal(same, same[:1].expand_as(same))


@pytest.mark.parametrize("gap", [7.0, 10.6, 14.0, 17.0])
@pytest.mark.parametrize("keys,spread", [(2048, 0.0), (32768, 0.0), (32768, 0.5), (131072, 0.0)])
@pytest.mark.parametrize("d", [64, 128])
def test_prompts_with_a_strong_first_key(d, keys, spread, gap):
    pages, scales = sink_cache(keys, 1, d, gap, spread, seed=keys)
    i32 = dict(dtype=torch.int32, device="cuda")
    for n in (160, 1):                                                       # sequences of the same pages: uncut, and cut where they are few
        new = 130
        table = torch.arange(pages.shape[0], **i32)[None].expand(n, -1).contiguous()
        seq = torch.arange(n, **i32).repeat_interleave(new)
        pos = (keys - new + torch.arange(new, **i32)).repeat(n)
        cu = torch.arange(n + 1, **i32) * new
        q = torch.ones(n * new, 1, d, dtype=torch.bfloat16, device="cuda")
        if n > 1:
            assert workspace(q, pages, scales, table, seq, pos, cu, new, keys) == 0
        got = kv8.attention(q, pages, scales, table, seq, pos, cu, max_new=new, max_len=keys)
        for t in (0, 5, 127, 128, 129):
            want, tol = _bounds(q[t:t + 1], pages, scales, pos[t:t + 1], torch.bfloat16, True)
            err = (got[t:t + 1].double() - want).abs()
            assert bool((err <= tol).all()), (n, t, float((err / tol).max()), float((err / want.abs().clamp(min=1e-3)).max()))
        assert torch.equal(got, got[:new].repeat(n, 1, 1))


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_near_the_largest_number(dtype, d):
    """Two keys of one score whose values are 2^126 and less: their mean, not infinity."""
    pages, scales = kv8.empty_cache(1, 1, d)
    pages[0, 0, 1, 0], pages[0, 0, 1, 1] = 127, 64
    scales[0, 0, 1, 0] = 2.0 ** 119
    i32 = dict(dtype=torch.int32, device="cuda")
    got = kv8.attention(torch.ones(1, 1, d, dtype=dtype, device="cuda"), pages, scales, torch.zeros(1, 1, **i32), torch.zeros(1, **i32), torch.ones(1, **i32), max_new=1)
    assert bool(((got.double() / (95.5 * 2.0 ** 119) - 1).abs() <= (2.0 ** -8 + 2.0 ** -15 if dtype == torch.bfloat16 else 2.0 ** -20)).all())


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_queries_near_the_largest_and_the_smallest_number(dtype, d):
    """Query values up to the type's largest, and near its smallest normal one, under a softmax scale that undoes them."""
    for size, scale in ((torch.finfo(dtype).max, 1.2e-38), (2.0 ** -120, 2.0 ** 118)):
        q, pages, scales, table, seq, pos, cu = setup_attention([300, 40], [60, 60], 1, 2, d, dtype, seed=24)
        scales[:, :, 0] *= 0.25
        x = torch.rand(q.shape, device="cuda", generator=gen(25)) * 2 - 1
        x[:, :, 3] = torch.sign(x[:, :, 3])
        q = (x.double() * size).to(dtype)
        assert bool(torch.isfinite(q).all())
        for kw in (dict(max_new=1), dict(cu_tok=cu)):
            check_attention((q, pages, scales, table, seq, pos, cu), dtype, scale=scale, max_len=360, **kw)


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scores_of_hundreds(dtype, d):
    """Two keys of nearly the same large score, which the query reaches by different values, 129 / 256 and 131 / 256 beside a largest of 1:
    a rounding of the query in steps that are not a power of two moves the scores apart."""
    a, b = d // 2 * 100 * 129, (d // 2 - 1) * 131
    kb = round(a / b)
    q = torch.full((1, 1, d), 131 / 256, device="cuda")
    q[..., 1::2], q[..., 0] = 129 / 256, 1.0
    pages, scales = kv8.empty_cache(1, 1, d)
    pages[0, 0, 0, 0, 1::2], pages[0, 0, 0, 1, 2::2] = 100, kb
    pages[0, 0, 1, 0], pages[0, 0, 1, 1] = 127, -127
    scales[0, 0, 0], scales[0, 0, 1] = 400 * 256 * d ** 0.5 / a, 1 / 127
    i32 = dict(dtype=torch.int32, device="cuda")
    args = (q.to(dtype), pages, scales, torch.zeros(1, 1, **i32), torch.zeros(1, **i32), torch.ones(1, **i32), torch.tensor([0, 1], **i32))
    for kw in (dict(max_new=1), dict(cu_tok=args[6])):
        check_attention(args, dtype, **kw)


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_random_scores_of_hundreds(dtype, d):
    """Scores so large that a rounding of the queries themselves, beyond their type's, would show in the weights."""
    q, pages, scales, table, seq, pos, cu = setup_attention([300, 40, 131, 200, 77, 260], [1] * 6, 2, 64, d, dtype, seed=26, sharp=6.0)
    scales[:, :, 0] *= 8
    for kw in (dict(max_new=1), dict(cu_tok=cu)):
        check_attention((q, pages, scales, table, seq, pos, cu), dtype, max_len=301, **kw)
