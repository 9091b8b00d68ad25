"""attention_quant where the scales of a cache differ by much: what a row's output may depend on, and to how many bits.

A row's output is a function of the positions that it sees.  Nothing else in the request, however large, may show in it, and
among the positions that it sees a value counts by its share of the sum, not by the size of other values.
"""
import math

import pytest
import torch

from test_gpu_kv_quant import attend, paged_cache, quantised, rand, values

pytestmark = pytest.mark.gpu

F16, BF16 = 2.0 ** -11, 2.0 ** -8                       # a rounding to the type, relative


def wanted(q, kc, ks, vc, vs, slots, n, nh, nkv, hd):
    """Float64 attention of a request's last n positions' queries over what each of them sees, [n, nkv, group, hd], with what a
    tolerance needs: sum p |v|, the largest sum |q k| / sqrt(hd), the largest |score|, the largest share p vs 448 of one position."""
    k, v = values(kc[slots], ks[:, slots]), values(vc[slots], vs[:, slots])
    scale = vs[:, slots].double()                                              # [nkv, l]
    l = len(slots)
    qq = q.double().view(n, nkv, nh // nkv, hd)
    seen = torch.arange(l, device="cuda")[None] <= (l - n + torch.arange(n, device="cuda"))[:, None]
    hidden = ~seen[:, None, None]
    k, v, scale = (torch.nan_to_num(x, 0.0, 0.0, 0.0) for x in (k, v, scale))      # what is not finite is put where nobody looks
    s = torch.einsum("nhgd,lhd->nhgl", qq, k) / math.sqrt(hd)
    size = torch.einsum("nhgd,lhd->nhgl", qq.abs(), k.abs()) / math.sqrt(hd)
    p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    out = torch.zeros_like(qq)
    a = torch.zeros_like(qq)
    for i in range(n):                                                         # by row, so that hidden values cannot cancel anything
        m = l - n + i + 1
        out[i] = torch.einsum("hgl,lhd->hgd", p[i, ..., :m], v[:m])
        a[i] = torch.einsum("hgl,lhd->hgd", p[i, ..., :m], v[:m].abs())
    top = lambda x: x.masked_fill(hidden, 0.0).amax(-1, keepdim=True)          # noqa: E731
    share = top(p * scale[None, :, None, :] * 448.0)
    return out, a, top(size), top(s.abs()), share


def check(got, want, a, size, score, share, l, dtype, products=256):
    """A weight is rounded to f16 (F32: to two of them).  Its score is off by `products` additions, each by 2^-23 of at most
    sum |q k|, and by four roundings of 2^-24 of itself (the scale, the factor of its row, their product with the sum, the
    difference from the reference); numerator and denominator both feel it.  The exponential and the sums: 2^-16.
    A weight below f16's normal range is off by 2^-25 instead, the largest being at least 2^-1 (its reference is at most 2^10
    above it), so a position's by 2^-24 of the largest share.  Float32 and bf16 end at 2^-126."""
    weight = F16 + 2.0 * products * 2.0 ** -23 * size + 8.0 * 2.0 ** -24 * score + 2.0 ** -16
    slack = a * weight + l * 2.0 ** -24 * share + 2.0 ** -126
    err = (got.double().view(want.shape) - want).abs()
    limit = (BF16 if dtype == torch.bfloat16 else 2.0 ** -24) * want.abs() * 1.01 + slack
    assert got.isfinite().all()
    assert (err <= limit).all(), f"{(err / limit).max().item():.3g} times the tolerance, {(err > limit).sum().item()} of {err.numel()}"


@pytest.mark.parametrize("news", [1, 2, 3, 65])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_are_not_rounded_to_sixteen_bits(backend, hd, news):
    """Keys that are one code times a scale with a full float32 fraction, one dimension only, scores of up to 300: a rounding of
    code times scale to 16 bits would be off by 2^-11 of a score, a weight by a tenth of itself.  The sum has one term."""
    nh, nkv, block, l = 8, 1, 16, 900
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, [l], block, 400)
    g = torch.Generator().manual_seed(401)
    k = torch.zeros(l, hd)
    k[:, 5] = (torch.rand(l, generator=g) * 2 - 1) * 8
    kc[slots[0]], ks[:, slots[0]] = quantised(k.cuda(), nkv)
    q = torch.zeros(news, nh, hd)
    q[..., 5] = 300 / 8 * math.sqrt(hd) * (0.7 + 0.3 * torch.rand(news, nh, generator=g))
    q = q.view(news, -1).to(torch.bfloat16).cuda()
    out = attend(backend, q, kc, ks, vc, vs, table, [l], [news], nh, nkv, hd, block, most)
    check(out, *wanted(q, kc, ks, vc, vs, slots[0], news, nh, nkv, hd), l, torch.bfloat16, products=1)


@pytest.mark.parametrize("news", [1, 4, 200])
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_of_chunks_are_as_exact_as_single_ones(backend, hd, news):
    """The last token's row, asked for alone, among four drafts or with a chunk of 200.  Its error is its output's rounding to
    bf16 (root mean square 0.42 * 2^-8 of a value) and that of its weights to f16: 0.42 * 2^-11 of each, independently, so of
    the sum as well, 1/8 of the former, and sqrt(1 + 1/64) < 1.01.  Sums of float32 add nothing.  Of 2048 outputs' rounding
    errors the root mean square varies by 1 or 2 %; a second rounding of keys and values to 16 bits would add 7 % and more."""
    nh, nkv, block, l = 16, 4, 16, 1000
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, [l], block, 410)
    q = rand(news, nh * hd, seed=411, loud=False).to(torch.bfloat16)
    q[-1] = rand(1, nh * hd, seed=412, loud=False)[0].to(torch.bfloat16)
    out = attend(backend, q, kc, ks, vc, vs, table, [l], [news], nh, nkv, hd, block, most)[-1:]
    want = wanted(q[-1:], kc, ks, vc, vs, slots[0], 1, nh, nkv, hd)[0]
    err = torch.linalg.vector_norm(out.double().view(want.shape) - want)
    own = torch.linalg.vector_norm(want.float().to(torch.bfloat16).double() - want)
    assert err <= 1.04 * own, (err / own).item()


OUTLIERS = [2.0 ** 24, 2.0 ** 40, 2.0 ** 90, math.inf, math.nan]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("size", OUTLIERS)
@pytest.mark.parametrize("hd,news", [(64, 4), (128, 3), (64, 70), (128, 150), (96, 20)])
def test_positions_that_a_row_does_not_see_do_not_show(backend, hd, news, size, which, dtype):
    """The last position, which only the last token sees, has a scale that is larger than the others by `size`."""
    nh, nkv, block, l = 8, 2, 16, 300
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, [l], block, 420)
    (ks if which == "keys" else vs)[:, slots[0][-1]] *= size
    q = rand(news, nh * hd, seed=421, loud=False).to(dtype)
    out = attend(backend, q, kc, ks, vc, vs, table, [l], [news], nh, nkv, hd, block, most)
    want = wanted(q, kc, ks, vc, vs, slots[0], news, nh, nkv, hd)
    rows = slice(0, news - 1)
    check(out[rows], *(x[rows] for x in want), l, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,news", [(64, 1), (128, 1), (128, 4), (64, 70), (128, 150), (96, 2)])
@pytest.mark.parametrize("at,size,depth", [(0, 2.0 ** 30, 300.0), (37, 2.0 ** 45, 300.0), (399, 2.0 ** 30, 300.0), (500, 2.0 ** 60, 300.0),
                                           (250, 2.0 ** 29, 20.0), (0, 2.0 ** 40, 20.0), (699, 2.0 ** 20, 40.0)])
def test_large_values_count_by_their_share(backend, hd, news, at, size, depth, dtype):
    """A position that is seen by every row (the last one: by the last) has a value `size` times the others and a score `depth`
    below them: what it adds is e^-depth of it, nothing at 300 (2^-433), about as much as the others at 20 and 2^29."""
    nh, nkv, block, l = 8, 2, 16, 700
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, [l], block, 430)
    q = rand(news, nh * hd, seed=431, loud=False).view(news, nh, hd)
    q[..., 0] = 4.0
    k = rand(l, nkv * hd, seed=432, loud=False).view(l, nkv, hd)
    k[at, :, :] = 0.0
    k[at, :, 0] = -depth / 4.0 * math.sqrt(hd)
    q = q.view(news, -1).to(dtype)
    kc[slots[0]], ks[:, slots[0]] = quantised(k.view(l, -1), nkv)
    vs[:, slots[0][at]] *= size
    out = attend(backend, q, kc, ks, vc, vs, table, [l], [news], nh, nkv, hd, block, most)
    check(out, *wanted(q, kc, ks, vc, vs, slots[0], news, nh, nkv, hd), l, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,news", [(64, 1), (128, 4), (64, 70), (128, 150), (96, 2)])
@pytest.mark.parametrize("low,high", [(-20, 20), (-60, 60), (-120, -80), (60, 100)])
def test_scales_of_all_sizes(backend, hd, news, low, high, dtype):
    """Values whose scales are spread evenly over many powers of two, position by position."""
    nh, nkv, block, l = 8, 2, 16, 700
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, [l], block, 440)
    g = torch.Generator().manual_seed(441)
    vs[:, slots[0]] = torch.exp2(torch.rand(nkv, l, generator=g) * (high - low) + low).cuda()
    q = rand(news, nh * hd, seed=442, loud=False).to(dtype)
    out = attend(backend, q, kc, ks, vc, vs, table, [l], [news], nh, nkv, hd, block, most)
    check(out, *wanted(q, kc, ks, vc, vs, slots[0], news, nh, nkv, hd), l, dtype)


@pytest.mark.parametrize("hd,news", [(64, 1), (128, 4), (128, 50)])
def test_keys_of_all_sizes(backend, hd, news):
    """Large keys under small queries and the other way round: the scores are ordinary, their factors are not."""
    nh, nkv, block, l = 8, 2, 16, 300
    for e in (-100, -60, 60, 100):
        kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, [l], block, 450)
        ks[:, slots[0]] *= 2.0 ** e
        q = (rand(news, nh * hd, seed=451, loud=False) * 2.0 ** -e).to(torch.bfloat16)
        out = attend(backend, q, kc, ks, vc, vs, table, [l], [news], nh, nkv, hd, block, most)
        check(out, *wanted(q, kc, ks, vc, vs, slots[0], news, nh, nkv, hd), l, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd,news", [(64, 1), (128, 4), (64, 70), (128, 150), (96, 2)])
def test_scales_of_either_sign_and_of_zero(backend, hd, news, dtype):
    """A cache that something else has filled: a third of the scales negative, a fifth zero; one head's values all zero, which
    makes its rows zero; one head's below float32's normal range but for one."""
    nh, nkv, block, l = 8, 4, 16, 300
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, [l], block, 470)
    g = torch.Generator().manual_seed(471)
    for s in (ks, vs):
        pick = torch.rand(nkv, l, generator=g)
        s[:, slots[0]] *= torch.where(pick < 1 / 3, -1.0, torch.where(pick < 1 / 3 + 1 / 5, 0.0, 1.0)).cuda()
    vs[2, slots[0]] = 0.0
    vs[3, slots[0]] = 2.0 ** -130
    vs[3, slots[0][7]] = 2.0 ** -100
    q = rand(news, nh * hd, seed=472, loud=False).to(dtype)
    out = attend(backend, q, kc, ks, vc, vs, table, [l], [news], nh, nkv, hd, block, most)
    check(out, *wanted(q, kc, ks, vc, vs, slots[0], news, nh, nkv, hd), l, dtype)
    assert not out.view(news, nkv, -1)[:, 2].any()


@pytest.mark.parametrize("group,tokens", [(1, 65), (3, 11), (4, 33), (5, 27), (7, 19), (8, 17), (17, 5), (32, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_row_counts_that_end_inside_a_warp(backend, hd, group, tokens):
    """Rows (token x head of the group) that fill no whole warp of 32, beside a second request, with tokens behind the last: the
    rows past the end are left as they were."""
    nkv, block, lens, news = 2, 16, [200, 150], [tokens, 1]
    nh = group * nkv
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, lens, block, 460)
    q = rand(tokens + 3, nh * hd, seed=461, loud=False).to(torch.bfloat16)
    out = attend(backend, q, kc, ks, vc, vs, table, lens, news, nh, nkv, hd, block, most)
    check(out[:tokens], *wanted(q[:tokens], kc, ks, vc, vs, slots[0], tokens, nh, nkv, hd), lens[0], torch.bfloat16)
    check(out[tokens:tokens + 1], *wanted(q[tokens:tokens + 1], kc, ks, vc, vs, slots[1], 1, nh, nkv, hd), lens[1], torch.bfloat16)
    assert (out[tokens + 1:] == 7.0).all()
