"""Scaled rotary positions and the 8-bit KV cache on the GPU, against plain 64-bit forms.

Tolerances.  A rounding to a type is off by at most half a step of it: bf16 2^-8, f16 2^-11, f32 2^-24, E4M3 2^-4
of the value (2^-10 below 2^-6, in units of the scale).
"""
import math

import numpy as np
import pytest
import torch

from llm_rs_b200 import BackendError, CudaBackend, DType, RopeScaling, rope_frequencies

pytestmark = pytest.mark.gpu

KINDS = {torch.bfloat16: DType.BF16, torch.float32: DType.F32, torch.int32: DType.I32, torch.float8_e4m3fn: DType.E4M3,
         torch.uint8: DType.E4M3}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
PAD = -1                      # 0xFFFFFFFF: a padding token's slot


def buf(be, t):
    """A CUDA tensor [rows, row] as the buffer [row, rows]."""
    assert t.is_contiguous()
    return be.wrap(t.data_ptr(), list(t.shape[::-1]), KINDS[t.dtype], keepalive=t)


def ints(x):
    return torch.as_tensor(x, dtype=torch.int64).to(torch.int32).cuda()


def rand(*shape, seed=0, loud=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if loud:
        x = x * torch.where(torch.rand(shape[-1], generator=g) < 0.05, 6.0, 1.0)
    return x.cuda()


def quantised(x, heads):
    """The definition of the cache, in float32: codes [slots, row] as bytes, scales [heads, slots].  (448 as a tensor on the
    GPU: by a Python number torch multiplies by the reciprocal there, which is not the division of the definition.)"""
    h = x.float().view(x.shape[0], heads, -1)
    scale = (h.abs().amax(-1) / torch.tensor(448.0, device=x.device)).clamp_min(2.0 ** -126)
    codes = (h / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.reshape(x.shape).contiguous(), scale.t().contiguous()


def values(codes, scales):
    return codes.view(torch.float8_e4m3fn).float().double().view(codes.shape[0], scales.shape[0], -1) * scales.double().t()[..., None]


# ---- rotation ------------------------------------------------------------------------------------

def rotated(x, hd, pos, freq, mag, half_layout):
    """Float64 rotation of x [tokens, heads * hd]."""
    n = freq.numel()
    y = x.double().view(x.shape[0], -1, hd).clone()
    ang = pos.long().bitwise_and(0xFFFFFFFF).double()[:, None, None] * freq.double()
    a = y[..., :n].clone() if half_layout else y[..., 0:2 * n:2].clone()
    b = y[..., n:2 * n].clone() if half_layout else y[..., 1:2 * n:2].clone()
    ra, rb = mag * (a * ang.cos() - b * ang.sin()), mag * (a * ang.sin() + b * ang.cos())
    if half_layout:
        y[..., :n], y[..., n:2 * n] = ra, rb
    else:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = ra, rb
    return y.view(x.shape)


def rope_slack(x, hd, mag):
    """|x| of the other member of a pair is at most the head's largest: cosine, sine, their product with the magnitude, two
    products and a sum, each off by 2^-24, and an angle off by 2^-22 (2 pi in float32 over half a turn): 2^-20 of it."""
    h = x.double().abs().view(x.shape[0], -1, hd).amax(-1, keepdim=True)
    return (h * max(mag, 1.0) * 2.0 ** -20).expand(-1, -1, hd).reshape(x.shape)


ROPE_CASES = [  # heads, kv heads, head_dim, rotary, tokens
    (32, 8, 128, 128, 1), (4, 2, 128, 64, 37), (14, 2, 64, 64, 5), (3, 1, 80, 20, 9), (2, 1, 256, 256, 3), (8, 8, 64, 16, 130),
    (5, 1, 96, 96, 2), (1, 1, 6, 2, 4), (7, 7, 32, 24, 11), (40, 8, 128, 32, 300),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,rot,tokens", ROPE_CASES)
def test_rope_scaled(backend, nh, nkv, hd, rot, tokens, half, dtype):
    freq, mag = rope_frequencies(rot, 500000.0, RopeScaling.YARN, 8.0, 8192, 1.0, 32.0)
    freq = torch.from_numpy(freq).cuda()
    q, k = rand(tokens, nh * hd, seed=1).to(dtype), rand(tokens, nkv * hd, seed=2).to(dtype)
    pos = ints(torch.linspace(0, 131071, tokens).long())
    pos[-1] = 131071
    q_out, k_out = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    qi, ki = q.clone(), k.clone()
    torch.cuda.synchronize()
    b = [buf(backend, t) for t in (q_out, k_out, q, k, pos, freq, qi, ki)]
    backend.rope_scaled(*b[:6], hd, mag, half)
    backend.rope_scaled(b[6], b[7], b[6], b[7], b[4], b[5], hd, mag, half)               # in place
    backend.sync()
    for got, inplace, x in ((q_out, qi, q), (k_out, ki, k)):
        want = rotated(x, hd, pos, freq, mag, half)
        err = (got.double() - want).abs()
        assert (err <= HALF_STEP[dtype] * want.abs() * 1.01 + rope_slack(x, hd, mag)).all(), err.max()
        assert torch.equal(got, inplace)
        rest = (slice(None), slice(None), slice(rot, None))
        assert torch.equal(got.view(tokens, -1, hd)[rest], x.view(tokens, -1, hd)[rest])


def test_rope_positions_are_unsigned_and_far(backend):
    """Position 2^32 - 1: the fraction of the angle in float64 is still good to 2^-20 turns."""
    freq = torch.tensor([1.0, 0.125, 3e-7, 1.0 / 3.0], device="cuda")
    q, k = rand(3, 8, seed=3), rand(3, 8, seed=4)
    pos = ints([-1, 2 ** 31, 2 ** 31 - 1])
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    torch.cuda.synchronize()
    backend.rope_scaled(*[buf(backend, t) for t in (qo, ko, q, k, pos, freq)], 8)
    backend.sync()
    want = rotated(q, 8, pos, freq, 1.0, False)
    # the product rounds at 2^-53 of 2^32 radians here and in the plain form alike, once or twice each
    assert ((qo.double() - want).abs() <= rope_slack(q, 8, 1.0) + q.abs().max().item() * 2.0 ** -18).all()


# ---- writing and reading back ---------------------------------------------------------------------

def empty_cache(slots, heads, hd, fill=0x7F):
    """A cache nobody has initialised: NaN codes and NaN scales."""
    return torch.full((slots, heads * hd), fill, dtype=torch.uint8, device="cuda"), torch.full((heads, slots), math.nan, device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,hd,tokens,slots", [(8, 128, 1, 40), (2, 64, 33, 100), (1, 256, 5, 7), (3, 32, 70, 70), (4, 96, 17, 64),
                                                   (1, 2, 9, 20), (5, 80, 130, 400), (8, 128, 1000, 1500)])
def test_scatter_and_gather(backend, heads, hd, tokens, slots, dtype):
    """Bit for bit the definition; the slots that are not named keep every byte; read back: code * scale, rounded once."""
    x = rand(tokens, heads * hd, seed=5).to(dtype)
    x[0] *= 1e-30
    x[-1, :hd] = 0.0
    x[tokens // 2, -hd:] = torch.finfo(dtype).tiny / 4
    where = torch.randperm(slots, generator=torch.Generator().manual_seed(6))[:tokens]
    codes, scales = empty_cache(slots, heads, hd)
    src, slot = x, ints(where)
    torch.cuda.synchronize()
    cb, sb = buf(backend, codes), buf(backend, scales)
    backend.scatter_kv_quant(cb, sb, buf(backend, src), buf(backend, slot), tokens)
    out = torch.full((tokens, heads * hd), 7.0, dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    backend.gather_quant(buf(backend, out), cb, sb, buf(backend, slot), tokens)
    backend.sync()
    want_codes, want_scales = quantised(x, heads)
    where = where.cuda()
    assert torch.equal(codes[where], want_codes)
    assert torch.equal(scales[:, where], want_scales)
    others = torch.ones(slots, dtype=torch.bool, device="cuda")
    others[where] = False
    assert (codes[others] == 0x7F).all() and scales[:, others].isnan().all()
    back = values(want_codes, want_scales).view(tokens, -1)
    assert torch.equal(out, back.float().to(dtype))
    # and the cache is what was written, to half a step of E4M3 (and of the type it is read into)
    step = want_scales.t().double()[..., None].expand(-1, -1, hd).reshape(tokens, -1) * 2.0 ** -10
    err = (back - x.double()).abs()
    assert (err <= torch.maximum(x.double().abs() * 2.0 ** -4, step) * (1 + 2.0 ** -20)).all()


def test_values_that_are_not_finite(backend):
    """Their head row becomes NaN, its codes 0; the other heads of the token notice nothing."""
    x = rand(4, 2 * 64, seed=7)
    x[0, 3], x[1, 64], x[2, 127] = math.inf, math.nan, -math.inf
    codes, scales = empty_cache(4, 2, 64)
    slot = ints([0, 1, 2, 3])
    torch.cuda.synchronize()
    backend.scatter_kv_quant(buf(backend, codes), buf(backend, scales), buf(backend, x), buf(backend, slot), 4)
    backend.sync()
    bad = torch.tensor([[1, 0, 0, 0], [0, 1, 1, 0]], dtype=torch.bool, device="cuda")
    assert torch.equal(scales.isnan(), bad)
    want, _ = quantised(torch.where(x.isfinite(), x, 0.0), 2)
    ok = ~bad.t()[..., None].expand(-1, -1, 64).reshape(4, -1)
    assert torch.equal(codes[ok], want[ok]) and (codes[~ok] == 0).all()


def test_padding_tokens_and_slots_beyond_the_pool(backend):
    x = rand(4, 64, seed=8)
    codes, scales = empty_cache(5, 1, 64)
    torch.cuda.synchronize()
    cb, sb, xb = buf(backend, codes), buf(backend, scales), buf(backend, x)
    slot = ints([4, PAD, 0, PAD])
    torch.cuda.synchronize()
    backend.scatter_kv_quant(cb, sb, xb, buf(backend, slot), 4)
    backend.sync()                                                        # padding is no error
    want, _ = quantised(x, 1)
    assert torch.equal(codes[[4, 0]], want[[0, 2]]) and (codes[1:4] == 0x7F).all()
    before = codes.clone()
    slot = ints([5, 2 ** 31 - 1, -2, 1])
    torch.cuda.synchronize()
    backend.scatter_kv_quant(cb, sb, xb, buf(backend, slot), 4)
    with pytest.raises(BackendError) as e:
        backend.sync()
    assert e.value.code == -4
    assert torch.equal(codes[1], want[3]) and torch.equal(codes[[0, 2, 3, 4]], before[[0, 2, 3, 4]])
    out = torch.full((3, 64), 7.0, device="cuda")
    idx = ints([1, 5, -1])
    torch.cuda.synchronize()
    backend.gather_quant(buf(backend, out), cb, sb, buf(backend, idx), 3)
    with pytest.raises(BackendError):
        backend.sync()
    assert (out[1:] == 7.0).all() and torch.equal(out[0].double(), values(codes, scales)[1].view(-1).float().double())
    backend.sync()                                                        # reported once


def test_zero_tokens_are_nothing(backend):
    x, (codes, scales), slot = rand(1, 64, seed=9), empty_cache(3, 1, 64), ints([0])
    torch.cuda.synchronize()
    backend.scatter_kv_quant(buf(backend, codes), buf(backend, scales), buf(backend, x), buf(backend, slot), 0)
    backend.gather_quant(buf(backend, x), buf(backend, codes), buf(backend, scales), buf(backend, slot), 0)
    backend.sync()
    assert (codes == 0x7F).all() and x.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,rot,tokens", ROPE_CASES)
def test_rope_scatter_kv_quant(backend, nh, nkv, hd, rot, tokens, half, dtype):
    freq, mag = rope_frequencies(rot, 10000.0, RopeScaling.WAVELENGTH, 4.0, 4096, 1.0, 4.0)
    mag = 1.25
    freq = torch.from_numpy(freq).cuda()
    q, k, v = (rand(tokens, n * hd, seed=s).to(dtype) for n, s in ((nh, 11), (nkv, 12), (nkv, 13)))
    pos = ints(torch.arange(tokens) * 17 + 100000)
    slots = tokens + 9
    where = torch.randperm(slots, generator=torch.Generator().manual_seed(14))[:tokens]
    slot = ints(where)
    if tokens > 4:
        slot[2] = PAD
    kc, ks = empty_cache(slots, nkv, hd)
    vc, vs = empty_cache(slots, nkv, hd)
    k0, v0 = k.clone(), v.clone()
    q_out, k_alone = torch.empty_like(q), torch.empty_like(k)
    torch.cuda.synchronize()
    b = {n: buf(backend, t) for n, t in dict(q=q, k=k, v=v, pos=pos, freq=freq, slot=slot, kc=kc, ks=ks, vc=vc, vs=vs, qo=q_out, ko=k_alone).items()}
    backend.rope_scatter_kv_quant(b["qo"], b["q"], b["k"], b["v"], b["pos"], b["freq"], hd, mag, b["kc"], b["ks"], b["vc"], b["vs"],
                                  b["slot"], half)
    backend.sync()
    got_q = q_out.clone()
    backend.rope_scaled(b["qo"], b["ko"], b["q"], b["k"], b["pos"], b["freq"], hd, mag, half)
    backend.rope_scatter_kv_quant(b["q"], b["q"], b["k"], b["v"], b["pos"], b["freq"], hd, mag, b["kc"], b["ks"], b["vc"], b["vs"],
                                  b["slot"], half)                       # q in place, the cache again
    backend.sync()
    assert torch.equal(got_q, q_out) and torch.equal(q, q_out)            # the same rotation as rope_scaled's
    assert torch.equal(k, k0) and torch.equal(v, v0)
    kept = torch.ones(tokens, dtype=torch.bool, device="cuda")
    if tokens > 4:
        kept[2] = False
    at = where.cuda()[kept]
    want_codes, want_scales = quantised(v, nkv)
    assert torch.equal(vc[at], want_codes[kept]) and torch.equal(vs[:, at], want_scales[:, kept])
    others = torch.ones(slots, dtype=torch.bool, device="cuda")
    others[at] = False
    assert (kc[others] == 0x7F).all() and (vc[others] == 0x7F).all() and ks[:, others].isnan().all()
    want = rotated(k, hd, pos, freq, mag, half)[kept]
    slack = rope_slack(k, hd, mag)[kept]
    scale = (want.abs().view(len(want), nkv, hd).amax(-1) / 448).t()
    rope_max = slack.view(len(want), nkv, hd).amax(-1).t() / 448
    assert ((ks[:, at].double() - scale).abs() <= rope_max + scale * 2.0 ** -23).all()
    sub = (scale.t()[..., None] * 2.0 ** -10).expand(-1, -1, hd).reshape(want.shape)
    err = (values(kc[at], ks[:, at]).view(want.shape) - want).abs()
    assert (err <= torch.maximum(want.abs() * 2.0 ** -4, sub) * (1 + 2.0 ** -16) + 2 * slack).all()


# ---- attention -----------------------------------------------------------------------------------

def paged_cache(nkv, hd, lens, block, seed, spare=3):
    """A pool whose pages lie in any order, whose unused slots were never written, and its page table."""
    pages = [-(-l // block) for l in lens]
    n = sum(pages) + spare
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed))
    most = max(max(pages), 1)
    table = torch.full((len(lens), most), 2 ** 31 - 1, dtype=torch.int32)         # entries past a request lead nowhere
    kc, ks = empty_cache(n * block, nkv, hd)
    vc, vs = empty_cache(n * block, nkv, hd, fill=0xFF)
    at, slots = 0, []
    for r, l in enumerate(lens):
        table[r, :pages[r]] = order[at:at + pages[r]]
        at += pages[r]
        p = torch.arange(l)
        slots.append((table[r].long()[p // block] * block + p % block).cuda())
        if l:
            kc[slots[r]], ks[:, slots[r]] = quantised(rand(l, nkv * hd, seed=seed + 2 * r + 1), nkv)
            vc[slots[r]], vs[:, slots[r]] = quantised(rand(l, nkv * hd, seed=seed + 2 * r + 2) * (1.0 + r), nkv)
    return kc, ks, vc, vs, table.cuda(), slots, most


def expected(q, kc, ks, vc, vs, slots, lens, news, nh, nkv, hd, of_many=False):
    """Float64 attention, and for each output what its error may be beside the rounding of the output itself."""
    group, f16 = nh // nkv, 2.0 ** -11
    out, slack = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    t0 = 0
    for r, (l, n) in enumerate(zip(lens, news)):
        if l and n:
            k, v = values(kc[slots[r]], ks[:, slots[r]]), values(vc[slots[r]], vs[:, slots[r]])
            qq = q[t0:t0 + n].double().view(n, nkv, nh // nkv, hd)
            s = torch.einsum("nhgd,lhd->nhgl", qq, k) / math.sqrt(hd)
            size = torch.einsum("nhgd,lhd->nhgl", qq.abs(), k.abs()) / math.sqrt(hd)
            seen = torch.arange(l, device="cuda")[None] <= (l - n + torch.arange(n, device="cuda"))[:, None]
            s = s.masked_fill(~seen[:, None, None], -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)                           # a row that sees nothing: zeros
            o = torch.einsum("nhgl,lhd->nhgd", p, v)
            a = torch.einsum("nhgl,lhd->nhgd", p, v.abs())
            size = size.masked_fill(~seen[:, None, None], 0.0).amax(-1, keepdim=True)
            out[t0:t0 + n] = o.reshape(n, -1)
            # A weight is off by its own rounding to f16 and by twice the error of a score: up to 256 additions each off by 2^-23
            # (a tensor core may cut instead of rounding) of at most sum |q k|, 2^-15 of it; the exponential and the sums of
            # weights and of weighted values over up to 2^7 partial ones, 2^-16.  Where many rows are worked on at once (bf16,
            # more than 16 rows a KV head), keys and values are rounded to f16 after their scale has been multiplied in: a
            # product of a score by 2^-11 each, so the score by 2^-11 of sum |q k|, a value by 2^-11 for its scale and as much for
            # the product.
            many = q.dtype == torch.bfloat16 and hd in (64, 128) and (n * group > 16 or of_many)      # of_many: a row of such a request
            weight = f16 + 2.0 * 2.0 ** -15 * size + 2.0 ** -16
            if many:
                weight = weight + 2.0 * f16 + 2.0 * f16 * size
            # Below the normal range of f16 a rounding is off by 2^-25 instead: of a weight, the largest being 2^9 or more, 2^-34,
            # at each position of at most |v|; of a value's scale, the largest being 2^5 or more, 2^-30 of the largest value
            # (the sum of the weights is at least the largest).  And float32 and bf16 end at 2^-126.
            flush = (l * 2.0 ** -34 + 2.0 ** -30) * v.abs().amax() + 2.0 ** -126
            slack[t0:t0 + n] = (a * weight).reshape(n, -1) + flush
        t0 += n
    return out, slack


def attend(be, q, kc, ks, vc, vs, table, lens, news, nh, nkv, hd, block, most, fill=7.0):
    out = torch.full_like(q, fill)
    starts, ln = ints(np.concatenate([[0], np.cumsum(news)])), ints(lens)
    torch.cuda.synchronize()
    be.attention_quant(*[buf(be, t) for t in (out, q, kc, ks, vc, vs, table, starts, ln)], nh, nkv, hd, block, most)
    be.sync()
    return out


def check_attention(be, nh, nkv, hd, block, lens, news, dtype, seed=20, behind=0):
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, lens, block, seed)
    q = rand(sum(news) + behind, nh * hd, seed=seed - 1, loud=False).to(dtype)
    out = attend(be, q, kc, ks, vc, vs, table, lens, news, nh, nkv, hd, block, most)
    want, slack = expected(q, kc, ks, vc, vs, slots, lens, news, nh, nkv, hd)
    n = sum(news)
    err = (out.double() - want).abs()
    assert (err[:n] <= HALF_STEP[dtype] * want[:n].abs() * 1.01 + slack[:n]).all(), (err[:n] - HALF_STEP[dtype] * want[:n].abs() - slack[:n]).max()
    # all in all: float32 in and out, no 16-bit rounding inside; bf16, no more than the rounding of the output may cost alone
    limit = 1e-5 if dtype == torch.float32 else 2.0 ** -8
    assert torch.linalg.norm(err[:n]) <= limit * torch.linalg.norm(want[:n]) + 1e-30
    assert (out[n:] == 7.0).all()                                               # tokens behind the last request
    return out


DECODE = [  # heads, kv heads, head_dim, page, lengths
    (32, 8, 128, 16, [1000]), (32, 8, 128, 16, [1]), (8, 8, 64, 32, [15, 16, 17]), (14, 2, 64, 24, [300, 1, 64, 63, 65]),
    (3, 1, 128, 1, [33, 2]), (40, 8, 128, 7, [129, 128, 127, 5]), (16, 1, 128, 64, [511]), (32, 1, 64, 16, [700, 3]),
    (17, 1, 128, 16, [90]), (4, 2, 256, 8, [300, 20]), (4, 4, 32, 16, [70]), (6, 2, 96, 5, [41, 200]), (5, 5, 160, 16, [77]),
    (8, 4, 64, 16, [30000] + [20] * 9), (4, 2, 128, 16, [3 + 5 * i for i in range(70)]), (3, 1, 128, 32, [9000] * 2 + [1] * 8),
    (32, 8, 128, 256, [5000, 4097]), (7, 7, 128, 16, [260] * 9), (12, 3, 64, 48, [1025, 1024]), (32, 8, 128, 100000, [3000]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd,block,lens", DECODE)
def test_attention_decode(backend, nh, nkv, hd, block, lens, dtype):
    check_attention(backend, nh, nkv, hd, block, lens, [1] * len(lens), dtype)


SEVERAL = [  # heads, kv heads, head_dim, page, lengths, query tokens
    (32, 8, 128, 16, [200], [200]), (8, 2, 128, 16, [65], [64]), (8, 2, 64, 24, [300, 5, 77], [100, 1, 77]),
    (14, 2, 64, 16, [500, 40, 333], [129, 40, 1]), (4, 4, 128, 3, [150, 149], [127, 128]), (5, 1, 128, 16, [400], [33]),
    (16, 2, 128, 32, [130, 2, 600], [2, 2, 2]), (4, 1, 64, 16, [90, 91, 92], [4, 3, 5]), (32, 1, 128, 16, [260], [50]),
    (8, 2, 128, 16, [200] * 3 + [90] * 9, [150, 1, 1] + [1] * 8 + [40]), (4, 1, 64, 24, [700] * 40, [1, 40] * 20),
    (8, 2, 128, 16, [100] + [5] * 50, [40] + [0] * 50), (8, 1, 64, 16, [300] * 3, [17, 1, 2]),
    (6, 3, 96, 16, [70], [70]), (2, 2, 256, 16, [130], [40]), (32, 8, 128, 64, [1500], [600]), (8, 8, 128, 16, [1030], [1030]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd,block,lens,news", SEVERAL)
def test_attention_several_query_tokens(backend, nh, nkv, hd, block, lens, news, dtype):
    check_attention(backend, nh, nkv, hd, block, lens, news, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_attention_rows_that_see_nothing(backend, hd, dtype):
    """Requests without query tokens, without positions, with more query tokens than positions; tokens behind the last."""
    check_attention(backend, 8, 2, hd, 16, [40, 0, 10, 3, 0, 90], [0, 1, 1, 20, 30, 90], dtype, behind=5)
    check_attention(backend, 8, 2, hd, 16, [0, 0], [1, 1], dtype, behind=1)
    check_attention(backend, 8, 2, hd, 16, [5], [130], dtype)


@pytest.mark.parametrize("news", [[1, 1], [1, 30], [40, 1], [70, 30]])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_attention_positions_that_are_nan(backend, hd, news):
    """A position whose key or value is NaN shows in the rows that see it, and in no other."""
    nh, nkv, block, lens = 8, 2, 16, [150, 61]
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, lens, block, 30)
    clean_k, clean_v = ks.clone(), vs.clone()
    ks[0, slots[0][149]] = math.nan                    # seen by the last query token of request 0 alone, first KV head
    kc[slots[0][149], :hd] = 0
    vs[1, slots[1][60]] = math.nan                     # the same of request 1, value, second KV head
    vc[slots[1][60], hd:] = 0
    q = rand(sum(news), nh * hd, seed=29, loud=False).to(torch.bfloat16)
    args = (table, lens, news, nh, nkv, hd, block, most)
    out = attend(backend, q, kc, ks, vc, vs, *args).view(sum(news), nkv, -1)
    ref = attend(backend, q, kc, clean_k, vc, clean_v, *args).view(sum(news), nkv, -1)
    bad = torch.zeros(sum(news), nkv, dtype=torch.bool, device="cuda")
    bad[news[0] - 1, 0] = bad[sum(news) - 1, 1] = True
    assert out[bad].isnan().all() and torch.equal(out[~bad], ref[~bad]) and ref.isfinite().all()


@pytest.mark.parametrize("hd", [64, 96, 128])
def test_attention_scores_far_apart(backend, hd):
    """Scores of several hundred: the running maximum moves by much between tiles, most weights underflow."""
    nh, nkv, block, lens, news = 8, 2, 16, [700, 300], [1, 40]
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, lens, block, 40)
    q = (rand(sum(news), nh * hd, seed=39, loud=False) * 60).to(torch.bfloat16)
    out = attend(backend, q, kc, ks, vc, vs, table, lens, news, nh, nkv, hd, block, most)
    want, slack = expected(q, kc, ks, vc, vs, slots, lens, news, nh, nkv, hd)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + slack).all()


@pytest.mark.parametrize("v_size", [1e-30, 1e30])
@pytest.mark.parametrize("news", [[1], [50]])
def test_attention_one_strong_position_and_sizes_of_values(backend, news, v_size):
    """One position takes most of the weight and thousands share the rest; values of any size, some of zero."""
    nh, nkv, hd, block, lens = 4, 1, 128, 16, [4000]
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, lens, block, 50)
    k = torch.zeros(4000, hd, device="cuda")
    k[7, 0] = 10.0 * math.sqrt(hd)
    v = rand(4000, hd, seed=51) * v_size + v_size
    v[1000:1010] = 0.0
    kc[slots[0]], ks[:, slots[0]] = quantised(k, 1)
    vc[slots[0]], vs[:, slots[0]] = quantised(v, 1)
    q = torch.zeros(sum(news), nh * hd, device="cuda")
    q.view(-1, nh, hd)[..., 0] = 1.0
    q = q.to(torch.bfloat16)
    out = attend(backend, q, kc, ks, vc, vs, table, lens, news, nh, nkv, hd, block, most)
    want, slack = expected(q, kc, ks, vc, vs, slots, lens, news, nh, nkv, hd)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + slack).all()


@pytest.mark.parametrize("news", [[1, 1], [1, 20], [64, 70]])
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_attention_pages_beyond_the_pool(backend, hd, news):
    """Their positions count as unseen, the call is reported, the context goes on."""
    nh, nkv, block, lens = 8, 2, 16, [150, 100]
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, lens, block, 60)
    table[0, 4] = ks.shape[1] // block                                           # the first page behind the pool
    table[1, 0] = -1
    q = rand(sum(news), nh * hd, seed=59, loud=False).to(torch.bfloat16)
    out = torch.zeros_like(q)
    starts, ln = ints(np.concatenate([[0], np.cumsum(news)])), ints(lens)
    torch.cuda.synchronize()
    backend.attention_quant(*[buf(backend, t) for t in (out, q, kc, ks, vc, vs, table, starts, ln)], nh, nkv, hd, block, most)
    with pytest.raises(BackendError) as e:
        backend.sync()
    assert e.value.code == -4
    t0 = 0
    for r, n in enumerate(news):
        for i in range(n):
            see = torch.arange(lens[r] - n + i + 1, device="cuda")
            see = see[(table[r].long()[see // block] >= 0) & (table[r].long()[see // block] < ks.shape[1] // block)]
            slot = table[r].long()[see // block] * block + see % block
            want, slack = expected(q[t0 + i:t0 + i + 1], kc, ks, vc, vs, [slot], [len(see)], [1], nh, nkv, hd, n * nh // nkv > 16)
            assert ((out[t0 + i].double() - want[0]).abs() <= 2.0 ** -8 * 1.01 * want[0].abs() + slack[0]).all()
        t0 += n
    check_attention(backend, nh, nkv, hd, block, [50], [1], torch.bfloat16)


def test_attention_lengths_and_starts_beyond_what_there_is(backend):
    """seq_lens longer than the page table, query_starts past q: cut, the first of them reported; nothing else is touched."""
    nh, nkv, hd, block = 4, 2, 64, 16
    kc, ks, vc, vs, table, slots, most = paged_cache(nkv, hd, [48], block, 70)
    q = rand(2, nh * hd, seed=69, loud=False).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    starts, ln = ints([0, 1]), ints([10 ** 9])
    torch.cuda.synchronize()
    backend.attention_quant(*[buf(backend, t) for t in (out, q, kc, ks, vc, vs, table, starts, ln)], nh, nkv, hd, block, most)
    with pytest.raises(BackendError):
        backend.sync()
    want, slack = expected(q[:1], kc, ks, vc, vs, slots, [48], [1], nh, nkv, hd)
    assert ((out[:1].double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + slack).all() and (out[1] == 7.0).all()
    starts, ln = ints([0, 50]), ints([48])                                       # 50 query tokens claimed, two are there
    torch.cuda.synchronize()
    backend.attention_quant(*[buf(backend, t) for t in (out, q, kc, ks, vc, vs, table, starts, ln)], nh, nkv, hd, block, most)
    backend.sync()
    want, slack = expected(q, kc, ks, vc, vs, slots, [48], [2], nh, nkv, hd)
    assert ((out.double() - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + slack).all()


def test_attention_needs_its_workspace_before_a_capture(cuda_lib):
    """A first call inside a capture would have to allocate: refused, and the context goes on."""
    stream = torch.cuda.Stream()
    be = CudaBackend(0, stream.cuda_stream)
    kc, ks, vc, vs, table, slots, most = paged_cache(2, 64, [40], 16, 85)
    q, out = torch.zeros(1, 256, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 256, dtype=torch.bfloat16, device="cuda")
    b = [buf(be, t) for t in (out, q, kc, ks, vc, vs, table, ints([0, 1]), ints([40]))]
    torch.cuda.synchronize()
    graph, refused = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(graph, stream=stream):
        try:
            be.attention_quant(*b, 4, 2, 64, 16, most)
        except BackendError as e:
            refused = e
    assert refused is not None and refused.code == -1 and "capture" in str(refused)
    be.attention_quant(*b, 4, 2, 64, 16, most)
    be.sync()
    assert out.isfinite().all() and out.any()            # queries of zeros: the mean of the values
    be.close()


def test_attention_twice_is_the_same(backend):
    """No sum depends on which block of threads came first."""
    for news in ([1] * 5, [70, 1, 30, 1, 2]):
        lens = [3000, 200, 77, 2500, 64]
        kc, ks, vc, vs, table, slots, most = paged_cache(8, 128, lens, 16, 80)
        q = rand(sum(news), 32 * 128, seed=79, loud=False).to(torch.bfloat16)
        a = [attend(backend, q, kc, ks, vc, vs, table, lens, news, 32, 8, 128, 16, most) for _ in range(4)]
        assert all(torch.equal(a[0], x) for x in a[1:])


# ---- refusals ------------------------------------------------------------------------------------

def _attention_args(**kw):
    t = dict(out=torch.zeros(2, 256, dtype=torch.bfloat16), q=torch.zeros(2, 256, dtype=torch.bfloat16),
             kc=torch.zeros(64, 128, dtype=torch.uint8), ks=torch.zeros(2, 64), vc=torch.zeros(64, 128, dtype=torch.uint8),
             vs=torch.zeros(2, 64), table=torch.zeros(2, 2, dtype=torch.int32), starts=torch.zeros(3, dtype=torch.int32),
             lens=torch.zeros(2, dtype=torch.int32))
    n = dict(nh=4, nkv=2, hd=64, block=16, most=2)
    for k, v in kw.items():
        (t if k in t else n)[k] = v
    return t, n


@pytest.mark.parametrize("change,code", [
    (dict(q=torch.zeros(2, 256)), -3), (dict(kc=torch.zeros(64, 128)), -3), (dict(ks=torch.zeros(2, 64, dtype=torch.int32)), -3),
    (dict(lens=torch.zeros(2)), -3), (dict(nh=3), -2), (dict(nkv=3), -2), (dict(hd=48), -2), (dict(hd=288), -2), (dict(block=0), -2),
    (dict(most=0), -2), (dict(most=3), -2), (dict(ks=torch.zeros(2, 63)), -2), (dict(vs=torch.zeros(4, 64)), -2),
    (dict(vc=torch.zeros(48, 128, dtype=torch.uint8)), -2), (dict(starts=torch.zeros(2, dtype=torch.int32)), -2),
    (dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)), -2), (dict(q=torch.zeros(2, 192, dtype=torch.bfloat16)), -2),
])
def test_attention_refusals(backend, change, code):
    t, n = _attention_args(**change)
    b = [buf(backend, x.cuda()) for x in t.values()]
    with pytest.raises(BackendError) as e:
        backend.attention_quant(*b, n["nh"], n["nkv"], n["hd"], n["block"], n["most"])
    assert e.value.code == code


def test_overlaps_are_refused(backend):
    t, n = _attention_args()
    b = [buf(backend, x.cuda()) for x in t.values()]
    with pytest.raises(BackendError) as e:
        backend.attention_quant(b[1], *b[1:], 4, 2, 64, 16, 2)                    # out is q
    assert e.value.code == -4
    q, k, pos, f = torch.zeros(4, 128, device="cuda"), torch.zeros(4, 128, device="cuda"), ints([0, 1, 2, 3]), torch.ones(32, device="cuda")
    qb, kb, pb, fb = (buf(backend, x) for x in (q, k, pos, f))
    shifted = backend.wrap(q.data_ptr() + 512, [128, 3], DType.F32, keepalive=q)
    k3 = backend.wrap(k.data_ptr(), [128, 3], DType.F32, keepalive=k)
    q3 = backend.wrap(q.data_ptr(), [128, 3], DType.F32, keepalive=q)
    for args in ((shifted, k3, q3, k3), (qb, qb, qb, kb), (kb, kb, qb, kb)):
        with pytest.raises(BackendError) as e:
            backend.rope_scaled(*args, pb, fb, 64)
        assert e.value.code == -4
    c, s, sl = torch.zeros(8, 128, dtype=torch.uint8, device="cuda"), torch.zeros(2, 8, device="cuda"), ints([0, 1, 2, 3])
    cb, sb, slb = (buf(backend, x) for x in (c, s, sl))
    with pytest.raises(BackendError) as e:                                        # one pool for keys and values
        backend.rope_scatter_kv_quant(qb, qb, kb, kb, pb, fb, 64, 1.0, cb, sb, cb, sb, slb)
    assert e.value.code == -4


def test_write_and_read_refusals(backend):
    x, c, s, i = torch.zeros(4, 128), torch.zeros(8, 128, dtype=torch.uint8), torch.zeros(2, 8), torch.zeros(4, dtype=torch.int32)

    def refused(code, call, *ts, extra=()):
        b = [buf(backend, t.cuda()) for t in ts]
        with pytest.raises(BackendError) as e:
            call(*b, *extra)
        assert e.value.code == code

    for call, data_first in ((backend.scatter_kv_quant, False), (backend.gather_quant, True)):
        order = lambda d, p, sc, ix: (d, p, sc, ix) if data_first else (p, sc, d, ix)  # noqa: E731
        refused(-3, call, *order(x, x, s, i), extra=(4,))
        refused(-3, call, *order(x, c, i.view(2, 2), i), extra=(2,))
        refused(-3, call, *order(x, c, s, x), extra=(4,))
        refused(-3, call, *order(c[:4].contiguous(), c, s, i), extra=(4,))
        refused(-2, call, *order(x, c, s, i), extra=(5,))
        refused(-2, call, *order(x[:, :64].contiguous(), c, s, i), extra=(4,))
        refused(-2, call, *order(x, c, torch.zeros(2, 9), i), extra=(4,))
        refused(-2, call, *order(x, c, torch.zeros(3, 8), i), extra=(4,))
    q = torch.zeros(4, 256)
    f = torch.zeros(32)
    refused(-3, backend.rope_scaled, q, x, q, x.bfloat16(), i, f, extra=(64,))
    refused(-3, backend.rope_scaled, q, x.bfloat16(), q, x, i, f, extra=(64,))
    refused(-3, backend.rope_scaled, q, x, q, x, f, f, extra=(64,))
    refused(-2, backend.rope_scaled, q, x, q, x, i, torch.zeros(33), extra=(64,))
    refused(-2, backend.rope_scaled, q, x, q, x, i[:3].contiguous(), f, extra=(64,))
    refused(-2, backend.rope_scaled, q, x, q, x, i, f, extra=(63,))
    refused(-2, backend.rope_scaled, q[:3].contiguous(), x, q, x, i, f, extra=(64,))
    refused(-4, backend.rope_scaled, q, x, q.clone(), x.clone(), i, f, extra=(64, math.nan))
    cache = (c, s, c.clone(), s.clone())
    refused(-2, lambda *b: backend.rope_scatter_kv_quant(*b[:6], 32, 1.0, *b[6:]), q, q.clone(), x, x.clone(), i, torch.zeros(8), *cache, i.clone())
    refused(-3, lambda *b: backend.rope_scatter_kv_quant(*b[:6], 64, 1.0, *b[6:]), q, q.clone(), x, x.bfloat16(), i, f, *cache, i.clone())
    refused(-2, lambda *b: backend.rope_scatter_kv_quant(*b[:6], 64, 1.0, *b[6:]), q, q.clone(), x, x.clone(), i, f, c, s,
            torch.zeros(9, 128, dtype=torch.uint8), torch.zeros(2, 9), i.clone())


def test_e4m3_buffers_elsewhere_are_refused(backend):
    codes, x = torch.zeros(256, 256, dtype=torch.uint8, device="cuda"), torch.zeros(1, 256, device="cuda")
    cb, xb = buf(backend, codes), buf(backend, x)
    out = backend.alloc([256], DType.F32)
    for call in (lambda: backend.matmul(out, cb, xb), lambda: backend.add(out, cb, cb), lambda: backend.read_to_vec_f32(cb),
                 lambda: backend.rms_norm(out, cb, xb, 1e-5)):
        with pytest.raises(BackendError) as e:
            call()
        assert e.value.code == -3
    pool = backend.alloc([256, 7], DType.E4M3)
    assert pool.nbytes == 7 * 256


# ---- together ------------------------------------------------------------------------------------

def test_a_run_of_them_captured_and_replayed(cuda_lib):
    """A prompt and then decode steps of two requests through one layer's calls: rotation and write, attention, rows read
    back.  The decode step is one CUDA graph, replayed with new contents of its buffers; a padding token rides along."""
    nh, nkv, hd, rot, block, most = 8, 2, 128, 64, 16, 8
    freq, mag = rope_frequencies(rot, 500000.0, RopeScaling.WAVELENGTH, 8.0, 64, 1.0, 4.0)
    freq = torch.from_numpy(freq).cuda()
    stream = torch.cuda.Stream()
    be = CudaBackend(0, stream.cuda_stream)
    n_slots = 20 * block
    kc, ks = empty_cache(n_slots, nkv, hd)
    vc, vs = empty_cache(n_slots, nkv, hd)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(90))[:2 * most].view(2, most).to(torch.int32).cuda()
    prompt = [37, 50]
    hist = [[], []]                                                              # float64 keys and values as they should be

    def slots_of(r, a, b):
        p = torch.arange(a, b)
        return (table.cpu()[r].long()[p // block] * block + p % block).tolist()

    def remember(r, k, v, pos):
        hist[r].append((rotated(k, hd, pos, freq, mag, True), v.double()))

    def check(out, q, news, lens):
        """Against attention over the cache as it is, and over the float64 keys and values that went into it."""
        slots = [torch.tensor(slots_of(r, 0, lens[r])).cuda() for r in range(2)]
        want, slack = expected(q, kc, ks, vc, vs, slots, lens, news, nh, nkv, hd)
        n = sum(news)
        assert ((out[:n].double() - want[:n]).abs() <= 2.0 ** -8 * 1.01 * want[:n].abs() + slack[:n]).all()
        for r in range(2):
            k = torch.cat([h[0] for h in hist[r]])
            err = (values(kc[slots[r]], ks[:, slots[r]]).view(k.shape) - k).abs()
            top = k.abs().view(len(k), nkv, hd).amax(-1, keepdim=True).expand(-1, -1, hd).reshape(k.shape)
            assert (err <= k.abs() * 2.0 ** -4 * 1.001 + top * (2.0 ** -10 / 448 + 2.0 ** -18)).all()

    with torch.cuda.stream(stream):
        # the prompts, as one batch
        n = sum(prompt)
        q, k, v = rand(n, nh * hd, seed=91, loud=False).bfloat16(), rand(n, nkv * hd, seed=92).bfloat16(), rand(n, nkv * hd, seed=93).bfloat16()
        pos, slot = ints(list(range(37)) + list(range(50))), ints(slots_of(0, 0, 37) + slots_of(1, 0, 50))
        starts, lens, qo, out = ints([0, 37, 87]), ints(prompt), torch.empty_like(q), torch.empty_like(q)
        b = {m: buf(be, t) for m, t in dict(q=q, k=k, v=v, pos=pos, freq=freq, slot=slot, kc=kc, ks=ks, vc=vc, vs=vs, starts=starts,
                                            lens=lens, qo=qo, out=out, table=table).items()}
        be.rope_scatter_kv_quant(b["qo"], b["q"], b["k"], b["v"], b["pos"], b["freq"], hd, mag, b["kc"], b["ks"], b["vc"], b["vs"], b["slot"], True)
        be.attention_quant(b["out"], b["qo"], b["kc"], b["ks"], b["vc"], b["vs"], b["table"], b["starts"], b["lens"], nh, nkv, hd, block, most)
        be.sync()
        remember(0, k[:37], v[:37], pos[:37])
        remember(1, k[37:], v[37:], pos[37:])
        check(out, qo, prompt, prompt)

        # decode: two requests and a padding token
        q, k, v = (torch.zeros(3, m * hd, dtype=torch.bfloat16, device="cuda") for m in (nh, nkv, nkv))
        pos, slot, starts, lens = ints([0, 0, 0]), ints([PAD] * 3), ints([0, 1, 2]), ints([1, 1])
        qo, out, back = torch.zeros_like(q), torch.full_like(q, 7.0), torch.zeros(2, nkv * hd, device="cuda")
        idx = ints([0, 0])
        d = {m: buf(be, t) for m, t in dict(q=q, k=k, v=v, pos=pos, slot=slot, starts=starts, lens=lens, qo=qo, out=out, back=back, idx=idx).items()}

        def step():
            be.rope_scatter_kv_quant(d["qo"], d["q"], d["k"], d["v"], d["pos"], b["freq"], hd, mag, b["kc"], b["ks"], b["vc"], b["vs"], d["slot"], True)
            be.attention_quant(d["out"], d["qo"], b["kc"], b["ks"], b["vc"], b["vs"], b["table"], d["starts"], d["lens"], nh, nkv, hd, block, most)
            be.gather_quant(d["back"], b["kc"], b["ks"], d["idx"], 2)

        step()                                                                   # outside the capture: the workspace grows here
        be.sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        at = list(prompt)
        for i in range(20):
            q.copy_(rand(3, nh * hd, seed=100 + i, loud=False)), k.copy_(rand(3, nkv * hd, seed=200 + i)), v.copy_(rand(3, nkv * hd, seed=300 + i))
            where = slots_of(0, at[0], at[0] + 1) + slots_of(1, at[1], at[1] + 1)
            pos.copy_(ints(at + [0])), slot.copy_(ints(where + [PAD])), idx.copy_(ints(where))
            at = [a + 1 for a in at]
            lens.copy_(ints(at))
            graph.replay()
            stream.synchronize()
            for r in range(2):
                remember(r, k[r:r + 1], v[r:r + 1], pos[r:r + 1])
            check(out, qo, [1, 1], at)
            assert (out[2] == 7.0).all()
            w = torch.tensor(where).cuda()
            assert torch.equal(back, values(kc[w], ks[:, w]).view(2, -1).float())
        be.sync()
        del graph
    be.close()


def test_on_another_stream_than_the_tensors(cuda_lib):
    """The calls run on the context's stream and nothing else: results are there once it has been waited for."""
    be = CudaBackend(0)
    for seed in range(3):
        check_attention(be, 32, 8, 128, 16, [700, 40], [1, 1], torch.bfloat16, seed=200 + seed)
    be.close()
