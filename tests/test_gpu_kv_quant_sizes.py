"""The 8-bit KV cache at sizes that the other tests do not reach."""
import pytest
import torch

from llm_rs_b200 import BackendError, CudaBackend, DType
from test_gpu_kv_quant import HALF_STEP, attend, buf, expected, ints, paged_cache, quantised, rand, values

pytestmark = pytest.mark.gpu


# ---- counts that do not fit ----------------------------------------------------------------------

def _nowhere(be, *buffers):
    """Buffers of any size at addresses that nothing lies at, far apart: for calls that are refused before anything is launched."""
    return [be.wrap((i + 1) << 44, shape, kind) for i, (shape, kind) in enumerate(buffers)]


@pytest.mark.parametrize("tokens", [1 << 30, (1 << 31) - 1])
def test_token_counts_of_31_bits_are_refused(backend, tokens):
    """The kernels' ints hold a count and what a grid adds to it: up to 2^30 - 1."""
    q, p, f = ([2, tokens], DType.F32), ([tokens], DType.I32), ([1], DType.F32)
    cache = (([2, 64], DType.E4M3), ([64], DType.F32))
    a, b, c = _nowhere(backend, q, q, q, q, p, f), _nowhere(backend, *cache, q, p), _nowhere(backend, q, q, q, q, p, f, *cache, *cache, p)
    for call in (lambda: backend.rope_scaled(*a, 2), lambda: backend.scatter_kv_quant(*b, tokens),
                 lambda: backend.rope_scatter_kv_quant(*c[:6], 2, 1.0, *c[6:])):
        with pytest.raises(BackendError) as e:
            call()
        assert e.value.code == -2


@pytest.mark.parametrize("requests", [1 << 30, (1 << 31) - 2])
def test_request_counts_of_31_bits_are_refused(backend, requests):
    """A loop over requests in steps of 32 passes 2^31 behind the last of them."""
    out, pool, scales = ([64, 1], DType.F32), ([64, 64], DType.E4M3), ([64], DType.F32)
    b = _nowhere(backend, out, out, pool, scales, pool, scales, ([requests], DType.I32), ([requests + 1], DType.I32), ([requests], DType.I32))
    with pytest.raises(BackendError) as e:
        backend.attention_quant(*b, 1, 1, 64, 16, 1)
    assert e.value.code == -2


def test_head_counts_of_31_bits_are_refused(backend):
    wide, one = ([(1 << 31) - 2, 1], DType.F32), ([1], DType.I32)
    b = _nowhere(backend, wide, wide, wide, wide, one, ([1], DType.F32))
    with pytest.raises(BackendError) as e:
        backend.rope_scaled(*b, 2)
    assert e.value.code == -2


# ---- long requests, large pools, padded batches ---------------------------------------------------

def _close(out, q, cache, slots, lens, news, nh, nkv, hd):
    want, slack = expected(q, *cache, slots, lens, news, nh, nkv, hd)
    n = sum(news)
    assert ((out[:n].double() - want[:n]).abs() <= HALF_STEP[q.dtype] * 1.01 * want[:n].abs() + slack[:n]).all()
    assert torch.linalg.vector_norm(out[:n].double() - want[:n]) <= (1e-5 if q.dtype == torch.float32 else 2.0 ** -8) * torch.linalg.vector_norm(want[:n])
    assert (out[n:] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv,hd,block,news", [(8, 2, 128, 256, [1]), (8, 2, 64, 48, [1]), (4, 1, 128, 16, [4]), (4, 1, 128, 16, [5]), (4, 1, 64, 24, [33])])
def test_131071_positions(backend, nh, nkv, hd, block, news, dtype):
    """One request of 131071 positions: a token, four and five drafts, a chunk of 33."""
    lens = [131071]
    *cache, table, slots, most = paged_cache(nkv, hd, lens, block, 500)
    q = rand(sum(news), nh * hd, seed=501, loud=False).to(dtype)
    _close(attend(backend, q, *cache, table, lens, news, nh, nkv, hd, block, most), q, cache, slots, lens, news, nh, nkv, hd)


@pytest.mark.parametrize("block", [16, 24])
def test_pools_of_more_than_31_bits(backend, block):
    """Rows behind 2^31 bytes of a pool are written, read back and attended over."""
    nh, nkv, hd, l = 16, 8, 128, 500
    pages = -(-((1 << 31) // (nkv * hd) + 100000) // block)
    n = pages * block
    kc, ks, vc, vs = (t for _ in range(2) for t in (torch.empty(n, nkv * hd, dtype=torch.uint8, device="cuda"), torch.empty(nkv, n, device="cuda")))
    most = -(-l // block)
    table = torch.arange(pages - 1, pages - 1 - most, -1)[None]                        # the last pages, in falling order
    p = torch.arange(l)
    slots = table[0][p // block] * block + p % block
    assert int(slots.min()) * nkv * hd > 1 << 31
    k, v = rand(l, nkv * hd, seed=510).bfloat16(), rand(l, nkv * hd, seed=511).bfloat16()
    slot, back = ints(slots), torch.empty(l, nkv * hd, device="cuda")
    torch.cuda.synchronize()
    b = [buf(backend, t) for t in (kc, ks, vc, vs, k, v, slot, back)]
    backend.scatter_kv_quant(b[0], b[1], b[4], b[6], l)
    backend.scatter_kv_quant(b[2], b[3], b[5], b[6], l)
    backend.gather_quant(b[7], b[0], b[1], b[6], l)
    backend.sync()
    at = slots.cuda()
    want, scales = quantised(k, nkv)
    assert torch.equal(kc[at], want) and torch.equal(ks[:, at], scales)
    assert torch.equal(back, values(want, scales).view(l, -1).float())
    for news in (1, 40):
        q = rand(news, nh * hd, seed=512 + news, loud=False).bfloat16()
        out = attend(backend, q, kc, ks, vc, vs, table.to(torch.int32).cuda(), [l], [news], nh, nkv, hd, block, most)
        small = [x[at].contiguous() for x in (kc, vc)], [x[:, at].contiguous() for x in (ks, vs)]
        _close(out, q, (small[0][0], small[1][0], small[0][1], small[1][1]), [torch.arange(l, device="cuda")], [l], [news], nh, nkv, hd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nh,nkv", [(17, 1), (32, 1), (40, 2), (8, 2)])
@pytest.mark.parametrize("hd", [64, 128])
def test_padded_decode_batches(backend, hd, nh, nkv, dtype):
    """Decoding requests with padding tokens behind the last one, groups of up to 32 query heads; idle requests between them."""
    lens, news = [300, 0, 1000, 64, 7], [1, 0, 1, 1, 1]
    *cache, table, slots, most = paged_cache(nkv, hd, lens, 16, 520)
    q = rand(sum(news) + 9, nh * hd, seed=521, loud=False).to(dtype)
    _close(attend(backend, q, *cache, table, lens, news, nh, nkv, hd, 16, most), q, cache, slots, lens, news, nh, nkv, hd)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,hd,tokens", [(8, 128, 3), (2, 64, 700), (8, 128, 2000), (3, 80, 50)])
def test_out_on_sixteen_bytes(backend, heads, hd, tokens, dtype):
    """Every buffer may start on 16 bytes; the widest stores need 32."""
    x = rand(tokens, heads * hd, seed=530).to(dtype)
    codes, scales = quantised(x, heads)
    room = torch.zeros(tokens * heads * hd * x.element_size() + 64, dtype=torch.uint8, device="cuda")
    at = 16 + (-room.data_ptr()) % 32
    out = room[at:at + tokens * heads * hd * x.element_size()].view(dtype).view(tokens, -1)
    assert out.data_ptr() % 32 == 16
    idx = ints(torch.arange(tokens - 1, -1, -1))
    torch.cuda.synchronize()
    backend.gather_quant(*[buf(backend, t) for t in (out, codes, scales, idx)], tokens)
    backend.sync()
    assert torch.equal(out, values(codes, scales).view(tokens, -1).float().to(dtype).flip(0))
    assert not room[:at].any() and not room[at + out.numel() * out.element_size():].any()


@pytest.mark.parametrize("side", [False, True])
def test_in_order_with_torch(cuda_lib, side):
    """A context on the stream that torch works on, its default stream (handle 1) or another: calls come after what torch has
    put there and before what it puts there next, without a wait between them."""
    nh, nkv, hd, lens = 8, 2, 128, [5000, 300]
    *cache, table, slots, most = paged_cache(nkv, hd, lens, 16, 540)
    x = rand(2, nh * hd, seed=541, loud=False).bfloat16()
    stream = torch.cuda.Stream() if side else torch.cuda.default_stream()
    be = CudaBackend(0, stream.cuda_stream or 1)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        q, out, big = torch.zeros_like(x), torch.full_like(x, 7.0), torch.ones(1 << 28, device="cuda")
        starts, ln = ints([0, 1, 2]), ints(lens)
        b = [buf(be, t) for t in (out, q, *cache, table, starts, ln)]
        be.attention_quant(*b, nh, nkv, hd, 16, most)                              # the workspace grows here
        got = []
        for scale in (1.0, -2.0, 0.5):
            big.mul_(1.0001)                                                       # keeps the stream busy
            q.copy_(x * scale)
            be.attention_quant(*b, nh, nkv, hd, 16, most)
            got.append(out.clone())
            out.fill_(7.0)
    torch.cuda.synchronize()
    be.sync()
    for scale, o in zip((1.0, -2.0, 0.5), got):
        _close(o, x * scale, cache, slots, lens, [1, 1], nh, nkv, hd)
    be.close()
