"""The 8-bit KV cache at sizes that the other tests do not reach."""
import pytest

from llm_rs_b200 import BackendError, DType

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
