"""Refusals of the paged 4-bit cache's entry points, which need no GPU: the C entries look at their arguments before they touch the device, and the Python functions at
their tensors before that."""
import math

import pytest
import torch

from qspec_b200 import _lib, ops

I32 = torch.int32
P = 1 << 20                       # stands for a pointer: on a 16-byte boundary, never followed


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, status, what):
    text = lib.qspec_last_error().decode()
    assert status in (1, 2, 4) and what in text, (status, text)


def append(lib, ptrs=(P,) * 9, ld=(8 + 4) * 128, cos_rows=9, q_ts=8 * 128, ntok=3, H=8, G=2, D=128, npages=9, page=64, dtype=0):
    qkv, cs, pos, slots, k, v, kw, vw, q = ptrs
    return lib.qspec_kv4_append(qkv, ld, cs, cos_rows, pos, slots, k, v, kw, vw, q, q_ts, ntok, H, G, D, npages, page, 1, dtype, None)


@pytest.mark.parametrize("kw,what", [*((dict(ptrs=tuple(None if j == i else P for j in range(9))), "null") for i in range(8)),
                                     *((dict(ptrs=tuple(P + 2 if j == i else P for j in range(9))), "16-byte") for i in (0, 1, 4, 5, 6, 7, 8)),
                                     (dict(D=96), "64 or 128"), (dict(page=256), "pages of"), (dict(G=0), "kv heads"), (dict(npages=0), "pages="), (dict(npages=1 << 27), "pages="),
                                     (dict(dtype=2), "float16"), (dict(ld=100), "16-byte"), (dict(ld=12 * 128 + 4), "16-byte"), (dict(q_ts=64), "16-byte"), (dict(H=0), "heads="),
                                     (dict(cos_rows=0), "table rows"), (dict(ntok=-1), "tokens="), (dict(ntok=1 << 24), "tokens=")])
def test_append_refuses(lib, kw, what):
    refused(lib, append(lib, **kw), what)


def read(lib, ptrs=(P,) * 7, rows=3, G=2, D=128, npages=9, page=64, dtype=0):
    return lib.qspec_kv4_read(*ptrs, rows, G, D, npages, page, dtype, None)


@pytest.mark.parametrize("kw,what", [*((dict(ptrs=tuple(None if j == i else P for j in range(7))), "null") for i in range(7)),
                                     *((dict(ptrs=tuple(P + 8 if j == i else P for j in range(7))), "16-byte") for i in (0, 1, 2, 3, 5, 6)), (dict(D=32), "64 or 128"),
                                     (dict(rows=-1), "rows"), (dict(rows=1 << 30, G=8), "too many"), (dict(dtype=2), "float16"), (dict(page=0), "pages of")])
def test_read_refuses(lib, kw, what):
    refused(lib, read(lib, **kw), what)


def attend(lib, ptrs=(P,) * 9, q_ts=1024, q_hs=128, o_ts=1024, o_hs=128, ntok=3, requests=2, width=4, H=8, G=2, D=128, npages=9, page=64, most=2, scale=0.1, dtype=0, work=P,
           nbytes=1 << 30):
    q, k, v, kw, vw, table, start, lens, out = ptrs
    return lib.qspec_kv4_attention(q, q_ts, q_hs, k, v, kw, vw, table, start, lens, out, o_ts, o_hs, ntok, requests, width, H, G, D, npages, page, most, scale, dtype, work, nbytes,
                                   None)


@pytest.mark.parametrize("kw,what", [*((dict(ptrs=tuple(None if j == i else P for j in range(9))), "null") for i in range(9)),
                                     *((dict(ptrs=tuple(P + 2 if j == i else P for j in range(9))), "16-byte") for i in (0, 1, 2, 3, 4, 8)),
                                     (dict(D=256), "64 or 128"), (dict(page=24), "pages of"), (dict(H=9), "query heads"), (dict(H=1), "query heads"), (dict(G=0), "query heads"),
                                     (dict(q_ts=1023), "16-byte"), (dict(o_hs=4), "16-byte"), (dict(requests=0), "requests="), (dict(width=0), "width="), (dict(width=1 << 26), "width="),
                                     (dict(most=0), "kv4_attention"), (dict(ntok=-1), "tokens="), (dict(dtype=2), "float16"), (dict(work=None), "workspace"),
                                     (dict(nbytes=1000), "workspace"), (dict(work=P + 4), "workspace"), *((dict(scale=s), "scale must be") for s in (0.0, -0.1, math.inf, math.nan, 1e-60))])
def test_attention_refuses(lib, kw, what):
    refused(lib, attend(lib, **kw), what)


def test_calls_of_nothing_are_no_errors(lib):
    assert append(lib, ntok=0) == 0 and read(lib, rows=0) == 0 and attend(lib, ntok=0) == 0


def test_python_functions_refuse_tensors_that_are_not_on_a_gpu():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)  # noqa: E731
    cache = (z(3, 2, 16, 32, dtype=torch.uint8), z(3, 2, 16, 32, dtype=torch.uint8), z(3, 2, 16, dtype=torch.int16), z(3, 2, 16, dtype=torch.int16))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_append(z(1, 512), z(8, 64), z(1, dtype=I32), z(1, dtype=I32), *cache, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_read(*cache, z(1, dtype=I32), z(1, 2, 64), z(1, 2, 64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_attention(z(1, 4, 64), *cache, z(1, 4, dtype=I32), z(2, dtype=I32), z(1, dtype=I32), z(1, 4, 64), 0.1, z(8, dtype=torch.uint8))
