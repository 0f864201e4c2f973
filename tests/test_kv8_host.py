"""Refusals of the paged 8-bit cache's entry points and of the draft verification, which need no GPU: the C entries look at their arguments before they
touch the device, and the Python functions at their tensors before that."""
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


def plan(lib, requests=4, width=8, npages=32, page=16, ntok=8, null=None):
    p = [P] * 11
    if null is not None:
        p[null] = None
    return lib.qspec_page_plan(*p[:5], requests, width, npages, page, ntok, *p[5:], None)


@pytest.mark.parametrize("kw,what", [(dict(null=0), "null"), (dict(null=4), "null"), (dict(null=8), "null"), (dict(null=10), "null"), (dict(requests=0), "requests"),
                                     (dict(requests=4097), "requests"), (dict(page=48), "pages of"), (dict(page=8), "pages of"), (dict(width=0), "width"),
                                     (dict(width=(1 << 18) + 1), "width"), (dict(npages=0), "pages="), (dict(npages=1 << 27, page=16), "pages="), (dict(ntok=-1), "tokens=")])
def test_page_plan_refuses(lib, kw, what):
    refused(lib, plan(lib, **kw), what)


def append(lib, ptrs=(P,) * 9, ld=(8 + 4) * 128, cos_rows=9, q_ts=8 * 128, ntok=3, H=8, G=2, D=128, npages=9, page=64, dtype=0):
    qkv, cs, pos, slots, k, v, ks, vs, q = ptrs
    return lib.qspec_kv8_append(qkv, ld, cs, cos_rows, pos, slots, k, v, ks, vs, q, q_ts, ntok, H, G, D, npages, page, dtype, None)


@pytest.mark.parametrize("kw,what", [*((dict(ptrs=tuple(None if j == i else P for j in range(9))), "null") for i in range(8)),
                                     *((dict(ptrs=tuple(P + 2 if j == i else P for j in range(9))), "16-byte") for i in (0, 1, 4, 5, 8)),
                                     (dict(D=96), "64 or 128"), (dict(page=256), "pages of"), (dict(G=0), "kv heads"), (dict(npages=0), "pages="), (dict(dtype=2), "float16"),
                                     (dict(ld=100), "16-byte"), (dict(ld=12 * 128 + 4), "16-byte"), (dict(q_ts=64), "16-byte"), (dict(H=0), "heads="), (dict(cos_rows=0), "table rows"),
                                     (dict(ntok=-1), "tokens=")])
def test_append_refuses(lib, kw, what):
    refused(lib, append(lib, **kw), what)


def read(lib, ptrs=(P,) * 7, rows=3, G=2, D=128, npages=9, page=64, dtype=0):
    return lib.qspec_kv8_read(*ptrs, rows, G, D, npages, page, dtype, None)


@pytest.mark.parametrize("kw,what", [*((dict(ptrs=tuple(None if j == i else P for j in range(7))), "null") for i in range(7)),
                                     *((dict(ptrs=tuple(P + 8 if j == i else P for j in range(7))), "16-byte") for i in (0, 1, 5, 6)), (dict(D=32), "64 or 128"),
                                     (dict(rows=-1), "rows"), (dict(rows=1 << 30, G=8), "too many"), (dict(dtype=2), "float16"), (dict(page=0), "pages of")])
def test_read_refuses(lib, kw, what):
    refused(lib, read(lib, **kw), what)


def attend(lib, ptrs=(P,) * 9, q_ts=1024, q_hs=128, o_ts=1024, o_hs=128, ntok=3, requests=2, width=4, H=8, G=2, D=128, npages=9, page=64, most=2, dtype=0, work=P, nbytes=1 << 30):
    q, k, v, ks, vs, table, start, lens, out = ptrs
    return lib.qspec_kv8_attention(q, q_ts, q_hs, k, v, ks, vs, table, start, lens, out, o_ts, o_hs, ntok, requests, width, H, G, D, npages, page, most, 0.1, dtype, work, nbytes,
                                   None)


@pytest.mark.parametrize("kw,what", [*((dict(ptrs=tuple(None if j == i else P for j in range(9))), "null") for i in range(9)),
                                     *((dict(ptrs=tuple(P + 2 if j == i else P for j in range(9))), "16-byte") for i in (0, 1, 2, 8)),
                                     (dict(D=256), "64 or 128"), (dict(page=24), "pages of"), (dict(H=9), "query heads"), (dict(H=1), "query heads"), (dict(G=0), "query heads"),
                                     (dict(q_ts=1023), "16-byte"), (dict(o_hs=4), "16-byte"), (dict(requests=0), "requests="), (dict(width=0), "width="), (dict(most=0), "kv8_attention"),
                                     (dict(ntok=-1), "tokens="), (dict(dtype=2), "float16"), (dict(work=None), "workspace"), (dict(nbytes=1000), "workspace"), (dict(work=P + 4), "workspace")])
def test_attention_refuses(lib, kw, what):
    refused(lib, attend(lib, **kw), what)


def verify(lib, ptrs=(P,) * 6, strides=(3000, 1000, 4000, 1000), requests=2, drafts=3, vocab=1000):
    drafted, draft, target, uniform, tokens, emitted = ptrs
    return lib.qspec_verify_drafts(drafted, draft, strides[0], strides[1], target, strides[2], strides[3], uniform, None, tokens, emitted, requests, drafts, vocab, None)


@pytest.mark.parametrize("kw,what", [*((dict(ptrs=tuple(None if j == i else P for j in range(6))), "null") for i in range(6)), (dict(drafts=32), "at most 31"),
                                     (dict(vocab=0), "vocabulary"), (dict(vocab=1 << 24), "vocabulary"), (dict(requests=-1), "requests"), (dict(strides=(-1, 1, 1, 1)), "stride"),
                                     (dict(strides=(1, 1, 1, -4)), "stride")])
def test_verify_refuses(lib, kw, what):
    refused(lib, verify(lib, **kw), what)


def test_calls_of_nothing_are_no_errors(lib):
    assert append(lib, ntok=0) == 0 and read(lib, rows=0) == 0 and attend(lib, ntok=0) == 0 and verify(lib, requests=0) == 0


def test_python_functions_refuse_tensors_that_are_not_on_a_gpu():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype)  # noqa: E731
    cache = (z(3, 2, 16, 64, dtype=torch.int8), z(3, 2, 16, 64, dtype=torch.int8), z(3, 2), z(3, 2))
    with pytest.raises(ValueError, match="CUDA"):
        ops.page_plan(z(2, dtype=I32), z(2, dtype=I32), z(2, 4, dtype=I32), z(8, dtype=I32), z(3, dtype=I32), 16, z(3, dtype=I32), z(2, dtype=I32), z(5, dtype=I32),
                      z(5, dtype=I32), z(5, dtype=I32), z(4, dtype=I32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_append(z(1, 512), z(8, 64), z(1, dtype=I32), z(1, dtype=I32), *cache, None)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_read(*cache, z(1, dtype=I32), z(1, 2, 64), z(1, 2, 64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv8_attention(z(1, 4, 64), *cache, z(1, 4, dtype=I32), z(2, dtype=I32), z(1, dtype=I32), z(1, 4, 64), 0.1, z(8, dtype=torch.uint8))
    with pytest.raises(ValueError, match="CUDA"):
        ops.verify_drafts(None, None, z(2, 1, 10), z(2, 1), z(2, 1, dtype=torch.int64), z(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="rows"):
        ops.sample_probs(z(2, 10), z(3), z(2, dtype=torch.int64))


@pytest.mark.parametrize("scale", [0.0, -0.1, math.inf, math.nan, 1e-60])
def test_attention_refuses_a_scale_that_is_none(lib, scale):
    assert lib.qspec_kv8_attention(P, 1024, 128, P, P, P, P, P, P, P, P, 1024, 128, 3, 2, 4, 8, 2, 128, 9, 64, 2, scale, 0, P, 1 << 30, None) == 1
    assert "scale must be" in lib.qspec_last_error().decode()
