"""The serving operators' C entry points without a GPU: what they refuse before
they touch a device, and that an empty call does nothing."""
import ctypes

import pytest

A = 1 << 20          # a well-aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    from fp8gq import _lib
    return _lib.load()


def cache(**kw):
    from fp8gq._lib import PagedCache
    d = dict(k=A, v=A, k_page_stride=4096, k_slot_stride=256, k_head_stride=128, v_page_stride=4096, v_slot_stride=256,
             v_head_stride=128, num_pages=4, page_size=16, dtype=0, k_scale=1.0, v_scale=1.0)
    return ctypes.byref(PagedCache(**{**d, **kw}))


def append(lib, c=None, qkv=A, ld=1024, pos=A, slots=A, cs=A, maxp=100, qo=A, ldq=512, ko=None, ldk=0, t=3, hq=4, hkv=2,
           d=128):
    return lib.fp8gq_qk_norm_rope_append(qkv, ld, pos, slots, cs, maxp, None, None, 1e-6, qo, ldq, ko, ldk,
                                         c or cache(), t, hq, hkv, d, None)


def decode(lib, c=None, q=A, qt=512, qh=128, table=A, ldt=8, pages=8, lens=A, out=A, b=2, hq=4, hkv=2, d=128, ws=A,
           n=1 << 30):
    return lib.fp8gq_paged_decode_attention(q, qt, qh, c or cache(), table, ldt, pages, lens, out, 512, 128, None, b, hq,
                                            hkv, d, 0.1, ws, n, None)


def prompt(lib, q=A, qt=512, qh=128, k=A, kt=256, kh=128, cu=A, b=1, tq=9, tk=9, hq=4, hkv=2, d=128):
    return lib.fp8gq_prompt_attention(q, qt, qh, k, kt, kh, A, 256, 128, A, 512, 128, None, cu, A, b, tq, tk, hq, hkv, d,
                                      0.1, 1, A, 1 << 20, None)


def score(lib, x=A, ld=100, dtype=1 * 2, tok=A, t=3, v=100, lp=A, ids=A, tops=A, k=5):
    return lib.fp8gq_token_logprobs(x, ld, dtype, tok, t, v, lp, A, ids, tops, k, None)


def test_append_refuses(lib):
    assert append(lib, qkv=None) == 1 and append(lib, slots=None) == 1 and append(lib, c=cache(k=None)) == 1
    assert append(lib, t=-1) == 2 and append(lib, hq=3) == 2 and append(lib, hkv=0) == 2 and append(lib, maxp=0) == 2
    assert append(lib, c=cache(num_pages=0)) == 2 and append(lib, c=cache(page_size=0)) == 2
    assert append(lib, d=96) == 8 and append(lib, c=cache(dtype=2)) == 8
    assert append(lib, c=cache(dtype=1, k_scale=0.0)) == 8 and append(lib, c=cache(dtype=1, v_scale=float("nan"))) == 8
    assert append(lib, ld=1016) == 4 and append(lib, ldq=500) == 4 and append(lib, ko=A, ldk=128) == 4
    assert append(lib, c=cache(k_head_stride=64)) == 4
    assert append(lib, qkv=A + 8) == 3 and append(lib, ld=1028) == 3 and append(lib, c=cache(v=A + 2)) == 3
    assert append(lib, c=cache(v_slot_stride=260)) == 3
    assert append(lib, t=0, qkv=None, qo=None) == 0


def test_decode_refuses(lib):
    assert decode(lib, q=None) == 1 and decode(lib, table=None) == 1 and decode(lib, lens=None) == 1
    assert decode(lib, b=-1) == 2 and decode(lib, hq=5) == 2 and decode(lib, pages=-1) == 2
    assert decode(lib, d=256) == 8
    assert decode(lib, qt=64) == 4 and decode(lib, qh=64) == 4 and decode(lib, ldt=7) == 4
    assert decode(lib, q=A + 4) == 3 and decode(lib, qt=516) == 3
    assert decode(lib, b=0, q=None, lens=None) == 0


def test_prompt_refuses(lib):
    assert prompt(lib, q=None) == 1 and prompt(lib, k=None) == 1 and prompt(lib, cu=None) == 1
    assert prompt(lib, tq=-1) == 2 and prompt(lib, hq=5) == 2 and prompt(lib, d=80) == 8
    assert prompt(lib, qh=120) == 4 and prompt(lib, kt=100) == 4
    assert prompt(lib, k=A + 2) == 3 and prompt(lib, kt=260) == 3
    assert prompt(lib, tq=0, q=None) == 0 and prompt(lib, b=0) == 0


def test_logprobs_refuses(lib):
    assert score(lib, x=None) == 1 and score(lib, tok=None) == 1 and score(lib, ids=None) == 1
    assert score(lib, t=-1) == 2 and score(lib, v=0) == 2 and score(lib, k=-1) == 2 and score(lib, v=4, k=5) == 2
    assert score(lib, k=33) == 8 and score(lib, dtype=1) == 8
    assert score(lib, ld=99) == 4 and score(lib, x=A + 2) == 3
    assert score(lib, t=0, x=None) == 0


def test_well_formed_calls_need_a_b200(lib):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert append(lib) == 6 and decode(lib) == 6 and prompt(lib) == 6 and score(lib) == 6
