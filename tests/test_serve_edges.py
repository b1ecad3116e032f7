"""The serving operators where values, flags or sizes are unusual.

Bounds are those of test_serve_ops.py, derived there from the kernels' roundings.
"""
import math

import numpy as np
import pytest
import torch

from tests.test_serve_ops import attend64, check_attention, check_logprobs, check_prompt, prompt_case, randn

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def f(cuda_device):
    import fp8gq
    fp8gq.device_error(clear=True)
    yield fp8gq
    torch.cuda.synchronize()
    assert fp8gq.device_error(clear=True) == 0


# --------------------------------------------------------------- logprobs --
@gpu
@pytest.mark.parametrize("t, v", [(6, 777), (6, 50257), (1, 151936)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_lowest_values_beside_ordinary_ones(f, dtype, t, v):
    """A mask of the type's lowest value is a finite logit: its log probability is
    the logit less the row's sum, not -inf."""
    low = torch.finfo(dtype).min
    x = randn(v, t, v, scale=3.0)
    masked = torch.rand(t, v, generator=torch.Generator("cuda").manual_seed(v), device="cuda") < 0.7
    x = x.masked_fill(masked, low).to(dtype)
    x[0, 5:] = low                                        # five left: the alternatives reach the masked
    x[0, :5] = torch.arange(5, device="cuda").to(dtype)
    tokens = masked.int().argmax(1)                       # of each row a masked one
    tokens[0] = v - 1
    if t > 3:
        x[2, 9], tokens[2] = -2.4e38, 9                   # x log2(e) leaves fp32, x does not
        x[3, 11] = -math.inf
    r = check_logprobs(f, x, tokens, 20)
    assert r.logprobs.isfinite().all() and r.top_logprobs[0].isfinite().all()


# ----------------------------------------------------------------- decode --
def check_e4m3_decode(f, q, k, v, scale):
    """q [1, Hq, D], k and v [N, Hkv, D] in pages of 16."""
    n, hkv, d = k.shape
    pages = (n + 15) // 16
    cache = torch.zeros(2, pages * 16, hkv, d, device="cuda")
    cache[0, :n], cache[1, :n] = k, v
    kc, vc = (c.view(pages, 16, hkv, d).to(torch.float8_e4m3fn) for c in cache)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    out, lse = f.paged_decode_attention(q, kc, vc, table, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=scale,
                                        return_lse=True)
    seen = torch.ones(1, n, dtype=torch.bool, device="cuda")
    check_attention(out, lse, *attend64(q, kc.view(-1, hkv, d)[:n].double(), vc.view(-1, hkv, d)[:n].double(), scale, seen))


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("drop", [5.0, 14.7, 20.3, 24.6, 26.0, 28.9])
def test_decode_e4m3_faint_tokens_count(f, d, drop):
    """One token in 16 has all the weight and v = 0, the others 2^-drop of it each
    and v = 1: what they add is the output."""
    n, hq, hkv = 1000, 8, 2
    q = torch.zeros(1, hq, d, device="cuda", dtype=torch.bfloat16)
    q[:, :, 0] = 1
    k, v = torch.zeros(n, hkv, d, device="cuda"), torch.ones(n, hkv, d, device="cuda")
    k[::16, :, 0], v[::16] = 8, 0
    check_e4m3_decode(f, q, k, v, drop * math.log(2) / 8)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("most", [2.0 ** 12, 2.0 ** 20, 2.0 ** 26])
def test_decode_e4m3_one_large_query_value(f, d, most):
    """A value of q that no key meets: the others give the scores, at full accuracy."""
    n, hq, hkv = 700, 16, 2
    q = randn(1, 1, hq, d).bfloat16()
    k, v = randn(2, n, hkv, d, scale=2.0), randn(3, n, hkv, d)
    q[:, :, 3], k[:, :, 3] = most, 0
    check_e4m3_decode(f, q, k, v, d ** -0.5)


# ----------------------------------------------------------------- prompt --
@gpu
@pytest.mark.parametrize("d, n", [(64, 300), (128, 300), (128, 4000)])
def test_prompt_large_values_behind_a_growing_maximum(f, d, n):
    """Scores that grow by 2^55 from one part of the keys to the next, and values of
    1e25 or 1e30: the weighted sums stay in range as long as the values do."""
    q = torch.zeros(40, 4, d, device="cuda")
    q[:, :, 0] = 1
    k, v = torch.zeros(n, 1, d, device="cuda"), randn(n, n, 1, d, scale=1e25)
    k[n // 2:, :, 0] = 38.0
    v[::7] *= 1e5
    cu = lambda m: torch.tensor([0, m], dtype=torch.int32, device="cuda")  # noqa: E731
    check_prompt(f, q.bfloat16(), k.bfloat16(), v.bfloat16(), cu(40), cu(n), scale=1.0)


@gpu
@pytest.mark.parametrize("with_out", [False, True])
def test_prompt_split_call_has_scratch_of_its_own(f, with_out):
    """A split call's two launches share nothing that another thread's launch between
    them could use: the scratch of the stream is as it was."""
    from fp8gq import ops
    q, k, v, cu_q, cu_k = prompt_case(21, [64], [6000], 16, 1, 128)
    dev, stream = torch.device("cuda", 0), torch.cuda.current_stream().cuda_stream
    assert f._lib.load().fp8gq_prompt_split_bytes(1, q.shape[0], k.shape[0], 16, 1, 128, 1) > 0
    scratch = ops.workspace(dev, 48 << 20, stream)
    scratch[16384:] = 0x5a
    out = torch.empty_like(q) if with_out else None
    f.prompt_attention(q, k, v, cu_q, cu_k, out=out)
    same = (scratch[16384:] == 0x5a).all() and (scratch[:16384] == 0).all()
    scratch.zero_()
    assert same


@gpu
def test_two_threads_on_one_stream(f):
    """One thread's split prompts and another's decodes, linears and split prompts."""
    import threading

    from tests.test_serve_ops import decode_case
    from tests.test_zz_no_alloc import _operands
    q, k, v, cu_q, cu_k = prompt_case(22, [40, 3], [3100, 2500], 8, 2, 128)
    q2, k2, v2, cu_q2, cu_k2 = prompt_case(23, [9], [4000], 4, 4, 64)
    kc, vc, table, ln = decode_case(24, [3000, 50], 2, 128, 16, torch.bfloat16)
    qd = randn(8, 2, 8, 128).bfloat16()
    x, wq, ws = _operands(4, 4096, 6144, 1, "cuda")
    calls = [lambda: f.prompt_attention(q, k, v, cu_q, cu_k), lambda: f.paged_decode_attention(qd, kc, vc, table, ln),
             lambda: f.fused_gemv_quant(x, wq, ws), lambda: f.prompt_attention(q2, k2, v2, cu_q2, cu_k2)]
    rows = [slice(0, 43), slice(None), slice(None), slice(0, 9)]
    prev = f.set_tm_options(f.TM_WORKSPACE_SPLITK)
    wrong, stream = [], torch.cuda.Stream()
    try:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            want = [c()[r].clone() for c, r in zip(calls, rows)]

        def run(which, out):
            with torch.cuda.stream(stream):
                got = []
                for _ in range(200):
                    for i in which:
                        if i == 0 and out:          # the path that lets go of the interpreter's lock
                            o = torch.empty_like(q)
                            f.prompt_attention(q, k, v, cu_q, cu_k, out=o)
                        else:
                            o = calls[i]()
                        got.append((i, o))
                wrong.extend(i for i, o in got if not torch.equal(o[rows[i]], want[i]))

        threads = [threading.Thread(target=run, args=a) for a in (([0], True), ([1, 2, 3], False))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        f.set_tm_options(prev)
    stream.synchronize()
    assert not wrong


# ------------------------------------------------------------------ flags --
@gpu
@pytest.mark.parametrize("yes", [1, np.bool_(True), "yes"])
@pytest.mark.parametrize("no", [0, np.bool_(False), None])
def test_flags_by_truth(f, yes, no):
    """return_lse, return_k and causal count by their truth, as everywhere in Python."""
    q, k, v, cu, _ = prompt_case(3, [5, 4], [5, 4], 4, 2, 64, spare=0)
    out, lse = f.prompt_attention(q, k, v, cu, return_lse=yes)
    assert out.shape == (9, 4, 64) and lse.shape == (9, 4)
    assert torch.equal(f.prompt_attention(q, k, v, cu, return_lse=no), out)
    assert torch.equal(f.prompt_attention(q, k, v, cu, causal=yes), out)
    assert torch.equal(f.prompt_attention(q, k, v, cu, causal=no), f.prompt_attention(q, k, v, cu, causal=False))
    kc = randn(4, 3, 4, 2, 64).bfloat16()
    table, lens = torch.tensor([[0, 1], [2, 1]], dtype=torch.int32, device="cuda"), torch.tensor([5, 8], dtype=torch.int32, device="cuda")
    o, s = f.paged_decode_attention(q[:2], kc, kc, table, lens, return_lse=yes)
    assert o.shape == (2, 4, 64) and s.shape == (2, 4)
    assert torch.equal(f.paged_decode_attention(q[:2], kc, kc, table, lens, return_lse=no), o)
    qkv, at = randn(5, 2, 8 * 64).bfloat16(), torch.arange(2, device="cuda")
    cs = torch.ones(4, 64, device="cuda")
    a, b = f.qk_norm_rope_append(qkv, at, at, cs, kc, kc.clone(), return_k=yes)
    assert a.shape == (2, 4, 64) and b.shape == (2, 2, 64)
    assert torch.equal(f.qk_norm_rope_append(qkv, at, at, cs, kc, kc.clone(), return_k=no), a)


# ----------------------------------------------------------- bounded waits --
@pytest.fixture
def shortest_limit(f):
    """Every bounded wait at its shortest limit (2 ms inside a kernel)."""
    torch.cuda.synchronize()
    prev = f.set_wait_limit_ns(1_000_000)
    yield
    torch.cuda.synchronize()
    f.set_wait_limit_ns(prev)
    f.device_error(clear=True)


@gpu
@pytest.mark.parametrize("t, v, k", [(1, 151936, 32), (37, 151936, 20), (700, 50257, 0), (1500, 4099, 3)])
def test_logprobs_under_the_shortest_limit(f, shortest_limit, t, v, k):
    """No ordinary wait comes near the limit, so none is given up, whatever the
    number of steps; the same row twice gives the same bits."""
    x = randn(t, t, v, scale=3.0)
    tokens = torch.arange(t, device="cuda") % v
    r = f.token_logprobs(x, tokens, top_k=k)
    torch.cuda.synchronize()
    assert f.device_error() == 0
    check_logprobs(f, x[:40], tokens[:40], k)
    assert all(torch.equal(a, b) for a, b in zip(r, f.token_logprobs(x, tokens, top_k=k)))


@gpu
@pytest.mark.parametrize("d, keys", [(128, 400_000), (64, 700_000)])
@pytest.mark.parametrize("rounds", [1, 2])
def test_prompt_items_longer_than_the_limit(f, shortest_limit, d, keys, rounds):
    """Whole items that take longer than the limit (some 6 ms against 2): the wait for the next
    item is given up and reported, the call ends, and the next one is right."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sms % 4 == 0
    n = rounds * sms // 4 * 256                            # an item for each SM and round
    q = randn(1, n, 4, d).bfloat16()
    k, v = randn(2, keys, 4, d).bfloat16(), randn(3, keys, 4, d).bfloat16()
    cu = lambda m: torch.tensor([0, m], dtype=torch.int32, device="cuda")  # noqa: E731
    cu_q, cu_k = cu(n), cu(keys)
    assert f._lib.load().fp8gq_prompt_split_bytes(1, n, keys, 4, 4, d, 0) == 0
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    out = f.prompt_attention(q, k, v, cu_q, cu_k, causal=False)
    end.record()
    end.synchronize()
    assert f.device_error(clear=True) == 0x80000000 | 11
    assert start.elapsed_time(end) < 100
    # the items that were begun are whole: the last rows of the sequence are the first
    check_attention(out[-40:, 1:2], None, *attend64(q[-40:, 1:2], k[:, 1:2], v[:, 1:2], d ** -0.5,
                                                    torch.ones(40, keys, dtype=torch.bool, device="cuda")))
    a, b, c, cu_a, _ = prompt_case(5, [900, 77, 2000], [900, 77, 2000], 8, 2, d)
    check_prompt(f, a, b, c, cu_a, None)
    assert f.device_error() == 0


@gpu
def test_decode_of_the_longest_sequence(f):
    """2^31 - 1 tokens (two pages in turn) beside 5: the sums of a lane have at most
    2^31 / (2 * 148 * 4 warps * 8 lanes) additions, those of o half as many, each
    within 2^-23, which bounds what they may be off by."""
    d, page = 64, 1 << 16
    kc, vc = randn(1, 2, page, 1, d).bfloat16(), randn(2, 2, page, 1, d).bfloat16()
    table = (torch.arange(2 ** 31 // page + 1, device="cuda") % 2).int().repeat(2, 1)
    lens = torch.tensor([2 ** 31 - 1, 5], dtype=torch.int32, device="cuda")
    q = randn(3, 2, 4, d).bfloat16()
    out, lse = f.paged_decode_attention(q, kc, vc, table, lens, return_lse=True)
    k, v = kc.view(-1, 1, d), vc.view(-1, 1, d)
    times = 2 ** 31 // (2 * page)
    ref, a, l64, size = attend64(q[:1], k, v, d ** -0.5, torch.ones(1, 2 * page, dtype=torch.bool, device="cuda"))
    off = 2 ** 31 / (2 * 148 * 4 * 8) * 2.0 ** -23
    # (the token that is missing weighs less than 2^-31 e^size)
    assert ((out[:1].double() - ref).abs() <= (2 * 2.0 ** -8 + off) * a + 2.0 ** -8 * ref.abs()).all()
    assert ((lse[:1].double() - l64 - math.log(times)).abs() <= off + 2.0 ** -16 * (1 + size)).all()
    check_attention(out[1:], lse[1:], *attend64(q[1:], k[:5], v[:5], d ** -0.5, torch.ones(1, 5, dtype=torch.bool, device="cuda")))


# ---------------------------------------------------------------- layouts --
def heads_first(t):
    """The same [tokens, heads, D] values laid out [heads, tokens, D]."""
    return t.transpose(0, 1).contiguous().transpose(0, 1)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq, lk", [([70, 1, 200], [70, 1, 200]), ([9], [5000])])
def test_prompt_heads_before_tokens(f, d, lq, lk):
    q, k, v, cu_q, cu_k = prompt_case(31, lq, lk, 8, 2, d)
    want, lse = check_prompt(f, q, k, v, cu_q, cu_k)
    n = sum(lq)
    out = heads_first(torch.zeros_like(q))
    got, l2 = f.prompt_attention(heads_first(q), heads_first(k), heads_first(v), cu_q, cu_k, out=out, return_lse=True)
    assert torch.equal(got[:n], want[:n]) and torch.equal(l2[:n], lse[:n])
    assert torch.equal(f.prompt_attention(heads_first(q), k, heads_first(v), cu_q, cu_k)[:n], want[:n])


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("order", [(0, 2, 1, 3), (2, 0, 1, 3), (1, 2, 0, 3)])
def test_cache_layouts(f, dtype, order):
    """Pages, slots and heads in other orders: append and decode as in the plain one."""
    pages, page, hkv, d, hq = 7, 16, 2, 128, 8
    k0, v0 = (randn(i, pages, page, hkv, d).to(dtype) for i in (1, 2))

    def laid(t):
        back = [order.index(i) for i in range(4)]
        return t.view(torch.uint8).permute(*order).contiguous().permute(*back).view(dtype)

    k1, v1 = laid(k0), laid(v0)
    assert not k1.is_contiguous()
    qkv, pos = randn(3, 5, (hq + 2 * hkv) * d).bfloat16(), torch.arange(5, device="cuda")
    slots, cs = torch.tensor([0, 33, 111, -1, 64], device="cuda"), randn(4, 9, d)
    a = f.qk_norm_rope_append(qkv, pos, slots, cs, k0, v0, k_scale=0.5, v_scale=0.25)
    b = f.qk_norm_rope_append(qkv, pos, slots, cs, k1, v1, k_scale=0.5, v_scale=0.25)
    bits = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731
    assert torch.equal(a, b) and torch.equal(bits(k0), bits(k1)) and torch.equal(bits(v0), bits(v1))
    table = torch.tensor([[3, 0, 5], [6, 1, 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([41, 20], dtype=torch.int32, device="cuda")
    q = heads_first(a[:2])
    want = f.paged_decode_attention(a[:2], k0, v0, table, lens, return_lse=True)
    got = f.paged_decode_attention(q, k1, v1, table, lens, out=heads_first(torch.zeros_like(a[:2])), return_lse=True)
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@gpu
def test_heads_that_share_memory_are_refused(f):
    """Broadcast heads (stride 0) have no place of their own: refused, not misread."""
    q, k, v, cu, _ = prompt_case(32, [20], [20], 4, 1, 64, spare=0)
    with pytest.raises(f.Fp8gqError):
        f.prompt_attention(q, k.expand(20, 4, 64), v.expand(20, 4, 64), cu)
    with pytest.raises(f.Fp8gqError):
        f.prompt_attention(q, k, v, cu, out=torch.zeros(20, 1, 64, dtype=torch.bfloat16, device="cuda").expand(20, 4, 64))
