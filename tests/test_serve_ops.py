"""The serving operators against plain implementations in 64 bits.

Tolerances are derived, per element, from the kernels' roundings:

  u = 2^-8      half an ulp of bf16 (8 significant bits), relative: the rounding of an output, and of a
                softmax weight where the weights meet v in bf16
  attention     |o - o64| <= u |o64| + u A + 2^-12 A,  A = sum_j p_j |v_j|: the
                output's rounding, the weights' (each at most u of itself), and
                the fp32 errors of scores and sums
  lse           2^-16 (1 + max_j scale sum_d |q_d k_jd|): D fp32 additions of the
                largest score, exponentials and a sum of positive terms
  logprob       r = (V / 256 + 64) 2^-24 + 2^-20 relative in a sum of V positive
                terms (a thread's own additions, then a tree; the exponential),
                plus 2^-22 (|x| + |lse|) for the roundings of the difference
  entropy       (2 r + 2^-22) (1 + entropy): log s and sum p |x - m| <= entropy, each within r, and a few roundings
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


@pytest.fixture(scope="module")
def f(cuda_device):
    import fp8gq
    fp8gq.device_error(clear=True)
    yield fp8gq
    torch.cuda.synchronize()
    assert fp8gq.device_error(clear=True) == 0


def randn(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale


def attend64(q, k, v, scale, visible):
    """q [Lq, Hq, D], k and v [Lk, Hkv, D]; visible [Lq, Lk] -> out, A, lse, largest score's size."""
    q, k, v = q.double(), k.double(), v.double()
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    if k.shape[0] == 0:
        z = torch.zeros_like(q)
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
        return z, z, lse, torch.zeros_like(lse)
    s = torch.einsum("qhd,khd->qhk", q, k) * scale
    s = s.masked_fill(~visible[:, None], -math.inf)
    size = torch.einsum("qhd,khd->qhk", q.abs(), k.abs()).amax(-1) * abs(scale)
    lse = torch.logsumexp(s, -1)
    p = torch.where(lse[..., None] == -math.inf, 0.0, (s - lse[..., None]).exp())
    p = torch.nan_to_num(p, nan=0.0)
    return torch.einsum("qhk,khd->qhd", p, v), torch.einsum("qhk,khd->qhd", p, v.abs()), lse, size


def check_attention(out, lse, ref, a, lse64, size):
    err = (out.double() - ref).abs()
    bound = U * ref.abs() + (U + 2.0 ** -12) * a + 1e-30
    assert torch.isfinite(out.float()).all()
    assert (err <= bound).all(), f"worst {(err / bound).max().item():.3g} of the bound"
    if lse is not None:
        none = lse64 == -math.inf
        assert (lse[none] == -math.inf).all()
        e = (lse.double() - lse64).abs()[~none]
        b = (2.0 ** -16 * (1 + size))[~none]
        assert (e <= b).all(), f"lse: worst {(e / b).max().item():.3g} of the bound"


# ----------------------------------------------------------------- append --
def append_case(seed, t, hq, hkv, d, page, dtype, pages=None, max_pos=4096):
    qkv = randn(seed, t, (hq + 2 * hkv) * d).bfloat16()
    pages = pages or (t + page - 1) // page + 1
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    pos = torch.randint(0, max_pos, (t,), generator=g, device="cuda")
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:t]
    ang = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * \
        1e4 ** (-torch.arange(d // 2, device="cuda", dtype=torch.float64) * 2 / d)
    cs = torch.cat([ang.cos(), ang.sin()], 1).float()
    kc = randn(seed + 2, pages, page, hkv, d).to(dtype)
    vc = randn(seed + 3, pages, page, hkv, d).to(dtype)
    qw, kw = (1 + 0.3 * randn(seed + 4, d)).bfloat16(), (1 + 0.3 * randn(seed + 5, d)).bfloat16()
    return qkv, pos, slots, cs, kc, vc, qw, kw


def append64(x, w, cs, eps=1e-6):
    """x [T, H, D] -> normed and rotated, and a bound on the fp32 error of each value."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    d = x.shape[-1]
    c, s = cs.double()[:, None, :d // 2], cs.double()[:, None, d // 2:]
    a, b = x[..., :d // 2], x[..., d // 2:]
    size = (a.abs() + b.abs()).repeat(1, 1, 2)
    return torch.cat([a * c - b * s, b * c + a * s], -1), size * 2.0 ** -19


@pytest.mark.parametrize("t, hq, hkv, d, page", [(1, 32, 8, 128, 16), (3, 1, 1, 64, 1), (37, 16, 2, 64, 32),
                                                 (130, 10, 2, 128, 64), (5, 7, 7, 128, 3), (257, 32, 8, 128, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("norm", [True, False])
def test_append(f, t, hq, hkv, d, page, dtype, norm):
    qkv, pos, slots, cs, kc, vc, qw, kw = append_case(7 * t + d, t, hq, hkv, d, page, dtype)
    if not norm:
        qw = kw = None
    ks, vs = (0.04, 0.03) if dtype != torch.bfloat16 else (1.0, 1.0)
    if t > 2:
        slots[1] = -1
        slots[2] = -7
    k0, v0 = kc.clone(), vc.clone()
    q, k = f.qk_norm_rope_append(qkv, pos, slots, cs, kc, vc, q_weight=qw, k_weight=kw, k_scale=ks, v_scale=vs,
                                 return_k=True)
    x = qkv.view(t, hq + 2 * hkv, d)
    for got, ref in ((q, append64(x[:, :hq], qw, cs[pos])), (k, append64(x[:, hq:hq + hkv], kw, cs[pos]))):
        assert ((got.double() - ref[0]).abs() <= U * ref[0].abs() * 1.01 + ref[1]).all()
    # the cache: untouched except at the slots, v exact, k within one rounding of its type
    held = slots >= 0
    rest = torch.ones(kc.shape[0] * page, dtype=torch.bool, device="cuda")
    rest[slots[held]] = False
    bits = torch.uint8 if dtype != torch.bfloat16 else torch.int16
    flat = lambda c: c.view(bits).view(-1, hkv, d)  # noqa: E731
    assert torch.equal(flat(kc)[rest], flat(k0)[rest]) and torch.equal(flat(vc)[rest], flat(v0)[rest])
    v = x[:, hq + hkv:].float()
    v = (v / vs).clamp(-448, 448).to(dtype) if dtype != torch.bfloat16 else v.to(dtype)
    assert torch.equal(flat(vc)[slots[held]], v.view(bits)[held])
    ref, tol = append64(x[:, hq:hq + hkv], kw, cs[pos])
    got = kc.view(-1, hkv, d)[slots[held]].double() * ks
    if dtype == torch.bfloat16:
        assert ((got - ref[held]).abs() <= U * ref[held].abs() * 1.01 + tol[held]).all()
    else:
        # half an e4m3 ulp: 2^-4 relative, 2^-10 of the scale below the normal range
        ref = ref.clamp(-448 * ks, 448 * ks)
        assert ((got - ref[held]).abs() <= ref[held].abs() * 2.0 ** -4 + ks * 2.0 ** -10 + 2 * tol[held]).all()


def test_append_in_place_strided_cache_and_extremes(f):
    t, hq, hkv, d, page = 40, 8, 2, 128, 8
    qkv, pos, slots, cs, _, _, qw, kw = append_case(3, t, hq, hkv, d, page, torch.bfloat16)
    qkv[0] = 0                                    # a head of zeros: norm by eps alone
    qkv[1] = 1e30
    both = torch.zeros(8, 2, page, hkv, d + 16, dtype=torch.bfloat16, device="cuda")   # k and v interleaved, padded heads
    kc, vc = both[:, 0, :, :, :d], both[:, 1, :, :, :d]
    want_q = f.qk_norm_rope_append(qkv, pos, slots, cs, kc, vc, q_weight=qw, k_weight=kw).clone()
    want = both.clone()
    both.zero_()
    x = qkv.view(t, -1, d)
    q = f.qk_norm_rope_append(qkv, pos, slots, cs, kc, vc, q_weight=qw, k_weight=kw, q_out=x[:, :hq],
                              k_out=x[:, hq:hq + hkv])
    assert torch.equal(q, want_q) and torch.equal(both, want)
    assert torch.equal(both[..., d:], torch.zeros_like(both[..., d:]))
    assert (q[0] == 0).all()
    assert torch.equal(x[2:, hq:hq + hkv], torch.stack([kc[s // page, s % page] for s in slots.tolist()])[2:])


def test_append_out_of_range_is_recorded(f):
    qkv, pos, slots, cs, kc, vc, qw, kw = append_case(5, 6, 4, 2, 64, 4, torch.bfloat16)
    k0 = kc.clone()
    slots[2] = kc.shape[0] * 4
    f.qk_norm_rope_append(qkv, pos, slots, cs, kc, vc, q_weight=qw, k_weight=kw)
    assert f.device_error(clear=True) & 0xFFFF == 12
    keep = torch.ones(kc.shape[0] * 4, dtype=torch.bool, device="cuda")
    keep[torch.cat([slots[:2], slots[3:]])] = False
    assert torch.equal(kc.view(-1, 2, 64)[keep], k0.view(-1, 2, 64)[keep])
    slots[2], pos[0] = -1, cs.shape[0]
    f.qk_norm_rope_append(qkv, pos, slots, cs, kc, vc, q_weight=qw, k_weight=kw)
    assert f.device_error(clear=True) & 0xFFFF == 12
    assert f.qk_norm_rope_append(qkv[:0], pos[:0], slots[:0], cs, kc, vc).shape == (0, 4, 64)


# ----------------------------------------------------------------- decode --
def decode_case(seed, lens, hkv, d, page, dtype, pages=None):
    """A cache whose unused slots and pages are NaN, and a table whose unused entries are -1."""
    need = [(n + page - 1) // page for n in lens]
    total = pages or sum(need) + 2
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = (total - 1 - torch.randperm(sum(need) + 1, generator=g, device="cuda")).tolist()
    width = max(need + [1]) + 1
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    kc = torch.full((total, page, hkv, d), math.nan, device="cuda", dtype=torch.bfloat16).to(dtype)
    vc = kc.clone()
    at = 0
    for b, n in enumerate(lens):
        for c in range(need[b]):
            table[b, c] = ids[at]
            m = min(page, n - c * page)
            kc[ids[at], :m] = randn(seed + 31 * at + 1, m, hkv, d, scale=2.0).clamp(-440, 440).to(dtype)
            vc[ids[at], :m] = randn(seed + 31 * at + 2, m, hkv, d).clamp(-440, 440).to(dtype)
            at += 1
    return kc, vc, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def check_decode(f, q, kc, vc, table, lens, ks=1.0, vs=1.0, scale=None):
    out, lse = f.paged_decode_attention(q, kc, vc, table, lens, return_lse=True, k_scale=ks, v_scale=vs, scale=scale)
    d, page = q.shape[2], kc.shape[1]
    scale = d ** -0.5 if scale is None else scale
    for b, n in enumerate(lens.tolist()):
        ids = table[b, :(n + page - 1) // page].long()
        k = kc[ids].reshape(-1, kc.shape[2], d)[:n].double() * ks
        v = vc[ids].reshape(-1, kc.shape[2], d)[:n].double() * vs
        seen = torch.ones(1, n, dtype=torch.bool, device="cuda")
        check_attention(out[b:b + 1], lse[b:b + 1], *attend64(q[b:b + 1], k, v, scale, seen))
    return out, lse


@pytest.mark.parametrize("lens", [[1], [0], [2, 0, 1], [15, 16, 17, 31, 32, 33], [63, 64, 65, 0, 127, 128, 129],
                                  [1000, 3, 513, 77], [2049]])
@pytest.mark.parametrize("hq, hkv, d, page", [(32, 8, 128, 16), (8, 8, 64, 1), (5, 1, 128, 64), (32, 2, 64, 7)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_decode(f, lens, hq, hkv, d, page, dtype):
    kc, vc, table, ln = decode_case(sum(lens) + hq, lens, hkv, d, page, dtype)
    q = randn(1, len(lens), hq, d, scale=1.5).bfloat16()
    s = (0.5, 0.25) if dtype != torch.bfloat16 else (1.0, 1.0)
    check_decode(f, q, kc, vc, table, ln, *s)


@pytest.mark.parametrize("hq, hkv", [(1, 1), (2, 1), (3, 1), (7, 1), (8, 1), (9, 1), (16, 1), (17, 1), (40, 2), (64, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_decode_groups(f, hq, hkv, dtype):
    kc, vc, table, ln = decode_case(hq, [300, 41, 700], hkv, 128, 16, dtype)
    check_decode(f, randn(2, 3, hq, 128).bfloat16(), kc, vc, table, ln)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_decode_long_and_many(f, dtype):
    kc, vc, table, ln = decode_case(11, [20011, 1], 2, 128, 64, dtype)
    check_decode(f, randn(3, 2, 8, 128).bfloat16(), kc, vc, table, ln)
    lens = [int(x) for x in np.random.RandomState(0).randint(0, 400, 300)]
    kc, vc, table, ln = decode_case(12, lens, 1, 64, 32, dtype)
    check_decode(f, randn(4, 300, 4, 64).bfloat16(), kc, vc, table, ln)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_decode_sharp_and_extreme_scores(f, dtype):
    """Scores in the hundreds (weights that underflow, a late maximum), zero and large queries, other scales."""
    kc, vc, table, ln = decode_case(13, [700, 700, 700], 2, 128, 16, dtype)
    q = randn(5, 3, 8, 128).bfloat16()
    q[0] *= 40
    q[1] = 0
    check_decode(f, q, kc, vc, table, ln)
    check_decode(f, q, kc, vc, table, ln, scale=-0.3)
    check_decode(f, (q[:1] * 2000).repeat(3, 1, 1), kc, vc, table, ln, scale=1e-5)
    check_decode(f, (q[:1] * 1e-6).repeat(3, 1, 1), kc, vc, table, ln, scale=1e4)


def test_decode_strides_streams_and_repeats(f):
    lens = [333, 90, 1, 0, 512]
    kc, vc, table, ln = decode_case(17, lens, 2, 128, 16, torch.bfloat16)
    both = torch.stack([kc, vc], 3)                       # [pages, page, heads, 2, D]
    kc, vc = both[:, :, :, 0], both[:, :, :, 1]
    qkv = randn(6, 5, 12, 128).bfloat16()
    wide = torch.full((5, table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    out, lse = check_decode(f, qkv[:, :8], kc, vc, wide[:, :table.shape[1]], ln)
    buf = torch.zeros(5, 10, 128, dtype=torch.bfloat16, device="cuda")
    f.paged_decode_attention(qkv[:, :8], kc, vc, table, ln, out=buf[:, 1:9])
    assert torch.equal(buf[:, 1:9], out) and (buf[:, 0] == 0).all() and (buf[:, 9] == 0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):                               # the same bits every time
            o, l = f.paged_decode_attention(qkv[:, :8], kc, vc, table, ln, return_lse=True)
            assert torch.equal(o, out) and torch.equal(l, lse)
    torch.cuda.current_stream().wait_stream(side)


def test_decode_in_a_graph_with_changing_lengths(f):
    """A captured step replayed while the lengths, pages and values move on."""
    kc, vc, table, ln = decode_case(19, [400, 400, 400], 2, 64, 16, torch.bfloat16)
    q = randn(7, 3, 16, 64).bfloat16()
    f.paged_decode_attention(q, kc, vc, table, ln, return_lse=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = f.paged_decode_attention(q, kc, vc, table, ln, return_lse=True)
    for lens in ([1, 400, 0], [257, 3, 399], [0, 0, 0]):
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(randn(sum(lens), 3, 16, 64).bfloat16())
        g.replay()
        want = f.paged_decode_attention(q, kc, vc, table, ln, return_lse=True)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        check_decode(f, q, kc, vc, table, ln)


def test_decode_between_tile_kernel_calls(f):
    """The workspace it shares with the linears stays good for both."""
    from tests.test_zz_no_alloc import _operands
    kc, vc, table, ln = decode_case(23, [3000, 50], 2, 128, 16, torch.bfloat16)
    q = randn(8, 2, 8, 128).bfloat16()
    x, wq, ws = _operands(4, 4096, 6144, 1, "cuda")
    a0, b0 = f.fused_gemv_quant(x, wq, ws), f.paged_decode_attention(q, kc, vc, table, ln)
    prev = f.set_tm_options(f.TM_WORKSPACE_SPLITK)
    try:
        c0 = f.fused_gemv_quant(x, wq, ws)
        for _ in range(5):
            assert torch.equal(f.paged_decode_attention(q, kc, vc, table, ln), b0)
            assert torch.equal(f.fused_gemv_quant(x, wq, ws), c0)
    finally:
        f.set_tm_options(prev)
    assert torch.equal(a0, c0)


def test_decode_offsets_past_32_bits(f):
    page, hkv, d = 16, 8, 128
    pages = 2 ** 32 // (page * hkv * d) + 8              # more than 2^32 elements
    kc = torch.empty(pages, page, hkv, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    lens = [50, 20]
    need = torch.tensor([[pages - 1, 3, pages - 2, pages // 2 + 1], [pages // 2, pages - 5, -1, -1]], dtype=torch.int32)
    for i in need.unique().tolist():
        if i >= 0:
            kc[i], vc[i] = randn(i, page, hkv, d), randn(i + 1, page, hkv, d)
    check_decode(f, randn(9, 2, 16, d).bfloat16(), kc, vc, need.cuda(),
                 torch.tensor(lens, dtype=torch.int32, device="cuda"))
    t = 3
    qkv, pos, _, cs, _, _, qw, kw = append_case(5, t, 16, hkv, d, page, torch.bfloat16)
    slots = torch.tensor([pages * page - 1, 5, (pages // 2) * page + 3], device="cuda")
    _, k = f.qk_norm_rope_append(qkv, pos, slots, cs, kc, vc, q_weight=qw, k_weight=kw, return_k=True)
    assert torch.equal(kc.view(-1, hkv, d)[slots], k)
    assert torch.equal(vc.view(-1, hkv, d)[slots], qkv.view(t, -1, d)[:, 16 + hkv:])


def test_decode_out_of_range_is_recorded(f):
    kc, vc, table, ln = decode_case(29, [100, 60], 2, 128, 16, torch.bfloat16)
    q = randn(10, 2, 8, 128).bfloat16()
    good = f.paged_decode_attention(q, kc, vc, table, ln)
    bad = table.clone()
    bad[1, 1] = kc.shape[0]
    out = f.paged_decode_attention(q, kc, vc, bad, ln)
    assert f.device_error(clear=True) & 0xFFFF == 12
    assert torch.equal(out[0], good[0])
    # the page counts as absent
    ids = table[1, [0, 2, 3]].long()
    k, v = (c[ids].reshape(-1, 2, 128)[:44] for c in (kc, vc))
    check_attention(out[1:], None, *attend64(q[1:], k, v, 128 ** -0.5, torch.ones(1, 44, dtype=torch.bool, device="cuda")))
    ln[0] = table.shape[1] * 16 + 1
    f.paged_decode_attention(q[:, :], kc, vc, table.clamp(min=0), ln)
    assert f.device_error(clear=True) & 0xFFFF == 12
    assert f.paged_decode_attention(q[:0], kc, vc, table[:0], ln[:0]).shape == (0, 8, 128)


# ----------------------------------------------------------------- prompt --
def prompt_case(seed, lq, lk, hq, hkv, d, spare=3):
    """Packed q, k, v with NaN rows after the last sequence."""
    cu = lambda n: torch.tensor([0] + n, device="cuda").cumsum(0).to(torch.int32)  # noqa: E731
    q, k, v = (randn(seed + i, sum(n) + spare, h, d, scale=s).bfloat16()
               for i, (n, h, s) in enumerate(((lq, hq, 1.5), (lk, hkv, 1.0), (lk, hkv, 1.0))))
    for t, n in ((q, lq), (k, lk), (v, lk)):
        t[sum(n):] = math.nan
    return q, k, v, cu(lq), cu(lk)


def check_prompt(f, q, k, v, cu_q, cu_k, causal=True, scale=None, **kw):
    out, lse = f.prompt_attention(q, k, v, cu_q, cu_k, causal=causal, scale=scale, return_lse=True, **kw)
    s = q.shape[2] ** -0.5 if scale is None else scale
    a, b = cu_q.tolist(), (cu_q if cu_k is None else cu_k).tolist()
    for i in range(len(a) - 1):
        n, m = a[i + 1] - a[i], b[i + 1] - b[i]
        if n == 0:
            continue
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril(m - n)
        for j in range(0, n, 512):
            r = slice(a[i] + j, min(a[i + 1], a[i] + j + 512))
            check_attention(out[r], lse[r], *attend64(q[r], k[b[i]:b[i + 1]], v[b[i]:b[i + 1]], s, seen[j:j + 512]))
    return out, lse


@pytest.mark.parametrize("lq, lk", [([1], None), ([1, 2, 3], None), ([127, 128, 129], None), ([300, 0, 5, 64], None),
                                    ([255, 256, 257], None), ([513, 1, 31], None),
                                    ([1, 17, 128], [200, 17, 400]), ([100, 5], [30, 0]), ([300], [129]),
                                    ([130, 70], [1000, 129])])
@pytest.mark.parametrize("hq, hkv, d", [(4, 2, 128), (3, 3, 64), (8, 1, 64), (5, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt(f, lq, lk, hq, hkv, d, causal):
    q, k, v, cu_q, cu_k = prompt_case(sum(lq) + hq, lq, lk or lq, hq, hkv, d)
    check_prompt(f, q, k, v, cu_q, cu_k, causal)


@pytest.mark.parametrize("d", [64, 128])
def test_prompt_long_and_many(f, d):
    check_prompt(f, *prompt_case(1, [1500], [2900], 4, 1, d))
    check_prompt(f, *prompt_case(2, [2100], [2100], 2, 2, d))
    lens = [int(x) for x in np.random.RandomState(1).randint(0, 60, 200)]
    check_prompt(f, *prompt_case(3, lens, lens, 4, 4, d))


def test_prompt_other_sequences_never_reach_a_row(f):
    """NaN and infinities in every other sequence, and between them: the rows of the rest are as they were."""
    lens = [70, 128, 33, 200, 1, 61]
    q, k, v, cu, _ = prompt_case(4, lens, lens, 8, 2, 128)
    want, lse = check_prompt(f, q, k, v, cu, None)
    at = cu.tolist()
    for i in range(1, 6, 2):
        r = slice(at[i], at[i + 1])
        q[r], k[r], v[r] = math.nan, math.inf, math.nan
        v[at[i]] = -math.inf
    got, lse2 = f.prompt_attention(q, k, v, cu, return_lse=True)
    for i in range(0, 6, 2):
        r = slice(at[i], at[i + 1])
        assert torch.equal(got[r], want[r]) and torch.equal(lse[r], lse2[r])


def test_prompt_sharp_scores_strides_and_streams(f):
    lens = [190, 300]
    qkv = randn(5, 490, 12, 128).bfloat16()
    qkv[:, :4] *= 20                                      # scores in the hundreds: weights underflow, the maximum moves
    qkv[100] = 0
    cu = torch.tensor([0, 190, 490], dtype=torch.int32, device="cuda")
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    out, lse = check_prompt(f, q, k, v, cu, None)
    check_prompt(f, q, k, v, cu, None, scale=-0.2)
    buf = torch.zeros(490, 10, 128, dtype=torch.bfloat16, device="cuda")
    f.prompt_attention(q, k, v, cu, out=buf[:, 1:9])
    assert torch.equal(buf[:, 1:9], out) and (buf[:, 0] == 0).all() and (buf[:, 9] == 0).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(10):
            assert torch.equal(f.prompt_attention(q, k, v, cu), out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = f.prompt_attention(q, k, v, cu)
    g.replay()
    assert torch.equal(o, out)
    # fewer tokens in the same captured call: the offsets are read on the device
    cu.copy_(torch.tensor([0, 17, 100], dtype=torch.int32))
    g.replay()
    assert torch.equal(o[:100], f.prompt_attention(q, k, v, cu)[:100])
    check_prompt(f, q, k, v, cu, None)


@pytest.mark.parametrize("lq,lk,hq,hkv,d", [
    ([1], [6000], 8, 2, 128), ([64], [5003], 16, 1, 128), ([1, 0, 33, 7], [4000, 900, 0, 3333], 8, 4, 64),
    ([300, 20], [2000, 4001], 10, 2, 128), ([700], [1900], 4, 4, 128), ([1300, 1], [1300, 5000], 4, 1, 64),
    ([130] * 3 + [5] * 29, [3000, 2999, 1] + [2000] * 29, 2, 1, 64), ([2], [3000], 128, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_few_rows_over_long_keys(f, lq, lk, hq, hkv, d, causal):
    """Items that several CTAs share."""
    q, k, v, cu_q, cu_k = prompt_case(sum(lk), lq, lk, hq, hkv, d)
    check_prompt(f, q, k, v, cu_q, cu_k, causal)


def test_prompt_shared_items_repeat_and_take_other_values(f):
    q, k, v, cu_q, cu_k = prompt_case(11, [40, 3], [3100, 2500], 8, 2, 128)
    out, lse = check_prompt(f, q, k, v, cu_q, cu_k)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, s = f.prompt_attention(q, k, v, cu_q, cu_k, return_lse=True)
    for _ in range(3):
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o[:43], out[:43]) and torch.equal(s[:43], lse[:43])
    # sharp scores in one part of the keys, the lowest in another; other lengths in the same graph
    k[100:140] *= 30
    k[2000:2100] *= -30
    cu_q.copy_(torch.tensor([0, 1, 43]))
    cu_k.copy_(torch.tensor([0, 2400, 5600]))
    g.replay()
    want, wlse = check_prompt(f, q, k, v, cu_q, cu_k)
    assert torch.equal(o[:43], want[:43]) and torch.equal(s[:43], wlse[:43])
    # a NaN key reaches the rows that see it, in whichever piece it lies
    k[50] = float("nan")
    o2, _ = f.prompt_attention(q, k, v, cu_q, cu_k, return_lse=True)
    assert torch.isnan(o2[0]).any() and torch.equal(o2[1:43], want[1:43])


def test_prompt_empty_and_out_of_range(f):
    q, k, v, cu, _ = prompt_case(6, [40], [40], 4, 2, 64, spare=0)
    assert f.prompt_attention(q[:0], k[:0], v[:0], torch.zeros(1, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)
    out, lse = f.prompt_attention(q, k[:0], v[:0], cu, torch.zeros_like(cu), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    f.prompt_attention(q, k, v, torch.tensor([0, 41], dtype=torch.int32, device="cuda"), cu)
    assert f.device_error(clear=True) & 0xFFFF == 12
    f.prompt_attention(q, k, v, cu, torch.tensor([0, 50], dtype=torch.int32, device="cuda"))
    assert f.device_error(clear=True) & 0xFFFF == 12
    f.prompt_attention(q, k, v, cu, torch.tensor([9, 5], dtype=torch.int32, device="cuda"))
    assert f.device_error(clear=True) & 0xFFFF == 12


# --------------------------------------------------------------- logprobs --
def check_logprobs(f, x, tokens, k):
    r = f.token_logprobs(x, tokens, top_k=k)
    t, v = x.shape
    x64 = x.double()
    p = torch.log_softmax(x64, -1)
    lse = torch.logsumexp(x64, -1)
    rel = (v / 256 + 64) * 2.0 ** -24 + 2.0 ** -20
    bound = lambda y: rel + 2.0 ** -22 * (y.abs() + (lse if y.dim() == 1 else lse[:, None]).abs())  # noqa: E731

    def close(got, want, at):
        same = (got == want) | (got.isnan() & want.isnan())        # -inf and NaN
        assert (same | ((got.double() - want).abs() <= bound(at))).all()

    if tokens is not None:
        given = tokens >= 0
        at = tokens.clamp(min=0)[:, None]
        assert (r.logprobs[~given] == 0).all()
        want = torch.where(given, p.gather(1, at)[:, 0], 0.0)
        close(r.logprobs, want, torch.where(x64.gather(1, at)[:, 0].isfinite(), x64.gather(1, at)[:, 0], 0.0))
    plogp = torch.where(p == -math.inf, 0.0, p.exp() * p)
    ent = -plogp.sum(-1)
    e = (r.entropy.double() - ent).abs()
    assert ((e <= (2 * rel + 2.0 ** -22) * (1 + ent)) | (r.entropy.isnan() & ent.isnan())).all()
    # alternatives: by descending value, then by ascending index
    y = torch.where(x64.isnan(), math.inf, x64).cpu().numpy()
    nan = x64.isnan().cpu().numpy()
    for i in range(t):
        order = np.lexsort((np.arange(v), -y[i], ~nan[i]))[:k]
        assert r.top_ids[i].tolist() == order.tolist()
    if k:
        at = x64.gather(1, r.top_ids)
        close(r.top_logprobs, p.gather(1, r.top_ids), torch.where(at.isfinite(), at, 0.0))
    return r


@pytest.mark.parametrize("t, v, k", [(1, 1, 1), (3, 5, 5), (2, 31, 20), (7, 32, 32), (5, 33, 3), (4, 1000, 0),
                                     (13, 1027, 8), (3, 50257, 20), (1, 151936, 32), (20, 151936, 5), (150, 4099, 7),
                                     (700, 777, 2)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs(f, t, v, k, dtype):
    x = randn(t + v, t, v, scale=3.0).to(dtype)
    tokens = torch.randint(0, v, (t,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(v))
    if t > 2:
        tokens[1] = -100
    check_logprobs(f, x, tokens, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_ties_masks_and_extremes(f, dtype):
    t, v = 12, 20001
    x = randn(5, t, v).round().to(dtype)                  # a handful of distinct values
    x[1] = 0.0
    x[1, 7::3] = -0.0
    x[2] = -math.inf
    x[2, 100:104] = 1.0                                    # fewer tokens left than alternatives
    x[3, 5000:] = -math.inf
    x[4] *= 1e30
    x[5] = -3e38
    x[5, v - 1] = -2.9e38
    x[6] = torch.arange(v, device="cuda").flip(0).to(dtype) / 64    # descending: the first is the largest
    x[7] = torch.arange(v, device="cuda").to(dtype) / 64            # ascending: every value enters the list
    x[8] = -math.inf
    x[9, 17] = math.nan
    x[10, 3] = math.inf
    x[11, v - 1] = 90.0
    tokens = torch.randint(0, v, (t,), device="cuda")
    tokens[2], tokens[3] = 101, 6000                      # a ruled-out token: -inf
    r = check_logprobs(f, x, tokens, 20)
    assert r.logprobs[3] == -math.inf
    for row in (8, 9, 10):
        assert r.logprobs[row].isnan() and r.entropy[row].isnan() and r.top_logprobs[row].isnan().all()
    assert abs(r.entropy[1].item() - math.log(v)) < 1e-4 and r.entropy[11].item() < 1e-3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_logprobs_strides_and_repeats(f, dtype):
    wide = randn(6, 9, 30011).to(dtype)
    for lo, hi in ((0, 30011), (1, 30000), (3, 29999), (7, 12), (5, 4000)):
        x = wide[:, lo:hi]
        tok = torch.randint(0, hi - lo, (9,), device="cuda")
        r = check_logprobs(f, x, tok, min(5, hi - lo))
        s = f.token_logprobs(x.clone(), tok, top_k=min(5, hi - lo))
        assert torch.equal(r.top_ids, s.top_ids)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(r, f.token_logprobs(x, tok, top_k=min(5, hi - lo))))
    check_logprobs(f, wide[2:3, 9:], None, 4)
    assert f.token_logprobs(wide[:0], None, top_k=3).top_ids.shape == (0, 3)


def test_logprobs_token_out_of_range_is_recorded(f):
    x = randn(7, 2, 100)
    r = f.token_logprobs(x, torch.tensor([100, 4], device="cuda"))
    assert f.device_error(clear=True) & 0xFFFF == 12
    assert r.logprobs[0].isnan() and r.logprobs[1].isfinite()


# --------------------------------------------------------------- refusals --
def test_refusals(f):
    kc, vc, table, ln = decode_case(1, [5], 2, 64, 4, torch.bfloat16)
    q = randn(1, 1, 4, 64).bfloat16()
    with pytest.raises(ValueError, match="CUDA"):
        f.paged_decode_attention(q.cpu(), kc, vc, table, ln)
    with pytest.raises(TypeError):
        f.paged_decode_attention(q.float(), kc, vc, table, ln)
    with pytest.raises(TypeError):
        f.paged_decode_attention(q, kc.float(), vc.float(), table, ln)
    with pytest.raises(f.ShapeError):
        f.paged_decode_attention(q[:, :3], kc, vc, table, ln)          # 3 heads over 2
    with pytest.raises(f.ShapeError):
        f.paged_decode_attention(q, kc, vc, table, ln.long())
    with pytest.raises(f.ShapeError):
        f.paged_decode_attention(q, kc, vc, table.long(), ln)
    with pytest.raises(f.ShapeError):
        f.paged_decode_attention(q, kc[..., :32], vc[..., :32], table, ln)
    with pytest.raises(ValueError):
        f.paged_decode_attention(q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, table, ln)
    with pytest.raises(f.Fp8gqError):                                   # rows not in multiples of 16 bytes
        f.paged_decode_attention(torch.zeros(1, 4 * 66, device="cuda", dtype=torch.bfloat16).view(1, 4, 66)[..., :64],
                                 kc, vc, table, ln)
    with pytest.raises(f.ShapeError):
        f.paged_decode_attention(q, kc, vc, table, ln, out=torch.empty(1, 4, 32, device="cuda", dtype=torch.bfloat16))
    x, cu = randn(2, 6, 4, 64).bfloat16(), torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    with pytest.raises(f.ShapeError):
        f.prompt_attention(x, x[:, :3], x[:, :3], cu)
    with pytest.raises(f.ShapeError):
        f.prompt_attention(x, x, x, cu.long())
    with pytest.raises(f.ShapeError):
        f.prompt_attention(x, x, x, cu, cu[:1])
    with pytest.raises(TypeError):
        f.prompt_attention(x.float(), x, x, cu)
    y = randn(3, 4, 40)
    with pytest.raises(f.ShapeError):
        f.token_logprobs(y, None, top_k=33)
    with pytest.raises(f.ShapeError):
        f.token_logprobs(y, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError):
        f.token_logprobs(y.double())
    with pytest.raises(ValueError):
        f.token_logprobs(y.t())
    qkv, pos, slots, cs, kc, vc, qw, kw = append_case(1, 3, 4, 2, 64, 4, torch.bfloat16)
    with pytest.raises(f.ShapeError):
        f.qk_norm_rope_append(qkv[:, :7 * 64], pos, slots, cs, kc, vc)     # 3 query heads over 2
    with pytest.raises(f.ShapeError):
        f.qk_norm_rope_append(qkv, pos[:2], slots, cs, kc, vc)
    with pytest.raises(f.ShapeError):
        f.qk_norm_rope_append(qkv, pos, slots.int(), cs, kc, vc)
    with pytest.raises(f.ShapeError):
        f.qk_norm_rope_append(qkv, pos, slots, cs[:, :32], kc, vc)
    with pytest.raises(f.Fp8gqError):
        f.qk_norm_rope_append(qkv, pos, slots, cs, kc.to(torch.float8_e4m3fn), vc.to(torch.float8_e4m3fn), k_scale=0.0)
