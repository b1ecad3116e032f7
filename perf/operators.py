"""Cases of the attention and scoring operators of a decoder's serving step.

Four operators that stand between the block-FP8 linears of a Qwen3-class decoder:

  append   per-head RMS norm and rotary positions of q and k, k and v written into the paged cache
  decode   attention of one new token per sequence over the paged cache
  prompt   causal attention over packed prompts, optionally behind a prefix
  score    log probabilities of given tokens, entropy and top alternatives from the lm_head's logits

``listed()`` gives the fixed cases, ``draw(rng)`` more of the same ranges.  ``run(state)`` is one
call: the plain torch form, or, where ``own`` is set, the framework's.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
PKG = str(Path(__file__).resolve().parent.parent / "sglang-triton-fusion_b200")


def listed():
    return [
        # one decode step of 24 sequences, Qwen3-8B heads, e4m3 cache in pages of 16: a call of a few microseconds
        dict(name="append-decode-24-e4m3", op="append", tokens=24, hq=32, hkv=8, d=128, page=16, cache="e4m3"),
        # a long prompt of odd length written into a bf16 cache in pages of 64
        dict(name="append-prompt-6001", op="append", tokens=6001, hq=32, hkv=8, d=128, page=64, cache="bf16"),
        # one user at the start of an answer: latency only
        dict(name="decode-1x333", op="decode", batch=1, length=333, lens="equal", hq=32, hkv=8, d=128, page=16,
             cache="bf16"),
        # a server's running batch: lengths from 1 to 6000, padded rows among them
        dict(name="decode-48-ragged-6000", op="decode", batch=48, length=6000, lens="ragged", hq=32, hkv=8, d=128,
             page=64, cache="bf16"),
        # a few long documents over an e4m3 cache: the split of a long axis
        dict(name="decode-8x32768-e4m3", op="decode", batch=8, length=32768, lens="equal", hq=32, hkv=8, d=128,
             page=32, cache="e4m3"),
        # many short chats on one tensor-parallel shard: 64-wide heads, groups of 8, token-granular cache
        dict(name="decode-128-ragged-d64", op="decode", batch=128, length=2047, lens="ragged", hq=16, hkv=2, d=64,
             page=1, cache="bf16"),
        # prompts of a batch of chats, packed: lengths from 1 to 700
        dict(name="prompt-8-ragged-700", op="prompt", batch=8, length=700, lens="ragged", prefix=0, hq=32, hkv=8,
             d=128, causal=True),
        # one long document
        dict(name="prompt-1x8192", op="prompt", batch=1, length=8192, lens="equal", prefix=0, hq=32, hkv=8, d=128,
             causal=True),
        # chunks of prompts behind a prefix already computed, 64-wide heads
        dict(name="prompt-4-chunks-prefix-5003", op="prompt", batch=4, length=1024, lens="ragged", prefix=5003, hq=16,
             hkv=4, d=64, causal=True),
        # the sampled token of one decode step
        dict(name="score-1-bf16", op="score", rows=1, vocab=151936, dtype="bf16", top=5, masked=False),
        # a decode batch under a grammar's mask, fp32 logits, the most alternatives an API returns
        dict(name="score-37-fp32-masked", op="score", rows=37, vocab=151936, dtype="fp32", top=20, masked=True),
        # every token of a prompt scored
        dict(name="score-2048-bf16", op="score", rows=2048, vocab=151936, dtype="bf16", top=8, masked=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prompt", "prompt", "score"])
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8, 16])
    d = rng.choice([64, 128])
    hq = hkv * group
    while hq > 32:                       # the listed cases have at most 32 query heads
        hq -= hkv
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 6000), hq=hq, hkv=hkv, d=d, page=rng.choice([1, 16, 32, 64, 128]),
                    cache=rng.choice(["bf16", "e4m3"]))
    if op == "decode":
        cache = rng.choice(["bf16", "e4m3"])
        batch = _log(rng, 1, 128)
        # at most the key-value bytes of the largest listed case
        most = min(32768, 8 * 32768 * 8 * 128 // (batch * hkv * d * (2 if cache == "bf16" else 1)))
        return dict(op=op, batch=batch, length=_log(rng, 1, max(2, most)), lens=rng.choice(["equal", "ragged"]), hq=hq,
                    hkv=hkv, d=d, page=rng.choice([1, 16, 32, 64, 128]), cache=cache)
    if op == "prompt":
        batch = _log(rng, 1, 16)
        length = _log(rng, 1, 8192 // batch)
        prefix = rng.choice([0, 0, _log(rng, 1, 6000 // batch)])
        causal = rng.random() < 0.8
        # at most the work of the largest listed case
        while batch * length * (prefix + length / (2 if causal else 1)) * hq * d > 8192 * 4096 * 32 * 128:
            length = length * 3 // 4
        return dict(op=op, batch=batch, length=length, lens=rng.choice(["equal", "ragged"]), prefix=prefix, hq=hq,
                    hkv=hkv, d=d, causal=causal)
    vocab = rng.choice([_log(rng, 1000, 151936), 50257, 151936])
    dtype = rng.choice(["bf16", "fp32"])
    return dict(op=op, rows=_log(rng, 1, 2048 if dtype == "bf16" else 1024), vocab=vocab, dtype=dtype,
                top=rng.choice([0, 1, 5, 20]), masked=rng.random() < 0.3)


def _lens(case):
    """The sequences' lengths: of the case alone, so that work() knows them."""
    n, most = case["batch"], case["length"]
    if case["lens"] == "equal":
        return [most] * n
    r = random.Random(1000003 * n + most)
    lens = [_log(r, 1, most) if r.random() < 0.5 else r.randint(1, most) for _ in range(n)]
    lens[r.randrange(n)] = most
    if n > 3 and case["op"] == "decode":                    # rows that pad a batch
        lens[lens.index(min(lens))] = 0
    return lens


def _cache_dtype(case):
    return torch.bfloat16 if case["cache"] == "bf16" else torch.float8_e4m3fn


def _randn(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    s = dict(case)
    if op == "score":
        x = _randn(g, case["rows"], case["vocab"], scale=2.5)
        # a few likely tokens stand out, as in a trained model's answer
        hot = torch.randint(0, case["vocab"], (case["rows"], 12), generator=g, device=DEV)
        x.scatter_add_(1, hot, _randn(g, case["rows"], 12).abs() * 6 + 4)
        if case["masked"]:
            x.masked_fill_(torch.rand(case["rows"], case["vocab"], generator=g, device=DEV) < 0.7, -math.inf)
        s["logits"] = x if case["dtype"] == "fp32" else x.to(torch.bfloat16)
        s["tokens"] = torch.where(torch.rand(case["rows"], generator=g, device=DEV) < 0.7, hot[:, 0],
                                  torch.randint(0, case["vocab"], (case["rows"],), generator=g, device=DEV))
        return s
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "append":
        n, page = case["tokens"], case["page"]
        pages = (n + page - 1) // page + 2
        s["qkv"] = _randn(g, n, (hq + 2 * hkv) * d).to(torch.bfloat16)
        s["qw"] = (1 + 0.2 * _randn(g, d)).to(torch.bfloat16)
        s["kw"] = (1 + 0.2 * _randn(g, d)).to(torch.bfloat16)
        most = 8192
        f = 1e6 ** (-torch.arange(0, d // 2, device=DEV, dtype=torch.float64) * 2 / d)
        a = torch.arange(most, device=DEV, dtype=torch.float64)[:, None] * f[None]
        s["cos_sin"] = torch.cat([a.cos(), a.sin()], 1).float()
        s["positions"] = torch.randint(0, most, (n,), generator=g, device=DEV)
        slots = torch.randperm(pages * page, generator=g, device=DEV)[:n]
        if n > 8:                                           # padding of a captured step: not stored
            slots[torch.randint(0, n, (1,), generator=g, device=DEV)] = -1
        s["slots"] = slots
        s["k_scale"], s["v_scale"] = (0.05, 0.03) if case["cache"] == "e4m3" else (1.0, 1.0)
        s["kc"] = _randn(g, pages, page, hkv, d).to(_cache_dtype(case))
        s["vc"] = _randn(g, pages, page, hkv, d).to(_cache_dtype(case))
        return s
    lens = _lens(case)
    if op == "decode":
        page = case["page"]
        need = [(n + page - 1) // page for n in lens]
        total = sum(need) + 3
        width = max(need) + 1
        ids = torch.randperm(total, generator=g, device=DEV)[:sum(need)].to(torch.int32)
        first = torch.tensor([0] + need, device=DEV).cumsum(0)[:-1]
        col = torch.arange(width, device=DEV)[None]
        held = col < torch.tensor(need, device=DEV)[:, None]
        at = (first[:, None] + col).clamp(max=max(0, sum(need) - 1))
        s["table"] = torch.where(held, ids[at], torch.full_like(ids[at], -1)).contiguous()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["q"] = _randn(g, len(lens), hq, d, scale=1.5).to(torch.bfloat16)
        s["k_scale"], s["v_scale"] = (0.02, 0.015) if case["cache"] == "e4m3" else (1.0, 1.0)
        kc = torch.empty(total, page, hkv, d, dtype=_cache_dtype(case), device=DEV)
        vc = torch.empty_like(kc)
        kc.copy_(_randn(g, total, page, hkv, d).div_(s["k_scale"]).clamp_(-448, 448))
        vc.copy_(_randn(g, total, page, hkv, d).div_(s["v_scale"]).clamp_(-448, 448))
        s["kc"], s["vc"] = kc, vc
        return s
    lk = [n + case["prefix"] for n in lens]
    cu = lambda v: torch.tensor([0] + v, device=DEV).cumsum(0).to(torch.int32)  # noqa: E731
    s["cu_q"], s["cu_k"] = cu(lens), cu(lk)
    # q, k and v as the qkv linear leaves them: views of one buffer where their lengths agree
    if case["prefix"] == 0:
        qkv = _randn(g, sum(lens), hq + 2 * hkv, d).to(torch.bfloat16)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    else:
        s["q"] = _randn(g, sum(lens), hq, d).to(torch.bfloat16)
        s["k"] = _randn(g, sum(lk), hkv, d).to(torch.bfloat16)
        s["v"] = _randn(g, sum(lk), hkv, d).to(torch.bfloat16)
    s["most_q"], s["most_k"] = max(lens), max(lk)
    return s


def _package():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import fp8gq
    return fp8gq


def run(s):
    op = s["op"]
    if own:
        f = _package()
        if op == "append":
            q = f.qk_norm_rope_append(s["qkv"], s["positions"], s["slots"], s["cos_sin"], s["kc"], s["vc"],
                                      q_weight=s["qw"], k_weight=s["kw"], k_scale=s["k_scale"], v_scale=s["v_scale"])
            return {"q": q, "k_cache": s["kc"], "v_cache": s["vc"]}
        if op == "decode":
            o, lse = f.paged_decode_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], k_scale=s["k_scale"],
                                              v_scale=s["v_scale"], return_lse=True)
            return {"out": o, "lse": lse}
        if op == "prompt":
            o, lse = f.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["causal"],
                                        return_lse=True)
            return {"out": o, "lse": lse}
        r = f.token_logprobs(s["logits"], s["tokens"], top_k=s["top"])
        return {"logprob": r.logprobs, "entropy": r.entropy, "top_id": r.top_ids, "top_logprob": r.top_logprobs}
    return {"append": _append, "decode": _decode, "prompt": _prompt, "score": _score}[op](s)


def _append(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    x = s["qkv"].view(-1, hq + 2 * hkv, d).float()
    cos, sin = s["cos_sin"][s["positions"]][:, None].chunk(2, dim=-1)

    def turned(y, w):
        y = y * (y.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.float()
        a, b = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    q, k, v = turned(x[:, :hq], s["qw"]), turned(x[:, hq:hq + hkv], s["kw"]), x[:, hq + hkv:]
    if s["cache"] == "e4m3":
        k, v = (k / s["k_scale"]).clamp(-448, 448), (v / s["v_scale"]).clamp(-448, 448)
    held = s["slots"] >= 0
    at = s["slots"][held]
    for c, y in ((s["kc"], k), (s["vc"], v)):
        bits = torch.uint8 if c.dtype == torch.float8_e4m3fn else torch.int16
        c.view(bits).view(-1, hkv, d)[at] = y.to(c.dtype).view(bits)[held]
    return {"q": q.to(torch.bfloat16), "k_cache": s["kc"], "v_cache": s["vc"]}


def _attend(q, k, v, seen, scale):
    """q [B,Lq,Hq,D], k and v [B,Lk,Hkv,D] in 32 bits, seen [B,Lq,Lk]: (out [B,Lq,Hq,D], lse [B,Lq,Hq])."""
    b, lq, hq, d = q.shape
    hkv = k.shape[2]
    x = torch.matmul(q.view(b, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d), k.permute(0, 2, 3, 1))
    x = x.view(b, hkv, hq // hkv, lq, -1).mul_(scale).masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    z = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hkv, -1, x.shape[-1]), v.permute(0, 2, 1, 3)).view(b, hkv, hq // hkv, lq, d)
    o = torch.where(z == 0, 0.0, o / z)
    lse = (m + z.log()).squeeze(-1)
    return o.permute(0, 3, 1, 2, 4).reshape(b, lq, hq, d), lse.permute(0, 3, 1, 2).reshape(b, lq, hq)


def _decode(s):
    page = s["page"]
    j = torch.arange(s["length"], device=DEV)
    seen = j[None] < s["lens"][:, None]
    at = s["table"].long()[:, j // page] * page + j % page
    at = torch.where(seen, at, 0)

    def taken(c, scale):
        return c.view(-1, s["hkv"], s["d"])[at].float().mul_(scale)

    o, lse = _attend(s["q"].float()[:, None], taken(s["kc"], s["k_scale"]), taken(s["vc"], s["v_scale"]), seen[:, None],
                     s["d"] ** -0.5)
    return {"out": o[:, 0].to(torch.bfloat16), "lse": lse[:, 0]}


def _prompt(s):
    cq, ck = s["cu_q"].long(), s["cu_k"].long()
    lq, lk = cq.diff(), ck.diff()
    i, j = torch.arange(s["most_q"], device=DEV), torch.arange(s["most_k"], device=DEV)
    row, col = i[None] < lq[:, None], j[None] < lk[:, None]
    seen = row[:, :, None] & col[:, None]
    if s["causal"]:
        seen &= j[None, None] <= (i[None] + (lk - lq)[:, None])[:, :, None]
    ai = torch.where(row, cq[:-1, None] + i[None], 0)
    aj = torch.where(col, ck[:-1, None] + j[None], 0)
    o, lse = _attend(s["q"].float()[ai], s["k"].float()[aj], s["v"].float()[aj], seen, s["d"] ** -0.5)
    return {"out": o[row].to(torch.bfloat16), "lse": lse[row]}


def _score(s):
    x, tok = s["logits"].float(), s["tokens"]
    n, v = x.shape
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    y = x - m
    ent = z.log()[:, 0] - torch.where(e == 0, 0.0, e * y).sum(-1) / z[:, 0]
    # unique keys: the value's bits in the order of the values, then the lowest index first
    b = (x + 0.0).view(torch.int32).long()
    b = torch.where(b < 0, b ^ 0x7FFFFFFF, b)
    key = b * (1 << 32) + (v - 1 - torch.arange(v, device=DEV))[None]
    top = v - 1 - (key.topk(s["top"], dim=-1, sorted=True).values & 0xFFFFFFFF) if s["top"] else tok.new_empty(n, 0)
    return {"logprob": (x.gather(1, tok[:, None]) - lse)[:, 0], "entropy": ent, "top_id": top,
            "top_logprob": x.gather(1, top) - lse}


def work(case):
    op = case["op"]
    if op == "score":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * (2 if case["dtype"] == "bf16" else 4) + n * (16 + 12 * case["top"]), "flops": 5 * n * v}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "append":
        n, c = case["tokens"], 2 if case["cache"] == "bf16" else 1
        return {"bytes": n * ((hq + 2 * hkv) * d * 2 + hq * d * 2 + 2 * hkv * d * c + 16) + min(n, 8192) * d * 4,
                "flops": n * (hq + hkv) * d * 7}
    lens = _lens(case)
    if op == "decode":
        c = 2 if case["cache"] == "bf16" else 1
        page = case["page"]
        return {"bytes": sum(2 * n * hkv * d * c + 4 * ((n + page - 1) // page) for n in lens)
                + len(lens) * (4 * hq * d + 4 * hq + 4), "flops": 4 * d * hq * sum(lens)}
    p = case["prefix"]
    pairs = sum(n * p + n * (n + 1) // 2 if case["causal"] else n * (n + p) for n in lens)
    return {"bytes": sum(n * hq * (4 * d + 4) + (n + p) * hkv * d * 4 for n in lens), "flops": 4 * d * hq * pairs}


def exact(case, seed):
    """The same from the definitions, in 64 bits, sequence by sequence and head by head."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "score":
        rows = []
        for x, tok in zip(s["logits"].split(64), s["tokens"].split(64)):
            p = torch.log_softmax(x.double(), -1)
            rows.append((p.gather(1, tok[:, None])[:, 0], -torch.special.xlogy(p.exp(), p.exp()).sum(-1),
                         p.sort(dim=-1, descending=True).values[:, :case["top"]]))
        a, b, c = (torch.cat(t) for t in zip(*rows))
        return {"logprob": a, "entropy": b, "top_id": None, "top_logprob": c}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if op == "append":
        x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
        half = d // 2
        c = s["cos_sin"].double()[s["positions"]]
        z = torch.complex(c[:, :half], c[:, half:])[:, None]

        def turned(y, w):
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / d + 1e-6) * w.double()
            y = torch.complex(y[..., :half], y[..., half:]) * z
            return torch.cat([y.real, y.imag], -1)

        if case["cache"] == "e4m3":
            return {"q": turned(x[:, :hq], s["qw"]), "k_cache": None, "v_cache": None}
        kc, vc = s["kc"].double().view(-1, hkv, d), s["vc"].double().view(-1, hkv, d)
        held = s["slots"] >= 0
        kc[s["slots"][held]] = turned(x[:, hq:hq + hkv], s["kw"])[held]
        vc[s["slots"][held]] = x[:, hq + hkv:][held]
        return {"q": turned(x[:, :hq], s["qw"]), "k_cache": kc.view(s["kc"].shape), "v_cache": vc.view(s["vc"].shape)}
    lens = _lens(case)
    outs, lses = [], []
    for i, n in enumerate(lens):
        if op == "decode":
            q = s["q"][i:i + 1]
            ids = s["table"][i, :(n + case["page"] - 1) // case["page"]].long()
            k = s["kc"][ids].view(-1, hkv, d)[:n].double() * s["k_scale"]
            v = s["vc"][ids].view(-1, hkv, d)[:n].double() * s["v_scale"]
        else:
            q = s["q"][s["cu_q"][i]:s["cu_q"][i + 1]]
            k, v = (s[t][s["cu_k"][i]:s["cu_k"][i + 1]].double() for t in "kv")
        o = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
        lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
        for h in range(hq if len(k) else 0):
            x = q[:, h].double() @ k[:, h * hkv // hq].T / math.sqrt(d)
            if op == "prompt" and case["causal"]:
                x += torch.full_like(x, -math.inf).triu(len(k) - len(q) + 1)
            lse[:, h] = torch.logsumexp(x, -1)
            o[:, h] = torch.softmax(x, -1) @ v[:, h * hkv // hq]
        outs.append(o)
        lses.append(lse)
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
