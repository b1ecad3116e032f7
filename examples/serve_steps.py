"""A small language model served with fp8gq: prompts, then decode steps.

The model is a stack of pre-norm decoder layers with block-FP8 linears, per-head
q and k norms and grouped query heads (the Qwen3-8B widths by default), with
random weights.  Prompts of different lengths are packed into one batch:

    qkv -> qk_norm_rope_append -> prompt_attention -> o -> gate_up -> down

which leaves their keys and values in a paged cache; then every step takes one
token per sequence through paged_decode_attention, and token_logprobs gives the
next tokens (the likeliest) with their log probabilities.  A step reads its
tokens, positions, slots and lengths from device memory, so one CUDA graph of it
is replayed for all.

    python examples/serve_steps.py [--layers 4] [--steps 32] [--cache e4m3]
"""
import argparse
import sys
from dataclasses import dataclass
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "sglang-triton-fusion_b200"))
import fp8gq  # noqa: E402


@dataclass
class Config:
    layers: int = 4
    hidden: int = 4096
    intermediate: int = 12288
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    vocab: int = 151936
    positions: int = 4096
    page: int = 64
    cache: torch.dtype = torch.bfloat16


def fp8_weight(n, k, gen):
    """A random (n, k) matrix as e4m3 codes with 128 x 128 block scales."""
    w = torch.randn(n, k, device="cuda", generator=gen) * k ** -0.5
    blocks = w.view(n // 128, 128, k // 128, 128)
    s = blocks.abs().amax(dim=(1, 3)) / 448.0
    codes = (blocks / s[:, None, :, None]).view(n, k).to(torch.float8_e4m3fn)
    return codes, s.contiguous()


def norm_linear(h, res, norm, w):
    """linear(rmsnorm(h + res)) and the new residual: one kernel for a decode batch."""
    if len(h) <= 16:
        return fp8gq.fused_add_rmsnorm_gemv_quant(h, res, norm, *w)
    y, res = fp8gq.add_rmsnorm(h, res, norm)
    return fp8gq.fused_gemv_quant(y, *w), res


class Model:
    def __init__(self, cfg: Config, seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        c = self.cfg = cfg

        def norm(n, at=1.0):
            return (at + 0.1 * torch.randn(n, device="cuda", generator=g)).bfloat16()

        self.embed = torch.randn(c.vocab, c.hidden, device="cuda", generator=g).bfloat16()
        self.layers = [dict(
            norm1=norm(c.hidden), qkv=fp8_weight((c.heads + 2 * c.kv_heads) * c.head_dim, c.hidden, g),
            q_norm=norm(c.head_dim, 1.5), k_norm=norm(c.head_dim, 1.5),
            o=fp8_weight(c.hidden, c.heads * c.head_dim, g),
            norm2=norm(c.hidden), gate_up=fp8_weight(2 * c.intermediate, c.hidden, g),
            down=fp8_weight(c.hidden, c.intermediate, g)) for _ in range(c.layers)]
        self.norm, self.lm_head = norm(c.hidden), fp8_weight(c.vocab, c.hidden, g)
        angle = torch.arange(c.positions, device="cuda")[:, None] * 10000.0 ** (
            -torch.arange(c.head_dim // 2, device="cuda") * 2.0 / c.head_dim)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous()

    def forward(self, tokens, positions, slots, cache, attend):
        """tokens, positions, slots int64 [T] -> logits (T, vocab).  ``attend(q,
        k, v, layer's cache)`` is the attention; k and v are the new tokens'."""
        c = self.cfg
        h = self.embed[tokens]
        res = torch.zeros_like(h)
        for w, (kc, vc) in zip(self.layers, cache.kv):
            qkv, res = norm_linear(h, res, w["norm1"], w["qkv"])
            q, k = fp8gq.qk_norm_rope_append(qkv, positions, slots, self.cos_sin, kc, vc, q_weight=w["q_norm"],
                                             k_weight=w["k_norm"], return_k=True)
            v = qkv.view(-1, c.heads + 2 * c.kv_heads, c.head_dim)[:, c.heads + c.kv_heads:]
            a = attend(q, k, v, kc, vc)
            h = fp8gq.fused_gemv_quant(a.view(-1, c.heads * c.head_dim), *w["o"])
            gu, res = norm_linear(h, res, w["norm2"], w["gate_up"])
            h = fp8gq.fused_swiglu_q_gemm(gu, *w["down"])
        return norm_linear(h, res, self.norm, self.lm_head)[0]

    def prompt(self, prompts, cache):
        """Token lists -> logits of all their tokens, packed in order.  The
        sequences' keys and values are in the cache afterwards."""
        lens = [len(p) for p in prompts]
        tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
        positions = torch.tensor([i for n in lens for i in range(n)], device="cuda")
        slots = torch.cat([cache.slots(b, torch.arange(n, device="cuda")) for b, n in enumerate(lens)])
        cu = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        cache.lens.copy_(torch.tensor(lens))
        return self.forward(tokens, positions, slots, cache, lambda q, k, v, kc, vc: fp8gq.prompt_attention(q, k, v, cu))

    def step(self, tokens, cache):
        """One more token (int64 [B]) of each sequence -> logits (B, vocab)."""
        b = torch.arange(len(tokens), device="cuda")
        at = cache.lens.long()
        cache.lens += 1
        return self.forward(tokens, at, cache.slots(b, at), cache,
                            lambda q, k, v, kc, vc: fp8gq.paged_decode_attention(q, kc, vc, cache.table, cache.lens))


class Cache:
    """Pages of keys and values of every layer; the sequences' pages lie in any order."""

    def __init__(self, cfg: Config, sequences, most):
        self.page, per = cfg.page, -(-most // cfg.page)
        shape = (sequences * per, cfg.page, cfg.kv_heads, cfg.head_dim)
        self.kv = [tuple(torch.zeros(shape, dtype=cfg.cache, device="cuda") for _ in "kv") for _ in range(cfg.layers)]
        self.table = torch.randperm(sequences * per, device="cuda").view(sequences, per).to(torch.int32)
        self.lens = torch.zeros(sequences, dtype=torch.int32, device="cuda")

    def slots(self, b, at):
        return self.table[b, at // self.page].long() * self.page + at % self.page


def generate(model, prompts, steps, graph=True):
    """The likeliest continuations: (tokens [B, steps], their log probabilities)."""
    cache = Cache(model.cfg, len(prompts), max(map(len, prompts)) + steps + 1)
    last = torch.tensor([len(p) for p in prompts], device="cuda").cumsum(0) - 1
    first = fp8gq.token_logprobs(model.prompt(prompts, cache)[last], top_k=1)
    tokens, logprobs = [first.top_ids[:, 0]], [first.top_logprobs[:, 0]]
    now = tokens[0].clone()

    def step():
        best = fp8gq.token_logprobs(model.step(now, cache), top_k=1)
        now.copy_(best.top_ids[:, 0])
        return now, best.top_logprobs[:, 0]

    run = step
    if graph:
        start, side = (cache.lens.clone(), now.clone()), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()                                 # scratch is made outside the graph
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        cache.lens.copy_(start[0])                 # (what the first call wrote to the cache is written again)
        now.copy_(start[1])

        def run():
            g.replay()
            return out
    for _ in range(steps - 1):
        t, lp = run()
        tokens.append(t.clone())
        logprobs.append(lp.clone())
    return torch.stack(tokens, 1), torch.stack(logprobs, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--cache", choices=["bf16", "e4m3"], default="bf16")
    args = ap.parse_args()
    cfg = Config(layers=args.layers, cache=torch.bfloat16 if args.cache == "bf16" else torch.float8_e4m3fn)
    model = Model(cfg)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(cfg.vocab, (n,), generator=gen).tolist() for n in (5, 130, 777, 1500)]
    tokens, logprobs = generate(model, prompts, args.steps)
    torch.cuda.synchronize()
    if fp8gq.device_error():
        raise RuntimeError(f"device error {fp8gq.device_error():#x}")
    for b, p in enumerate(prompts):
        print(f"prompt of {len(p)}: {tokens[b, :8].tolist()} ... sum of log probabilities {logprobs[b].sum():.2f}")
    # the same sequences as prompts: what the steps said of each token, scored in one pass
    whole = [p + t[:-1] for p, t in zip(prompts, tokens.tolist())]
    logits = model.prompt(whole, Cache(cfg, len(whole), max(map(len, whole))))
    at = 0
    for b, p in enumerate(prompts):
        rows = logits[at + len(p) - 1:at + len(whole[b])]
        diff = (fp8gq.token_logprobs(rows, tokens[b]).logprobs - logprobs[b]).abs().max()
        print(f"prompt of {len(p)}: steps and one pass differ by {diff:.3f} at most")
        at += len(whole[b])


if __name__ == "__main__":
    main()
