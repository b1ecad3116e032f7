"""The example that runs the serving operators together (examples/serve_steps.py)."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("serve_steps", Path(__file__).parent.parent / "examples/serve_steps.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def small(ex, **kw):
    return ex.Config(**dict(dict(layers=2, hidden=512, intermediate=1024, heads=8, kv_heads=2, head_dim=64, vocab=1024,
                                 positions=512, page=16), **kw))


def prompts(vocab, lens):
    g = torch.Generator().manual_seed(3)
    return [torch.randint(vocab, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("kw", [dict(), dict(head_dim=128, heads=4, page=5), dict(cache=torch.float8_e4m3fn)])
def test_steps_agree_with_one_pass(ex, kw):
    """The steps' log probabilities against those of the same tokens as prompts.

    The logits have a deviation of about 1.  The two paths round differently (bf16
    values, half an ulp 2^-8), which moves 1 in 16 of a linear's e4m3 inputs (steps
    of 2^-3 at most) to the next code: 2^-5 rms of a linear's input, through 2
    layers of 4 linears about 0.09 rms at the logits.  An e4m3 cache adds roundings
    of 2^-4 at most, 2^-5 rms, of k and v to the steps alone, so about as much
    again.  A token at a wrong place, slot or length changes them by about 1."""
    cfg = small(ex, **kw)
    model = ex.Model(cfg)
    ps = prompts(cfg.vocab, (1, 17, 60, 200))
    tokens, logprobs = ex.generate(model, ps, 12)
    whole = [p + t[:-1] for p, t in zip(ps, tokens.tolist())]
    logits = model.prompt(whole, ex.Cache(cfg, len(ps), max(map(len, whole))))
    at, diffs = 0, []
    for b, p in enumerate(ps):
        rows = logits[at + len(p) - 1:at + len(whole[b])]
        diffs.append(ex.fp8gq.token_logprobs(rows, tokens[b]).logprobs - logprobs[b])
        at += len(whole[b])
    d = torch.cat(diffs)
    assert d.square().mean().sqrt() < 0.25 and d.abs().max() < 0.9
    assert ex.fp8gq.device_error() == 0


def test_graph_and_calls_give_the_same(ex):
    cfg = small(ex)
    model = ex.Model(cfg)
    ps = prompts(cfg.vocab, (3, 50, 128))
    a, b = ex.generate(model, ps, 10), ex.generate(model, ps, 10, graph=False)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_page_order_does_not_matter(ex):
    """Each run draws the order of the pages anew."""
    cfg = small(ex)
    model = ex.Model(cfg)
    ps = prompts(cfg.vocab, (40, 40, 40, 40))
    one, again = ex.generate(model, ps, 8), ex.generate(model, ps, 8)
    assert torch.equal(one[0], again[0]) and torch.equal(one[1], again[1])
