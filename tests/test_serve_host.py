"""The serving operators' host side without a GPU: stand-ins for CUDA tensors, the
library and the device guard."""
import contextlib

import pytest
import torch

fp8gq = pytest.importorskip("fp8gq")
from fp8gq import serve  # noqa: E402


def on(index):
    """The class of CPU tensors that say they are on cuda:index."""
    class Elsewhere(torch.Tensor):
        is_cuda = True
        device = torch.device("cuda", index)
    return Elsewhere


class Lib:
    """Records each entry point's arguments and the device that was current."""

    def __init__(self):
        self.current, self.calls = 0, []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, self.current, args))
            return 4096 if name.endswith("workspace_bytes") else 0
        return call


@pytest.fixture
def lib(monkeypatch):
    """The library and torch's allocation and device guard, replaced; the binding steps aside."""
    lib = Lib()

    @contextlib.contextmanager
    def device(d):
        before, lib.current = lib.current, d.index
        yield
        lib.current = before

    class Native:
        def __getattr__(self, name):
            return lambda *args: None
    empty = torch.empty
    monkeypatch.setattr(serve, "_native", Native())
    monkeypatch.setattr(serve._lib, "load", lambda *a: lib)
    monkeypatch.setattr(torch, "empty", lambda *s, device=None, **kw: empty(*s, **kw).as_subclass(on(device.index)))
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(serve, "_stream", lambda dev: 1000 + dev.index)
    monkeypatch.setattr(serve, "_workspace_entry", lambda dev, n, s: (None, 1 << 20, n))
    monkeypatch.setattr(serve, "_decode_ws_bytes", {})
    return lib


def operands(name):
    """Positional operands of an operator (CPU tensors)."""
    b, i, f = torch.bfloat16, torch.int32, torch.float32
    cache = [torch.zeros(3, 4, 2, 64, dtype=b) for _ in "kv"]
    if name == "qk_norm_rope_append":
        return [torch.zeros(5, 8 * 64, dtype=b), torch.zeros(5, dtype=torch.int64), torch.zeros(5, dtype=torch.int64),
                torch.zeros(9, 64, dtype=f), *cache]
    if name == "paged_decode_attention":
        return [torch.zeros(5, 4, 64, dtype=b), *cache, torch.zeros(5, 2, dtype=i), torch.zeros(5, dtype=i)]
    if name == "prompt_attention":
        return [torch.zeros(5, 4, 64, dtype=b), torch.zeros(5, 2, 64, dtype=b), torch.zeros(5, 2, 64, dtype=b),
                torch.zeros(2, dtype=i), torch.zeros(2, dtype=i)]
    return [torch.zeros(5, 40, dtype=f), torch.zeros(5, dtype=torch.int64)]


NAMES = ["qk_norm_rope_append", "paged_decode_attention", "prompt_attention", "token_logprobs"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("index", [0, 1])
def test_runs_on_the_tensors_device(lib, name, index):
    getattr(fp8gq, name)(*[t.as_subclass(on(index)) for t in operands(name)])
    assert any(c[0] == f"fp8gq_{name}" and c[2][-1] == 1000 + index for c in lib.calls)
    assert all(c[1] == index for c in lib.calls) and lib.current == 0


@pytest.mark.parametrize("name", NAMES)
def test_operands_on_two_devices_are_refused(lib, name):
    n = len(operands(name))
    for at in range(n):
        ts = [t.as_subclass(on(1 if i == at else 0)) for i, t in enumerate(operands(name))]
        with pytest.raises(ValueError, match="one device"):
            getattr(fp8gq, name)(*ts)
    ts = [t.as_subclass(on(0)) for t in operands(name)]
    out = torch.zeros(5, 4, 64, dtype=torch.bfloat16).as_subclass(on(1))
    if name != "token_logprobs":
        with pytest.raises(ValueError, match="one device"):
            getattr(fp8gq, name)(*ts, **{"q_out" if name == "qk_norm_rope_append" else "out": out})
    if name == "qk_norm_rope_append":
        for kw in ("q_weight", "k_weight"):
            with pytest.raises(ValueError, match="one device"):
                fp8gq.qk_norm_rope_append(*ts, **{kw: torch.ones(64, dtype=torch.bfloat16).as_subclass(on(1))})
    assert not lib.calls


EMPTY = torch.empty          # (the fixture replaces it)


def huge(*shape, dtype):
    return EMPTY(*shape, dtype=dtype, device="meta").as_subclass(on(0))


def test_sizes_past_32_bits_are_refused(lib):
    """The entry points take 32-bit sizes; a larger one must not be cut to its low bits."""
    n, b, i = 2 ** 32 + 5, torch.bfloat16, torch.int32
    for x in (huge(n, 1, dtype=b), huge(1, n, dtype=torch.float32), huge(3, 2 ** 31, dtype=b)):
        with pytest.raises(fp8gq.ShapeError, match="2.31"):
            fp8gq.token_logprobs(x)
    q, kc, vc, table, lens = [t.as_subclass(on(0)) for t in operands("paged_decode_attention")]
    with pytest.raises(fp8gq.ShapeError, match="2.31"):
        fp8gq.paged_decode_attention(q, kc, vc, huge(5, n, dtype=i), lens)
    with pytest.raises(fp8gq.ShapeError, match="2.31"):
        fp8gq.paged_decode_attention(q, huge(1, n, 2, 64, dtype=b), huge(1, n, 2, 64, dtype=b), table, lens)
    big = huge(n, 2, 64, dtype=b)
    with pytest.raises(fp8gq.ShapeError, match="2.31"):
        fp8gq.prompt_attention(q, big, big, *[t.as_subclass(on(0)) for t in operands("prompt_attention")[3:]])
    qkv, pos, slots, cs, kc, vc = [t.as_subclass(on(0)) for t in operands("qk_norm_rope_append")]
    with pytest.raises(fp8gq.ShapeError, match="2.31"):
        fp8gq.qk_norm_rope_append(huge(n, 8 * 64, dtype=b), huge(n, dtype=torch.int64), huge(n, dtype=torch.int64), cs, kc, vc)
    assert not lib.calls


def test_rows_that_32_bit_loops_cannot_walk_are_refused():
    from fp8gq import _lib
    a = 1 << 20
    for v, want in ((2 ** 31 - 1, 8), (2 ** 31 - 100, 8)):
        assert _lib.load().fp8gq_token_logprobs(a, v, 0, a, 1, v, a, a, a, a, 1, None) == want
