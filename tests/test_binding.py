"""The serving operators' C++ binding: of one torch and Python, and not needed."""
import pytest
import torch

pytest.importorskip("fp8gq")
from fp8gq import _build, _lib, serve  # noqa: E402


@pytest.fixture
def binding(monkeypatch):
    """A binding that was not loaded yet."""
    monkeypatch.setattr(serve, "_native", serve._Binding())
    return monkeypatch


def check_steps_aside():
    with pytest.warns(RuntimeWarning, match="without their C[+][+] binding"):
        assert serve._native.token_logprobs(None, None, 0) is None
    for name in ("qk_norm_rope_append", "paged_decode_attention", "prompt_attention", "token_logprobs"):
        assert getattr(serve._native, name)(1, 2, 3) is None         # and says so once


def test_no_compiler(binding, tmp_path):
    binding.setattr(_build, "native_path", lambda: tmp_path / "none.so")
    binding.setattr(_build, "_native_command", lambda target: [str(tmp_path / "no-such-compiler"), target])
    check_steps_aside()


def test_compiler_fails(binding, tmp_path):
    binding.setattr(_build, "native_path", lambda: tmp_path / "none.so")
    binding.setattr(_build, "_native_command", lambda target: ["false"])
    check_steps_aside()


def test_file_that_does_not_load(binding, tmp_path):
    bad = tmp_path / "bad.so"
    bad.write_bytes(b"not a library")
    binding.setattr(_build, "native_path", lambda: bad)
    check_steps_aside()


def test_another_torch_has_another_binding(monkeypatch):
    here = _build.native_path()
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    assert _build.native_path() != here and not _build.native_up_to_date()


def test_library_loads_without_a_compiler_for_the_binding(monkeypatch, tmp_path):
    _lib.load()                                    # (there and current from here on)
    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_build, "native_path", lambda: tmp_path / "none.so")
    monkeypatch.setattr(_build, "_native_command", lambda target: pytest.fail("the library needs no binding"))
    assert _lib.load().fp8gq_version() == 2


def test_binding_loads(binding):
    assert serve._native.token_logprobs(None, None, 0) is None
    assert serve._native.__name__ == "_serve_native"
