"""The module of native calls: what build and import do where it cannot be had."""
import sys

import pytest

pytest.importorskip("torch")

from webgllm_b200 import build  # noqa: E402


@pytest.fixture
def target(monkeypatch, tmp_path):
    """build_host into a folder of its own, where an older module lies."""
    monkeypatch.setattr(build, "HOST", tmp_path / "_host.so")
    monkeypatch.setattr(build, "OBJ_DIR", tmp_path)
    build.HOST.write_bytes(b"older")
    (tmp_path / "host_torch").write_text("older")
    return tmp_path


@pytest.mark.parametrize("compiler", ["/nonexistent/c++", "false"])
def test_no_compiler_or_a_failed_one_leaves_the_python_calls(target, monkeypatch, capfd, compiler):
    """The library is built all the same: build_host reports, and leaves no
    module of another build behind."""
    monkeypatch.setenv("CXX", compiler)
    assert build.build_host() is None
    assert not build.HOST.exists() and "not built" in capfd.readouterr().err


def test_headers_that_are_missing(target, monkeypatch, capfd):
    """As with a torch without CUDA, or a Python without its headers."""
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": "/nonexistent"})
    assert build.build_host() is None
    assert not build.HOST.exists() and "not built" in capfd.readouterr().err


def test_a_module_of_another_torch_is_not_used(monkeypatch):
    """After an upgrade without a rebuild the module would read the new torch's
    tensors by the old one's layout: it is left alone, before any call."""
    from types import SimpleNamespace

    import webgllm_b200
    from webgllm_b200 import q4

    def used(*args):
        raise AssertionError("bound")

    for built_for in ("2.0.0 3.12", "", build.host_target().replace(" ", "x ")):
        old = SimpleNamespace(built_for=built_for, bind=used)
        monkeypatch.setitem(sys.modules, "webgllm_b200._host", old)
        monkeypatch.setattr(webgllm_b200, "_host", old, raising=False)
        assert q4.host_calls.__wrapped__() is None
    old = SimpleNamespace(bind=used)  # from before modules said so
    monkeypatch.setitem(sys.modules, "webgllm_b200._host", old)
    monkeypatch.setattr(webgllm_b200, "_host", old, raising=False)
    assert q4.host_calls.__wrapped__() is None


def test_the_module_says_what_it_is_built_for():
    from webgllm_b200 import q4

    host = q4.host_calls()
    if host is None:
        pytest.skip("webgllm_b200._host is not built")
    assert host.built_for == build.host_target()
