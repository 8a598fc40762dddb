"""The module of native calls: what build and import do where it cannot be had."""
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
