"""The build's parts do not hang together: a library whose compiler succeeded is put in place, whatever became of
the others, and the build raises with what each of those said."""
import os
import sys

import pytest

from vllm_sly_radiance_amd import build as B


@pytest.fixture
def recipe(monkeypatch, tmp_path):
    """build() with commands that write their output's name, or fail, in place of the compilers."""
    paths = {}
    for name in ("LIB_PATH", "KV4_LIB_PATH", "KV4_TORCH_PATH"):
        paths[name] = str(tmp_path / getattr(B, name).split("/")[-1])
        monkeypatch.setattr(B, name, paths[name])

    def write(path, code=0):
        return [sys.executable, "-c", f"import sys; open({path!r}, 'w').write('new'); print('words of', "
                                      f"{os.path.basename(path)!r}); sys.exit({code})"]
    fail = set()
    monkeypatch.setattr(B, "_command", lambda sources, out: write(out, out[:-4] in fail))
    monkeypatch.setattr(B, "_torch_commands", lambda out: (write(out + ".o", "compile" in fail),
                                                           write(out, "link" in fail)))
    return paths, fail


def built(paths):
    return {n for n, p in paths.items() if os.path.exists(p)}


def test_all(recipe):
    paths, _ = recipe
    assert B.build() == paths["LIB_PATH"] and built(paths) == set(paths)
    assert not [f for f in os.listdir(os.path.dirname(paths["LIB_PATH"])) if ".tmp" in f]


@pytest.mark.parametrize("broken,there", [
    ("compile", {"LIB_PATH", "KV4_LIB_PATH"}), ("link", {"LIB_PATH", "KV4_LIB_PATH"}),
    ("KV4_LIB_PATH", {"LIB_PATH"}), ("LIB_PATH", {"KV4_LIB_PATH", "KV4_TORCH_PATH"})])
def test_one_fails(recipe, broken, there):
    paths, fail = recipe
    fail.add(paths.get(broken, broken))
    with pytest.raises(RuntimeError, match="words of"):
        B.build()
    assert built(paths) == there


@pytest.mark.parametrize("error", [FileNotFoundError("no g++"), ImportError("no torch"), AttributeError("abi")])
def test_no_host_compiler_or_torch(recipe, monkeypatch, error):
    paths, _ = recipe
    if isinstance(error, FileNotFoundError):
        monkeypatch.setattr(B, "_torch_commands", lambda out: (["/nowhere/g++"], ["/nowhere/g++"]))
    else:
        def missing(out):
            raise error
        monkeypatch.setattr(B, "_torch_commands", missing)
    with pytest.raises(RuntimeError, match="_kv4_torch"):
        B.build()
    assert built(paths) == {"LIB_PATH", "KV4_LIB_PATH"}
