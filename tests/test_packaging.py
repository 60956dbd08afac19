"""What an installed package holds of the extension on PyTorch's headers: it is found there, without a compiler."""
import importlib.util
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _module(path):
    spec = importlib.util.spec_from_file_location("installed_build", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.fixture
def installed(tmp_path):
    """The package's native folder as installation lays it out, from a tree in which the extension (of no content here) was built."""
    native = tmp_path / "tree" / "ipex_llm_b200" / "native"
    shutil.copytree(os.path.join(ROOT, "ipex_llm_b200", "native", "torch"), native / "torch")
    for name in ("__init__.py", "build.py"):
        shutil.copy(os.path.join(ROOT, "ipex_llm_b200", "native", name), native)
    shutil.copy(os.path.join(ROOT, "ipex_llm_b200", "__init__.py"), native.parent)
    shutil.copy(os.path.join(ROOT, "setup.py"), tmp_path / "tree")

    def compiled(cmd, **kw):
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
    tree = _module(native / "build.py")
    tree.subprocess = type("", (), {"check_call": staticmethod(compiled)})
    assert tree.build_calls() == str(native / "libipex_calls.so")
    subprocess.run([sys.executable, "setup.py", "-q", "build_py", "-d", str(tmp_path / "site")], cwd=tmp_path / "tree", check=True,
                   capture_output=True)
    return tmp_path / "site" / "ipex_llm_b200" / "native"


def test_the_extension_is_found_without_a_compiler(installed):
    def none(*a, **kw):
        raise OSError("there is no compiler")
    site = _module(installed / "build.py")
    site.subprocess = type("", (), {"check_call": staticmethod(none)})
    assert site.build_calls() == str(installed / "libipex_calls.so")
    # another patch release of Python, or build of it, takes extensions of the same version
    site.sys = type("", (), {"version": "another"})
    assert site.build_calls() == str(installed / "libipex_calls.so")
    # of another PyTorch, or changed sources, it is not the one
    with open(installed / "torch" / "calls.cpp", "a") as f:
        f.write("// changed\n")
    with pytest.raises(OSError, match="no compiler"):
        site.build_calls()
