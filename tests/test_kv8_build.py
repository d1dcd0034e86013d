"""Building the PyTorch binding of the 8-bit cache (make -C bz-ggml_b200): the library itself needs no Python. The
compiler and the interpreter are scripts that write down how they were called."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def script(path, text):
    path.write_text("#!/bin/sh\n" + text)
    path.chmod(0o755)
    return str(path)


@pytest.fixture
def tree(tmp_path):
    """A copy of the sources whose library and model writer count as built; make(python) builds the rest."""
    pkg = tmp_path / "pkg"
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    shutil.copytree(os.path.join(ROOT, "bz-ggml_b200", "csrc"), pkg / "csrc")
    shutil.copy(os.path.join(ROOT, "bz-ggml_b200", "Makefile"), pkg)
    (pkg / "bin").mkdir()
    for f in ("libbreeze.so", "bin/breeze-synth"):
        (pkg / f).touch()
    calls = tmp_path / "calls"
    calls.touch()
    cxx = script(tmp_path / "cxx", f'echo "$@" >> {calls}\nwhile [ "$1" != -o ]; do shift; done\ntouch "$2"\n')

    def make(python):
        r = subprocess.run(["make", "-C", str(pkg), "-o", "libbreeze.so", "-o", "bin/breeze-synth", "all", f"PYTHON={python}", f"CXX={cxx}"],
                           capture_output=True, text=True, timeout=300)
        return r, calls.read_text().splitlines()

    return tmp_path, pkg, make


@pytest.mark.parametrize("python", ["without torch", "missing"])
def test_the_library_builds_without_pytorch(tree, python):
    tmp, pkg, make = tree
    path = str(tmp / "nowhere") if python == "missing" else script(tmp / "py", "echo 'No module named torch' >&2\nexit 1\n")
    r, calls = make(path)
    assert r.returncode == 0, r.stderr
    assert "_kv8_torch.so" in r.stderr and "not built" in r.stderr
    assert not calls and not (pkg / "_kv8_torch.so").exists()


def test_a_binding_that_does_not_compile_is_an_error(tree):
    tmp, pkg, make = tree
    script(tmp / "cxx", "exit 1\n")
    r, _ = make(script(tmp / "py", "echo -DFLAGS\n"))
    assert r.returncode != 0


def test_another_interpreter_or_pytorch_builds_the_binding_again(tree):
    tmp, pkg, make = tree
    version = tmp / "version"
    version.write_text("torch 1\n")
    python = script(tmp / "py", f'if [ "$2" = --stamp ]; then cat {version}; else echo -DFLAGS; fi\n')
    assert len(make(python)[1]) == 1
    assert len(make(python)[1]) == 1, "nothing changed"
    version.write_text("torch 2\n")
    assert len(make(python)[1]) == 2
    assert len(make(python)[1]) == 2


def test_the_stamp_names_interpreter_and_pytorch():
    import sys
    import torch
    out = subprocess.run([sys.executable, os.path.join(ROOT, "bz-ggml_b200", "csrc", "torch_flags.py"), "--stamp"], capture_output=True,
                         text=True, check=True).stdout
    assert sys.version.split()[0] in out and torch.__version__ in out
